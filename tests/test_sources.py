"""Rules that the GPU sources follow by themselves, checked on the text (CPU)."""
import glob
import os
import re

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DIRS = ["nanopolish_amd/csrc", "tools"]


def _gpu_sources():
    out = []
    for d in DIRS:
        for f in sorted(glob.glob(os.path.join(ROOT, d, "*"))):
            if f.endswith((".hip", ".h")):
                out.append(f)
    assert len(out) >= 8
    return out


def test_scalar_instructions_in_inline_assembly_do_not_write_memory():
    """Inline assembly uses scalar instructions for arithmetic, branches and waits only; memory is written through vector stores.  (The
    pattern names what is allowed: every scalar arithmetic instruction ends in its operand type; a probe's printed
    labels leave it off.)"""
    ok = re.compile(r"s_(mov|add|cmp|cselect|bitcmp1|waitcnt|nop|memtime|branch|cbranch_[a-z0-9]+|[a-z0-9_]+_(b32|b64|i32|u32|i64|u64))")
    for f in _gpu_sources():
        for lit in re.findall(r'"((?:[^"\\\n]|\\.)*)"', open(f).read()):
            if not re.search(r"(^|\\n|\\t|\s)[sv]_[a-z0-9_]+ ", lit + " "):
                continue
            for w in re.findall(r"(?:(?<=^)|(?<=\\n)|(?<=\\t)|(?<=\s))(s_[a-z0-9_]+)", lit):
                assert ok.fullmatch(w), (os.path.relpath(f, ROOT), w)
