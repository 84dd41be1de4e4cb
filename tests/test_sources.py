"""Rules that the GPU sources follow by themselves, checked on the text (CPU)."""
import ast
import glob
import os
import re
import subprocess

import pytest

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


def _makefile_flags():
    text = open(os.path.join(ROOT, "nanopolish_amd", "csrc", "Makefile")).read()
    return re.search(r"^CXXFLAGS = (.*)$", text, re.M).group(1).replace("$(ARCH)", "gfx950").split()


def test_the_product_is_built_without_packed_fp32(tmp_path):
    """The compiler makes packed fp32 instructions from ordinary float code; the Makefile's flags keep them out of the device code (the event
    detector's translation unit is the one where it finds pairs)."""
    hipcc = "/opt/rocm/bin/hipcc"
    if not os.path.exists(hipcc):
        pytest.skip("no hipcc")
    out = str(tmp_path / "events.s")
    subprocess.run([hipcc] + _makefile_flags() + ["-S", "--cuda-device-only", os.path.join(ROOT, "nanopolish_amd", "csrc", "np_events_kernels.hip"), "-o", out],
                   check=True, capture_output=True)
    text = open(out).read()
    assert "v_add_f32" in text
    assert re.findall(r"\bv_pk_(?:add|mul|fma)_f32\b", text) == []


def test_no_packed_fp32_by_hand():
    for f in _gpu_sources():
        for lit in re.findall(r'"((?:[^"\\\n]|\\.)*)"', open(f).read()):
            assert not re.search(r"\bv_pk_(add|mul|fma)_f32\b", lit), (os.path.relpath(f, ROOT), lit)


def test_streams_keep_the_default_priority():
    """Work on streams of different priorities has hung here for good: no stream or process group asks for one."""
    files = [f for d in ("", "nanopolish_amd", "tools", "tests", "oracle") for f in glob.glob(os.path.join(ROOT, d, "*.py"))]
    assert len(files) > 40
    for f in files:
        for node in ast.walk(ast.parse(open(f).read())):
            if isinstance(node, ast.Call):
                assert not {k.arg for k in node.keywords} & {"priority", "is_high_priority_stream"}, (os.path.relpath(f, ROOT), node.lineno)
    for f in _gpu_sources() + glob.glob(os.path.join(ROOT, "nanopolish_amd", "csrc", "*.cpp")):
        assert "StreamCreateWithPriority" not in open(f).read(), f
