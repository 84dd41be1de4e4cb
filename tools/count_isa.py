#!/usr/bin/env python3
"""Static instruction counts of kernel A's FAST pair loop, from the assembly hipcc generates:

    hipcc -O3 -std=c++17 -ffp-contract=off --offload-arch=gfx950 -Iinclude -Inanopolish_amd/csrc -S --cuda-device-only \
          nanopolish_amd/csrc/np_align_kernel.hip -o /tmp/align.s && python tools/count_isa.py /tmp/align.s

The pair loop is the innermost loop that contains the `s_min_u32 ..., 0xff7fffff` of the even band's move decision.  Its
basic blocks are classified by what they do (straight band code; the right-move update; the eight-slot re-target; the trace
store), counted per class, and weighted: a right move in 0.405 of the bands ((K + 51) / (E + K + 2) for the bench's reads), a
re-target in one right move of eight, a trace store in one band of eight (one pair of four).  Prints one JSON object."""
import json
import re
import sys

lines = open(sys.argv[1]).read().splitlines()
anchor = next(i for i, l in enumerate(lines) if "s_min_u32" in l and "0xff7fffff" in l)
# the loop: from its header label (first label above the anchor that a later s_branch / s_cbranch jumps back to) to that branch
labels = {m.group(1): i for i, l in enumerate(lines) for m in [re.match(r"^(\.LBB\d+_\d+):", l)] if m}
head = None
for i in range(anchor, 0, -1):
    m = re.match(r"^(\.LBB\d+_\d+):", lines[i])
    if m and "Inner Loop Header" in lines[i + 2]:
        head = i; name = m.group(1); break
end = max(i for i, l in enumerate(lines) if re.search(r"s_c?branch\S*\s+" + re.escape(name) + r"\b", l) and i > anchor)
body = lines[head:end + 1]

def klass(op):
    if op.startswith(("v_readlane", "v_writelane")): return "lane"
    if op.startswith("v_cmpx"): return "valu"
    if op.startswith("v_"): return "valu"
    if op.startswith(("s_waitcnt", "s_nop", "s_setprio")): return "wait"
    if op.startswith(("s_cbranch", "s_branch")): return "branch"
    if op.startswith(("s_load", "s_buffer")): return "smem"
    if op.startswith("s_"): return "salu"
    if op.startswith(("buffer_", "global_", "flat_", "scratch_")): return "vmem"
    if op.startswith("ds_"): return "lds"
    return None

# split into blocks at labels; tag blocks
blocks, cur = [], []
for l in body:
    if re.match(r"^\.LBB", l):
        if cur: blocks.append(cur)
        cur = []
    t = l.strip()
    if not t or t.startswith(";") or t.startswith("."): continue
    cur.append(t.split()[0])
if cur: blocks.append(cur)
# a fall-through block continues until a branch: split blocks further at conditional branches so that the conditional parts
# (right move, re-target, store) can be told apart
parts, cur = [], []
for b in blocks:
    for op in b:
        cur.append(op)
        if op.startswith(("s_cbranch", "s_branch")):
            parts.append(cur); cur = []
    if cur: parts.append(cur); cur = []

def tag(p):
    s = " ".join(p)
    if "v_cmpx" in s: return "retarget"
    if "s_bitcmp1_b32" in s and "s_cselect_b64" in s: return "right_move"
    if "buffer_store_dword" in s: return "trace_store"
    if sum(o.startswith("v_") for o in p) > 20: return "band"
    return "glue"

W = dict(band=1.0, glue=None, right_move=0.405, retarget=0.405 / 8, trace_store=1.0 / 8)
out = {"loop": name, "parts": []}
tot = {}
for p in parts:
    t = tag(p)
    c = {}
    for op in p:
        k = klass(op)
        if k: c[k] = c.get(k, 0) + 1
    out["parts"].append(dict(tag=t, **c))
    # per-band weights: a `band` or `glue` part runs once per pair (1/2 per band); a right-move / re-target part exists once per
    # band position and runs with the probability of its event (p / 2 per band each, two positions); the trace store exists in
    # the second position only and runs once per four pairs
    w = 0.5 if t in ("band", "glue") else (0.125 if t == "trace_store" else W[t] / 2)
    for k, v in c.items():
        tot[k] = tot.get(k, 0.0) + w * v
out["per_band"] = {k: round(v, 2) for k, v in sorted(tot.items())}
out["note"] = "weights: band / glue parts 1/2 (once per pair), right move 0.405, re-target 0.405/8, trace store 1/8 (per band position, two positions)"
print(json.dumps(out, indent=1))
