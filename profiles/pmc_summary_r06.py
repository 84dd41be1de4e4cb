#!/usr/bin/env python3
"""Summary of the counter passes of profiles/collect_r06_pmc.sh -> profiles/pmc_shipped.json (the shipped kernels; r06_pmc.json: an earlier state).

    pmc_summary_r06.py <folder of the passes>  [> profiles/pmc_shipped.json]

Round 6 re-collects every family on the round's code (the recalibration kernel is new: np_recalibrate_half_kernel).  Round 5 added the families the round-4 review missed: the event detector of the from-raw / eventalign steps
(np_ed_peaks_par_kernel<true> -- the fused t-statistics + peak walk --, np_ed_check_kernel, np_ed_events_kernel, np_mom_fill_kernel; unit =
raw SAMPLE) and the rewritten glue kernels (np_build_map_kernel, np_recalibrate_kernel, np_resolve_kernel; unit = read), otherwise as round 4:

Per kernel family (event_align = np_event_align_kernel, hmm_forward = every size class of np_hmm_forward_kernel in the call-methylation
step, hmm_forward_variants = the same kernels on the variants screening shape, chain = np_eventalign_chain2_kernel): counter totals per
launch, instructions per unit of work (band / HMM call / segment; the units come from tools/pmc_workload.py's own JSON lines), HBM bytes
per unit (FETCH_SIZE x 2, WRITE_SIZE x 1: the gfx950 corrections calibrated in round 1, tools/hbm_counter_calib.hip), and the
VECTOR-ISSUE UTILISATION the round-3 review asked for, from counters a reader can recompute:

    valu_issue_floor  = SQ_INSTS_VALU per launch x FAST / (UNPROFILED launch time x 2.4 GHz x 1024 SIMDs)
    valu_issue_priced = SQ_INSTS_VALU per launch x MEAN / (the same)

FAST (2.49 cycles) is the issue time of a wave-instruction in the fastest class a SIMD sustains with eight waves resident
(profiles/r04_valu_calibration.json, gpurun r04l: v_add/sub/mul_f32, v_and/or_b32, v_mov_b32, 32-bit integer add; the guide's 2 cycles plus
the loop overhead of the stream).  Every vector instruction costs at least that, so `valu_issue_floor` is a LOWER bound of the fraction of
time the vector port is busy.  MEAN prices each instruction by its own class: conversions, compares, selects, maxima, shifts, DPP, everything
64-bit and ANY instruction with a scalar-register source 4.37 cycles, packed fp32 4.85, lane reads 4.51, fma 2.56 (same calibration), with
the class mix read off the kernel's loops in the generated assembly (tools/issue_cost.py, static: every loop block counts once) -- an
ESTIMATE of the busy fraction, good to a few per cent (it reads 1.03 for the variants shape of kernel B, where the true figure cannot
exceed 1).  SQ_ACTIVE_INST_VALU ticks ONCE per instruction whatever its class, so rocprof's VALUBusy formula (x 4 cycles) is an instruction
rate, not a busy time: round 3's "49.5 %" was neither.  The first calibration of this round (gpurun r04a: 3.74 / 6.3 cycles) ran ten waves
per CU instead of 32 (16 KB of LDS per one-wave workgroup) and overstated every cost 1.5 x; `profiles/r04_kernel_b_staged.md`'s closing
arithmetic used it and is corrected in DESIGN section 11.
The counter passes slow some kernels (A: ~1.7 x); all times here are the unprofiled ones (the workload's own HIP events in a run without
counters).
"""
import csv
import glob
import json
import os
import subprocess
import sys
from collections import defaultdict

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "tools"))
root = sys.argv[1]
FETCH_CORR, WRITE_CORR, N_SIMD, CLK = 2.0, 1.0, 1024, 2.4e9
_cal = {c["name"]: c["cycles_per_inst_simd"] for c in json.load(open(os.path.join(ROOT, "profiles", "r04_valu_calibration.json")))["classes"]}
FAST_CYCLES = round(sum(_cal[k] for k in ("v_add_f32", "v_sub_f32", "v_mul_f32", "v_and_b32", "v_or_b32", "v_mov_b32", "v_add_u32", "v_sub_u32")) / 8, 2)
FAM = (("event_align", "np_event_align_kernel"), ("hmm_forward", "np_hmm_forward_kernel"), ("chain", "np_eventalign_chain"),
       ("recalibrate", "np_recalibrate_"), ("build_map", "np_build_map_kernel"), ("cm_items", "np_cm_items_kernel"),
       ("cm_groups", "np_cm_groups_kernel"), ("resolve", "np_resolve_"), ("ed_peaks", "np_ed_peaks_par_kernel"), ("ed_check", "np_ed_check_kernel"),
       ("ed_events", "np_ed_events_kernel"), ("mom_fill", "np_mom_fill_kernel"))


def units_of(name):
    try:
        for line in open(os.path.join(root, name)):
            if line.startswith("{"):
                return json.loads(line)
    except OSError:
        pass
    return {}


units, units_var = units_of("units.json"), units_of("units_variants.json")
reps = units.get("reps", 2)
tot = defaultdict(lambda: defaultdict(float))
rows = defaultdict(list)
for f in sorted(glob.glob(root + "/*/**/*counter_collection.csv", recursive=True)):
    var = os.path.basename(os.path.dirname(f)).startswith("var_") or "/var_" in f
    for r in csv.DictReader(open(f)):
        for key, pat in FAM:
            if pat in r["Kernel_Name"]:
                k = "hmm_forward_variants" if (var and key == "hmm_forward") else (None if var else key)
                if k:
                    rows[(k, f)].append((int(r["Dispatch_Id"]), r["Counter_Name"], float(r["Counter_Value"])))
for (key, f), lst in rows.items():
    ids = sorted({d for d, _, _ in lst})
    # the workload runs the call-methylation step first, then the eventalign step, which launches kernel A again on ITS batch (more
    # events per read): only the call-methylation launches (the first `reps` dispatches) are normalised by that step's bands
    keep = set(ids[:reps]) if key == "event_align" else set(ids)
    for d, name, v in lst:
        if d in keep:
            tot[key][name] += v

# class mix of the kernels' loops from the assembly of the tree the summary runs in
mix = {}
try:
    import issue_cost
    tmp = "/tmp/np_pmc_summary"
    os.makedirs(tmp, exist_ok=True)
    for unit, pats in (("np_align_kernel", {"event_align": "np_event_align_kernelE"}),
                       ("np_hmm_kernels", {"hmm_forward": "np_hmm_forward_kernelILi2ELi8ELi512ELb1", "hmm_forward_variants": "np_hmm_forward_kernelILi3ELi8ELi512ELb1"}),
                       ("np_eventalign_kernel", {"chain": "ea_fill2ILi3"}), ("np_events_kernels", {"ed_peaks": "np_ed_peaks_par_kernelILb1"})):
        sfile = os.path.join(tmp, unit + ".s")
        subprocess.run(["/opt/rocm/bin/hipcc", "-O3", "-std=c++17", "-fPIC", "-ffp-contract=off", "-fno-slp-vectorize", "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops", "--offload-arch=gfx950", "-S", "--cuda-device-only",
                        os.path.join(ROOT, "nanopolish_amd", "csrc", unit + ".hip"), "-o", sfile], check=True, capture_output=True)
        for key, pat in pats.items():
            mix[key] = issue_cost.loop_mix(sfile, pat)
except Exception as e:  # noqa: BLE001
    mix["error"] = repr(e)

out = {"source": "rocprofv3 --kernel-trace --pmc over tools/pmc_workload.py (profiles/collect_r06_pmc.sh), pass folder %s" % root.rstrip("/").split("/")[-1],
       "units": units, "units_variants": units_var, "fetch_size_correction": FETCH_CORR, "write_size_correction": WRITE_CORR,
       "fast_class_cycles_per_instruction": FAST_CYCLES, "calibration": "profiles/r04_valu_calibration.json"}
cm, ea, va = units.get("call_methylation", {}), units.get("eventalign", {}), units_var.get("variants", {})
for key, c in tot.items():
    d = {}
    per = {k: v / reps for k, v in c.items()}
    for name, v in sorted(per.items()):
        d[name + "_per_step"] = v
    if per.get("SQ_WAVE_CYCLES"):
        wc = per["SQ_WAVE_CYCLES"]
        for nm in ("SQ_WAIT_ANY", "SQ_WAIT_INST_ANY", "SQ_ACTIVE_INST_ANY", "SQ_ACTIVE_INST_VALU", "SQ_ACTIVE_INST_SCA"):
            if nm in per:
                d[nm.lower() + "_over_wave_cycles"] = round(per[nm] / wc, 4)
    if per.get("SQ_LDS_IDX_ACTIVE") and "SQ_LDS_BANK_CONFLICT" in per:
        d["lds_bank_conflict_frac"] = round(per["SQ_LDS_BANK_CONFLICT"] / per["SQ_LDS_IDX_ACTIVE"], 4)
        if per.get("SQ_INSTS_LDS"):
            d["lds_cycles_per_lds_inst"] = round(per["SQ_LDS_IDX_ACTIVE"] / per["SQ_INSTS_LDS"], 3)
    fb = per["FETCH_SIZE"] * 1024 * FETCH_CORR if "FETCH_SIZE" in per else None
    wb = per["WRITE_SIZE"] * 1024 * WRITE_CORR if "WRITE_SIZE" in per else None
    unit, ms = None, None
    if key == "event_align" and cm.get("bands"):
        unit = ("band", cm["bands"]); d["reads_per_launch"] = cm["reads"]; d["algo_bytes_per_band"] = cm["algo_bytes_align"] / cm["bands"]
        ms = cm["unprofiled_ms"]["event_align"]
    elif key == "hmm_forward" and cm.get("hmm_calls"):
        unit = ("call", cm["hmm_calls"]); d["algo_bytes_per_call"] = cm["hmm_algo_bytes"] / cm["hmm_calls"]; ms = cm["unprofiled_ms"]["hmm_forward"]
    elif key == "hmm_forward_variants" and va.get("calls"):
        unit = ("call", va["calls"]); d["algo_bytes_per_call"] = va["algo_bytes"] / va["calls"]; ms = va["unprofiled_ms"]
    elif key == "chain" and ea.get("segments"):
        unit = ("segment", ea["segments"]); d["reads_per_launch"] = ea["reads"]; ms = ea["unprofiled_chain_ms"]
        d["algo_bytes_per_segment"] = (ea["lattice_cells"] + 4 * ea["lattice_rows"] + 2 * ea["lattice_kmers"] + 9 * ea["rows_out"]) / ea["segments"]
    elif key in ("ed_peaks", "ed_check", "ed_events", "mom_fill") and ea.get("raw_samples"):
        unit = ("sample", ea["raw_samples"]); d["reads_per_launch"] = ea["reads"]; ms = (ea.get("unprofiled_ms") or {}).get(key)
    elif key in ("recalibrate", "build_map", "resolve", "cm_items", "cm_groups") and cm.get("reads"):
        # (the eventalign step launches build_map / recalibrate on its batch too: per read of BOTH steps)
        unit = ("read", cm["reads"] + (ea.get("reads", 0) if key in ("recalibrate", "build_map") else 0))
    if unit:
        nm, n = unit
        for cname, label in (("SQ_INSTS_VALU", "valu"), ("SQ_INSTS_SALU", "salu"), ("SQ_INSTS_LDS", "lds"), ("SQ_INSTS_VMEM_RD", "vmem_rd"),
                             ("SQ_INSTS_VMEM_WR", "vmem_wr"), ("SQ_INSTS_SMEM", "smem")):
            if cname in per:
                d["%s_per_%s" % (label, nm)] = round(per[cname] / n, 3)
        if fb is not None:
            d["fetch_bytes_per_%s" % nm] = round(fb / n, 3)
        if wb is not None:
            d["write_bytes_per_%s" % nm] = round(wb / n, 3)
        if ms:
            d["unprofiled_ms_per_launch"] = ms
            simd_cycles = ms * 1e-3 * CLK * N_SIMD
            d["simd_cycles_per_%s" % nm] = round(simd_cycles / n, 2)
            if "SQ_INSTS_VALU" in per:
                d["valu_issue_floor"] = round(per["SQ_INSTS_VALU"] * FAST_CYCLES / simd_cycles, 4)
                if key in mix:
                    d["valu_issue_priced"] = round(per["SQ_INSTS_VALU"] * mix[key]["mean_cycles"] / simd_cycles, 4)
                    d["loop_class_mix"] = mix[key]
    out[key] = d
json.dump(out, sys.stdout, indent=1)
print()
