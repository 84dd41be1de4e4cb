"""The eventalign segment chain on the device (np_eventalign_dev, csrc/np_eventalign_kernel.hip) against the oracle's chain
(oracle/workloads.py:eventalign_read over npo_profile_hmm_align), in every form of the kernel: three k-mer blocks per lane at both register
budgets, four blocks (the direct-RNA model), a segment whose back-track outgrows the list that LDS holds, odd numbers of reads, reads of one
segment, both strands."""
import os

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
HERE = os.path.dirname(os.path.abspath(__file__))


def _oracle_rows(orc, model, k, rd, events, batch, i, rds, monkeypatch, lens=None):
    """the chain on the oracle, from what the device holds for read i: its event alignment and its scalings"""
    import oracle.workloads as W
    monkeypatch.setattr(W, "K", k)
    pairs = batch.pairs_of(i)
    epb = float(batch.epb()[i])
    S = orc.scalings(float(rds["shift"][i]), float(rds["scale"][i]), float(rds["var"][i]))

    def align(fwd, rc_s, e1, e2, stride, rc):
        r = orc.hmm_align(model, S, events, orc.sequence_kmer_ranks("nucleotide", fwd, rc_s, k, rc), e1, e2, stride, epb)
        if r is not None and lens is not None:
            lens.append(len(r[0]))
        return r

    rows, n_calls, _ = W.eventalign_read(orc, dict(seq=rd["seq"], rc=rd["rc"]), pairs, align)
    return rows, n_calls


def _check(got, want, n_calls):
    assert got["status"] == 0 and got["n_calls"] == n_calls
    assert list(zip(got["ref_position"].tolist(), got["event_idx"].tolist(), got["hmm_state"].tolist())) == want


def _records(reads):
    from nanopolish_amd import api
    out = []
    for r in reads:
        ref = api.reverse_complement("nucleotide", r["seq"]) if r["rc"] else r["seq"]
        rec = {f: r[f] for f in ("events", "raw", "shift", "scale", "var") if f in r}
        out.append(dict(rec, seq=r["seq"], rc=int(r["rc"]), pos=0, cigar=api.cigar_words([("M", len(ref))]), contig=ref))
    return out


@pytest.mark.parametrize("waves_per_cu", [16, 20])
@pytest.mark.parametrize("lengths", [[400], [1500, 320, 900], [700, 1100, 260, 1300, 500]], ids=str)
def test_three_blocks_per_lane(models, orc, monkeypatch, waves_per_cu, lengths):
    from nanopolish_amd.api import Context
    from nanopolish_amd.pipeline import build_host_batch_records, CallMethylationBatch
    from nanopolish_amd.synth import synth_read
    ctx = Context(0)
    try:
        ctx.register_model(models["nucleotide"], "nucleotide")
        ctx.set_option("ea_waves_per_cu", waves_per_cu)
        reads = [synth_read(900 + i, models["nucleotide"], L=n) for i, n in enumerate(lengths)]
        hb = build_host_batch_records(models, _records(reads), "", with_jobs=False)
        batch = CallMethylationBatch(ctx, hb, "cuda:0", workload="eventalign")
        batch.step()
        got = batch.eventalign_results()
        rds = batch.reads_scored()
        mn = orc.model(models["nucleotide"])
        for i, rd in enumerate(reads):
            want, n_calls = _oracle_rows(orc, mn, 6, rd, rd["events"], batch, i, rds, monkeypatch)
            assert len(want) > lengths[i] // 2
            _check(got[i], want, n_calls)
    finally:
        ctx.close()


def test_four_blocks_per_lane_direct_rna(ctx, orc, monkeypatch):
    from nanopolish_amd.pipeline import build_host_batch_records, CallMethylationBatch
    from nanopolish_amd.synth import synth_raw_rna
    z = np.load(os.path.join(HERE, "golden", "models_r9.4_70bps_rna.npz"))
    m = dict(k=5, level_mean=z["u_to_t_rna_level_mean"], level_stdv=z["u_to_t_rna_level_stdv"], level_log_stdv=z["u_to_t_rna_level_log_stdv"])
    if "u_to_t_rna" not in ctx.models:
        ctx.register_model(m, "u_to_t_rna")
    reads = [dict(synth_raw_rna(760 + i, m, L=n), rc=0) for i, n in enumerate([700, 420, 1500, 900, 300])]
    for r in reads:
        r.pop("events", None)
    hb = build_host_batch_records({"nucleotide": m}, _records(reads), "", k=5, with_jobs=False)
    batch = CallMethylationBatch(ctx, hb, "cuda:0", calibrate=True, from_raw=True, workload="eventalign", rna=True, base_model="u_to_t_rna")
    batch.step()
    got = batch.eventalign_results()
    rds, cal = batch.reads_scored(), batch.calibrated()
    mo = orc.model(m)
    checked = 0
    for i, rd in enumerate(reads):
        if not cal[i] or len(batch.pairs_of(i)) == 0 or batch.epb()[i] > 5.0:
            assert len(got[i]["event_idx"]) == 0
            continue
        want, n_calls = _oracle_rows(orc, mo, 5, rd, batch.detected(i)[3], batch, i, rds, monkeypatch)
        _check(got[i], want, n_calls)
        checked += len(want)
    assert checked > 2000


def test_a_segment_that_outgrows_the_burst_list(ctx, models, orc, monkeypatch):
    """A stretch of slow translocation: twenty events a base over ~80 bases in a read that averages two.  A burst of walk steps holds ten at
    most, LDS 112 of them: a segment of more than 1 120 states spills its list for certain."""
    from nanopolish_amd.pipeline import build_host_batch_records, CallMethylationBatch
    from nanopolish_amd.synth import synth_read
    nuc = models["nucleotide"]
    rng = np.random.default_rng(17)
    reads = []
    for rid, L, lo in ((930, 1600, 700), (931, 1900, 40), (932, 800, 300)):
        rd = synth_read(rid, nuc, L=L)
        n_ev = rng.integers(1, 3, len(rd["ranks"]))
        if rid != 932:
            n_ev[lo:lo + 80] = 20
        rk = np.repeat(rd["ranks"], n_ev)
        ev = (nuc["level_mean"][rk] + 0.6 * nuc["level_stdv"][rk] * rng.standard_normal(len(rk))).astype(np.float32)
        reads.append(dict(seq=rd["seq"], rc=rd["rc"], events=ev, shift=0.0, scale=1.0, var=1.0))
    hb = build_host_batch_records(models, _records(reads), "", with_jobs=False)
    batch = CallMethylationBatch(ctx, hb, "cuda:0", workload="eventalign")
    batch.step()
    got = batch.eventalign_results()
    rds = batch.reads_scored()
    mn = orc.model(nuc)
    lens = []
    for i, rd in enumerate(reads):
        want, n_calls = _oracle_rows(orc, mn, 6, rd, rd["events"], batch, i, rds, monkeypatch, lens)
        assert len(want) > 500
        _check(got[i], want, n_calls)
    assert max(lens) > 1120
