"""The constants that a host function of the stream forms between two kernels (np_mom_fill_dev, np_resolve_jobs_dev, np_calibrate_resolve_dev,
np_hmm_score_set_combine_dev): large batches (several threads share them), sets of any size, calls in flight behind each other, reads whose
scalings stay as they were, and the refusal of a captured call."""
import ctypes as C
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def _p(t):
    return C.c_void_p(t.data_ptr())


def _fill_records(rng, n):
    from nanopolish_amd.pipeline import READ_DT
    rd = np.zeros(n, READ_DT)
    rd["n_kmers"] = rng.integers(1, 60, n)
    ne = rng.integers(0, 120, n).astype(np.int32)
    rd["event_off"] = np.concatenate([[0], np.cumsum(ne)[:-1]])
    rd["rank_off"] = np.concatenate([[0], np.cumsum(rd["n_kmers"].astype(np.int64))[:-1]])
    return rd, ne


@pytest.mark.parametrize("n", [1, 63, 4097, 40001])
def test_aligner_constants_of_a_batch(ctx, models, orc, n):
    """lp_* of every read, one read to a batch that several threads share, are the process's; a read without events too (log 0 = -inf)."""
    import torch
    from nanopolish_amd.pipeline import READ_DT
    rng = np.random.default_rng(n)
    rd, ne = _fill_records(rng, n)
    ne[0] = 0 if n > 1 else 50
    dev = torch.device("cuda:0")
    up = lambda a: torch.from_numpy(np.ascontiguousarray(a).view(np.uint8).reshape(-1)).to(dev)
    d_rd = up(rd); d_ne = up(ne)
    d_ev = torch.rand(int(ne.sum()) + 64, dtype=torch.float32, device=dev) * 50 + 60
    d_rk = up(rng.integers(0, 4096, int(rd["n_kmers"].sum())).astype(np.uint16))
    torch.cuda.synchronize()
    ctx._chk(ctx.L.np_mom_fill_dev(ctx.h, None, n, _p(d_rd), None, _p(d_ev), _p(d_ne), _p(d_rk), ctx.models["nucleotide"]), "np_mom_fill_dev")
    ctx.sync()
    got = d_rd.cpu().numpy().view(READ_DT)
    pick = np.arange(n) if n < 5000 else rng.integers(0, n, 3000)
    for i in [0, n - 1] + list(pick):
        want = orc.aligner_constants(int(ne[i]), int(rd["n_kmers"][i]))
        assert (got["lp_skip"][i], got["lp_stay"][i], got["lp_step"][i], got["lp_trim"][i]) == want, i
        assert got["n_events"][i] == ne[i]


def test_set_combination_of_any_size(ctx, orc):
    """log n of sets up to thousands of members, empty sets among them, many sets in one call."""
    import torch
    rng = np.random.default_rng(5)
    sizes = np.concatenate([[0, 1, 2, 63, 64, 65, 66, 127, 1000, 4097, 0], rng.integers(1, 9, 9000)])
    off = np.zeros(len(sizes) + 1, np.int64); off[1:] = np.cumsum(sizes)
    sc = (-rng.uniform(100, 140, int(off[-1]))).astype(np.float32)
    dev = torch.device("cuda:0")
    d_off, d_sc = torch.from_numpy(off).to(dev), torch.from_numpy(sc).to(dev)
    d_out = torch.zeros(len(sizes), dtype=torch.float32, device=dev)
    torch.cuda.synchronize()
    ctx._chk(ctx.L.np_hmm_score_set_combine_dev(ctx.h, None, len(sizes), _p(d_off), None, _p(d_sc), _p(d_out)), "np_hmm_score_set_combine_dev")
    ctx.sync()
    got = d_out.cpu().numpy()
    for q in list(range(11)) + list(rng.integers(11, len(sizes), 1500)):
        n = int(sizes[q])
        want = np.float32(orc.combine_score_set(sc[off[q]:off[q + 1]])) if n else np.float32(-np.inf)
        assert got[q] == want, (q, n)
    # no sets: nothing is touched
    ctx._chk(ctx.L.np_hmm_score_set_combine_dev(ctx.h, None, 0, None, None, None, None), "np_hmm_score_set_combine_dev")


def test_reads_that_are_not_rescaled_keep_their_log_var(ctx, models):
    """recalibrate_model leaves a read with too few 'M' events alone (src/nanopolish_methyltrain.cpp:204-306): shift, scale, var AND log_var
    stay what the caller put there; the transitions are formed for it all the same."""
    import torch
    from nanopolish_amd.pipeline import build_host_batch, CallMethylationBatch
    hb = build_host_batch(models, [84, 85, 86, 87], L=[150, 2000, 150, 1200])
    hb["reads_b"] = hb["reads_b"].copy()
    hb["reads_b"]["log_var"] = [0.25, 0.5, 0.75, 1.0]
    before = hb["reads_b"].copy()
    batch = CallMethylationBatch(ctx, hb, "cuda:0", calibrate=True)
    batch.step()
    rds, cal = batch.reads_scored(), batch.calibrated()
    assert list(cal) == [0, 1, 0, 1]
    for i in range(4):
        if cal[i]:
            assert rds["var"][i] != before["var"][i] and rds["log_var"][i] == math.log(rds["var"][i])
        else:
            for f in ("shift", "scale", "var", "log_var"):
                assert rds[f][i] == before[f][i], (i, f)
        from nanopolish_amd import api
        assert np.array_equal(rds["trans"][i], api.calculate_transitions(float(batch.epb()[i])))


def test_calls_in_flight_behind_each_other(ctx, models):
    """Batches of growing and shrinking size, enqueued without a wait in between, on the context's stream and on others: every call's
    constants are its own."""
    import torch
    from nanopolish_amd.pipeline import build_host_batch, tile_host_batch, CallMethylationBatch
    small = build_host_batch(models, [3, 4], L=900, raw=True)
    big = tile_host_batch(build_host_batch(models, [5, 6, 7, 8, 9, 10], L=1100, raw=True), 40)
    mk = lambda hb: CallMethylationBatch(ctx, hb, "cuda:0", calibrate=True, from_raw=True)
    want = []
    for hb in (small, big):
        b = mk(hb); b.step()
        want.append((b.scores(), b.reads_aligned().tobytes(), b.reads_scored().tobytes()))
    streams = [None, torch.cuda.Stream(), torch.cuda.Stream()]
    runs = [(mk(small), 0), (mk(big), 1), (mk(small), 0), (mk(big), 1), (mk(small), 0), (mk(big), 1)]
    for _ in range(2):
        for i, (b, _w) in enumerate(runs):
            st = streams[i % 3]
            b.stream = st.cuda_stream if st is not None else None
            b.step()
    for b, w in runs:
        assert np.array_equal(b.scores(), want[w][0], equal_nan=True)
        assert b.reads_aligned().tobytes() == want[w][1] and b.reads_scored().tobytes() == want[w][2]


def test_a_captured_call_is_refused(ctx, models):
    """A host function's argument block lives for one run: a call on a capturing stream is refused before it enqueues anything, and the
    context goes on working."""
    import torch
    n = 3
    rd, ne = _fill_records(np.random.default_rng(1), n)
    dev = torch.device("cuda:0")
    up = lambda a: torch.from_numpy(np.ascontiguousarray(a).view(np.uint8).reshape(-1)).to(dev)
    d_rd, d_ne = up(rd), up(ne)
    d_ev = torch.rand(400, dtype=torch.float32, device=dev)
    d_rk = up(np.zeros(400, np.uint16)); d_x = torch.zeros(8, device=dev)
    torch.cuda.synchronize()
    g, st = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(g, stream=st):
        d_x.add_(1.0)
        s = C.c_void_p(st.cuda_stream)
        rc = [ctx.L.np_mom_fill_dev(ctx.h, s, n, _p(d_rd), None, _p(d_ev), _p(d_ne), _p(d_rk), ctx.models["nucleotide"]),
              ctx.L.np_hmm_score_set_combine_dev(ctx.h, s, 1, _p(d_rk), None, _p(d_ev), _p(d_x))]
    assert rc == [-4, -4] and "captured" in ctx.L.np_last_error(ctx.h).decode()
    g.replay(); torch.cuda.synchronize()
    assert float(d_x[0]) == 1.0
    ctx._chk(ctx.L.np_mom_fill_dev(ctx.h, None, n, _p(d_rd), None, _p(d_ev), _p(d_ne), _p(d_rk), ctx.models["nucleotide"]), "np_mom_fill_dev")
    ctx.sync()


def test_two_contexts_on_two_threads(models):
    """Two contexts, a host thread each, their steps in flight side by side (ctypes releases the GIL): each forms its own constants."""
    import threading
    from nanopolish_amd.api import Context
    from nanopolish_amd.pipeline import build_host_batch, tile_host_batch, CallMethylationBatch
    hbs = [tile_host_batch(build_host_batch(models, ids, L=1000, raw=True), 30) for ids in ([20, 21, 22], [23, 24, 25, 26])]
    ctxs, batches, want = [], [], []
    for hb in hbs:
        c = Context(0)
        c.register_model(models["nucleotide"], "nucleotide"); c.register_model(models["cpg"], "cpg")
        b = CallMethylationBatch(c, hb, "cuda:0", calibrate=True, from_raw=True)
        b.step()
        ctxs.append(c); batches.append(b); want.append((b.scores(), b.reads_aligned().tobytes(), b.reads_scored().tobytes()))
    errors = []

    def run(b):
        try:
            for _ in range(12):
                b.step()
            b.sync()
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=run, args=(b,)) for b in batches]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert errors == []
    for b, w in zip(batches, want):
        assert np.array_equal(b.scores(), w[0], equal_nan=True) and b.reads_aligned().tobytes() == w[1] and b.reads_scored().tobytes() == w[2]
    for c in ctxs:
        c.close()
