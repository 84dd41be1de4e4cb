// np_eventalign_kernel.hip -- the eventalign segment chain on the device: align_read_to_ref
// (src/alignment/nanopolish_eventalign.cpp:612-826) for a batch of reads, two reads per wavefront.
//
// The reference realigns a read to its reference in ~100-base segments.  Every segment is one profile_hmm_align (Viterbi
// fill + back-track, src/hmm/nanopolish_profile_hmm_r9.cpp:73-204, r9.inl:130-197, flags 0) over the events between the
// segment's start event and the closest event of its last aligned base; of the aligned states only the first ~50 are
// emitted, and the next segment starts at the last emitted (event, reference k-mer).  The chain is data-dependent from
// segment to segment but independent between reads, so a persistent wave walks one read's chain from end to end:
//   * segment geometry from the read's CIGAR without materialising aligned pairs (np_cigar.h; get_end_pair :196-205 is a
//     "last aligned pair with ref_pos <= x" search), closest events from the read's event map (np_device.h);
//   * Viterbi fill as an anti-diagonal sweep, two segments (of two reads) per wave, one per half-wave: lane j of a half owns three
//     k-mer blocks (a segment has <= 96 k-mers; four for the k = 5 model), computes row t - j at step t; previous row in registers,
//     left neighbour through DPP; candidates in HMMMovementType order, later index wins ties; only back-pointers leave the wave, seven
//     bits per block, one dword per lane and one 256-byte line per sweep STEP (cell (row r, k-mer b) sits in line r + b / BPL, dword
//     b / BPL of its half), into a per-wave scratch (ea_fill2);
//   * back-track of both halves' segments as vector code over a window of lines staged in LDS, in bursts of steps whose number is known in advance; the visited states go to a per-half list, one 64-bit word per burst
//     (ea_walk2); then a lane per burst replays it and emits (ballots + prefix counts reproduce the reference's "first 50 that are not K
//     and not the start event" cut, ea_emit_segment).
// Output rows are (ref_position relative to the record's pos, event_idx, state 'M'/'B'); ref_kmer / model_kmer of the TSV
// follow from them on the host (nanopolish_amd/eventalign.py).
#include "np_kernels.h"
#include "np_cigar.h"

#define NP_EA_MAX_KMERS 128

namespace {

__device__ __forceinline__ float readlane_f32(float v, int l)
{
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), l));
}

__device__ __forceinline__ uint32_t base_code(char c) { return c == 'C' ? 1u : c == 'G' ? 2u : c == 'T' ? 3u : 0u; }   // disambiguated to ACGT upstream


struct ea_trans { float mm_self, mb, mk, mm_next, bb, bk, bm_next, bm_self, kk, km; };

// ---------------------------------------------------------------------------------------------------------------------------
// Round 3: TWO reads per wave.  A segment has <= 96 k-mers: at two blocks per lane the sweep above keeps 48 of 64 lanes busy and
// spends e + 47 steps per segment.  Here a half-wave (32 lanes) owns a segment at THREE blocks per lane -- 96 k-mers exactly --
// and the two halves sweep two segments of two different reads in the same instruction stream: every lane busy, e + 31 steps,
// the per-step overhead (neighbour exchange, event distribution, store) shared by two segments.  The two chains are independent
// and data-dependent, so everything around the sweep (segment geometry, back-track, emission) is scalar code run for half 0,
// then for half 1; a half whose read is finished pulls the next read from the queue, a half without work sweeps an empty
// segment.  The per-read state that survives from segment to segment is ten integers per half (ea_half); what only depends on
// the read's index is reloaded where it is needed (wave-uniform loads).
// ---------------------------------------------------------------------------------------------------------------------------
// Back-pointers: SEVEN bits per k-mer block, "this candidate is the cell's maximum" for every candidate but each state's first (which is
// the move when no other bit is set; of several set bits the reference's "later index wins" takes the highest candidate).  A bit is the
// sign of (candidate - maximum), shifted into the lane's word: one subtraction and one v_alignbit_b32 per candidate, no lane masks.
//   bits 5 c .. 5 c + 4              block c:  B from its own B;  M from K, B, own B, M to the left (PREV_K, PREV_B, SAME_B, PREV_M)
//   bits 5 BPL + 2 (BPL - 1 - c) ..  block c:  K from PREV_K, PREV_B
// i.e. in every state the bits rise as the candidates' indices fall, and the walk takes the lowest set one.  A line is 64 dwords, 256
// bytes, one coalesced vector store: half h's walk reads its 128-byte half of a line.
// Measured, 50 000 reads from raw signal: 229 ms; with lane masks (a compare per candidate) combined to six bits by scalar logic and added
// into the word with carries 242 ms.
// BPL, the k-mer blocks per lane: a segment spans up to 101 reference bases (eventalign.cpp:695-735), i.e. 102 - k k-mers: 96 for the
// DNA models (k = 6: three blocks on each of a half-wave's 32 lanes), 97 for the direct-RNA model (k = 5): that one k-mer more takes a
// fourth block per lane (np_eventalign_chain2_kernel<WAVES, 4>: the same code, 28 bits of the dword).
#define NP_EA2_LINE_BYTES 256

// Arguments of a (not inlined) device function arrive in vector registers, and the compiler cannot know that they are wave-uniform:
// everything computed from them would become vector code (the back-track as exec-masked vector loops, the argument block read with
// flat loads).  These put a uniform value back into scalar registers.
template <class T> __device__ __forceinline__ T* ea_uniform(T* p)
{
    const uint64_t u = (uint64_t)p;
    const uint32_t lo = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)u), hi = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(u >> 32));
    return (T*)(((uint64_t)hi << 32) | lo);
}
__device__ __forceinline__ float ea_uniform(float v) { return __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, v))); }
__device__ __forceinline__ int ea_uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

struct ea_read {                 // what the chain needs of a read, all derived from its index
    const np_read_dev* rd; const float* ev; const int32_t* ms; const char* ref;
    cig_view cv;
    int K, ref_n, rl; bool rc;
    int64_t o0; int out_cap;
};
__device__ __forceinline__ ea_read ea_load_read(const np_ea_args& a, int ri)
{
    ea_read R;
    R.rd = a.reads + ri;
    R.ev = a.event_mean + R.rd->event_off;
    R.ms = a.map_start + R.rd->rank_off;
    R.K = (int)R.rd->n_kmers;
    R.ref = a.genome + a.ref_begin[ri];
    R.ref_n = a.ref_len[ri];
    R.rl = a.read_len[ri];
    R.rc = a.read_rc[ri] != 0;
    R.cv = cig_view{a.cigar + a.cigar_off[ri], a.op_ref + a.cigar_off[ri] + ri, a.op_read + a.cigar_off[ri] + ri,
                    (int)(a.cigar_off[ri + 1] - a.cigar_off[ri])};
    R.o0 = a.out_off[ri];
    R.out_cap = (int)(a.out_off[ri + 1] - R.o0);
    return R;
}

struct ea_half {                 // chain state of the read a half-wave works on (wave-uniform scalars)
    int ri;                      // -1: no read
    int n_out, n_calls, status;
    int curr_start_event, curr_start_ref, last_event, forward, q_last, r_last;
    // the segment about to be swept / just swept
    int e_start, stride, e, n, last_section;
};

// One k-mer block of one lattice row (the candidates of r9.inl:130-197 in HMMMovementType order, later index wins ties; (lM_r, lB_r,
// lK_r): the block to the left in this row, (lM_p, ...): in the previous row), in two halves so that a step needs no copy of the previous
// row.  The M and B cells of row r read row r-1 of their own block and of the block to the left; K reads row r of the block to the left.
// Sweeping M and B over the lane's blocks in DESCENDING order, in place, every block still finds its left neighbour's row r-1 untouched; K
// then runs ASCENDING, in place, behind the new M and B (and M has already used the old K).  The soft clip (block 0 of row 1) has no bit:
// no other candidate of that cell is finite, its walk takes the move of "no bit set" (SAME_M) to row 0 and ends there.

// x = 2 x + the sign of d, "this candidate is NOT the maximum" (the finished word is complemented): d = candidate - maximum is +0 or
// negative.  (A cell without any path, everything -inf, gets the sign of a NaN: no walk comes there.)
__device__ __forceinline__ uint32_t ea_push(const uint32_t x, const float d) { return __builtin_amdgcn_alignbit(x, __builtin_bit_cast(uint32_t, d), 31); }
template <bool FIRST>
__device__ __forceinline__ void ea_block_mb(float& M, float& B, const float lM_p, const float lB_p, const float lK_p, const float x, const np_gauss& g,
                                            const ea_trans& tr, const float soft, uint32_t& word)
{
    const float em = np_emission(x, g);
    const float a0 = tr.mm_self + M, a1 = tr.mm_next + lM_p, a2 = tr.bm_self + B, a3 = tr.bm_next + lB_p, a4 = tr.km + lK_p;
    float v = __builtin_fmaxf(__builtin_fmaxf(__builtin_fmaxf(__builtin_fmaxf(a0, a1), a2), a3), a4);      // two three-input maxima
    if (FIRST) v = __builtin_fmaxf(v, soft);
    word = ea_push(ea_push(ea_push(ea_push(word, a1 - v), a2 - v), a3 - v), a4 - v);
    const float newM = v + em;
    const float b0 = tr.mb + M, b2 = tr.bb + B;
    const float newB = __builtin_fmaxf(b0, b2);
    word = ea_push(word, b2 - newB);
    M = newM; B = newB;
}
__device__ __forceinline__ void ea_block_k(float& K, const float lM_r, const float lB_r, const float lK_r, const ea_trans& tr, uint32_t& word)
{
    const float k1 = tr.mk + lM_r, k3 = tr.bk + lB_r, k4 = tr.kk + lK_r;
    const float newK = __builtin_fmaxf(__builtin_fmaxf(k1, k3), k4);
    word = ea_push(ea_push(word, k3 - newK), k4 - newK);
    K = newK;
}

struct ea_seg { const float* ev; int e_start, stride, e, n; };

// The sweep of two segments, one per half-wave (e == 0: no segment).  tr, g[]: the lane's half's transitions and the scaled Gaussians
// of the lane's BPL blocks.  Returns the value of (last row, MATCH of the last k-mer) of each segment.
template <int BPL> struct ea_gauss { np_gauss g[BPL]; };
template <int BPL>
__device__ __attribute__((noinline)) float2 ea_fill2(const ea_gauss<BPL> G, const ea_trans tr, const float flank0, const ea_seg s0, const ea_seg s1,
                                                     uint8_t* __restrict__ bp, const int lane)
{
    const int sl = lane & 31;
    const bool hi_half = lane >= 32;
    const int lu0 = (s0.n + BPL - 1) / BPL, lu1 = (s1.n + BPL - 1) / BPL;
    const int steps0 = __builtin_amdgcn_readfirstlane(s0.e > 0 ? s0.e + lu0 - 1 : 0), steps1 = __builtin_amdgcn_readfirstlane(s1.e > 0 ? s1.e + lu1 - 1 : 0);
    const int s_min = steps0 < steps1 ? steps0 : steps1, s_max = steps0 < steps1 ? steps1 : steps0;
    float M[BPL], B[BPL], K[BPL];                                           // row r-1 of this lane's blocks
#pragma unroll
    for (int c = 0; c < BPL; ++c) M[c] = B[c] = K[c] = NP_NEG_INF;
    float oM = NP_NEG_INF, oB = NP_NEG_INF, oK = NP_NEG_INF;                // row r-1 of the block to the left
    // events: lane sl of a half computes row t - sl at step t, i.e. needs event t - 1 - sl of ITS segment: every lane loads its own event
    // of the next step through its half's range-checked descriptor (an index before the segment's first or past its last event reads as
    // 0 and only feeds rows nobody reads), one step ahead.  Both descriptors are scalar, so every lane requests from both and keeps its
    // half's: two loads, two offset additions and one select per step.  (Until round 4 a wave fetched 64 events per 64 steps with one
    // coalesced load, the half's first lane took its event with v_readlane and the others by a DPP shift: two lane reads with a scalar
    // lane select, two scalar-to-vector moves, a shift and a select per step -- 35 issue cycles of the step's ~350; the loads are not
    // vector-ALU instructions.)
    const __amdgpu_buffer_rsrc_t evr0 = make_rsrc(s0.ev + (s0.stride > 0 ? s0.e_start : s0.e_start - (s0.e - 1)), (uint32_t)s0.e * 4u);
    const __amdgpu_buffer_rsrc_t evr1 = make_rsrc(s1.ev + (s1.stride > 0 ? s1.e_start : s1.e_start - (s1.e - 1)), (uint32_t)s1.e * 4u);
    int off0 = s0.stride > 0 ? -4 * sl : 4 * (s0.e - 1 + sl), off1 = s1.stride > 0 ? -4 * sl : 4 * (s1.e - 1 + sl);        // byte offset of event t - 1 - sl at t = 1
    int d0 = s0.stride > 0 ? 4 : -4, d1 = s1.stride > 0 ? 4 : -4;
    asm("" : "+v"(d0), "+v"(d1));                          // (vector registers: an addition with a scalar-register source issues in the slow class)
    float xn;                                             // the lane's event of the NEXT step
    { const float xa = buf_f32(evr0, off0), xb = buf_f32(evr1, off1); xn = hi_half ? xb : xa; }
    // line t - 1: the wave's 64 dwords of step t (device memory by name: through a generic pointer the store would be a flat one, which
    // makes every later wait for an event load a wait for the store too)
    typedef __attribute__((address_space(1))) uint32_t global_u32;
    global_u32* lines = (global_u32*)ea_uniform(bp);
    // the first lane of a half has no left neighbour (block -1 = -inf): instead of a select after the lane shift, the shift ADDS a
    // per-lane constant -- -inf in lanes 0 and 32, else 0 (v + 0 == v for every value the lattice holds, v + -inf == -inf) -- in the
    // same DPP instruction (bound_ctrl: lane 0's missing source reads as 0)
    const float head = sl == 0 ? NP_NEG_INF : 0.0f;
    auto shr_add = [&](const float v) {
        float r;
        asm("v_add_f32_dpp %0, %1, %2 wave_shr:1 row_mask:0xf bank_mask:0xf bound_ctrl:0" : "=v"(r) : "v"(v), "v"(head));
        return r;
    };
    float soft = sl == 0 ? flank0 : NP_NEG_INF;                                  // HMT_FROM_SOFT: block 0 of row 1 only (flags 0)
    auto step = [&](const int t) {
        const float nM = shr_add(M[BPL - 1]), nB = shr_add(B[BPL - 1]), nK = shr_add(K[BPL - 1]);
        const float x = xn;
        off0 += d0; off1 += d1;
        { const float xa = buf_f32(evr0, off0), xb = buf_f32(evr1, off1); xn = hi_half ? xb : xa; }
        uint32_t wm = 0u, wk = 0u;
#pragma unroll
        for (int c = BPL - 1; c >= 1; --c) ea_block_mb<false>(M[c], B[c], M[c - 1], B[c - 1], K[c - 1], x, G.g[c], tr, NP_NEG_INF, wm);
        ea_block_mb<true>(M[0], B[0], oM, oB, oK, x, G.g[0], tr, soft, wm);
        ea_block_k(K[0], nM, nB, nK, tr, wk);
#pragma unroll
        for (int c = 1; c < BPL; ++c) ea_block_k(K[c], M[c - 1], B[c - 1], K[c - 1], tr, wk);
        oM = nM; oB = nB; oK = nK;
        soft = NP_NEG_INF;
        const uint32_t word = ~((wk << (5 * BPL)) | wm);          // set: the candidate IS the maximum
        lines[(size_t)(t - 1) * (NP_EA2_LINE_BYTES / 4) + lane] = word;
    };
    int t = 1;
    for (; t + 1 <= s_min; t += 2) { step(t); step(t + 1); }      // two steps per iteration: the values a step hands to the next need no move back to fixed registers
    for (; t <= s_min; ++t) step(t);
    // the segment with fewer steps has just computed its last row in the lane that owns its last k-mer: keep that row (the lanes
    // go on computing rows nobody reads)
    float zM[BPL];
#pragma unroll
    for (int c = 0; c < BPL; ++c) zM[c] = M[c];
    for (; t + 1 <= s_max; t += 2) { step(t); step(t + 1); }
    for (; t <= s_max; ++t) step(t);
    const int ec_0 = s0.n > 0 ? (s0.n - 1) % BPL : 0, ec_1 = s1.n > 0 ? (s1.n - 1) % BPL : 0;
    const int my_ec = hi_half ? ec_1 : ec_0;
    float live = M[0], snap = zM[0];
#pragma unroll
    for (int c = 1; c < BPL; ++c) { live = my_ec == c ? M[c] : live; snap = my_ec == c ? zM[c] : snap; }
    const int el0 = s0.n > 0 ? (s0.n - 1) / BPL : 0, el1 = 32 + (s1.n > 0 ? (s1.n - 1) / BPL : 0);
    float2 out;
    out.x = s0.e > 0 ? readlane_f32(steps0 == s_max ? live : snap, el0) : NP_NEG_INF;
    out.y = s1.e > 0 ? readlane_f32(steps1 == s_max ? live : snap, el1) : NP_NEG_INF;
    return out;
}

// The scalar phases are separate (not inlined) functions over a state block in LDS, and the launch arguments are read through a
// pointer to a device copy of np_ea_args: inlined into one kernel body, the two halves' states, the ~40 argument pointers and the
// walk's own variables competed for 102 scalar registers, and the compiler parked hundreds of them in vector-register lanes
// (v_writelane / v_readlane on every use) -- the first form of this kernel was slower than the one-read kernel for that reason alone.
struct ea_wave_state { ea_half h[2]; int drained; };

__device__ __forceinline__ ea_half ea_get(const ea_wave_state* W, int q)
{
    ea_half h;
    const int* p = (const int*)&W->h[q];
    int* d = (int*)&h;
#pragma unroll
    for (int i = 0; i < (int)(sizeof(ea_half) / 4); ++i) d[i] = __builtin_amdgcn_readfirstlane(p[i]);
    return h;
}
__device__ __forceinline__ void ea_put(ea_wave_state* W, int q, const ea_half& h, int lane)
{
    __builtin_amdgcn_wave_barrier();
    if (lane == 0) W->h[q] = h;
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
    __builtin_amdgcn_s_waitcnt(0);
    __builtin_amdgcn_wave_barrier();
}
__device__ __forceinline__ void ea_finish_read(const np_ea_args& a, ea_half& h, int lane)
{
    if (lane == 0) {
        const int cap = (int)(a.out_off[h.ri + 1] - a.out_off[h.ri]);
        a.n_out[h.ri] = h.n_out < cap ? h.n_out : cap; a.status[h.ri] = h.status; a.n_calls[h.ri] = h.n_calls;
    }
    h.ri = -1;
}

// leaves half q with the geometry of its read's next segment (taking new reads from the queue as reads end), or without a read
__device__ __attribute__((noinline)) void ea_next_segment(const np_ea_args* __restrict__ ap_, ea_wave_state* W, const int q_, const int lane)
{
    const np_ea_args& a = *ea_uniform(ap_);
    const int q = ea_uniform(q_);
    ea_half h = ea_get(W, q);
    int drained = __builtin_amdgcn_readfirstlane(W->drained);
    const int k = a.k;
    for (;;) {
        if (h.ri < 0) {
            if (drained) break;
            const int ri = __builtin_amdgcn_readfirstlane((int)atomicAdd(a.counter, lane == 0 ? 1u : 0u));
            if (ri >= a.n_reads) { drained = 1; break; }
            h.ri = ri; h.n_out = 0; h.n_calls = 0; h.status = NP_EA_OK;
            const ea_read R = ea_load_read(a, ri);
            const int max_kmer_idx = R.rl - k;                       // trim_aligned_pairs_to_kmer, :167-177
            int q_first = 0, r_first = 0, q_last = 0, r_last = 0;
            // a read without events in the reference (failed alignment / calibration / events-per-base QC, squiggle_read.cpp:320-335) is skipped
            bool have = a.cig_reads[4 * ri + 2] != 0 && R.rd->n_events > 0 && a.n_pairs[ri] > 0 && !(a.events_per_base[ri] > 5.0) &&
                        (!a.calibrated || a.calibrated[ri] != 0) && first_aligned_read_ge(R.cv, 0, q_first, r_first) &&
                        last_aligned_read_le_r(R.cv, max_kmer_idx, q_last, r_last) && q_first <= q_last;
            int first_event = -1, last_event = -1;
            if (have) {
                const int ks = R.rc ? R.rl - q_first - k : q_first, ke = R.rc ? R.rl - q_last - k : q_last;      // flip_k_strand
                if (ks < 0 || ks >= R.K || ke < 0 || ke >= R.K) { have = false; h.status = NP_EA_BAD_RECORD; }    // the reference asserts / reads out of range
                else { first_event = closest_event(R.ms, R.K, ks); last_event = closest_event(R.ms, R.K, ke); }
            }
            if (!have) { ea_finish_read(a, h, lane); continue; }
            h.forward = first_event < last_event ? 1 : 0;
            h.curr_start_event = __builtin_amdgcn_readfirstlane(first_event); h.curr_start_ref = __builtin_amdgcn_readfirstlane(r_first);
            h.last_event = __builtin_amdgcn_readfirstlane(last_event); h.q_last = __builtin_amdgcn_readfirstlane(q_last);
            h.r_last = __builtin_amdgcn_readfirstlane(r_last);
        }
        if (!((h.forward && h.curr_start_event < h.last_event) || (!h.forward && h.curr_start_event > h.last_event))) { ea_finish_read(a, h, lane); continue; }
        const ea_read R = ea_load_read(a, h.ri);
        // ---- segment geometry (:695-735) ----
        int q_end = 0, r_end = 0;
        if (!last_aligned_ref_le(R.cv, h.curr_start_ref + 100, q_end, r_end)) { ea_finish_read(a, h, lane); continue; }   // cannot happen
        if (q_end > h.q_last) { q_end = h.q_last; r_end = h.r_last; }
        const bool last_section = q_end == h.q_last;
        const int curr_end_read = R.rc ? R.rl - q_end - k : q_end;
        const int l = r_end - h.curr_start_ref + 1;
        if (l < 2 * k) { ea_finish_read(a, h, lane); continue; }                                     // hmm_sequence.length() < 2 * k
        if (h.curr_start_ref + l > R.ref_n || curr_end_read < 0 || curr_end_read >= R.K) { h.status = NP_EA_BAD_RECORD; ea_finish_read(a, h, lane); continue; }
        const int e_start = __builtin_amdgcn_readfirstlane(h.curr_start_event), e_stop = __builtin_amdgcn_readfirstlane(closest_event(R.ms, R.K, curr_end_read));
        const int span = e_start > e_stop ? e_start - e_stop : e_stop - e_start;
        if (span < 2) { ea_finish_read(a, h, lane); continue; }
        const int e = span + 1, n = __builtin_amdgcn_readfirstlane(l - k + 1);
        if (n > a.max_kmers || e > a.rows_cap) { h.status = NP_EA_OVERFLOW; ea_finish_read(a, h, lane); continue; }
        h.n_calls++;
        h.e_start = e_start; h.stride = e_start < e_stop ? 1 : -1; h.e = e; h.n = n; h.last_section = last_section ? 1 : 0;
        break;
    }
    ea_put(W, q, h, lane);
    if (lane == 0) W->drained = drained;
    __builtin_amdgcn_wave_barrier();
}

// Back-track (profile_hmm_align_r9, r9.cpp:117-196) of BOTH halves' segments as vector code: lanes 0..31 walk half 0's path, lanes
// 32..63 half 1's (every lane of a half computes the same).  A walk step is one dependent chain around an LDS read; as scalar
// code, one segment after the other, it took ~550-790 cycles per step and half of this kernel's time (the scalar unit's latency
// per dependent instruction, ~40-55 of them per step), and two scalar chains interleaved in one loop were no faster.  As vector
// code the chain is ~25 instructions for BOTH segments.
// Per half: a window of NP_EA_WIN lines of its dwords staged in LDS (refilled when the walk leaves it) and the list of visited
// states in LDS (ea_lds; a longer path spills the full buffer to the half's global list and goes on).
typedef __attribute__((address_space(3))) uint32_t lds_u32;
#ifndef NP_EA_EARLY
#define NP_EA_EARLY 5                     // refill a window that has fewer than this many lines left (experiment)
#endif
#define NP_EA_WIN 24                      // lines of a half's window: three rounds of 64 lanes' 16-byte requests
#define NP_EA_LDW 32                      // dwords of a half's line
#ifndef NP_EA_BCAP
#define NP_EA_BCAP 112                    // bursts of a half's list that LDS holds (a longer list spills to the half's global list): twenty
                                          // waves' blocks fit a CU's LDS beside their windows
#endif
#define NP_EA_BURST 10                    // steps of a burst at most: their codes share a dword
// The list of visited states, per half: one 64-bit word per BURST of walk steps (round 5; until then one dword per visited state, written
// by every step -- six of a step's vector instructions).  Low dword: the state the burst starts in, row | k-mer << 16 | state << 24, and
// the number of steps << 26; high dword: the steps' move codes, three bits each, first step lowest.  The emission replays a burst from
// its first state (row -= state != KMER_SKIP, k-mer -= code >> 2, state = code & 3).
struct alignas(16) ea_lds {
    uint32_t stage[2][NP_EA_WIN * NP_EA_LDW];        // back-pointer windows
    uint64_t bursts[2][NP_EA_BCAP];        // oldest first
    ea_wave_state W;
};
static_assert(20 * sizeof(ea_lds) <= 163840, "twenty waves of a CU");
typedef __attribute__((address_space(3))) uint64_t lds_u64;
typedef __attribute__((address_space(3))) uint8_t lds_u8;
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) u32x4 lds_u32x4;
struct ea_walk_result { int nb0, nb1, spilled0, spilled1; };       // bursts in all, bursts spilled

// A walk step takes its move from the dword of the lane that owns the k-mer: the state walked in (0 KMER_SKIP, 1 BAD_EVENT, 2 MATCH) has
// its bits from pos = first bit + stride x (k % BPL) on; the lowest set one -- or the end mark behind the state's last bit -- is the
// candidate, its move code three bits of NP_EA_CODES.  The numbers of a state are bytes of constants.
#define NP_EA_POS0(BPL) (7u * (BPL) - 2u + 0x010000u)       // per state: first bit of block 0 (K 5 BPL + 2 (BPL - 1), B 0, M 1)
#define NP_EA_STRIDE 0x0505fe            // per state: what a block adds to its first bit (5, 5, -2)
#define NP_EA_END   0x100204u            // per state: the bit after its last candidate's
#define NP_EA_ROW   0x0f0900u            // per state: first bit of its row of NP_EA_CODES
#define NP_EA_CODES ((4u | 5u << 3 | 6u << 6) | (1u << 9 | 2u << 12) | (4u << 15 | 5u << 18 | 1u << 21 | 6u << 24 | 2u << 27))

// the lane (of its half) that owns k-mer k = k / BPL, as full-rate instructions (a 32-bit multiply-high is quarter rate); 5 bits, as the
// shifts that use it take
// (the full-rate 24-bit multiply by name: the compiler takes the quarter-rate v_mul_lo_u32 for these small products whatever it is told
//  about the operands)
__device__ __forceinline__ uint32_t ea_mul24(const uint32_t a, const uint32_t b)
{
    uint32_t p;
    asm("v_mul_u32_u24 %0, %1, %2" : "=v"(p) : "v"(a), "v"(b));
    return p;
}
__device__ __forceinline__ uint32_t ea_mad24(const uint32_t a, const int b, const uint32_t c)
{
    uint32_t p;
    asm("v_mad_i32_i24 %0, %1, %2, %3" : "=v"(p) : "v"(a), "v"(b), "v"(c));
    return p;
}
template <int BPL> __device__ __forceinline__ uint32_t ea_owner(const uint32_t k)
{
    if constexpr (BPL == 3) return __builtin_amdgcn_ubfe(ea_mul24(k, 171u), 9, 5);      // exact for k < 512 (k < 96 here)
    else { static_assert((BPL & (BPL - 1)) == 0, "k-mers per lane"); return (k / BPL) & 31u; }
}

template <int BPL>
__device__ __attribute__((noinline)) ea_walk_result ea_walk2(ea_lds* L, const float sv0_, const float sv1_, const uint8_t* __restrict__ bp_,
                                                             uint32_t* __restrict__ path0_, uint32_t* __restrict__ path1_, const int lane)
{
    constexpr int LINE = NP_EA2_LINE_BYTES, WIN = NP_EA_WIN;
    const float sv0 = ea_uniform(sv0_), sv1 = ea_uniform(sv1_);
    const uint8_t* __restrict__ bp = ea_uniform(bp_);

    uint32_t* __restrict__ path0 = ea_uniform(path0_); uint32_t* __restrict__ path1 = ea_uniform(path1_);
    const ea_half H0 = ea_get(&L->W, 0), H1 = ea_get(&L->W, 1);
    const bool hi_half = lane >= 32;
    const int sl = lane & 31;
    // per-lane state, uniform within a half
    const int e = hi_half ? H1.e : H0.e, n = hi_half ? H1.n : H0.n;
    int row = e, k = n - 1, ps = 2, nb = 0, spilled = 0;               // nb: bursts recorded; k: the k-mer; lane k / BPL (of the half) owns it, as its block k % BPL
    int lo = 0x7fffffff;                                  // no window yet
    // assert(get(vm, row, col) != -INFINITY): no path, nothing to emit
    bool alive = (hi_half ? (H1.ri >= 0 && sv1 != NP_NEG_INF) : (H0.ri >= 0 && sv0 != NP_NEG_INF)) && e > 0 && n > 0;
    // (L arrives as a generic pointer -- a not-inlined function's argument; without the address space the compiler reads the staged
    //  lines with flat loads behind null checks and 64-bit address arithmetic, in the middle of the walk's dependent chain)
    const lds_u8* st = (const lds_u8*)&L->stage[hi_half ? 1 : 0][0];
    lds_u64* bl = (lds_u64*)&L->bursts[hi_half ? 1 : 0][0];
    static_assert(WIN * NP_EA_LDW * 4 % (64 * 16) == 0, "whole rounds of 16-byte requests");
    constexpr int ROUNDS = WIN * NP_EA_LDW * 4 / (64 * 16);
    while (__builtin_amdgcn_ballot_w64(alive) != 0ull) {
        // ---- per half, by scalar control: refill the window of a walk that is outside it; spill a full list ----
        const int line0 = (int)((uint32_t)row + (uint32_t)k / BPL);
        const bool need = alive && (line0 < lo || (NP_EA_EARLY > 0 && line0 < lo + NP_EA_EARLY && lo > 1)), full = alive && nb - spilled >= NP_EA_BCAP;
        const uint64_t need_m = __builtin_amdgcn_ballot_w64(need), full_m = __builtin_amdgcn_ballot_w64(full);
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            if ((need_m >> (32 * h)) & 1ull) {
                const int hi = __builtin_amdgcn_readlane(line0, 32 * h);
                const int nlo = hi - (WIN - 1) > 1 ? hi - (WIN - 1) : 1;
                // the half's 128 bytes of every line of the window, eight 16-byte requests per line (lane i of round r: piece i & 7 of line
                // 8 r + i / 8), all of a refill in flight at once, at agent scope: they bypass the vector L1, which may still hold the
                // previous segment's lines at these addresses.  A piece past the window's last line is outside the descriptor's range and
                // reads as 0 (nobody reads it).
                const __amdgpu_buffer_rsrc_t lr = make_rsrc(bp + (size_t)(nlo - 1) * LINE, (uint32_t)(hi - nlo + 1) * LINE);
                u32x4 v[ROUNDS];
#pragma unroll
                for (int it = 0; it < ROUNDS; ++it)
                    v[it] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(lr, whole_offset((8 * it + (lane >> 3)) * LINE + h * (LINE / 2) + (lane & 7) * 16), 0, 16 /* sc1 */));
                lds_u32x4* dst = (lds_u32x4*)&L->stage[h][0];
#pragma unroll
                for (int it = 0; it < ROUNDS; ++it) dst[64 * it + lane] = v[it];
                lo = (hi_half == (h == 1)) ? nlo : lo;
            }
            if ((full_m >> (32 * h)) & 1ull) {
                const int sp = __builtin_amdgcn_readlane(spilled, 32 * h);
                uint64_t* __restrict__ dstp = (uint64_t*)(h ? path1 : path0) + sp;
                for (int i = lane; i < NP_EA_BCAP; i += 64) dstp[i] = L->bursts[h][i];
                spilled = (hi_half == (h == 1)) ? spilled + NP_EA_BCAP : spilled;
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
        __builtin_amdgcn_s_waitcnt(0);
        __builtin_amdgcn_wave_barrier();
        // ---- a burst of steps: as many as no live walk can leave its window in.  A step lowers row + k / BPL by at most 2, so the count
        //      is known before the first one and the steps themselves carry no window test, no ballot and no branch (round 5: the
        //      per-step test and the selects that froze a waiting walk were a third of the chain's instructions)
        const int room = (int)(((uint32_t)line0 - (uint32_t)lo) >> 1) + 1;      // (unsigned: a finished walk's numbers are anything)
        const int mine = alive ? room : NP_EA_BURST;
        const int b0 = __builtin_amdgcn_readlane(mine, 0), b1 = __builtin_amdgcn_readlane(mine, 32);
        const int b01 = b0 < b1 ? b0 : b1, burst = b01 < NP_EA_BURST ? b01 : NP_EA_BURST;
        // the dword of cell (row, k): stage[(row + k / BPL - lo) * 32 + k / BPL], i.e. byte 128 (row - lo) + 132 (k / BPL).  (A finished
        // walk's offset is anything: the min keeps its reads inside the window.)
        const uint32_t lo128 = (uint32_t)lo * (4u * NP_EA_LDW);
        const uint32_t first = (uint32_t)row | ((uint32_t)k << 16) | ((uint32_t)ps << 24);
        uint32_t codes = 0u;
        uint32_t steps0 = 0u, steps1 = 0u;                // steps each half's walk was alive at
        uint64_t am = __builtin_amdgcn_ballot_w64(alive); // inside the burst "alive" is this scalar mask, the counts scalar additions
        for (int s = 0; s < burst; ++s) {
            steps0 += (uint32_t)am & 1u; steps1 += (uint32_t)(am >> 32) & 1u;
            // the move out of this cell: the dword of the lane that owns the k-mer, of it the state's bits of the k-mer's block
            const uint32_t own = ea_owner<BPL>((uint32_t)k);
            const uint32_t off = ea_mul24(own, 4u * NP_EA_LDW + 4u) + (((uint32_t)row * (4u * NP_EA_LDW)) - lo128);
            const uint32_t w = *(const lds_u32*)(st + (off < (uint32_t)(4 * (WIN * NP_EA_LDW - 1)) ? off : (uint32_t)(4 * (WIN * NP_EA_LDW - 1))));
            const uint32_t b8 = (uint32_t)ps * 8u;
            const uint32_t blk = (uint32_t)k - ea_mul24(own, BPL);
            const uint32_t pos = ea_mad24(blk, __builtin_amdgcn_sbfe(NP_EA_STRIDE, b8, 8), __builtin_amdgcn_ubfe(NP_EA_POS0(BPL), b8, 8));
            const uint32_t f = (w >> (pos & 31u)) | __builtin_amdgcn_ubfe(NP_EA_END, b8, 8);
            const uint32_t c = __builtin_amdgcn_ubfe(NP_EA_CODES, (uint32_t)__builtin_ctz(f) * 3u + __builtin_amdgcn_ubfe(NP_EA_ROW, b8, 8), 3);
            codes |= c << (3 * s);
            row -= ps != 0 ? 1 : 0;                                     // K states are silent (r9.cpp:176-178)
            k -= (int)(c >> 2);
            ps = (int)(c & 3u);
            // the walk ends at row 0 or k-mer -1 (the soft clip leads to row 0: no test of its own).  A finished walk's row, k and state are
            // not used again.
            am &= __builtin_amdgcn_ballot_w64(row > 0) & __builtin_amdgcn_ballot_w64(k >= 0);      // (two ballots: each is its compare's own result register)
        }
        alive = __builtin_amdgcn_inverse_ballot_w64(am);
        const uint32_t steps = hi_half ? steps1 : steps0;
        if (sl == 0 && steps > 0u) bl[nb - spilled] = (uint64_t)(first | (steps << 26)) | ((uint64_t)codes << 32);
        nb += steps > 0u ? 1 : 0;
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
    __builtin_amdgcn_s_waitcnt(0);
    __builtin_amdgcn_wave_barrier();
    ea_walk_result r;
    r.nb0 = __builtin_amdgcn_readlane(nb, 0); r.nb1 = __builtin_amdgcn_readlane(nb, 32);
    r.spilled0 = __builtin_amdgcn_readlane(spilled, 0); r.spilled1 = __builtin_amdgcn_readlane(spilled, 32);
    return r;
}

// emission (eventalign.cpp:774-812) of half q's segment from its list of bursts (those from `spilled` on in LDS, older ones in the half's
// global list).  Ascending order = the list read backwards: a round takes the last 64 bursts not yet seen, lane 0 the last of them; a
// lane replays its burst from its first state and then goes through the states last to first.
__device__ __attribute__((noinline)) void ea_emit_segment(const np_ea_args* __restrict__ ap_, ea_lds* L, const int q_, const int nb_, const int spilled_,
                                                          const uint32_t* __restrict__ path_, const int lane)
{
    const np_ea_args& a = *ea_uniform(ap_);
    const int q = ea_uniform(q_), nb = ea_uniform(nb_), spilled = ea_uniform(spilled_);
    const uint64_t* __restrict__ path = (const uint64_t*)ea_uniform(path_);
    ea_wave_state* W = &L->W;
    ea_half h = ea_get(W, q);
    const int e_start = h.e_start, stride = h.stride;
    const int64_t o0 = a.out_off[h.ri];
    const int out_cap = (int)(a.out_off[h.ri + 1] - o0);
    int32_t* __restrict__ out_ref = a.out_ref + o0; int32_t* __restrict__ out_event = a.out_event + o0; uint8_t* __restrict__ out_state = a.out_state + o0;
    const lds_u64* bl = (const lds_u64*)&L->bursts[q][0];
    const uint64_t below = (1ull << lane) - 1ull;
    int num_output = 0, last_event_output = 0, last_ref_kmer_output = 0;
    for (int base = 0; base < nb && (num_output < 50 || h.last_section); base += 64) {
        const int w = nb - 1 - base - lane;
        uint64_t word = 0ull;                             // (no burst: no steps)
        if (w >= 0) word = w >= spilled ? bl[w - spilled] : path[w];
        const uint32_t first = (uint32_t)word, codes = (uint32_t)(word >> 32);
        const int n = (int)((first >> 26) & 15u);
        int row = (int)(first & 0xffffu), k = (int)((first >> 16) & 0xffu), ps = (int)((first >> 24) & 3u);
        int evi[NP_EA_BURST], km[NP_EA_BURST]; bool qq[NP_EA_BURST], is_m[NP_EA_BURST];
        int mine = 0;                                     // states of this burst that are output candidates: not K, not the start event
#pragma unroll
        for (int j = 0; j < NP_EA_BURST; ++j) {
            evi[j] = e_start + (row - 1) * stride; km[j] = k; is_m[j] = ps == 2;
            qq[j] = j < n && ps != 0 && evi[j] != h.curr_start_event;
            mine += qq[j] ? 1 : 0;
            const uint32_t c = (codes >> (3 * j)) & 7u;
            row -= ps != 0 ? 1 : 0; k -= (int)(c >> 2); ps = (int)(c & 3u);
        }
        // candidates of the lanes before this one, and of the round (mine <= 10: four bits)
        int before = 0, total = 0;
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            const uint64_t m = __builtin_amdgcn_ballot_w64(((mine >> b) & 1) != 0);
            before += __builtin_popcountll(m & below) << b; total += __builtin_popcountll(m) << b;
        }
        int pos = num_output + before;
        bool any = false; int my_event = 0, my_kmer = 0;  // the last state this lane wrote
#pragma unroll
        for (int j = NP_EA_BURST - 1; j >= 0; --j) {
            const bool wr = qq[j] && (pos < 50 || h.last_section);
            const int o = h.n_out + (pos - num_output);
            if (wr && o < out_cap) {
                out_ref[o] = h.curr_start_ref + km[j];
                out_event[o] = evi[j];
                out_state[o] = is_m[j] ? (uint8_t)'M' : (uint8_t)'B';
            }
            any = any || wr; my_event = wr ? evi[j] : my_event; my_kmer = wr ? km[j] : my_kmer;
            pos += qq[j] ? 1 : 0;
        }
        const uint64_t wm = __builtin_amdgcn_ballot_w64(any);
        const int left = 50 - num_output;
        const int nw = h.last_section ? total : (total < left ? total : (left > 0 ? left : 0));
        if (wm != 0ull) {
            const int last_lane = 63 - __builtin_clzll(wm);
            last_event_output = __shfl(my_event, last_lane, 64);
            last_ref_kmer_output = h.curr_start_ref + __shfl(my_kmer, last_lane, 64);
        }
        if (h.n_out + nw > out_cap) h.status = NP_EA_OVERFLOW;
        h.n_out += nw; num_output += nw;
    }
    if (h.status != NP_EA_OK) ea_finish_read(a, h, lane);
    else {
        h.curr_start_event = __builtin_amdgcn_readfirstlane(last_event_output);
        h.curr_start_ref = __builtin_amdgcn_readfirstlane(last_ref_kmer_output);
        if (num_output == 0) ea_finish_read(a, h, lane);
    }
    ea_put(W, q, h, lane);
}

// WAVES: resident waves per SIMD the register budget is set for (4: 128 registers, no spills in the sweep; 5: 96)
template <int WAVES, int BPL>
__global__ void __launch_bounds__(64, WAVES) np_eventalign_chain2_kernel(const np_ea_args* __restrict__ ap)
{
    __shared__ ea_lds lds;
    ea_wave_state& W = lds.W;
    const np_ea_args& a = *ap;
    const int lane = threadIdx.x;
    const int wave_slot = blockIdx.x;
    uint8_t* __restrict__ bp = a.bp + (size_t)wave_slot * a.bp_stride;
    uint32_t* __restrict__ path = a.path + (size_t)wave_slot * a.path_stride;
    const int k = a.k;
    if (lane == 0) { W.h[0].ri = -1; W.h[1].ri = -1; W.drained = 0; }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
    __builtin_amdgcn_s_waitcnt(0);
    __builtin_amdgcn_wave_barrier();

    unsigned long long cells = 0ull, rows = 0ull, kmers = 0ull;
    unsigned long long t_next = 0ull, t_fill = 0ull, t_fin = 0ull;      // shader cycles this wave spent in the three phases (statistics)
    for (;;) {
        unsigned long long t0 = __builtin_amdgcn_s_memtime();
        ea_next_segment(ap, &W, 0, lane);
        ea_next_segment(ap, &W, 1, lane);
        const ea_half H0 = ea_get(&W, 0), H1 = ea_get(&W, 1);
        if (H0.ri < 0 && H1.ri < 0) break;
        unsigned long long t1 = __builtin_amdgcn_s_memtime();
        t_next += t1 - t0;

        // ---- the lane's BPL blocks of its half's segment (ProfileHMMViterbiOutputR9, r9.inl:130-197) ----
        const bool hi_half = lane >= 32;
        const int sl = lane & 31;
        ea_seg S0, S1;
        ea_gauss<BPL> G;
        ea_trans tr;
        {
            const ea_read R0 = ea_load_read(a, H0.ri >= 0 ? H0.ri : 0), R1 = ea_load_read(a, H1.ri >= 0 ? H1.ri : 0);
            S0 = H0.ri >= 0 ? ea_seg{R0.ev, H0.e_start, H0.stride, H0.e, H0.n} : ea_seg{R0.ev, 0, 1, 0, 0};
            S1 = H1.ri >= 0 ? ea_seg{R1.ev, H1.e_start, H1.stride, H1.e, H1.n} : ea_seg{R1.ev, 0, 1, 0, 0};
            cells += (unsigned long long)(S0.e > 0 ? (S0.e + 1) * 3 * (S0.n + 2) : 0) + (unsigned long long)(S1.e > 0 ? (S1.e + 1) * 3 * (S1.n + 2) : 0);
            rows += (unsigned long long)(S0.e + S1.e); kmers += (unsigned long long)(S0.n + S1.n);
            const np_read_dev* rd = hi_half ? R1.rd : R0.rd;
            const char* ref = hi_half ? R1.ref : R0.ref;
            const bool rc = hi_half ? R1.rc : R0.rc;
            const int n = hi_half ? S1.n : S0.n, csr = hi_half ? H1.curr_start_ref : H0.curr_start_ref;
            const double scale = rd->scale, shift = rd->shift, var = rd->var, log_var = rd->log_var;
            tr = ea_trans{rd->trans[0], rd->trans[1], rd->trans[2], rd->trans[3], rd->trans[4], rd->trans[5], rd->trans[6], rd->trans[7],
                          rd->trans[8], rd->trans[9]};
#pragma unroll
            for (int c = 0; c < BPL; ++c) {
                const int b = BPL * sl + c;
                uint32_t rank = 0;
                if (b < n) {
                    // HMMInputSequence::get_kmer_rank(b, k, rc): the forward k-mer at b, or its reverse complement's rank
                    for (int t = 0; t < k; ++t) {
                        const uint32_t code = rc ? 3u - base_code(ref[csr + b + k - 1 - t]) : base_code(ref[csr + b + t]);
                        rank = rank * 4u + code;
                    }
                }
                G.g[c] = np_scale_state(a.model, rank, scale, shift, var, log_var);
            }
        }
        const float2 start_v = ea_fill2<BPL>(G, tr, a.flank[0], S0, S1, bp, lane);
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
        __builtin_amdgcn_s_waitcnt(0);
        unsigned long long t2 = __builtin_amdgcn_s_memtime();
        t_fill += t2 - t1;
        const bool prio = __builtin_amdgcn_readfirstlane(a.walk_prio) != 0;
        if (prio) __builtin_amdgcn_s_setprio(3);
        uint32_t* path1 = path + (a.path_stride >> 1);
        const ea_walk_result wr = ea_walk2<BPL>(&lds, start_v.x, start_v.y, bp, path, path1, lane);
        if (H0.ri >= 0) ea_emit_segment(ap, &lds, 0, wr.nb0, wr.spilled0, path, lane);
        if (H1.ri >= 0) ea_emit_segment(ap, &lds, 1, wr.nb1, wr.spilled1, path1, lane);
        if (prio) __builtin_amdgcn_s_setprio(0);
        t_fin += __builtin_amdgcn_s_memtime() - t2;
    }
    if (lane == 0 && a.stats && cells) {
        atomicAdd(a.stats, cells); atomicAdd(a.stats + 1, rows); atomicAdd(a.stats + 2, kmers);
        atomicAdd(a.stats + 3, t_next); atomicAdd(a.stats + 4, t_fill); atomicAdd(a.stats + 5, t_fin);
    }
}

} // namespace

// variant 2 / 3: the register budget of 4 / 5 resident waves per SIMD (three k-mer blocks per lane: segments of up to 96 k-mers, k >= 6);
// variant 4: four blocks per lane at 4 waves per SIMD (up to 128 k-mers: the direct-RNA model, k = 5, whose segments reach 97).
// (Rounds 1-3 also carried a one-read-per-wave kernel; round 4 removed it: the two-read kernel is the faster one on every input
// measured, both were pinned by the same tests, and a divergence seen once while refactoring the old kernel's walk was never
// explained.)
hipError_t np_launch_eventalign_chain(const np_ea_args& a, const np_ea_args* a_dev /* a device copy of a */, int n_blocks, int variant, hipStream_t s)
{
    (void)a;
    if (variant == 2) hipLaunchKernelGGL((np_eventalign_chain2_kernel<4, 3>), dim3(n_blocks), dim3(64), 0, s, a_dev);
    else if (variant == 3) hipLaunchKernelGGL((np_eventalign_chain2_kernel<5, 3>), dim3(n_blocks), dim3(64), 0, s, a_dev);
    else hipLaunchKernelGGL((np_eventalign_chain2_kernel<4, 4>), dim3(n_blocks), dim3(64), 0, s, a_dev);
    return hipGetLastError();
}
int np_eventalign_line_bytes(int variant) { (void)variant; return NP_EA2_LINE_BYTES; }
int np_eventalign_max_kmers(int variant) { return variant == 4 ? 128 : 96; }
