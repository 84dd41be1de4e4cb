// np_constants.h -- the per-read constants that go through the C library's log / exp / logf, formed on the HOST by calling the
// process's own functions in the reference's own expressions:
//   * the event aligner's lp_skip / lp_stay / lp_step / lp_trim   (src/nanopolish_raw_loader.cpp:99-108)
//   * the HMM transitions                                         (src/hmm/nanopolish_profile_hmm_r9.inl:17-76)
// (set4's log(var), src/nanopolish_squiggle_read.cpp:38-65, and profile_hmm_score_set's log(n), src/hmm/nanopolish_profile_hmm.cpp:38,
// are single calls where they are needed.)
//
// Why on the host: a constant that is one unit in the last place away from the reference's can flip a p7_FLogsum table index or an
// arg-max of the aligner, and the C library rounds these functions its own way -- the device's math library need not agree with it in
// the last bit, and another C library need not agree with this one.  Calling the process's functions gives the reference's bits with
// whatever library both are linked to.  np_capi.hip (host_fix) says how the device-resident pass reaches them.
#pragma once
#include <cmath>
#include <stdint.h>

// The ten transition PROBABILITIES, in the order of BlockTransitions (src/hmm/nanopolish_profile_hmm_r9.h:75-95): mm_self, mb, mk,
// mm_next, bb, bk, bm_next, bm_self, kk, km.  Only mm_self and mm_next depend on the read.
static inline void np_transition_probs(double events_per_base, double indel_bias, float p[10])
{
    double read_events_per_base = events_per_base;
    read_events_per_base *= indel_bias;
    read_events_per_base = read_events_per_base > 1.25 ? read_events_per_base : 1.25;   // std::max(1.25, x)
    const float p_stay = (float)(1 - (1 / read_events_per_base));
    const float p_skip = 0.0025f, p_bad = 0.001f, p_bad_self = p_bad, p_skip_self = 0.3f;
    const float p_mk = p_skip, p_mb = p_bad, p_mm_self = p_stay;
    const float p_mm_next = 1.0f - p_mm_self - p_mk - p_mb;
    const float p_bb = p_bad_self;
    const float p_bk = (1.0f - p_bb) / 3;
    const float p_kk = p_skip_self;
    p[0] = p_mm_self; p[1] = p_mb; p[2] = p_mk; p[3] = p_mm_next; p[4] = p_bb;
    p[5] = p_bk; p[6] = p_bk; p[7] = p_bk; p[8] = p_kk; p[9] = 1.0f - p_kk;
}
static inline void np_transitions(double events_per_base, double indel_bias, float out[10])
{
    float p[10];
    np_transition_probs(events_per_base, indel_bias, p);
    for (int i = 0; i < 10; ++i) out[i] = logf(p[i]);                       // the float overload of log, as r9.inl:61-72
}

#define NP_ALIGN_EPSILON 1e-10
#define NP_ALIGN_P_TRIM 0.01
// lp_stay and lp_step of one read; lp_skip = log(NP_ALIGN_EPSILON) and its exp do not depend on the read
static inline void np_aligner_lp(uint32_t n_events, uint32_t n_kmers, double exp_lp_skip, double* lp_stay, double* lp_step)
{
    const double events_per_kmer = (double)n_events / (double)n_kmers;
    const double p_stay = 1 - (1 / (events_per_kmer + 1));
    *lp_stay = log(p_stay);
    *lp_step = log(1.0 - exp_lp_skip - exp(*lp_stay));
}
