// Losses over rows of class scores: what their kernels are given.
#pragma once
#include "evt_internal.h"

// what a kernel makes of a row
enum { SC_LOGP = 0, SC_GRAD = 1, SC_DISTILL = 2, SC_POLICY = 3 };

#define EVT_SCORES_MAX_TOP 1024 // entries of a teacher a row

struct ScoreArgs {
    const void *x;
    void *g; // nullptr: no gradient; x itself: in place
    int64_t xs, gs; // elements from row to row
    int64_t N;
    int64_t row0; // the launch's first row
    int32_t V;
    int32_t past;   // the gradient is stored past the caches
    double inv_t;   // 1 / temperature
    float exp_mul;  // log2(e) / temperature: exp(d / T) = exp2(d * exp_mul)
    const void *labels;
    int32_t label64;
    // rows outside [bounds[0], bounds[n_bounds - 1]) are left out (nullptr: none is)
    const int32_t *bounds;
    int32_t n_bounds;
    const float *weights; // a row's, ws elements apart, nullptr: ones
    int64_t ws;
    float *loss, *logp, *stats;
    float *slope; // SC_GRAD reads a row's dloss / dlogp here; SC_LOGP clears it for the kernel that fills it in (nullptr: does not)
    // SC_DISTILL
    const void *ids, *top;
    int32_t id64, top_type, n_top;
    float t_mul, t2_mul; // temperature and its square
    // SC_POLICY
    const float *old_logp, *adv, *ref_logp;
    double log_lo, log_hi; // the bounds of logp - old_logp
    double lo, hi, kl;
};

void score_scale(ScoreArgs &a, double temperature);
int launch_distill_f32(hipStream_t s, const ScoreArgs &a); // loss nullptr: none
