// Losses over rows of class scores with their gradients, for scores of any number of classes in device memory: log-probabilities of chosen
// classes, distillation from a teacher's top scores, the preference loss of paired sequences and the clipped policy loss.
//
// With m the row's maximum, e_c = exp((x_c - m) / T) and S = sum_c e_c, the class probabilities are q_c = e_c / S.  Every gradient here is
// a multiple of q plus something at a few classes:
//   d logp(label) / dx_c = ([c == label] - q_c) / T
//   d KL(p || q) / dx_c  = (q_c - p_c) / T
// so a kernel finds m and S, then the row's loss and its factor, then writes factor * q for every class and writes the few classes again.
//
// Scores are 16 or 32 bits wide; differences, exponentials, sums and losses are 32-bit, a gradient is rounded once, when it is written.
#include "scores.h"
#include <math.h>
#include <utility>

typedef _Float16 half_t;
typedef __bf16 bf16_t;

// (m, s): the maximum of some scores and the sum of their exp((x - m) / T).  Scores of -inf count nothing, a NaN or +inf makes s a NaN.
struct MaxSum {
    float m, s;
};
__device__ __forceinline__ float finite_or_zero(float m) { return m == -INFINITY ? 0.0f : m; }
__device__ __forceinline__ MaxSum join(MaxSum a, MaxSum b, float mul) {
    const float m = fmaxf(a.m, b.m), z = finite_or_zero(m);
    return {m, a.s * __builtin_amdgcn_exp2f((a.m - z) * mul) + b.s * __builtin_amdgcn_exp2f((b.m - z) * mul)};
}
__device__ __forceinline__ MaxSum wave_join(MaxSum a, float mul) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) a = join(a, {__shfl_xor(a.m, o), __shfl_xor(a.s, o)}, mul);
    return a;
}
__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    return v;
}
template <int WAVES>
__device__ __forceinline__ MaxSum block_join(MaxSum a, float mul) {
    __shared__ MaxSum s_a[WAVES];
    a = wave_join(a, mul);
    if ((threadIdx.x & 63) == 0) s_a[threadIdx.x >> 6] = a;
    __syncthreads();
    a = s_a[0];
#pragma unroll
    for (int w = 1; w < WAVES; w++) a = join(a, s_a[w], mul);
    __syncthreads();
    return a;
}
template <int WAVES>
__device__ __forceinline__ float block_sum(float v) {
    __shared__ float s_v[WAVES];
    v = wave_sum(v);
    if ((threadIdx.x & 63) == 0) s_v[threadIdx.x >> 6] = v;
    __syncthreads();
    v = s_v[0];
#pragma unroll
    for (int w = 1; w < WAVES; w++) v += s_v[w];
    __syncthreads();
    return v;
}

__device__ __forceinline__ int64_t load_id(const void *p, int wide, int64_t i) { return wide ? ((const int64_t *)p)[i] : ((const int32_t *)p)[i]; }
__device__ __forceinline__ float load_score(const void *p, int type, int64_t i) {
    return type == EVT_F32 ? ((const float *)p)[i] : type == EVT_BF16 ? (float)((const bf16_t *)p)[i] : (float)((const half_t *)p)[i];
}

// A row of score x at its label: its log-probability.  Nothing is left of a row whose scores are all -inf: every class has probability 0.
// 64 bits for the two terms: a policy's ratio is compared with its bounds.
__device__ __forceinline__ double row_logp(const ScoreArgs &a, MaxSum r, float x) {
    if (r.s == 0.0f) return -INFINITY;
    return (double)(x - finite_or_zero(r.m)) * a.inv_t - log((double)r.s);
}
__device__ __forceinline__ float inverse_sum(MaxSum r) { return r.s == 0.0f ? 0.0f : 1.0f / r.s; }

// The policy loss of a token and its derivative by logp: -min(r A, clip(r) A) + kl (exp(ref - logp) - (ref - logp) - 1), r = exp(logp - old).
// An advantage of zero has no share in it, however far apart the two policies are, a weight of zero no loss.
__device__ __forceinline__ void policy_row(const ScoreArgs &a, int64_t row, float w, double logp, float &loss, float &slope) {
    double l = 0.0, d = 0.0;
    const double adv = a.adv[row];
    if (adv != 0.0) {
        const double r = exp(logp - (double)a.old_logp[row]);
        const double lo = 1.0 - a.clip_lo, hi = 1.0 + a.clip_hi;
        const double held = (r < lo ? lo : r > hi ? hi : r) * adv, free = r * adv; // a NaN stays one
        l = free <= held ? -free : -held;
        d = free <= held ? -free : 0.0;
        if (free != free) l = d = free;
    }
    if (a.kl != 0.0) {
        const double back = (double)a.ref_logp[row] - logp;
        const double e = expm1(back);
        l += a.kl * (e - back);
        d -= a.kl * e;
    }
    loss = w == 0.0f ? 0.0f : (float)((double)w * l);
    slope = w == 0.0f ? 0.0f : (float)((double)w * d);
}

// One block to a row, two passes over its scores: the simplest form.
template <typename T, int OP>
__global__ __launch_bounds__(256) void k_scores(ScoreArgs a) {
    constexpr int WAVES = 4;
    const int64_t row = blockIdx.x;
    const int t = threadIdx.x, V = a.V;
    const T *x = (const T *)a.x + row * a.xs;
    T *g = a.g ? (T *)a.g + row * a.gs : nullptr;
    const float w = a.weights ? a.weights[row] : 1.0f;
    __shared__ float s_p[OP == SC_DISTILL ? EVT_SCORES_MAX_TOP : 1], s_x[OP == SC_DISTILL ? EVT_SCORES_MAX_TOP : 1];
    __shared__ int32_t s_id[OP == SC_DISTILL ? EVT_SCORES_MAX_TOP : 1];
    bool live = OP != SC_DISTILL || w != 0.0f, bad = false;
    int64_t label = -1;
    float x_label = 0.0f, slope = 0.0f;
    MaxSum teacher = {-INFINITY, 0.0f};
    if (a.bounds) live = live && row >= a.bounds[0] && row < a.bounds[a.n_bounds - 1];
    if (OP == SC_DISTILL) {
        if (live) { // uniform
            bool mine = false;
            for (int j = t; j < a.n_top; j += 256) {
                const int64_t id = load_id(a.ids, a.id64, row * a.n_top + j);
                const float s = id < 0 ? -INFINITY : load_score(a.top, a.top_type, row * a.n_top + j);
                mine |= id >= V;
                s_id[j] = id < 0 || id >= V ? -1 : (int32_t)id;
                s_x[j] = id < 0 || id >= V ? 0.0f : (float)x[id];
                s_p[j] = s;
                teacher = join(teacher, {s, s == -INFINITY ? 0.0f : s - s + 1.0f}, a.exp_mul);
            }
            bad = __syncthreads_or(mine);
            teacher = block_join<WAVES>(teacher, a.exp_mul);
            live = teacher.s != 0.0f; // a NaN is live
        }
    } else {
        label = load_id(a.labels, a.label64, row);
        live = live && label >= 0;
        if (OP == SC_GRAD && live) {
            slope = a.slope[row];
            live = slope != 0.0f; // nothing asked of it: not read
        }
        bad = live && label >= V;
        if (live && !bad) x_label = (float)x[label];
    }
    if (!live) { // the row has no part in the loss
        if (t == 0) {
            if (OP != SC_GRAD && OP != SC_LOGP) a.loss[row] = 0.0f;
            if (OP == SC_LOGP || OP == SC_POLICY) a.logp[row] = 0.0f;
            if (OP == SC_LOGP && a.stats) a.stats[2 * row] = a.stats[2 * row + 1] = 0.0f;
            if (OP == SC_LOGP && a.slope) a.slope[row] = 0.0f;
        }
        if (OP != SC_LOGP && g)
            for (int c = t; c < V; c += 256) g[c] = (T)0.0f;
        return;
    }
    MaxSum r = {-INFINITY, 0.0f};
    if (OP == SC_GRAD) r = {a.stats[2 * row], a.stats[2 * row + 1]};
    else {
        for (int c = t; c < V; c += 256) {
            const float v = (float)x[c];
            r = join(r, {v, v == -INFINITY ? 0.0f : v - v + 1.0f}, a.exp_mul); // 1, or a NaN for a score that is none
        }
        r = block_join<WAVES>(r, a.exp_mul);
    }
    const float z = finite_or_zero(r.m), inv = inverse_sum(r);
    float factor = 0.0f; // of q
    if (OP == SC_DISTILL) {
        const double log_ts = log((double)teacher.s);
        const double log_s = r.s == 0.0f ? 0.0 : log((double)r.s);
        const float tz = finite_or_zero(teacher.m);
        float sum = 0.0f;
        for (int j = t; j < a.n_top; j += 256) {
            const float d = s_p[j] - tz, p = __builtin_amdgcn_exp2f(d * a.exp_mul) / teacher.s;
            if (s_id[j] >= 0 && p != 0.0f) {
                const double lq = r.s == 0.0f ? -INFINITY : (double)(s_x[j] - z) * a.inv_t - log_s;
                sum += p * (float)((double)d * a.inv_t - log_ts - lq);
            }
            s_p[j] = p;
        }
        sum = block_sum<WAVES>(sum);
        if (t == 0) a.loss[row] = bad ? NAN : w * a.t2_mul * sum;
        factor = bad ? NAN : w * a.t_mul;
    } else if (OP == SC_GRAD) {
        slope = bad ? NAN : (float)(slope * a.inv_t);
        factor = -slope;
    } else {
        const double logp = bad ? NAN : row_logp(a, r, x_label);
        if (OP == SC_POLICY) {
            float loss;
            policy_row(a, row, w, logp, loss, slope);
            slope = (float)(slope * a.inv_t);
            factor = -slope;
            if (t == 0) a.loss[row] = loss;
        }
        if (t == 0) {
            a.logp[row] = (float)logp;
            if (OP == SC_LOGP && a.stats) a.stats[2 * row] = r.m, a.stats[2 * row + 1] = r.s;
            if (OP == SC_LOGP && a.slope) a.slope[row] = 0.0f;
        }
    }
    if (OP == SC_LOGP || !g) return;
    if (OP == SC_POLICY && slope == 0.0f) { // clipped
        __syncthreads(); // every thread has read its label's score
        for (int c = t; c < V; c += 256) g[c] = (T)0.0f;
        return;
    }
    const float fq = factor * inv;
    __syncthreads(); // every score of another thread's class has been read
    for (int c = t; c < V; c += 256) g[c] = (T)(fq * __builtin_amdgcn_exp2f(((float)x[c] - z) * a.exp_mul));
    __syncthreads();
    if (OP == SC_DISTILL) {
        for (int j = t; j < a.n_top; j += 256) {
            const int32_t id = s_id[j];
            if (id < 0) continue;
            float p = 0.0f; // an id that comes twice has both shares
            for (int i = 0; i < a.n_top; i++) p += s_id[i] == id ? s_p[i] : 0.0f;
            g[id] = (T)(factor * (__builtin_amdgcn_exp2f((s_x[j] - z) * a.exp_mul) * inv - p));
        }
    } else if (t == 0 && !bad) {
        g[label] = (T)(slope * (1.0f - __builtin_amdgcn_exp2f((x_label - z) * a.exp_mul) * inv));
    }
}

// Every pair's loss: the sequences' sums of logp (means with `average`), h = beta ((lp_c - lp_r) - (ref_c - ref_r)) - margin,
// loss = w (-(1 - e) log sigma(h) - e log sigma(-h)), and the slope dloss / dlogp of every row of the two.  Sequences 0 .. pairs - 1 are the chosen
// ones, the rest the rejected.  One block to a pair; sums of 64 bits in an order that the lengths alone decide.
__global__ __launch_bounds__(1024) void k_scores_pairs(ScoreArgs a, int pairs, const float *__restrict__ ref_logp, double beta, double soft, double margin,
                                                       int average, float *__restrict__ seq_logp) {
    __shared__ double s_sum[2][16];
    __shared__ int s_cnt[2][16];
    const int t = threadIdx.x, p = blockIdx.x;
    int64_t from[2], to[2];
    double lp[2], len[2];
    bool bad = false;
    for (int k = 0; k < 2; k++) {
        from[k] = a.bounds[p + k * pairs];
        to[k] = a.bounds[p + k * pairs + 1];
        if (from[k] < 0 || to[k] > a.N || to[k] < from[k]) { // not ascending, or out of the rows
            bad = true;
            from[k] = to[k] = 0;
        }
        double sum = 0.0;
        int cnt = 0;
        for (int64_t i = from[k] + t; i < to[k]; i += 1024) {
            sum += (double)a.logp[i];
            cnt += load_id(a.labels, a.label64, i) >= 0;
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) {
            sum += __shfl_xor(sum, o);
            cnt += __shfl_xor(cnt, o);
        }
        if ((t & 63) == 0) s_sum[k][t >> 6] = sum, s_cnt[k][t >> 6] = cnt;
    }
    __syncthreads();
    for (int k = 0; k < 2; k++) {
        double sum = 0.0;
        int cnt = 0;
        for (int w = 0; w < 16; w++) sum += s_sum[k][w], cnt += s_cnt[k][w];
        len[k] = average && cnt ? cnt : 1;
        lp[k] = sum / len[k];
    }
    const double w = a.weights ? a.weights[p] : 1.0;
    const double h = beta * ((lp[0] - lp[1]) - ((double)ref_logp[p] - (double)ref_logp[p + pairs])) - margin;
    const double up = log1p(exp(-fabs(h))) + (h < 0.0 ? -h : 0.0); // -log sigma(h)
    const double sig = h < 0.0 ? exp(h) / (1.0 + exp(h)) : 1.0 / (1.0 + exp(-h));
    // the smaller of the two probabilities exactly: 1 - sigma(h) where h is large is sigma(-h)
    const double lose = h < 0.0 ? 1.0 / (1.0 + exp(h)) : exp(-h) / (1.0 + exp(-h));
    double dh = w * (soft * sig - (1.0 - soft) * lose);
    double loss = w * (up + (soft != 0.0 ? soft * h : 0.0));
    if (w == 0.0) dh = loss = 0.0;
    if (bad) dh = loss = NAN;
    if (t == 0) {
        a.loss[p] = (float)loss;
        seq_logp[p] = bad ? NAN : (float)lp[0];
        seq_logp[p + pairs] = bad ? NAN : (float)lp[1];
    }
    for (int k = 0; k < 2; k++) {
        const float d = (float)((k ? -dh : dh) * beta / len[k]);
        for (int64_t i = from[k] + t; i < to[k]; i += 1024) a.slope[i] = d;
    }
}

template <int OP>
static int launch_scores(hipStream_t s, const ScoreArgs &a, int dtype) {
    const dim3 grid((unsigned)a.N), block(256);
    if (dtype == EVT_F32) hipLaunchKernelGGL((k_scores<float, OP>), grid, block, 0, s, a);
    else if (dtype == EVT_BF16) hipLaunchKernelGGL((k_scores<bf16_t, OP>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((k_scores<half_t, OP>), grid, block, 0, s, a);
    HIPCHK(hipGetLastError());
    return EVT_OK;
}

// ---- entry points ---------------------------------------------------------------------------
static bool on_device(const void *p) {
    hipPointerAttribute_t attr;
    const bool ok = hipPointerGetAttributes(&attr, p) == hipSuccess && attr.devicePointer != nullptr &&
                    (attr.type == hipMemoryTypeDevice || attr.type == hipMemoryTypeHost || attr.type == hipMemoryTypeManaged);
    (void)hipGetLastError();
    return ok;
}
template <typename... P>
static int check_device(int32_t flags, P... ptrs) {
    if (flags & EVT_STATIC_TRUSTED) return EVT_OK;
    const void *all[] = {(const void *)ptrs...};
    for (const void *p : all) ARGCHK(!p || on_device(p), "losses over class scores take device memory only");
    return EVT_OK;
}

// The checks that every entry point makes of its scores; fills in what they say.
static int take_scores(const evt_scores *s, bool grad_needed, int32_t flags, ScoreArgs &a) {
    ARGCHK(s, "scores must not be NULL");
    ARGCHK(flags == 0 || flags == EVT_STATIC_TRUSTED, "flags takes 0 or EVT_STATIC_TRUSTED");
    ARGCHK(s->dtype == EVT_F32 || s->dtype == EVT_BF16 || s->dtype == EVT_F16, "scores must be EVT_F32, EVT_BF16 or EVT_F16");
    ARGCHK(s->nrows >= 0 && s->nrows <= INT32_MAX && s->nclass >= 1, "nrows must be in [0, 2^31 - 1], nclass >= 1");
    ARGCHK(s->temperature > 0.0 && s->temperature < INFINITY, "temperature must be positive and finite");
    a.N = s->nrows;
    a.V = s->nclass;
    if (a.N == 0) return EVT_OK;
    ARGCHK(s->x, "scores must not be NULL");
    ARGCHK(s->row_stride >= 0, "row_stride must not be negative");
    ARGCHK(s->grad || !grad_needed, "grad must not be NULL");
    const int size = s->dtype == EVT_F32 ? 4 : 2;
    ARGCHK((uintptr_t)s->x % size == 0 && (uintptr_t)s->grad % size == 0, "scores and gradients must be aligned to their type");
    if (s->grad) {
        ARGCHK(a.N == 1 || s->grad_stride >= s->nclass, "grad_stride must be at least nclass");
        if (!(s->grad == s->x && (a.N == 1 || s->grad_stride == s->row_stride))) { // in place, or apart
            const uintptr_t x0 = (uintptr_t)s->x, x1 = x0 + ((size_t)(a.N - 1) * s->row_stride + a.V) * size;
            const uintptr_t g0 = (uintptr_t)s->grad, g1 = g0 + ((size_t)(a.N - 1) * s->grad_stride + a.V) * size;
            ARGCHK(g1 <= x0 || x1 <= g0, "grad must be the scores' own memory, row for row, or lie apart from them");
        }
    }
    a.x = s->x;
    a.g = s->grad;
    a.xs = s->row_stride;
    a.gs = s->grad_stride;
    a.inv_t = 1.0 / s->temperature;
    a.exp_mul = (float)(1.4426950408889634 / s->temperature);
    a.t_mul = (float)s->temperature;
    a.t2_mul = (float)(s->temperature * s->temperature);
    return check_device(flags, s->x, s->grad);
}
static int take_labels(const void *labels, int32_t dtype, ScoreArgs &a) {
    ARGCHK(dtype == EVT_I32 || dtype == EVT_I64, "labels must be EVT_I32 or EVT_I64");
    ARGCHK(labels || a.N == 0, "labels must not be NULL");
    a.labels = labels;
    a.label64 = dtype == EVT_I64;
    return EVT_OK;
}
#define TRY(call)                        \
    do {                                 \
        const int _r = (call);           \
        if (_r != EVT_OK) return _r;     \
    } while (0)

extern "C" int evt_class_logp(void *stream, const evt_scores *s, const void *labels, int32_t label_dtype, float *logp, float *stats, int32_t flags) {
    return guarded([&]() -> int {
    ScoreArgs a = {};
    TRY(take_scores(s, false, flags, a));
    TRY(take_labels(labels, label_dtype, a));
    if (a.N == 0) return EVT_OK;
    ARGCHK(logp && stats, "logp and stats must not be NULL");
    TRY(check_device(flags, labels, logp, stats));
    a.logp = logp;
    a.stats = stats;
    return launch_scores<SC_LOGP>((hipStream_t)stream, a, s->dtype);
    });
}

extern "C" int evt_class_logp_grad(void *stream, const evt_scores *s, const void *labels, int32_t label_dtype, const float *stats, const float *dlogp,
                                   int32_t flags) {
    return guarded([&]() -> int {
    ScoreArgs a = {};
    TRY(take_scores(s, true, flags, a));
    TRY(take_labels(labels, label_dtype, a));
    if (a.N == 0) return EVT_OK;
    ARGCHK(stats && dlogp, "stats and dlogp must not be NULL");
    TRY(check_device(flags, labels, stats, dlogp));
    a.stats = const_cast<float *>(stats);
    a.slope = const_cast<float *>(dlogp);
    return launch_scores<SC_GRAD>((hipStream_t)stream, a, s->dtype);
    });
}

extern "C" int evt_distill_loss(void *stream, const evt_scores *s, const void *top_ids, int32_t id_dtype, const void *top_scores, int32_t top_dtype,
                                int32_t n_top, const float *weights, float *loss, int32_t flags) {
    return guarded([&]() -> int {
    ScoreArgs a = {};
    TRY(take_scores(s, false, flags, a));
    ARGCHK(id_dtype == EVT_I32 || id_dtype == EVT_I64, "top_ids must be EVT_I32 or EVT_I64");
    ARGCHK(top_dtype == EVT_F32 || top_dtype == EVT_BF16 || top_dtype == EVT_F16, "top_scores must be EVT_F32, EVT_BF16 or EVT_F16");
    ARGCHK(n_top >= 1 && n_top <= EVT_SCORES_MAX_TOP, "n_top must be in [1, 1024]");
    if (a.N == 0) return EVT_OK;
    ARGCHK(top_ids && top_scores && loss, "top_ids, top_scores and loss must not be NULL");
    TRY(check_device(flags, top_ids, top_scores, weights, loss));
    a.ids = top_ids;
    a.id64 = id_dtype == EVT_I64;
    a.top = top_scores;
    a.top_type = top_dtype;
    a.n_top = n_top;
    a.weights = weights;
    a.loss = loss;
    return launch_scores<SC_DISTILL>((hipStream_t)stream, a, s->dtype);
    });
}

extern "C" int evt_policy_loss(void *stream, const evt_scores *s, const void *labels, int32_t label_dtype, const float *old_logp, const float *advantages,
                               const float *ref_logp, const float *weights, double clip_low, double clip_high, double kl_coef, float *loss, float *logp,
                               int32_t flags) {
    return guarded([&]() -> int {
    ScoreArgs a = {};
    TRY(take_scores(s, false, flags, a));
    TRY(take_labels(labels, label_dtype, a));
    ARGCHK(clip_low >= 0.0 && clip_low <= 1.0 && clip_high >= 0.0, "clip_low must be in [0, 1], clip_high >= 0");
    ARGCHK(kl_coef >= 0.0 && kl_coef < INFINITY, "kl_coef must be >= 0 and finite");
    if (a.N == 0) return EVT_OK;
    ARGCHK(kl_coef == 0.0 || ref_logp, "ref_logp must not be NULL with a kl_coef");
    ARGCHK(old_logp && advantages && loss && logp, "old_logp, advantages, loss and logp must not be NULL");
    TRY(check_device(flags, labels, old_logp, advantages, ref_logp, weights, loss, logp));
    a.old_logp = old_logp;
    a.adv = advantages;
    a.ref_logp = ref_logp;
    a.weights = weights;
    a.clip_lo = clip_low;
    a.clip_hi = clip_high;
    a.kl = kl_coef;
    a.loss = loss;
    a.logp = logp;
    return launch_scores<SC_POLICY>((hipStream_t)stream, a, s->dtype);
    });
}

extern "C" int evt_preference_loss(void *stream, const evt_scores *s, const void *labels, int32_t label_dtype, const int32_t *offsets, int32_t n_pairs,
                                   const float *ref_logp, const float *weights, double beta, double label_smoothing, double margin, int32_t average,
                                   float *loss, float *seq_logp, float *work, int32_t flags) {
    return guarded([&]() -> int {
    ScoreArgs a = {};
    TRY(take_scores(s, false, flags, a));
    TRY(take_labels(labels, label_dtype, a));
    ARGCHK(n_pairs >= 1 && n_pairs < (1 << 30), "n_pairs must be in [1, 2^30 - 1]");
    ARGCHK(beta > 0.0 && beta < INFINITY && label_smoothing >= 0.0 && label_smoothing <= 0.5 && margin > -INFINITY && margin < INFINITY,
           "beta must be positive, label_smoothing in [0, 0.5], margin finite");
    ARGCHK(average == 0 || average == 1, "average takes 0 or 1");
    ARGCHK(offsets && ref_logp && loss && seq_logp, "offsets, ref_logp, loss and seq_logp must not be NULL");
    ARGCHK(work || a.N == 0, "work must not be NULL");
    TRY(check_device(flags, labels, offsets, ref_logp, weights, loss, seq_logp, work));
    const hipStream_t st = (hipStream_t)stream;
    a.bounds = offsets;
    a.n_bounds = 2 * n_pairs + 1;
    a.logp = work;
    a.slope = work + a.N;
    a.stats = work + 2 * a.N;
    a.loss = loss;
    if (a.N) TRY(launch_scores<SC_LOGP>(st, a, s->dtype));
    ScoreArgs pa = a;
    pa.weights = weights;
    hipLaunchKernelGGL(k_scores_pairs, dim3((unsigned)n_pairs), dim3(1024), 0, st, pa, n_pairs, ref_logp, beta, label_smoothing,
                       margin, average, seq_logp);
    HIPCHK(hipGetLastError());
    if (!a.N || !a.g) return EVT_OK;
    return launch_scores<SC_GRAD>(st, a, s->dtype);
    });
}
