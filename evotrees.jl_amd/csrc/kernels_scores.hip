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
#include "pieces.h"
#include <math.h>

// (m, s): the maximum of some scores, at least the lowest finite number, and the sum of their exp((x - m) / T).  Scores of -inf count nothing, a
// NaN or +inf makes s a NaN, and s is 0 where every score is -inf.
struct MaxSum {
    float m, s;
};
#define LOWEST (-3.402823466e38f)
__device__ __forceinline__ float exp_of(float x, float m, float mul) { return __builtin_amdgcn_exp2f((x - m) * mul); }
// a with E more scores
template <int E>
__device__ __forceinline__ MaxSum take(MaxSum a, const float *f, float mul) {
    float m = a.m;
#pragma unroll
    for (int k = 0; k < E; k++) m = fmaxf(m, f[k]);
    float s[E];
#pragma unroll
    for (int k = 0; k < E; k++) s[k] = exp_of(f[k], m, mul);
#pragma unroll
    for (int w = E / 2; w > 0; w /= 2)
#pragma unroll
        for (int k = 0; k < w; k++) s[k] += s[k + w];
    return {m, a.s * exp_of(a.m, m, mul) + s[0]};
}
template <int G>
__device__ __forceinline__ MaxSum lanes_join(MaxSum a, float mul) {
    const float m = over_lanes<G>(a.m, [](float x, float y) { return fmaxf(x, y); });
    return {m, lanes_sum<G>(a.s * exp_of(a.m, m, mul))};
}
// What every lane of a wavefront has alike, in scalar registers: a block that holds 16 pieces a thread has no vector register to spare
__device__ __forceinline__ float uniform(float v) { return __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(v))); }
__device__ __forceinline__ MaxSum uniform(MaxSum a) { return {uniform(a.m), uniform(a.s)}; }
// v, of which the compiler does not know that it is v: what is computed from it is computed where it is used, and does not stay in registers from the
// loads to the stores (16 offsets did, in pairs: 128 registers and spills in the largest blocks, 111 and none so)
__device__ __forceinline__ int again(int v) {
    asm volatile("" : "+v"(v));
    return v;
}
template <int G>
__device__ __forceinline__ bool lanes_any(bool v) {
    const uint64_t set = __ballot(v);
    return G == 64 ? set != 0 : ((set >> (threadIdx.x & 63 & ~(G - 1))) & ((1ull << (G & 63)) - 1)) != 0;
}

// The threads that share a row: G lanes of a wavefront, or W whole wavefronts, a block.
template <int G>
struct Lanes {
    static constexpr int SIZE = G, ROWS = 256 / G, THREADS = 256;
    __device__ static int rank() { return threadIdx.x & (G - 1); }
    __device__ static int slot() { return threadIdx.x / G; } // of the block's rows
    __device__ static void sync() {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
    __device__ static MaxSum all(MaxSum a, float mul) { // the group's joined; what its lanes wrote to shared memory before can be read
        a = lanes_join<G>(a, mul);
        sync();
        return a;
    }
};
template <int W>
struct Waves {
    static constexpr int SIZE = 64 * W, ROWS = 1, THREADS = 64 * W;
    __device__ static int rank() { return threadIdx.x; }
    __device__ static int slot() { return 0; }
    __device__ static void sync() { __syncthreads(); }
    __device__ static MaxSum all(MaxSum a, float mul) {
        __shared__ MaxSum s_a[W];
        a = lanes_join<64>(a, mul);
        if ((threadIdx.x & 63) == 0) s_a[threadIdx.x >> 6] = a;
        __syncthreads();
        return uniform(lanes_join<W>(s_a[threadIdx.x & (W - 1)], mul));
    }
};

__device__ __forceinline__ int64_t load_id(const void *p, int wide, int64_t i) { return wide ? ((const int64_t *)p)[i] : ((const int32_t *)p)[i]; }
__device__ __forceinline__ float load_score(const void *p, int type, int64_t i) {
    return type == EVT_F32 ? ((const float *)p)[i] : type == EVT_BF16 ? (float)((const bf16_t *)p)[i] : (float)((const half_t *)p)[i];
}

// log(s) to 3e-8: the exponent's share in 64 bits, the mantissa's, of at most 0.35, in 32.  (In 32 bits altogether the logarithm of a sum over a large
// vocabulary is off by 5e-7; in 64 it is some hundred instructions of every wavefront.)
__device__ __forceinline__ double log_sum(float s) {
    int k;
    float f = frexpf(s, &k);
    if (f < 0.70710678f) f += f, k--;
    return (double)k * 0.6931471805599453 + (double)logf(f);
}
// A row of score x at its label: its log-probability.  Nothing is left of a row whose scores are all -inf: every class has probability 0.
// 64 bits for the two terms: a policy's ratio is compared with its bounds.
__device__ __forceinline__ double row_logp(const ScoreArgs &a, MaxSum r, float x) {
    if (r.s == 0.0f) return -INFINITY;
    return (double)(x - r.m) * a.inv_t - log_sum(r.s);
}
__device__ __forceinline__ float inverse_sum(MaxSum r) { return r.s == 0.0f ? 0.0f : 1.0f / r.s; }

// exp(x) with 32 bits of digits and the exponents of 64
__device__ __forceinline__ double exp_wide(double x) {
    x = x > 1500.0 ? 1500.0 : x < -1500.0 ? -1500.0 : x; // infinite or 0 either way; a NaN stays
    const int k = x == x ? (int)rint(x * 1.4426950408889634) : 0;
    return ldexp((double)expf((float)(x - k * 0.6931471805599453)), k);
}
// The policy loss of a token and its derivative by logp: -min(r A, clip(r) A) + kl (exp(b) - b - 1), r = exp(logp - old), b = ref - logp.
// The differences are 64-bit, and the side of the bounds that r is on is found from them: a ratio next to a bound has a whole row's gradient or none.
// An advantage of zero has no share in it, however far apart the two policies are, a weight of zero no loss.
__device__ __forceinline__ void policy_row(const ScoreArgs &a, int64_t row, float w, double logp, float &loss, float &slope) {
    double l = 0.0, d = 0.0;
    const float adv = a.adv[row];
    if (adv != 0.0f) {
        const double gap = logp - (double)a.old_logp[row];
        // beyond float's range an advantage or a weight may bring the product back into it
        double ratio = expf((float)gap);
        if (__builtin_expect(fabsf((float)gap) > 80.0f, 0)) ratio = exp_wide(gap);
        const double free = -ratio * adv;
        if (adv > 0.0f ? gap > a.log_hi : adv < 0.0f && gap < a.log_lo) l = -(adv > 0.0f ? a.hi : a.lo) * adv;
        else l = d = free; // a NaN too, of the ratio or the advantage
    }
    if (a.kl != 0.0) {
        const double back = (double)a.ref_logp[row] - logp;
        const float b = (float)back, e32 = expm1f(b);
        // e - b cancels where the policies are close: there the series up to b^7 / 7!, the rest of which is under 2^-26 of it
        const float r32 = fabsf(b) < 0.25f ? b * b * (0.5f + b * (1.0f / 6 + b * (1.0f / 24 + b * (1.0f / 120 + b * (1.0f / 720 + b * (1.0f / 5040)))))) : e32 - b;
        double e = e32, rest = r32;
        if (__builtin_expect(b > 80.0f, 0)) {
            e = exp_wide(back);
            rest = e - back;
        }
        l += a.kl * rest;
        d -= a.kl * e;
    }
    loss = w == 0.0f ? 0.0f : (float)(w * l);
    slope = w == 0.0f ? 0.0f : (float)(w * d);
}

// What an operator makes of a labelled row's (m, s): its values are written by the thread that `writes`; the slope dloss / dx_label + ... = dloss /
// dlogp / T is returned (SC_LOGP: 0).
template <int OP>
__device__ __forceinline__ float labelled_row(const ScoreArgs &a, int64_t row, bool bad, MaxSum r, float x_label, float given, bool writes) {
    if (OP == SC_GRAD) return bad ? NAN : (float)(given * a.inv_t);
    const double logp = bad ? NAN : row_logp(a, r, x_label);
    float slope = 0.0f;
    if (OP == SC_POLICY) {
        float loss;
        policy_row(a, row, a.weights ? a.weights[row * a.ws] : 1.0f, logp, loss, slope);
        slope = (float)(slope * a.inv_t);
        if (writes) a.loss[row] = loss;
    }
    if (writes) {
        a.logp[row] = (float)logp;
        if (OP == SC_LOGP && a.stats) {
            a.stats[2 * row] = r.s == 0.0f ? -INFINITY : r.m;
            a.stats[2 * row + 1] = r.s;
        }
        if (OP == SC_LOGP && a.slope) a.slope[row] = 0.0f;
    }
    return slope;
}
template <int OP>
__device__ __forceinline__ void left_out(const ScoreArgs &a, int64_t row) {
    if ((OP == SC_DISTILL && a.loss) || OP == SC_POLICY) a.loss[row] = 0.0f;
    if (OP == SC_LOGP || OP == SC_POLICY) a.logp[row] = 0.0f;
    if (OP == SC_LOGP && a.stats) a.stats[2 * row] = a.stats[2 * row + 1] = 0.0f;
    if (OP == SC_LOGP && a.slope) a.slope[row] = 0.0f;
}

// A gradient of 0 for V classes
template <typename T>
__device__ __forceinline__ void clear_row(T *g, int V, int rank, int size, bool past) {
    constexpr int E = Piece<T>::E;
    Piece<T> p;
    p.r = {};
    const int n = V / E;
    for (int v = rank; v < n; v += size) p.store(g + (size_t)v * E, past);
    for (int c = n * E + rank; c < V; c += size) g[c] = (T)0.0f;
}

// E classes' gradients: fq * exp((x - m) / T), and at the label, if it is among them, slope (1 - q)
template <int E>
__device__ __forceinline__ void gradients(float *f, MaxSum r, float fq, float mul, int label_at, float slope, float inv) {
    float e[E];
#pragma unroll
    for (int k = 0; k < E; k++) e[k] = exp_of(f[k], r.m, mul);
#pragma unroll
    for (int k = 0; k < E; k++) f[k] = fq * e[k];
    if ((unsigned)label_at < (unsigned)E) {
#pragma unroll
        for (int k = 0; k < E; k++) f[k] = k == label_at ? slope * (1.0f - e[k] * inv) : f[k];
    }
}

// A row to a group of threads.  The first NV pieces of every thread stay in registers between the two passes over the row, the rest
// (rows of more classes than the largest form holds) is read again.  V is at least a piece's: the last one reaches back over classes of the one before it.
template <typename T, int OP, int NV, class G>
__global__ __launch_bounds__(G::THREADS) void k_rows(ScoreArgs a) {
    constexpr int E = Piece<T>::E;
    static_assert(OP != SC_DISTILL || G::ROWS == 1, "k_distill_short has the others");
    extern __shared__ __align__(16) unsigned char s_dyn[]; // SC_DISTILL: n_top (id, probability) pairs, then the scores of these classes
    __shared__ int s_state;                  // SC_DISTILL: 1 a teacher, 2 with an id of no class or a score that is no number or +inf
    const int64_t row = a.row0 + (int64_t)blockIdx.x * G::ROWS + G::slot();
    if (G::ROWS > 1 && row >= a.N) return;
    const int t = G::rank(), V = a.V;
    const T *x = (const T *)a.x + row * a.xs;
    T *g = a.g ? (T *)a.g + row * a.gs : nullptr;
    const float mul = a.exp_mul;
    // a teacher's classes are stored a second time: behind the caches that is a line read and written for each (89 448 x 3001 f32 of 32 entries: 520 us past the
    // caches, 462 not; 2048 x 131072 of 64 454 | 494)
    const bool past = a.past && (OP != SC_DISTILL || V > 4096 * E);
    float w = 1.0f, x_label = 0.0f, given = 0.0f;
    bool live = true, bad = false;
    int64_t label = -1;
    Piece<T> p[NV];
    // A piece at an odd 16-bit address costs (10 732 x 50 021 bf16, log-probabilities: 225 us, 181 so): in rows that start there pieces start an element earlier, the first of
    // them at the row's start all the same.  first: where the thread's piece would start; at: where it is
    const int base = sizeof(T) == 2 && ((uintptr_t)x & 2) ? -1 : 0;
    const auto at = [&](int first) { return first < 0 ? 0 : first + E <= V ? first : V - E; };
    if (OP == SC_DISTILL) {
        w = a.weights ? a.weights[row * a.ws] : 1.0f;
        live = w != 0.0f;
    } else {
        label = load_id(a.labels, a.label64, row);
        live = label >= 0;
        if (a.bounds) live = live && row >= a.bounds[0] && row < a.bounds[a.n_bounds - 1];
        if (OP == SC_GRAD && live) {
            given = a.slope[row];
            live = given != 0.0f; // nothing asked of it: not read
        }
        bad = live && label >= V;
        if (live && !bad) x_label = (float)x[label];
    }
    if (!live) { // the row has no part in the loss
        if (t == 0) left_out<OP>(a, row);
        if (OP != SC_LOGP && g) clear_row(g, V, t, G::SIZE, past);
        return;
    }
#pragma unroll
    for (int i = 0; i < NV; i++) {
        const int o = base + (t + i * G::SIZE) * E;
        // past the row's end: the last piece, which counts once.  Lanes leave out what no lane has; between the loads of a block the branches cost
        // more than the loads (8192 x 131072 bf16: 1020 for 790 us)
        if (G::ROWS == 1 || base + i * G::SIZE * E < V) p[i].load(x, at(o));
    }
    int2 *const s_top = (int2 *)s_dyn;
    float *const s_x = (float *)(s_top + a.n_top);
    MaxSum teacher = {LOWEST, 0.0f};
    if (OP == SC_DISTILL && t < 64) { // the first wavefront looks after the teacher while the row is on its way
        bool none = false;
#pragma unroll 1
        for (int j = t; j < a.n_top; j += 64) {
            const int64_t id = load_id(a.ids, a.id64, row * a.n_top + j);
            const float s = id < 0 ? -INFINITY : load_score(a.top, a.top_type, row * a.n_top + j);
            const bool in = id >= 0 && id < V;
            none |= id >= V;
            s_top[j] = {in ? (int)id : -1, __float_as_int(s)};
            s_x[j] = in ? (float)x[id] : 0.0f;
            teacher = take<1>(teacher, &s, mul);
        }
        teacher = uniform(lanes_join<64>(teacher, mul));
        none = __any(none);
        if (t == 0) s_state = teacher.s == 0.0f ? 0 : none || teacher.s != teacher.s ? 2 : 1;
#pragma unroll 1
        for (int j = t; j < a.n_top; j += 64) s_top[j].y = __float_as_int(exp_of(__int_as_float(s_top[j].y), teacher.m, mul) * (1.0f / teacher.s));
    }
    MaxSum r = {LOWEST, 0.0f};
    if (OP == SC_GRAD) {
        r = {fmaxf(a.stats[2 * row], LOWEST), a.stats[2 * row + 1]};
    } else {
        const int tt = again(t);
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const int o = base + (tt + i * G::SIZE) * E;
            if (o < V) {
                float f[E];
                p[i].get(f);
                const int off = at(o) - o; // not 0: classes that the piece behind or before counts
                if (off != 0) {
#pragma unroll
                    for (int k = 0; k < E; k++) f[k] = (unsigned)(k + off) < (unsigned)E ? f[k] : -INFINITY;
                }
                r = take<E>(r, f, mul);
            }
        }
        int64_t o = base + (int64_t)(t + NV * G::SIZE) * E;
        for (; o + 3 * G::SIZE * E + E <= V; o += 4 * G::SIZE * E) { // four pieces in flight
            Piece<T> q[4];
            float f[E];
#pragma unroll
            for (int i = 0; i < 4; i++) q[i].load(x + o + i * G::SIZE * E);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                q[i].get(f);
                r = take<E>(r, f, mul);
            }
        }
        for (; o < V; o += G::SIZE * E) {
            float f[E];
            if (o + E <= V) {
                Piece<T> q;
                q.load(x + o);
                q.get(f);
            } else {
#pragma unroll
                for (int k = 0; k < E; k++) f[k] = o + k < V ? (float)x[o + k] : -INFINITY;
            }
            r = take<E>(r, f, mul);
        }
        r = G::all(r, mul);
    }
    const float inv = inverse_sum(r);
    float fq, slope = 0.0f, factor = 0.0f;
    if (OP == SC_DISTILL) {
        const int state = s_state;
        if (state == 0) {
            if (t == 0) left_out<OP>(a, row);
            if (g) clear_row(g, V, t, G::SIZE, past);
            return;
        }
        if (t < 64) {
            // log p_j - log q_j = ((t_j - t_max) - (x_j - m)) / T + log(S / S_teacher), and the p_j add up to 1
            const double logs = r.s == 0.0f ? 0.0 : log_sum(r.s) - log_sum(teacher.s);
            float sum = 0.0f;
#pragma unroll 1
            for (int j = t; j < a.n_top; j += 64) {
                const int2 e = s_top[j];
                const float pj = __int_as_float(e.y);
                if (e.x >= 0 && pj != 0.0f) sum += pj * ((load_score(a.top, a.top_type, row * a.n_top + j) - teacher.m) - (s_x[j] - r.m));
            }
            sum = lanes_sum<64>(sum);
            if (t == 0 && a.loss) a.loss[row] = state == 2 ? NAN : w * a.t2_mul * (float)((double)sum * a.inv_t + logs);
        }
        factor = state == 2 ? NAN : w * a.t_mul;
    } else {
        slope = labelled_row<OP>(a, row, bad, r, x_label, given, t == 0);
        if (OP == SC_POLICY && slope == 0.0f && g) { // clipped, or of no weight
            clear_row(g, V, t, G::SIZE, past);
            return;
        }
        factor = -slope;
    }
    if (OP == SC_LOGP || !g) return;
    fq = factor * inv;
    const int tt = again(t);
#pragma unroll
    for (int i = 0; i < NV; i++) {
        int o = base + (tt + i * G::SIZE) * E;
        if (o < V) {
            o = at(o);
            float f[E];
            p[i].get(f);
            gradients<E>(f, r, fq, mul, OP == SC_DISTILL ? -1 : (int)(label - o), slope, inv);
            p[i].set(f);
            p[i].store(g, o, past);
        }
    }
    for (int64_t o = base + (int64_t)(t + NV * G::SIZE) * E; o < V; o += G::SIZE * E) {
        float f[E];
        if (o + E <= V) {
            Piece<T> q;
            q.load(x + o);
            q.get(f);
            gradients<E>(f, r, fq, mul, OP == SC_DISTILL ? -1 : (int)(label - o), slope, inv);
            q.set(f);
            q.store(g + o, past);
        } else { // not reaching back: in place, the classes in front are gradients already
            for (int64_t c = o; c < V; c++) {
                f[0] = (float)x[c];
                gradients<1>(f, r, fq, mul, OP == SC_DISTILL ? -1 : (int)(label - c), slope, inv);
                g[c] = (T)f[0];
            }
        }
    }
    if (OP == SC_DISTILL) { // the teacher's classes again, behind the others' stores
        G::sync();
        for (int j = t; j < a.n_top; j += G::SIZE) {
            const int id = s_top[j].x;
            if (id < 0) continue;
            float pj = 0.0f; // an id that comes twice has both shares
            for (int i = 0; i < a.n_top; i++) {
                const int2 e = s_top[i];
                pj += e.x == id ? __int_as_float(e.y) : 0.0f;
            }
            g[id] = (T)(factor * (exp_of(s_x[j], r.m, mul) * inv - pj));
        }
    }
}

// A row to a thread: fewer classes than a piece has.
template <typename T, int OP>
__global__ __launch_bounds__(256) void k_few_classes(ScoreArgs a) {
    constexpr int KM = Piece<T>::E;
    const int64_t row = a.row0 + (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (row >= a.N) return;
    const int V = a.V;
    const T *x = (const T *)a.x + row * a.xs;
    T *g = a.g ? (T *)a.g + row * a.gs : nullptr;
    const int64_t label = load_id(a.labels, a.label64, row);
    float given = 0.0f;
    bool live = label >= 0;
    if (a.bounds) live = live && row >= a.bounds[0] && row < a.bounds[a.n_bounds - 1];
    if (OP == SC_GRAD && live) {
        given = a.slope[row];
        live = given != 0.0f;
    }
    const bool bad = live && label >= V;
    if (!live) {
        left_out<OP>(a, row);
        if (OP != SC_LOGP && g) clear_row(g, V, 0, 1, false);
        return;
    }
    float f[KM], x_label = 0.0f;
#pragma unroll
    for (int k = 0; k < KM; k++) f[k] = (float)x[k < V ? k : V - 1];
#pragma unroll
    for (int k = 0; k < KM; k++) {
        f[k] = k < V ? f[k] : -INFINITY;
        x_label = k == (int)label ? f[k] : x_label;
    }
    MaxSum r = {LOWEST, 0.0f};
    if (OP == SC_GRAD) r = {fmaxf(a.stats[2 * row], LOWEST), a.stats[2 * row + 1]};
    else r = take<KM>(r, f, a.exp_mul);
    const float inv = inverse_sum(r), slope = labelled_row<OP>(a, row, bad, r, x_label, given, true);
    if (OP == SC_LOGP || !g) return;
    if (OP == SC_POLICY && slope == 0.0f) return clear_row(g, V, 0, 1, false);
    gradients<KM>(f, r, -slope * inv, a.exp_mul, (int)label, slope, inv);
#pragma unroll
    for (int k = 0; k < KM; k++)
        if (k < V) g[k] = (T)f[k];
}

// Distillation of rows that a group of lanes holds.  The entries of the block's rows are one stretch of memory: the block copies them to shared memory
// in whole lines (read by each row's lanes they are a line an entry: 8M rows of 16 bfloat16 classes and 16 entries 1.85 -> 0.50 ms), and a row's
// teacher is spread over all its classes there, so that no gradient is written twice.
template <typename T, int NV, class G>
__global__ __launch_bounds__(256) void k_distill_short(ScoreArgs a, uint32_t top_magic) {
    constexpr int E = Piece<T>::E;
    constexpr bool FEW = NV == 0; // V < E: every lane has the whole row, and shares the teacher's entries
    extern __shared__ __align__(16) unsigned char s_dyn[];
    const int V = a.V, k1 = a.n_top, ks = k1 | 1, vs = (V + 2) | 1; // odd distances: rows that lanes read side by side start in different banks
    int2 *const s_all = (int2 *)s_dyn; // (class, V for no entry, V + 1 for no class; score)
    float *const s_share = (float *)(s_all + G::ROWS * ks);
    const int64_t row0 = a.row0 + (int64_t)blockIdx.x * G::ROWS, row = row0 + G::slot();
    const int t = G::rank();
    const bool in_range = row < a.N;
    const T *x = (const T *)a.x + (in_range ? row : a.N - 1) * a.xs;
    T *g = a.g ? (T *)a.g + row * a.gs : nullptr;
    const float mul = a.exp_mul;
    const bool past = a.past;
    const float w = !in_range ? 0.0f : a.weights ? a.weights[row * a.ws] : 1.0f;
    Piece<T> p[FEW ? 1 : NV];
    float few[FEW ? E : 1];
    if constexpr (FEW) {
#pragma unroll
        for (int k = 0; k < E; k++) few[k] = (float)x[k < V ? k : V - 1];
    } else {
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const int o = (t + i * G::SIZE) * E;
            if (i * G::SIZE * E < V) p[i].load(x, o + E <= V ? o : V - E);
        }
    }
    {
        const int64_t at = row0 * k1, left = (a.N - row0) * k1;
        const int n = (int)(left < G::ROWS * k1 ? left : G::ROWS * k1);
        for (int e0 = threadIdx.x; e0 < n; e0 += 1024) { // four entries in flight
            int64_t id[4];
            float v[4];
#pragma unroll
            for (int i = 0; i < 4; i++) id[i] = load_id(a.ids, a.id64, at + (e0 + 256 * i < n ? e0 + 256 * i : n - 1));
#pragma unroll
            for (int i = 0; i < 4; i++) v[i] = load_score(a.top, a.top_type, at + (e0 + 256 * i < n ? e0 + 256 * i : n - 1));
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int e = e0 + 256 * i, r = k1 == 1 ? e : (int)__umulhi((uint32_t)e, top_magic); // e / n_top
                if (e < n) s_all[r * ks + e - r * k1] = {id[i] < 0 ? V : id[i] < V ? (int)id[i] : V + 1, __float_as_int(id[i] < 0 ? -INFINITY : v[i])};
            }
        }
        for (int e = threadIdx.x; e < G::ROWS * vs; e += 256) s_share[e] = 0.0f;
    }
    __syncthreads();
    if (w == 0.0f) {
        if (in_range) {
            if (t == 0) left_out<SC_DISTILL>(a, row);
            if (g) clear_row(g, V, t, G::SIZE, past);
        }
        return;
    }
    int2 *const s_top = s_all + G::slot() * ks;
    float *const share = s_share + G::slot() * vs;
    MaxSum r = {LOWEST, 0.0f};
    if constexpr (FEW) {
#pragma unroll
        for (int k = 0; k < E; k++) few[k] = k < V ? few[k] : -INFINITY;
        r = take<E>(r, few, mul);
    } else {
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const int o = (t + i * G::SIZE) * E;
            if (o < V) {
                float f[E];
                p[i].get(f);
                if (o + E > V) {
#pragma unroll
                    for (int k = 0; k < E; k++) f[k] = k < o + E - V ? -INFINITY : f[k];
                }
                r = take<E>(r, f, mul);
            }
        }
        r = lanes_join<G::SIZE>(r, mul);
    }
    // The teacher's entries, four at a time, for each is a trip to shared memory or two: their maximum while each leaves its number at its class, then
    // exp of each in the number's place - another number there is an entry of the same class.  (Added up there by float atomics, some 165 cycles a
    // wavefront each, 8M rows of 7 classes and entries take 347 us for 237.)
    float most = LOWEST, total = 0.0f, sum = 0.0f;
    bool none = false, twice = false;
    for (int j0 = t; j0 < k1; j0 += 4 * G::SIZE) {
        int2 e[4];
#pragma unroll
        for (int i = 0; i < 4; i++) e[i] = s_top[j0 + i * G::SIZE < k1 ? j0 + i * G::SIZE : j0];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            most = fmaxf(most, __int_as_float(e[i].y));
            none |= e[i].x == V + 1;
            if (j0 + i * G::SIZE < k1) share[e[i].x] = __int_as_float(j0 + i * G::SIZE);
        }
    }
    G::sync();
    most = over_lanes<G::SIZE>(most, [](float a, float b) { return fmaxf(a, b); });
    for (int j0 = t; j0 < k1; j0 += 4 * G::SIZE) {
        int2 e[4];
        float at[4];
#pragma unroll
        for (int i = 0; i < 4; i++) e[i] = s_top[j0 + i * G::SIZE < k1 ? j0 + i * G::SIZE : j0];
#pragma unroll
        for (int i = 0; i < 4; i++) at[i] = share[e[i].x];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if (j0 + i * G::SIZE < k1) {
                const float d = __int_as_float(e[i].y) - most, u = __builtin_amdgcn_exp2f(d * mul);
                total += u;
                sum += u != 0.0f ? u * d : 0.0f;
                share[e[i].x] = u;
                twice |= e[i].x < V && __float_as_int(at[i]) != j0 + i * G::SIZE;
            }
        }
    }
    total = lanes_sum<G::SIZE>(total);
    sum = lanes_sum<G::SIZE>(sum);
    none = lanes_any<G::SIZE>(none);
    if (total == 0.0f) { // no entry; a total that is no number is one
        if (t == 0) left_out<SC_DISTILL>(a, row);
        if (g) clear_row(g, V, t, G::SIZE, past);
        return;
    }
    if (lanes_any<G::SIZE>(twice)) { // a class that comes twice has both shares, added up in their order
        G::sync();
        for (int j = t; j < k1; j += G::SIZE) {
            const int id = s_top[j].x;
            if (id >= V) continue;
            float u = 0.0f;
            for (int i = 0; i < k1; i++) {
                const int2 e = s_top[i];
                u += e.x == id ? __builtin_amdgcn_exp2f((__int_as_float(e.y) - most) * mul) : 0.0f;
            }
            share[id] = u;
        }
    }
    G::sync();
    const float one = 1.0f / total, factor = none ? NAN : w * a.t_mul, fq = factor * inverse_sum(r), fp = factor * one;
    float cross = 0.0f; // the sum of share (x - m)
    if constexpr (FEW) {
#pragma unroll
        for (int k = 0; k < E; k++) {
            const float u = share[k < V ? k : V - 1];
            if (k < V && u != 0.0f) cross += u * (few[k] - r.m);
            if (g && k < V && t == 0) g[k] = (T)(fq * exp_of(few[k], r.m, mul) - fp * u);
        }
    } else {
#pragma unroll
        for (int i = 0; i < NV; i++) {
            int o = (t + i * G::SIZE) * E;
            if (o < V) {
                const int twofold = o + E <= V ? 0 : o + E - V; // classes of the piece before
                o = o + E <= V ? o : V - E;
                float f[E];
                p[i].get(f);
#pragma unroll
                for (int k = 0; k < E; k++) {
                    const float u = share[o + k], d = f[k] - r.m;
                    cross += u != 0.0f && k >= twofold ? u * d : 0.0f; // not 0 times infinity
                    f[k] = fq * __builtin_amdgcn_exp2f(d * mul) - fp * u;
                }
                if (g) {
                    p[i].set(f);
                    p[i].store(g, o, past);
                }
            }
        }
        cross = lanes_sum<G::SIZE>(cross);
    }
    if (t == 0 && a.loss) {
        const double logs = r.s == 0.0f ? 0.0 : log_sum(r.s * one);
        a.loss[row] = none ? NAN : w * a.t2_mul * (float)((double)((sum - cross) * one) * a.inv_t + logs);
    }
}

// What the pairs' loss is computed from beside the rows' log-probabilities
struct PairArgs {
    int pairs, average;
    const float *ref_logp, *weights;
    double beta, soft, margin;
    float *seq_logp;
};
// A pair's loss by a block of 64 W threads: the sequences' sums of logp (means with `average`), h = beta ((lp_c - lp_r) - (ref_c - ref_r)) - margin,
// loss = w (-(1 - e) log sigma(h) - e log sigma(-h)), and the slope dloss / dlogp of a row of either.  Sequences 0 .. pairs - 1 are the chosen
// ones, the rest the rejected.  Sums of 64 bits in an order that the lengths and W decide.
struct Pair {
    int64_t from[2], to[2];
    double lp[2];
    float loss, slope[2];
    bool bad;
};
// Rows from .. to - 1 ascend, are rows of the scores and lie between the first offset and the last: rows outside have no logp
__device__ __forceinline__ bool is_sequence(const ScoreArgs &a, int64_t from, int64_t to, int64_t first, int64_t last) {
    return from >= 0 && to <= a.N && from <= to && from >= first && to <= last;
}
// flag: one thread's, and then any thread's
template <int W>
__device__ __forceinline__ Pair pair_loss(const ScoreArgs &a, const PairArgs &q, int p, bool &flag) {
    __shared__ double s_sum[2][W];
    __shared__ int s_cnt[2][W], s_flag[W];
    const int t = threadIdx.x;
    Pair r;
    double len[2];
    int cnt[2] = {0, 0};
    const int64_t first = a.bounds[0], last = a.bounds[a.n_bounds - 1];
    r.bad = false;
#pragma unroll
    for (int k = 0; k < 2; k++) {
        r.from[k] = a.bounds[p + k * q.pairs];
        r.to[k] = a.bounds[p + k * q.pairs + 1];
        r.lp[k] = 0.0;
    }
#pragma unroll
    for (int k = 0; k < 2; k++) {
        if (!is_sequence(a, r.from[k], r.to[k], first, last)) {
            r.bad = true;
            r.from[k] = r.to[k] = 0;
        }
    }
    const int64_t longer = r.to[0] - r.from[0] > r.to[1] - r.from[1] ? r.to[0] - r.from[0] : r.to[1] - r.from[1];
    for (int64_t i = t; i < longer; i += 64 * W) {
#pragma unroll
        for (int k = 0; k < 2; k++) {
            if (r.from[k] + i < r.to[k]) {
                r.lp[k] += (double)a.logp[r.from[k] + i];
                cnt[k] += load_id(a.labels, a.label64, r.from[k] + i) >= 0;
            }
        }
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1)
#pragma unroll
        for (int k = 0; k < 2; k++) {
            r.lp[k] += __shfl_xor(r.lp[k], o);
            cnt[k] += __shfl_xor(cnt[k], o);
        }
    flag = __any(flag);
    if ((t & 63) == 0) {
        for (int k = 0; k < 2; k++) s_sum[k][t >> 6] = r.lp[k], s_cnt[k][t >> 6] = cnt[k];
        s_flag[t >> 6] = flag;
    }
    __syncthreads();
    flag = __any(s_flag[t & (W - 1)]);
#pragma unroll
    for (int k = 0; k < 2; k++) {
        r.lp[k] = s_sum[k][t & (W - 1)];
        cnt[k] = s_cnt[k][t & (W - 1)];
    }
#pragma unroll
    for (int o = W / 2; o > 0; o >>= 1)
#pragma unroll
        for (int k = 0; k < 2; k++) {
            r.lp[k] += __shfl_xor(r.lp[k], o);
            cnt[k] += __shfl_xor(cnt[k], o);
        }
#pragma unroll
    for (int k = 0; k < 2; k++) {
        len[k] = q.average && cnt[k] ? cnt[k] : 1;
        r.lp[k] /= len[k];
    }
    const double w = q.weights ? q.weights[p] : 1.0;
    const double h = q.beta * ((r.lp[0] - r.lp[1]) - ((double)q.ref_logp[p] - (double)q.ref_logp[p + q.pairs])) - q.margin;
    const double e = exp(-fabs(h)), one = log1p(e), up = one + (h < 0.0 ? -h : 0.0), down = one + (h > 0.0 ? h : 0.0); // -log sigma(h), -log sigma(-h)
    // the smaller of the two probabilities exactly: 1 - sigma(h) where h is large is sigma(-h)
    const double sig = (h < 0.0 ? e : 1.0) / (1.0 + e), lose = (h < 0.0 ? 1.0 : e) / (1.0 + e);
    double dh = w * (q.soft * sig - (1.0 - q.soft) * lose), loss = w * up;
    // an answer that cannot be has an infinite h: the two terms apart, neither of which is a difference
    if (q.soft != 0.0) loss = w * ((1.0 - q.soft) * up + q.soft * down);
    if (w == 0.0) dh = loss = 0.0;
    if (r.bad) dh = loss = NAN;
    r.loss = (float)loss;
#pragma unroll
    for (int k = 0; k < 2; k++) r.slope[k] = (float)((k ? -dh : dh) * q.beta / len[k]) + 0.0f; // no -0: most_bits
    return r;
}
__device__ __forceinline__ void write_pair(const ScoreArgs &a, const PairArgs &q, int p, const Pair &r) {
    a.loss[p] = r.loss;
#pragma unroll
    for (int k = 0; k < 2; k++) q.seq_logp[p + k * q.pairs] = r.bad ? NAN : (float)r.lp[k];
}
// Sequences share rows only where offsets descend somewhere between them.  Such a row has the slope of the most bits, an order that depends neither on which
// block comes first nor on the form; a slope of 0, which SC_LOGP left as well, has none.
__device__ __forceinline__ uint32_t most_bits(uint32_t a, float slope) { return a > __float_as_uint(slope) ? a : __float_as_uint(slope); }
// One block to a pair, which leaves its slope at every row of the two: by atomics where the offsets descend, or are so many that looking costs more (one block's
// 500 000 rows: 370 us by atomics, 328 without)
#define LOOK_FOR_SHARED 4096 // offsets
template <int W>
__global__ __launch_bounds__(64 * W) void k_scores_pairs(ScoreArgs a, PairArgs q) {
    const int n = 2 * q.pairs;
    bool shared = n > LOOK_FOR_SHARED;
    if (!shared)
        for (int k = threadIdx.x; k < n; k += 64 * W) shared |= a.bounds[k + 1] < a.bounds[k];
    const Pair r = pair_loss<W>(a, q, blockIdx.x, shared);
    if (threadIdx.x == 0) write_pair(a, q, blockIdx.x, r);
#pragma unroll
    for (int k = 0; k < 2; k++) {
        if (shared)
            for (int64_t i = r.from[k] + threadIdx.x; i < r.to[k]; i += 64 * W) atomicMax((uint32_t *)&a.slope[i], most_bits(0, r.slope[k]));
        else
            for (int64_t i = r.from[k] + threadIdx.x; i < r.to[k]; i += 64 * W) a.slope[i] = r.slope[k];
    }
}

// The gradient of given slopes, where rows are long: nothing is joined, a block has a part of a row.
// PAIRS: of the preference loss, few blocks (all of them run at once): each finds its row's pair and the pair's slope by itself, a launch less (256 rows of
// 8192 bf16: 6.6 us for 5.0 + 4.8); the last blocks write the losses.
template <typename T, bool PAIRS>
__global__ __launch_bounds__(256) void k_slope_rows(ScoreArgs a, PairArgs q, int parts) {
    constexpr int E = Piece<T>::E;
    // classes, at most 1024 pieces; the parts alike (32 764 x 8193 bf16, 1025 pieces a row: 308 us by 1024 and 1, 224 so)
    const int part = ((a.V + E - 1) / E + parts - 1) / parts * E;
    __shared__ int2 s_two[4];
    const int64_t blocks = a.N * parts;
    const bool past = a.past;
    if (PAIRS && blockIdx.x >= blocks) {
        const int p = (int)(blockIdx.x - blocks);
        bool none = false;
        const Pair r = pair_loss<4>(a, q, p, none);
        if (threadIdx.x == 0) write_pair(a, q, p, r);
        return;
    }
    for (int64_t b = blockIdx.x; b < blocks; b += gridDim.x) {
        const int64_t row = b / parts;
        const int64_t c0 = (b - row * parts) * part;
        const T *x = (const T *)a.x + row * a.xs + c0;
        T *g = (T *)a.g + row * a.gs + c0;
        const int V = (int)(a.V - c0 < part ? a.V - c0 : part), t = threadIdx.x;
        const int64_t label = load_id(a.labels, a.label64, row);
        float given = 0.0f;
        bool live = label >= 0;
        if (!PAIRS && a.bounds) live = live && row >= a.bounds[0] && row < a.bounds[a.n_bounds - 1];
        if (PAIRS && live) { // the sequences that have the row: none, one, or more where offsets descend
            const int n = 2 * q.pairs, first = a.bounds[0] < 0 ? 0 : a.bounds[0], last = a.bounds[n] < a.N ? a.bounds[n] : (int)a.N, at = (int)row;
            uint32_t best = 0;
            for (int from = 0; from < n;) {
                int seq = -1, next = n; // the first of them from `from` on, and the one behind it
                // up to 64 by every wavefront, more by a wavefront each and handed round (1000 pairs, 1000 rows of 2048 bf16: 19.1 us by every one)
                const bool each = n - from <= 64;
                for (int k0 = each ? from : from + (t & ~63); k0 < n && next == n; k0 += 256) {
                    const int k = k0 + (t & 63), c = k < n ? k : n - 1, b0 = a.bounds[c], b1 = a.bounds[c + 1];
                    uint64_t has = __ballot(k < n && at >= b0 && at < b1 && b0 >= first && b1 <= last); // is_sequence
                    if (has && seq < 0) {
                        seq = k0 + __builtin_ctzll(has);
                        has &= has - 1;
                    }
                    if (has) next = k0 + __builtin_ctzll(has);
                }
                if (!each) {
                    if ((t & 63) == 0) s_two[t >> 6] = {seq, next};
                    __syncthreads();
                    seq = -1, next = n;
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const int2 two = s_two[i];
                        if (two.x < 0) continue;
                        const int later = seq < 0 ? n : seq < two.x ? two.x : seq; // the second of the two firsts
                        seq = seq < 0 || two.x < seq ? two.x : seq;
                        next = min(next, min(later, two.y));
                    }
                }
                if (seq < 0) break;
                if (from) __syncthreads(); // everyone has read the sums of the pair before
                bool none = false;
                const Pair r = pair_loss<4>(a, q, seq < q.pairs ? seq : seq - q.pairs, none);
                best = most_bits(best, r.slope[seq >= q.pairs]);
                from = next;
            }
            given = __uint_as_float(best);
        } else if (live) {
            given = a.slope[row];
        }
        if (given == 0.0f) {
            clear_row(g, V, t, 256, past);
            continue;
        }
        const MaxSum r = {fmaxf(a.stats[2 * row], LOWEST), a.stats[2 * row + 1]};
        const float inv = inverse_sum(r), slope = label >= a.V ? NAN : (float)(given * a.inv_t), fq = -slope * inv;
        const int64_t at = label - c0; // of the label, in this part if at all
        Piece<T> p[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int o = (t + i * 256) * E;
            if (o + E <= V) p[i].load(x + o);
        }
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int o = (t + i * 256) * E;
            float f[E];
            if (o + E <= V) {
                p[i].get(f);
                gradients<E>(f, r, fq, a.exp_mul, (int)(at - o), slope, inv);
                p[i].set(f);
                p[i].store(g + o, past);
            }
        }
        const int c = V / E * E + t; // behind the last whole piece
        if (c < V) {
            float f = (float)x[c];
            gradients<1>(&f, r, fq, a.exp_mul, (int)(at - c), slope, inv);
            g[c] = (T)f;
        }
    }
}

// A launch has fewer than 2^32 threads: more rows go in several.  f(args, blocks) for each
template <typename F>
static void slices(ScoreArgs a, int rows, int threads, F &&f) {
    const int64_t most = (int64_t)(1 << 22) * 1024 / threads - 1; // blocks
    for (a.row0 = 0; a.row0 < a.N; a.row0 += most * rows) {
        const int64_t left = (a.N - a.row0 + rows - 1) / rows;
        f(a, dim3((unsigned)(left < most ? left : most)));
    }
}
template <typename T, int OP, int NV, class G>
static int launch_rows(hipStream_t s, ScoreArgs a) {
    const size_t lds = OP == SC_DISTILL ? (size_t)a.n_top * 12 : 0;
    slices(a, G::ROWS, G::THREADS, [&](const ScoreArgs &b, dim3 grid) { hipLaunchKernelGGL((k_rows<T, OP, NV, G>), grid, dim3(G::THREADS), lds, s, b); });
    return EVT_OK;
}
// Distillation of short rows: true where the lanes hold a row of n pieces and a block's memory its teachers: 25 KB, six blocks to a unit, or more lanes to a row
// (bf16, 32 entries, at 52 | 25 | 20 KB: 2.7M x 100 670 | 429 | 590 us, 8M x 33 1461 | 921 | 901)
template <typename T, int NV, class G>
static bool launch_distill(hipStream_t s, const ScoreArgs &a, int64_t n) {
    const size_t lds = G::ROWS * ((size_t)(a.n_top | 1) * 8 + (size_t)((a.V + 2) | 1) * 4);
    if ((NV ? a.V < Piece<T>::E || n > (int64_t)G::SIZE * NV : a.V >= Piece<T>::E) || (lds > 26000 && G::SIZE < 64) || lds > 65536) return false;
    const uint32_t magic = a.n_top > 1 ? (uint32_t)(((1ull << 32) + a.n_top - 1) / a.n_top) : 0u; // exact for e / n_top, e * n_top < 2^32
    slices(a, G::ROWS, 256, [&](const ScoreArgs &b, dim3 grid) { hipLaunchKernelGGL((k_distill_short<T, NV, G>), grid, dim3(256), lds, s, b, magic); });
    return true;
}
template <typename T, int OP>
static int launch_typed(hipStream_t s, const ScoreArgs &a) {
    constexpr int E = Piece<T>::E;
    const int64_t n = ((int64_t)a.V + E - 1) / E;
    const bool few = a.N <= 256; // no more than a unit each
    if constexpr (OP == SC_DISTILL) {
        if (launch_distill<T, 0, Lanes<1>>(s, a, n) || launch_distill<T, 0, Lanes<8>>(s, a, n) || launch_distill<T, 0, Lanes<64>>(s, a, n)) return EVT_OK;
        // few rows of more than a few classes: a block to each (4 rows of 2048 bf16, on the device: 6.9 us by lanes, 5.9 so; 256 rows of 512: 5.8 | 6.4)
        if ((!few || n <= 32) &&
            (launch_distill<T, 4, Lanes<1>>(s, a, n) || launch_distill<T, 4, Lanes<2>>(s, a, n) || launch_distill<T, 4, Lanes<4>>(s, a, n) ||
             launch_distill<T, 4, Lanes<8>>(s, a, n) || launch_distill<T, 4, Lanes<16>>(s, a, n) || launch_distill<T, 4, Lanes<32>>(s, a, n) ||
             launch_distill<T, 4, Lanes<64>>(s, a, n) || (E == 4 && launch_distill<T, 8, Lanes<64>>(s, a, n))))
            return EVT_OK;
        if (a.V < E) {
            evt_set_error("no form for %d classes and %d entries", a.V, a.n_top); // k_rows' last piece would start in front of the row
            return EVT_ERR_INTERNAL;
        }
    } else {
        if (a.V < E) {
            slices(a, 256, 256, [&](const ScoreArgs &b, dim3 grid) { hipLaunchKernelGGL((k_few_classes<T, OP>), grid, dim3(256), 0, s, b); });
            return EVT_OK;
        }
        // Lanes to a row: four pieces each (one each pays a row's own work and its reductions four times as often: 4.2M x 64 bf16, log-probabilities | policy,
        // 170 | 330 us for 135 | 270)
        if (n <= 4) return launch_rows<T, OP, 4, Lanes<1>>(s, a);
        if (n <= 8) return launch_rows<T, OP, 4, Lanes<2>>(s, a);
        if (n <= 16) return launch_rows<T, OP, 4, Lanes<4>>(s, a);
        if (n <= 32) return launch_rows<T, OP, 4, Lanes<8>>(s, a);
        if (n <= 64) return launch_rows<T, OP, 4, Lanes<16>>(s, a);
        if (n <= 128) return launch_rows<T, OP, 4, Lanes<32>>(s, a);
        if (n <= 256) return launch_rows<T, OP, 4, Lanes<64>>(s, a);
    }
    if constexpr (OP != SC_DISTILL) {
        // a wavefront to a row, eight pieces a lane (89 478 x 3000 bf16, log-probabilities: 140 us by blocks of 256, 88 so); few rows are done sooner by blocks
        if (!few && n <= 512) return launch_rows<T, OP, 8, Lanes<64>>(s, a);
    }
    if constexpr (OP == SC_GRAD) {
        const int64_t parts = (n + 1023) / 1024, blocks = a.N * parts;
        hipLaunchKernelGGL((k_slope_rows<T, false>), dim3((unsigned)(blocks < (1 << 23) ? blocks : (1 << 23))), dim3(256), 0, s, a, PairArgs{}, (int)parts);
        return EVT_OK;
    } else {
        // No gradient: the row streams by.  Blocks of 1024 for few rows (16 x 32 768 bf16: 5.5 us by 256, 5.1) and long ones (4096 x 65 536: 95 | 86 us),
        // of 256 for the others (16 384 x 16 384: 127 us by 1024, 88)
        if (OP == SC_LOGP || !a.g) return few || n >= 8192 ? launch_rows<T, OP, 4, Waves<16>>(s, a) : launch_rows<T, OP, 4, Waves<4>>(s, a);
        // The row stays in registers, 1024 pieces a unit, in the smallest blocks that hold it: while one waits for its row another computes and a third stores
        // (policy, bf16, 1024 threads | so: 16 384 x 16 384 224 | 195 us, 8192 x 32 768 225 | 213, 4096 x 65 536 243 | 203).  No more rows than
        // units: 1024 threads each (16 x 32 768: 9.7 us by 256, 7.4; 256 rows 12.3 | 10.5, but 384 14.2 | 15.3)
        if constexpr (OP != SC_LOGP) {
            if (few) return n <= 4096 ? launch_rows<T, OP, 4, Waves<16>>(s, a) : launch_rows<T, OP, 16, Waves<16>>(s, a);
            if (n <= 1024) return launch_rows<T, OP, 4, Waves<4>>(s, a);
            if (n <= 2048) return launch_rows<T, OP, 8, Waves<4>>(s, a);
            if (n <= 4096) return launch_rows<T, OP, 16, Waves<4>>(s, a);
            if (n <= 8192) return launch_rows<T, OP, 16, Waves<8>>(s, a);
            return launch_rows<T, OP, 16, Waves<16>>(s, a);
        }
    }
}
template <int OP>
static int launch_scores(hipStream_t s, const ScoreArgs &a, int dtype) {
    const int r = dtype == EVT_F32 ? launch_typed<float, OP>(s, a) : dtype == EVT_BF16 ? launch_typed<bf16_t, OP>(s, a) : launch_typed<half_t, OP>(s, a);
    HIPCHK(hipGetLastError());
    return r;
}

// The preference loss's gradient and losses in one launch where few blocks do it: false where they are more
template <typename T>
static bool launch_pairs(hipStream_t s, const ScoreArgs &a, const PairArgs &q) {
    const int64_t parts = (((int64_t)a.V + Piece<T>::E - 1) / Piece<T>::E + 1023) / 1024, blocks = a.N * parts + q.pairs;
    if (blocks > 2048) return false; // what runs at once
    hipLaunchKernelGGL((k_slope_rows<T, true>), dim3((unsigned)blocks), dim3(256), 0, s, a, q, (int)parts);
    return true;
}

void score_scale(ScoreArgs &a, double temperature) {
    a.inv_t = 1.0 / temperature;
    a.exp_mul = (float)(1.4426950408889634 / temperature);
    a.t_mul = (float)temperature;
    a.t2_mul = (float)(temperature * temperature);
}
int launch_distill_f32(hipStream_t s, const ScoreArgs &a) { return launch_scores<SC_DISTILL>(s, a, EVT_F32); }

// ---- entry points ---------------------------------------------------------------------------
static bool on_device(const void *p) {
    hipPointerAttribute_t attr;
    const bool ok = hipPointerGetAttributes(&attr, p) == hipSuccess && attr.type == hipMemoryTypeDevice; // pinned host memory has no atomics
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
    ARGCHK(s->nrows >= 0 && s->nrows <= INT32_MAX && s->nclass >= 1 && s->nclass <= (1 << 30), "nrows must be in [0, 2^31 - 1], nclass in [1, 2^30]");
    ARGCHK(s->temperature >= 1e-4 && s->temperature <= 1e4, "temperature must be in [1e-4, 1e4]"); // factors and their squares stay far from float's ends
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
    a.ws = 1;
    score_scale(a, s->temperature);
    a.past = (double)a.N * a.V * size > 256e6 && a.V > 256 * 16 / size;
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

extern "C" int evt_class_logp(void *stream, const void *scores, const void *labels, int32_t label_dtype, float *logp, float *stats, int32_t flags) {
    return guarded([&]() -> int {
    const evt_scores *const s = static_cast<const evt_scores *>(scores);
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

extern "C" int evt_class_logp_grad(void *stream, const void *scores, const void *labels, int32_t label_dtype, const float *stats, const float *dlogp,
                                   int32_t flags) {
    return guarded([&]() -> int {
    const evt_scores *const s = static_cast<const evt_scores *>(scores);
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

extern "C" int evt_distill_loss(void *stream, const void *scores, const void *top_ids, int32_t id_dtype, const void *top_scores, int32_t top_dtype,
                                int32_t n_top, const float *weights, float *loss, int32_t flags) {
    return guarded([&]() -> int {
    const evt_scores *const s = static_cast<const evt_scores *>(scores);
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

extern "C" int evt_policy_loss(void *stream, const void *scores, const void *labels, int32_t label_dtype, const float *old_logp, const float *advantages,
                               const float *ref_logp, const float *weights, double clip_low, double clip_high, double kl_coef, float *loss, float *logp,
                               int32_t flags) {
    return guarded([&]() -> int {
    const evt_scores *const s = static_cast<const evt_scores *>(scores);
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
    a.lo = 1.0 - clip_low;
    a.hi = 1.0 + clip_high;
    a.log_lo = log(1.0 - clip_low); // -inf of 1: no lower bound
    a.log_hi = log1p(clip_high);
    a.kl = kl_coef;
    a.loss = loss;
    a.logp = logp;
    return launch_scores<SC_POLICY>((hipStream_t)stream, a, s->dtype);
    });
}

extern "C" int evt_preference_loss(void *stream, const void *scores, const void *labels, int32_t label_dtype, const int32_t *offsets, int32_t n_pairs,
                                   const float *ref_logp, const float *weights, double beta, double label_smoothing, double margin, int32_t average,
                                   float *loss, float *seq_logp, float *work, int32_t flags) {
    return guarded([&]() -> int {
    const evt_scores *const s = static_cast<const evt_scores *>(scores);
    ScoreArgs a = {};
    TRY(take_scores(s, false, flags, a));
    TRY(take_labels(labels, label_dtype, a));
    ARGCHK(n_pairs >= 1 && n_pairs < (1 << 22), "n_pairs must be in [1, 2^22 - 1]");
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
    const PairArgs q = {n_pairs, average, ref_logp, weights, beta, label_smoothing, margin, seq_logp};
    if (a.N && a.g && (s->dtype == EVT_F32 ? launch_pairs<float>(st, a, q) : s->dtype == EVT_BF16 ? launch_pairs<bf16_t>(st, a, q) : launch_pairs<half_t>(st, a, q))) {
        HIPCHK(hipGetLastError());
        return EVT_OK;
    }
    // many pairs are short ones (1M rows of 7 classes in 100 000 pairs, the whole call: 1076 us by 1024 threads, 251 by 256)
    if (q.pairs * 2 > LOOK_FOR_SHARED) hipLaunchKernelGGL(k_scores_pairs<4>, dim3((unsigned)n_pairs), dim3(256), 0, st, a, q);
    else hipLaunchKernelGGL(k_scores_pairs<16>, dim3((unsigned)n_pairs), dim3(1024), 0, st, a, q);
    HIPCHK(hipGetLastError());
    if (!a.N || !a.g) return EVT_OK;
    return launch_scores<SC_GRAD>(st, a, s->dtype);
    });
}
