// The choice of each row's experts from its class scores, and the gradient of their weights (formulas: include/evotrees_hip.h).
//
// A score is read once, in pieces of sixteen bytes, by a group of lanes that share a row; exponentials and sums are 32-bit, a gradient is rounded once.  Wide rows are
// bound by memory, narrow ones by the comparisons that find the best.
#include "experts.h"

struct RouteArgs {
    const void *x;
    void *g;
    int64_t xs, gs, N;
    int32_t V, top, renormalize, id64;
    float inv_t, exp_mul; // 1 / temperature, log2(e) / temperature
    int32_t *ids;
    float *w;
    const void *ids_in;
    const float *w_in, *dw;
};

// What a wavefront's lanes wrote to shared memory before can be read by its others
__device__ __forceinline__ void lanes_wait() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}
__device__ __forceinline__ float exp_gap(float x, float m, float mul) { return __builtin_amdgcn_exp2f((x - m) * mul); }

// A score and its class as one number that is the greater the better, and no two are alike: the score in an order that numbers have (zeros alike), and below it the
// class as a tag, counted from the last one down, so that of two equal scores the lower class's is the greater.  Scores of -inf, and what is behind a row, are below every other.
template <typename T>
struct Best {
    // 16-bit scores: a whole number of 32 bits, the score's sign and magnitude as its upper half
    typedef int32_t type;
    static constexpr int32_t INF = std::is_same<T, bf16_t>::value ? 0x7F80 : 0x7C00;
    static constexpr uint32_t NONE = (0x8000u | INF) << 16 | 0x8000u | INF; // -inf, twice
    static __device__ __forceinline__ int32_t lowest() { return INT32_MIN; }
    // the scores of a piece, with the tags that count down from `tag`
    static __device__ __forceinline__ void of(const Piece<T> &p, uint32_t tag, int32_t *v, bool &odd) {
        typedef short s2 __attribute__((ext_vector_type(2)));
        typedef unsigned short us2 __attribute__((ext_vector_type(2)));
        us2 most = {0, 0};
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const uint32_t x = p.r.w[j], size = x & 0x7FFF7FFFu;
            const s2 m = __builtin_bit_cast(s2, x) >> (short)15;
            const uint32_t s = __builtin_bit_cast(uint32_t, __builtin_bit_cast(s2, size ^ __builtin_bit_cast(uint32_t, m)) - m);
            most = __builtin_elementwise_max(most, __builtin_bit_cast(us2, size));
            v[2 * j] = (int32_t)(s << 16 | (tag - 2 * j));
            v[2 * j + 1] = (int32_t)((s & 0xFFFF0000u) | (tag - 2 * j - 1));
        }
        odd |= most[0] > INF || most[1] > INF;
    }
    // scores that are no numbers are the best there are
    static __device__ void nan_first(const Piece<T> &p, int32_t *v) {
#pragma unroll
        for (int j = 0; j < 8; j++)
            if (((p.r.w[j / 2] >> (16 * (j & 1))) & 0x7FFFu) > INF) v[j] = (int32_t)(0x7FFF0000u | ((uint32_t)v[j] & 0xFFFFu));
    }
    static __device__ __forceinline__ void add_tag(int32_t &k, uint32_t tag) { k ^= (int32_t)tag; }
    static __device__ __forceinline__ bool is_class(int32_t k) { return (k >> 16) > -INF; }
    static __device__ __forceinline__ int tag_of(int32_t k) { return k & 0xFFFF; }
    static __device__ __forceinline__ float score(int32_t k) {
        const int32_t s = k >> 16;
        const uint32_t bits = (uint32_t)(s < 0 ? 0x8000 - s : s);
        return (float)__builtin_bit_cast(T, (uint16_t)bits);
    }
    static __device__ __forceinline__ int32_t greater(int32_t a, int32_t b) { return a > b ? a : b; }
    static __device__ __forceinline__ int32_t lesser(int32_t a, int32_t b) { return a < b ? a : b; }
    template <int CTRL>
    static __device__ __forceinline__ int32_t moved(int32_t v) { return __builtin_amdgcn_update_dpp(0, v, CTRL, 0xf, 0xf, true); }
    // the two that lanes D apart have, in both of them
    template <int D>
    static __device__ __forceinline__ void both(int32_t v, int32_t &x, int32_t &y) {
        const auto h = D == 16 ? __builtin_amdgcn_permlane16_swap((uint32_t)v, (uint32_t)v, false, false) : __builtin_amdgcn_permlane32_swap((uint32_t)v, (uint32_t)v, false, false);
        x = (int32_t)h[0];
        y = (int32_t)h[1];
    }
};
template <>
struct Best<float> {
    // 32-bit scores: a double of the score, exact, with the class in the lowest 12 of the 29 bits that the score leaves 0.  Doubles have a maximum and a minimum of one
    // instruction each where a pair of words takes a comparison and four choices.
    typedef double type;
    static constexpr uint32_t NONE = 0xFF800000u;
    static __device__ __forceinline__ double lowest() { return -0x1p129; }
    // the lesser bits make a negative number the greater one: its tag is turned round
    static __device__ __forceinline__ uint64_t turned(uint64_t b) { return b | ((uint32_t)((int32_t)(b >> 32) >> 31) & 0xFFFu); }
    static __device__ __forceinline__ double tagged(double d, uint32_t tag) { return __builtin_bit_cast(double, turned(__builtin_bit_cast(uint64_t, d)) ^ tag); }
    static __device__ __forceinline__ void of(const Piece<float> &p, uint32_t tag, double *v, bool &odd) {
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const float x = __uint_as_float(p.r.w[j]) + 0.0f; // -0 becomes 0
            odd |= !(x < INFINITY);
            v[j] = tagged(x == -INFINITY ? -0x1p129 : (double)x, tag - j);
        }
    }
    static __device__ __forceinline__ void add_tag(double &k, uint32_t tag) { k = __builtin_bit_cast(double, __builtin_bit_cast(uint64_t, k) ^ tag); }
    static __device__ void nan_first(const Piece<float> &p, double *v) {
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const float x = __uint_as_float(p.r.w[j]);
            // +inf with a tag would be no number
            if (!(x < INFINITY)) v[j] = tagged(x != x ? 0x1p130 : 0x1p129, tag_of(v[j]));
        }
    }
    static __device__ __forceinline__ bool is_class(double k) { return k > -0x1p128; }
    static __device__ __forceinline__ int tag_of(double k) {
        const uint64_t b = __builtin_bit_cast(uint64_t, k);
        return (int)(((uint32_t)b ^ (uint32_t)((int32_t)(b >> 32) >> 31)) & 0xFFFu);
    }
    static __device__ __forceinline__ float score(double k) { // infinite for no number, too
        return (float)__builtin_bit_cast(double, __builtin_bit_cast(uint64_t, k) & ~0xFFFull);
    }
    static __device__ __forceinline__ double greater(double a, double b) { return fmax(a, b); }
    static __device__ __forceinline__ double lesser(double a, double b) { return fmin(a, b); }
    template <int CTRL>
    static __device__ __forceinline__ double moved(double v) {
        const uint64_t b = __builtin_bit_cast(uint64_t, v);
        return __builtin_bit_cast(double, (uint64_t)(uint32_t)Best<bf16_t>::moved<CTRL>((int32_t)(b >> 32)) << 32 | (uint32_t)Best<bf16_t>::moved<CTRL>((int32_t)b));
    }
    template <int D>
    static __device__ __forceinline__ void both(double v, double &x, double &y) {
        const uint64_t b = __builtin_bit_cast(uint64_t, v);
        int32_t x1, y1, x0, y0;
        Best<bf16_t>::both<D>((int32_t)(b >> 32), x1, y1);
        Best<bf16_t>::both<D>((int32_t)b, x0, y0);
        x = __builtin_bit_cast(double, (uint64_t)(uint32_t)x1 << 32 | (uint32_t)x0);
        y = __builtin_bit_cast(double, (uint64_t)(uint32_t)y1 << 32 | (uint32_t)y0);
    }
};

template <typename T, typename V>
__device__ __forceinline__ void order(V &a, V &b) { // the greater one first
    const V x = Best<T>::greater(a, b), y = Best<T>::lesser(a, b);
    a = x;
    b = y;
}
// Batcher's odd-even merge sort of N values, descending
template <typename T, int N, typename V>
__device__ __forceinline__ void sort_values(V *v) {
#pragma unroll
    for (int p = 1; p < N; p *= 2)
#pragma unroll
        for (int k = p; k >= 1; k /= 2)
#pragma unroll
            for (int j = k % p; j + k < N; j += 2 * k)
#pragma unroll
                for (int i = 0; i < k; i++)
                    if (i + j + k < N && (i + j) / (2 * p) == (i + j + k) / (2 * p)) order<T>(v[i + j], v[i + j + k]);
}
// The K best of two descending lists of K, into the first: the greater ones of the first and the second turned round are they, in an order that rises and falls, which
// the halves' exchanges (Batcher's bitonic ones) make descend.
template <typename T, int K, typename V, typename F>
__device__ __forceinline__ void join(V *a, F &&other) {
    V c[K];
#pragma unroll
    for (int i = 0; i < K; i++) c[i] = Best<T>::greater(a[i], other(K - 1 - i));
#pragma unroll
    for (int i = 0; i < K; i++) a[i] = c[i];
#pragma unroll
    for (int k = K / 2; k >= 1; k /= 2)
#pragma unroll
        for (int i = 0; i < K; i++)
            if ((i & k) == 0) order<T>(a[i], a[i + k]);
}
// ... of the G lanes that share a row, in every one of them
template <typename T, int K, int G, typename V>
__device__ __forceinline__ void join_lanes(V *a) {
    typedef Best<T> B;
    if (G >= 2) join<T, K>(a, [&](int i) { return B::template moved<0xB1>(a[i]); });
    if (G >= 4) join<T, K>(a, [&](int i) { return B::template moved<0x4E>(a[i]); });
    if (G >= 8) join<T, K>(a, [&](int i) { return B::template moved<0x141>(a[i]); });
    if (G >= 16) join<T, K>(a, [&](int i) { return B::template moved<0x140>(a[i]); });
    V b[K];
    if (G >= 32) {
#pragma unroll
        for (int i = 0; i < K; i++) B::template both<16>(a[i], a[i], b[i]);
        join<T, K>(a, [&](int i) { return b[i]; });
    }
    if (G >= 64) {
#pragma unroll
        for (int i = 0; i < K; i++) B::template both<32>(a[i], a[i], b[i]);
        join<T, K>(a, [&](int i) { return b[i]; });
    }
}

template <typename T, int NV, int G>
__device__ __forceinline__ void load_scores(Piece<T> *p, const T *x, int rank, int V) {
    constexpr int E = Piece<T>::E;
    constexpr uint32_t NONE = Best<T>::NONE;
    if (V >= E) {
#pragma unroll
        for (int i = 0; i < NV; i++) load_piece<false>(p[i], x, rank + i * G, V); // behind the row: its last piece again
        if (V < NV * G * E) {
#pragma unroll
            for (int i = 0; i < NV; i++) {
                settle_piece<false>(p[i], rank + i * G, V, NONE);
#pragma unroll
                for (int k = 0; k < 4; k++) p[i].r.w[k] = (rank + i * G) * E < V ? p[i].r.w[k] : NONE;
            }
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < NV; i++)
#pragma unroll
        for (int k = 0; k < 4; k++) p[i].r.w[k] = NONE;
    if (rank == 0) {
        p[0].load_some(x, V);
#pragma unroll
        for (int k = 0; k < E; k++)
            if (k >= V) {
                if (sizeof(T) == 4) p[0].r.w[k & 3] = NONE;
                else p[0].r.w[k / 2] = k & 1 ? (p[0].r.w[k / 2] & 0xFFFFu) | (NONE & 0xFFFF0000u) : (p[0].r.w[k / 2] & 0xFFFF0000u) | (NONE & 0xFFFFu);
            }
    }
}

// A row to G lanes of a wavefront, NV pieces a lane: each lane finds the K best of its scores by sorting K at a time and joining, then the lanes join theirs.  MORE: any
// number: each lane sorts all that it has, the lanes' first ones are compared, and the lane that has the best moves up.
template <typename T, int G, int NV, int K, bool MORE>
__global__ __launch_bounds__(256) void k_route(RouteArgs a) {
    constexpr int E = Piece<T>::E, N = E * NV, ROWS = 256 / G, KEPT = MORE ? N : K;
    typedef Best<T> B;
    typedef typename B::type Value;
    extern __shared__ __align__(16) unsigned char s_dyn[]; // MORE: [ROWS][top] of the best
    const int rank = threadIdx.x & (G - 1), slot = threadIdx.x / G, V = a.V;
    for (int64_t row = (int64_t)blockIdx.x * ROWS + slot; row < a.N; row += (int64_t)gridDim.x * ROWS) {
        Piece<T> p[NV];
        load_scores<T, NV, G>(p, (const T *)a.x + row * a.xs, rank, V);
        Value v[N];
        bool odd = false;
#pragma unroll
        for (int i = 0; i < NV; i++) B::of(p[i], (NV - 1 - i) * G * E + E - 1, v + i * E, odd);
        if (__builtin_expect(__any(odd), 0)) {
#pragma unroll
            for (int i = 0; i < NV; i++) B::nan_first(p[i], v + i * E);
        }
#pragma unroll
        for (int i = 0; i < N; i += KEPT) sort_values<T, KEPT>(v + i);
        // a lane's share of the tag comes when few are left
        const uint32_t lane_tag = (G - 1 - rank) * E;
        float most, total = 0.0f;
        Value *const s_best = (Value *)s_dyn + slot * a.top;
        if constexpr (MORE) {
#pragma unroll
            for (int i = 0; i < N; i++) B::add_tag(v[i], lane_tag);
            for (int j = 0; j < a.top; j++) {
                Value best[1] = {v[0]};
                join_lanes<T, 1, G>(best);
                if (j == 0) most = B::score(best[0]);
                if (B::is_class(best[0])) total += exp_gap(B::score(best[0]), most, a.exp_mul);
                if (rank == 0) s_best[j] = best[0];
                if (v[0] == best[0]) {
#pragma unroll
                    for (int i = 0; i + 1 < N; i++) v[i] = v[i + 1];
                    v[N - 1] = B::lowest();
                }
            }
        } else {
#pragma unroll
            for (int s = K; s < N; s *= 2)
#pragma unroll
                for (int i = 0; i + s < N; i += 2 * s) join<T, K>(v + i, [&](int k) { return v[i + s + k]; });
#pragma unroll
            for (int i = 0; i < K; i++) B::add_tag(v[i], lane_tag);
            join_lanes<T, K, G>(v);
            most = B::score(v[0]);
        }
        if (!a.renormalize) {
            total = 0.0f;
#pragma unroll
            for (int i = 0; i < NV; i++) {
                float f[E];
                p[i].get(f);
#pragma unroll
                for (int k = 0; k < E; k++) total += f[k] == -INFINITY ? 0.0f : exp_gap(f[k], most, a.exp_mul);
            }
            total = lanes_sum<G>(total);
        }
        if constexpr (MORE) {
            lanes_wait();
            const float inv = 1.0f / total;
            for (int j = rank; j < a.top; j += G) {
                const Value best = s_best[j];
                const bool is = B::is_class(best);
                a.ids[row * a.top + j] = is ? G * N - 1 - B::tag_of(best) : -1;
                a.w[row * a.top + j] = is ? exp_gap(B::score(best), most, a.exp_mul) * inv : 0.0f;
            }
            lanes_wait();
        } else { // lane j has the j-th best, or each lane every G-th
            constexpr int MINE = K > G ? K / G : 1;
            float e[MINE];
            int id[MINE];
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < MINE; i++) {
                Value best = v[0];
#pragma unroll
                for (int k = 1; k < K; k++) best = rank + i * G == k ? v[k] : best;
                const bool is = rank + i * G < a.top && B::is_class(best);
                id[i] = is ? G * N - 1 - B::tag_of(best) : -1;
                e[i] = is ? exp_gap(B::score(best), most, a.exp_mul) : 0.0f;
                sum += e[i];
            }
            if (a.renormalize) total = lanes_sum<G>(sum);
            const float inv = 1.0f / total;
#pragma unroll
            for (int i = 0; i < MINE; i++)
                if (rank + i * G < a.top) {
                    a.ids[row * a.top + rank + i * G] = id[i];
                    a.w[row * a.top + rank + i * G] = id[i] >= 0 ? e[i] * inv : 0.0f;
                }
        }
    }
}

// The gradient of weights that are probabilities among all experts: a row to G lanes.  What the chosen classes have is put together in shared memory, a word to a class.
template <typename T, int G, int NV>
__global__ __launch_bounds__(256) void k_route_grad(RouteArgs a) {
    constexpr int E = Piece<T>::E, ROWS = 256 / G, ROW = G * NV * E;
    extern __shared__ __align__(16) float s_rows[]; // [ROWS][ROW]
    const int rank = threadIdx.x & (G - 1), slot = threadIdx.x / G, V = a.V;
    float *const s_row = s_rows + slot * ROW;
    // a class's word: sixteen bytes of each lane side by side, so that no two lanes of a read meet in a bank
    const auto at_class = [&](int c) -> float & {
        const int v = c / E, i = v / G, lane = v % G;
        return s_row[((i * (E / 4) + c % E / 4) * G + lane) * 4 + c % 4];
    };
    for (int64_t row = (int64_t)blockIdx.x * ROWS + slot; row < a.N; row += (int64_t)gridDim.x * ROWS) {
        Piece<T> p[NV];
        load_scores<T, NV, G>(p, (const T *)a.x + row * a.xs, rank, V);
        // a lane's first entry stays in registers, the others of long choices are read twice
        const int64_t e0 = row * a.top;
        const auto id_at = [&](int j) { return a.id64 ? ((const int64_t *)a.ids_in)[e0 + j] : (int64_t)((const int32_t *)a.ids_in)[e0 + j]; };
        const bool has = rank < a.top;
        const int64_t id = has ? id_at(rank) : -1;
        const float w = has ? a.w_in[e0 + rank] : 0.0f, dw = has ? a.dw[e0 + rank] : 0.0f;
        float mean = id >= V ? NAN : id >= 0 ? w * dw : 0.0f; // an id of no class makes the row's gradient NaN
        for (int j = rank + G; j < a.top; j += G) {
            const int64_t i = id_at(j);
            if (i >= 0) mean += i >= V ? NAN : a.w_in[e0 + j] * a.dw[e0 + j];
        }
        mean = lanes_sum<G>(mean);
#pragma unroll
        for (int k = 0; k < NV * E; k += 4) *(float4 *)(s_row + (k / 4 * G + rank) * 4) = {0.0f, 0.0f, 0.0f, 0.0f};
        lanes_wait();
        // Every entry writes its number at its class and looks whether it is still there: an expert that is chosen twice is none of a choice's, but may be given
        bool twice = false;
        if (id >= 0 && id < V) at_class((int)id) = (float)(rank + 1);
        for (int j = rank + G; j < a.top; j += G) {
            const int64_t i = id_at(j);
            if (i >= 0 && i < V) at_class((int)i) = (float)(j + 1);
        }
        lanes_wait();
        if (id >= 0 && id < V) twice = at_class((int)id) != (float)(rank + 1);
        for (int j = rank + G; j < a.top; j += G) {
            const int64_t i = id_at(j);
            if (i >= 0 && i < V) twice |= at_class((int)i) != (float)(j + 1);
        }
        if (__builtin_expect(!__any(twice), 1)) {
            if (id >= 0 && id < V) at_class((int)id) = w * dw * a.inv_t;
            for (int j = rank + G; j < a.top; j += G) {
                const int64_t i = id_at(j);
                if (i >= 0 && i < V) at_class((int)i) = a.w_in[e0 + j] * a.dw[e0 + j] * a.inv_t;
            }
        } else { // sums, in the entries' order
            for (int pass = 0; pass < 2; pass++)
                for (int j = 0; j < a.top; j++) {
                    lanes_wait();
                    if (rank != (j & (G - 1))) continue;
                    const int64_t i = id_at(j);
                    if (i >= 0 && i < V) at_class((int)i) = pass ? at_class((int)i) + a.w_in[e0 + j] * a.dw[e0 + j] * a.inv_t : 0.0f;
                }
        }
        lanes_wait();
        float f[NV * E], m = -INFINITY, total = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; i++) p[i].get(f + i * E);
#pragma unroll
        for (int k = 0; k < NV * E; k++) m = fmaxf(m, f[k]);
        m = over_lanes<G>(m, [](float u, float v) { return fmaxf(u, v); });
        m = m == -INFINITY ? 0.0f : m;
#pragma unroll
        for (int k = 0; k < NV * E; k++) {
            f[k] = exp_gap(f[k], m, a.exp_mul);
            total += f[k];
        }
        total = lanes_sum<G>(total);
        // a row of -inf has no shares; what makes its gradient NaN does so all the same
        const float factor = total == 0.0f && mean == mean ? 0.0f : -mean * a.inv_t / total;
        T *g = (T *)a.g + row * a.gs;
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const int c = (rank + i * G) * E;
            if (c < V) {
                float o[E];
#pragma unroll
                for (int k = 0; k < E; k += 4) *(float4 *)(o + k) = *(const float4 *)(s_row + ((i * (E / 4) + k / 4) * G + rank) * 4);
#pragma unroll
                for (int k = 0; k < E; k++) o[k] = __builtin_fmaf(f[i * E + k], factor, o[k]);
                Piece<T> q;
                q.set(o);
                if (c + E <= V) q.store(g + c, false);
                else q.store_some(g + c, V - c);
            }
        }
        lanes_wait();
    }
}

// ... of weights that sum to one: the scores have no part in it, and few classes have a gradient.  A block's rows lie in shared memory as they will in the result, L lanes to a
// row put their entries there, and all of the block's threads write the rows.
template <typename T, int L>
__global__ __launch_bounds__(256) void k_chosen_grad(RouteArgs a, int rows, int wide) {
    constexpr int E = Piece<T>::E;
    typedef std::conditional_t<sizeof(T) == 2, uint16_t, uint32_t> Bits;
    extern __shared__ __align__(16) unsigned char s_dyn[]; // [rows][wide] of T
    Bits *const s_rows = (Bits *)s_dyn;
    const int rank = threadIdx.x & (L - 1), V = a.V;
    const int64_t first = (int64_t)blockIdx.x * rows;
    const int here = a.N - first < rows ? (int)(a.N - first) : rows;
    for (int k = threadIdx.x * E; k < here * wide; k += 256 * E) *(uint4 *)(s_rows + k) = {0, 0, 0, 0};
    __syncthreads();
    const int r = threadIdx.x / L;
    if (r < here) {
        Bits *const s = s_rows + r * wide;
        const int64_t at = (first + r) * a.top + rank;
        const bool has = rank < a.top;
        const int64_t id = has ? (a.id64 ? ((const int64_t *)a.ids_in)[at] : (int64_t)((const int32_t *)a.ids_in)[at]) : -1;
        const float w = has ? a.w_in[at] : 0.0f, dw = has ? a.dw[at] : 0.0f;
        const bool in = id >= 0 && id < V;
        const float mean = lanes_sum<L>(id >= V ? NAN : id >= 0 ? w * dw : 0.0f); // an id of no class makes the row's gradient NaN
        float value = w * (dw - mean) * a.inv_t;
        // Every entry writes its number at its class and looks whether it is still there: an expert that is chosen twice is none of a choice's, but may be given
        if (in) s[id] = (Bits)(rank + 1);
        lanes_wait();
        const bool twice = in && s[id] != (Bits)(rank + 1);
        if (__builtin_expect(__any(twice), 0)) { // each of them has the sum, in the entries' order
            float sum = 0.0f;
            for (int j = 0; j < L; j++) {
                const int other = __shfl(in ? (int)id : -1, j, L);
                const float more = __shfl(value, j, L);
                if (in && other == (int)id) sum += more;
            }
            value = sum;
        }
        lanes_wait();
        if (in) s[id] = __builtin_bit_cast(Bits, (T)value);
        if (__builtin_expect(mean != mean, 0)) {
            lanes_wait();
            for (int c = rank; c < V; c += L) s[c] = __builtin_bit_cast(Bits, (T)NAN);
        }
    }
    __syncthreads();
    const uint32_t pieces = (V + E - 1) / E;
    for (uint32_t i = threadIdx.x; i < here * pieces; i += 256) {
        const uint32_t r = i / pieces, v = i - r * pieces;
        T *const g = (T *)a.g + (first + r) * a.gs + v * E;
        const uint4 o = *(const uint4 *)(s_rows + r * wide + v * E);
        Piece<T> q;
        q.r = {{o.x, o.y, o.z, o.w}};
        if ((int)(v * E) + E <= V) q.store(g, false);
        else q.store_some(g, V - v * E);
    }
}

// ---- launches --------------------------------------------------------------------------------

template <typename T, int G, int N, int K>
static void launch_best(hipStream_t s, const RouteArgs &a) {
    constexpr int ROWS = 256 / G;
    const int64_t blocks = (a.N + ROWS - 1) / ROWS;
    const dim3 grid((unsigned)(blocks < (1 << 22) ? blocks : 1 << 22));
    hipLaunchKernelGGL((k_route<T, G, N / Piece<T>::E, K ? K : 1, K == 0>), grid, dim3(256), K ? 0 : ROWS * a.top * sizeof(typename Best<T>::type), s, a);
}
template <typename T, int G, int N>
static void launch_route_as(hipStream_t s, const RouteArgs &a) {
    if (a.top <= 2) launch_best<T, G, N, 2>(s, a);
    else if (a.top <= 4) launch_best<T, G, N, 4>(s, a);
    else if (a.top <= 8) launch_best<T, G, N, 8>(s, a);
    else if constexpr (N % 16 == 0) {
        // lists of 16 doubles are too many registers (131 072 x 10 of 1000 f32: 306 us, 244 so; bf16 124 | 148, 16 of 256 30.1 | 52.9)
        if constexpr (sizeof(T) == 2) {
            if (a.top <= 16) return launch_best<T, G, N, 16>(s, a);
        }
        launch_best<T, G, N, 0>(s, a);
    }
}
// Lanes that share a row, and scores of each: 24 where they are enough (131 072 x 8 of 96 bf16: 14.3 us without, 10.9 so; of 384 42.9 | 34.2, f32 88.1 | 57; lists of 16 need a
// multiple of that); more scores a lane are fewer lists to join between lanes, but their registers leave fewer wavefronts to a unit, with 32-bit scores twice as soon.
template <typename T>
static void launch_route_typed(hipStream_t s, const RouteArgs &a) {
    const int V = a.V;
    const bool thirds = a.top <= 8;
    constexpr bool half = sizeof(T) == 2;
    if (V <= 16) return launch_route_as<T, 1, 16>(s, a);
    if (V <= 32) return launch_route_as<T, 2, 16>(s, a);
    if (V <= 48 && thirds) return launch_route_as<T, 2, 24>(s, a);
    if (V <= 64) return launch_route_as<T, 4, 16>(s, a);
    if (V <= 96 && thirds) return launch_route_as<T, 4, 24>(s, a);
    if (V <= 128) return launch_route_as<T, 8, 16>(s, a);
    if (V <= 192 && thirds) return launch_route_as<T, 8, 24>(s, a);
    if (V <= 256) return launch_route_as<T, half ? 8 : 16, half ? 32 : 16>(s, a);
    if (V <= 384 && thirds) return launch_route_as<T, 16, 24>(s, a);
    // ... of 32-bit scores as long as the lists are short (131 072 x 8 of 512: 90.6 us by 16, 72.2 by 32; of 1000 189 | 154; but 12 of 256, all sorted, 70 | 80)
    if (V <= 512 && (half || thirds)) return launch_route_as<T, 16, 32>(s, a);
    if (V <= 768 && thirds) return launch_route_as<T, 32, 24>(s, a);
    if (V <= 1024 && (half || thirds)) return launch_route_as<T, 32, 32>(s, a);
    if constexpr (!half) {
        if (V <= 512) return launch_best<T, 32, 16, 0>(s, a);
        if (V <= 1024) return launch_best<T, 64, 16, 0>(s, a);
    }
    if (V <= 1536 && thirds) return launch_route_as<T, 64, 24>(s, a);
    if (V <= 2048) return launch_route_as<T, 64, 32>(s, a);
    launch_route_as<T, 64, 64>(s, a);
}
// Sixteen values of the gradient a lane, of more than 1024 classes 32 or 64
template <typename T, int G, int N>
static void launch_grad_as(hipStream_t s, const RouteArgs &a) {
    constexpr int ROWS = 256 / G;
    const int64_t blocks = (a.N + ROWS - 1) / ROWS;
    hipLaunchKernelGGL((k_route_grad<T, G, N / Piece<T>::E>), dim3((unsigned)(blocks < (1 << 22) ? blocks : 1 << 22)), dim3(256), ROWS * G * N * 4, s, a);
}
// As many rows as the block has lanes for their entries, or as 16 KB hold, ten blocks to a unit (131 072 rows of 8 of 256 bf16: 16.8 us with 8 KB, 15.3 so and with 32; of 10 of
// 1000 77.3, 57.8, 55.6; of 8 of 2048 109.8 with 32, 105.5 so; four times the lanes: 6 of 64 9.3 | 7.7 us, 1024 rows of these 4.9 | 3.1)
template <typename T, int L>
static void launch_chosen(hipStream_t s, RouteArgs a) {
    const int wide = (a.V + 7) / 8 * 8, bytes = wide * (int)sizeof(T), rows = 16384 / bytes < 256 / L ? 16384 / bytes : 256 / L;
    const int64_t all = a.N, some = (int64_t)rows << 22;
    for (int64_t row0 = 0; row0 < all; row0 += some) {
        a.N = all - row0 < some ? all - row0 : some;
        hipLaunchKernelGGL((k_chosen_grad<T, L>), dim3((unsigned)((a.N + rows - 1) / rows)), dim3(256), (size_t)rows * bytes, s, a, rows, wide);
        a.ids_in = (const char *)a.ids_in + a.N * a.top * (a.id64 ? 8 : 4);
        a.w_in += a.N * a.top;
        a.dw += a.N * a.top;
        a.g = (T *)a.g + a.N * a.gs;
    }
}
template <typename T>
static void launch_grad_typed(hipStream_t s, const RouteArgs &a) {
    if (a.renormalize) {
        if (a.top <= 1) return launch_chosen<T, 1>(s, a);
        if (a.top <= 2) return launch_chosen<T, 2>(s, a);
        if (a.top <= 4) return launch_chosen<T, 4>(s, a);
        if (a.top <= 8) return launch_chosen<T, 8>(s, a);
        if (a.top <= 16) return launch_chosen<T, 16>(s, a);
        if (a.top <= 32) return launch_chosen<T, 32>(s, a);
        return launch_chosen<T, 64>(s, a);
    }
    const int n = (a.V + 15) / 16;
    if (n <= 1) launch_grad_as<T, 1, 16>(s, a);
    else if (n <= 2) launch_grad_as<T, 2, 16>(s, a);
    else if (n <= 4) launch_grad_as<T, 4, 16>(s, a);
    else if (n <= 8) launch_grad_as<T, 8, 16>(s, a);
    else if (n <= 16) launch_grad_as<T, 16, 16>(s, a);
    else if (n <= 32) launch_grad_as<T, 32, 16>(s, a);
    else if (n <= 64) launch_grad_as<T, 64, 16>(s, a);
    else if (n <= 128) launch_grad_as<T, 64, 32>(s, a);
    else launch_grad_as<T, 64, 64>(s, a);
}
template <bool GRAD>
static int launch_route(hipStream_t s, const RouteArgs &a, int dtype) {
    const auto go = [&](auto t) {
        if (GRAD) launch_grad_typed<decltype(t)>(s, a);
        else launch_route_typed<decltype(t)>(s, a);
    };
    if (dtype == EVT_F32) go(float());
    else if (dtype == EVT_BF16) go(bf16_t());
    else go(half_t());
    HIPCHK(hipGetLastError());
    return EVT_OK;
}

// ---- entry points ------------------------------------------------------------------------------
static int take_route(const evt_scores *s, int32_t top, int32_t renormalize, int32_t flags, RouteArgs &a) {
    ARGCHK(s, "scores must not be NULL");
    TRY(check_flags(flags));
    ARGCHK(s->dtype == EVT_F32 || s->dtype == EVT_BF16 || s->dtype == EVT_F16, "scores must be EVT_F32, EVT_BF16 or EVT_F16");
    ARGCHK(s->nrows >= 0 && s->nrows <= INT32_MAX && s->nclass >= 1 && s->nclass <= MAX_EXPERTS, "nrows must be in [0, 2^31 - 1], nclass in [1, 4096]");
    ARGCHK(top >= 1 && top <= MAX_TOP && top <= s->nclass, "top must be in [1, 64] and at most nclass");
    ARGCHK(renormalize == 0 || renormalize == 1, "renormalize takes 0 or 1");
    ARGCHK(s->temperature >= 1e-4 && s->temperature <= 1e4, "temperature must be in [1e-4, 1e4]");
    ARGCHK(s->row_stride >= 0, "row_stride must not be negative");
    a.N = s->nrows;
    a.V = s->nclass;
    a.top = top;
    a.renormalize = renormalize;
    a.x = s->x;
    a.xs = s->row_stride;
    a.inv_t = (float)(1.0 / s->temperature);
    a.exp_mul = (float)(1.4426950408889634 / s->temperature);
    if (a.N) ARGCHK(s->x && (uintptr_t)s->x % size_of(s->dtype) == 0, "scores must not be NULL and be aligned to their type");
    return EVT_OK;
}

extern "C" int evt_route_rows(void *stream, const void *scores, int32_t top, int32_t renormalize, int32_t *experts, float *weights, int32_t flags) {
    return guarded([&]() -> int {
    const evt_scores *const s = static_cast<const evt_scores *>(scores);
    RouteArgs a = {};
    TRY(take_route(s, top, renormalize, flags, a));
    if (a.N == 0) return EVT_OK;
    ARGCHK(experts && weights, "experts and weights must not be NULL");
    TRY(check_aligned(experts, weights));
    TRY(check_device(flags, s->x, experts, weights));
    const Bytes x = bytes_of({s->x, s->row_stride, a.N}, a.V, size_of(s->dtype)), ids = bytes_of(experts, a.N * top * 4), w = bytes_of(weights, a.N * top * 4);
    ARGCHK(apart(ids, x) && apart(w, x) && apart(ids, w), "experts and weights must lie apart from the scores and from each other");
    a.ids = experts;
    a.w = weights;
    return launch_route<false>((hipStream_t)stream, a, s->dtype);
    });
}

extern "C" int evt_route_rows_grad(void *stream, const void *scores, int32_t top, int32_t renormalize, const void *experts, int32_t id_dtype,
                                   const float *weights, const float *dweights, int32_t flags) {
    return guarded([&]() -> int {
    const evt_scores *const s = static_cast<const evt_scores *>(scores);
    RouteArgs a = {};
    TRY(take_route(s, top, renormalize, flags, a));
    ARGCHK(id_dtype == EVT_I32 || id_dtype == EVT_I64, "experts must be EVT_I32 or EVT_I64");
    if (a.N == 0) return EVT_OK;
    const int size = size_of(s->dtype);
    ARGCHK(experts && weights && dweights && s->grad, "experts, weights, dweights and grad must not be NULL");
    ARGCHK((uintptr_t)s->grad % size == 0, "gradients must be aligned to their type");
    ARGCHK(a.N == 1 || s->grad_stride >= s->nclass, "grad_stride must be at least nclass");
    const Extent x = {s->x, s->row_stride, a.N}, g = {s->grad, s->grad_stride, a.N};
    ARGCHK(same(x, g) || apart(x, g, a.V, size), "grad must be the scores' own memory, row for row, or lie apart from them");
    TRY(check_ids(experts, id_dtype));
    TRY(check_aligned(weights, dweights));
    TRY(check_device(flags, s->x, s->grad, experts, weights, dweights));
    const Bytes grad = bytes_of(g, a.V, size);
    const int64_t n = a.N * top * 4;
    ARGCHK(apart(grad, bytes_of(experts, id_dtype == EVT_I64 ? 2 * n : n)) && apart(grad, bytes_of(weights, n)) && apart(grad, bytes_of(dweights, n)),
           "grad must lie apart from experts, weights and dweights");
    a.g = s->grad;
    a.gs = s->grad_stride;
    a.ids_in = experts;
    a.id64 = id_dtype == EVT_I64;
    a.w_in = weights;
    a.dw = dweights;
    return launch_route<true>((hipStream_t)stream, a, s->dtype);
    });
}

