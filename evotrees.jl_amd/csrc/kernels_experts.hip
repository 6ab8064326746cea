// Rows through experts: the tables that order rows by expert, rows sorted by them and combined again, dropout, and the gradients of these (formulas:
// include/evotrees_hip.h).
//
// All of it moves bytes, in pieces of sixteen: of what is read or written in order memory is the bound, of scattered rows a little less of it (262 144 rows of 4096 bf16
// sorted: of one expert 6.16 TB/s, of 8 5.67, of 64 5.33, of 512 5.30).  Products and sums are 32-bit, and a value is rounded once, when it is written.
#include "experts.h"

// ---- the tables of rows by expert ------------------------------------------------------------

struct PlanArgs {
    const void *ids;
    int64_t n; // rows x top
    int32_t id64, E, bits, nb;
    int32_t *place, *source, *offsets, *table;
};

__device__ __forceinline__ int expert_of(const PlanArgs &a, int64_t i) {
    if (i >= a.n) return -1;
    const int64_t id = a.id64 ? ((const int64_t *)a.ids)[i] : ((const int32_t *)a.ids)[i];
    return id >= 0 && id < a.E ? (int)id : -1;
}

// How many entries of each block's an expert has: table[block][expert], or [expert][block] for many blocks
template <int ITEMS>
__global__ __launch_bounds__(256) void k_plan_count(PlanArgs a, int by_expert) {
    extern __shared__ __align__(16) int s_plan[]; // [E]
    for (int e = threadIdx.x; e < a.E; e += 256) s_plan[e] = 0;
    const int64_t first = (int64_t)blockIdx.x * (256 * ITEMS) + threadIdx.x;
    int id[ITEMS];
#pragma unroll
    for (int i = 0; i < ITEMS; i++) id[i] = expert_of(a, first + i * 256);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < ITEMS; i++)
        if (id[i] >= 0) atomicAdd(s_plan + id[i], 1);
    __syncthreads();
    for (int e = threadIdx.x; e < a.E; e += 256) a.table[by_expert ? (int64_t)e * a.nb + blockIdx.x : (int64_t)blockIdx.x * a.E + e] = s_plan[e];
}

// Inclusive sum over the wavefront's lanes: within rows of sixteen by shifts, then the rows' last ones go to the rows behind
template <int CTRL, int ROWS>
__device__ __forceinline__ int sum_from(int v) { return v + __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xf, false); }
__device__ __forceinline__ int lanes_inclusive(int v) {
    v = sum_from<0x111, 0xf>(v); // row_shr 1, 2, 4, 8
    v = sum_from<0x112, 0xf>(v);
    v = sum_from<0x114, 0xf>(v);
    v = sum_from<0x118, 0xf>(v);
    v = sum_from<0x142, 0xa>(v); // row_bcast 15
    return sum_from<0x143, 0xc>(v); // row_bcast 31
}
// The block's exclusive sum over its threads' values, and all of it
__device__ __forceinline__ int block_exclusive(int v, int &all) {
    constexpr int W = 4;
    __shared__ int s_w[W];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, sum = lanes_inclusive(v);
    if (lane == 63) s_w[wave] = sum;
    __syncthreads();
    int before = 0;
    all = 0;
#pragma unroll
    for (int w = 0; w < W; w++) {
        const int n = s_w[w];
        if (w < wave) before += n;
        all += n;
    }
    __syncthreads();
    return before + sum - v;
}

// Each expert's counts become what the blocks before have, the expert's total goes behind the table: a block to an expert
__global__ __launch_bounds__(256) void k_plan_sums(PlanArgs a) {
    int32_t *t = a.table + (int64_t)blockIdx.x * a.nb;
    int carry = 0;
    for (int b0 = 0; b0 < a.nb; b0 += 256 * 8) {
        int v[8], sum = 0, all;
        const int b = b0 + (int)threadIdx.x * 8;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            v[i] = b + i < a.nb ? t[b + i] : 0;
            sum += v[i];
        }
        int at = carry + block_exclusive(sum, all);
#pragma unroll
        for (int i = 0; i < 8; i++) {
            if (b + i < a.nb) t[b + i] = at;
            at += v[i];
        }
        carry += all;
    }
    if (threadIdx.x == 0) a.table[(int64_t)a.E * a.nb + blockIdx.x] = carry;
}

// Where the counts before a block come from
enum { PLAN_ALONE, PLAN_BLOCKS, PLAN_SUMS };

// Every entry's place: the experts before its own, its expert's entries of the blocks before, of the wavefronts before, and of its wavefront's before it.  The last are found by
// comparing the experts' bits over the wavefront, 64 consecutive entries at a time, without atomics: many entries of one expert would queue up at one word.
// JOIN: a block's entries are put in order in shared memory, so that what goes to the source's places in a row goes there together: four bytes by themselves are a request each (1 000 000 x
// 8 of 64 experts 67 us, 56 so; of 1000 142 | 109; of few experts it is no gain: 262 144 x 8 of 8 24.7 | 25.9).  Blocks of 1024 entries are not joined: with few of them that costs (2048 x 8 of
// 256 11.0 us, 11.5 joined, 32 768 x 8 of 64 11.4 | 11.6), with many it would give a tenth, which is left (131 072 x 8 of 64 17.3 | 15.7, of 256 22.2 | 20.1, of 1000 38.3 | 37.2).
template <int ITEMS, int FROM, bool JOIN>
__global__ __launch_bounds__(256) void k_plan_place(PlanArgs a) {
    constexpr int W = 4, THREADS = 64 * W;
    // [E] where the block's entries of an expert start, [W][E] the wavefronts' counts, 16 bits each, then
    // PLAN_BLOCKS: [2][E] the blocks' sums; JOIN: [E] where an expert's entries start among the block's, and the block's in order, the expert above an entry's bits
    extern __shared__ __align__(16) int s_plan[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), E = a.E;
    int *const s_base = s_plan, *const s_all = s_plan + E * (1 + W / 2), *const s_before = s_all + E, *const s_local = s_all, *const s_order = s_local + E;
    uint16_t *const s_wave = (uint16_t *)(s_plan + E), *const s_mine = s_wave + wave * E;
    for (int e = threadIdx.x; e < E * (W / 2 + (FROM == PLAN_BLOCKS ? 2 : 0)); e += THREADS) s_plan[E + e] = 0;
    const int64_t wave0 = ((int64_t)blockIdx.x * W + wave) * (64 * ITEMS), first = wave0 + lane;
    int id[ITEMS], rank[ITEMS];
#pragma unroll
    for (int i = 0; i < ITEMS; i++) id[i] = expert_of(a, first + i * 64);
    __syncthreads();
    if (FROM == PLAN_BLOCKS) { // all of the blocks' counts, which are few
        const int cells = a.nb * E, mine = blockIdx.x * E, step = THREADS % E;
        int e = threadIdx.x % E;
#pragma unroll 8
        for (int c = threadIdx.x; c < cells; c += THREADS) {
            const int n = a.table[c];
            if (n) {
                atomicAdd(s_all + e, n);
                if (c < mine) atomicAdd(s_before + e, n);
            }
            e += step;
            e -= e >= E ? E : 0;
        }
    }
#pragma unroll
    for (int i = 0; i < ITEMS; i++) {
        rank[i] = 0;
        if (wave0 + i * 64 < a.n) {
            const int e = id[i];
            const uint64_t some = __ballot(e >= 0); // the lanes with the same expert
            uint32_t lo = (uint32_t)some, hi = (uint32_t)(some >> 32);
            for (int b = 0; b < a.bits; b++) {
                const uint32_t set = (uint32_t)__builtin_amdgcn_sbfe(e, b, 1); // all ones or none
                const uint64_t with = __ballot(set != 0);
                lo &= ~((uint32_t)with ^ set);
                hi &= ~((uint32_t)(with >> 32) ^ set);
            }
            if (e >= 0) {
                volatile uint16_t *const c = s_mine + e;
                rank[i] = *c + __builtin_amdgcn_mbcnt_hi(hi, __builtin_amdgcn_mbcnt_lo(lo, 0));
                __builtin_amdgcn_wave_barrier();
                if ((((uint64_t)hi << 32 | lo) >> lane) == 1) *c = (uint16_t)(rank[i] + 1); // the last of them
            }
            __builtin_amdgcn_wave_barrier();
        }
    }
    __syncthreads();
    // an expert's start: the threads have consecutive experts
    const int per = (E + THREADS - 1) / THREADS, e0 = threadIdx.x * per, e1 = e0 + per < E ? e0 + per : E;
    int sum = 0, all, own = 0, here;
    for (int e = e0; e < e1; e++) {
        int total, before = 0, mine = 0;
#pragma unroll
        for (int w = 0; w < W; w++) {
            uint16_t &c = s_wave[w * E + e];
            const int n = c;
            c = (uint16_t)mine;
            mine += n;
        }
        if (FROM == PLAN_ALONE) total = mine;
        else if (FROM == PLAN_SUMS) {
            total = a.table[(int64_t)E * a.nb + e];
            before = a.table[(int64_t)e * a.nb + blockIdx.x];
        } else {
            total = s_all[e];
            before = s_before[e];
        }
        s_base[e] = sum + before;
        if (blockIdx.x == 0) a.offsets[e] = sum;
        sum += total;
        if (JOIN) s_local[e] = own;
        own += mine;
    }
    const int start = block_exclusive(sum, all), own_start = JOIN ? block_exclusive(own, here) : 0;
    for (int e = e0; e < e1; e++) {
        s_base[e] += start;
        if (JOIN) s_local[e] += own_start;
        if (blockIdx.x == 0) a.offsets[e] += start;
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) a.offsets[E] = all;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < ITEMS; i++) {
        const int64_t at = first + i * 64;
        const int e = id[i];
        int pos = -1;
        if (e >= 0) {
            const int n = s_mine[e] + rank[i];
            pos = s_base[e] + n;
            if (JOIN) s_order[s_local[e] + n] = (int)(at - (int64_t)blockIdx.x * (THREADS * ITEMS)) | e << 12;
            else if (pos < a.n) a.source[pos] = (int)at; // always, unless somebody writes the ids meanwhile
        }
        if (at < a.n) a.place[at] = pos;
    }
    if (JOIN) {
        __syncthreads();
        for (int l = threadIdx.x; l < here; l += THREADS) {
            const int o = s_order[l], e = o >> 12, pos = s_base[e] + l - s_local[e];
            if (pos < a.n) a.source[pos] = (int)blockIdx.x * (THREADS * ITEMS) + (o & 0xFFF);
        }
    }
    // behind the last
    for (int64_t p = all + (int64_t)blockIdx.x * THREADS + threadIdx.x; p < a.n; p += (int64_t)gridDim.x * THREADS) a.source[p] = -1;
}

// ---- rows ------------------------------------------------------------------------------------

struct RowArgs {
    const void *x, *res;
    void *out;
    int64_t xs, rs, os; // elements from row to row
    const int32_t *place, *count;
    const float *w;
    const void *y;
    int64_t ys;
    float *dw;
    uint32_t N, n;                     // rows; sorted rows, rows x top
    uint32_t row0;                     // the launch's first row
    uint32_t H, top, pieces, parts;    // pieces of a row; parts: of 64 pieces
    uint32_t tail;                     // blocks that clear sorted rows that no entry has
    // dropout: an element is dropped whose 32 bits are below this
    uint32_t drop, layer;
    float scale;
    const uint64_t *seed_at; // nullptr: seed
    uint64_t seed;
};

#define GAMMA 0x9E3779B97F4A7C15ull
__device__ __forceinline__ uint64_t mixed(uint64_t z) {
    z = (z ^ (z >> 30)) * 0xBF58476D1CE4E5B9ull;
    z = (z ^ (z >> 27)) * 0x94D049BB133111EBull;
    return z ^ (z >> 31);
}
// Dropout of E values of a row from piece v on, whose bits come from SplitMix64 (Steele, Lea, Flood 2014), as a row sample's do: nothing is stored, the gradient draws
// them again.  Four values have the sixteen-bit quarters of one output, which decide unless one of them is just the threshold's upper half: one in 65 536, whose lower
// half is drawn then.
template <int E>
__device__ __forceinline__ void drop_values(const RowArgs &a, uint64_t key, uint32_t row, uint32_t v, float *f) {
    const uint32_t hi = a.drop >> 16, lo = a.drop & 0xFFFFu, words = (a.H + 3) / 4;
    const uint64_t first = (uint64_t)row * words + 1;
#pragma unroll
    for (int q = 0; q < E / 4; q++) {
        const uint64_t at = (first + (v * (E / 4) + q)) * GAMMA, word = mixed(key + at);
        const uint32_t half[2] = {(uint32_t)word, (uint32_t)(word >> 32)};
        bool tie = false;
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const uint32_t bits = (half[k / 2] >> (16 * (k & 1))) & 0xFFFFu;
            tie |= bits == hi;
            f[4 * q + k] = bits < hi ? 0.0f : f[4 * q + k] * a.scale;
        }
        if (__builtin_expect(lo != 0 && tie, 0)) {
            const uint64_t second = mixed(~key + at);
#pragma unroll
            for (int k = 0; k < 4; k++)
                if (((word >> (16 * k)) & 0xFFFF) == hi && ((second >> (16 * k)) & 0xFFFF) < lo) f[4 * q + k] = 0.0f;
        }
    }
}
__device__ __forceinline__ uint64_t drop_key(const RowArgs &a) { return mixed((a.seed_at ? *a.seed_at : a.seed) + ((uint64_t)a.layer + 1) * GAMMA); }

template <bool TINY, typename T>
__device__ __forceinline__ void store_piece(const Piece<T> &p, T *x, uint32_t v, uint32_t H, bool past = false) {
    constexpr uint32_t E = Piece<T>::E;
    T *const o = x + (size_t)v * E;
    if (!TINY && v * E + E <= H) p.store(o, past);
    else p.store_some(o, H % E);
}

// The block of rows that a block has, of as many as the 8 dies divide.  Blocks go round the dies, and each of them has the next of its own eighth of the rows: neighbours among an
// expert's sorted rows come from neighbouring rows, so that the line where one ends and the next begins is put together in one die's cache (32 768 x 8 rows of 4099
// bf16 sorted: 571 us with the blocks as they come, 520 so; of 4096 values, whole lines, 472 | 476; gradients at the leaves of 200 003 x 100 f32 60.7 | 56.5)
__device__ __forceinline__ uint32_t own_block(uint32_t block, uint32_t blocks) { return (block & 7) * (blocks / 8) + block / 8; }
// The row and piece that a thread has.  ROW: a wavefront's are of one row, which the compiler knows; otherwise the pieces of all rows follow each other, and
// no lane is idle.
template <bool ROW>
struct Share {
    uint32_t row, v;
    bool in;
    __device__ __forceinline__ Share(const RowArgs &a, uint32_t block) {
        if (ROW) {
            const uint32_t i = __builtin_amdgcn_readfirstlane(block * 4 + threadIdx.x / 64), r = i / a.parts;
            v = (i - r * a.parts) * 64 + (threadIdx.x & 63);
            row = a.row0 + r;
            in = row < a.N && v < a.pieces;
        } else {
            const uint32_t i = block * 256 + threadIdx.x, r = i / a.pieces;
            v = i - r * a.pieces;
            row = a.row0 + r;
            in = row < a.N;
        }
    }
};

// Sorted rows that no entry has: 0, by the launch's first blocks, beside the others (65 536 x 4 x 201 bf16 with 16 000 rows of padding sorted: by 64 blocks a row
// to a block 198 us, by 1024 46, by 1024 whose rows' pieces follow each other 37)
template <bool TINY, typename T>
__device__ void clear_behind(const RowArgs &a, uint32_t block) {
    Piece<T> z;
    z.r = {};
    const int count = *a.count;
    const uint32_t first = count < 0 ? 0u : (uint32_t)count < a.n ? (uint32_t)count : a.n;
    const uint64_t pieces = (uint64_t)(a.n - first) * a.pieces, step = (uint64_t)a.tail * blockDim.x;
    uint64_t i = (uint64_t)block * blockDim.x + threadIdx.x;
    uint32_t row = first + (uint32_t)(i / a.pieces), v = (uint32_t)(i % a.pieces);
    const uint32_t rows = (uint32_t)(step / a.pieces), more = (uint32_t)(step % a.pieces);
    for (; i < pieces; i += step) {
        store_piece<TINY>(z, (T *)a.out + row * a.os, v, a.H);
        v += more;
        row += rows + (v >= a.pieces ? 1 : 0);
        v -= v >= a.pieces ? a.pieces : 0;
    }
}

// Rows to their places: each row is read once and written `top` times, times a weight if there are weights
template <typename T, bool ROW, bool TINY, bool DROP>
__global__ __launch_bounds__(256) void k_spread(RowArgs a) {
    constexpr int E = Piece<T>::E, TOP = 8;
    if (blockIdx.x < a.tail) {
        if (a.row0 == 0) clear_behind<TINY, T>(a, blockIdx.x);
        return;
    }
    const Share<ROW> me(a, own_block(blockIdx.x - a.tail, gridDim.x - a.tail));
    if (!me.in) return;
    Piece<T> p;
    load_piece<TINY>(p, (const T *)a.x + me.row * a.xs, me.v, a.H);
    settle_piece<TINY>(p, me.v, a.H);
    float f[E];
    if (DROP || a.w) p.get(f);
    if (DROP) drop_values<E>(a, drop_key(a), me.row, me.v, f);
    const size_t e0 = (size_t)me.row * a.top;
    for (uint32_t j0 = 0; j0 < a.top; j0 += TOP) {
        uint32_t at[TOP];
#pragma unroll
        for (int j = 0; j < TOP; j++) at[j] = j0 + j < a.top ? (uint32_t)a.place[e0 + j0 + j] : ~0u;
#pragma unroll
        for (int j = 0; j < TOP; j++)
            if (at[j] < a.n) {
                if (DROP || a.w) {
                    const float w = a.w ? a.w[e0 + j0 + j] : 1.0f;
                    float g[E];
#pragma unroll
                    for (int k = 0; k < E; k++) g[k] = f[k] * w;
                    p.set(g);
                }
                store_piece<TINY>(p, (T *)a.out + at[j] * a.os, me.v, a.H);
            }
    }
}

// ... and the sums of its products with the rows that lie at these places in y: a row to G lanes, or (G = 0) to a block of as many wavefronts as it has.
template <typename T, int G, int TOP, bool TINY, bool DROP>
__global__ __launch_bounds__(G ? 256 : 512) void k_spread_dot(RowArgs a) {
    constexpr int E = Piece<T>::E, ROWS = G ? 256 / G : 1;
    __shared__ float s_dot[G ? 1 : 8][TOP];
    const uint32_t size = G ? G : blockDim.x;
    if (blockIdx.x < a.tail) {
        if (a.row0 == 0) clear_behind<TINY, T>(a, blockIdx.x);
        return;
    }
    const uint32_t rank = G ? threadIdx.x & (G - 1) : threadIdx.x, slot = G == 0 ? 0 : G == 64 ? __builtin_amdgcn_readfirstlane(threadIdx.x / 64) : threadIdx.x / (G ? G : 1);
    const uint32_t row = a.row0 + own_block(blockIdx.x - a.tail, gridDim.x - a.tail) * ROWS + slot;
    if (row >= a.N) return;
    const T *x = (const T *)a.x + row * a.xs;
    const uint64_t key = DROP ? drop_key(a) : 0;
    const size_t e0 = (size_t)row * a.top;
    for (uint32_t j0 = 0; j0 < a.top; j0 += TOP) {
        uint32_t at[TOP];
        float w[TOP], dot[TOP];
#pragma unroll
        for (int j = 0; j < TOP; j++) {
            at[j] = j0 + j < a.top ? (uint32_t)a.place[e0 + j0 + j] : ~0u;
            w[j] = j0 + j < a.top ? a.w[e0 + j0 + j] : 0.0f;
            dot[j] = 0.0f;
        }
        for (uint32_t v = rank; v < a.pieces; v += size) {
            Piece<T> p, q[TOP];
            float f[E];
            load_piece<TINY>(p, x, v, a.H);
#pragma unroll
            for (int j = 0; j < TOP; j++)
                if (at[j] < a.n) load_piece<TINY>(q[j], (const T *)a.y + at[j] * a.ys, v, a.H);
            settle_piece<TINY>(p, v, a.H);
            p.get(f);
            if (DROP) drop_values<E>(a, key, row, v, f);
#pragma unroll
            for (int j = 0; j < TOP; j++)
                if (at[j] < a.n) {
                    float g[E];
#pragma unroll
                    for (int k = 0; k < E; k++) g[k] = f[k] * w[j];
                    p.set(g);
                    store_piece<TINY>(p, (T *)a.out + at[j] * a.os, v, a.H);
                    settle_piece<TINY>(q[j], v, a.H);
                    q[j].get(g);
                    float sum = f[0] * g[0];
#pragma unroll
                    for (int k = 1; k < E; k++) sum = __builtin_fmaf(f[k], g[k], sum);
                    dot[j] += sum;
                }
        }
#pragma unroll
        for (int j = 0; j < TOP; j++) dot[j] = lanes_sum<(G ? G : 64)>(dot[j]);
        if constexpr (G == 0) {
            if (j0) __syncthreads();
            if ((threadIdx.x & 63) == 0) {
#pragma unroll
                for (int j = 0; j < TOP; j++) s_dot[threadIdx.x >> 6][j] = dot[j];
            }
            __syncthreads();
            if (threadIdx.x < TOP && j0 + threadIdx.x < a.top) {
                float sum = 0.0f;
                for (uint32_t k = 0; k < blockDim.x / 64; k++) sum += s_dot[k][threadIdx.x];
                a.dw[e0 + j0 + threadIdx.x] = sum;
            }
        } else if (rank == 0) {
#pragma unroll
            for (int j = 0; j < TOP; j++)
                if (j0 + j < a.top) a.dw[e0 + j0 + j] = dot[j];
        }
    }
}

// Every row's sum over its places, times the weights if there are any, with dropout and a residual
template <typename T, bool ROW, bool TINY, int TOP, bool DROP, bool PAST>
__global__ __launch_bounds__(256) void k_combine(RowArgs a) {
    constexpr int E = Piece<T>::E;
    const Share<ROW> me(a, own_block(blockIdx.x, gridDim.x));
    if (!me.in) return;
    Piece<T> res;
    float sum[E] = {};
    if (a.res) load_piece<TINY, PAST>(res, (const T *)a.res + me.row * a.rs, me.v, a.H);
    const size_t e0 = (size_t)me.row * a.top;
    for (uint32_t j0 = 0; j0 < a.top; j0 += TOP) {
        uint32_t at[TOP];
        float w[TOP];
        Piece<T> p[TOP];
#pragma unroll
        for (int j = 0; j < TOP; j++) at[j] = j0 + j < a.top ? (uint32_t)a.place[e0 + j0 + j] : ~0u;
#pragma unroll
        for (int j = 0; j < TOP; j++) w[j] = a.w && j0 + j < a.top ? a.w[e0 + j0 + j] : 1.0f;
#pragma unroll
        for (int j = 0; j < TOP; j++)
            if (at[j] < a.n) load_piece<TINY, PAST>(p[j], (const T *)a.x + at[j] * a.xs, me.v, a.H);
#pragma unroll
        for (int j = 0; j < TOP; j++)
            if (at[j] < a.n) {
                float f[E];
                settle_piece<TINY>(p[j], me.v, a.H);
                p[j].get(f);
#pragma unroll
                for (int k = 0; k < E; k++) sum[k] = __builtin_fmaf(w[j], f[k], sum[k]);
            }
    }
    if (DROP) drop_values<E>(a, drop_key(a), me.row, me.v, sum);
    if (a.res) {
        float f[E];
        settle_piece<TINY>(res, me.v, a.H);
        res.get(f);
#pragma unroll
        for (int k = 0; k < E; k++) sum[k] += f[k];
    }
    Piece<T> o;
    o.set(sum);
    store_piece<TINY>(o, (T *)a.out + me.row * a.os, me.v, a.H, PAST);
}

template <typename T, bool ROW, bool TINY, bool PAST>
__global__ __launch_bounds__(256) void k_drop(RowArgs a) {
    constexpr int E = Piece<T>::E;
    const Share<ROW> me(a, blockIdx.x);
    if (!me.in) return;
    Piece<T> p, res;
    float f[E];
    load_piece<TINY, PAST>(p, (const T *)a.x + me.row * a.xs, me.v, a.H);
    if (a.res) load_piece<TINY, PAST>(res, (const T *)a.res + me.row * a.rs, me.v, a.H);
    settle_piece<TINY>(p, me.v, a.H);
    p.get(f);
    if (a.drop) drop_values<E>(a, drop_key(a), me.row, me.v, f);
    if (a.res) {
        float g[E];
        settle_piece<TINY>(res, me.v, a.H);
        res.get(g);
#pragma unroll
        for (int k = 0; k < E; k++) f[k] += g[k];
    }
    p.set(f);
    store_piece<TINY>(p, (T *)a.out + me.row * a.os, me.v, a.H, PAST);
}

// ---- launches --------------------------------------------------------------------------------

static unsigned round_up(unsigned blocks) { return (blocks + 7) / 8 * 8; }
enum { ROWS_SPREAD, ROWS_COMBINE, ROWS_DROP };
template <typename T, bool ROW, bool TINY, bool PAST, int OP>
static void launch_rows_as(hipStream_t s, const RowArgs &a, unsigned grid) {
    grid = round_up(grid);
    if constexpr (OP == ROWS_DROP) hipLaunchKernelGGL((k_drop<T, ROW, TINY, PAST>), dim3(grid), dim3(256), 0, s, a);
    else if constexpr (OP == ROWS_SPREAD) {
        if (a.drop) hipLaunchKernelGGL((k_spread<T, ROW, TINY, true>), dim3(grid + a.tail), dim3(256), 0, s, a);
        else hipLaunchKernelGGL((k_spread<T, ROW, TINY, false>), dim3(grid + a.tail), dim3(256), 0, s, a);
    } else {
        const auto go = [&](auto top) {
            if (a.drop) hipLaunchKernelGGL((k_combine<T, ROW, TINY, decltype(top)::value, true, PAST>), dim3(grid), dim3(256), 0, s, a);
            else hipLaunchKernelGGL((k_combine<T, ROW, TINY, decltype(top)::value, false, PAST>), dim3(grid), dim3(256), 0, s, a);
        };
        if (a.top <= 2) go(std::integral_constant<int, 2>());
        else if (a.top <= 4) go(std::integral_constant<int, 4>());
        else go(std::integral_constant<int, 8>());
    }
}
template <typename T, int G, bool TINY>
static void launch_dot_as(hipStream_t s, const RowArgs &a, unsigned groups, int threads = 256) {
    constexpr int ROWS = G ? 256 / G : 1;
    const unsigned grid = round_up((groups + ROWS - 1) / ROWS) + a.tail;
    const auto go = [&](auto top) {
        if (a.drop) hipLaunchKernelGGL((k_spread_dot<T, G, decltype(top)::value, TINY, true>), dim3(grid), dim3(threads), 0, s, a);
        else hipLaunchKernelGGL((k_spread_dot<T, G, decltype(top)::value, TINY, false>), dim3(grid), dim3(threads), 0, s, a);
    };
    if (a.top <= 2) go(std::integral_constant<int, 2>());
    else if (a.top <= 4) go(std::integral_constant<int, 4>());
    else go(std::integral_constant<int, 8>());
}
template <typename T, int OP>
static void launch_rows_typed(hipStream_t s, RowArgs &a) {
    constexpr int E = Piece<T>::E;
    a.pieces = (a.H + E - 1) / E;
    a.parts = (a.pieces + 63) / 64;
    // One block for every 4096 pieces that may have to be cleared: 16 rows of 6 x 2048 have 6 of them
    const uint64_t clear = OP == ROWS_SPREAD ? (uint64_t)a.n * a.pieces / 4096 + 1 : 0;
    a.tail = (uint32_t)(clear < 1024 ? clear : 1024);
    // Results of more than half of what the second caches hold (8 x 4 MB) go past them, and what they come from is read as something that nobody reads again soon (32 768 x 8 x 4096
    // bf16 combined: 486 us, 432 so; dropout of 65 536 x 8192 with a residual 537 | 499; 4096 x 8 x 2048 33.2 | 29.2).  With the kernel that reads the result behind it, combined rows with a
    // residual gain as much (4096 x 8 x 2048, 17 MB, 42.2 us, 39.0 so; 8192 x 8 x 4096 164 | 148; 32 768 x 8 x 4096 618 | 557), dropout alone loses what its reader then fetches from memory
    // (4096 x 2048 14.5 | 15.7, 16 384 x 4096 88 | 100, 32 768 x 8192 359 | 363).  Not what goes to scattered places: parts of lines would leave the second cache before their neighbours come (rows of 4099 sorted: 535 us, 667
    // so), not rows that pieces do not divide (200 003 x 97 f32 combined 37.7 | 42.3, of 100 37.9 | 33.9), and gradients are no sooner done (909 | 910)
    const bool past = OP != ROWS_SPREAD && (double)a.N * a.H * sizeof(T) > 16e6 && (uintptr_t)a.out % 16 == 0 && a.os % E == 0 && a.H % E == 0;
    // Wavefronts of one row, whose places and weights are scalars, from 512 pieces on (32 768 x 8 x 4096 bf16 combined with a residual: 467 us with the rows' pieces behind each
    // other, 462 so; of 4099 sorted 531 | 507); below, lanes without a piece cost more than that gives (65 536 x 4 x 520 combined: 62.5 | 74.6, dropout with a residual 34.8 | 43.8)
    const bool tiny = a.H < E, by_row = a.pieces >= 512;
    const uint32_t each = a.pieces < 64 ? 64 : a.parts * 64; // threads a row, at most
    const uint32_t some = (1u << 30) / each > 0 ? (1u << 30) / each : 1, all = a.N; // rows of a launch
    for (uint64_t row0 = 0; row0 < all; row0 += some) {
        const uint32_t rows = all - row0 < some ? (uint32_t)(all - row0) : some;
        a.row0 = (uint32_t)row0;
        a.N = a.row0 + rows; // the launch's own: rows done twice in place would be done twice
        if (OP == ROWS_SPREAD && a.dw) {
            if (tiny) launch_dot_as<T, 8, true>(s, a, rows);
            else if (a.pieces <= 8) launch_dot_as<T, 8, false>(s, a, rows);
            else if (a.pieces <= 16) launch_dot_as<T, 16, false>(s, a, rows);
            else if (a.pieces <= 32) launch_dot_as<T, 32, false>(s, a, rows);
            else if (a.pieces <= 64) launch_dot_as<T, 64, false>(s, a, rows);
            else {
                // blocks of up to 8 wavefronts in as many turns as it takes (by 4, 6, 8 and 16: 32 768 rows of 8 x 4099 bf16 with dropout 1033, 990, 1004, 1220 us, 65 536 of 4 x 1391 359, 351, 364,
                // 363, 16 rows of 8 x 16 384 14.5, 11.9, 10.3, 10.4: few long rows decide for 8, batches of odd rows lose 1 to 4 %)
                const int turns = (a.parts + 7) / 8;
                launch_dot_as<T, 0, false>(s, a, rows, 64 * ((a.parts + turns - 1) / turns));
            }
        } else {
            const uint64_t threads = by_row ? (uint64_t)rows * a.parts * 64 : (uint64_t)rows * a.pieces;
            const unsigned grid = (unsigned)((threads + 255) / 256);
            if (tiny) launch_rows_as<T, false, true, false, OP>(s, a, grid);
            else if (OP != ROWS_SPREAD && past) by_row ? launch_rows_as<T, true, false, OP != ROWS_SPREAD, OP>(s, a, grid) : launch_rows_as<T, false, false, OP != ROWS_SPREAD, OP>(s, a, grid);
            else by_row ? launch_rows_as<T, true, false, false, OP>(s, a, grid) : launch_rows_as<T, false, false, false, OP>(s, a, grid);
        }
    }
}

template <int OP>
static int launch_rows(hipStream_t s, RowArgs &a, int dtype) {
    if (dtype == EVT_F32) launch_rows_typed<float, OP>(s, a);
    else if (dtype == EVT_BF16) launch_rows_typed<bf16_t, OP>(s, a);
    else launch_rows_typed<half_t, OP>(s, a);
    HIPCHK(hipGetLastError());
    return EVT_OK;
}

// One block for the smallest (16 x 6 of 64 experts: 3.0 us on the device).  Then a launch that counts, in blocks of 1024 entries up to 2^20 of them (131 072 x 2 of 64 experts: 11.3 us, of 4096
// 21.1; 131 072 x 8 of 256 22.2 | 27.3) and of 4096 beyond (262 144 x 8 of 256 29.6 us, of 1024 32.8; of 1000 41.6 | 62.0; 2 000 000 x 1 of 1023 41.0 | 58.1), and one that finds the places.  The
// number of experts, which this does not look at, moves that limit: 131 072 x 8 of 1000 take 38.3 us in blocks of 1024 and 33.5 in blocks of 4096, 262 144 x 8 of 64 27.0 us in blocks of
// 4096 and 23.3 in blocks of 1024, of 8 25.9 | 18.7.  Up to 2048 counts each block that finds places adds up what is before it by itself (2048 x 8 of 64: 9.3 us, 10.3 with a launch for the
// sums; 16 384 x 8 of 16 10.3 | 10.0; of 4096 counts, 8192 x 8 of 64: 12.5 | 10.5).
static void launch_plan(hipStream_t s, PlanArgs &a) {
    a.bits = 0;
    while ((1 << a.bits) < a.E) a.bits++;
    a.nb = 1;
    const dim3 block(256);
    const size_t count_lds = a.E * 4, place_lds = a.E * 12;
    if (a.n <= 1024) {
        hipLaunchKernelGGL((k_plan_place<4, PLAN_ALONE, false>), dim3(1), block, place_lds, s, a);
        return;
    }
    const int chunk = EVT_PLAN_BLOCK(a.n);
    const bool small = chunk == 1024;
    a.nb = (int)((a.n + chunk - 1) / chunk);
    const dim3 grid(a.nb);
    const bool few = small && a.nb * a.E <= 2048;
    if (small) hipLaunchKernelGGL(k_plan_count<4>, grid, block, count_lds, s, a, few ? 0 : 1);
    else hipLaunchKernelGGL(k_plan_count<16>, grid, block, count_lds, s, a, 1);
    if (few) {
        hipLaunchKernelGGL((k_plan_place<4, PLAN_BLOCKS, false>), grid, block, a.E * 20, s, a);
        return;
    }
    hipLaunchKernelGGL(k_plan_sums, dim3(a.E), block, 0, s, a);
    if (small) hipLaunchKernelGGL((k_plan_place<4, PLAN_SUMS, false>), grid, block, place_lds, s, a);
    else if (a.E <= 2048) hipLaunchKernelGGL((k_plan_place<16, PLAN_SUMS, true>), grid, block, place_lds + a.E * 4 + 16384, s, a);
    else hipLaunchKernelGGL((k_plan_place<16, PLAN_SUMS, false>), grid, block, place_lds, s, a);
}

// ---- entry points ------------------------------------------------------------------------------
extern "C" int evt_plan_rows(void *stream, const void *experts, int32_t id_dtype, int64_t nrows, int32_t top, int32_t nexperts, int32_t *place, int32_t *source,
                             int32_t *offsets, int32_t *work, int32_t flags) {
    return guarded([&]() -> int {
    TRY(check_flags(flags));
    ARGCHK(id_dtype == EVT_I32 || id_dtype == EVT_I64, "experts must be EVT_I32 or EVT_I64");
    ARGCHK(nexperts >= 1 && nexperts <= MAX_EXPERTS, "nexperts must be in [1, 4096]");
    ARGCHK(top >= 1 && nrows >= 0 && nrows <= INT32_MAX / top, "top must be at least 1, nrows * top in [0, 2^31 - 1]");
    ARGCHK(offsets, "offsets must not be NULL");
    PlanArgs a = {};
    a.n = nrows * top;
    ARGCHK(a.n == 0 || (experts && place && source && work), "experts, place, source and work must not be NULL");
    TRY(check_ids(experts, id_dtype));
    TRY(check_aligned(place, source, offsets, work));
    TRY(check_device(flags, experts, place, source, offsets, work));
    const int64_t n = a.n * 4;
    const Bytes all[] = {bytes_of(place, n), bytes_of(source, n), bytes_of(offsets, (nexperts + 1) * (int64_t)4), bytes_of(work, a.n ? EVT_PLAN_WORK(a.n, nexperts) * 4 : 0),
                         bytes_of(experts, id_dtype == EVT_I64 ? 2 * n : n)};
    for (int i = 0; i < 4; i++)
        for (int j = i + 1; j < 5; j++) ARGCHK(apart(all[i], all[j]), "place, source, offsets, work and experts must lie apart from each other");
    a.ids = experts;
    a.id64 = id_dtype == EVT_I64;
    a.E = nexperts;
    a.place = place;
    a.source = source;
    a.offsets = offsets;
    a.table = work;
    launch_plan((hipStream_t)stream, a);
    HIPCHK(hipGetLastError());
    return EVT_OK;
    });
}

// What every entry point checks of its rows: x has nx of them, out and residual no
static int take_rows(const evt_rows *r, int64_t nx, int64_t no, int32_t flags, RowArgs &a) {
    TRY(check_flags(flags));
    ARGCHK(r->dtype == EVT_F32 || r->dtype == EVT_BF16 || r->dtype == EVT_F16, "rows must be EVT_F32, EVT_BF16 or EVT_F16");
    ARGCHK(r->nfeats >= 1 && r->nfeats <= (1 << 24), "nfeats must be in [1, 2^24]");
    ARGCHK(r->p >= 0.0 && r->p < 1.0, "p must be in [0, 1)");
    const int size = size_of(r->dtype);
    ARGCHK(r->x_stride >= 0 && r->residual_stride >= 0, "strides must not be negative");
    ARGCHK(nx <= 0 || no <= 0 || (r->x && r->out), "rows and out must not be NULL");
    ARGCHK((uintptr_t)r->x % size == 0 && (uintptr_t)r->out % size == 0 && (uintptr_t)r->residual % size == 0, "rows must be aligned to their type");
    ARGCHK((uintptr_t)r->seed_dev % 8 == 0, "seed_dev must be aligned to its type");
    ARGCHK(no <= 1 || r->out_stride >= r->nfeats, "out_stride must be at least nfeats");
    a.x = r->x;
    a.xs = r->x_stride;
    a.out = r->out;
    a.os = r->out_stride;
    a.res = r->residual;
    a.rs = r->residual_stride;
    a.N = (uint32_t)r->nrows;
    a.H = (uint32_t)r->nfeats;
    const double drop = rint(r->p * 4294967296.0);
    a.drop = drop < 4294967295.0 ? (uint32_t)drop : 4294967295u;
    a.scale = (float)(4294967296.0 / (4294967296.0 - a.drop));
    a.seed = r->seed;
    a.seed_at = r->seed_dev;
    a.layer = r->layer;
    const Extent x = {r->x, r->x_stride, nx}, out = {r->out, r->out_stride, no}, res = {r->residual, r->residual_stride, no};
    ARGCHK((nx == no && same(x, out)) || apart(x, out, a.H, size), "out must lie apart from the rows, or of drop_rows be their own memory, row for row");
    ARGCHK(same(res, out) || apart(res, out, a.H, size), "out must be the residual's own memory, row for row, or lie apart from it");
    return check_device(flags, r->x, r->out, r->residual, r->seed_dev);
}
static int take_places(int64_t nrows, int32_t top, int32_t nexperts, const int32_t *place, RowArgs &a) {
    ARGCHK(nexperts >= 1 && nexperts <= MAX_EXPERTS, "nexperts must be in [1, 4096]");
    ARGCHK(top >= 1 && nrows >= 0 && nrows <= INT32_MAX / top, "top must be at least 1, nrows * top in [0, 2^31 - 1]");
    ARGCHK(place || nrows == 0, "place must not be NULL");
    a.place = place;
    a.top = top;
    a.n = (uint32_t)(nrows * top);
    return EVT_OK;
}

// What a call writes lies apart from the tables that it reads: a row may be written before another thread has read its places
static bool clear_of_tables(Bytes out, const evt_rows *r, const RowArgs &a, const int32_t *offsets, int32_t nexperts, const float *weights) {
    const int64_t n = (int64_t)a.n * 4;
    return apart(out, bytes_of(a.place, n)) && apart(out, bytes_of(weights, n)) && apart(out, bytes_of(offsets, (nexperts + 1) * (int64_t)4)) &&
           apart(out, bytes_of(a.drop ? r->seed_dev : nullptr, 8));
}
static int check_tables(const evt_rows *r, int64_t no, const RowArgs &a, const int32_t *offsets, int32_t nexperts, const float *weights) {
    ARGCHK(clear_of_tables(bytes_of({r->out, r->out_stride, no}, a.H, size_of(r->dtype)), r, a, offsets, nexperts, weights),
           "out must lie apart from place, offsets, weights and the seed");
    return EVT_OK;
}

extern "C" int evt_sort_rows(void *stream, const void *rows, const int32_t *place, const int32_t *offsets, int32_t top, int32_t nexperts, int32_t flags) {
    return guarded([&]() -> int {
    const evt_rows *const r = static_cast<const evt_rows *>(rows);
    ARGCHK(r, "rows must not be NULL");
    RowArgs a = {};
    TRY(take_places(r->nrows, top, nexperts, place, a));
    TRY(take_rows(r, r->nrows, a.n, flags, a));
    ARGCHK(!r->residual && r->p == 0.0, "sorted rows have no residual and no dropout");
    if (a.N == 0) return EVT_OK;
    ARGCHK(top > 1 || r->x != r->out, "sorted rows must lie apart from the rows");
    ARGCHK(offsets, "offsets must not be NULL");
    TRY(check_aligned(place, offsets));
    TRY(check_device(flags, place, offsets));
    TRY(check_tables(r, a.n, a, offsets, nexperts, nullptr));
    a.count = offsets + nexperts;
    return launch_rows<ROWS_SPREAD>((hipStream_t)stream, a, r->dtype);
    });
}

extern "C" int evt_combine_rows(void *stream, const void *rows, const int32_t *place, const float *weights, int32_t top, int32_t flags) {
    return guarded([&]() -> int {
    const evt_rows *const r = static_cast<const evt_rows *>(rows);
    ARGCHK(r, "rows must not be NULL");
    RowArgs a = {};
    TRY(take_places(r->nrows, top, 1, place, a));
    TRY(take_rows(r, a.n, r->nrows, flags, a));
    if (a.N == 0) return EVT_OK;
    ARGCHK(top > 1 || r->x != r->out, "combined rows must lie apart from the experts' rows");
    TRY(check_aligned(place, weights));
    TRY(check_device(flags, place, weights));
    TRY(check_tables(r, a.N, a, nullptr, 0, weights));
    a.w = weights;
    return launch_rows<ROWS_COMBINE>((hipStream_t)stream, a, r->dtype);
    });
}

extern "C" int evt_combine_rows_grad(void *stream, const void *rows, const void *y, int64_t y_stride, const int32_t *place, const int32_t *offsets,
                                     const float *weights, float *dweights, int32_t top, int32_t nexperts, int32_t flags) {
    return guarded([&]() -> int {
    const evt_rows *const r = static_cast<const evt_rows *>(rows);
    ARGCHK(r, "rows must not be NULL");
    RowArgs a = {};
    TRY(take_places(r->nrows, top, nexperts, place, a));
    TRY(take_rows(r, r->nrows, a.n, flags, a));
    ARGCHK(!r->residual, "the gradient takes no residual");
    ARGCHK((y != nullptr) == (dweights != nullptr) && (!y || weights), "y and dweights come together, and with weights");
    ARGCHK(y_stride >= 0 && (uintptr_t)y % size_of(r->dtype) == 0, "y must be aligned to its type, its stride not negative");
    if (a.N == 0) return EVT_OK;
    ARGCHK(top > 1 || r->x != r->out, "the experts' gradients must lie apart from the rows'");
    ARGCHK(apart({y, y_stride, a.n}, {r->out, r->out_stride, a.n}, a.H, size_of(r->dtype)), "the experts' gradients must lie apart from y");
    ARGCHK(offsets, "offsets must not be NULL");
    TRY(check_aligned(place, offsets, weights, dweights));
    TRY(check_device(flags, y, place, offsets, weights, dweights));
    TRY(check_tables(r, a.n, a, offsets, nexperts, weights));
    const Bytes slopes = bytes_of(dweights, (int64_t)a.n * 4);
    const int size = size_of(r->dtype);
    ARGCHK(clear_of_tables(slopes, r, a, offsets, nexperts, weights) && apart(slopes, bytes_of({r->x, r->x_stride, a.N}, a.H, size)) &&
               apart(slopes, bytes_of({y, y_stride, a.n}, a.H, size)) && apart(slopes, bytes_of({r->out, r->out_stride, a.n}, a.H, size)),
           "dweights must lie apart from the rows and the tables");
    a.count = offsets + nexperts;
    a.y = y;
    a.ys = y_stride;
    a.w = weights;
    a.dw = dweights;
    return launch_rows<ROWS_SPREAD>((hipStream_t)stream, a, r->dtype);
    });
}

extern "C" int evt_drop_rows(void *stream, const void *rows, int32_t flags) {
    return guarded([&]() -> int {
    const evt_rows *const r = static_cast<const evt_rows *>(rows);
    ARGCHK(r, "rows must not be NULL");
    ARGCHK(r->nrows >= 0 && r->nrows <= INT32_MAX, "nrows must be in [0, 2^31 - 1]");
    RowArgs a = {};
    TRY(take_rows(r, r->nrows, r->nrows, flags, a));
    if (a.N == 0) return EVT_OK;
    TRY(check_tables(r, a.N, a, nullptr, 0, nullptr));
    return launch_rows<ROWS_DROP>((hipStream_t)stream, a, r->dtype);
    });
}
