// Rows of 16- and 32-bit values in pieces of sixteen bytes, and reductions over the lanes that share a row.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <type_traits>

typedef _Float16 half_t;
typedef __bf16 bf16_t;

// Sixteen bytes of values as they lie in memory, at any address their type allows.
template <typename T>
struct Piece {
    static constexpr int E = 16 / sizeof(T);
    struct __attribute__((packed, aligned(sizeof(T)))) Raw {
        uint32_t w[4];
    };
    Raw r;
    __device__ __forceinline__ void load(const T *p) { r = *(const Raw *)p; }
    // past: by the caches.  A gradient that the last of them (256 MB) cannot hold only drives out what the next pass reads (8 pairs, 5003 x 32 768 bf16, loss and
    // gradient again and again: the first pass over the scores 67 us, 39 so); a smaller one stays for its reader.  Not of short rows, where a store has parts of
    // lines that the second cache would put together (4.2M x 64 bf16: 290 us, 530 so; from 256 pieces on 0 to 5 % less)
    __device__ __forceinline__ void store(T *p, bool past) const {
        typedef uint32_t u4 __attribute__((ext_vector_type(4), aligned(2)));
        const u4 v = {r.w[0], r.w[1], r.w[2], r.w[3]};
        if (past) {
            asm volatile(""); // in front and behind, so that the two stores stay apart: joined, the hint is lost
            __builtin_nontemporal_store(v, (u4 *)p);
            asm volatile("");
        } else {
            *(u4 *)p = v;
        }
    }
    // o elements behind a base: a 32-bit offset is an operand of the access where a pointer is two registers for every piece
    __device__ __forceinline__ void load(const T *p, uint32_t o) { r = *(const Raw *)((const char *)p + o * (uint32_t)sizeof(T)); }
    __device__ __forceinline__ void store(T *p, uint32_t o, bool past) const { store((T *)((char *)p + o * (uint32_t)sizeof(T)), past); }
    // the first n of them, 0 < n < E, the others 0: a row's last piece
    __device__ __forceinline__ void load_some(const T *p, int n) {
        typedef uint32_t u2 __attribute__((ext_vector_type(2), aligned(2)));
        typedef uint32_t u1 __attribute__((aligned(2)));
        u2 a = {0, 0};
        uint32_t b = 0, c = 0;
        if constexpr (sizeof(T) == 4) {
            if (n & 2) a = *(const u2 *)p;
            if (n & 1) c = *(const u1 *)(p + (n & 2));
            r.w[0] = n & 2 ? a[0] : c;
            r.w[1] = a[1];
            r.w[2] = n & 2 ? c : 0;
            r.w[3] = 0;
        } else {
            if (n & 4) a = *(const u2 *)p;
            if (n & 2) b = *(const u1 *)(p + (n & 4));
            if (n & 1) c = *(const uint16_t *)(p + (n & 6));
            const uint32_t d = n & 2 ? b : c;
            r.w[0] = n & 4 ? a[0] : d;
            r.w[1] = n & 4 ? a[1] : n & 2 ? c : 0;
            r.w[2] = n & 4 ? d : 0;
            r.w[3] = (n & 6) == 6 ? c : 0;
        }
    }
    __device__ __forceinline__ void store_some(T *p, int n) const {
        typedef uint32_t u2 __attribute__((ext_vector_type(2), aligned(2)));
        typedef uint32_t u1 __attribute__((aligned(2)));
        const uint32_t w0 = r.w[0], w1 = r.w[1], w2 = r.w[2], w3 = r.w[3]; // values: a choice between places would keep the piece in memory
        const u2 a = {w0, w1};
        if constexpr (sizeof(T) == 4) {
            if (n & 2) *(u2 *)p = a;
            if (n & 1) *(u1 *)(p + (n & 2)) = n & 2 ? w2 : w0;
        } else {
            const uint32_t low = n & 2 ? w1 : w0, high = n & 2 ? w3 : w2;
            if (n & 4) *(u2 *)p = a;
            if (n & 2) *(u1 *)(p + (n & 4)) = n & 4 ? w2 : w0;
            if (n & 1) *(uint16_t *)(p + (n & 6)) = (uint16_t)(n & 4 ? high : low);
        }
    }
    __device__ __forceinline__ void get(float *f) const {
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int k = 0; k < 4; k++) f[k] = __uint_as_float(r.w[k]);
        } else if constexpr (std::is_same<T, bf16_t>::value) {
#pragma unroll
            for (int k = 0; k < 4; k++) {
                f[2 * k] = __uint_as_float(r.w[k] << 16);
                f[2 * k + 1] = __uint_as_float(r.w[k] & 0xffff0000u);
            }
        } else {
            typedef half_t h2 __attribute__((ext_vector_type(2)));
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const h2 v = __builtin_bit_cast(h2, r.w[k]);
                f[2 * k] = (float)v[0];
                f[2 * k + 1] = (float)v[1];
            }
        }
    }
    __device__ __forceinline__ void set(const float *f) { // rounds to nearest
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int k = 0; k < 4; k++) r.w[k] = __float_as_uint(f[k]);
        } else {
            typedef T t2 __attribute__((ext_vector_type(2)));
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const t2 v = {(T)f[2 * k], (T)f[2 * k + 1]};
                r.w[k] = __builtin_bit_cast(uint32_t, v);
            }
        }
    }
};

typedef uint32_t u4 __attribute__((ext_vector_type(4), aligned(2)));
// Piece v of a row of H values, in two steps, so that several are on their way before the first is waited for.  The last one, where it is not whole, is read from where
// the row ends...  TINY: rows of less than a piece.  ONCE: nobody reads it again soon, and it need not stay in the caches
template <bool TINY, bool ONCE = false, typename T>
__device__ __forceinline__ void load_piece(Piece<T> &p, const T *x, uint32_t v, uint32_t H) {
    constexpr uint32_t E = Piece<T>::E;
    if (TINY) {
        p.load_some(x, H);
        return;
    }
    const uint32_t at = v * E, last = H - E;
    const u4 *const from = (const u4 *)((const char *)x + (size_t)(at < last ? at : last) * sizeof(T));
    const u4 r = ONCE ? __builtin_nontemporal_load(from) : *from;
#pragma unroll
    for (int k = 0; k < 4; k++) p.r.w[k] = r[k];
}
// ... and moved down here; what is behind the row becomes `fill`, two or one values of a word.
template <bool TINY, typename T>
__device__ __forceinline__ void settle_piece(Piece<T> &p, uint32_t v, uint32_t H, uint32_t fill = 0) {
    constexpr uint32_t E = Piece<T>::E;
    const uint32_t n = H % E;
    if (TINY || n == 0) return; // of all lanes alike
    const uint32_t up = E - n, words = up * sizeof(T) / 4;
    const bool moves = v * E > H - E;
    uint32_t w[5];
#pragma unroll
    for (uint32_t k = 0; k < 4; k++) {
        w[k] = p.r.w[k];
#pragma unroll
        for (uint32_t d = 1; d < 4; d++) w[k] = words == d ? (d + k < 4 ? p.r.w[(d + k) & 3] : fill) : w[k];
    }
    w[4] = fill;
#pragma unroll
    for (int k = 0; k < 4; k++) {
        if (sizeof(T) == 2) w[k] = up & 1 ? __builtin_amdgcn_alignbit(w[k + 1], w[k], 16) : w[k];
        p.r.w[k] = moves ? w[k] : p.r.w[k];
    }
}

// Reductions over G neighbouring lanes whose result every one of them has: by moves within rows of sixteen lanes and gfx950's swaps of rows between two
// registers, a few cycles a step where a trip through the LDS crossbar is a hundred (8 rows of 32 768 classes: 6.3 us, 4.8 so).
template <int CTRL>
__device__ __forceinline__ float moved(float v) {
    return __int_as_float(__builtin_amdgcn_update_dpp(__float_as_int(v), __float_as_int(v), CTRL, 0xf, 0xf, false));
}
template <int G, typename F>
__device__ __forceinline__ float over_lanes(float v, F &&f) {
    if (G >= 2) v = f(v, moved<0xB1>(v));   // quad_perm: lane ^ 1
    if (G >= 4) v = f(v, moved<0x4E>(v));   // quad_perm: lane ^ 2
    if (G >= 8) v = f(v, moved<0x141>(v));  // row_half_mirror: the other four of eight
    if (G >= 16) v = f(v, moved<0x140>(v)); // row_mirror: the other eight of sixteen
    if (G >= 32) {
        const auto h = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = f(__uint_as_float(h[0]), __uint_as_float(h[1]));
    }
    if (G >= 64) {
        const auto h = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = f(__uint_as_float(h[0]), __uint_as_float(h[1]));
    }
    return v;
}
template <int G>
__device__ __forceinline__ float lanes_sum(float v) {
    return over_lanes<G>(v, [](float x, float y) { return x + y; });
}
