// Rows through experts: limits, and the checks of arguments that their entry points share.
#pragma once
#include "evt_internal.h"
#include "pieces.h"
#include <math.h>

#define MAX_EXPERTS 4096
#define MAX_TOP 64

static bool on_device(const void *p) {
    hipPointerAttribute_t attr;
    const bool ok = hipPointerGetAttributes(&attr, p) == hipSuccess && attr.type == hipMemoryTypeDevice;
    (void)hipGetLastError();
    return ok;
}
template <typename... P>
static int check_device(int32_t flags, P... ptrs) {
    if (flags & EVT_STATIC_TRUSTED) return EVT_OK;
    const void *all[] = {(const void *)ptrs...};
    for (const void *p : all) ARGCHK(!p || on_device(p), "rows through experts take device memory only");
    return EVT_OK;
}
// Tables and weights lie at multiples of their type's size: a scalar load takes no other address, and reads what lies in front instead
template <typename... P>
static int check_aligned(P... ptrs) {
    const void *all[] = {(const void *)ptrs...};
    for (const void *p : all) ARGCHK((uintptr_t)p % 4 == 0, "tables and weights must be aligned to their type");
    return EVT_OK;
}
static int check_ids(const void *ids, int32_t id_dtype) {
    ARGCHK((uintptr_t)ids % (id_dtype == EVT_I64 ? 8 : 4) == 0, "experts must be aligned to their type");
    return EVT_OK;
}
#define TRY(call)                        \
    do {                                 \
        const int _r = (call);           \
        if (_r != EVT_OK) return _r;     \
    } while (0)

static int check_flags(int32_t flags) {
    ARGCHK(flags == 0 || flags == EVT_STATIC_TRUSTED, "flags takes 0 or EVT_STATIC_TRUSTED");
    return EVT_OK;
}
static int size_of(int32_t dtype) { return dtype == EVT_F32 ? 4 : 2; }
struct Extent { // rows in memory, in elements
    const void *p;
    int64_t stride, rows;
};
struct Bytes {
    uintptr_t at;
    uint64_t stride, rows, width;
    uintptr_t end() const { return at + (rows - 1) * stride + width; }
};
// No byte in common: one lies behind the other, or they are columns of one matrix, whose rows are equally far apart.  Rows at two strides that reach into each other's range
// count as lying on each other.
static bool apart(Bytes a, Bytes b) {
    if (!a.at || !b.at || !a.rows || !b.rows || a.end() <= b.at || b.end() <= a.at) return true;
    if ((a.rows > 1 && b.rows > 1 && a.stride != b.stride) || (a.rows == 1 && b.rows == 1)) return false;
    const uint64_t stride = (a.rows > 1 ? a : b).stride;
    if (stride < a.width + b.width) return false;
    const uint64_t gap = a.at < b.at ? (b.at - a.at) % stride : (stride - (a.at - b.at) % stride) % stride; // from a row of a's to the next of b's
    return gap >= a.width && gap + b.width <= stride;
}
static Bytes bytes_of(Extent e, int64_t width, int size) { return {(uintptr_t)e.p, (uint64_t)e.stride * size, (uint64_t)e.rows, (uint64_t)width * size}; }
static Bytes bytes_of(const void *p, int64_t bytes) { return {(uintptr_t)p, 0, bytes > 0, (uint64_t)bytes}; }
static bool apart(Extent a, Extent b, int64_t width, int size) { return apart(bytes_of(a, width, size), bytes_of(b, width, size)); }
static bool same(Extent a, Extent b) { return a.p == b.p && (a.rows <= 1 || a.stride == b.stride); }
