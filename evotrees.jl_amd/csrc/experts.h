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
// Two matrices' rows of `width` values have no byte in common: one lies behind the other, or both are columns of one matrix, whose rows are equally far apart.  Rows at
// two strides that reach into each other's range count as lying on each other.
static bool apart(Extent a, Extent b, int64_t width, int size) {
    if (!a.p || !b.p || !a.rows || !b.rows) return true;
    const uintptr_t a0 = (uintptr_t)a.p, b0 = (uintptr_t)b.p;
    const uintptr_t a1 = a0 + ((a.rows - 1) * a.stride + width) * size, b1 = b0 + ((b.rows - 1) * b.stride + width) * size;
    if (a1 <= b0 || b1 <= a0) return true;
    if ((a.rows > 1 && b.rows > 1 && a.stride != b.stride) || (a.rows == 1 && b.rows == 1)) return false;
    const uint64_t stride = (uint64_t)(a.rows > 1 ? a : b).stride * size, bytes = (uint64_t)width * size;
    if (stride < 2 * bytes) return false;
    const uint64_t gap = (a0 < b0 ? b0 - a0 : a0 - b0) % stride; // from a row of the one to the next of the other
    return gap >= bytes && stride - gap >= bytes;
}
static bool same(Extent a, Extent b) { return a.p == b.p && (a.rows <= 1 || a.stride == b.stride); }
