// paged_finish.cuh -- how a paged-attention tile's rows end: normalising and
// storing them, and redoing the rows that a masked key spoilt.
//
// The tensor-core kernels form weight 0 times V for keys that a row does not
// see but its neighbours do.  That is 0 unless such a V is NaN or infinite.
// So every stored value is looked at, and a row with one that is not finite
// is computed again by paged_row.cuh, which does not read the keys that the
// row does not see.  Rows that are not finite by right come out the same.
// Rows whose weights lost their bits (paged_codes.cuh) carry a maximum of NaN
// and are computed again too.
#pragma once
#include "paged_row.cuh"
#include "paged_sched.cuh"

namespace zl {

// token and query head of row r of a tile (rows: token-major, then head)
struct RowPlace {
    int token, head;
};
__device__ __forceinline__ RowPlace row_place(const PagedAttn& a, const Segment& g, int row) {
    const int tok = row / a.group;
    return {g.q.q0 + g.i0 + tok, g.head * a.group + row - tok * a.group};
}

__device__ __forceinline__ float lse_of(float m2, float l) {
    return l == 0.f ? -INFINITY : m2 * 0.6931471805599453f + logf(l);
}

// the larger one, NaN if either is
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// by a warp
static __device__ __noinline__ void repair_row(const PagedAttn& a, const Segment& g, int row) {
    const RowPlace p = row_place(a, g, row);
    const int seen = keys_seen(a, g.q, p.token - g.q.q0);
    RowState r;
    r.clear();
    row_keys(a, g.s, a.q + (p.token * a.qr + p.head * a.qh) * 2, g.head, 0, seen, 32, r);
    row_store(a, p.token, p.head, r);
}
}  // namespace zl
