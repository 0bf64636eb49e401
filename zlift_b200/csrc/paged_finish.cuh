// paged_finish.cuh -- how a paged-attention tile's rows end: normalising and
// storing them, and redoing the rows that a masked key spoilt.
//
// The tensor-core kernels form weight 0 times V for keys that a row does not
// see but its neighbours do.  That is 0 unless such a V is NaN or infinite.
// So every stored value is looked at, and a row with one that is not finite
// is computed again by paged_row.cuh, which does not read the keys that the
// row does not see, unless it is so by right (redo_row).  Rows whose weights
// lost their bits (paged_codes.cuh) carry a maximum of NaN and are computed
// again too.
//
// A row takes one warp some 4 us per 32 keys.  Where nobody waits for the warp
// it is done at once; the chunk kernel, whose warps wait for one another,
// marks the row in O and does it when all of a block's tiles are finished.
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

// Whether a row has to be computed again, from its maximum (log2 units), its
// sum and z (not zero where a stored value is not finite); a sum of NaN comes
// from scores that it sees.
__device__ __forceinline__ bool spoilt(float m2, float l, float z) {
    return m2 != m2 || (z != 0.f && l == l);
}
// If so: not when all the keys that were multiplied for it are its own (`seen`
// of them), so that the NaN or infinity is; but bf16 values near the type's
// end, times weights above one, may overflow fp32 on the way.
__device__ __forceinline__ bool redo_row(const PagedAttn& a, float m2, int seen, int multiplied) {
    return m2 != m2 || seen < multiplied || a.type == kBF16;
}

// first element of a row that is to be computed again: a NaN that no
// conversion gives
constexpr uint16_t kRedo = 0xffff;

// by a warp
static __device__ __noinline__ void repair_row(const PagedAttn& a, const Segment& g, int row) {
    const RowPlace p = row_place(a, g, row);
    const int seen = keys_seen(a, g.q, p.token - g.q.q0);
    RowState r;
    r.clear();
    __syncwarp();                                    // what the other lanes stored of it comes first
    row_keys(a, g.s, a.q + (p.token * a.qr + p.head * a.qh) * 2, g.head, 0, seen, 32, r);
    row_store(a, p.token, p.head, r);
}

}  // namespace zl
