// paged_row.cuh -- attention of one query row over a paged cache by one warp,
// for any dim up to 256, type, stride and page size.
//
// Keys go 32 at a time: lane i owns key i of the group, forms its whole dot
// product (q's elements come by shuffle) and the softmax runs across the
// lanes; then every lane owns the output columns lane + 32c and the group's
// V rows are added in key order.  Keys past the row's limit are not read, so
// nothing they hold can reach the result.  fp32 throughout, exp in full
// precision.
#pragma once
#include "paged.h"

namespace zl {

constexpr int kRowCols = 8;              // output columns per lane: dim <= 256

struct RowState {
    float m, l, acc[kRowCols];
    __device__ __forceinline__ void clear() {
        m = -INFINITY;
        l = 0.f;
#pragma unroll
        for (int c = 0; c < kRowCols; c++) acc[c] = 0.f;
    }
};

// keys [k0, k1) of sequence s, group by group with a distance of `step` keys
static __device__ __noinline__ void row_keys(const PagedAttn& a, int s, const char* qrow, int hk,
                                             int k0, int k1, int step, RowState& r) {
    const int lane = threadIdx.x & 31;
    const int dim = a.c.dim, eb = a.type >= kI8 ? 1 : 2;
    float q[kRowCols];
#pragma unroll
    for (int c = 0; c < kRowCols; c++)
        q[c] = lane + 32 * c < dim ? load_as_float(qrow + (lane + 32 * c) * 2, a.elem) : 0.f;
    const int* table = a.table + s * a.tstride;
    for (int kb = k0; kb < k1; kb += step) {
        const int j = kb + lane;
        long long at = 0, sat = 0;
        bool ok = j < k1;
        if (ok) {
            const unsigned i = a.c.by_ps.div((unsigned)j);
            const int off = j - (int)i * a.c.ps;
            const int page = __ldg(table + i);
            if (page < 0 || page >= a.c.pages) {
                note_bad_index();
                ok = false;
            } else {
                at = (page * a.c.page + off * a.c.row + hk * a.c.head) * eb;
                sat = page * a.c.spage + hk * a.c.shead + off;
            }
        }
        float x = 0.f;
        const char* krow = a.c.k + at;
#pragma unroll
        for (int c = 0; c < kRowCols; c++)
            for (int t = 0; t < 32 && 32 * c + t < dim; t++) {
                const float qd = __shfl_sync(0xffffffffu, q[c], t);
                if (ok) x = fmaf(qd, load_as_float(krow + (32 * c + t) * eb, a.type), x);
            }
        if (a.type >= kI8 && ok) x *= __ldg(a.c.ks + sat);
        x = ok ? x * a.scale : -INFINITY;
        float mx = x;
        for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
        const float m = fmaxf(r.m, mx);
        const float base = m == -INFINITY ? 0.f : m;
        const float alpha = expf(r.m - base);
        float p = ok ? expf(x - base) : 0.f;
        float sum = p;
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        r.l = r.l * alpha + sum;
        r.m = m;
        if (a.type >= kI8 && ok) p *= __ldg(a.c.vs + sat);
#pragma unroll
        for (int c = 0; c < kRowCols; c++) r.acc[c] *= alpha;
        const unsigned there = __ballot_sync(0xffffffffu, ok);
        for (int t = 0; t < 32; t++) {
            const float pt = __shfl_sync(0xffffffffu, p, t);
            const long long vt = __shfl_sync(0xffffffffu, at, t);
            if (!((there >> t) & 1u)) continue;
#pragma unroll
            for (int c = 0; c < kRowCols; c++)
                if (lane + 32 * c < dim)
                    r.acc[c] = fmaf(pt, load_as_float(a.c.v + vt + (lane + 32 * c) * eb, a.type),
                                    r.acc[c]);
        }
    }
}

// the row's O and LSE
__device__ __forceinline__ void row_store(const PagedAttn& a, int token, int head,
                                          const RowState& r) {
    const int lane = threadIdx.x & 31;
    const float inv = r.l == 0.f ? 0.f : 1.f / r.l;      // NaN stays NaN
    char* o = a.o + (token * a.orow + head * a.oh) * 2;
#pragma unroll
    for (int c = 0; c < kRowCols; c++)
        if (lane + 32 * c < a.c.dim) store_as(o + (lane + 32 * c) * 2, a.elem, r.acc[c] * inv);
    if (a.lse && lane == 0)
        a.lse[head * a.lh + token] = r.l == 0.f ? -INFINITY : r.m + logf(r.l);
}

// keys that query i of a chunk sees
__device__ __forceinline__ int keys_seen(const PagedAttn& a, const SeqInfo& q, int i) {
    return a.causal ? max(0, min(q.len, q.len - q.n + i + 1)) : q.len;
}

}  // namespace zl
