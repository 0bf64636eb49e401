// paged_simt.cu -- attention over the paged cache on the CUDA cores: any dim
// up to 256, page size, stride and alignment.
//
// One block per query token and head, its four warps taking every fourth
// group of 32 keys (paged_row.cuh) and joining their softmax states at the
// end.  It reads a key's row once per query head, so it is bound by L2
// traffic and issue, not by memory; it serves the layouts that the tensor
// core kernels leave out.
#include "gemm.h"
#include "paged_row.cuh"

namespace zl {

namespace {

constexpr int kWarps = 4;

__global__ void __launch_bounds__(kWarps * 32) paged_attn_simt_kernel(const __grid_constant__ PagedAttn a) {
    __shared__ float sm[kWarps], sl[kWarps], sacc[kWarps][32 * kRowCols];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int head = blockIdx.y;
    for (int token = blockIdx.x; token < a.total_q; token += gridDim.x) {
        // the sequence whose chunk holds this token
        int lo = 0, hi = a.batch;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (__ldg(a.cu + mid) <= token) lo = mid;
            else hi = mid;
        }
        const SeqInfo q = seq_info(a, lo);
        if (token < q.q0 || token >= q.q0 + q.n) continue;    // in no chunk: left alone
        const int seen = keys_seen(a, q, token - q.q0);
        RowState r;
        r.clear();
        row_keys(a, lo, a.q + (token * a.qr + head * a.qh) * 2, head / a.group, warp * 32, seen,
                 kWarps * 32, r);
        if (lane == 0) {
            sm[warp] = r.m;
            sl[warp] = r.l;
        }
#pragma unroll
        for (int c = 0; c < kRowCols; c++) sacc[warp][lane + 32 * c] = r.acc[c];
        __syncthreads();
        if (warp == 0) {
            RowState t;
            t.clear();
            for (int w = 0; w < kWarps; w++) t.m = fmaxf(t.m, sm[w]);
            const float base = t.m == -INFINITY ? 0.f : t.m;
            for (int w = 0; w < kWarps; w++) {
                const float f = expf(sm[w] - base);
                t.l += sl[w] * f;
#pragma unroll
                for (int c = 0; c < kRowCols; c++) t.acc[c] += sacc[w][lane + 32 * c] * f;
            }
            row_store(a, token, head, t);
        }
        __syncthreads();
    }
}

}  // namespace

int paged_attn_simt(const PagedAttn& a, cudaStream_t s) {
    const dim3 grid((unsigned)min(a.total_q, 1 << 20), (unsigned)a.heads);
    paged_attn_simt_kernel<<<grid, kWarps * 32, 0, s>>>(a);
    const cudaError_t e = cudaGetLastError();
    if (e == cudaSuccess) note_launch();
    return e == cudaSuccess ? 0 : (int)e;
}

int paged_simt_error(bool clear) {
    int v = 0;
    cudaMemcpyFromSymbol(&v, g_dev_error, sizeof(int));
    if (clear && v) {
        int z = 0;
        cudaMemcpyToSymbol(g_dev_error, &z, sizeof(int));
    }
    return v;
}

}  // namespace zl
