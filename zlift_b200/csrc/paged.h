// paged.h -- what the paged-cache units share: the cache as kernels see it,
// exact small-divisor division, 8-bit conversions, and the launch functions
// behind include/zlift_paged.h.
#pragma once
#include "../../include/zlift_paged.h"
#include "ptx.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <cmath>

namespace zl {

// A page or slot number outside the cache (or a length outside its bounds)
// was met and not followed.
constexpr int kErrBadIndex = 2;

static __device__ __noinline__ void note_bad_index() {
    atomicCAS(&g_dev_error, 0, kErrBadIndex);
}

// Waits for copies or products that are under way, whoever has given up
// (bounded too, by the default limit: a shorter one that was set is for waits
// on other parts of a kernel).
__device__ __forceinline__ void copy_wait(uint64_t* bar, uint32_t parity) {
    volatile int never = 0;
    mbar_wait_for(bar, parity, &never, kDefaultWaitLimitNs);
}

// n / d for 0 <= n < 2^31, d >= 1: one multiply-high and a shift.  With
// s = ceil(log2 d) and m = floor(2^32 (2^s - d) / d) + 1 the quotient is
// (mulhi(m, n) + n) >> s (Granlund and Montgomery 1994, figure 4.1); the sum
// stays below 2^32 because n < 2^31.
struct FastDiv {
    unsigned d = 1, m = 1, s = 0;
    FastDiv() = default;
    explicit FastDiv(unsigned div) : d(div) {
        while (s < 31 && (1u << s) < d) s++;
        m = (unsigned)((((unsigned long long)1 << 32) * (((unsigned long long)1 << s) - d)) / d + 1);
    }
    __device__ __forceinline__ unsigned div(unsigned n) const { return (__umulhi(m, n) + n) >> s; }
};

// Element types of the cache as template arguments.
enum KvType : int { kF16 = 0, kBF16 = 1, kF32 = 2, kI8 = 3, kE4M3 = 4 };
template <int T>
constexpr int kv_bytes = T == kF32 ? 4 : T >= kI8 ? 1 : 2;

struct KvView {
    char *k, *v;                         // elements of the cache's type
    float *ks, *vs;
    long long page, row, head;           // strides, elements
    long long spage, shead;
    int pages, ps, heads, dim;
    FastDiv by_ps;
};

struct PagedAttn {
    KvView c;
    const char* q;
    char* o;
    float* lse;
    long long qr, qh, orow, oh, lh;
    const int *cu, *len, *table;
    long long tstride;
    int tpages, batch, total_q, max_q, heads, group, causal;
    float scale;
    char* ws;
    size_t ws_bytes;
    int elem, type;
};

__device__ __forceinline__ float load_as_float(const char* p, int type) {
    switch (type) {
    case kF16: return __half2float(*reinterpret_cast<const __half*>(p));
    case kBF16: return __bfloat162float(*reinterpret_cast<const __nv_bfloat16*>(p));
    case kI8: return (float)*reinterpret_cast<const signed char*>(p);
    case kE4M3: return (float)*reinterpret_cast<const __nv_fp8_e4m3*>(p);
    default: return *reinterpret_cast<const float*>(p);
    }
}

__device__ __forceinline__ void store_as(char* p, int type, float x) {
    switch (type) {
    case kF16: *reinterpret_cast<__half*>(p) = __float2half_rn(x); break;
    case kBF16: *reinterpret_cast<__nv_bfloat16*>(p) = __float2bfloat16_rn(x); break;
    default: *reinterpret_cast<float*>(p) = x;
    }
}

// The chunk and the cached tokens of sequence s, with every length clamped
// to what the arrays hold: first query row, queries, keys.
struct SeqInfo {
    int q0, n, len;
};
__device__ __forceinline__ SeqInfo seq_info(const PagedAttn& a, int s) {
    SeqInfo r;
    const int c0 = __ldg(a.cu + s), c1 = __ldg(a.cu + s + 1), l = __ldg(a.len + s);
    r.q0 = min(max(c0, 0), a.total_q);
    r.n = max(min(c1, a.total_q) - r.q0, 0);
    const long long room = (long long)a.tpages * a.c.ps;
    r.len = (int)min((long long)max(l, 0), room);
    if (r.q0 != c0 || c1 < c0 || c1 > a.total_q || r.len != l) note_bad_index();
    return r;
}

// Launches, 0 done, 1 not this kernel's, > 1 a CUDA error.
int kv_write(const KvView& c, int type, const zlift_kv_rows& r, const int* slots, cudaStream_t s);
int kv_read(const KvView& c, int type, const zlift_kv_rows& r, const int* table,
            long long tstride, int tpages, const int* starts, const int* cu, int batch,
            cudaStream_t s);
int paged_attn_simt(const PagedAttn& a, cudaStream_t s);
int paged_decode(const PagedAttn& a, cudaStream_t s);
int decode_max_rows();
size_t paged_decode_workspace(const PagedAttn& a);
int paged_chunk(const PagedAttn& a, cudaStream_t s);
int chunk_blocks();
size_t paged_chunk_workspace(const PagedAttn& a);

}  // namespace zl
