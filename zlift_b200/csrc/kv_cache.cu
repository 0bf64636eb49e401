// kv_cache.cu -- writing tokens into the paged cache (quantising to 8 bits
// where it holds 8 bits) and reading them back.
//
// Both move every byte once and do a few operations on it, so memory bounds
// them (small calls: the launch).  A block takes a few tokens, looks their
// slots up once into shared memory, and then its threads take 16-byte pieces
// (8 elements of 16 bits) of the rows [token][K or V][head][dim], dim
// fastest: global accesses are contiguous along dim on both sides, and a
// thread has kUnroll independent pieces in flight.  A row's maximum is
// reduced over the dim / 8 neighbouring lanes that hold it, so the row is
// read once.  Rows that do not split into such pieces take a lane per
// element, two reads (the second hits in cache).
//
// Measured on one B200, 8 heads of 128: reading 131072 int8 tokens back in bf16
// 129 us, 6.3 TB/s, 96% of the copy rate; writing 8 x 4096 bf16 tokens to e4m3
// 55 us, 3.7 TB/s (what is left is issue: a maximum, two quotients and eight
// conversions per 16 bytes); 64 tokens written to int8 and read back 6 us,
// two launches.
#include "gemm.h"
#include "paged.h"

#include <algorithm>

namespace zl {

namespace {

constexpr int kThreads = 256;
constexpr int kUnroll = 4;
constexpr int kMaxTokens = 64;      // tokens per block, at most

// Smallest amax that is quantised: below it top / amax could overflow.
constexpr float kTiny = 0x1p-100f;

struct Rows {
    char *k, *v;
    long long kr, kh, vr, vh;       // strides, bytes
    int tokens, per_block;
    FastDiv by_heads;
};

template <int IN>
__device__ __forceinline__ void unpack8(const uint4& w, float (&x)[8]) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if constexpr (IN == kBF16) {
            x[2 * i] = __uint_as_float(u[i] << 16);
            x[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
        } else {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
            x[2 * i] = f.x;
            x[2 * i + 1] = f.y;
        }
    }
}

template <int OUT>
__device__ __forceinline__ uint32_t pack16(float a, float b) {
    if constexpr (OUT == kBF16) {
        const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&v);
    } else {
        const __half2 v = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&v);
    }
}

// One code of value v (already x * (top / amax)).  |v| <= top * (1 + 2^-23)
// rounds to at most top in both types.  int8: adding 1.5 * 2^23 rounds to the
// nearest even integer and leaves it in the low bits (conversion instructions
// run at a quarter of an addition's rate).
template <int CT>
__device__ __forceinline__ uint32_t code_of(float v) {
    if constexpr (CT == kI8) return __float_as_uint(__fadd_rn(v, 12582912.f)) & 0xffu;
    else return __nv_cvt_float_to_fp8(v, __NV_SATFINITE, __NV_E4M3);
}
// four codes, lowest byte first
template <int CT>
__device__ __forceinline__ uint32_t code4(float a, float b, float c, float d) {
    if constexpr (CT == kI8) {
        const uint32_t lo = __byte_perm(__float_as_uint(__fadd_rn(a, 12582912.f)),
                                        __float_as_uint(__fadd_rn(b, 12582912.f)), 0x0040);
        const uint32_t hi = __byte_perm(__float_as_uint(__fadd_rn(c, 12582912.f)),
                                        __float_as_uint(__fadd_rn(d, 12582912.f)), 0x0040);
        return __byte_perm(lo, hi, 0x5410);
    } else {
        const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
        const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
        return lo | hi << 16;
    }
}

// scale and multiplier of a row with maximum `amax` (NaN: not all finite)
template <int CT>
__device__ __forceinline__ void row_scale(float amax, float& scale, float& mul) {
    constexpr float top = CT == kI8 ? 127.f : 448.f;
    const bool full = amax >= kTiny;                 // false for NaN
    scale = full ? __fdiv_rn(amax, top) : amax < kTiny ? 0.f : amax;
    mul = full ? __fdiv_rn(top, amax) : 0.f;
}

// |x| as an ordering key: the bits without the sign, where NaN and infinity
// compare above every finite value
__device__ __forceinline__ float amax_of(unsigned key) {
    return key >= 0x7f800000u ? __uint_as_float(0x7fffffffu) : __uint_as_float(key);
}

__device__ __forceinline__ bool slot_place(const KvView& c, int slot, int& page, int& off) {
    page = (int)c.by_ps.div((unsigned)max(slot, 0));
    off = slot - page * c.ps;
    if (slot >= 0 && page >= c.pages) note_bad_index();
    return slot >= 0 && page < c.pages;
}

// LPR lanes hold one row (8 elements each).
template <int IN, int CT, int LPR>
__global__ void __launch_bounds__(kThreads)
kv_write_kernel(const KvView c, const Rows r, const int* __restrict__ slots) {
    __shared__ long long s_at[kMaxTokens], s_sc[kMaxTokens];
    const int t0 = blockIdx.x * r.per_block;
    const int nt = min(r.per_block, r.tokens - t0);
    constexpr int kRows = kThreads / LPR;            // rows per pass of the block
    constexpr int EB = kv_bytes<CT>;
    const int part = threadIdx.x % LPR;
    const unsigned rows = (unsigned)nt * 2u * (unsigned)c.heads;
    uint4 in[kUnroll];
    auto fetch = [&](unsigned r0) {
#pragma unroll
        for (int u = 0; u < kUnroll; u++) {
            const unsigned row = r0 + u * kRows + threadIdx.x / LPR;
            const unsigned q = r.by_heads.div(row);  // 2 * token + (K or V)
            const unsigned head = row - q * c.heads;
            in[u] = make_uint4(0u, 0u, 0u, 0u);
            if (row < rows) {
                const char* p = q & 1u ? r.v + (t0 + (int)(q >> 1)) * r.vr + head * r.vh
                                       : r.k + (t0 + (int)(q >> 1)) * r.kr + head * r.kh;
                in[u] = __ldcs(reinterpret_cast<const uint4*>(p) + part);
            }
        }
    };
    fetch(0);                                        // the rows need no slot to be read
    for (int i = threadIdx.x; i < nt; i += kThreads) {
        int page, off;
        const bool ok = slot_place(c, __ldg(slots + t0 + i), page, off);
        s_at[i] = ok ? page * c.page + off * c.row : LLONG_MIN;
        s_sc[i] = page * c.spage + off;
    }
    __syncthreads();
    for (unsigned r0 = 0; r0 < rows; r0 += kRows * kUnroll) {
        if (r0) fetch(r0);
#pragma unroll
        for (int u = 0; u < kUnroll; u++) {
            const unsigned row = r0 + u * kRows + threadIdx.x / LPR;
            const unsigned q = r.by_heads.div(row);
            const unsigned head = row - q * c.heads;
            const bool is_v = q & 1u;
            const long long place = row < rows ? s_at[q >> 1] : LLONG_MIN;
            const bool live = place != LLONG_MIN;
            const long long at = live ? place + head * c.head + part * 8 : 0;
            char* dst = (is_v ? c.v : c.k) + at * EB;
            if constexpr (EB == 2) {
                if (live) *reinterpret_cast<uint4*>(dst) = in[u];
            } else {
                float x[8];
                unpack8<IN>(in[u], x);
                unsigned key = 0;
#pragma unroll
                for (int i = 0; i < 8; i++) key = max(key, __float_as_uint(x[i]) & 0x7fffffffu);
#pragma unroll
                for (int o = LPR / 2; o > 0; o >>= 1)
                    key = max(key, __shfl_xor_sync(0xffffffffu, key, o));
                float scale, mul;
                row_scale<CT>(amax_of(key), scale, mul);
                uint32_t w[2] = {0u, 0u};
                if (mul > 0.f) {
#pragma unroll
                    for (int i = 0; i < 8; i++) x[i] = __fmul_rn(x[i], mul);
                    w[0] = code4<CT>(x[0], x[1], x[2], x[3]);
                    w[1] = code4<CT>(x[4], x[5], x[6], x[7]);
                }
                if (live) {
                    *reinterpret_cast<uint2*>(dst) = make_uint2(w[0], w[1]);
                    if (part == 0) (is_v ? c.vs : c.ks)[s_sc[q >> 1] + head * c.shead] = scale;
                }
            }
        }
    }
}

// Any dim, stride and alignment: one warp per row.
__global__ void __launch_bounds__(kThreads)
kv_write_any_kernel(const KvView c, const Rows r, const int* __restrict__ slots, int in, int ct) {
    const int lane = threadIdx.x & 31;
    const long long rows = (long long)r.tokens * 2 * c.heads;
    const int ib = 2, eb = ct >= kI8 ? 1 : 2;
    for (long long row = (long long)blockIdx.x * (kThreads / 32) + threadIdx.x / 32; row < rows;
         row += (long long)gridDim.x * (kThreads / 32)) {
        const int head = (int)(row % c.heads);
        const long long q = row / c.heads;
        const int tok = (int)(q >> 1);
        const bool is_v = q & 1;
        int page, off;
        if (!slot_place(c, __ldg(slots + tok), page, off)) continue;
        const char* src = is_v ? r.v + tok * r.vr + head * r.vh : r.k + tok * r.kr + head * r.kh;
        char* dst = (is_v ? c.v : c.k) + (page * c.page + off * c.row + head * c.head) * eb;
        if (eb == 2) {
            for (int d = lane; d < c.dim; d += 32)
                reinterpret_cast<uint16_t*>(dst)[d] = reinterpret_cast<const uint16_t*>(src)[d];
            continue;
        }
        unsigned key = 0;
        for (int d = lane; d < c.dim; d += 32)
            key = max(key, __float_as_uint(load_as_float(src + d * ib, in)) & 0x7fffffffu);
        for (int o = 16; o > 0; o >>= 1) key = max(key, __shfl_xor_sync(0xffffffffu, key, o));
        float scale, mul;
        if (ct == kI8) row_scale<kI8>(amax_of(key), scale, mul);
        else row_scale<kE4M3>(amax_of(key), scale, mul);
        for (int d = lane; d < c.dim; d += 32) {
            const float x = mul > 0.f ? __fmul_rn(load_as_float(src + d * ib, in), mul) : 0.f;
            dst[d] = (char)(ct == kI8 ? code_of<kI8>(x) : code_of<kE4M3>(x));
        }
        if (lane == 0)
            (is_v ? c.vs : c.ks)[page * c.spage + head * c.shead + off] = scale;
    }
}

struct Seqs {
    const int *table, *starts, *cu;
    long long tstride;
    int tpages, batch;
};

// (page, offset) of output token t; page < 0: not written (past cu[batch]),
// page >= c.pages: outside, reads as zeros
__device__ __forceinline__ void token_place(const KvView& c, const Seqs& s, int t, int& page,
                                            int& off) {
    page = -1;
    off = 0;
    if (t >= __ldg(s.cu + s.batch)) return;
    int lo = 0, hi = s.batch;                        // cu[lo] <= t < cu[hi]
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (__ldg(s.cu + mid) <= t) lo = mid;
        else hi = mid;
    }
    const long long pos = (long long)t - __ldg(s.cu + lo) + (s.starts ? __ldg(s.starts + lo) : 0);
    page = c.pages;
    if (pos >= 0 && pos < (long long)s.tpages * c.ps) {
        const unsigned i = c.by_ps.div((unsigned)pos);
        off = (int)pos - (int)i * c.ps;
        const int p = __ldg(s.table + lo * s.tstride + i);
        if (p >= 0 && p < c.pages) page = p;
    }
    if (page == c.pages) note_bad_index();
}

template <int CT, int OUT>
__device__ __forceinline__ void decode8(uint2 w, float scale, float (&x)[8]) {
    const uint32_t u[2] = {w.x, w.y};
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const uint32_t b = (u[i >> 2] >> (8 * (i & 3))) & 0xffu;
        if constexpr (CT == kI8) {
            x[i] = (float)(signed char)b * scale;
        } else {
            __nv_fp8_e4m3 e;
            e.__x = (__nv_fp8_storage_t)b;
            x[i] = (float)e * scale;
        }
    }
}

template <int CT, int OUT, int LPR>
__global__ void __launch_bounds__(kThreads)
kv_read_kernel(const KvView c, const Rows r, const Seqs s) {
    __shared__ long long s_at[kMaxTokens], s_sc[kMaxTokens];
    __shared__ int s_ok[kMaxTokens];                 // -1 skip, 0 zeros, 1 read
    const int t0 = blockIdx.x * r.per_block;
    const int nt = min(r.per_block, r.tokens - t0);
    for (int i = threadIdx.x; i < nt; i += kThreads) {
        int page, off;
        token_place(c, s, t0 + i, page, off);
        s_ok[i] = page < 0 ? -1 : page < c.pages;
        s_at[i] = page * c.page + off * c.row;
        s_sc[i] = page * c.spage + off;
    }
    __syncthreads();
    constexpr int kRows = kThreads / LPR;
    constexpr int EB = kv_bytes<CT>;
    const int part = threadIdx.x % LPR;
    const unsigned rows = (unsigned)nt * 2u * (unsigned)c.heads;
    for (unsigned r0 = 0; r0 < rows; r0 += kRows * kUnroll) {
        uint4 in[kUnroll];
        float sc[kUnroll];
        char* dst[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; u++) {
            const unsigned row = r0 + u * kRows + threadIdx.x / LPR;
            const unsigned q = r.by_heads.div(row);
            const unsigned head = row - q * c.heads;
            const int tok = q >> 1;
            const int ok = row < rows ? s_ok[tok] : -1;
            dst[u] = nullptr;
            in[u] = make_uint4(0u, 0u, 0u, 0u);
            sc[u] = 0.f;
            if (ok >= 0)
                dst[u] = q & 1u ? r.v + (t0 + tok) * r.vr + head * r.vh
                                : r.k + (t0 + tok) * r.kr + head * r.kh;
            if (ok > 0) {
                const char* p = (q & 1u ? c.v : c.k) + (s_at[tok] + head * c.head + part * 8) * EB;
                if constexpr (EB == 2) {
                    in[u] = __ldg(reinterpret_cast<const uint4*>(p));
                } else {
                    const uint2 w = __ldg(reinterpret_cast<const uint2*>(p));
                    in[u].x = w.x;
                    in[u].y = w.y;
                    sc[u] = __ldg((q & 1u ? c.vs : c.ks) + s_sc[tok] + head * c.shead);
                }
            }
        }
#pragma unroll
        for (int u = 0; u < kUnroll; u++) {
            if (!dst[u]) continue;
            if constexpr (EB == 2) {
                __stcs(reinterpret_cast<uint4*>(dst[u]) + part, in[u]);
            } else {
                float x[8];
                decode8<CT, OUT>(make_uint2(in[u].x, in[u].y), sc[u], x);
                if constexpr (OUT == kF32) {
                    float4* d = reinterpret_cast<float4*>(dst[u]) + 2 * part;
                    __stcs(d, make_float4(x[0], x[1], x[2], x[3]));
                    __stcs(d + 1, make_float4(x[4], x[5], x[6], x[7]));
                } else {
                    __stcs(reinterpret_cast<uint4*>(dst[u]) + part,
                           make_uint4(pack16<OUT>(x[0], x[1]), pack16<OUT>(x[2], x[3]),
                                      pack16<OUT>(x[4], x[5]), pack16<OUT>(x[6], x[7])));
                }
            }
        }
    }
}

__global__ void __launch_bounds__(kThreads)
kv_read_any_kernel(const KvView c, const Rows r, const Seqs s, int ct, int out) {
    const int lane = threadIdx.x & 31;
    const long long rows = (long long)r.tokens * 2 * c.heads;
    const int eb = ct >= kI8 ? 1 : 2, ob = out == kF32 ? 4 : 2;
    for (long long row = (long long)blockIdx.x * (kThreads / 32) + threadIdx.x / 32; row < rows;
         row += (long long)gridDim.x * (kThreads / 32)) {
        const int head = (int)(row % c.heads);
        const long long q = row / c.heads;
        const int tok = (int)(q >> 1);
        const bool is_v = q & 1;
        int page, off;
        token_place(c, s, tok, page, off);
        if (page < 0) continue;
        char* dst = is_v ? r.v + tok * r.vr + head * r.vh : r.k + tok * r.kr + head * r.kh;
        const bool ok = page < c.pages;
        const char* src = (is_v ? c.v : c.k) + (page * c.page + off * c.row + head * c.head) * eb;
        if (eb == 2) {
            for (int d = lane; d < c.dim; d += 32)
                reinterpret_cast<uint16_t*>(dst)[d] =
                    ok ? reinterpret_cast<const uint16_t*>(src)[d] : (uint16_t)0;
            continue;
        }
        const float scale =
            ok ? __ldg((is_v ? c.vs : c.ks) + page * c.spage + head * c.shead + off) : 0.f;
        for (int d = lane; d < c.dim; d += 32)
            store_as(dst + d * ob, out, ok ? load_as_float(src + d, ct) * scale : 0.f);
    }
}

bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// Rows split into 8-element pieces whose lanes fit a warp, every piece
// aligned: 16 bytes on a 16-bit side, 8 on an 8-bit one, 16 on an fp32 one.
bool pieces(const KvView& c, int type, const Rows& r) {
    if (c.dim != 32 && c.dim != 64 && c.dim != 128 && c.dim != 256) return false;
    const int eb = type >= kI8 ? 1 : 2;
    const long long m = type >= kI8 ? 8 : 16;
    for (long long st : {c.page, c.row, c.head})
        if ((st * eb) % m) return false;
    for (long long st : {r.kr, r.kh, r.vr, r.vh})
        if (st % 16) return false;
    auto ok = [&](const void* p) { return (reinterpret_cast<uintptr_t>(p) & (m - 1)) == 0; };
    return ok(c.k) && ok(c.v) && al16(r.k) && al16(r.v);
}

Rows make_rows(const KvView& c, const zlift_kv_rows& z) {
    Rows r;
    const long long b = z.elem == kF32 ? 4 : 2;
    r.k = static_cast<char*>(z.k);
    r.v = static_cast<char*>(z.v);
    r.kr = z.k_row_stride * b; r.kh = z.k_head_stride * b;
    r.vr = z.v_row_stride * b; r.vh = z.v_head_stride * b;
    r.tokens = z.tokens;
    r.by_heads = FastDiv((unsigned)c.heads);
    // a block's tokens: one pass of kUnroll pieces per thread when there are
    // enough tokens to fill the GPU with such blocks, fewer when not
    const int piece_rows = kThreads / std::max(1, c.dim / 8) * kUnroll;
    const long long want = std::max(1, piece_rows / (2 * c.heads));
    const long long spread = std::max(1LL, (long long)z.tokens / (2 * num_sms()));
    r.per_block = (int)std::max(1LL, std::min({want, spread, (long long)kMaxTokens}));
    return r;
}

int done() {
    const cudaError_t e = cudaGetLastError();
    if (e == cudaSuccess) note_launch();
    return e == cudaSuccess ? 0 : (int)e;
}

template <int IN, int CT>
int write_lpr(const KvView& c, const Rows& r, const int* slots, cudaStream_t s) {
    const unsigned grid = (unsigned)((r.tokens + r.per_block - 1) / r.per_block);
    switch (c.dim) {
    case 32: kv_write_kernel<IN, CT, 4><<<grid, kThreads, 0, s>>>(c, r, slots); break;
    case 64: kv_write_kernel<IN, CT, 8><<<grid, kThreads, 0, s>>>(c, r, slots); break;
    case 128: kv_write_kernel<IN, CT, 16><<<grid, kThreads, 0, s>>>(c, r, slots); break;
    default: kv_write_kernel<IN, CT, 32><<<grid, kThreads, 0, s>>>(c, r, slots); break;
    }
    return done();
}

template <int CT, int OUT>
int read_lpr(const KvView& c, const Rows& r, const Seqs& q, cudaStream_t s) {
    const unsigned grid = (unsigned)((r.tokens + r.per_block - 1) / r.per_block);
    switch (c.dim) {
    case 32: kv_read_kernel<CT, OUT, 4><<<grid, kThreads, 0, s>>>(c, r, q); break;
    case 64: kv_read_kernel<CT, OUT, 8><<<grid, kThreads, 0, s>>>(c, r, q); break;
    case 128: kv_read_kernel<CT, OUT, 16><<<grid, kThreads, 0, s>>>(c, r, q); break;
    default: kv_read_kernel<CT, OUT, 32><<<grid, kThreads, 0, s>>>(c, r, q); break;
    }
    return done();
}

unsigned any_grid(const KvView& c, int tokens) {
    const long long rows = (long long)tokens * 2 * c.heads;
    return (unsigned)std::min((rows + kThreads / 32 - 1) / (kThreads / 32), 1LL << 20);
}

}  // namespace

int kv_write(const KvView& c, int type, const zlift_kv_rows& z, const int* slots, cudaStream_t s) {
    const Rows r = make_rows(c, z);
    if (!pieces(c, type, r)) {
        kv_write_any_kernel<<<any_grid(c, r.tokens), kThreads, 0, s>>>(c, r, slots, z.elem, type);
        return done();
    }
    // a 16-bit cache takes the bits as they are, whichever type they are
    if (type == kF16 || type == kBF16) return write_lpr<kBF16, kBF16>(c, r, slots, s);
    if (type == kI8)
        return z.elem == kBF16 ? write_lpr<kBF16, kI8>(c, r, slots, s)
                               : write_lpr<kF16, kI8>(c, r, slots, s);
    return z.elem == kBF16 ? write_lpr<kBF16, kE4M3>(c, r, slots, s)
                           : write_lpr<kF16, kE4M3>(c, r, slots, s);
}

int kv_read(const KvView& c, int type, const zlift_kv_rows& z, const int* table,
            long long tstride, int tpages, const int* starts, const int* cu, int batch,
            cudaStream_t s) {
    const Rows r = make_rows(c, z);
    const Seqs q{table, starts, cu, tstride, tpages, batch};
    if (!pieces(c, type, r)) {
        kv_read_any_kernel<<<any_grid(c, r.tokens), kThreads, 0, s>>>(c, r, q, type, z.elem);
        return done();
    }
    if (type == kF16 || type == kBF16) return read_lpr<kBF16, kBF16>(c, r, q, s);
    if (type == kI8)
        return z.elem == kBF16 ? read_lpr<kI8, kBF16>(c, r, q, s)
             : z.elem == kF16 ? read_lpr<kI8, kF16>(c, r, q, s)
                              : read_lpr<kI8, kF32>(c, r, q, s);
    return z.elem == kBF16 ? read_lpr<kE4M3, kBF16>(c, r, q, s)
         : z.elem == kF16 ? read_lpr<kE4M3, kF16>(c, r, q, s)
                          : read_lpr<kE4M3, kF32>(c, r, q, s);
}

int kv_cache_error(bool clear) {
    int v = 0;
    cudaMemcpyFromSymbol(&v, g_dev_error, sizeof(int));
    if (clear && v) {
        int z = 0;
        cudaMemcpyToSymbol(g_dev_error, &z, sizeof(int));
    }
    return v;
}

}  // namespace zl
