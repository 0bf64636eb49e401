// paged_decode.cu -- attention of a few query rows per KV head over the
// paged cache: single tokens and short chunks, where reading the cache once
// is the whole cost.
//
// Rows.  The group's query heads times the chunk's tokens are the rows of one
// matrix operand (16 per tile), so K and V are read once for all of them.
// Bytes bound it: per key and head 2 * dim * (2 or 1) bytes against 16 * dim
// * 4 operations per 16 rows, some 64 operations a byte at most, far left of
// the ridge.  That is why the products go through mma.sync m16n8k16 and not
// tcgen05: operands come from registers in the layout that a plain row of the
// cache already has, rows that do not exist cost little, and there is no
// tile of 128 rows to fill nor a trip through tensor memory to wait for.
//
// Loads.  A warp works alone: blocks of BK keys, its own online softmax, its
// own ring of kStages blocks in shared memory filled by cp.async.  Each lane
// fetches exactly the 16-byte pieces that it will itself use as operands, so
// the ring needs no barrier, no swizzle and no bank conflicts (piece i of lane
// l sits at i * 512 + l * 16).  The freedom that makes this work is the order
// of the contraction: with the same permutation of dim on both sides,
// q.k is unchanged, so lane (g, t) (g = lane / 4, t = lane % 4) takes 16
// consecutive bytes of key g and the query operand is loaded to match; in P.V
// it takes 16 consecutive bytes of its four keys, whose columns become the n
// index of 8 or 16 products.  8-bit codes turn into 16-bit operands in
// registers, exactly; a key's K scale multiplies its score and its V scale its
// weight.
//
// Softmax in log2 units: x = s * scale * log2(e) (* K scale), weights
// ex2(x - m) rounded to the 16-bit type for the product, summed unrounded in
// fp32.  m is the running maximum, or up to 2^kLazy below it: O and l are
// rescaled only when it grew by more, and both carry the same m, so the
// quotient does not change.  In fp16 the V scale could leave the type's
// range, so weights carry a power of two beside it that follows the largest V
// scale seen.
//
// Work is split as in paged_sched.cuh; a block's four warps take blocks of
// keys in turn and join through shared memory.
#include "gemm.h"
#include "paged_codes.cuh"
#include "paged_finish.cuh"

#include <algorithm>
#include <atomic>

namespace zl {

namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kRows = 16;
constexpr int kStages = 3;
constexpr int kBlocksPerSM = 2;
constexpr float kLazy = 6.f;
constexpr uint32_t kNone = 0xffffffffu;
constexpr float kLog2e = 1.4426950408889634f;

template <int D, int CT>
struct DCfg {
    static constexpr int EB = kv_bytes<CT>;
    static constexpr bool Q8 = CT >= kI8;
    static constexpr int BK = 4096 / (D * EB);           // keys per block: 4 KB of K, 4 KB of V
    static constexpr int NT = BK / 8;                    // score tiles
    static constexpr int KCH = D * EB / 64;              // 16-byte K pieces per lane and key
    static constexpr int VP = D * EB >= 128 ? 16 : 8;    // bytes of a V piece
    static constexpr int VCH = D * EB / (8 * VP);        // V pieces per lane and key
    static constexpr int VE = VP / EB;                   // elements of one
    static constexpr int STAGE = 8192 + (Q8 ? 2 * BK * 4 : 0) + 16;
    static constexpr int RING = kStages * STAGE;
    static constexpr int JOIN = kWarps * kRows * (D + 4) * 4;
    static constexpr int SMEM = kWarps * RING > JOIN ? kWarps * RING : JOIN;
    static_assert(NT * KCH == 8 && BK / 4 * VCH * VP == 128, "a block is 8 KB");
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t s) {
    return __byte_perm(a, b, s);
}

template <int ELEM>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    if constexpr (ELEM == kBF16) {
        const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&v);
    } else {
        const __half2 v = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&v);
    }
}

// 16 x 8 += 16 x 16 . 16 x 8
template <int ELEM>
__device__ __forceinline__ void mma16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                      uint32_t b1) {
    if constexpr (ELEM == kBF16)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
            "{%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
            "{%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// copies N bytes, or writes N zeros where `there` is false (src is not read then)
template <int N>
__device__ __forceinline__ void copy_async(uint32_t dst, const char* src, bool there) {
    const int bytes = there ? N : 0;
    if constexpr (N == 16)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;"
                     :: "r"(dst), "l"(src), "r"(bytes) : "memory");
    else
        asm volatile("cp.async.ca.shared.global [%0], [%1], %3, %2;"
                     :: "r"(dst), "l"(src), "r"(bytes), "n"(N) : "memory");
}
__device__ __forceinline__ void copy_commit() {
    asm volatile("cp.async.commit_group;" ::: "memory");
}
template <int N>
__device__ __forceinline__ void copy_wait() {
    asm volatile("cp.async.wait_group %0;" :: "n"(N) : "memory");
}

__device__ __forceinline__ uint4 lds16(uint32_t a) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
    return v;
}
__device__ __forceinline__ uint2 lds8(uint32_t a) {
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a));
    return v;
}
__device__ __forceinline__ uint32_t lds4(uint32_t a) {
    uint32_t v;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(a));
    return v;
}

template <int D, int ELEM, int CT>
__global__ void __launch_bounds__(kThreads, kBlocksPerSM)
paged_decode_kernel(const __grid_constant__ PagedAttn a, const SchedShape shape) {
    using C = DCfg<D, CT>;
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ float s_m[kWarps][kRows], s_l[kWarps][kRows];
    __shared__ int s_last, s_bad[kRows];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = lane >> 2, t = lane & 3;
    const int block = blockIdx.x;
    const uint32_t ring = smem_u32(smem) + warp * C::RING;
    const float cscale = a.scale * kLog2e * (CT == kE4M3 ? Code<ELEM, CT>::kUnscale : 1.f);

    Walker walk;
    walk.start(a, shape, block, gridDim.x);
    Segment sg;
    while (walk.next(a, shape, block, sg)) {
        const int rows = sg.ni * a.group;
        const char* kbase = a.c.k + (long long)sg.head * a.c.head * C::EB;
        const char* vbase = a.c.v + (long long)sg.head * a.c.head * C::EB;
        const float* ksb = a.c.ks + sg.head * a.c.shead;
        const float* vsb = a.c.vs + sg.head * a.c.shead;
        const int* table = a.table + sg.s * a.tstride;

        // ---- queries: rows g and g + 8, dim permuted as the K pieces are
        uint32_t qa[D / 16][4];
        int lim[2];                                  // keys that the row sees
#pragma unroll
        for (int r = 0; r < 2; r++) {
            const int row = g + 8 * r;
            const bool live = row < rows;
            const int tok = live ? row / a.group : 0;
            const int hd = sg.head * a.group + (live ? row - tok * a.group : 0);
            lim[r] = live ? tile_end(a, sg.q, sg.i0 + tok + 1) : 0;
            const char* qrow = a.q + ((sg.q.q0 + sg.i0 + tok) * a.qr + hd * a.qh) * 2;
            if constexpr (C::EB == 2) {
#pragma unroll
                for (int c = 0; c < D / 32; c++) {
                    uint4 w = make_uint4(0u, 0u, 0u, 0u);
                    if (live) w = __ldg(reinterpret_cast<const uint4*>(qrow + c * 64 + t * 16));
                    qa[2 * c][r] = w.x;
                    qa[2 * c][r + 2] = w.y;
                    qa[2 * c + 1][r] = w.z;
                    qa[2 * c + 1][r + 2] = w.w;
                }
            } else {
#pragma unroll
                for (int c = 0; c < D / 64; c++)
#pragma unroll
                    for (int h = 0; h < 2; h++) {    // 8 of the piece's 16 elements
                        uint4 w = make_uint4(0u, 0u, 0u, 0u);
                        if (live)
                            w = __ldg(reinterpret_cast<const uint4*>(qrow + c * 128 + t * 32 + h * 16));
                        qa[4 * c + 2 * h][r] = w.x;
                        qa[4 * c + 2 * h][r + 2] = w.y;
                        qa[4 * c + 2 * h + 1][r] = w.z;
                        qa[4 * c + 2 * h + 1][r + 2] = w.w;
                    }
            }
        }
        // below this key no row of the tile masks anything
        const int lim_all = tile_end(a, sg.q, sg.i0 + 1);

        float o[D / 8][4];
#pragma unroll
        for (int j = 0; j < D / 8; j++)
#pragma unroll
            for (int i = 0; i < 4; i++) o[j][i] = 0.f;
        float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
        float vmost = 0.f, vpow = 1.f;               // fp16: see v_power
        const int stride = kWarps * C::BK;
        const int first = sg.k0 + warp * C::BK;
        const int mine = sg.k1 > first ? (sg.k1 - first + stride - 1) / stride : 0;

        // ---- loads: block i into stage i % kStages
        constexpr int PL = C::BK > 32 ? 2 : 1;       // keys per lane
        int page[PL];
        auto fetch_pages = [&](int i) {
#pragma unroll
            for (int h = 0; h < PL; h++) {
                const int key = first + i * stride + h * 32 + lane;
                page[h] = -2;                        // past the end
                if (lane < C::BK && key < sg.k1) page[h] = __ldg(table + a.c.by_ps.div(key));
            }
        };
        auto load_block = [&](int i) {
            const uint32_t st = ring + (i % kStages) * C::STAGE;
            uint32_t at[PL];
            uint32_t there[PL];
#pragma unroll
            for (int h = 0; h < PL; h++) {
                const int key = first + i * stride + h * 32 + lane;
                const int off = key - (int)a.c.by_ps.div(key) * a.c.ps;
                const bool ok = page[h] >= 0 && page[h] < a.c.pages;
                if (!ok && page[h] != -2) note_bad_index();
                at[h] = ok ? (uint32_t)((page[h] * a.c.page + off * a.c.row) * C::EB / 32) : kNone;
                there[h] = __ballot_sync(0xffffffffu, ok);
                if constexpr (C::Q8) {
                    if (lane < C::BK) {
                        const long long sat = ok ? page[h] * a.c.spage + off : 0;
                        const uint32_t d = st + 8192 + (h * 32 + lane) * 4;
                        copy_async<4>(d, reinterpret_cast<const char*>(ksb + sat), ok);
                        copy_async<4>(d + C::BK * 4, reinterpret_cast<const char*>(vsb + sat), ok);
                    }
                }
            }
            if (lane == 0) {
                const uint32_t d = st + 8192 + (C::Q8 ? 2 * C::BK * 4 : 0);
                asm volatile("st.shared.v2.u32 [%0], {%1,%2};"
                             :: "r"(d), "r"(there[0]), "r"(there[PL - 1]) : "memory");
            }
#pragma unroll
            for (int n = 0; n < C::NT; n++) {
                const uint32_t x = __shfl_sync(0xffffffffu, at[PL > 1 ? n / 4 : 0], (n * 8 + g) & 31);
                const char* p = kbase + (x == kNone ? 0ull : (unsigned long long)x * 32) + t * 16;
#pragma unroll
                for (int c = 0; c < C::KCH; c++)
                    copy_async<16>(st + (n * C::KCH + c) * 512 + lane * 16, p + c * 64, x != kNone);
            }
#pragma unroll
            for (int n = 0; n < C::BK / 4; n++) {    // keys 2t, 2t+1, 2t+8, 2t+9 of each 16
                const int key = (n >> 2) * 16 + 2 * t + (n & 1) + 8 * ((n >> 1) & 1);
                const uint32_t x = __shfl_sync(0xffffffffu, at[PL > 1 ? n / 8 : 0], key & 31);
                const char* p = vbase + (x == kNone ? 0ull : (unsigned long long)x * 32) + g * C::VP;
#pragma unroll
                for (int c = 0; c < C::VCH; c++)
                    copy_async<C::VP>(st + 4096 + (n * C::VCH + c) * (32 * C::VP) + lane * C::VP,
                                      p + c * 8 * C::VP, x != kNone);
            }
        };

        fetch_pages(0);
#pragma unroll
        for (int i = 0; i < kStages - 1; i++) {
            if (i < mine) load_block(i);
            fetch_pages(i + 1);
            copy_commit();
        }
        for (int i = 0; i < mine; i++) {
            copy_wait<kStages - 2>();
            __syncwarp();
            if (i + kStages - 1 < mine) load_block(i + kStages - 1);
            fetch_pages(i + kStages);
            copy_commit();
            const uint32_t st = ring + (i % kStages) * C::STAGE;
            const int kb = first + i * stride;

            // ---- scores
            float x[C::NT][4];
#pragma unroll
            for (int n = 0; n < C::NT; n++) {
                x[n][0] = x[n][1] = x[n][2] = x[n][3] = 0.f;
#pragma unroll
                for (int c = 0; c < C::KCH; c++) {
                    const uint4 w = lds16(st + (n * C::KCH + c) * 512 + lane * 16);
                    if constexpr (C::EB == 2) {
                        mma16<ELEM>(x[n], qa[2 * c], w.x, w.y);
                        mma16<ELEM>(x[n], qa[2 * c + 1], w.z, w.w);
                    } else {
                        const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            uint32_t b0, b1;
                            Code<ELEM, CT>::widen(u[e], b0, b1);
                            mma16<ELEM>(x[n], qa[4 * c + e], b0, b1);
                        }
                    }
                }
            }
            const uint2 there = lds8(st + 8192 + (C::Q8 ? 2 * C::BK * 4 : 0));
            const uint32_t all = C::BK >= 32 ? 0xffffffffu : (1u << C::BK) - 1u;
            const bool edge = kb + C::BK > lim_all || there.x != all || there.y != all;
#pragma unroll
            for (int n = 0; n < C::NT; n++) {
                float f0 = cscale, f1 = cscale;
                if constexpr (C::Q8) {
                    const uint2 ks = lds8(st + 8192 + (n * 8 + 2 * t) * 4);
                    f0 *= __uint_as_float(ks.x);
                    f1 *= __uint_as_float(ks.y);
                }
                x[n][0] *= f0;
                x[n][1] *= f1;
                x[n][2] *= f0;
                x[n][3] *= f1;
                if (edge) {
                    const uint32_t mask = PL > 1 && n >= 4 ? there.y : there.x;
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        const int j = n * 8 + 2 * t + e;
                        const bool here = (mask >> (j & 31)) & 1u;
                        if (!here || kb + j >= lim[0]) x[n][e] = -INFINITY;
                        if (!here || kb + j >= lim[1]) x[n][2 + e] = -INFINITY;
                    }
                }
            }

            // ---- running maximum
            float alpha[2] = {1.f, 1.f}, base[2];
            bool grow = false;
#pragma unroll
            for (int r = 0; r < 2; r++) {
                float mx = x[0][2 * r];
#pragma unroll
                for (int n = 0; n < C::NT; n++) mx = fmaxf(mx, fmaxf(x[n][2 * r], x[n][2 * r + 1]));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                if (mx > m[r] + kLazy) {             // also from -inf
                    alpha[r] = ex2(m[r] - mx);
                    m[r] = mx;
                    grow = true;
                }
                base[r] = m[r] == -INFINITY ? 0.f : m[r];
            }
            float vfix = 1.f;
            if constexpr (C::Q8 && ELEM == kF16) {
                float big = 0.f;
                if (lane < C::BK) {
                    big = __uint_as_float(lds4(st + 8192 + (C::BK + lane) * 4));
                    if (PL > 1)
                        big = fmaxf(big, __uint_as_float(lds4(st + 8192 + (C::BK + 32 + lane) * 4)));
                }
#pragma unroll
                for (int o2 = 16; o2 > 0; o2 >>= 1)
                    big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, o2));
                vfix = v_power(big, vmost, vpow);
                grow = grow || vfix != 1.f;
            }
            if (__any_sync(0xffffffffu, grow)) {
                l[0] *= alpha[0];
                l[1] *= alpha[1];
#pragma unroll
                for (int j = 0; j < D / 8; j++) {
                    o[j][0] *= alpha[0] * vfix;
                    o[j][1] *= alpha[0] * vfix;
                    o[j][2] *= alpha[1] * vfix;
                    o[j][3] *= alpha[1] * vfix;
                }
            }

            // ---- weights, and P.V sixteen keys at a time
#pragma unroll
            for (int kk = 0; kk < C::BK / 16; kk++) {
                uint32_t pa[4];
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const int n = 2 * kk + h;
                    float p[4];
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        p[e] = ex2(x[n][e] - base[e >> 1]);
                        l[e >> 1] += p[e];
                    }
                    if constexpr (C::Q8) {
                        const uint2 vs = lds8(st + 8192 + (C::BK + n * 8 + 2 * t) * 4);
                        float v0 = __uint_as_float(vs.x), v1 = __uint_as_float(vs.y);
                        if constexpr (ELEM == kF16) {
                            v0 *= vpow;
                            v1 *= vpow;
                        }
                        p[0] *= v0;
                        p[1] *= v1;
                        p[2] *= v0;
                        p[3] *= v1;
                        if (edge) {                  // 0 * NaN: a masked key's scale
                            if (x[n][0] == -INFINITY) p[0] = 0.f;
                            if (x[n][1] == -INFINITY) p[1] = 0.f;
                            if (x[n][2] == -INFINITY) p[2] = 0.f;
                            if (x[n][3] == -INFINITY) p[3] = 0.f;
                        }
                    }
                    pa[2 * h] = pack2<ELEM>(p[0], p[1]);
                    pa[2 * h + 1] = pack2<ELEM>(p[2], p[3]);
                }
#pragma unroll
                for (int c = 0; c < C::VCH; c++) {
                    uint32_t w[4][C::VP / 4];
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        const uint32_t p = st + 4096 + ((kk * 4 + k) * C::VCH + c) * (32 * C::VP) +
                                           lane * C::VP;
                        if constexpr (C::VP == 16) {
                            const uint4 v = lds16(p);
                            w[k][0] = v.x; w[k][1] = v.y; w[k][2] = v.z; w[k][3] = v.w;
                        } else {
                            const uint2 v = lds8(p);
                            w[k][0] = v.x; w[k][1] = v.y;
                        }
                    }
#pragma unroll
                    for (int i4 = 0; i4 < C::VP / 4; i4++) {
                        if constexpr (C::EB == 2) {
                            mma16<ELEM>(o[c * C::VE + 2 * i4], pa, prmt(w[0][i4], w[1][i4], 0x5410),
                                        prmt(w[2][i4], w[3][i4], 0x5410));
                            mma16<ELEM>(o[c * C::VE + 2 * i4 + 1], pa,
                                        prmt(w[0][i4], w[1][i4], 0x7632),
                                        prmt(w[2][i4], w[3][i4], 0x7632));
                        } else {
#pragma unroll
                            for (int h = 0; h < 2; h++) {
                                const uint32_t sel = h ? 0x7362 : 0x5140;
                                uint32_t lo0, hi0, lo1, hi1;
                                Code<ELEM, CT>::widen(prmt(w[0][i4], w[1][i4], sel), lo0, hi0);
                                Code<ELEM, CT>::widen(prmt(w[2][i4], w[3][i4], sel), lo1, hi1);
                                mma16<ELEM>(o[c * C::VE + 4 * i4 + 2 * h], pa, lo0, lo1);
                                mma16<ELEM>(o[c * C::VE + 4 * i4 + 2 * h + 1], pa, hi0, hi1);
                            }
                        }
                    }
                }
            }
        }
        copy_wait<0>();

        // ---- join the warps: maxima and sums, then O through shared memory
#pragma unroll
        for (int r = 0; r < 2; r++) {
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
            if (t == 0) {
                s_m[warp][g + 8 * r] = m[r];
                s_l[warp][g + 8 * r] = l[r];
            }
        }
        __syncthreads();                             // also: every ring is drained
        float* so = reinterpret_cast<float*>(smem);  // [warp][row][D + 4]
        const float unv = (CT == kE4M3 ? Code<ELEM, CT>::kUnscale : 1.f) / vpow;
#pragma unroll
        for (int c = 0; c < C::VCH; c++)
#pragma unroll
            for (int e = 0; e < C::VE; e++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int row = g + 8 * (i >> 1);
                    const int d = c * 8 * C::VE + (2 * t + (i & 1)) * C::VE + e;
                    if (row < rows) so[(warp * kRows + row) * (D + 4) + d] = o[c * C::VE + e][i] * unv;
                }
        if (threadIdx.x < kRows) s_bad[threadIdx.x] = 0;
        __syncthreads();
        const bool whole = sg.parts == 1;
        float* slot = whole ? nullptr : part_slot(a, kRows, block, sg.part == 0);
        for (int i = threadIdx.x; i < rows * D; i += kThreads) {
            const int row = i / D, d = i - row * D;
            float mm = s_m[0][row];
#pragma unroll
            for (int w = 1; w < kWarps; w++) mm = fmaxf(mm, s_m[w][row]);
            const float b = mm == -INFINITY ? 0.f : mm;
            float ll = 0.f, v = 0.f;
#pragma unroll
            for (int w = 0; w < kWarps; w++) {
                const float f = ex2(s_m[w][row] - b);
                ll += s_l[w][row] * f;
                v += so[(w * kRows + row) * (D + 4) + d] * f;
            }
            if (whole) {
                write_out<ELEM>(a, sg, row, d, mm, ll, v, s_bad);
            } else {
                slot[2 * kRows + i] = v;
                if (d == 0) {
                    slot[2 * row] = mm;
                    slot[2 * row + 1] = ll;
                }
            }
        }
        bool final = whole;
        if (!whole) {
            __threadfence();
            __syncthreads();
            if (threadIdx.x == 0) s_last = count_part(a, sg);
            __syncthreads();
            final = s_last;
            if (final) {
                __threadfence();
                for (int i = threadIdx.x; i < rows * D; i += kThreads) {
                    const int row = i / D, d = i - row * D;
                    float mm = -INFINITY, ll = 0.f, v = 0.f;
                    for (int p = 0; p < sg.parts; p++) {
                        const float* ps = part_slot(a, kRows, sg.first + p, p == 0);
                        const float pm = __ldcg(ps + 2 * row), pl = __ldcg(ps + 2 * row + 1);
                        const float pv = __ldcg(ps + 2 * kRows + i);
                        const float nm = fmaxf(mm, pm);
                        const float b = nm == -INFINITY ? 0.f : nm;
                        const float f0 = ex2(mm - b), f1 = ex2(pm - b);
                        ll = ll * f0 + pl * f1;
                        v = v * f0 + pv * f1;
                        mm = nm;
                    }
                    write_out<ELEM>(a, sg, row, d, mm, ll, v, s_bad);
                }
            }
        }
        __syncthreads();
        if (final) repair_rows(a, sg, rows, s_bad, warp, kWarps);
        __syncthreads();
    }
}

template <int D, int ELEM, int CT>
int launch(const PagedAttn& a, cudaStream_t s) {
    using C = DCfg<D, CT>;
    auto kern = paged_decode_kernel<D, ELEM, CT>;
    static std::atomic<unsigned long long> attr_set{0};
    int dev = 0;
    cudaGetDevice(&dev);
    const unsigned long long bit = 1ull << (dev & 63);
    if (!(attr_set.load() & bit)) {
        const cudaError_t e =
            cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
        if (e != cudaSuccess) return (int)e;
        attr_set.fetch_or(bit);
    }
    const SchedShape shape{kRows / a.group, kWarps * C::BK, 2};
    kern<<<decode_blocks(), kThreads, C::SMEM, s>>>(a, shape);
    const cudaError_t e = cudaGetLastError();
    if (e == cudaSuccess) note_launch();
    return e == cudaSuccess ? 0 : (int)e;
}

template <int ELEM, int CT>
int launch_dim(const PagedAttn& a, cudaStream_t s) {
    return a.c.dim == 128 ? launch<128, ELEM, CT>(a, s) : launch<64, ELEM, CT>(a, s);
}

}  // namespace

int decode_blocks() { return std::min(kBlocksPerSM * num_sms(), kMaxBlocks); }

size_t paged_decode_workspace(const PagedAttn& a) {
    return kCounterBytes + 2ull * decode_blocks() * slot_floats(kRows, a.c.dim) * sizeof(float);
}

int paged_decode(const PagedAttn& a, cudaStream_t s) {
    if (a.elem == kBF16)
        return a.type == kI8 ? launch_dim<kBF16, kI8>(a, s)
             : a.type == kE4M3 ? launch_dim<kBF16, kE4M3>(a, s)
                               : launch_dim<kBF16, kBF16>(a, s);
    return a.type == kI8 ? launch_dim<kF16, kI8>(a, s)
         : a.type == kE4M3 ? launch_dim<kF16, kE4M3>(a, s)
                           : launch_dim<kF16, kF16>(a, s);
}

int paged_decode_error(bool clear) {
    int v = 0;
    cudaMemcpyFromSymbol(&v, g_dev_error, sizeof(int));
    if (clear && v) {
        int z = 0;
        cudaMemcpyToSymbol(g_dev_error, &z, sizeof(int));
    }
    return v;
}

}  // namespace zl
