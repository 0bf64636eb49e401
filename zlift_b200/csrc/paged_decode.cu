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
constexpr int kMaxNB = 3;
constexpr int kLeast = 2;                // steps of a piece, at least
constexpr int kExtra = 2;                // small pieces for each large one
constexpr int kShare = 200;              // 256ths of the work in large pieces
constexpr float kLazy = 6.f;
constexpr float kLog2e = 1.4426950408889634f;

template <int D, int CT, int NB>
struct DCfg {
    static constexpr int EB = kv_bytes<CT>;
    static constexpr bool Q8 = CT >= kI8;
    static constexpr int ROWS = 8 * NB;
    static constexpr int BK = 4096 / (D * EB);           // keys per block: 4 KB of K, 4 KB of V
    static constexpr int NT = BK / 8;
    static constexpr int KCH = D * EB / 64;              // 16-byte K pieces per lane and key
    static constexpr int VP = D * EB >= 128 ? 16 : 8;    // bytes of a V piece
    static constexpr int VCH = D * EB / (8 * VP);        // V pieces per lane and key
    static constexpr int VE = VP / EB;                   // elements of one
    static constexpr int RB = D * EB > 128 ? 128 : D * EB;   // bytes of a row in a box
    static constexpr int CB = D * EB / RB;               // boxes side by side
    static constexpr int PER_SM = NB == 1 ? 3 : 2;       // blocks per SM
    static constexpr int STAGES = NB == 1 ? 2 : 3;
    static constexpr int RING = STAGES * 8192;
    static constexpr int SIDE = (Q8 ? 2 * BK * 4 : 0) + 16;  // scales, keys there; per stage
    static constexpr int SIDE_OFF = kWarps * RING;
    static constexpr int JOIN = kWarps * ROWS * (D + 4) * 4;
    static constexpr int SMEM = SIDE_OFF + kWarps * STAGES * SIDE + 1024;
    static_assert(JOIN <= SIDE_OFF, "the join reuses the rings");
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
__device__ __forceinline__ void mma16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                      uint32_t a3, const uint32_t (&b)[2]) {
    if constexpr (ELEM == kBF16)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
            "{%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b[0]), "r"(b[1]));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
            "{%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b[0]), "r"(b[1]));
}

// an 8 x 8 matrix of 16-bit values across the warp, transposed
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

// copies a scale, or writes zero where `there` is false (src is not read then)
__device__ __forceinline__ void copy_async4(uint32_t dst, const float* src, bool there) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;"
                 :: "r"(dst), "l"(src), "r"(there ? 4 : 0) : "memory");
}
__device__ __forceinline__ void copy_commit() {
    asm volatile("cp.async.commit_group;" ::: "memory");
}
template <int N>
__device__ __forceinline__ void copy_wait() {
    asm volatile("cp.async.wait_group %0;" :: "n"(N) : "memory");
}

// N (2 or 4) floats at an address aligned for them
template <int N>
__device__ __forceinline__ void load_vec(float (&x)[N], const float* p) {
    if constexpr (N == 4) {
        const float4 v = *reinterpret_cast<const float4*>(p);
        x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
    } else {
        const float2 v = *reinterpret_cast<const float2*>(p);
        x[0] = v.x; x[1] = v.y;
    }
}
template <int N>
__device__ __forceinline__ void load_vec_cg(float (&x)[N], const float* p) {
    if constexpr (N == 4) {
        const float4 v = __ldcg(reinterpret_cast<const float4*>(p));
        x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
    } else {
        const float2 v = __ldcg(reinterpret_cast<const float2*>(p));
        x[0] = v.x; x[1] = v.y;
    }
}
template <int N>
__device__ __forceinline__ void store_vec(float* p, const float (&x)[N]) {
    if constexpr (N == 4) *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
    else *reinterpret_cast<float2*>(p) = make_float2(x[0], x[1]);
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

// Row block nb of the query operand from bf16 to fp16, the type that codes
// widen to most cheaply and weights keep most bits in.  A row is brought to a
// maximum of [1, 2) by a power of two (returned: its inverse): bf16's 8 bits fit
// fp16's 11, and what lies 2^14 below the row's maximum and loses bits to
// fp16's subnormals is off by 2^-25 of that maximum, as fp32 sums are.
template <int D, int NB>
__device__ __forceinline__ float halve_row(uint32_t (&qb)[D / 16][NB][2], int nb) {
    unsigned most = 0;
#pragma unroll
    for (int i = 0; i < D / 16; i++)
#pragma unroll
        for (int h = 0; h < 2; h++)
            most = max(most, max(qb[i][nb][h] << 16 & 0x7fffffffu, qb[i][nb][h] & 0x7fff0000u));
    most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
    most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
    const int e = most ? min(max((int)(most >> 23) - 127, -120), 120) : 0;
    const float f = __uint_as_float((uint32_t)(127 - e) << 23);
#pragma unroll
    for (int i = 0; i < D / 16; i++)
#pragma unroll
        for (int h = 0; h < 2; h++)
            qb[i][nb][h] = pack2<kF16>(__uint_as_float(qb[i][nb][h] << 16) * f,
                                       __uint_as_float(qb[i][nb][h] & 0xffff0000u) * f);
    return __uint_as_float((uint32_t)(127 + e) << 23);
}

template <int D, int ELEM, int CT, int NB>
__global__ void __launch_bounds__(kThreads, DCfg<D, CT, NB>::PER_SM)
paged_decode_kernel(const __grid_constant__ CUtensorMap tmK,
                    const __grid_constant__ CUtensorMap tmV,
                    const __grid_constant__ PagedAttn a, const SchedShape shape, const int box) {
    using C = DCfg<D, CT, NB>;
    constexpr int kRows = C::ROWS, kStages = C::STAGES;
    constexpr int MT = C::Q8 ? kF16 : ELEM;          // type of the products' operands
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>(
        (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    __shared__ uint64_t s_full[kWarps][kStages];
    __shared__ int s_abort;
    __shared__ float s_m[kWarps][kRows], s_l[kWarps][kRows];
    __shared__ int s_last, s_bad[kRows];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = lane >> 2, t = lane & 3;
    const int block = blockIdx.x;
    uint8_t* ring = smem + warp * C::RING;
    const uint32_t side = smem_u32(smem + C::SIDE_OFF) + warp * kStages * C::SIDE;
    const float cscale = a.scale * kLog2e;
    if (threadIdx.x == 0) {
        for (int w = 0; w < kWarps; w++)
            for (int i = 0; i < kStages; i++) mbar_init(&s_full[w][i], 1);
        s_abort = 0;
        fence_mbar_init();
    }
    __syncthreads();
    // where this lane's operands sit in a stage: K pieces t and t + 4 of row g,
    // V piece g of rows 2t and 2t + 1 (swizzled as TMA stores them)
    const uint32_t k_even = C::RB == 128 ? g * 128 + ((t ^ g) << 4) : g * 64 + ((t ^ (g >> 1)) << 4);
    const uint32_t k_odd = k_even ^ 64;
    const uint32_t v_even = C::RB == 128 ? 2 * t * 128 + ((g ^ (2 * t)) << 4)
                                         : 2 * t * 64 + (((g >> 1) ^ t) << 4) + (g & 1) * 8;
    const uint32_t v_odd = C::RB == 128 ? (2 * t + 1) * 128 + ((g ^ (2 * t + 1)) << 4) : v_even + 64;
    // the boxes this lane fetches: K or V, box column, box row
    const int box_kv = lane & 1, box_col = (lane >> 1) % C::CB, box_row = (lane >> 1) / C::CB;
    const bool box_mine = box_row * box < C::BK;
    uint32_t filled = 0, used = 0;                   // blocks so far
    bool alive = true;

    Walker walk;
    walk.start(a, shape, block);
    Segment sg;
    while (walk.next(a, shape, block, sg)) {
        const int rows = sg.ni * a.group;
        const float* ksb = a.c.ks + sg.head * a.c.shead;
        const float* vsb = a.c.vs + sg.head * a.c.shead;
        const int* table = a.table + sg.s * a.tstride;
        const int stride = kWarps * C::BK;
        const int first = sg.k0 + warp * C::BK;
        const int mine = alive && sg.k1 > first ? (sg.k1 - first + stride - 1) / stride : 0;

        // ---- loads: block i into stage i % kStages
        constexpr int PL = C::BK > 32 ? 2 : 1;       // keys per lane
        int page[PL];
        auto fetch_pages = [&](int i) {
#pragma unroll
            for (int h = 0; h < PL; h++) {
                const int key = first + i * stride + h * 32 + lane;
                page[h] = -2;                        // past the end
                if ((C::BK >= 32 || lane < C::BK) && key < sg.k1)
                    page[h] = __ldg(table + a.c.by_ps.div(key));
            }
        };
        auto load_block = [&](int i) {
            const uint32_t stage = filled % kStages;
            filled++;
            uint32_t there[PL];
#pragma unroll
            for (int h = 0; h < PL; h++) {
                const bool ok = (unsigned)page[h] < (unsigned)a.c.pages;
                if (!ok && page[h] != -2) note_bad_index();
                there[h] = __ballot_sync(0xffffffffu, ok);
                if constexpr (C::Q8) {
                    if (C::BK >= 32 || lane < C::BK) {
                        const int key = first + i * stride + h * 32 + lane;
                        const int off = key - (int)a.c.by_ps.div(key) * a.c.ps;
                        const long long sat = ok ? page[h] * a.c.spage + off : 0;
                        const uint32_t d = side + stage * C::SIDE + 16 + (h * 32 + lane) * 4;
                        copy_async4(d, ksb + sat, ok);
                        copy_async4(d + C::BK * 4, vsb + sat, ok);
                    }
                }
            }
            if (lane == 0) {
                asm volatile("st.shared.v2.u32 [%0], {%1,%2};" :: "r"(side + stage * C::SIDE),
                             "r"(there[0]), "r"(there[PL - 1]) : "memory");
                mbar_expect_tx(&s_full[warp][stage], 8192);
            }
            __syncwarp();
            const int r = box_row * box;
            int pg = __shfl_sync(0xffffffffu, page[0], r & 31);
            if constexpr (PL > 1) {
                const int p1 = __shfl_sync(0xffffffffu, page[1], r & 31);
                if (r >= 32) pg = p1;
            }
            if (box_mine) {
                const int key = first + i * stride + r;
                const int off = key - (int)a.c.by_ps.div(key) * a.c.ps;
                // a page that is not there, or not wanted, is asked for out of
                // range and arrives as zeros
                if ((unsigned)pg >= (unsigned)a.c.pages) pg = a.c.pages;
                tma_load_4d(ring + stage * 8192 + box_kv * 4096 + box_col * (C::BK * C::RB) + r * C::RB,
                            box_kv ? &tmV : &tmK, &s_full[warp][stage], box_col * (128 / C::EB), off,
                            sg.head, pg);
            }
        };

        fetch_pages(0);
#pragma unroll
        for (int i = 0; i < kStages - 1; i++) {
            if (i < mine) load_block(i);
            fetch_pages(i + 1);
            copy_commit();
        }

        // ---- queries: row nb * 8 + g, dim permuted as the K pieces are
        uint32_t qb[D / 16][NB][2];
        float qscale[NB][2];                         // of rows nb*8 + 2t, + 1 (8-bit caches)
        int lim[NB][2];                              // keys that rows nb*8 + 2t, + 1 see
#pragma unroll
        for (int nb = 0; nb < NB; nb++) {
            const int row = nb * 8 + g;
            const bool live = row < rows;
            const RowPlace pl = row_place(a, sg, live ? row : 0);
            const char* qrow = a.q + (pl.token * a.qr + pl.head * a.qh) * 2;
            // 16-byte pieces of q: one for two 16-bit steps, half of one K piece of codes
#pragma unroll
            for (int c = 0; c < D / 32; c++) {
                const int at = C::EB == 2 ? c * 64 + t * 16 : (c >> 1) * 128 + t * 32 + (c & 1) * 16;
                uint4 w = make_uint4(0u, 0u, 0u, 0u);
                if (live) w = __ldg(reinterpret_cast<const uint4*>(qrow + at));
                qb[2 * c][nb][0] = w.x;
                qb[2 * c][nb][1] = w.y;
                qb[2 * c + 1][nb][0] = w.z;
                qb[2 * c + 1][nb][1] = w.w;
            }
            if constexpr (C::Q8 && ELEM == kBF16) {
                const float f = halve_row<D>(qb, nb);
                qscale[nb][0] = cscale * __shfl_sync(0xffffffffu, f, 8 * t);
                qscale[nb][1] = cscale * __shfl_sync(0xffffffffu, f, 8 * t + 4);
            } else {
                qscale[nb][0] = qscale[nb][1] = cscale;
            }
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const int r = nb * 8 + 2 * t + e;
                lim[nb][e] = r < rows ? tile_end(a, sg.q, sg.i0 + r / a.group + 1) : 0;
            }
        }
        // up to this key no row of the tile masks anything
        const int lim_all = tile_end(a, sg.q, sg.i0 + 1);

        float o[D / 16][NB][4];
        float m[NB][2], base[NB][2], l[NB][2];
#pragma unroll
        for (int nb = 0; nb < NB; nb++) {
#pragma unroll
            for (int j = 0; j < D / 16; j++)
#pragma unroll
                for (int i = 0; i < 4; i++) o[j][nb][i] = 0.f;
            m[nb][0] = m[nb][1] = -INFINITY;
            base[nb][0] = base[nb][1] = 0.f;
            l[nb][0] = l[nb][1] = 0.f;
        }
        float vmost = 0.f, vpow = 1.f, lpow = 0.f;   // fp16: see v_power

        for (int i = 0; i < mine; i++) {
            __syncwarp();                            // the stage to fill is no longer read
            if (i + kStages - 1 < mine) load_block(i + kStages - 1);
            fetch_pages(i + kStages);
            copy_commit();
            const uint32_t stage = used % kStages;
            const uint32_t st = smem_u32(ring) + stage * 8192, sc = side + stage * C::SIDE;
            copy_wait<kStages - 1>();
            alive = __all_sync(0xffffffffu, mbar_wait(&s_full[warp][stage], (used / kStages) & 1, &s_abort));
            if (!alive) break;
            used++;
            const int kb = first + i * stride;
            // V rows past the keys, in a box that is partly wanted, may hold
            // anything: 0 times them must be 0
            const int left = sg.k1 - kb;
            if (left < C::BK) {
                constexpr int PIECES = C::RB / 16;
                for (int j = lane; j < (C::BK - left) * PIECES * C::CB; j += 32) {
                    const int row = left + j / (PIECES * C::CB), c = j % (PIECES * C::CB);
                    *reinterpret_cast<uint4*>(ring + stage * 8192 + 4096 + (c / PIECES) * (C::BK * C::RB) +
                                              row * C::RB + (c % PIECES) * 16) = make_uint4(0u, 0u, 0u, 0u);
                }
                fence_async_smem();                  // before TMA fills the stage again
                __syncwarp();
            }

            // ---- scores: keys g and g + 8 of each 16, rows 2t and 2t + 1
            float x[C::BK / 16][NB][4];
#pragma unroll
            for (int kk = 0; kk < C::BK / 16; kk++) {
#pragma unroll
                for (int nb = 0; nb < NB; nb++)
                    x[kk][nb][0] = x[kk][nb][1] = x[kk][nb][2] = x[kk][nb][3] = 0.f;
#pragma unroll
                for (int c = 0; c < C::KCH; c++) {
                    const uint32_t p = st + (c & 1 ? k_odd : k_even) + (c >> 1) * (C::BK * C::RB) +
                                       kk * 16 * C::RB;
                    const uint4 w = lds16(p), v = lds16(p + 8 * C::RB);
                    if constexpr (C::EB == 2) {
#pragma unroll
                        for (int nb = 0; nb < NB; nb++) {
                            mma16<MT>(x[kk][nb], w.x, v.x, w.y, v.y, qb[2 * c][nb]);
                            mma16<MT>(x[kk][nb], w.z, v.z, w.w, v.w, qb[2 * c + 1][nb]);
                        }
                    } else {
                        const uint32_t wu[4] = {w.x, w.y, w.z, w.w}, vu[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            uint32_t a0, a1, a2, a3;
                            Code<MT, CT>::widen(wu[e], a0, a2);
                            Code<MT, CT>::widen(vu[e], a1, a3);
#pragma unroll
                            for (int nb = 0; nb < NB; nb++)
                                mma16<MT>(x[kk][nb], a0, a1, a2, a3, qb[4 * c + e][nb]);
                        }
                    }
                }
            }
            const uint2 there = lds8(sc);
            constexpr uint32_t ALL = C::BK >= 32 ? 0xffffffffu : (1u << (C::BK & 31)) - 1u;
            const bool edge = kb + C::BK > lim_all || there.x != ALL || there.y != ALL;
            bool grow = false;
            float alpha[NB][2];
#pragma unroll
            for (int kk = 0; kk < C::BK / 16; kk++) {
                float f0 = 1.f, f1 = 1.f;
                if constexpr (C::Q8) {
                    f0 = __uint_as_float(lds4(sc + 16 + (kk * 16 + g) * 4));
                    f1 = __uint_as_float(lds4(sc + 16 + (kk * 16 + g + 8) * 4));
                }
#pragma unroll
                for (int nb = 0; nb < NB; nb++) {
                    x[kk][nb][0] *= f0 * qscale[nb][0];
                    x[kk][nb][1] *= f0 * qscale[nb][1];
                    x[kk][nb][2] *= f1 * qscale[nb][0];
                    x[kk][nb][3] *= f1 * qscale[nb][1];
                }
                if (edge) {
                    const uint32_t mask = PL > 1 && kk >= 2 ? there.y : there.x;
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        const int j = kk * 16 + g + 8 * h;
                        const bool here = (mask >> (j & 31)) & 1u;
#pragma unroll
                        for (int nb = 0; nb < NB; nb++)
#pragma unroll
                            for (int e = 0; e < 2; e++)
                                if (!here || kb + j >= lim[nb][e]) x[kk][nb][2 * h + e] = -INFINITY;
                    }
                }
            }

            // ---- running maximum
#pragma unroll
            for (int nb = 0; nb < NB; nb++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    float mx = fmaxf(x[0][nb][e], x[0][nb][2 + e]);
#pragma unroll
                    for (int kk = 1; kk < C::BK / 16; kk++)
                        mx = fmaxf(mx, fmaxf(x[kk][nb][e], x[kk][nb][2 + e]));
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
                    alpha[nb][e] = 1.f;
                    if (mx > m[nb][e] + kLazy) {     // also from -inf
                        alpha[nb][e] = ex2(m[nb][e] - mx);
                        m[nb][e] = mx;
                        grow = true;
                    }
                }
            float vfix = 1.f;
            if constexpr (C::Q8) {
                float big = 0.f;
                if (C::BK >= 32 || lane < C::BK)
                    big = __uint_as_float(lds4(sc + 16 + (C::BK + lane) * 4));
                if (PL > 1)
                    big = fmaxf(big, __uint_as_float(lds4(sc + 16 + (C::BK + 32 + lane) * 4)));
#pragma unroll
                for (int o2 = 16; o2 > 0; o2 >>= 1)
                    big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, o2));
                vfix = v_power(big, vmost, vpow);
                if (vfix != 1.f) lpow = log2f(vpow); // a power of two: exact
                grow = grow || vfix != 1.f;
            }
            if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
                for (int nb = 0; nb < NB; nb++)
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        const float f = alpha[nb][e] * vfix;
                        // the power of two rides in the exponent, on O and l alike
                        base[nb][e] = (m[nb][e] == -INFINITY ? 0.f : m[nb][e]) - lpow;
                        l[nb][e] *= f;
#pragma unroll
                        for (int j = 0; j < D / 16; j++) {
                            o[j][nb][e] *= f;
                            o[j][nb][2 + e] *= f;
                        }
                    }
            }

            // ---- weights, and P.V sixteen keys at a time
#pragma unroll
            for (int kk = 0; kk < C::BK / 16; kk++) {
                float v0 = 1.f, v1 = 1.f;
                if constexpr (C::Q8) {
                    v0 = __uint_as_float(lds4(sc + 16 + (C::BK + kk * 16 + g) * 4));
                    v1 = __uint_as_float(lds4(sc + 16 + (C::BK + kk * 16 + g + 8) * 4));
                }
                uint32_t pb[NB][2];
#pragma unroll
                for (int nb = 0; nb < NB; nb++) {
                    float p[4];
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        p[e] = ex2(x[kk][nb][e] - base[nb][e & 1]);
                        l[nb][e & 1] += p[e];
                    }
                    if constexpr (C::Q8) {
                        // (a masked key's scale may be NaN: paged_finish.cuh)
                        p[0] *= v0;
                        p[1] *= v0;
                        p[2] *= v1;
                        p[3] *= v1;
                    }
                    pb[nb][0] = transpose8(pack2<MT>(p[0], p[1]));
                    pb[nb][1] = transpose8(pack2<MT>(p[2], p[3]));
                }
#pragma unroll
                for (int c = 0; c < C::VCH; c++) {
                    uint32_t w[4][C::VP / 4];
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        const uint32_t p = st + 4096 + (k & 1 ? v_odd : v_even) + c * (C::BK * C::RB) +
                                           (kk * 16 + (k >> 1) * 8) * C::RB;
                        if constexpr (C::VP == 16) {
                            const uint4 v = lds16(p);
                            w[k][0] = v.x; w[k][1] = v.y; w[k][2] = v.z; w[k][3] = v.w;
                        } else {
                            const uint2 v = lds8(p);
                            w[k][0] = v.x; w[k][1] = v.y;
                        }
                    }
                    // columns e and e + 1 of this lane's VE: output rows g, g + 8
#pragma unroll
                    for (int i4 = 0; i4 < C::VP / 4; i4++) {
                        if constexpr (C::EB == 2) {
                            const uint32_t a0 = prmt(w[0][i4], w[1][i4], 0x5410);
                            const uint32_t a1 = prmt(w[0][i4], w[1][i4], 0x7632);
                            const uint32_t a2 = prmt(w[2][i4], w[3][i4], 0x5410);
                            const uint32_t a3 = prmt(w[2][i4], w[3][i4], 0x7632);
#pragma unroll
                            for (int nb = 0; nb < NB; nb++)
                                mma16<MT>(o[c * C::VE / 2 + i4][nb], a0, a1, a2, a3, pb[nb]);
                        } else {
#pragma unroll
                            for (int h = 0; h < 2; h++) {
                                const uint32_t sel = h ? 0x7362 : 0x5140;
                                uint32_t a0, a1, a2, a3;
                                Code<MT, CT>::widen(prmt(w[0][i4], w[1][i4], sel), a0, a1);
                                Code<MT, CT>::widen(prmt(w[2][i4], w[3][i4], sel), a2, a3);
#pragma unroll
                                for (int nb = 0; nb < NB; nb++)
                                    mma16<MT>(o[c * C::VE / 2 + 2 * i4 + h][nb], a0, a1, a2, a3, pb[nb]);
                            }
                        }
                    }
                }
            }
        }
        copy_wait<0>();

        // ---- join the warps: maxima and sums, then O through shared memory
#pragma unroll
        for (int nb = 0; nb < NB; nb++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
                float sum = l[nb][e];
                sum += __shfl_xor_sync(0xffffffffu, sum, 4);
                sum += __shfl_xor_sync(0xffffffffu, sum, 8);
                sum += __shfl_xor_sync(0xffffffffu, sum, 16);
                if (g == 0) {
                    s_m[warp][nb * 8 + 2 * t + e] = m[nb][e] - lpow;
                    s_l[warp][nb * 8 + 2 * t + e] = sum;
                }
            }
        if (threadIdx.x < kRows) s_bad[threadIdx.x] = 0;
        __syncthreads();                             // also: every ring is drained
        float* so = reinterpret_cast<float*>(smem);  // [warp][row][D + 4]
#pragma unroll
        for (int j = 0; j < D / 16; j++)
#pragma unroll
            for (int nb = 0; nb < NB; nb++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int row = nb * 8 + 2 * t + (i & 1);
                    const int e = 2 * j + (i >> 1);  // column within the lane's pieces
                    const int d = (e / C::VE) * 8 * C::VE + g * C::VE + e % C::VE;
                    if (row < rows) so[(warp * kRows + row) * (D + 4) + d] = o[j][nb][i];
                }
        __syncthreads();
        const bool whole = sg.parts == 1;
        float* slot = whole ? nullptr : part_slot(a, kRows, block, sg.part == 0);
        constexpr int VL = D / 32;                   // columns per lane
        for (int row = warp; row < rows; row += kWarps) {
            float mm = s_m[0][row];
#pragma unroll
            for (int w = 1; w < kWarps; w++) mm = fmaxf(mm, s_m[w][row]);
            const float b = mm == -INFINITY ? 0.f : mm;
            float ll = 0.f, v[VL] = {};
#pragma unroll
            for (int w = 0; w < kWarps; w++) {
                const float f = ex2(s_m[w][row] - b);
                ll += s_l[w][row] * f;
                float x[VL];
                load_vec<VL>(x, so + (w * kRows + row) * (D + 4) + lane * VL);
#pragma unroll
                for (int i = 0; i < VL; i++) v[i] += x[i] * f;
            }
            if (whole) {
                write_out<ELEM, VL>(a, sg, row, lane * VL, mm, ll, v, s_bad);
            } else {
                store_vec<VL>(slot + 2 * kRows + row * D + lane * VL, v);
                if (lane == 0) *reinterpret_cast<float2*>(slot + 2 * row) = make_float2(mm, ll);
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
                for (int row = warp; row < rows; row += kWarps) {
                    float mm = -INFINITY, ll = 0.f, v[VL] = {};
                    for (int p0 = 0; p0 < sg.parts; p0 += 32) {
                        // lane i: maximum and sum of part p0 + i
                        const int np = min(32, sg.parts - p0);
                        float2 ml = make_float2(-INFINITY, 0.f);
                        if (lane < np)
                            ml = __ldcg(reinterpret_cast<const float2*>(
                                part_slot(a, kRows, sg.first + p0 + lane, p0 + lane == 0) + 2 * row));
                        float nm = ml.x;
#pragma unroll
                        for (int o2 = 16; o2 > 0; o2 >>= 1)
                            nm = fmaxf(nm, __shfl_xor_sync(0xffffffffu, nm, o2));
                        nm = fmaxf(nm, mm);
                        const float b = nm == -INFINITY ? 0.f : nm;
                        const float f = ex2(ml.x - b), back = ex2(mm - b);
                        float sum = ml.y * f;
#pragma unroll
                        for (int o2 = 16; o2 > 0; o2 >>= 1)
                            sum += __shfl_xor_sync(0xffffffffu, sum, o2);
                        ll = ll * back + sum;
#pragma unroll
                        for (int i = 0; i < VL; i++) v[i] *= back;
                        mm = nm;
                        for (int p = 0; p < np; p += 8) {
                            float x[8][VL];
#pragma unroll
                            for (int u = 0; u < 8; u++)
                                if (p + u < np)
                                    load_vec_cg<VL>(x[u], part_slot(a, kRows, sg.first + p0 + p + u,
                                                                    p0 + p + u == 0) +
                                                              2 * kRows + row * D + lane * VL);
#pragma unroll
                            for (int u = 0; u < 8; u++) {
                                const float fu = __shfl_sync(0xffffffffu, f, (p + u) & 31);
                                if (p + u < np) {
#pragma unroll
                                    for (int i = 0; i < VL; i++) v[i] = fmaf(x[u][i], fu, v[i]);
                                }
                            }
                        }
                    }
                    write_out<ELEM, VL>(a, sg, row, lane * VL, mm, ll, v, s_bad);
                }
            }
        }
        __syncthreads();
        if (final) repair_rows(a, sg, rows, s_bad, warp, kWarps);
        fence_async_smem();                          // the rings are TMA's again
        __syncthreads();
    }
}

// row blocks of 8: those of the longest chunk, as the caller tells it
int row_blocks(const PagedAttn& a) {
    const long long rows = (long long)std::max(1, a.max_q) * a.group;
    return (int)std::min<long long>((rows + 7) / 8, kMaxNB);
}

// How many pieces the work is cut into: those that start together, fewer when
// the page table cannot hold that much work, and the small ones behind them.
struct Pieces {
    int blocks, extra;
};
int most_together(const PagedAttn& a) {
    return std::min((row_blocks(a) == 1 ? 3 : 2) * num_sms(), kMaxBlocks / (1 + kExtra));
}
Pieces pieces(const PagedAttn& a) {
    const int nb = row_blocks(a), together = most_together(a);
    const int step = kWarps * 4096 / (a.c.dim * (a.type >= kI8 ? 1 : 2));
    const long long keys = (long long)a.tpages * a.c.ps;
    const long long tile_tokens = 8 * nb / a.group;
    const long long tiles = (a.total_q + tile_tokens - 1) / tile_tokens + a.batch;
    const long long most = std::max(1LL, (keys + step - 1) / step) * std::min<long long>(tiles, 1 << 20) *
                           a.c.heads;
    if (most <= (long long)together * 2 * kLeast)
        return {(int)std::max(1LL, (most + kLeast - 1) / kLeast), 0};
    return {together, kExtra * together};
}

using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*,
                              const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                              const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeFn encode_fn() {
    static std::atomic<EncodeFn> fn{nullptr};
    EncodeFn f = fn.load();
    if (f) return f;
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) ==
            cudaSuccess && q == cudaDriverEntryPointSuccess) {
        f = reinterpret_cast<EncodeFn>(ptr);
        fn.store(f);
    }
    return f;
}

// {dim, page_size, heads, pages}, boxes of `box` rows of row_bytes
bool cache_map(CUtensorMap* tm, const PagedAttn& a, const void* base, int row_bytes, int box_rows) {
    EncodeFn enc = encode_fn();
    if (!enc) return false;
    const int eb = a.type >= kI8 ? 1 : 2;
    const cuuint64_t dims[4] = {(cuuint64_t)a.c.dim, (cuuint64_t)a.c.ps, (cuuint64_t)a.c.heads,
                                (cuuint64_t)a.c.pages};
    const cuuint64_t st[3] = {a.c.ps > 1 ? (cuuint64_t)a.c.row * eb : 16,
                              a.c.heads > 1 ? (cuuint64_t)a.c.head * eb : 16,
                              a.c.pages > 1 ? (cuuint64_t)a.c.page * eb : 16};
    const cuuint32_t box[4] = {(cuuint32_t)(row_bytes / eb), (cuuint32_t)box_rows, 1, 1};
    const cuuint32_t ones[4] = {1, 1, 1, 1};
    const CUtensorMapDataType type = a.type >= kI8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8
                                   : a.type == kBF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                     : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    return enc(tm, type, 4, const_cast<void*>(base), dims, st, box, ones,
               CU_TENSOR_MAP_INTERLEAVE_NONE,
               row_bytes == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
               CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int D, int ELEM, int CT, int NB>
int launch(const PagedAttn& a, cudaStream_t s) {
    using C = DCfg<D, CT, NB>;
    auto kern = paged_decode_kernel<D, ELEM, CT, NB>;
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
    const Pieces pc = pieces(a);
    const SchedShape shape{C::ROWS / a.group, kWarps * C::BK, kLeast, pc.blocks, pc.extra, kShare};
    int box = 8;                                     // tokens of a page side by side
    while (box < C::BK && a.c.ps % (2 * box) == 0) box *= 2;
    CUtensorMap tk, tv;
    if (!cache_map(&tk, a, a.c.k, C::RB, box) || !cache_map(&tv, a, a.c.v, C::RB, box)) return 1;
    kern<<<pc.blocks + pc.extra, kThreads, C::SMEM, s>>>(tk, tv, a, shape, box);
    const cudaError_t e = cudaGetLastError();
    if (e == cudaSuccess) note_launch();
    return e == cudaSuccess ? 0 : (int)e;
}

template <int D, int ELEM, int CT>
int launch_rows(const PagedAttn& a, cudaStream_t s) {
    switch (row_blocks(a)) {
    case 1: return launch<D, ELEM, CT, 1>(a, s);
    case 2: return launch<D, ELEM, CT, 2>(a, s);
    default: return launch<D, ELEM, CT, 3>(a, s);
    }
}

template <int ELEM, int CT>
int launch_dim(const PagedAttn& a, cudaStream_t s) {
    return a.c.dim == 128 ? launch_rows<128, ELEM, CT>(a, s) : launch_rows<64, ELEM, CT>(a, s);
}

}  // namespace

int decode_max_rows() { return 8 * kMaxNB; }

size_t paged_decode_workspace(const PagedAttn& a) {
    // (not by the length of the page table, which may grow between calls)
    return kCounterBytes +
           2ull * (1 + kExtra) * most_together(a) * slot_floats(8 * row_blocks(a), a.c.dim) * sizeof(float);
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
