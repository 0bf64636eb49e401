// paged_decode.cu -- attention of a few query rows per KV head over the
// paged cache: single tokens and short chunks, where reading the cache once
// is the whole cost.
//
// Bytes bound it: per key and KV head 2 * dim * (2 or 1) of them against 4 *
// dim operations per row, and a row is a query head of the group times a
// token: at most 24 rows here, so some 24 to 48 operations a byte, far left of
// the ridge (250).  That is why the products go through mma.sync m16n8k16 and
// not tcgen05: there is no tile of 128 rows to fill nor a trip through tensor
// memory to wait for, and 8-bit codes become operands in registers.
//
// Products.  Keys are the long side: S^T = K.Q^T has 16 keys by 8 rows, O^T =
// V^T.P^T 16 columns by 8 rows, so 8 rows (the usual group) waste nothing, and
// NB = 1 to 3 blocks of 8 rows share every K and V operand.  P^T comes from S^T
// by one 8 x 8 transposition in registers per 8 keys.  The contraction may
// take dim in any order that both sides share: lane (g, t) = (lane / 4, lane %
// 4) takes 16 consecutive bytes of key g, and the query operand is loaded to
// match; in P.V it takes 16 consecutive bytes of its four keys, whose columns
// become output rows g and g + 8 of the products.  Codes of an 8-bit cache widen
// to fp16 exactly; a key's K scale multiplies its scores and its V scale its
// weights.
//
// Loads.  A warp works alone on a piece of the keys (paged_sched.cuh): blocks
// of 8 KB (16 to 64 keys, K and V), its own online softmax, its own ring of
// blocks filled by TMA boxes of up to a page, in the swizzled layout in which
// the lanes' 16-byte reads of V meet no bank conflict and those of K a double
// one.  Lanes that copied their own operands by cp.async had fetched 1.6 times
// the bytes from L2 (32-byte pieces of 64-byte requests): 172 against 124 us on
// the case below.  The next segment's first blocks are asked for before this
// one's rows are stored.
//
// Softmax in log2 units: x = s * scale * log2(e) (* K scale), weights
// ex2(x - m) rounded to the 16-bit type for the product, summed unrounded in
// fp32.  m is the running maximum, or up to kLazy (kLazy8) below it: O and l are
// rescaled only when it grew by more, and both carry the same m, so the
// quotient does not change.  In fp16 a V scale could leave the type's range:
// see v_power.
//
// Measured on one B200 (32 query and 8 KV heads of 128 unless said otherwise):
// 64 ragged sequences of up to 4096 bf16 tokens 125 us, 5.5 TB/s, 84% of the
// copy rate, every byte read from DRAM once.  Handing the last 15 to 30% of the
// keys out in small pieces to whoever was free cost more in parts to join than
// it gained (145 us and up).  16 x 32768 int8 175 us, 3.9 TB/s of codes and
// scales: some 790 warp instructions per block of 8 KB, at 43% of the issue
// slots, and DRAM reads 1.35 times the bytes (5.3 TB/s).  32 sequences of up to
// 4096 e4m3 tokens with 5 drafted ones 80 us (20 rows, three row blocks); 16
// heads of 64, e4m3, 24 x up to 2047 tokens 30 us; one bf16 sequence of 515
// tokens, 8/2 heads 13.6 us, all of it latency (launch, look-ups, first bytes,
// blocks, join).
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
constexpr int kMaxStages = 6;
constexpr int kLeast = 3;                // blocks of keys of a piece, at least
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
    static constexpr int SIDE = (Q8 ? 2 * BK * 4 : 0) + 16;  // scales, keys there; per stage
    static constexpr int smem(int stages) { return kWarps * stages * (8192 + SIDE) + 1024; }
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
// one arrival on `bar` once this thread's copies so far have landed
__device__ __forceinline__ void copy_arrive(uint64_t* bar) {
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" :: "r"(smem_u32(bar)) : "memory");
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
// fp16's 11, and what lies more than 2^17 below the row's maximum and loses bits
// to fp16's subnormals is off by 2^-25 of that maximum (K's codes are off by
// 2^-8 of theirs).
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

// This warp's fragments to (and, summed in key order, from) part slots.
template <int D, int NB>
__device__ __forceinline__ void store_part(float* slot, const float (&o)[D / 16][NB][4],
                                           const float (&m)[NB][2], const float (&l)[NB][2]) {
    const int lane = threadIdx.x & 31, t = lane & 3;
    if (lane < 4) {
#pragma unroll
        for (int nb = 0; nb < NB; nb++)
            reinterpret_cast<float4*>(slot)[nb * 4 + t] = make_float4(m[nb][0], l[nb][0], m[nb][1], l[nb][1]);
    }
    float4* so = reinterpret_cast<float4*>(slot + 16 * NB) + lane;
#pragma unroll
    for (int nb = 0; nb < NB; nb++)
#pragma unroll
        for (int j = 0; j < D / 16; j++)
            so[(nb * (D / 16) + j) * 32] = make_float4(o[j][nb][0], o[j][nb][1], o[j][nb][2], o[j][nb][3]);
}

template <int D, int NB>
__device__ __forceinline__ void join_parts(const PagedAttn& a, const Segment& sg, const Climb& c,
                                           float (&o)[D / 16][NB][4], float (&m)[NB][2],
                                           float (&l)[NB][2]) {
    const int lane = threadIdx.x & 31, t = lane & 3;
    auto slot = [&](int u) { return part_slot(a, 8 * NB, sg.first + c.part(u), c.part(u) == 0); };
#pragma unroll
    for (int nb = 0; nb < NB; nb++) {
        // maxima first (a load each, all independent), then sums and O
        float mm[2] = {-INFINITY, -INFINITY};
#pragma unroll 8
        for (int u = 0; u < c.members; u++) {
            const float4 ml = __ldcg(reinterpret_cast<const float4*>(slot(u)) + nb * 4 + t);
            mm[0] = max_nan(mm[0], ml.x);
            mm[1] = max_nan(mm[1], ml.z);
        }
        m[nb][0] = mm[0];
        m[nb][1] = mm[1];
        const float b0 = mm[0] == -INFINITY ? 0.f : mm[0], b1 = mm[1] == -INFINITY ? 0.f : mm[1];
        l[nb][0] = l[nb][1] = 0.f;
#pragma unroll
        for (int j = 0; j < D / 16; j++)
#pragma unroll
            for (int i = 0; i < 4; i++) o[j][nb][i] = 0.f;
#pragma unroll 4
        for (int u = 0; u < c.members; u++) {
            const float4 ml = __ldcg(reinterpret_cast<const float4*>(slot(u)) + nb * 4 + t);
            const float4* so = reinterpret_cast<const float4*>(slot(u) + 16 * NB) + lane;
            float4 v[D / 16];
#pragma unroll
            for (int j = 0; j < D / 16; j++) v[j] = __ldcg(so + (nb * (D / 16) + j) * 32);
            const float f0 = ex2(ml.x - b0), f1 = ex2(ml.z - b1);
            l[nb][0] = fmaf(ml.y, f0, l[nb][0]);
            l[nb][1] = fmaf(ml.w, f1, l[nb][1]);
#pragma unroll
            for (int j = 0; j < D / 16; j++) {
                o[j][nb][0] = fmaf(v[j].x, f0, o[j][nb][0]);
                o[j][nb][1] = fmaf(v[j].y, f1, o[j][nb][1]);
                o[j][nb][2] = fmaf(v[j].z, f0, o[j][nb][2]);
                o[j][nb][3] = fmaf(v[j].w, f1, o[j][nb][3]);
            }
        }
    }
}

// Rows whose largest |O| is below `from`: a maximum of NaN (paged_codes.cuh).
template <int D, int NB>
__device__ __forceinline__ void distrust_rows(const float (&o)[D / 16][NB][4], float (&m)[NB][2],
                                              const float (&l)[NB][2], float from) {
#pragma unroll
    for (int nb = 0; nb < NB; nb++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
            float mx = 0.f;
#pragma unroll
            for (int j = 0; j < D / 16; j++)
                mx = fmaxf(mx, fmaxf(fabsf(o[j][nb][e]), fabsf(o[j][nb][2 + e])));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
            if (m[nb][e] != -INFINITY && mx < from) m[nb][e] = __uint_as_float(0x7fffffffu);
        }
}

// Normalises and stores a tile's rows, and redoes those a masked key spoilt.
template <int D, int ELEM, int CT, int NB>
__device__ __forceinline__ void finish_rows(const PagedAttn& a, const Segment& sg, int rows,
                                            const float (&o)[D / 16][NB][4], const float (&m)[NB][2],
                                            const float (&l)[NB][2]) {
    using C = DCfg<D, CT, NB>;
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int end = tile_end(a, sg.q, sg.i0 + sg.ni);
    const bool vec = ((reinterpret_cast<uintptr_t>(a.o) | (a.orow * 2) | (a.oh * 2)) & 15) == 0;
#pragma unroll
    for (int nb = 0; nb < NB; nb++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
            const int row = nb * 8 + 2 * t + e;
            const bool live = row < rows;
            const RowPlace pl = row_place(a, sg, live ? row : 0);
            const float inv = l[nb][e] == 0.f ? 0.f : 1.f / l[nb][e];
            char* orow = a.o + (pl.token * a.orow + pl.head * a.oh) * 2;
            float z = 0.f;
#pragma unroll
            for (int c = 0; c < D / 64; c++) {       // 8 columns that follow one another
                uint32_t w[4];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float x = o[4 * c + i][nb][e] * inv, y = o[4 * c + i][nb][2 + e] * inv;
                    z = fmaf(x, 0.f, fmaf(y, 0.f, z));       // NaN once one is not finite
                    w[i] = pack2<ELEM>(x, y);
                }
                const int d = C::VE == 8 ? c * 64 + g * 8 : g * 16 + c * 8;
                char* p = orow + d * 2;
                if (live && vec) {
                    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
                } else if (live) {
#pragma unroll
                    for (int i = 0; i < 8; i++)
                        reinterpret_cast<uint16_t*>(p)[i] = (uint16_t)(w[i >> 1] >> (16 * (i & 1)));
                }
            }
            if (live && g == 0 && a.lse) a.lse[pl.head * a.lh + pl.token] = lse_of(m[nb][e], l[nb][e]);
            const unsigned bad = __ballot_sync(
                0xffffffffu, live && spoilt(m[nb][e], l[nb][e], z) &&
                                redo_row(a, m[nb][e], keys_seen(a, sg.q, pl.token - sg.q.q0), end));
            if (bad)
                for (int i = 0; i < 4; i++)
                    if ((bad >> i) & 0x11111111u) repair_row(a, sg, nb * 8 + 2 * i + e);
        }
}

template <int D, int ELEM, int CT, int NB>
__global__ void __launch_bounds__(kThreads, DCfg<D, CT, NB>::PER_SM)
paged_decode_kernel(const __grid_constant__ CUtensorMap tmK,
                    const __grid_constant__ CUtensorMap tmV,
                    const __grid_constant__ PagedAttn a, const SchedShape shape, const int box,
                    const uint32_t stages) {
    using C = DCfg<D, CT, NB>;
    constexpr int MT = C::Q8 ? kF16 : ELEM;          // type of the products' operands
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>(
        (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    __shared__ uint64_t s_full[kWarps][kMaxStages];
    __shared__ int s_abort;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = lane >> 2, t = lane & 3;
    const int piece = blockIdx.x * kWarps + warp;
    uint8_t* ring = smem + warp * stages * 8192;
    const uint32_t side = smem_u32(smem) + kWarps * stages * 8192 + warp * stages * C::SIDE;
    const float cscale = a.scale * kLog2e;
    if (threadIdx.x == 0) {
        for (int w = 0; w < kWarps; w++)
            for (int i = 0; i < kMaxStages; i++)     // the bytes, and every lane's scales
                mbar_init(&s_full[w][i], C::Q8 ? 33 : 1);
        s_abort = 0;
        fence_mbar_init();
    }
    __syncthreads();                                 // from here on every warp is alone
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
    struct Turn {                                    // a place in the ring, and its phase
        uint32_t at = 0, phase = 0;
        __device__ __forceinline__ void next(uint32_t n) {
            if (++at == n) {
                at = 0;
                phase ^= 1;
            }
        }
    } in, out;
    int in_flight = 0;
    bool alive = true;

    Walker walk;
    walk.start(a, shape, piece);
    Segment sg, nx;
    bool more = walk.next(a, shape, piece, sg);

    // ---- loads: block i of a segment into the next stage
    constexpr int PL = C::BK > 32 ? 2 : 1;           // keys per lane
    auto blocks_of = [&](const Segment& z) { return alive ? (z.k1 - z.k0 + C::BK - 1) / C::BK : 0; };
    auto page_at = [&](const Segment& z, int i, int h) {     // -2: past the end
        const int key = z.k0 + i * C::BK + h * 32 + lane;
        return (C::BK >= 32 || lane < C::BK) && key < z.k1
                   ? __ldg(a.table + z.s * a.tstride + a.c.by_ps.div(key)) : -2;
    };
    auto load_block = [&](const Segment& z, int i, const int (&page)[PL]) {
        const uint32_t stage = in.at;
        in.next(stages);
        in_flight++;
        uint32_t there[PL];
#pragma unroll
        for (int h = 0; h < PL; h++) {
            const bool ok = (unsigned)page[h] < (unsigned)a.c.pages;
            if (!ok && page[h] != -2) note_bad_index();
            there[h] = __ballot_sync(0xffffffffu, ok);
            if constexpr (C::Q8) {
                if (C::BK >= 32 || lane < C::BK) {
                    const int key = z.k0 + i * C::BK + h * 32 + lane;
                    const int off = key - (int)a.c.by_ps.div(key) * a.c.ps;
                    const long long sat = (ok ? page[h] * a.c.spage + off : 0) + z.head * a.c.shead;
                    const uint32_t d = side + stage * C::SIDE + 16 + (h * 32 + lane) * 4;
                    copy_async4(d, a.c.ks + sat, ok);
                    copy_async4(d + C::BK * 4, a.c.vs + sat, ok);
                }
            }
        }
        if constexpr (C::Q8) copy_arrive(&s_full[warp][stage]);
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
            const int key = z.k0 + i * C::BK + r;
            const int off = key - (int)a.c.by_ps.div(key) * a.c.ps;
            // a page that is not there, or not wanted, is asked for out of
            // range and arrives as zeros
            if ((unsigned)pg >= (unsigned)a.c.pages) pg = a.c.pages;
            tma_load_4d(ring + stage * 8192 + box_kv * 4096 + box_col * (C::BK * C::RB) + r * C::RB,
                        box_kv ? &tmV : &tmK, &s_full[warp][stage], box_col * (128 / C::EB), off,
                        z.head, pg);
        }
    };
    // of a segment's first blocks, all but one of which are loaded ahead
    int page[kMaxStages][PL];
    auto first_pages = [&](const Segment& z) {
#pragma unroll
        for (int i = 0; i < kMaxStages; i++)
#pragma unroll
            for (int h = 0; h < PL; h++) page[i][h] = i < stages ? page_at(z, i, h) : -2;
    };
    auto first_blocks = [&](const Segment& z) {
        const int n = blocks_of(z);
#pragma unroll
        for (int i = 0; i < kMaxStages - 1; i++)
            if (i < stages - 1 && i < n) load_block(z, i, page[i]);
    };
    if (more) {
        first_pages(sg);
        first_blocks(sg);
    }

    while (more) {
        const int rows = sg.ni * a.group;
        const int mine = blocks_of(sg);
        int ahead[PL];                               // pages of the next block to load
#pragma unroll
        for (int h = 0; h < PL; h++) {
            ahead[h] = page[kMaxStages - 1][h];
#pragma unroll
            for (int i = 1; i < kMaxStages - 1; i++)
                if (stages - 1 == i) ahead[h] = page[i][h];
        }

        // ---- queries: row nb * 8 + g, dim permuted as the K pieces are
        uint32_t qb[D / 16][NB][2];
        float qscale[NB][2];                         // of rows nb*8 + 2t, + 1
        int lim[NB][2];                              // keys that they see
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
        float vmost = 0.f, vpow = 1.f, lpow = 0.f;   // 8 bit: see v_power
        uint32_t vleast = 0xffffffffu;               // of this lane's keys

        for (int i = 0; i < mine; i++) {
            __syncwarp();                            // the stage to fill is no longer read
            if (i + (int)stages - 1 < mine) load_block(sg, i + stages - 1, ahead);
#pragma unroll
            for (int h = 0; h < PL; h++) ahead[h] = page_at(sg, i + stages, h);
            const uint32_t stage = out.at;
            const uint32_t st = smem_u32(ring) + stage * 8192, sc = side + stage * C::SIDE;
            alive = __all_sync(0xffffffffu, mbar_wait(&s_full[warp][stage], out.phase, &s_abort));
            if (!alive) break;
            out.next(stages);
            in_flight--;
            const int kb = sg.k0 + i * C::BK;
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
                    if (mx > m[nb][e] + (C::Q8 ? kLazy8 : kLazy)) {     // also from -inf
                        alpha[nb][e] = ex2(m[nb][e] - mx);
                        m[nb][e] = mx;
                        grow = true;
                    }
                }
            float vfix = 1.f;
            if constexpr (C::Q8) {
                uint32_t big = 0;
#pragma unroll
                for (int h = 0; h < PL; h++)
                    if (C::BK >= 32 || lane < C::BK) {
                        const float s = __uint_as_float(lds4(sc + 16 + (C::BK + h * 32 + lane) * 4));
                        big = max(big, scale_key(s, 0u));
                        vleast = min(vleast, scale_key(s, 0xffffffffu));
                    }
                vfix = v_power(__uint_as_float(__reduce_max_sync(0xffffffffu, big)), vmost, vpow);
                if (vfix != 1.f) lpow = exponent_of(vpow);
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

        // ---- the next segment's pages are on their way while this one ends
        more = walk.next(a, shape, piece, nx);
        if (more) first_pages(nx);
#pragma unroll
        for (int nb = 0; nb < NB; nb++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
                l[nb][e] += __shfl_xor_sync(0xffffffffu, l[nb][e], 4);
                l[nb][e] += __shfl_xor_sync(0xffffffffu, l[nb][e], 8);
                l[nb][e] += __shfl_xor_sync(0xffffffffu, l[nb][e], 16);
                m[nb][e] -= lpow;                    // log2 units, of O and l alike
            }
        if constexpr (C::Q8) {
            if (wide_scales(__reduce_min_sync(0xffffffffu, vleast), vmost, vpow))
                distrust_rows<D, NB>(o, m, l, trusted_from<ELEM, CT>(sg.k1 - sg.k0, vmost, vpow));
        }
        bool final = sg.parts == 1;
        if (!final) store_part<D, NB>(part_slot(a, C::ROWS, piece, sg.part == 0), o, m, l);
        if (more) first_blocks(nx);
        if (!final) {
            Climb c(sg);
#pragma unroll 1
            for (;; c.up()) {
                __threadfence();
                __syncwarp();
                int last = 0;
                if (lane == 0) last = c.arrive(a, sg, 0);
                if (!__shfl_sync(0xffffffffu, last, 0)) break;
                if (c.members > 1) {
                    __threadfence();
                    join_parts<D, NB>(a, sg, c, o, m, l);
                }
                if (c.top()) {
                    final = true;
                    break;
                }
                if (c.members > 1)
                    store_part<D, NB>(part_slot(a, C::ROWS, sg.first + c.part(0), c.part(0) == 0), o, m, l);
            }
        }
        if (final) finish_rows<D, ELEM, CT, NB>(a, sg, rows, o, m, l);
        sg = nx;
    }
    if (!alive) {                                    // gave up: not before the copies have landed
        for (; in_flight > 0; in_flight--, out.next(stages)) copy_wait(&s_full[warp][out.at], out.phase);
    }
}

// row blocks of 8: those of the longest chunk, as the caller tells it
int row_blocks(const PagedAttn& a) {
    const long long rows = (long long)std::max(1, a.max_q) * a.group;
    return (int)std::min<long long>((rows + 7) / 8, kMaxNB);
}

// How many blocks share the work: all that fit the GPU, or fewer when the page
// table cannot hold that much.
int most_blocks(const PagedAttn& a) {
    return std::min((row_blocks(a) == 1 ? 3 : 2) * num_sms(), kMaxPieces / kWarps);
}
int blocks_for(const PagedAttn& a) {
    const int step = 4096 / (a.c.dim * (a.type >= kI8 ? 1 : 2));
    const long long keys = (long long)a.tpages * a.c.ps;
    const long long tile_tokens = 8 * row_blocks(a) / a.group;
    const long long tiles = (a.total_q + tile_tokens - 1) / tile_tokens + a.batch;
    const long long most = std::max(1LL, (keys + step - 1) / step) * std::min<long long>(tiles, 1 << 20) *
                           a.c.heads;
    return (int)std::min<long long>(most_blocks(a), (most + kLeast * kWarps - 1) / (kLeast * kWarps));
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
            cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 C::smem(kMaxStages));
        if (e != cudaSuccess) return (int)e;
        attr_set.fetch_or(bit);
    }
    const int blocks = blocks_for(a);
    const SchedShape shape = sched_shape(a, C::ROWS / a.group, C::BK, kLeast, blocks * kWarps);
    int box = 8;                                     // tokens of a page side by side
    while (box < C::BK && a.c.ps % (2 * box) == 0) box *= 2;
    CUtensorMap tk, tv;
    if (!cache_map(&tk, a, a.c.k, C::RB, box) || !cache_map(&tv, a, a.c.v, C::RB, box)) return 1;
    // stages that fit beside the other blocks of the SM; all of them where a
    // block has its SM to itself
    const int per_sm = (blocks + num_sms() - 1) / num_sms();
    const int stages = per_sm == 1 ? kMaxStages : per_sm == 2 ? 3 : 2;
    kern<<<blocks, kThreads, C::smem(stages), s>>>(tk, tv, a, shape, box, stages);
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
           2ull * kWarps * most_blocks(a) * slot_floats(8 * row_blocks(a), a.c.dim) * sizeof(float);
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

int paged_decode_set_wait_limit(unsigned long long ns) { return set_unit_wait_limit(ns); }

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
