// paged_chunk.cu -- attention of a chunk of new tokens over the paged cache
// on the sm_100a tensor cores.
//
// The matrix products bound it (4 * dim operations per query row and key
// against 2 * dim bytes per key shared by 256 rows), so it has the shape of
// the contiguous forward kernel (fmha.cu): two tiles of 128 query rows, key
// tiles of 128, S = Q.K^T and O += P.V by tcgen05.mma, P in the tensor memory
// of S, one softmax thread per row, the two tiles taking turns on the tensor
// core.  What differs:
//
//   rows    A tile's rows are (token, head of the group), token-major: K and V
//           are read once for all query heads that share them, and a causal
//           chunk of few tokens still fills its tile.  One TMA box
//           {64 dims, group, tokens} of Q puts them in that order.
//   work    paged_sched.cuh: 148 blocks, each an equal piece of all key tiles
//           of all row tiles, so that a short chunk over a long context uses
//           the whole GPU.  The rings and barriers run on across a block's
//           segments; the next segment's loads and first products run under
//           the epilogue of the last.
//   16 bit  One warp loads: lane i takes box i of the tile (the largest power
//           of two of tokens that divides the page, 8 to 128), looks its page
//           up and issues its TMA.  Boxes past the sequence, or whose page is
//           not in the cache, are asked for out of range and arrive as zeros.
//           What a page holds behind the sequence's last token may be
//           anything, NaN included, and 0 times that must be 0: those V rows
//           are zeroed in shared memory before the tile is handed on.
//   8 bit   Six warps load codes (16 bytes a lane, eight lanes a row of 128),
//           widen them to 16 bits exactly and store them in the swizzled
//           layout that the tensor core reads; K of the next tile is on its
//           way while V of this one is widened, and the other way round.  The
//           K scale of a key multiplies its column of S and the V scale its
//           column of P, which is fp16 (what that loses where the scales lie
//           far apart: paged_codes.cuh).
//
// Measured on one B200 (32/8 heads of 128): 512 new tokens over 32768, bf16,
// 295 us in short runs (925 TFLOP/s), 345 us at the power cap; 4 ragged chunks
// of up to 2048 over up to 4096 tokens, bf16 366 us, int8 594 us, e4m3 590 us.
// What 8 bits cost there: the loaders' and the softmax's instructions share the
// issue slots (45% used, 0.65 of 8.4 warps waiting for instructions) and 128
// registers a thread, with some 190 bytes of spills.  Earlier forms, when this
// one took 565 us: three loader warps in place of six 842 us; the softmax
// unrolled for both halves of a warp's rows 646 us; a row of scores per thread,
// whose 128 scales every thread reads, 760 us.
//
// Roles (warps): 0-3 and 4-7 softmax of tile 0 and 1, then the loaders (one
// or six), then the MMA issuer.
#include "gemm.h"
#include "paged_codes.cuh"
#include "paged_finish.cuh"

#include <algorithm>
#include <atomic>

namespace zl {

namespace {

constexpr int BQ = 128;              // rows per tile
constexpr int BKEY = 128;            // keys per tile
constexpr float kLog2e = 1.4426950408889634f;
constexpr int kBoxBytes = 128 * 128; // 128 rows of one 128-byte column box

template <int D, bool Q8>
struct PCfg {
    static constexpr int BOXES = D / 64;
    static constexpr int TILE_BYTES = 128 * D * 2;
    // warps; with six and the issuer a block has 15, and 128 registers a thread
    static constexpr int LOADERS = Q8 ? 6 : 1;
    static constexpr int THREADS = 256 + LOADERS * 32 + 32;
    static constexpr int MMA_WARP = 8 + LOADERS;
    static constexpr int KV_OFF = 2 * TILE_BYTES;
    static constexpr int SIDE = 8192;                        // barriers, scales, walkers
    static constexpr int FIT = (227 * 1024 - 1024 - SIDE - KV_OFF) / TILE_BYTES;
    static constexpr int NSLOT = FIT > 8 ? 8 : FIT;
    static constexpr int KV_BARS = NSLOT / 2 + 1;
    static constexpr int SIDE_OFF = KV_OFF + NSLOT * TILE_BYTES;
    static constexpr int SMEM = SIDE_OFF + SIDE + 1024;
    static_assert(NSLOT >= 4 && SMEM <= 227 * 1024, "shared memory");
    static constexpr uint32_t S_COL0 = 0, S_COL1 = 128, O_COL0 = 256, O_COL1 = 256 + D;
};

constexpr int kMaxBars = 5;          // KV_BARS at most (NSLOT 8)

// what sits behind the tiles in shared memory
struct Side {
    uint64_t qfull, qempty, vtail;
    uint64_t sfull[2], ofinal[2], drained;
    uint64_t kvfull[kMaxBars];
    uint64_t kvempty[8];
    uint32_t pready[2];              // softmax -> MMA: warps done, 4 per key tile
    uint32_t tmem;
    int abort;
    int last[2];
    int ended[2][2];                 // of the partial unit that began before, begins here: tile joined here
    int redo;                        // rows are marked in O
    alignas(16) uint32_t there[kMaxBars][4];     // which keys of the tile are in the cache
    alignas(16) uint32_t vbig[kMaxBars][4];      // 8 bit: largest V scale of 32 keys,
    alignas(16) uint32_t vleast[kMaxBars][4];    // and the smallest (scale_key)
    alignas(16) float kscale[kMaxBars][BKEY];
    alignas(16) float vscale[kMaxBars][BKEY];
    uint32_t rowat[3][BKEY];         // 8 bit: where a key's row is; three steps
    Walker walk[15];
};
static_assert(sizeof(Side) <= 8192, "side area");

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
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

// Piece c (16 codes) of rows r0, r0 + RP, ... widened to type T in a tile of
// two (dim 64: one) swizzled column boxes.
template <int T, int CT, int NP, int RP>
__device__ __forceinline__ void store_codes(const uint4 (&w)[NP], uint8_t* tile, int c, int r0) {
    uint8_t* dst = tile + (c >> 2) * kBoxBytes;
    // 16-byte piece p of a row sits at p ^ (row % 8); the odd half first where
    // that spreads the eight lanes of a row over all banks
    const int p = 2 * (c & 3), swap = c >> 2;
#pragma unroll
    for (int i = 0; i < NP; i++) {
        const int row = i * RP + r0;
        uint4 lo, hi;
        Code<T, CT>::widen(w[i].x, lo.x, lo.y);
        Code<T, CT>::widen(w[i].y, lo.z, lo.w);
        Code<T, CT>::widen(w[i].z, hi.x, hi.y);
        Code<T, CT>::widen(w[i].w, hi.z, hi.w);
        uint8_t* d = dst + row * 128;
        if (row < BKEY) {
            *reinterpret_cast<uint4*>(d + ((p + swap) ^ (row & 7)) * 16) = swap ? hi : lo;
            *reinterpret_cast<uint4*>(d + ((p + 1 - swap) ^ (row & 7)) * 16) = swap ? lo : hi;
        }
    }
}

struct ChunkShape {
    SchedShape sched;                // tokens: of both tiles
    int tile_tokens;                 // of one
    int box;                         // tokens per K/V box (16 bit)
};

// key tiles [s0, s0 + n0) and [s0, s0 + n1) of the two row tiles in a segment
struct Span {
    int s0, n0, n1, nmax;
};
__device__ __forceinline__ Span span_of(const PagedAttn& a, const ChunkShape& c,
                                        const Segment& g) {
    Span p;
    p.s0 = g.k0 / BKEY;
    const int s1 = (g.k1 + BKEY - 1) / BKEY;
    const int ni0 = min(g.ni, c.tile_tokens);
    const int e0 = tile_end(a, g.q, g.i0 + ni0);
    const int e1 = g.ni > c.tile_tokens ? tile_end(a, g.q, g.i0 + g.ni) : 0;
    p.n0 = max(0, min((e0 + BKEY - 1) / BKEY, s1) - p.s0);
    p.n1 = max(0, min((e1 + BKEY - 1) / BKEY, s1) - p.s0);
    p.nmax = max(p.n0, p.n1);
    return p;
}

// A warp's walker lives in shared memory: in registers it would cost the
// softmax threads twenty of them.
__device__ __forceinline__ bool next_segment(const PagedAttn& a, const ChunkShape& c, Walker* w,
                                             Segment& g) {
    __syncwarp();
    Walker t = *w;
    const bool more = t.next(a, c.sched, blockIdx.x, g);
    __syncwarp();
    if ((threadIdx.x & 31) == 0) *w = t;
    __syncwarp();
    return more;
}

// the part of tile t of a block's slot: (maximum, sum) of 128 rows, then O as
// [dim / 4][row][4]
template <int D>
__device__ __forceinline__ float* chunk_slot(const PagedAttn& a, int block, bool begins, int t) {
    return reinterpret_cast<float*>(a.ws + kCounterBytes) +
           ((2LL * block + (begins ? 1 : 0)) * 2 + t) * slot_floats(BQ, D);
}

// Row r over the members of a join: maximum (log2 units) and sum, then 32
// columns of O.
template <int D>
__device__ __forceinline__ void join_sums(const PagedAttn& a, const Segment& g, const Climb& c, int t,
                                          int r, float& m2, float& l) {
    float2 ml[kFan];
    m2 = -INFINITY;
#pragma unroll
    for (int u = 0; u < kFan; u++) {
        ml[u] = make_float2(-INFINITY, 0.f);
        if (u < c.members)
            ml[u] = __ldcg(reinterpret_cast<const float2*>(
                chunk_slot<D>(a, g.first + c.part(u), c.part(u) == 0, t) + 2 * r));
        m2 = max_nan(m2, ml[u].x);
    }
    const float b = m2 == -INFINITY ? 0.f : m2;
    l = 0.f;
#pragma unroll
    for (int u = 0; u < kFan; u++) l = fmaf(ml[u].y, ex2(ml[u].x - b), l);
}
template <int D>
__device__ __forceinline__ void join_columns(const PagedAttn& a, const Segment& g, const Climb& c,
                                             int t, int r, float m2, int c0, float (&v)[32]) {
    const float b = m2 == -INFINITY ? 0.f : m2;
#pragma unroll
    for (int i = 0; i < 32; i++) v[i] = 0.f;
#pragma unroll 1
    for (int u = 0; u < c.members; u++) {
        const float* ps = chunk_slot<D>(a, g.first + c.part(u), c.part(u) == 0, t);
        const float pm = __ldcg(ps + 2 * r);
        float4 x[8];
#pragma unroll
        for (int i = 0; i < 8; i++)
            x[i] = __ldcg(reinterpret_cast<const float4*>(ps + 2 * BQ + ((c0 / 4 + i) * BQ + r) * 4));
        if (pm == -INFINITY) continue;               // its O may never have been written
        const float f = ex2(pm - b);
#pragma unroll
        for (int i = 0; i < 8; i++) {
            v[4 * i] = fmaf(x[i].x, f, v[4 * i]);
            v[4 * i + 1] = fmaf(x[i].y, f, v[4 * i + 1]);
            v[4 * i + 2] = fmaf(x[i].z, f, v[4 * i + 2]);
            v[4 * i + 3] = fmaf(x[i].w, f, v[4 * i + 3]);
        }
    }
}

// The row's maximum, or NaN where its largest |O| is below `from`
// (paged_codes.cuh).
template <int D>
static __device__ __noinline__ float trusted_max(uint32_t o_addr, float m2, float from) {
    float mx = 0.f;
#pragma unroll 1
    for (int c0 = 0; c0 < D; c0 += 32) {
        uint32_t v[32];
        tmem_ld32(o_addr + c0, v);
        tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < 32; i++) mx = fmaxf(mx, fabsf(__uint_as_float(v[i])));
    }
    return m2 != -INFINITY && mx < from ? __uint_as_float(0x7fffffffu) : m2;
}

// by a thread, after it has stored row r
static __device__ __noinline__ void mark_row(const PagedAttn& a, const Segment& g, int r, float m2, int* redo) {
    const int end = (tile_end(a, g.q, g.i0 + g.ni) + BKEY - 1) / BKEY * BKEY;
    const RowPlace p = row_place(a, g, r);
    if (!redo_row(a, m2, keys_seen(a, g.q, p.token - g.q.q0), min(end, g.q.len))) return;
    *reinterpret_cast<uint16_t*>(a.o + (p.token * a.orow + p.head * a.oh) * 2) = kRedo;
    *redo = 1;
}

// Once a block's tiles are finished: its warps walk the piece again and compute
// the marked rows of the tiles that it stored.
static __device__ __noinline__ void redo_marked(const PagedAttn& a, const ChunkShape& c, const Side& sd) {
    const int warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    Walker w;
    w.start(a, c.sched, blockIdx.x);
    Segment g;
    while (w.next(a, c.sched, blockIdx.x, g)) {
        const int i0 = g.i0, ni = g.ni;
        for (int t = 0; t < 2; t++) {
            if (g.parts > 1 && !sd.ended[g.part == 0][t]) continue;
            g.i0 = i0 + t * c.tile_tokens;
            g.ni = max(0, min(ni - t * c.tile_tokens, c.tile_tokens));
            for (int r = warp; r < g.ni * a.group; r += warps) {
                const RowPlace p = row_place(a, g, r);
                const char* o = a.o + (p.token * a.orow + p.head * a.oh) * 2;
                if (*reinterpret_cast<const volatile uint16_t*>(o) == kRedo) repair_row(a, g, r);
            }
        }
    }
}

template <int D, int ELEM, int CT>
__global__ void __launch_bounds__(PCfg<D, (CT >= kI8)>::THREADS, 1)
paged_chunk_kernel(const __grid_constant__ CUtensorMap tmQ,
                   const __grid_constant__ CUtensorMap tmK,
                   const __grid_constant__ CUtensorMap tmV,
                   const __grid_constant__ PagedAttn a, const ChunkShape shape) {
    constexpr bool Q8 = CT >= kI8;
    using C = PCfg<D, Q8>;
    // P and V of an 8-bit cache in fp16, to which codes widen most cheaply and
    // in which weights keep three bits more than in bf16
    constexpr int PV = Q8 ? kF16 : ELEM;
    constexpr int NSLOT = C::NSLOT, KV_BARS = C::KV_BARS;
    constexpr uint32_t IDESC_QK = make_idesc(1, ELEM == kBF16 ? 1 : 0, 0, 0, BQ, BKEY);
    constexpr uint32_t IDESC_PV = make_idesc(1, PV == kBF16 ? 1 : 0, 0, 1, BQ, D);

    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>(
        (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    Side& sd = *reinterpret_cast<Side*>(smem + C::SIDE_OFF);
    volatile int* abort_flag = &sd.abort;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        mbar_init(&sd.qfull, 1);
        mbar_init(&sd.qempty, 1);
        mbar_init(&sd.vtail, 1);
        mbar_init(&sd.drained, 1);
        // 16 bit: one arrival for K and one for V, each with its byte count (a V
        // tile that had to be cleaned: once it is);
        // 8 bit: each loader warp, once for K and once for V
        for (int i = 0; i < KV_BARS; i++) mbar_init(&sd.kvfull[i], Q8 ? 2 * C::LOADERS : 2);
        for (int i = 0; i < NSLOT; i++) mbar_init(&sd.kvempty[i], 1);
        for (int i = 0; i < 2; i++) {
            mbar_init(&sd.sfull[i], 1);
            mbar_init(&sd.ofinal[i], 1);
            sd.pready[i] = 0;
        }
        sd.abort = 0;
        sd.redo = 0;
        for (int i = 0; i < 4; i++) sd.ended[i >> 1][i & 1] = 0;
        fence_mbar_init();
    }
    if (warp == C::MMA_WARP) {
        tmem_alloc(&sd.tmem, 512);
        tmem_relinquish();
    }
    {
        Walker w;
        w.start(a, shape.sched, blockIdx.x);
        if (lane == 0) sd.walk[warp] = w;
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = sd.tmem;

    if (warp >= 8 && warp < C::MMA_WARP) {
        // ---------------- loaders ----------------
        uint32_t step = 0, segs = 0, tails = 0;      // key tiles, segments, cleaned tails so far
        uint32_t asked = 0, asked_q = 0;             // key tiles and Q tiles on their way or here
        bool ok = true;
        Segment sg;
        // (8 bit: a warp that gave up goes on through the named barriers that
        // the others may be waiting at)
        while ((Q8 || ok) && next_segment(a, shape, &sd.walk[warp], sg)) {
            const Span sp = span_of(a, shape, sg);
            if (sp.nmax == 0) continue;
            if (warp == 8 && ok) {
                if (segs > 0) ok = mbar_wait(&sd.qempty, (segs - 1) & 1, abort_flag);
                ok = __all_sync(0xffffffffu, ok);
                asked_q += ok;
                if (ok && lane == 0) {
                    // the box clips nothing but the end of q, and counts its
                    // bytes there too
                    mbar_expect_tx(&sd.qfull, 2 * C::BOXES * shape.tile_tokens * a.group * 128);
                    for (int t = 0; t < 2; t++)
                        for (int x = 0; x < C::BOXES; x++)
                            tma_load_3d(smem + t * C::TILE_BYTES + x * kBoxBytes, &tmQ, &sd.qfull,
                                        x * 64, sg.head * a.group,
                                        sg.q.q0 + sg.i0 + t * shape.tile_tokens);
                }
            }
            segs++;
            const int* table = a.table + sg.s * a.tstride;
            if constexpr (!Q8) {
                const int box = shape.box, nbox = BKEY / box;
                const int bi = lane % nbox, bx = lane / nbox;    // box of tokens, of dims
                const bool mine = bx < C::BOXES;
                auto page_of = [&](int j) {          // of this lane's box in key tile j
                    const int key = (sp.s0 + j) * BKEY + bi * box;
                    return mine && j < sp.nmax && key < sg.q.len
                               ? __ldg(table + a.c.by_ps.div(key)) : -2;
                };
                int page = page_of(0);
                for (int j = 0; ok && j < sp.nmax; j++, step++) {
                    const int key0 = (sp.s0 + j) * BKEY, key = key0 + bi * box;
                    const int off = key - (int)a.c.by_ps.div(key) * a.c.ps;
                    const bool bad = page != -2 && (page < 0 || page >= a.c.pages);
                    if (bad) note_bad_index();
                    const int pc = page < 0 || page >= a.c.pages ? a.c.pages : page;
                    page = page_of(j + 1);
                    const unsigned gone = __ballot_sync(0xffffffffu, bad && bx == 0);
                    const int bar = step % KV_BARS;
                    uint64_t* full = &sd.kvfull[bar];
                    // a V tile in which the sequence ends inside a box
                    const int left = sg.q.len - key0;
                    const bool tail = left < BKEY && left % box != 0;
#pragma unroll
                    for (int kv = 0; kv < 2; kv++) {
                        const uint32_t item = 2 * step + kv, slot = item % NSLOT;
                        ok = mbar_wait(&sd.kvempty[slot], ((item / NSLOT) & 1) ^ 1u, abort_flag);
                        ok = __all_sync(0xffffffffu, ok);
                        if (!ok) {                   // (K's phase shall end with its bytes)
                            if (kv && lane == 0) mbar_arrive(full);
                            break;
                        }
                        asked = step + 1;
                        if (lane == 0) mbar_expect_tx(kv && tail ? &sd.vtail : full, C::TILE_BYTES);
                        if (kv == 0 && lane < 4) {
                            uint32_t w = 0xffffffffu;
                            if (gone)
                                for (int i = 0; i < 32; i++)
                                    if ((gone >> ((lane * 32 + i) / box)) & 1u) w &= ~(1u << i);
                            sd.there[bar][lane] = w;
                        }
                        __syncwarp();
                        uint8_t* dst = smem + C::KV_OFF + slot * C::TILE_BYTES;
                        if (mine)
                            tma_load_4d(dst + bx * kBoxBytes + bi * box * 128, kv ? &tmV : &tmK,
                                        kv && tail ? &sd.vtail : full, bx * 64, off, sg.head, pc);
                        if (kv && tail) {
                            ok = mbar_wait(&sd.vtail, tails & 1, abort_flag);
                            ok = __all_sync(0xffffffffu, ok);
                            if (!ok) {
                                if (lane == 0) {
                                    copy_wait(&sd.vtail, tails & 1);
                                    mbar_arrive(full);
                                }
                                break;
                            }
                            tails++;
                            const int end = (left + box - 1) / box * box;
                            constexpr int PIECES = 8 * C::BOXES;
                            for (int i = lane; i < (end - left) * PIECES; i += 32) {
                                const int row = left + i / PIECES, c = i % PIECES;
                                *reinterpret_cast<uint4*>(dst + (c >> 3) * kBoxBytes + row * 128 +
                                                          (c & 7) * 16) = make_uint4(0u, 0u, 0u, 0u);
                            }
                            fence_async_smem();
                            __syncwarp();
                            if (lane == 0) mbar_arrive(full);
                        }
                    }
                }
            } else {
                constexpr int CPR = D / 16;          // 16-byte pieces of a row
                constexpr int LT = 32 * C::LOADERS;  // loader threads
                constexpr int RP = LT / CPR;         // rows per pass of them
                constexpr int NP = (BKEY + RP - 1) / RP;
                constexpr uint32_t kNone = 0xffffffffu;
                const int lt = threadIdx.x - 256, lw = warp - 8;
                const int c = lt % CPR, r0 = lt / CPR;
                const char* kb = a.c.k + sg.head * a.c.head + c * 16;
                const char* vb = a.c.v + sg.head * a.c.head + c * 16;
                const float* ksb = a.c.ks + sg.head * a.c.shead;
                const float* vsb = a.c.vs + sg.head * a.c.shead;
                // Thread lt < 128 looks up key lt of a tile: the row's place for
                // all, its scales to keep.
                struct Look {
                    float ks, vs;
                    bool bad;
                };
                auto look_up = [&](int j, uint32_t buf) {
                    Look q{0.f, 0.f, false};
                    const int key = (sp.s0 + j) * BKEY + lt;
                    uint32_t at = kNone;
                    if (lt < BKEY && j < sp.nmax && key < sg.q.len) {
                        const unsigned n = a.c.by_ps.div(key);
                        const int off = key - (int)n * a.c.ps;
                        const int page = __ldg(table + n);
                        if (page >= 0 && page < a.c.pages) {
                            at = (uint32_t)((page * a.c.page + off * a.c.row) / 32);
                            q.ks = __ldg(ksb + page * a.c.spage + off);
                            q.vs = __ldg(vsb + page * a.c.spage + off);
                        } else {
                            q.bad = true;
                            note_bad_index();
                        }
                    }
                    if (lt < BKEY) sd.rowat[buf][lt] = at;
                    return q;
                };
                auto fetch = [&](uint4 (&w)[NP], const char* base, uint32_t buf) {
#pragma unroll
                    for (int i = 0; i < NP; i++) {
                        const int row = i * RP + r0;
                        const uint32_t at = row < BKEY ? sd.rowat[buf][row] : kNone;
                        w[i] = make_uint4(0u, 0u, 0u, 0u);
                        if (at != kNone) w[i] = __ldg(reinterpret_cast<const uint4*>(base + (size_t)at * 32));
                    }
                };
                auto slot_free = [&](uint32_t item) {
                    if (ok) ok = mbar_wait(&sd.kvempty[item % NSLOT], ((item / NSLOT) & 1) ^ 1u, abort_flag);
                    ok = __all_sync(0xffffffffu, ok);
                    return ok;
                };
                uint4 wk[NP], wv[NP];
                uint32_t buf = 0;                    // of step j
                auto after = [](uint32_t b, int n) { return (b + n) % 3; };
                named_bar_sync(3, LT);               // the last segment's places are read
                Look now = look_up(0, 0), next = look_up(1, 1);
                named_bar_sync(3, LT);
                fetch(wk, kb, 0);
                fetch(wv, vb, 0);
                for (int j = 0; j < sp.nmax; j++, step++, buf = after(buf, 1)) {
                    const int bar = step % KV_BARS;
                    if (slot_free(2 * step)) {
                        if (lw < BKEY / 32) {
                            sd.kscale[bar][lt] = now.ks * (a.scale * kLog2e);
                            sd.vscale[bar][lt] = now.vs;
                            const unsigned there = __ballot_sync(0xffffffffu, !now.bad);
                            const uint32_t big = __reduce_max_sync(0xffffffffu, scale_key(now.vs, 0u));
                            const uint32_t least =
                                __reduce_min_sync(0xffffffffu, scale_key(now.vs, 0xffffffffu));
                            if (lane == 0) {
                                sd.there[bar][lw] = there;
                                sd.vbig[bar][lw] = big;
                                sd.vleast[bar][lw] = least;
                            }
                        }
                        store_codes<ELEM, CT, NP, RP>(wk, smem + C::KV_OFF + (2 * step) % NSLOT * C::TILE_BYTES, c, r0);
                        fence_async_smem();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&sd.kvfull[bar]);
                    }
                    // the places of step j + 1 were written a step ago, those of
                    // j + 2 go where those of j - 1 were
                    named_bar_sync(3, LT);
                    fetch(wk, kb, after(buf, 1));
                    now = next;
                    next = look_up(j + 2, after(buf, 2));
                    if (slot_free(2 * step + 1)) {
                        store_codes<PV, CT, NP, RP>(wv, smem + C::KV_OFF + (2 * step + 1) % NSLOT * C::TILE_BYTES, c, r0);
                        fence_async_smem();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&sd.kvfull[bar]);
                    }
                    fetch(wv, vb, after(buf, 1));
                }
            }
        }
        // no commit may still be on its way to this block's barriers when it
        // exits: wait for the last release of every slot and of Q
        if (warp == 8 && lane == 0 && ok && segs > 0) {
            const uint32_t items = 2 * step;
            for (uint32_t i = items > NSLOT ? items - NSLOT : 0; ok && i < items; i++)
                ok = mbar_wait(&sd.kvempty[i % NSLOT], (i / NSLOT) & 1, abort_flag);
            ok = ok && mbar_wait(&sd.qempty, (segs - 1) & 1, abort_flag);
        }
        // gave up: not before the copies have landed
        if (warp == 8 && lane == 0 && !ok) {
            if (asked_q > 0) copy_wait(&sd.qfull, (asked_q - 1) & 1);
            for (uint32_t j = asked > KV_BARS ? asked - KV_BARS : 0; j < asked; j++)
                copy_wait(&sd.kvfull[j % KV_BARS], (j / KV_BARS) & 1);
        }
    } else if (warp == C::MMA_WARP) {
        // ---------------- MMA issuer ----------------
        const uint32_t sq_base = smem_u32(smem);
        const uint32_t kv_base = smem_u32(smem + C::KV_OFF);
        uint32_t step = 0, segs = 0, done0 = 0, done1 = 0;
        auto kv_wait = [&](uint32_t j) {
            return mbar_wait(&sd.kvfull[j % KV_BARS], (j / KV_BARS) & 1, abort_flag);
        };
        auto slot_addr = [&](uint32_t item) { return kv_base + (item % NSLOT) * C::TILE_BYTES; };
        auto issue_qk = [&](int t, uint32_t j) {
            const uint64_t kd = sw128_desc(slot_addr(2 * j), 16, 1024);
            const uint64_t qd = sw128_desc(sq_base + t * C::TILE_BYTES, 16, 1024);
            const uint32_t s_tm = tmem_base + (t ? C::S_COL1 : C::S_COL0);
#pragma unroll
            for (int ks = 0; ks < D / 16; ks++) {
                const uint64_t off = ((ks >> 2) * kBoxBytes + (ks & 3) * 32) >> 4;
                mma_f16_ss(s_tm, qd + off, kd + off, IDESC_QK, ks > 0 ? 1u : 0u);
            }
            mma_commit(&sd.sfull[t]);
        };
        auto issue_pv = [&](int t, uint32_t j, bool fresh) {
            const uint64_t vd = sw128_desc(slot_addr(2 * j + 1), kBoxBytes, 1024);
            const uint32_t o_tm = tmem_base + (t ? C::O_COL1 : C::O_COL0);
            const uint32_t p_tm = tmem_base + (t ? C::S_COL1 : C::S_COL0);
#pragma unroll
            for (int ks = 0; ks < BKEY / 16; ks++)
                mma_f16_ts(o_tm, p_tm + ks * 8, vd + ((ks * 16 * 128) >> 4), IDESC_PV,
                           (!fresh || ks > 0) ? 1u : 0u);
        };
        bool ok = true;
        Segment sg;
        while (ok && next_segment(a, shape, &sd.walk[warp], sg)) {
            const Span sp = span_of(a, shape, sg);
            if (sp.nmax == 0) continue;
            if (lane == 0) {
                ok = mbar_wait(&sd.qfull, segs & 1, abort_flag) && kv_wait(step);
                if (ok) {
                    tc_fence_after();
                    if (sp.n0 > 0) issue_qk(0, step);
                    if (sp.n1 > 0) issue_qk(1, step);
                    mma_commit(&sd.kvempty[(2 * step) % NSLOT]);
                    if (sp.nmax == 1) mma_commit(&sd.qempty);
                }
                for (int j = 0; ok && j < sp.nmax; j++) {
                    bool have_next_k = false;
#pragma unroll
                    for (int t = 0; t < 2; t++) {
                        const int ntt = t ? sp.n1 : sp.n0;
                        if (j >= ntt) continue;
                        const bool last_reader = t == 1 || j >= sp.n1;
                        uint32_t& done = t ? done1 : done0;
                        if (!flag_wait(&sd.pready[t], 4u * ++done, abort_flag)) { ok = false; break; }
                        tc_fence_after();
                        issue_pv(t, step + j, j == 0);
                        if (last_reader) mma_commit(&sd.kvempty[(2 * (step + j) + 1) % NSLOT]);
                        if (j + 1 == ntt) mma_commit(&sd.ofinal[t]);
                        if (j + 1 < ntt) {
                            if (!have_next_k) {
                                if (!kv_wait(step + j + 1)) { ok = false; break; }
                                tc_fence_after();
                                have_next_k = true;
                            }
                            issue_qk(t, step + j + 1);
                            if (t == 1 || j + 1 >= sp.n1) {
                                mma_commit(&sd.kvempty[(2 * (step + j) + 2) % NSLOT]);
                                if (j + 2 == sp.nmax) mma_commit(&sd.qempty);
                            }
                        }
                    }
                }
            }
            ok = __shfl_sync(0xffffffffu, ok, 0);
            step += sp.nmax;
            segs++;
        }
        // whatever the other roles have waited for: no product and no commit
        // outlives the block
        if (lane == 0) {
            mma_commit(&sd.drained);
            copy_wait(&sd.drained, 0);
        }
    } else {
        // ---------------- softmax and epilogue (warps 0-7) ----------------
        const int t = warp >> 2, quarter = warp & 3;
        const int r = quarter * 32 + lane;
        const uint32_t lane_off = (uint32_t)(quarter * 32) << 16;
        const uint32_t s_addr = tmem_base + lane_off + (t ? C::S_COL1 : C::S_COL0);
        const uint32_t o_addr = tmem_base + lane_off + (t ? C::O_COL1 : C::O_COL0);
        const float c = Q8 ? 1.f : a.scale * kLog2e;     // 8 bit: in the K scales already
        constexpr float kLazyLog2 = Q8 ? kLazy8 : 8.f;   // weights reach 2^this
        uint32_t step = 0, tiles = 0, finals = 0;
        bool alive = true;
        Segment sg;
        while (next_segment(a, shape, &sd.walk[warp], sg)) {
            const Span sp = span_of(a, shape, sg);
            const int tnt = t ? sp.n1 : sp.n0;
            sg.i0 += t * shape.tile_tokens;          // from here on: this tile's rows
            sg.ni = max(0, min(sg.ni - t * shape.tile_tokens, shape.tile_tokens));
            const bool row_ok = r < sg.ni * a.group;
            const int lim = row_ok ? tile_end(a, sg.q, sg.i0 + r / a.group + 1) : 0;
            const int lim_all = tile_end(a, sg.q, sg.i0 + 1);
            float m_used = -INFINITY, l = 0.f, lpow = 0.f;
            float vmost = 0.f, vpow = 1.f;           // 8 bit: see v_power
            uint32_t vleast = 0xffffffffu;
            if constexpr (!Q8) {
                for (int j = 0; j < tnt && alive; j++, tiles++) {
                    alive = __all_sync(0xffffffffu, mbar_wait(&sd.sfull[t], tiles & 1, abort_flag));
                    if (!alive) break;
                    tc_fence_after();
                    float s[BKEY];
#pragma unroll
                    for (int c0 = 0; c0 < BKEY; c0 += 32)
                        tmem_ld32(s_addr + c0, *reinterpret_cast<uint32_t(*)[32]>(&s[c0]));
                    tmem_wait_ld();
                    const int key0 = (sp.s0 + j) * BKEY;
                    const uint4 th = *reinterpret_cast<const uint4*>(sd.there[(step + j) % KV_BARS]);
                    if (key0 + BKEY > lim_all || (th.x & th.y & th.z & th.w) != 0xffffffffu) {
                        const uint32_t tw[4] = {th.x, th.y, th.z, th.w};
#pragma unroll
                        for (int i = 0; i < BKEY; i++)
                            if (key0 + i >= lim || !((tw[i >> 5] >> (i & 31)) & 1u)) s[i] = -INFINITY;
                    }
                    float mx8[8];
#pragma unroll
                    for (int i = 0; i < 8; i++) mx8[i] = s[i];
#pragma unroll
                    for (int i = 8; i < BKEY; i++) mx8[i & 7] = fmaxf(mx8[i & 7], s[i]);
                    const float mx = fmaxf(fmaxf(fmaxf(mx8[0], mx8[1]), fmaxf(mx8[2], mx8[3])),
                                           fmaxf(fmaxf(mx8[4], mx8[5]), fmaxf(mx8[6], mx8[7])));
                    const float m_new = fmaxf(m_used, mx);
                    if (j == 0) {
                        m_used = m_new;
                    } else {
                        const bool grow = m_new != -INFINITY &&
                                          (m_used == -INFINITY || (m_new - m_used) * c > kLazyLog2);
                        if (__any_sync(0xffffffffu, grow)) {
                            float alpha = 1.f;
                            if (grow) {
                                alpha = ex2((m_used - m_new) * c);
                                l *= alpha;
                                m_used = m_new;
                            }
#pragma unroll 1
                            for (int c0 = 0; c0 < D; c0 += 16) {
                                uint32_t o[16];
                                tmem_ld16(o_addr + c0, o);
                                tmem_wait_ld();
#pragma unroll
                                for (int i = 0; i < 16; i++)
                                    o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
                                tmem_st16(o_addr + c0, o);
                            }
                        }
                    }
                    const float mc = m_used == -INFINITY ? 0.f : m_used * c;
                    float sum8[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int c0 = 0; c0 < BKEY / 2; c0 += 16) {
                        uint32_t pk[16];
#pragma unroll
                        for (int i = 0; i < 16; i++) {
                            const int k = 2 * (c0 + i);
                            const float p0 = ex2(fmaf(s[k], c, -mc)), p1 = ex2(fmaf(s[k + 1], c, -mc));
                            sum8[i & 7] += p0 + p1;
                            pk[i] = pack2<ELEM>(p0, p1);
                        }
                        tmem_st16(s_addr + c0, pk);
                    }
                    tmem_wait_st();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) flag_add_release(&sd.pready[t]);
                    l += ((sum8[0] + sum8[1]) + (sum8[2] + sum8[3])) +
                         ((sum8[4] + sum8[5]) + (sum8[6] + sum8[7]));
                }
            } else {
                // Every key has a factor of its own here.  With a whole row in a
                // thread each thread would read all of them, and shared memory
                // is what the tensor core lives on; as a matrix fragment,
                // thread (g, t4) has 32 keys of the four rows g + 8k and reads the
                // factors of those 32.
                const int g = lane >> 2, t4 = lane & 3;
                auto turn = [](auto& x, auto& y) {
                    const auto z = x;
                    x = y;
                    y = z;
                };
                float m4[4], l4[4], b4[4];          // of rows g + 8k
                int lim4[4];
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    m4[k] = -INFINITY;
                    l4[k] = b4[k] = 0.f;
                    lim4[k] = __shfl_sync(0xffffffffu, lim, g + 8 * k);
                }
                for (int j = 0; j < tnt && alive; j++, tiles++) {
                    alive = __all_sync(0xffffffffu, mbar_wait(&sd.sfull[t], tiles & 1, abort_flag));
                    if (!alive) break;
                    tc_fence_after();
                    const int bar = (step + j) % KV_BARS;
                    const float2* ks = reinterpret_cast<const float2*>(sd.kscale[bar]) + t4;
                    const float2* vs = reinterpret_cast<const float2*>(sd.vscale[bar]) + t4;
                    const int key0 = (sp.s0 + j) * BKEY;
                    const uint4 th = *reinterpret_cast<const uint4*>(sd.there[bar]);
                    const uint32_t tw[4] = {th.x, th.y, th.z, th.w};
                    const bool edge = key0 + BKEY > lim_all ||
                                      (th.x & th.y & th.z & th.w) != 0xffffffffu;
                    float vfix = 1.f;
                    {
                        const uint4 b = *reinterpret_cast<const uint4*>(sd.vbig[bar]);
                        vfix = v_power(__uint_as_float(max(max(b.x, b.y), max(b.z, b.w))), vmost, vpow);
                        if (vfix != 1.f) lpow = exponent_of(vpow);
                        const uint4 s = *reinterpret_cast<const uint4*>(sd.vleast[bar]);
                        vleast = min(min(vleast, min(s.x, s.y)), min(s.z, s.w));
                    }
                    // Lanes 0-15, then 16-31, by one piece of code (unrolled
                    // twice, it and the loaders' would not fit the instruction
                    // cache together): the rows' state is turned round after
                    // each.
#pragma unroll 1
                    for (int h = 0; h < 2; h++) {
                        const uint32_t half = (uint32_t)h << 20;
                        float x[64];                 // scores in log2 units
                        tmem_ld_frag128(s_addr + half, reinterpret_cast<uint32_t(&)[64]>(x));
                        tmem_wait_ld();
#pragma unroll
                        for (int i = 0; i < 16; i++) {
                            const float2 f = ks[4 * i];
                            x[4 * i] *= f.x;
                            x[4 * i + 1] *= f.y;
                            x[4 * i + 2] *= f.x;
                            x[4 * i + 3] *= f.y;
                        }
                        if (edge) {
#pragma unroll
                            for (int i = 0; i < 16; i++)
#pragma unroll
                                for (int e = 0; e < 2; e++) {
                                    const int k = 8 * i + 2 * t4 + e;
                                    const bool gone = !((tw[i >> 2] >> (k & 31)) & 1u);
                                    if (gone || key0 + k >= lim4[0]) x[4 * i + e] = -INFINITY;
                                    if (gone || key0 + k >= lim4[1]) x[4 * i + 2 + e] = -INFINITY;
                                }
                        }
                        bool grow = vfix != 1.f;
                        float alpha[2];
#pragma unroll
                        for (int r2 = 0; r2 < 2; r2++) {
                            const int o = 2 * r2;
                            float& mk = m4[r2];
                            float mx[4];
#pragma unroll
                            for (int i = 0; i < 4; i++) mx[i] = fmaxf(x[4 * i + o], x[4 * i + o + 1]);
#pragma unroll
                            for (int i = 4; i < 16; i++)
                                mx[i & 3] = fmaxf(mx[i & 3], fmaxf(x[4 * i + o], x[4 * i + o + 1]));
                            float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
                            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                            alpha[r2] = vfix;
                            if (top > mk + kLazyLog2) {      // also from -inf
                                alpha[r2] *= ex2(mk - top);
                                mk = top;
                                grow = true;
                            }
                        }
                        if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
                            for (int r2 = 0; r2 < 2; r2++) {
                                // the power of two rides in the exponent, on O and l alike
                                b4[r2] = (m4[r2] == -INFINITY ? 0.f : m4[r2]) - lpow;
                                l4[r2] *= alpha[r2];
                            }
                            if (j > 0) {
#pragma unroll 1
                                for (int c0 = 0; c0 < D; c0 += 32) {
                                    uint32_t o[16];
                                    tmem_ld_frag32(o_addr + half + c0, o);
                                    tmem_wait_ld();
#pragma unroll
                                    for (int i = 0; i < 16; i++)
                                        o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha[(i >> 1) & 1]);
                                    tmem_st_frag32(o_addr + half + c0, o);
                                }
                            }
                        }
#pragma unroll
                        for (int i0 = 0; i0 < 16; i0 += 8) {
                            uint32_t pk[16];
#pragma unroll
                            for (int i = 0; i < 8; i++) {
                                const float2 f = vs[4 * (i0 + i)];
#pragma unroll
                                for (int r2 = 0; r2 < 2; r2++) {
                                    const int o = 4 * (i0 + i) + 2 * r2;
                                    const float p0 = ex2(x[o] - b4[r2]);
                                    const float p1 = ex2(x[o + 1] - b4[r2]);
                                    l4[r2] += p0 + p1;
                                    pk[2 * i + r2] = pack2<PV>(p0 * f.x, p1 * f.y);
                                }
                            }
                            tmem_st_frag32p(s_addr + half + 4 * i0, pk);
                        }
#pragma unroll
                        for (int k = 0; k < 2; k++) {
                            turn(m4[k], m4[k + 2]);
                            turn(l4[k], l4[k + 2]);
                            turn(b4[k], b4[k + 2]);
                            turn(lim4[k], lim4[k + 2]);
                        }
                    }
                    tmem_wait_st();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) flag_add_release(&sd.pready[t]);
                }
                // back to a row for each thread: row `lane` of the warp's 32
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    l4[k] += __shfl_xor_sync(0xffffffffu, l4[k], 1);
                    l4[k] += __shfl_xor_sync(0xffffffffu, l4[k], 2);
                    const float mk = __shfl_sync(0xffffffffu, m4[k], (lane & 7) * 4);
                    const float lk = __shfl_sync(0xffffffffu, l4[k], (lane & 7) * 4);
                    if (k == lane >> 3) {
                        m_used = mk;
                        l = lk;
                    }
                }
            }
            step += sp.nmax;

            // ---- epilogue
            bool have_o = tnt > 0;
            if (have_o && alive) {
                if (!mbar_wait(&sd.ofinal[t], finals & 1, abort_flag)) alive = false;
                else tc_fence_after();
            }
            if (tnt > 0) finals++;
            alive = __all_sync(0xffffffffu, alive);
            have_o = have_o && alive;
            // log2 units; -inf: no key
            float m2 = m_used == -INFINITY ? -INFINITY : m_used * c - lpow;
            if constexpr (Q8) {
                if (have_o && wide_scales(vleast, vmost, vpow))
                    m2 = trusted_max<D>(o_addr, m2, trusted_from<ELEM, CT>(tnt * BKEY, vmost, vpow));
            }
            const bool split = sg.parts > 1;
            bool final = !split;
            Climb up(sg);
            if (split) {
                float* ps = chunk_slot<D>(a, blockIdx.x, sg.part == 0, t);
                *reinterpret_cast<float2*>(ps + 2 * r) = make_float2(m2, l);
                if (have_o) {
#pragma unroll 1
                    for (int c0 = 0; c0 < D; c0 += 32) {
                        uint32_t v[32];
                        tmem_ld32(o_addr + c0, v);
                        tmem_wait_ld();
#pragma unroll
                        for (int i = 0; i < 8; i++)
                            *reinterpret_cast<float4*>(ps + 2 * BQ + ((c0 / 4 + i) * BQ + r) * 4) =
                                make_float4(__uint_as_float(v[4 * i]), __uint_as_float(v[4 * i + 1]),
                                            __uint_as_float(v[4 * i + 2]), __uint_as_float(v[4 * i + 3]));
                    }
                }
#pragma unroll 1
                for (;; up.up()) {
                    __threadfence();
                    named_bar_sync(1 + t, 128);
                    if (r == 0) sd.last[t] = up.arrive(a, sg, t);
                    named_bar_sync(1 + t, 128);
                    const bool last = *static_cast<volatile int*>(&sd.last[t]);
                    named_bar_sync(1 + t, 128);      // (before anyone writes it again)
                    if (!last) break;
                    __threadfence();
                    join_sums<D>(a, sg, up, t, r, m2, l);
                    if (up.top()) {
                        final = true;
                        break;
                    }
                    if (up.members == 1) continue;
                    // into the first member's slot, each thread its own row
                    float* to = chunk_slot<D>(a, sg.first + up.part(0), up.part(0) == 0, t);
#pragma unroll 1
                    for (int c0 = 0; c0 < D; c0 += 32) {
                        float v[32];
                        join_columns<D>(a, sg, up, t, r, m2, c0, v);
#pragma unroll
                        for (int i = 0; i < 8; i++)
                            *reinterpret_cast<float4*>(to + 2 * BQ + ((c0 / 4 + i) * BQ + r) * 4) =
                                make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
                    }
                    *reinterpret_cast<float2*>(to + 2 * r) = make_float2(m2, l);
                }
            }
            if (final && alive) {
                const float inv = l == 0.f ? 0.f : 1.f / l;
                const RowPlace pl = row_place(a, sg, row_ok ? r : 0);
                char* orow = a.o + (pl.token * a.orow + pl.head * a.oh) * 2;
                float z = 0.f;
#pragma unroll 1
                for (int c0 = 0; c0 < D; c0 += 32) {
                    float v[32];
                    if (!split) {
                        if (have_o) {
                            tmem_ld32(o_addr + c0, *reinterpret_cast<uint32_t(*)[32]>(&v[0]));
                            tmem_wait_ld();
                        } else {
#pragma unroll
                            for (int i = 0; i < 32; i++) v[i] = 0.f;
                        }
                    } else {
                        join_columns<D>(a, sg, up, t, r, m2, c0, v);
                    }
                    if (row_ok) {
                        uint32_t w[16];
#pragma unroll
                        for (int i = 0; i < 16; i++) {
                            const float x = v[2 * i] * inv, y = v[2 * i + 1] * inv;
                            z = fmaf(x, 0.f, fmaf(y, 0.f, z));   // NaN once one is not finite
                            w[i] = pack2<ELEM>(x, y);
                        }
                        uint4* dst = reinterpret_cast<uint4*>(orow + c0 * 2);
#pragma unroll
                        for (int i = 0; i < 4; i++)
                            dst[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
                    }
                }
                if (row_ok && a.lse) a.lse[pl.head * a.lh + pl.token] = lse_of(m2, l);
                if (row_ok && spoilt(m2, l, z)) mark_row(a, sg, r, m2, &sd.redo);
                if (split && r == 0) sd.ended[sg.part == 0][t] = 1;
            }
            __syncwarp();
        }
    }

    tc_fence_before();
    __syncthreads();
    if (warp == C::MMA_WARP) {
        tc_fence_after();
        tmem_dealloc(tmem_base, 512);
    }
    if (sd.redo && !sd.abort) redo_marked(a, shape, sd);
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

// 16-bit tensor of `rank` dimensions, strides in elements (of dimensions 1
// and up; one that is never stepped over may be anything)
bool tensor_map(CUtensorMap* tm, int elem, const void* base, int rank, const cuuint64_t* dims,
                const long long* strides, const cuuint32_t* box) {
    EncodeFn enc = encode_fn();
    if (!enc) return false;
    cuuint64_t st[4];
    const cuuint32_t ones[5] = {1, 1, 1, 1, 1};
    for (int i = 1; i < rank; i++) st[i - 1] = dims[i] > 1 ? (cuuint64_t)strides[i] * 2 : 16;
    return enc(tm, elem == kBF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
               (cuuint32_t)rank, const_cast<void*>(base), dims, st, box, ones,
               CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
               CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int D, int ELEM, int CT>
int launch(const PagedAttn& a, cudaStream_t s) {
    using C = PCfg<D, (CT >= kI8)>;
    ChunkShape shape;
    shape.tile_tokens = BQ / a.group;
    shape.sched = sched_shape(a, 2 * shape.tile_tokens, BKEY, 2, chunk_blocks());
    shape.box = 8;
    while (shape.box < BKEY && a.c.ps % (2 * shape.box) == 0) shape.box *= 2;
    CUtensorMap tq, tk, tv;
    {
        const cuuint64_t dims[3] = {(cuuint64_t)D, (cuuint64_t)a.heads, (cuuint64_t)a.total_q};
        const long long st[3] = {0, a.qh, a.qr};
        const cuuint32_t box[3] = {64, (cuuint32_t)a.group, (cuuint32_t)shape.tile_tokens};
        if (!tensor_map(&tq, ELEM, a.q, 3, dims, st, box)) return 1;
    }
    tk = tv = tq;
    if (CT < kI8) {
        const cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)a.c.ps, (cuuint64_t)a.c.heads,
                                    (cuuint64_t)a.c.pages};
        const long long st[4] = {0, a.c.row, a.c.head, a.c.page};
        const cuuint32_t box[4] = {64, (cuuint32_t)shape.box, 1, 1};
        if (!tensor_map(&tk, ELEM, a.c.k, 4, dims, st, box)) return 1;
        if (!tensor_map(&tv, ELEM, a.c.v, 4, dims, st, box)) return 1;
    }
    auto kern = paged_chunk_kernel<D, ELEM, CT>;
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
    kern<<<chunk_blocks(), C::THREADS, C::SMEM, s>>>(tq, tk, tv, a, shape);
    const cudaError_t e = cudaGetLastError();
    if (e == cudaSuccess) note_launch();
    return e == cudaSuccess ? 0 : (int)e;
}

template <int ELEM, int CT>
int launch_dim(const PagedAttn& a, cudaStream_t s) {
    return a.c.dim == 128 ? launch<128, ELEM, CT>(a, s) : launch<64, ELEM, CT>(a, s);
}

}  // namespace

int chunk_blocks() { return std::min(num_sms(), kMaxPieces); }

size_t paged_chunk_workspace(const PagedAttn& a) {
    return kCounterBytes + 4ull * chunk_blocks() * slot_floats(BQ, a.c.dim) * sizeof(float);
}

int paged_chunk(const PagedAttn& a, cudaStream_t s) {
    if (a.elem == kBF16)
        return a.type == kI8 ? launch_dim<kBF16, kI8>(a, s)
             : a.type == kE4M3 ? launch_dim<kBF16, kE4M3>(a, s)
                               : launch_dim<kBF16, kBF16>(a, s);
    return a.type == kI8 ? launch_dim<kF16, kI8>(a, s)
         : a.type == kE4M3 ? launch_dim<kF16, kE4M3>(a, s)
                           : launch_dim<kF16, kF16>(a, s);
}

int paged_chunk_set_wait_limit(unsigned long long ns) { return set_unit_wait_limit(ns); }

int paged_chunk_error(bool clear) {
    int v = 0;
    cudaMemcpyFromSymbol(&v, g_dev_error, sizeof(int));
    if (clear && v) {
        int z = 0;
        cudaMemcpyToSymbol(g_dev_error, &z, sizeof(int));
    }
    return v;
}

}  // namespace zl
