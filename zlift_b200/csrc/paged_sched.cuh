// paged_sched.cuh -- how a paged-attention launch is split over its blocks.
//
// A unit is a tile of query rows of one sequence and KV head; its steps are
// the key tiles that its rows see (one at least, so that rows which see
// nothing are written too).  All steps of all units, in the order sequence,
// head, tile, key, form one line, which is cut into equal pieces, one for
// each worker (a block, or a warp where warps work alone).  Lengths live on
// the device, so every worker finds its piece from them: nothing is planned
// on the host, a ragged batch is as even as a regular one, and a graph
// replays with new lengths.  Positions are 32 bits: where the work that the
// arrays can hold would pass that, a step is several key tiles (sched_shape).
//
// A unit that spans several pieces is joined by whichever worker finishes
// last: each leaves its unnormalised O with the maximum and the sum of every
// row in the workspace and counts itself; the last one sums the parts in key
// order (so the result does not depend on who came last) and puts the counter
// back to zero for the next call.  A piece has at most two partial units: one
// that began before it (slot 0, also where it ends after it) and one that
// begins in it (slot 1).
#pragma once
#include "paged.h"

namespace zl {

struct SchedShape {
    int tokens;          // query tokens per tile
    int step;            // keys per step
    int least;           // steps per piece, at least
    int pieces;
};

// Of tiles of `tokens` query tokens and `keys` keys.  A long chunk in tiles of
// single tokens is 2^32 key tiles soon (131072 tokens, 16 keys, 8 heads), so
// the step is doubled until the longest line that total_q, batch and the page
// table's width allow is below 2^31 steps.
inline SchedShape sched_shape(const PagedAttn& a, int tokens, int keys, int least, int pieces) {
    SchedShape h{tokens, keys, least, pieces};
    const double tiles = ((double)a.total_q / tokens + a.batch) * a.c.heads;
    const double room = (double)a.tpages * a.c.ps;
    while (h.step < (1 << 29) && tiles * (room / h.step + 2) >= 2147483648.0) {
        h.step *= 2;
        h.least = (h.least + 1) / 2;
    }
    return h;
}

// a unit, or what of it falls into one piece
struct Segment {
    int s, head;         // sequence, KV head
    SeqInfo q;
    int i0, ni;          // the tile's first token in the chunk, and tokens
    int k0, k1;          // its keys in this piece (k1 is not rounded up)
    int parts, part;     // pieces that share the unit; this one's place
    int first;           // the piece in which the unit begins
};

__device__ __forceinline__ int tile_end(const PagedAttn& a, const SeqInfo& q, int i1) {
    return a.causal ? max(0, min(q.len, q.len - q.n + i1)) : q.len;
}

__device__ __forceinline__ int tile_steps(const PagedAttn& a, const SchedShape& h,
                                          const SeqInfo& q, int tile) {
    const int e = tile_end(a, q, min(q.n, (tile + 1) * h.tokens));
    return max(1, (int)((unsigned)(e + h.step - 1) / (unsigned)h.step));
}

// steps of all tiles of one head of a sequence
__device__ __forceinline__ unsigned head_steps(const PagedAttn& a, const SchedShape& h,
                                               const SeqInfo& q) {
    if (q.n <= h.tokens) return q.n ? tile_steps(a, h, q, 0) : 0;
    const int tiles = (q.n + h.tokens - 1) / h.tokens;
    if (!a.causal) return (unsigned)tiles * tile_steps(a, h, q, 0);
    unsigned sum = 0;
    for (int t = 0; t < tiles; t++) sum += tile_steps(a, h, q, t);
    return sum;
}

// inclusive sum over the lanes
__device__ __forceinline__ unsigned lane_sums(unsigned v) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned x = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += x;
    }
    return v;
}

// Walks a piece.  Every warp keeps one of its own (the search runs
// across the lanes; all lanes hold the same state afterwards).
struct Walker {
    unsigned pos, end, begin;            // on the line; begin: of the unit
    unsigned per;                        // steps of a piece
    SeqInfo q;
    int s, head, tile;
    unsigned steps;

    __device__ __forceinline__ void enter(const PagedAttn& a, const SchedShape& h) {
        steps = tile_steps(a, h, q, tile);
    }

    __device__ void start(const PagedAttn& a, const SchedShape& h, int piece) {
        const int lane = threadIdx.x & 31;
        // lane l sums sequences [l * each, (l + 1) * each)
        const int each = (a.batch + 31) / 32;
        unsigned mine = 0;
        for (int i = 0; i < each; i++) {
            const int b = lane * each + i;
            if (b < a.batch) mine += head_steps(a, h, seq_info(a, b));
        }
        mine *= a.c.heads;
        const unsigned sum = lane_sums(mine);
        const unsigned total = __shfl_sync(0xffffffffu, sum, 31);
        per = max((total + h.pieces - 1) / h.pieces, (unsigned)h.least);
        pos = min((unsigned long long)total, (unsigned long long)piece * per);
        end = min((unsigned long long)total, (unsigned long long)pos + per);
        if (pos >= end) return;
        // the lane whose sequences hold pos, then the sequence
        int l = __ffs(__ballot_sync(0xffffffffu, sum > pos)) - 1;
        unsigned base = __shfl_sync(0xffffffffu, sum - mine, l);
        s = l * each;
        if (each > 1) {
            for (int b0 = l * each; b0 < (l + 1) * each; b0 += 32) {
                const int b = b0 + lane;
                const unsigned v = b < min(a.batch, (l + 1) * each)
                                       ? head_steps(a, h, seq_info(a, b)) * a.c.heads : 0;
                const unsigned x = lane_sums(v);
                const unsigned past = __ballot_sync(0xffffffffu, base + x > pos);
                if (past) {
                    const int f = __ffs(past) - 1;
                    s = b0 + f;
                    base += __shfl_sync(0xffffffffu, x - v, f);
                    break;
                }
                base += __shfl_sync(0xffffffffu, x, 31);
            }
        }
        q = seq_info(a, s);
        const unsigned hs = max(1u, head_steps(a, h, q));
        head = min((int)((pos - base) / hs), a.c.heads - 1);
        begin = base + head * hs;
        tile = 0;
        enter(a, h);
        while (pos - begin >= steps && (tile + 1) * h.tokens < q.n) {
            begin += steps;
            tile++;
            enter(a, h);
        }
    }

    // the next piece of a unit; false at the end of the line's piece
    __device__ __forceinline__ bool next(const PagedAttn& a, const SchedShape& h, int piece,
                                         Segment& g) {
        if (pos >= end) return false;
        g.s = s;
        g.head = head;
        g.q = q;
        g.i0 = tile * h.tokens;
        g.ni = min(h.tokens, q.n - g.i0);
        const unsigned st0 = pos - begin;
        const unsigned st1 = min(steps, end - begin);
        const int e = tile_end(a, q, g.i0 + g.ni);
        g.k0 = (int)min((unsigned)e, st0 * h.step);
        g.k1 = (int)min((unsigned)e, st1 * h.step);
        if (st0 == 0 && st1 == steps) {
            g.parts = 1;
            g.part = 0;
            g.first = piece;
        } else {
            g.first = (int)(begin / per);
            g.parts = (int)((begin + steps - 1) / per) - g.first + 1;
            g.part = piece - g.first;
        }
        pos = begin + st1;
        if (st1 == steps && pos < end) {
            begin += steps;
            if (++tile * h.tokens >= q.n) {
                tile = 0;
                if (++head == a.c.heads) {
                    head = 0;
                    do q = seq_info(a, ++s);
                    while (q.n == 0 && s + 1 < a.batch);
                }
            }
            enter(a, h);
        }
        return true;
    }
};

// ---- the workspace --------------------------------------------------------------

constexpr int kMaxPieces = 2048;
constexpr int kFan = 8;                          // parts joined at once
constexpr int kLevels = 4;                       // kFan ^ kLevels >= kMaxPieces
constexpr size_t kCounterBytes = kLevels * 2 * kMaxPieces * sizeof(int);

// floats of one slot: (maximum, sum) of every row, then O
__host__ __device__ constexpr long long slot_floats(int rows, int dim) {
    return (long long)rows * (2 + dim);
}

__device__ __forceinline__ float* part_slot(const PagedAttn& a, int rows, int piece, bool begins) {
    return reinterpret_cast<float*>(a.ws + kCounterBytes) +
           (2LL * piece + (begins ? 1 : 0)) * slot_floats(rows, a.c.dim);
}

// Joining many parts one after another would take longer than computing them,
// so they are joined as a tree: parts 8i .. 8i + 7 by whichever of them comes
// last, into the slot of part 8i; those sums the same way, and so on.  One
// step of a worker's way up: what was part `index` of `count` (`stride` parts
// each) belongs to `members` ones from `from` on.
struct Climb {
    int index, count, stride = 1, level = 0;
    int from, members;
    __device__ __forceinline__ Climb(const Segment& g) : index(g.part), count(g.parts) { look(); }
    __device__ __forceinline__ void look() {
        from = index / kFan * kFan;
        members = min(kFan, count - from);
    }
    __device__ __forceinline__ bool top() const { return count <= kFan; }
    __device__ __forceinline__ void up() {
        index /= kFan;
        count = (count + kFan - 1) / kFan;
        stride *= kFan;
        level++;
        look();
    }
    // the part (of the unit's) whose slot holds member u
    __device__ __forceinline__ int part(int u) const { return (from + u) * stride; }
    // By one thread of a worker once all its threads have stored and passed a
    // __threadfence() and a barrier: whether it was the last of the members.
    // Counters are named by the piece of the first member; members of one unit
    // are the only ones to share it where there are two or more.  `which` of two:
    // the row tiles of a unit that joins them apart.
    __device__ __forceinline__ bool arrive(const PagedAttn& a, const Segment& g, int which) const {
        if (members == 1) return true;
        int* counter = reinterpret_cast<int*>(a.ws) + level * 2 * kMaxPieces + 2 * (g.first + part(0)) + which;
        const bool last = atomicAdd(counter, 1) == members - 1;
        if (last) atomicExch(counter, 0);
        return last;
    }
};

}  // namespace zl
