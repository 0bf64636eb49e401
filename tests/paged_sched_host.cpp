// The work line of paged_sched.cuh on the host: a warp is 32 threads that meet
// at every exchange between lanes.  Reads calls from standard input,
//     tokens keys least pieces causal heads page_size table_pages batch  then  n len  for each sequence
// walks every piece and prints, for each call, the step that was chosen, the
// work it found (units, keys) and whether every unit's keys came exactly once
// and in as many parts as the segments say.
#include <pthread.h>

#include <algorithm>
#include <cstdint>
#include <cstdio>
#include <thread>
#include <vector>

#include <cuda_runtime.h>

using std::max;
using std::min;

struct Lane { unsigned x; };
static thread_local Lane lane_id;
#define threadIdx lane_id
#define blockIdx lane_id
static pthread_barrier_t meet;
static unsigned long long cell[32];
template <class T>
static T exchange(T v, int from) {
    cell[lane_id.x] = (unsigned long long)v;
    pthread_barrier_wait(&meet);
    const T r = (T)cell[from & 31];
    pthread_barrier_wait(&meet);
    return r;
}
static bool solo;                        // outside of start() every lane does the same
template <class T> static T __shfl_sync(unsigned, T v, int from) { return solo ? v : exchange(v, from); }
template <class T> static T __shfl_up_sync(unsigned, T v, int d) {
    const int at = (int)lane_id.x - d;
    const T r = exchange(v, at < 0 ? lane_id.x : at);
    return r;
}
static unsigned __ballot_sync(unsigned, bool p) {
    cell[lane_id.x] = p;
    pthread_barrier_wait(&meet);
    unsigned r = 0;
    for (int i = 0; i < 32; i++) r |= (unsigned)cell[i] << i;
    pthread_barrier_wait(&meet);
    return r;
}
static int __ffs(unsigned v) { return __builtin_ffs((int)v); }
static unsigned __umulhi(unsigned a, unsigned b) { return (unsigned)((unsigned long long)a * b >> 32); }
template <class T> static T __ldg(const T* p) { return *p; }
static int atomicCAS(int* p, int a, int b) { const int v = *p; if (v == a) *p = b; return v; }
static int atomicAdd(int* p, int d) { const int v = *p; *p += d; return v; }
static int atomicExch(int* p, int d) { const int v = *p; *p = d; return v; }
static unsigned __cvta_generic_to_shared(const void*) { return 0; }
static void __nanosleep(unsigned) {}

#define __noinline__ __attribute__((noinline))
#define cudaMemcpyToSymbol(...) cudaErrorNotSupported
#define cudaMemcpyFromSymbol(...) cudaErrorNotSupported
#include "paged_sched.cuh"

int main() {
    pthread_barrier_init(&meet, nullptr, 32);
    long long tokens, keys, least, pieces, causal, heads, ps, tpages, batch;
    while (scanf("%lld %lld %lld %lld %lld %lld %lld %lld %lld", &tokens, &keys, &least, &pieces, &causal, &heads,
                 &ps, &tpages, &batch) == 9) {
        std::vector<int> cu(batch + 1, 0), len(batch);
        for (int i = 0; i < batch; i++) {
            int n;
            if (scanf("%d %d", &n, &len[i]) != 2) return 1;
            cu[i + 1] = cu[i] + n;
        }
        zl::PagedAttn a{};
        a.cu = cu.data(); a.len = len.data();
        a.tpages = (int)tpages; a.batch = (int)batch; a.total_q = cu[batch];
        a.causal = (int)causal;
        a.c.heads = (int)heads; a.c.ps = (int)ps;
        const zl::SchedShape h = zl::sched_shape(a, (int)tokens, (int)keys, (int)least, (int)pieces);
        long long units = 0, found = 0, bad = 0;
        // where the line stands: the unit, and its keys and parts so far
        int s = 0, head = 0, i0 = 0, at = 0, part = 0;
        auto first = [&] { while (s < batch && cu[s + 1] == cu[s]) s++; };
        first();
        for (int piece = 0; piece < h.pieces; piece++) {
            zl::Walker w[32];
            std::vector<std::thread> warp;
            for (unsigned l = 0; l < 32; l++)
                warp.emplace_back([&, l] {
                    lane_id.x = l;
                    w[l].start(a, h, piece);
                });
            for (auto& t : warp) t.join();
            for (int l = 1; l < 32; l++) bad += w[l].pos != w[0].pos || w[l].end != w[0].end || (w[0].pos < w[0].end && (w[l].begin != w[0].begin || w[l].s != w[0].s));
            solo = true;
            zl::Segment g;
            while (w[0].next(a, h, piece, g)) {
                if (s >= batch) { bad++; break; }
                const int n = cu[s + 1] - cu[s], last = min(n, i0 + (int)tokens);
                const int e = causal ? max(0, min(len[s], len[s] - n + last)) : len[s];
                bad += g.s != s || g.head != head || g.i0 != i0 || g.ni != last - i0 || g.k0 != at || g.k1 > e ||
                       g.k0 % (int)keys || (g.k1 != e && g.k1 % (int)keys) || g.part != part || g.first != piece - part;
                found += g.k1 - g.k0;
                at = g.k1;
                if (++part == g.parts) {             // the unit ends
                    bad += at != e;
                    units++;
                    at = part = 0;
                    i0 = last;
                    if (i0 == n) {
                        i0 = 0;
                        if (++head == heads) {
                            head = 0;
                            s++;
                            first();
                        }
                    }
                }
            }
            solo = false;
        }
        bad += s != batch || part != 0;
        printf("%d %lld %lld %lld\n", h.step, units, found, bad);
    }
    return 0;
}
