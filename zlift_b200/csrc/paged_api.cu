// paged_api.cu -- the C entries of include/zlift_paged.h: argument checks
// and the choice of kernel.
#include "gemm.h"
#include "paged.h"

#include <cstdio>

namespace {

using namespace zl;

int declined(const char* who, const char* why) {
    if (tracing()) fprintf(stderr, "[zblas] %s declined: %s\n", who, why);
    return 1;
}

int finish(const char* who, int rc) {
    if (rc == 0) return 0;
    if (rc == 1) return declined(who, "shape or layout outside the kernels");
    if (tracing()) fprintf(stderr, "[zblas] %s launch failed: %d\n", who, rc);
    cudaGetLastError();
    return 2;
}

bool view(const zlift_kv_cache* z, KvView& c, const char* who) {
    auto no = [&](const char* why) {
        declined(who, why);
        return false;
    };
    if (!z || !z->k || !z->v) return no("null cache");
    if (z->type != ZLIFT_KV_F16 && z->type != ZLIFT_KV_BF16 && z->type != ZLIFT_KV_I8 &&
        z->type != ZLIFT_KV_E4M3)
        return no("cache type");
    if (z->type >= ZLIFT_KV_I8 && (!z->k_scale || !z->v_scale)) return no("no scales");
    if (z->num_pages <= 0 || z->page_size <= 0 || z->heads <= 0 || z->dim <= 0)
        return no("empty cache");
    if ((long long)z->num_pages * z->page_size > 0x7fffffffLL) return no("cache of 2^31 slots");
    if (z->heads > 65535 || z->dim > 65536) return no("heads or dim");
    c.k = static_cast<char*>(z->k);
    c.v = static_cast<char*>(z->v);
    c.ks = z->k_scale;
    c.vs = z->v_scale;
    c.page = z->page_stride; c.row = z->row_stride; c.head = z->head_stride;
    c.spage = z->scale_page_stride; c.shead = z->scale_head_stride;
    c.pages = z->num_pages; c.ps = z->page_size; c.heads = z->heads; c.dim = z->dim;
    c.by_ps = FastDiv((unsigned)c.ps);
    return true;
}

bool describe(const zlift_kv_cache* cache, const zlift_paged_attn_params* p, PagedAttn& a) {
    const char* who = "paged attention";
    auto no = [&](const char* why) {
        declined(who, why);
        return false;
    };
    if (!view(cache, a.c, who)) return false;
    if (!p) return no("null parameters");
    if (p->elem != ZLIFT_KV_F16 && p->elem != ZLIFT_KV_BF16) return no("element type");
    if (cache->type < ZLIFT_KV_I8 && cache->type != p->elem) return no("cache of another type");
    if (a.c.dim > 256) return no("dim above 256");
    if (p->batch < 0 || p->total_q < 0 || p->table_pages < 0) return no("negative size");
    if (p->heads <= 0 || p->heads > 65535 || p->heads % a.c.heads) return no("head grouping");
    // (some room below 2^31, so that key numbers a few tiles past the end fit)
    if ((long long)p->table_pages * a.c.ps > 0x7fff0000LL) return no("2^31 keys in a sequence");
    if (p->batch > 0 && p->total_q > 0 &&
        (!p->q || !p->o || !p->cu_q || !p->seq_k || (!p->page_table && p->table_pages > 0)))
        return no("null operand");
    a.q = static_cast<const char*>(p->q);
    a.o = static_cast<char*>(p->o);
    a.lse = p->lse;
    a.qr = p->q_row_stride; a.qh = p->q_head_stride;
    a.orow = p->o_row_stride; a.oh = p->o_head_stride;
    a.lh = p->lse_head_stride;
    a.cu = p->cu_q; a.len = p->seq_k; a.table = p->page_table;
    a.tstride = p->table_stride;
    a.tpages = p->table_pages; a.batch = p->batch; a.total_q = p->total_q; a.max_q = p->max_q;
    a.heads = p->heads; a.group = p->heads / a.c.heads;
    a.causal = p->causal ? 1 : 0;
    a.scale = p->scale;
    a.ws = static_cast<char*>(p->workspace);
    a.ws_bytes = p->workspace_bytes;
    a.elem = p->elem; a.type = cache->type;
    return true;
}

enum class Way { Simt, Decode, Chunk };

// Which kernel serves a call.  The tensor-core kernels take rows in 16-byte
// pieces, find a token by a 32-bit count of 32 bytes, and scale by a positive
// factor after the running maximum.
Way choose(const PagedAttn& a) {
    const int eb = a.type >= kI8 ? 1 : 2;
    if (a.c.dim != 64 && a.c.dim != 128) return Way::Simt;
    if (!(a.scale > 0.f) || !std::isfinite(a.scale)) return Way::Simt;
    if (a.c.page < 0 || a.c.row < 0 || a.c.head < 0) return Way::Simt;
    if ((a.c.page * eb) % 32 || (a.c.row * eb) % 32 || (a.c.head * eb) % 16) return Way::Simt;
    const double span = ((double)(a.c.pages - 1) * a.c.page + (double)(a.c.ps - 1) * a.c.row) * eb;
    if (span / 32 >= 4294967295.0) return Way::Simt;
    if ((a.qr * 2) % 16 || (a.qh * 2) % 16) return Way::Simt;
    for (const void* p : {(const void*)a.q, (const void*)a.c.k, (const void*)a.c.v})
        if (reinterpret_cast<uintptr_t>(p) & 15u) return Way::Simt;
    auto steps = [](long long stride, int count) { return stride > 0 || count == 1; };
    if (a.c.ps % 8 || !steps(a.c.row, a.c.ps) || !steps(a.c.head, a.c.heads) ||
        !steps(a.c.page, a.c.pages))
        return Way::Simt;
    // the chunk kernel's boxes: whole ones inside a page (16 bit), queries and
    // output rows by 16-byte pieces
    const bool boxes = steps(a.qr, a.total_q) && steps(a.qh, a.heads) &&
                       a.group <= 128 && (reinterpret_cast<uintptr_t>(a.o) & 15u) == 0 &&
                       (a.orow * 2) % 16 == 0 && (a.oh * 2) % 16 == 0;
    // Few rows go to the kernel that reads the cache once for 24 of them; more,
    // to the one with tiles of 128 rows.  Over 32 x up to 4096 tokens, dim 128, 8 KV
    // heads, in us:
    //              bf16 cache                e4m3 cache
    //   rows   4   24   32   48  128     4   24   32   64  128
    //   few   70   84   88  132  274    56   77   82  151  228   (from 32 on: one
    //   tiles 101  105  101  113  116   174  177  173  199  179    read per 24 rows)
    // So the tiles win from some 40 rows on over 16 bits and from some 80 over 8.
    // The limit is the rows of one tile all the same.
    const long long rows = (long long)(a.max_q > 1 ? a.max_q : 1) * a.group;
    if (a.group <= decode_max_rows() && (rows <= decode_max_rows() || !boxes)) return Way::Decode;
    return boxes ? Way::Chunk : Way::Simt;
}

size_t workspace_of(const PagedAttn& a) {
    switch (choose(a)) {
    case Way::Decode: return paged_decode_workspace(a);
    case Way::Chunk: return paged_chunk_workspace(a);
    default: return 0;
    }
}

}  // namespace

extern "C" {

int zlift_kv_write(const zlift_kv_cache* cache, const zlift_kv_rows* rows, const int32_t* slots,
                   void* stream) {
    const char* who = "kv write";
    KvView c;
    if (!view(cache, c, who)) return 1;
    if (!rows) return declined(who, "null rows");
    if (rows->elem != ZLIFT_KV_F16 && rows->elem != ZLIFT_KV_BF16)
        return declined(who, "element type");
    if (cache->type < ZLIFT_KV_I8 && cache->type != rows->elem)
        return declined(who, "cache of another type");
    if (rows->tokens < 0) return declined(who, "negative size");
    if (rows->tokens == 0) return 0;
    if (!rows->k || !rows->v || !slots) return declined(who, "null operand");
    return finish(who, kv_write(c, cache->type, *rows, slots, static_cast<cudaStream_t>(stream)));
}

int zlift_kv_read(const zlift_kv_cache* cache, const zlift_kv_rows* rows,
                  const int32_t* page_table, long long table_stride, int table_pages,
                  const int32_t* starts, const int32_t* cu, int batch, void* stream) {
    const char* who = "kv read";
    KvView c;
    if (!view(cache, c, who)) return 1;
    if (!rows) return declined(who, "null rows");
    if (rows->elem != ZLIFT_KV_F16 && rows->elem != ZLIFT_KV_BF16 && rows->elem != ZLIFT_KV_F32)
        return declined(who, "element type");
    if (cache->type < ZLIFT_KV_I8 && cache->type != rows->elem)
        return declined(who, "cache of another type");
    if (rows->tokens < 0 || batch < 0 || table_pages < 0) return declined(who, "negative size");
    if ((long long)table_pages * c.ps > 0x7fffffffLL) return declined(who, "2^31 positions");
    if (rows->tokens == 0 || batch == 0) return 0;
    if (!rows->k || !rows->v || !cu || (!page_table && table_pages > 0))
        return declined(who, "null operand");
    return finish(who, kv_read(c, cache->type, *rows, page_table, table_stride, table_pages, starts,
                               cu, batch, static_cast<cudaStream_t>(stream)));
}

size_t zlift_paged_attn_workspace(const zlift_kv_cache* cache, const zlift_paged_attn_params* p) {
    PagedAttn a;
    if (!describe(cache, p, a)) return 0;
    return workspace_of(a);
}

int zlift_paged_attn(const zlift_kv_cache* cache, const zlift_paged_attn_params* p, void* stream) {
    PagedAttn a;
    if (!describe(cache, p, a)) return 1;
    if (a.batch == 0 || a.total_q == 0) return 0;
    const char* who = "paged attention";
    const size_t need = workspace_of(a);
    if (need && (!a.ws || a.ws_bytes < need || (reinterpret_cast<uintptr_t>(a.ws) & 255u)))
        return declined(who, "workspace missing, small or unaligned");
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    switch (choose(a)) {
    case Way::Decode: return finish(who, paged_decode(a, s));
    case Way::Chunk: return finish(who, paged_chunk(a, s));
    default: return finish(who, paged_attn_simt(a, s));
    }
}

}  // extern "C"
