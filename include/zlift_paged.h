/*
 * zlift_paged.h -- a paged key/value cache in 16 or 8 bits, and attention of
 * each sequence's newest tokens over it.
 *
 * No counterpart in the reference: its attention entries decline a block
 * with a K/V cache (seqlen_knew) and ragged batches
 * (zblas/zblas_gpu.cpp:1424-1535).  These entries keep the manner of
 * zlift_attention.h: everything is enqueued on `stream` (0: the legacy
 * default stream) of the current device, which has to be the operands', and
 * nothing synchronises, allocates or copies to the host.
 *
 * Return value of every entry: 0 = done (enqueued), 1 = declined (the
 * arguments ask for something the kernels do not do; nothing was launched;
 * ZBLAS_TRACE prints the reason), 2 = the launch failed.
 *
 * What the host cannot see is checked on the device: a page or slot number
 * outside the cache is never followed.  A write to it is dropped, a read of
 * it gives zeros, attention treats its keys as absent, and
 * zlift_device_error() then reports 2.  Lengths are clamped to what the page
 * table and `total_q` can hold.  Index arrays must not change while a call
 * that reads them runs.
 *
 * Strides are in elements and may be anything (also negative or zero where
 * that makes sense for reading) unless stated; elements of one row (dim) are
 * contiguous.  The fast kernels need base pointers and strides that are
 * multiples of 16 bytes (attention: cache strides of 32), dim 64 or 128,
 * pages of a multiple of 8 tokens and a positive scale; everything else runs
 * on the CUDA cores, correct and slower.
 */
#ifndef ZLIFT_PAGED_H
#define ZLIFT_PAGED_H

#include <stddef.h>
#include <stdint.h>

#ifndef ZLIFT_API
#define ZLIFT_API __attribute__((visibility("default")))
#endif

#ifdef __cplusplus
extern "C" {
#endif

/* Types: those of `elem` in zlift_attention.h, and the 8-bit ones. */
enum {
    ZLIFT_KV_F16 = 0,
    ZLIFT_KV_BF16 = 1,
    ZLIFT_KV_F32 = 2,      /* kv_read's output only */
    ZLIFT_KV_I8 = 3,       /* codes -127..127 and one fp32 scale per row */
    ZLIFT_KV_E4M3 = 4      /* e4m3 codes and one fp32 scale per row */
};

/* The cache.  K and V of token slot s = page * page_size + offset and head h
 * are the `dim` elements at page*page_stride + offset*row_stride +
 * h*head_stride, the same in both.  An 8-bit row's scale is at
 * page*scale_page_stride + h*scale_head_stride + offset of k_scale/v_scale;
 * the row stands for code * scale. */
typedef struct zlift_kv_cache {
    void *k, *v;
    float *k_scale, *v_scale;               /* null for 16-bit caches */
    long long page_stride, row_stride, head_stride;
    long long scale_page_stride, scale_head_stride;
    int num_pages, page_size, heads, dim;   /* num_pages*page_size < 2^31 */
    int type;                               /* ZLIFT_KV_* (not F32) */
} zlift_kv_cache;

/* Packed tokens: K and V of token t and head h at t*row + h*head. */
typedef struct zlift_kv_rows {
    void *k, *v;
    long long k_row_stride, k_head_stride, v_row_stride, v_head_stride;
    int tokens;
    int elem;
} zlift_kv_rows;

/* Writes token t's K and V rows into slot slots[t] (device, int32; a negative
 * slot skips the token, as padding needs it; the others must differ: what two
 * tokens leave in one slot is undefined, codes of one beside the scale of the
 * other included).  rows->elem is F16 or BF16; a 16-bit cache has the same
 * type.
 *
 * An 8-bit row x is stored as scale = amax / top and codes
 * round(x * (top / amax)), amax = max |x|, top = 127 (I8) or 448 (E4M3);
 * both quotients and the product are rounded once to fp32, the codes to
 * nearest even.  amax < 2^-100 (all zeros included) stores scale 0 and codes
 * 0.  A row with a NaN or an infinity stores scale NaN and codes 0: 8 bits
 * cannot hold it, so the row reads as NaN rather than as wrong numbers.  The
 * NaN code of e4m3 is never stored, and what a reader makes of it is
 * undefined. */
ZLIFT_API int zlift_kv_write(const zlift_kv_cache *cache, const zlift_kv_rows *rows,
                             const int32_t *slots, void *stream);

/* Reads the tokens of `batch` sequences into packed rows: token t of
 * [cu[s], cu[s+1]) is position t - cu[s] (+ starts[s], when not null) of
 * sequence s, whose pages are page_table[s*table_stride ...], table_pages of
 * them.  cu has batch + 1 non-decreasing entries from 0; tokens of the
 * output at or past cu[batch] are left alone.  rows->elem is F16, BF16 or
 * F32 for an 8-bit cache (code * scale in fp32, rounded once), the cache's
 * own type otherwise.  All index arrays are int32 on the device. */
ZLIFT_API int zlift_kv_read(const zlift_kv_cache *cache, const zlift_kv_rows *rows,
                            const int32_t *page_table, long long table_stride, int table_pages,
                            const int32_t *starts, const int32_t *cu, int batch, void *stream);

/* One attention call: the newest cu_q[s+1] - cu_q[s] tokens of sequence s
 * (queries, packed) over all seq_k[s] tokens that its pages hold (the new
 * ones, already written, among them).  Query head h reads KV head
 * h / (heads / cache->heads).  Causal: query i of n sees key j when
 * j <= i + seq_k - n.  A query that sees no key gets O = 0, LSE = -inf.
 * Keys that a query does not see have no effect on it, whatever they hold. */
typedef struct zlift_paged_attn_params {
    const void *q;                          /* [total_q] x row, head strides */
    void *o;                                /* q's type */
    float *lse;                             /* [heads] x [total_q], or null */
    long long q_row_stride, q_head_stride, o_row_stride, o_head_stride;
    long long lse_head_stride;
    const int32_t *cu_q;                    /* [batch + 1], device */
    const int32_t *seq_k;                   /* [batch], device */
    const int32_t *page_table;              /* device */
    long long table_stride;
    int table_pages;                        /* entries of a sequence's row */
    int batch, total_q;
    int max_q;                              /* longest chunk; a hint that picks the kernel */
    int heads;
    int elem;                               /* F16 or BF16: q, o and a 16-bit cache */
    int causal;
    float scale;                            /* of Q.K^T, natural-log units */
    void *workspace;                        /* zeroed once by its owner, see below */
    size_t workspace_bytes;
} zlift_paged_attn_params;

/* Device bytes zlift_paged_attn wants for such a call (workspace fields not
 * read).  The workspace is 256-byte aligned and zero before its first use;
 * every call leaves it fit for the next one of any shape.  Calls that share
 * one must run one after another; after device error 1 (a wait ran out) it has
 * to be zeroed again.  0 for calls that will be declined or need none. */
ZLIFT_API size_t zlift_paged_attn_workspace(const zlift_kv_cache *cache,
                                            const zlift_paged_attn_params *p);

ZLIFT_API int zlift_paged_attn(const zlift_kv_cache *cache, const zlift_paged_attn_params *p,
                               void *stream);

#ifdef __cplusplus
}
#endif
#endif
