/*
 * kv_pages.h -- a paged KV cache that sequences share, and the attention that reads it (none of
 * this exists in typhoon-ocr-server, whose cache is one contiguous block per request,
 * kernel/kv_cache.h:11-26).
 *
 * A pool holds `num_pages` pages of `page_size` rows for every layer; a sequence is a row of the
 * table that names its pages in order, and a page may be named by several sequences (ref counts
 * them), so that requests about one document hold its rows once.  Everything the calls below
 * read and write is memory of the pool's DEVICE, bookkeeping included (another device's is refused): a
 * call queues work on the library stream (attn_set_stream) and returns; nothing is read back.  A call may be captured in a CUDA graph
 * once a call of the same sizes has been made on that pool (it sizes the pool's workspace; a captured
 * call that would need more is refused).  Later calls of any size leave such a graph valid.
 *
 * Errors: what the host can see is refused with a nonzero return and attn_last_error().  What only
 * the device can see raises a bit that the next attn_sync() reports: a sequence, page or length
 * outside its bounds ("index check failed"), or a pool without enough free pages ("out of
 * pages").  A maintenance call that raises one changes nothing, except kv_pages_write: it writes the
 * rows whose places are there, and raises one for the others.  A wait that ran out ("wait timed out")
 * in a single-token attention call is raised again by those that follow on its pool, replays among
 * them, until attn_sync() has reported it; from then on they are right.
 *
 * A pool is driven from one stream at a time, replays of the graphs captured from it among the work
 * that this counts.
 */
#pragma once
#include "kv_cache.h"

#ifdef __cplusplus
extern "C" {
#endif

typedef struct {
    void *k, *v;   /* device [num_layers][num_pages][kv_heads][page_size][head_dim], ATTN_KV_* elements */
    int  *table;   /* device [max_seqs][max_pages]: page of rows [i * page_size, (i + 1) * page_size), -1: none */
    int  *len;     /* device [max_seqs]: tokens of the sequence (0: not in use) */
    int  *ref;     /* device [num_pages]: table entries that name the page (0: free) */
    int   num_layers, num_pages, page_size, kv_heads, head_dim, max_seqs, max_pages, kv_dtype;
} KVPages;

/* An empty pool: page_size 16, 32, 64 or 128 rows; head_dim 64 or 128; kv_dtype ATTN_KV_F32 or
 * ATTN_KV_BF16; num_layers * num_pages * kv_heads * page_size < 2^31.  NULL on failure. */
KVPages *kv_pages_alloc(int num_layers, int num_pages, int page_size, int kv_heads, int head_dim,
                        int max_seqs, int max_pages, int kv_dtype);
/* The same over the caller's device memory (16-byte aligned K and V), in whatever state its
 * bookkeeping is; kv_pages_release leaves that memory alone. */
KVPages *kv_pages_attach(void *k, void *v, int *table, int *len, int *ref, int num_layers, int num_pages,
                         int page_size, int kv_heads, int head_dim, int max_seqs, int max_pages, int kv_dtype);
/* Waits for the library stream, then frees the handle, its workspace (what a captured call was given of
 * that is kept until exit) and the memory that kv_pages_alloc made. */
void     kv_pages_release(KVPages *p);

/* ---- maintenance ------------------------------------------------------------------------
 * seqs, src, dst, counts, starts: device int32.  New pages are the lowest-numbered free ones, given
 * out in the order of the list, so that equal states and calls give equal tables.  0 on success.
 *
 * kv_pages_extend: sequence seqs[i] grows by counts[i] >= 0 tokens (pages taken, len advanced; the
 * rows are then written, layer by layer, with kv_pages_write).  A sequence appears once. */
int kv_pages_extend(KVPages *p, const int *seqs, const int *counts, int n);
/* The last starts[i + 1] - starts[i] rows of each sequence, from rows starts[i].. of k_new and v_new
 * [rows][kv_heads][head_dim] in `in_dtype` (ATTN_DT_*), rows `stride` elements apart; starts[n] = rows.
 * Each row is placed by itself: one without a place (no such sequence, not so long, its page given back)
 * is reported and the others are written.  Table, lengths and counts stay as they are. */
int kv_pages_write(KVPages *p, int layer, const int *seqs, const int *starts, int n, int rows, const void *k_new,
                   const void *v_new, int in_dtype, long long stride);
/* Rows [0, cache->seq_len) of all 28 layers of a static cache become sequence `seq` (not in use
 * before; the pool has 28 layers, 8 KV heads, head_dim 128 and the cache's element type). */
int kv_pages_import(KVPages *p, int seq, const KVCache *cache);
/* Sequence dst[i] (not in use before, named once, no src) becomes a branch of src[i]: it names the
 * same pages, except a partly filled last page, which it gets a copy of.  Either may then grow. */
int kv_pages_fork(KVPages *p, const int *src, const int *dst, int n);
/* The same with pages of its own throughout. */
int kv_pages_copy(KVPages *p, const int *src, const int *dst, int n);
/* The sequences are no longer in use; pages that no other sequence names are free. */
int kv_pages_free(KVPages *p, const int *seqs, int n);
/* Gives back the pages that no token from the sequence's last one on can see through a window
 * (>= 1) with sinks (attention_pages_window_gqa): those wholly at or past row `sinks` and before row
 * len - window. */
int kv_pages_trim(KVPages *p, const int *seqs, int n, int window, int sinks);
/* Moves pages so that those in use are [0, live): the pages in use from `live` on go, in order, to
 * the free ones below it.  live_out: NULL, or a device int that receives `live`. */
int kv_pages_compact(KVPages *p, int *live_out);

/* ---- attention --------------------------------------------------------------------------
 * Queries and the rows in the pool are taken as they are: normalised and rotated by the caller where the
 * model asks for it.  Query head h reads KV head h / (q_heads / kv_heads); q_heads is a multiple of kv_heads, at most
 * 16 times it.  q: token rows [..][q_heads][head_dim], rows q_stride elements apart; output
 * [..][q_heads][head_dim], contiguous; both in io_dtype (ATTN_DT_*).  Scores are scale * q . k; sums
 * and softmax statistics are FP32.  An ATTN_KV_BF16 pool multiplies BF16 operands (an FP32 query is
 * rounded); an ATTN_KV_F32 pool keeps FP32 accuracy throughout.  A row that sees nothing gives zeros.
 * Rows of a page that has been given back (table entry -1) are not seen, and what lies in a page
 * beyond its sequence's rows is never used.  A non-finite K or V row makes the outputs of the
 * queries that see it non-finite; in a chunk, it may do the same to queries near them.
 * max_len: at least the length of every sequence of the call (the work is split by it).
 * 0 on success.
 *
 * One token for each of `batch` sequences (their last one, its row written) that hold the same
 * first prefix_len tokens, in the same pages as far as those are full (what kv_pages_fork leaves):
 * the shared pages are read and multiplied once for all sequences, every sequence's further rows
 * by themselves, and the two parts joined.  All of len[seqs[b]] is seen.  A sequence that is shorter
 * than the shared pages is reported ("index check failed"); one not in use may fill up a batch, though
 * not as the first of any 1,024, and its output means nothing. */
int attention_pages_prefix_gqa(const void *q, long long q_stride, const KVPages *p, int layer, const int *seqs,
                               int batch, int q_heads, int prefix_len, int max_len, void *output, int io_dtype,
                               float scale);
/* Causal attention of each sequence's last tokens, a sliding window with sinks: sequence seqs[b]'s
 * queries are rows starts[b] .. starts[b + 1] of q, its last starts[b + 1] - starts[b] tokens; the one
 * at position i sees rows j <= i with j > i - window or j < sinks.  window 0: all j <= i.  max_new: at
 * least the queries of every sequence; 1 (single tokens: starts may be NULL, one each) takes the
 * decode form.  rows: starts[batch]. */
int attention_pages_window_gqa(const void *q, long long q_stride, const KVPages *p, int layer, const int *seqs,
                               const int *starts, int batch, int rows, int q_heads, int max_new, int max_len,
                               int window, int sinks, void *output, int io_dtype, float scale);

#ifdef __cplusplus
}
#endif
