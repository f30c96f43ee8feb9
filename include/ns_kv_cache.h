/* ns_kv_cache.h: C-ABI of the MI355X paged KV cache: the store of new key and value rows, and the pages.
 *
 * Replaces, around the attention of ns_paged_attention.h:
 *   nanoserve/model/rope.py:78-91       (apply_rope) and nanoserve/model/attention.py:55-72
 *                                       (write_kv_to_cache): ns_kv_store, one launch;
 *   nanoserve/cache/block_allocator.py:14-47 (BlockAllocator, a free list on the host): ns_kv_extend and
 *                                       ns_kv_free on device tables.  Forking, releasing pages behind
 *                                       a window and compacting have no counterpart in the reference.
 *
 * All pointers are device pointers unless said otherwise; nothing is read on the host, no call
 * synchronizes or allocates, and every call can be captured into a graph.  Calls that change one pool
 * run one after another (on one stream, or ordered by the caller).
 */
#ifndef NS_KV_CACHE_H
#define NS_KV_CACHE_H

#include <stddef.h>
#include <stdint.h>
#include <hip/hip_runtime_api.h>

#ifdef __cplusplus
extern "C" {
#endif

#define NS_KV_ABI_VERSION 1

#define NS_KV_DTYPE_F32 0
#define NS_KV_DTYPE_BF16 1
#define NS_KV_DTYPE_F16 2

/* rows of one ns_kv_extend or ns_kv_fork call */
#define NS_KV_MAX_ROWS 4096

/* status bits, OR-ed into the word that `status` points to (when not NULL) */
#define NS_KV_STATUS_BAD_PAGE 1    /* a page number outside the cache, or a position past the table's columns:
                                      that row or page is not stored, copied or counted */
#define NS_KV_STATUS_NO_PAGES 2    /* not enough free pages for a listed row (it is left as it was), or for
                                      ns_kv_compact's smaller cache (nothing is moved) */
#define NS_KV_STATUS_BAD_ROW 4     /* a listed row outside the tables, listed before in the same call, or a child
                                      that holds a sequence already: left alone */
#define NS_KV_STATUS_BAD_LENGTH 8  /* a new length below the row's, or past the table's columns: row left alone */

/* New tokens' keys and values into their pages; queries and keys rotated by position when inv_freq is set.
 *
 * Token i of sequence s (rows query_start_loc[s] .. + query_lens[s] - 1 of key, value and query) is at
 * position p = seq_lens[s] - query_lens[s] + (i - query_start_loc[s]), the position that ns_paged_attention
 * gives it, and its row goes to page block_tables[s][p / block_size], slot p % block_size.  Rows that are no
 * sequence's token (a padded batch's) are left alone, in out too.  Two tokens of one call are not to have the
 * same page and slot (tables that share a page that is written): which row's pieces stay is not defined then.
 *
 * Rotation (the reference's rotate-half form): with a_j = p * inv_freq[j], j < head_dim / 2, the pair
 * (x_j, x_{j + head_dim / 2}) becomes (x_j cos a_j - x_{j + head_dim/2} sin a_j,
 * x_{j + head_dim/2} cos a_j + x_j sin a_j).  a_j is formed and reduced in 64 bits, the rest is float32,
 * rounded once to the type. */
typedef struct ns_kv_store_args {
  const void*    query;            /* (total, num_heads_q, head_dim) or NULL */
  const void*    key;              /* (total, num_kv_heads, head_dim) */
  const void*    value;            /* (total, num_kv_heads, head_dim) */
  void*          k_cache;          /* (num_blocks, block_size, num_kv_heads, head_dim) */
  void*          v_cache;          /* the same shape */
  void*          out;              /* the rotated query, like query (may be the query itself), or NULL with it */
  const float*   inv_freq;         /* (head_dim / 2), or NULL: nothing is rotated and query is NULL */
  const int32_t* block_tables;     /* (num_seqs, stride_bt_seq) */
  const int32_t* seq_lens;         /* (num_seqs): lengths with the new tokens */
  const int32_t* query_start_loc;  /* (num_seqs + 1) */
  const int32_t* query_lens;       /* (num_seqs) */
  int32_t*       status;           /* optional: NS_KV_STATUS_BAD_PAGE */
  int64_t        stride_q_token, stride_q_head;
  int64_t        stride_key_token, stride_key_head;
  int64_t        stride_value_token, stride_value_head;
  int64_t        stride_k_block, stride_k_token, stride_k_head;
  int64_t        stride_v_block, stride_v_token, stride_v_head;
  int64_t        stride_o_token, stride_o_head;
  int64_t        stride_bt_seq;
  int32_t        total, num_seqs, num_heads_q, num_kv_heads;
  int32_t        head_dim;         /* 64 or 128; rows are 16-byte aligned with a unit head_dim stride */
  int32_t        block_size, num_blocks, max_blocks_per_seq;
  int32_t        dtype;            /* NS_KV_DTYPE_* */
} ns_kv_store_args;

/* A pool of pages: the caches of all layers, whose pages are numbered alike, and who holds them.
 * Row r holds seq_lens[r] tokens in pages block_tables[r][0 .. ceil(seq_lens[r] / block_size) - 1], -1 for a
 * page released behind a window.  page_refs[p] counts the table entries that name page p, plus one for a
 * page that is never to be handed out (the reference's padding page 0); 0: free. */
typedef struct ns_kv_pool {
  int32_t*       block_tables;     /* (num_rows, stride_bt_row), num_cols of it used */
  int32_t*       seq_lens;         /* (num_rows) */
  int32_t*       page_refs;        /* (num_pages), 16-byte aligned */
  int32_t*       status;           /* optional */
  const uint64_t* tensors;         /* (num_tensors, 2): each cache tensor's address and bytes from page to page */
  int32_t*       scratch;          /* ns_kv_scratch_bytes() bytes, any contents, this pool's own */
  uint64_t       scratch_bytes;
  int64_t        stride_bt_row;
  int64_t        slot_bytes;       /* bytes of a token in a page of one tensor, a multiple of 16 */
  int32_t        num_rows, num_cols, num_pages, num_tensors;
  int32_t        block_size;
} ns_kv_pool;

/* Version of this ABI (NS_KV_ABI_VERSION). */
int ns_kv_abi_version(void);

/* Message of the last failed call on this thread. */
const char* ns_kv_last_error(void);

/* Every function below returns 0, or nonzero on invalid arguments. */
int ns_kv_store(const ns_kv_store_args* args, hipStream_t stream);

/* Bytes of the scratch memory of a pool of num_pages pages. */
int ns_kv_scratch_bytes(int32_t num_pages, uint64_t* bytes);

/* Rows rows[0 .. n-1] grow to lens[0 .. n-1] tokens and get the pages that these need, the lowest free pages
 * first, in the order of the list.  A row is served if the pages that it and the rows listed before it ask for
 * are all there, or if it asks for none. */
int ns_kv_extend(const ns_kv_pool* pool, const int32_t* rows, const int32_t* lens, int32_t n, hipStream_t stream);

/* children[i], an empty row, becomes a copy of row parents[i]: the full pages are shared, the filled slots of a
 * last page that is not full are copied, in every tensor, into a page of its own (the lowest free one, in the
 * order of the list; a child for which none is left stays empty). */
int ns_kv_fork(const ns_kv_pool* pool, const int32_t* parents, const int32_t* children, int32_t n, hipStream_t stream);

/* The listed rows give up their pages and become empty.  A row may be listed more than once. */
int ns_kv_free(const ns_kv_pool* pool, const int32_t* rows, int32_t n, hipStream_t stream);

/* The listed rows give up the pages that no later token sees through `window` and `sinks` (those of
 * ns_paged_attention_windowed): columns j with j * block_size >= sinks and (j + 1) * block_size <=
 * seq_lens[row] - window + 1. Their entries become -1. */
int ns_kv_release(const ns_kv_pool* pool, const int32_t* rows, int32_t n, int32_t window, int32_t sinks,
                  hipStream_t stream);

/* Pages src[0 .. n-1] of `pool` copied to pages dst[0 .. n-1] of `to` (the same pool or one of equal tensors), in
 * every tensor.  No page is to be named twice by dst or, within one pool, by both. */
int ns_kv_copy(const ns_kv_pool* pool, const ns_kv_pool* to, const int32_t* src, const int32_t* dst, int32_t n,
               hipStream_t stream);

/* The m pages in use become pages 0 .. m-1: those numbered m or higher move, in ascending order, to the free
 * ones below m.  page_map[p] (num_pages) receives page p's new number, -1 for a free page.  With `to` NULL the
 * pages move within the pool and its tables and counts follow; else the pool stays as it is and `to`, a pool of
 * as many rows, columns and tensors and of at least m pages, receives its pages, tables, lengths and counts (its memory
 * is none of the pool's). */
int ns_kv_compact(const ns_kv_pool* pool, const ns_kv_pool* to, int32_t* page_map, hipStream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* NS_KV_CACHE_H */
