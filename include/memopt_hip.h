/*
 * memopt_hip.h — C ABI of the MI355X (gfx950) INT4 KV-cache data plane.
 *
 * Every entry point takes plain device pointers, 64-bit sizes and a
 * hipStream_t (passed as void*), returns an int status (MEMOPT_OK == 0) and
 * records a human-readable message retrievable with memopt_last_error()
 * (thread-local). No libtorch types cross this boundary: callers allocate
 * device memory themselves (the Python `memopt_C` shim uses torch tensors)
 * and keep it alive while the library uses it.
 *
 * Each declaration names the reference interface it replaces:
 * TheRadDani/memopt-transformer-runtime, pybind11 module `memopt_C`
 * (src/csrc/extension.cpp) and the C++ functions it binds.
 *
 * Kernel entry points are asynchronous on `stream`; launch errors are
 * reported through the status code.
 */
#ifndef MEMOPT_HIP_H
#define MEMOPT_HIP_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* ------------------------------------------------------------------------ */
/* Status codes                                                             */
/* ------------------------------------------------------------------------ */
#define MEMOPT_OK               0
#define MEMOPT_ERR_INVALID      1  /* contract violation (shape/dtype/range) */
#define MEMOPT_ERR_STATE        2  /* pool not initialized                    */
#define MEMOPT_ERR_HIP          3  /* HIP runtime / launch error              */
#define MEMOPT_ERR_UNSUPPORTED  4  /* configuration not compiled in           */

/* KV storage formats (memopt_init_pool `kv_format`, memopt_attn_desc.kv_format). */
#define MEMOPT_KV_FP16       0  /* fp16 [num_blocks, block_size, H, D] (reference layout)  */
#define MEMOPT_KV_INT4       1  /* INT4 page pool, one u8 buffer [num_blocks, H, B] with    *
                                 * B = 16*D + 64*(D/64) bytes per (page, head):             *
                                 *   K codes (8*D) | V codes (8*D) | K scales | V scales    *
                                 * (fp16 scales, 32*(D/64) bytes each); 16-token pages;     *
                                 * codes laid out for the wave64 decode kernel: lane 8p+c   *
                                 * owns tokens (p, p+8) x dims [c*D/8, (c+1)*D/8); see      *
                                 * memopt-transformer-runtime_amd/csrc/page_format.hpp.     */
#define MEMOPT_KV_INT4_ROWS  2  /* attention input only: INT4 codes in the reference's      *
                                 * quantize_kv_cache_int4 byte order with arbitrary         *
                                 * page/head/token strides + separate f32/f16 scales        */

/* Scale element types for INT4 caches passed to attention. */
#define MEMOPT_SCALE_F32 0
#define MEMOPT_SCALE_F16 1

/* Message of the last failed call on this thread ("" if none). */
const char *memopt_last_error(void);

/* Replaces get_hello() — src/csrc/extension.cpp:6-8. */
const char *memopt_get_hello(void);

/* ------------------------------------------------------------------------ */
/* Paged pool (host free list + registered device storage)                 */
/* ------------------------------------------------------------------------ */

/* Replaces init_pool(num_blocks, block_size, num_heads, head_dim) —
 * src/csrc/kv_cache.cu:112-153, bound at src/csrc/extension.cpp:20-26.
 * The caller allocates the storage, filled with the empty-row pattern, and
 * passes it in:
 *   MEMOPT_KV_FP16: key/value = fp16 [nb, bs, H, D] zeros; scale pointers unused.
 *   MEMOPT_KV_INT4: key_pool = the page buffer (codes 0x88, scales 1.0);
 *                   value_pool / key_scales / value_scales unused (NULL);
 *                   block_size must be 16 and head_dim a multiple of 64.
 * The free list is reseeded FIFO 0..nb-1. Invalid parameters tear the pool
 * down and return MEMOPT_ERR_INVALID. */
int memopt_init_pool(int64_t num_blocks, int32_t block_size, int32_t num_heads,
                     int32_t head_dim, int32_t kv_format, void *key_pool,
                     void *value_pool, void *key_scales, void *value_scales);

/* Reports the live pool's parameters; returns 1 if a pool is initialized,
 * 0 otherwise (outputs untouched). Used for init_pool's idempotency
 * (src/csrc/kv_cache.cu:115-122). */
int memopt_pool_info(int64_t *num_blocks, int32_t *block_size, int32_t *num_heads,
                     int32_t *head_dim, int32_t *kv_format);

/* Drops the pool (storage pointers are forgotten; the caller frees them). */
int memopt_reset_pool(void);

/* Swaps the live pool's storage and format (fp16 <-> INT4 pages) for the same
 * geometry, keeping the free list, so block tables stay valid across the
 * switch. No counterpart in the reference: it serves the policy forward
 * wrapper that applies MemoryScheduler.use_int4 (src/memopt/scheduler.py:15-18
 * documents the switch; no reference code performs it). The caller fills the
 * new storage (memopt_write_cache into INT4 pages, memopt_int4_pages_to_fp16
 * into fp16 pools) on the stream before using the pool. */
int memopt_pool_set_storage(int32_t kv_format, void *key_pool, void *value_pool);

/* Replaces allocate_block() — src/csrc/kv_cache.cu:163-172. *block_idx = -1
 * when exhausted (not an error). */
int memopt_allocate_block(int64_t *block_idx);

/* Replaces free_block(block_idx) — src/csrc/kv_cache.cu:179-185. */
int memopt_free_block(int64_t block_idx);

/* `count` calls of memopt_allocate_block / memopt_free_block as one, in the
 * same FIFO order (a prompt takes hundreds of pages at a time). All or none:
 * allocate leaves the list as it is and sets block_idx[0] = -1 when fewer
 * than `count` blocks are free; free checks every index first. */
int memopt_allocate_blocks(int64_t count, int64_t *block_idx);
int memopt_free_blocks(int64_t count, const int64_t *block_idx);

/* Replaces free_blocks_count() — src/csrc/kv_cache.cu:198-201. */
int memopt_free_blocks_count(int64_t *count);

/* Replaces write_cache(keys, values, block_tables, slot_mapping) —
 * src/csrc/kv_cache.cu:282-348. keys/values: fp16 [num_tokens, H, D]
 * contiguous; slot_mapping: int32 [num_tokens], slot = block*bs + pos.
 * FP16 pools get a scatter copy; INT4 pools get a fused group-64 quantize
 * into the page (codes bit-exact with memopt_quantize_kv_cache_int4, scales
 * stored as RNE fp16 of the fp32 scale, 9360 = RNE(65504/7) stored as 9352
 * so that 7 * scale stays finite). Slots outside the pool are skipped
 * on device; the caller validates them beforehand. */
int memopt_write_cache(const void *keys, const void *values, int64_t num_tokens,
                       int32_t num_heads, int32_t head_dim,
                       const int32_t *slot_mapping, void *stream);

/* Replaces evict_cache(block_tables, attention_scores, retain_ratio,
 * num_sink_tokens) — src/csrc/kv_cache.cu:379-559. scores: f32
 * [num_blocks, block_size, H]. Per (block, head): keep = max(1,
 * floor(r*bs)); rows scoring below the keep-th largest of the scores above
 * -1e38 (below -1e38 itself when fewer than keep exceed it) are zeroed: the
 * reference's selection with its -1e38 sentinel. Sinks ignored, as in the
 * reference. block_size up to 8192. */
int memopt_evict_cache(const float *attention_scores, int64_t num_blocks,
                       float retain_ratio, int32_t num_sink_tokens, void *stream);

/* Replaces evict_tokens(attention_scores, block_tables, is_block_free,
 * retain_ratio, num_sink_tokens) — src/csrc/kv_cache.cu:640-1156.
 * scores f32 [num_seqs, H, seq_len]; block_tables i32 [num_seqs, max_blocks]
 * (mutated); is_block_free i32 [total_pool_blocks] (mutated, caller zeroes).
 * Per (seq, head): sinks t < num_sink_tokens always kept; keep =
 * clamp(ceilf(r*L), 1, L); tokens scoring below the exact keep-th largest
 * (sink-boosted) score are evicted; their (token, head) rows are zeroed
 * (INT4: every group scale of the row set to 0, codes kept, so the row
 * dequantizes to zeros). A logical block with all block_size positions
 * evicted votes is_block_free[phys] += 1; the vote reaching H unlinks
 * block_tables[seq, lb] = -1. No seq_len cap (rows longer than 32768
 * tokens run as several workgroups per row). A physical page named by more
 * than one live entry of block_tables (shared between sequences) receives
 * the union of their evictions and no votes: it is never unlinked or
 * counted free by this call.
 * `workspace` is device scratch of at least memopt_evict_workspace_size
 * bytes, 16-byte aligned, of any content; nothing in it is kept between
 * calls. The call allocates no device memory. Calls sharing a workspace
 * must not overlap (nor may calls on one pool: they mutate it). */
int memopt_evict_tokens(const float *attention_scores, int32_t num_seqs,
                        int32_t num_heads, int32_t seq_len, int32_t *block_tables,
                        int32_t max_blocks_per_seq, int32_t *is_block_free,
                        int64_t total_pool_blocks, float retain_ratio,
                        int32_t num_sink_tokens, void *workspace,
                        int64_t workspace_bytes, void *stream);

/* Workspace bytes memopt_evict_tokens needs for these sizes: page marks for
 * total_pool_blocks pages plus, for seq_len > 32768, the long-row
 * selection state. No counterpart in the reference, whose kernels keep this
 * state in shared memory (it caps seq_len at 4096). */
int memopt_evict_workspace_size(int32_t num_seqs, int32_t num_heads, int32_t seq_len,
                                int32_t max_blocks_per_seq, int64_t total_pool_blocks,
                                int64_t *bytes);

/* ------------------------------------------------------------------------ */
/* Quantization (surface, whole-tensor)                                     */
/* ------------------------------------------------------------------------ */

/* Replaces quantize_kv_cache_int4(cache, group_size) —
 * src/csrc/quantization.cu:104-203, :294-353. cache: fp16, numel elements,
 * contiguous; packed_out: u8 [numel/2]; scales_out: f32 [numel/64].
 * scale = absmax>0 ? absmax/7 : 1 (IEEE fp32); code = clamp(roundf(v/scale)
 * + 8, 0, 15); byte = code[2i] | code[2i+1] << 4. */
int memopt_quantize_kv_cache_int4(const void *cache, int64_t numel, int64_t last_dim,
                                  int32_t group_size, uint8_t *packed_out,
                                  float *scales_out, void *stream);

/* Replaces dequantize_kv_cache_int4(q_cache, scales, group_size) —
 * src/csrc/quantization.cu:232-270, :371-428. out: fp16 [2*packed_numel],
 * value = fp16(RNE(float(code-8) * scale)). */
int memopt_dequantize_kv_cache_int4(const uint8_t *packed, int64_t packed_numel,
                                    const float *scales, int64_t num_scales,
                                    int32_t group_size, void *out, void *stream);

/* Dequantizes an INT4 page pool [num_blocks, H, B] into fp16 pools
 * key_out/value_out [num_blocks, 16, H, D]: value = fp16(RN(float(code-8) *
 * page scale)), the dequantize_kv_cache_int4 arithmetic of
 * src/csrc/quantization.cu:232-270 applied to this build's page layout
 * (fp16 page scales). head_dim 64 or 128. */
int memopt_int4_pages_to_fp16(const uint8_t *pages, int64_t num_blocks, int32_t num_heads,
                              int32_t head_dim, void *key_out, void *value_out, void *stream);

/* ------------------------------------------------------------------------ */
/* Paged attention                                                          */
/* ------------------------------------------------------------------------ */

/* Replaces dynamic_sparse_attention(query, key_cache, value_cache,
 * block_tables, context_lens, max_seq_len, window_size) —
 * src/csrc/attention.cu:98-339, :371-521 — with reference semantics:
 * non-causal, keys j in [max(0, ctx-W), ctx) for every query, pages with
 * block_tables < 0 skipped, W <= 0 or W > max_seq_len -> max_seq_len,
 * scale 1/sqrtf(D), empty key set -> 0. fp16 pool [nb, bs, H, D]. */
int memopt_dynamic_sparse_attention(const void *query, int32_t batch, int32_t q_len,
                                    int32_t num_heads, int32_t head_dim,
                                    const void *key_cache, const void *value_cache,
                                    int64_t num_kv_blocks, int32_t block_size,
                                    const int32_t *block_tables,
                                    int32_t max_blocks_per_seq,
                                    const int32_t *context_lens, int32_t max_seq_len,
                                    int32_t window_size, void *out, void *stream);

/* Extended paged attention: the reference semantics above plus
 *   - INT4 caches — the INT4 page pool, or reference-order codes with
 *     f32/f16 group-64 scales and arbitrary page/head/token strides —
 *     dequantized just in time; replaces the reference's
 *     dequantize_kv_cache_int4 -> dynamic_sparse_attention composition;
 *   - attention sinks (keys j < num_sink_tokens always visible, the token
 *     rule of src/memopt/triton_attention.py:523-532);
 *   - causal mode (query i at absolute position ctx-q_len+i sees
 *     j <= pos && (j < sinks || j >= pos-W+1), scripts/bench_accuracy.py:253-280).
 * With num_sink_tokens == 0, causal == 0 and an fp16 cache it computes the
 * same function as memopt_dynamic_sparse_attention.
 * `workspace` (device, >= memopt_attention_workspace_size bytes) holds the
 * decode's split-K partials and arrival counters, or a multi-query call's
 * staged K/V and staging flags or split partials; it may be NULL when that
 * size is 0 (and for multi-query calls that attend straight from the cache,
 * which then run unsplit). A decode
 * (q_len == 1) workspace must be zero before its first use; later calls may
 * reuse it without clearing (each call's counters carry the call's id, so
 * what an earlier call left is never taken for its own). A multi-query
 * workspace may hold anything (the call clears its flags itself). */
typedef struct memopt_attn_desc {
  const void *query;          /* fp16 [batch, q_len, H, D] contiguous        */
  void *out;                  /* fp16 [batch, q_len, H, D] contiguous        */
  int32_t batch, q_len, num_heads, head_dim;
  int32_t kv_format;          /* MEMOPT_KV_FP16 / _INT4 (page pool) / _INT4_ROWS */
  const void *key_cache;      /* fp16 elements, INT4 page buffer, or u8 codes */
  const void *value_cache;    /* unused for MEMOPT_KV_INT4                   */
  const void *key_scales;     /* MEMOPT_KV_INT4_ROWS only                    */
  const void *value_scales;
  int32_t scale_dtype;        /* MEMOPT_SCALE_F32 / MEMOPT_SCALE_F16 (ROWS)  */
  int32_t block_size;         /* tokens per page                             */
  int64_t num_kv_blocks;
  /* Strides (FP16 / INT4_ROWS only; derived for INT4 pages): fp16 cache in
   * elements, INT4 codes in bytes, scales in elements. */
  int64_t kv_page_stride, kv_head_stride, kv_token_stride;
  int64_t sc_page_stride, sc_head_stride, sc_token_stride;
  const int32_t *block_tables; /* [batch, max_blocks_per_seq]                */
  int32_t max_blocks_per_seq;
  const int32_t *context_lens; /* [batch]                                    */
  int32_t max_seq_len, window_size, num_sink_tokens, causal;
  void *workspace;
  int64_t workspace_bytes;
} memopt_attn_desc;

int memopt_attention_workspace_size(const memopt_attn_desc *desc, int64_t *bytes);
/* `workspace` must hold at least memopt_attention_workspace_size bytes;
 * a smaller one is an error (MEMOPT_ERR_INVALID). Only
 * memopt_dynamic_sparse_attention, whose reference signature has no
 * workspace, runs a decode that would split unsplit instead. */
int memopt_paged_attention(const memopt_attn_desc *desc, void *stream);

/* Bytes of the per-GPU static scratch of memopt_paged_attention_noalloc. */
#define MEMOPT_NOALLOC_SCRATCH_BYTES (4LL << 20)

/* No counterpart in the reference. For callers that cannot allocate device
 * memory: code under HIP graph capture, tight serving loops, harnesses that
 * forbid hipMalloc. Computes what memopt_paged_attention computes for the
 * same descriptor (desc->workspace is ignored) and allocates nothing: the
 * decode kernels' split-K partials, and the staged K/V of a multi-query call
 * when they fit, live in a static device array of
 * MEMOPT_NOALLOC_SCRATCH_BYTES (4 MiB) per GPU, held until the process ends;
 * its last 64 KiB hold the decode's arrival counters (zero at load, then
 * only ever counters) and the rest the partials or staged K/V.
 * Results are bit-identical to memopt_paged_attention's except for
 * multi-query calls whose staged K/V or split partials do not fit: those run
 * the in-kernel staging kernel, or fewer splits, and agree with the other to
 * within fp16 attention tolerance, not bit for bit. A decode whose partials exceed the rest
 * (B * H * splits * (head_dim + 2) * 4 + 8 * B * H bytes; splits grow only
 * while B * H is below two workgroups per CU) returns MEMOPT_ERR_INVALID. Every call on
 * a GPU shares that GPU's array, so calls that overlap on one GPU (other
 * streams or host threads) race: the caller serializes them. The first call
 * on each device resolves the array's device address there. */
int memopt_paged_attention_noalloc(const memopt_attn_desc *desc, void *stream);

/* Diagnostics, no counterpart in the reference: the path that multi-query
 * calls of the calling thread over INT4 pages and fp16 pools take (workspace
 * query included). Both compute the same function; AUTO, the default, takes
 * the one estimated to be faster. The others are for tests and measurements
 * that need one of them at any size. */
#define MEMOPT_PATH_AUTO   0
#define MEMOPT_PATH_STAGED 1  /* K and V staged as fp16, then attended (csrc/prefill.hip) */
#define MEMOPT_PATH_DIRECT 2  /* attended straight from the cache (csrc/direct.hip)       */
int memopt_multi_query_path(int32_t path);

/* ------------------------------------------------------------------------ */
/* Packed batches: grouped heads, sequences of different lengths            */
/* ------------------------------------------------------------------------ */
/* No counterparts in the reference, whose attention takes one query head per
 * cached head and the same number of queries from every sequence, and whose
 * callers build block tables and slots on the host.
 *
 * A packed tensor holds the rows of `batch` sequences one behind the other:
 * query_starts (int32 [batch + 1], device, ascending from >= 0 to <= tokens)
 * gives sequence b the rows query_starts[b] .. query_starts[b + 1] - 1.
 * Entries outside [0, tokens] are clamped; rows of no sequence are neither
 * read nor written. Query head h reads key head h / (num_heads /
 * num_kv_heads). Strides are in elements; a row's head_dim elements are
 * contiguous, rows are 16-byte aligned. */

/* Element types of memopt_prompt_desc. */
#define MEMOPT_FP16 0
#define MEMOPT_BF16 1

/* Causal attention over whole prompts from q, k and v as a layer's
 * projections leave them (views of a fused projection included): row i of a
 * sequence sees its rows j <= i with j < num_sink_tokens or j > i -
 * window_size (window_size <= 0: all j <= i), scale 1/sqrt(head_dim).
 * Elements of hidden rows never reach a result, inf and NaN included (bf16
 * values from 2^112 on may overflow the sums).
 * head_dim 64 or 128; key and value token strides from head_dim to 2^23 - 1.
 * `out` must not overlap the inputs. */
typedef struct memopt_prompt_desc {
  const void *query, *key, *value;   /* [tokens, heads, head_dim]              */
  void *out;                         /* [tokens, num_heads, head_dim]          */
  int32_t dtype;                     /* MEMOPT_FP16 / MEMOPT_BF16              */
  int32_t tokens, batch, num_heads, num_kv_heads, head_dim;
  int64_t q_token_stride, q_head_stride, k_token_stride, k_head_stride;
  int64_t v_token_stride, v_head_stride, o_token_stride, o_head_stride;
  const int32_t *query_starts;
  int32_t window_size, num_sink_tokens;
} memopt_prompt_desc;
int memopt_prompt_attention(const memopt_prompt_desc *desc, void *stream);

/* Attention of packed queries over a paged cache: sequence b's rows are the
 * last positions of its context_lens[b] tokens (row i of n at position
 * context_lens[b] - n + i), and see what the causal rule of
 * memopt_paged_attention shows them (window, sinks, unlinked pages skipped,
 * window_size <= 0 or > max_seq_len: max_seq_len; a row that sees nothing
 * gives 0). Sequences may bring different numbers of rows, none included.
 * Caches: MEMOPT_KV_INT4 page buffers (key_cache; value_cache unused) and
 * contiguous MEMOPT_KV_FP16 pools with block_size a multiple of 16, both with
 * num_kv_heads heads; head_dim 64 or 128; INT4 values are (code - 8) * scale.
 * max_query_len bounds the rows of any one sequence (rows past it may be left
 * unwritten). Block tables hold up to 2^30 tokens. */
typedef struct memopt_packed_desc {
  const void *query;                 /* fp16 [tokens, num_heads, head_dim]     */
  void *out;                         /* fp16 [tokens, num_heads, head_dim]     */
  int32_t tokens, batch, num_heads, num_kv_heads, head_dim;
  int64_t q_token_stride, q_head_stride, o_token_stride, o_head_stride;
  int32_t kv_format;                 /* MEMOPT_KV_FP16 / MEMOPT_KV_INT4        */
  const void *key_cache, *value_cache;
  int32_t block_size;
  int64_t num_kv_blocks;
  const int32_t *block_tables;       /* [batch, max_blocks_per_seq]            */
  int32_t max_blocks_per_seq;
  const int32_t *context_lens;       /* [batch]                                */
  const int32_t *query_starts;       /* [batch + 1]                            */
  int32_t max_query_len, max_seq_len, window_size, num_sink_tokens;
  void *workspace;                   /* >= memopt_packed_workspace_size bytes, 16-byte aligned */
  int64_t workspace_bytes;
} memopt_packed_desc;
/* The workspace's first `zeroed` bytes (arrival counters) must be zero before
 * its first use; every call leaves them zero. The rest may hold anything.
 * Calls sharing a workspace must not overlap. */
int memopt_packed_workspace_size(const memopt_packed_desc *desc, int64_t *bytes, int64_t *zeroed);
int memopt_packed_attention(const memopt_packed_desc *desc, void *stream);

/* The index tensors of a batch's next step, built on the device. Request b
 * holds context_lens[b] tokens in the pages of its block table row and asks
 * for new_tokens[b] more. Free pages are a ring: free_pages[(free_span[0] +
 * i) % num_free_pages] for i < free_span[1], taken from the front in request
 * order (the FIFO order of memopt_allocate_block). Requests are served in
 * order while the sums of what the valid requests so far ask for stay within
 * the free pages and num_rows (one that needs no page is not refused for
 * pages). Written: the new entries of block_tables; context_lens_out and
 * free_span_out (which may be the inputs); query_starts [num_requests + 1];
 * slots and positions [num_rows], request by request, -1 behind the last row
 * (memopt_write_cache skips those); status [num_requests]: */
#define MEMOPT_STEP_SERVED   0
#define MEMOPT_STEP_INVALID  1  /* a negative count, or more tokens than the table's row holds */
#define MEMOPT_STEP_UNLINKED 2  /* the page that holds its last token was evicted               */
#define MEMOPT_STEP_NO_PAGES 3
#define MEMOPT_STEP_NO_ROWS  4
/* A request that is not served stays as it was and gets no rows. At most 4096
 * requests; calls on one batch must not overlap. */
typedef struct memopt_advance_desc {
  const int32_t *new_tokens, *context_lens;  /* [num_requests]                 */
  int32_t *block_tables;                     /* [num_requests, max_blocks_per_seq] */
  const int32_t *free_pages, *free_span;     /* [num_free_pages], [2]          */
  int32_t *context_lens_out, *free_span_out, *query_starts, *slots, *positions, *status;
  int32_t num_requests, max_blocks_per_seq, num_free_pages, block_size, num_rows;
} memopt_advance_desc;
int memopt_advance_batch(const memopt_advance_desc *desc, void *stream);

/* Attention weights per cached token: out[b, h, j] = scores[b, h, j] + the sum
 * of the softmax weights that sequence b's query rows, in the num_heads /
 * num_kv_heads heads of key head h, give token j; the rows, masks and caches
 * are memopt_packed_attention's, and a row that sees nothing adds nothing. The
 * order of all sums is fixed. Tokens from max_seq_len on are not looked at;
 * weights of tokens from scores_len on are not written. `scores` may be null
 * (zeros) or `out` itself, else the two must not overlap. Query rows: 31 token strides and a group's head
 * strides together less than 2^29 elements. */
typedef struct memopt_scores_desc {
  const void *query;                 /* fp16 [tokens, num_heads, head_dim]     */
  const float *scores;               /* [batch, num_kv_heads, scores_len]      */
  float *out;                        /* the same                               */
  int32_t tokens, batch, num_heads, num_kv_heads, head_dim;
  int64_t q_token_stride, q_head_stride;
  int32_t kv_format;                 /* MEMOPT_KV_FP16 / MEMOPT_KV_INT4        */
  const void *key_cache;             /* fp16 keys, or INT4 pages               */
  int32_t block_size;
  int64_t num_kv_blocks;
  const int32_t *block_tables;       /* [batch, max_blocks_per_seq]            */
  int32_t max_blocks_per_seq;
  const int32_t *context_lens;       /* [batch]                                */
  const int32_t *query_starts;       /* [batch + 1]                            */
  int32_t max_query_len, max_seq_len, window_size, num_sink_tokens, scores_len;
  void *workspace;                   /* >= memopt_scores_workspace_size bytes, 16-byte aligned, any content */
  int64_t workspace_bytes;
} memopt_scores_desc;
/* Calls sharing a workspace must not overlap. */
int memopt_scores_workspace_size(const memopt_scores_desc *desc, int64_t *bytes);
int memopt_attention_scores(const memopt_scores_desc *desc, void *stream);

/* Tokens of least weight leave the cache. Of request b's context_lens[b]
 * tokens, n = min(keep[b], those whose pages are linked) stay in every key
 * head: the first num_sink_tokens, the last num_recent_tokens (as far as n
 * reaches, the sinks first), and of the others those with the largest
 * scores[b, h] (ties: the first; NaN counts as the lowest). They keep their
 * order and become tokens 0 .. n - 1: their rows are copied, bit for bit, into
 * fresh pages from the front of the ring of free pages (memopt_advance_batch),
 * and the old linked pages go to its end, both in request order. Nothing else
 * of the cache changes, rows of the fresh pages behind token n - 1 included.
 *
 * Written for every request: block_tables_out (the fresh pages, -1 behind),
 * context_lens_out, scores_out (the kept tokens' scores, 0 behind), kept (old
 * positions, -1 behind), status; a request that is not compacted keeps its
 * tables, length and scores, and its `kept` are -1. free_span_out may be
 * free_span; apart from that results must not overlap the inputs, nor each
 * other. At most 4096 requests; calls on one batch must not overlap. Status: */
#define MEMOPT_COMPACT_DONE     0
#define MEMOPT_COMPACT_INVALID  1  /* a length past the table or scores_len, or keep past max_keep  */
#define MEMOPT_COMPACT_LEFT     2  /* it may keep all it has (negative keep: always)                */
#define MEMOPT_COMPACT_NO_PAGES 3  /* the free pages, or the ring's room for the old ones, did not  */
                                   /* last (sums over all that ask so far, as in advance_batch);    */
                                   /* pages that this call gives back serve the next one            */
#define MEMOPT_COMPACT_SHARED   4  /* one of its pages is listed twice in this call's contexts,     */
                                   /* those of invalid requests that fit their tables among them    */
typedef struct memopt_compact_desc {
  const float *scores;               /* [num_requests, num_kv_heads, scores_len] */
  float *scores_out;                 /* the same                               */
  int32_t *kept;                     /* [num_requests, num_kv_heads, max_keep] */
  int32_t kv_format;                 /* MEMOPT_KV_FP16 / MEMOPT_KV_INT4        */
  void *key_cache, *value_cache;     /* (value_cache unused for INT4 pages)    */
  int64_t num_kv_blocks;
  const int32_t *block_tables, *context_lens, *keep;
  int32_t *block_tables_out, *context_lens_out, *status;
  int32_t *free_pages;               /* [num_free_pages]; written at the end of the span */
  const int32_t *free_span;
  int32_t *free_span_out;
  int32_t num_requests, num_kv_heads, head_dim, max_blocks_per_seq, block_size, num_free_pages, scores_len, max_keep;
  int32_t num_sink_tokens, num_recent_tokens;
  void *workspace;                   /* >= memopt_compact_workspace_size bytes, 16-byte aligned, any content */
  int64_t workspace_bytes;
} memopt_compact_desc;
/* Calls sharing a workspace must not overlap. */
int memopt_compact_workspace_size(const memopt_compact_desc *desc, int64_t *bytes);
int memopt_compact_cache(const memopt_compact_desc *desc, void *stream);

/* Attention over a paged cache of one vector per token for all heads (latent
 * attention, absorbed form): cache [num_kv_blocks, block_size, rank +
 * rope_dim], contiguous; keys are its whole rows, values their first `rank`
 * elements:
 *   out[t, h] = sum_j softmax_j(scale query[t, h] . cache_j) cache_j[: rank]
 * Packed rows, positions, windows, sinks, unlinked pages and rows that see
 * nothing are memopt_packed_attention's. Elements of hidden tokens never reach
 * a result, inf and NaN included. Tokens from max_seq_len on are not looked
 * at; rows past max_query_len of a sequence may be left unwritten. dtype is
 * that of query, cache and out; rank 128, 256 or 512, rope_dim 32 or 64,
 * block_size a multiple of 16. */
typedef struct memopt_latent_desc {
  const void *query;                 /* [tokens, num_heads, rank + rope_dim]   */
  const void *cache;
  void *out;                         /* [tokens, num_heads, rank]              */
  int32_t dtype;                     /* MEMOPT_FP16 / MEMOPT_BF16              */
  int32_t tokens, batch, num_heads, rank, rope_dim;
  int64_t q_token_stride, q_head_stride, o_token_stride, o_head_stride;
  int32_t block_size;
  int64_t num_kv_blocks;
  const int32_t *block_tables;       /* [batch, max_blocks_per_seq]            */
  int32_t max_blocks_per_seq;
  const int32_t *context_lens;       /* [batch]                                */
  const int32_t *query_starts;       /* [batch + 1]                            */
  int32_t max_query_len, max_seq_len, window_size, num_sink_tokens;
  float scale;
  void *workspace;                   /* >= memopt_latent_workspace_size bytes, 16-byte aligned, any content */
  int64_t workspace_bytes;
} memopt_latent_desc;
/* Calls sharing a workspace must not overlap. */
int memopt_latent_workspace_size(const memopt_latent_desc *desc, int64_t *bytes);
int memopt_latent_attention(const memopt_latent_desc *desc, void *stream);

/* Rows of the latent cache from their two parts: token t's latents [rank] and
 * rotary keys [rope_dim] (16-bit elements, strides in elements, rows 16-byte
 * aligned) go to row slots[t] of the cache's num_slots; slots outside are
 * skipped. Two tokens of one slot: either's elements. */
int memopt_write_latent(const void *latents, int64_t latent_stride, const void *rope_keys, int64_t rope_stride,
                        int32_t num_tokens, int32_t rank, int32_t rope_dim, const int32_t *slots, void *cache,
                        int64_t num_slots, void *stream);

/* Causal attention over whole packed prompts with keys of two parts, one per
 * head and a rotary one shared by all heads (latent attention, expanded form):
 *   score = scale (query[.. : head_dim] . key + query[head_dim ..] . rope_key)
 * with values of head_dim elements. Rows, masks, strides and hidden elements
 * as in memopt_prompt_attention; every head has keys and values of its own.
 * head_dim 64 or 128, rope_dim 32 or 64. `out` must not overlap the inputs. */
typedef struct memopt_latent_prompt_desc {
  const void *query;                 /* [tokens, num_heads, head_dim + rope_dim] */
  const void *key;                   /* [tokens, num_heads, head_dim]          */
  const void *rope_key;              /* [tokens, rope_dim]                     */
  const void *value;                 /* [tokens, num_heads, head_dim]          */
  void *out;                         /* [tokens, num_heads, head_dim]          */
  int32_t dtype;                     /* MEMOPT_FP16 / MEMOPT_BF16              */
  int32_t tokens, batch, num_heads, head_dim, rope_dim;
  int64_t q_token_stride, q_head_stride, k_token_stride, k_head_stride, r_token_stride;
  int64_t v_token_stride, v_head_stride, o_token_stride, o_head_stride;
  const int32_t *query_starts;
  int32_t window_size, num_sink_tokens;
  float scale;
} memopt_latent_prompt_desc;
int memopt_latent_prompt_attention(const memopt_latent_prompt_desc *desc, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* MEMOPT_HIP_H */
