/*
 * flexengine_amd_span.h -- attention over long contexts: a KV cache held in 4 bits, and a
 * sliding window with sinks (same library, conventions and return codes as flexengine_amd.h).
 *
 * Window.  A query at position p of its sequence sees the keys j <= p with p - j < window, and
 * the sequence's first `sinks` keys whatever the distance.  window 0: every key j <= p (the
 * 4-bit forms; the _window forms take window >= 1), sinks then has no effect.  Pages that no
 * query of the call sees, and their table entries, are not read and may hold anything, as may
 * keys of other pages that none sees.  The prefill forms compute up to 128 (fp32: 16; long 4-bit
 * prompts: 256) rows of a sequence together: a V that is infinite or NaN and seen by one of them
 * makes NaN of the others too (0 * inf).
 *
 * 4-bit pools.  A row of one token and KV head is cut into blocks of 32 dims: 32 e2m1 codes (0,
 * 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives) with one e8m0 scale byte s, values code *
 * 2^(s - 127).  Per pool (K and V alike):
 *   codes   uint8 [num_blocks, kv_heads, block_size, head_dim / 2], 16-byte aligned; dim 2i in
 *           the low half of byte i
 *   scales  uint8 [num_blocks, kv_heads, block_size, head_dim / 32]
 * The _strided forms take the same dims in any order and with gaps between rows (fe_kv4_strides).
 * A write takes the smallest power of two 2^e with max|x| <= 7 * 2^e, -23 <= e <= 13 (fp16
 * rows) or 125 (bf16 rows), and rounds to the nearest code, ties to the even one.  Every value
 * is exact in the rows' type.  fp16 magnitudes above 49152 are held as 49152, a block (of either
 * type) whose largest magnitude is at most 2^-25 as zeros; one with an infinity or a NaN as NaN.  Two rows of one call in the same slot leave it undefined.
 *
 * Shapes: block_size a power of two, of at least 16 for attention; head_dim a multiple of 32 up
 * to 256 (4-bit), a multiple of 8 up to 256 (fp16, bf16 windows) or up to 128 (fp32 windows);
 * tables of up to 262144 tokens (decode); any number of query heads per KV head (above 16 the
 * decode attends them in groups, each reading K and V), batch * kv_heads * groups up to 65536
 * there.  No plans, and no shared-prefix form.
 */
#ifndef FLEXENGINE_AMD_SPAN_H
#define FLEXENGINE_AMD_SPAN_H

#include "flexengine_amd.h"

#ifdef __cplusplus
extern "C" {
#endif

/*
 * Where the rows of 4-bit pools are: bytes between blocks, KV heads and tokens, of the codes
 * (multiples of 16) and of the scales; K's and V's alike.  The bytes of a row are side by side
 * and rows lie apart: each stride is at least what the smaller ones span (else
 * FE_ERR_INVALID_ARGUMENT); block strides below 2^36 and 2^32, token strides below 2^26.  The
 * stride of a dim of size 1 counts for nothing.  Null: the layout above.
 */
typedef struct {
  int64_t codes[3];
  int64_t scales[3];
} fe_kv4_strides;

/*
 * Page writes into 4-bit pools: fe_write_kv, fe_write_kv_decode and fe_write_kv_ragged
 * (flexengine_amd.h) with the same slot maps, from fp16 (or _bf16) rows.  Rows whose slot,
 * page or block is out of range are skipped.
 */
int fe_write_kv4(const void* k_new, const void* v_new, int64_t new_token_stride, void* k_codes,
                 void* k_scales, void* v_codes, void* v_scales, int num_blocks,
                 const int32_t* slot_block, const int32_t* slot_offset, int num_tokens,
                 int kv_heads, int head_dim, int block_size, fe_stream_t stream);
int fe_write_kv4_bf16(const void* k_new, const void* v_new, int64_t new_token_stride,
                      void* k_codes, void* k_scales, void* v_codes, void* v_scales,
                      int num_blocks, const int32_t* slot_block, const int32_t* slot_offset,
                      int num_tokens, int kv_heads, int head_dim, int block_size,
                      fe_stream_t stream);
int fe_write_kv4_decode(const void* k_new, const void* v_new, int64_t new_batch_stride,
                        void* k_codes, void* k_scales, void* v_codes, void* v_scales,
                        int num_blocks, const int32_t* block_tables, int table_stride,
                        const int32_t* context_lens, int batch, int kv_heads, int head_dim,
                        int block_size, fe_stream_t stream);
int fe_write_kv4_decode_bf16(const void* k_new, const void* v_new, int64_t new_batch_stride,
                             void* k_codes, void* k_scales, void* v_codes, void* v_scales,
                             int num_blocks, const int32_t* block_tables, int table_stride,
                             const int32_t* context_lens, int batch, int kv_heads, int head_dim,
                             int block_size, fe_stream_t stream);
int fe_write_kv4_ragged(const void* k_new, const void* v_new, int64_t new_token_stride,
                        void* k_codes, void* k_scales, void* v_codes, void* v_scales,
                        int num_blocks, const int32_t* block_tables, int table_stride,
                        const int32_t* q_offsets, const int32_t* context_lens, int num_seqs,
                        int total_tokens, int kv_heads, int head_dim, int block_size,
                        fe_stream_t stream);
int fe_write_kv4_ragged_bf16(const void* k_new, const void* v_new, int64_t new_token_stride,
                             void* k_codes, void* k_scales, void* v_codes, void* v_scales,
                             int num_blocks, const int32_t* block_tables, int table_stride,
                             const int32_t* q_offsets, const int32_t* context_lens, int num_seqs,
                             int total_tokens, int kv_heads, int head_dim, int block_size,
                             fe_stream_t stream);

/* fe_gather_kv from 4-bit pools: the rows' values in fp16 (or bfloat16), exact. */
int fe_gather_kv4(const void* k_codes, const void* k_scales, const void* v_codes,
                  const void* v_scales, int num_blocks, const int32_t* block_tables,
                  int table_stride, const int32_t* context_lens, const int32_t* out_offsets,
                  void* k_out, void* v_out, int batch, int total_tokens, int kv_heads,
                  int head_dim, int block_size, fe_stream_t stream);
int fe_gather_kv4_bf16(const void* k_codes, const void* k_scales, const void* v_codes,
                       const void* v_scales, int num_blocks, const int32_t* block_tables,
                       int table_stride, const int32_t* context_lens, const int32_t* out_offsets,
                       void* k_out, void* v_out, int batch, int total_tokens, int kv_heads,
                       int head_dim, int block_size, fe_stream_t stream);

/*
 * Workspace bytes of the decode forms below (zero-filled before its first use; every call
 * leaves it ready for the next; calls that overlap in time need separate ones).  max_context =
 * table_stride * block_size.
 */
size_t fe_span_decode_workspace_size(int batch, int num_q_heads, int kv_heads, int head_dim,
                                     int max_context, int target_splits);

/*
 * fe_paged_decode (flexengine_amd.h) under a window with sinks: the same arguments, page write
 * of k_new / v_new and zero rows, with a workspace of fe_span_decode_workspace_size.
 */
int fe_paged_decode_window(const void* q, int64_t q_batch_stride, void* out, const void* k_new,
                           const void* v_new, int64_t new_batch_stride, void* k_pool,
                           void* v_pool, int num_blocks, const int32_t* block_tables,
                           int table_stride, const int32_t* context_lens, void* workspace,
                           size_t workspace_bytes, int batch, int num_q_heads, int kv_heads,
                           int head_dim, int block_size, float scale, int window, int sinks,
                           int target_splits, fe_stream_t stream);
int fe_paged_decode_window_bf16(const void* q, int64_t q_batch_stride, void* out,
                                const void* k_new, const void* v_new, int64_t new_batch_stride,
                                void* k_pool, void* v_pool, int num_blocks,
                                const int32_t* block_tables, int table_stride,
                                const int32_t* context_lens, void* workspace,
                                size_t workspace_bytes, int batch, int num_q_heads, int kv_heads,
                                int head_dim, int block_size, float scale, int window, int sinks,
                                int target_splits, fe_stream_t stream);
int fe_paged_decode_window_f32(const void* q, int64_t q_batch_stride, void* out,
                               const void* k_new, const void* v_new, int64_t new_batch_stride,
                               void* k_pool, void* v_pool, int num_blocks,
                               const int32_t* block_tables, int table_stride,
                               const int32_t* context_lens, void* workspace,
                               size_t workspace_bytes, int batch, int num_q_heads, int kv_heads,
                               int head_dim, int block_size, float scale, int window, int sinks,
                               int target_splits, fe_stream_t stream);

/*
 * The same over 4-bit pools (q, out, k_new and v_new in fp16 or bfloat16; window 0: all keys).
 * With k_new and v_new the new rows are written in 4 bits and attended as written.
 */
int fe_paged_decode_kv4(const void* q, int64_t q_batch_stride, void* out, const void* k_new,
                        const void* v_new, int64_t new_batch_stride, void* k_codes,
                        void* k_scales, void* v_codes, void* v_scales, int num_blocks,
                        const int32_t* block_tables, int table_stride,
                        const int32_t* context_lens, void* workspace, size_t workspace_bytes,
                        int batch, int num_q_heads, int kv_heads, int head_dim, int block_size,
                        float scale, int window, int sinks, int target_splits,
                        fe_stream_t stream);
int fe_paged_decode_kv4_bf16(const void* q, int64_t q_batch_stride, void* out, const void* k_new,
                             const void* v_new, int64_t new_batch_stride, void* k_codes,
                             void* k_scales, void* v_codes, void* v_scales, int num_blocks,
                             const int32_t* block_tables, int table_stride,
                             const int32_t* context_lens, void* workspace,
                             size_t workspace_bytes, int batch, int num_q_heads, int kv_heads,
                             int head_dim, int block_size, float scale, int window, int sinks,
                             int target_splits, fe_stream_t stream);

/* Workspace bytes of the prefill forms below (the decode's rules). */
size_t fe_span_prefill_workspace_size(int num_seqs, int total_q, int num_q_heads, int kv_heads,
                                      int head_dim);

/*
 * Rows (query heads of a KV head times positions) of a sequence that a prefill of these sizes
 * computes together: 16 (elem_bytes 4), 128, or 256 (long prompts over 4-bit pools, kv4 != 0); a
 * negative FE_ERR_* code for bad sizes.  Launches nothing; for tests and profiles.
 */
int fe_span_prefill_rows(int num_seqs, int total_q, int num_q_heads, int kv_heads, int head_dim,
                         int window, int kv4, int elem_bytes);

/*
 * fe_prefill_paged (flexengine_amd.h) under a window with sinks: the same rows, tables and
 * offsets, scale > 0.  A context past what the table addresses ends there; one of fewer tokens than
 * its rows counts as just those rows.  No page past the table's last entry is read for it.
 */
int fe_prefill_paged_window(const void* q, void* out, const void* k_pool, const void* v_pool,
                            int num_blocks, const int32_t* block_tables, int table_stride,
                            const int32_t* q_offsets, const int32_t* context_lens, int num_seqs,
                            int total_q, int num_q_heads, int kv_heads, int head_dim,
                            int block_size, float scale, int window, int sinks, void* workspace,
                            size_t workspace_bytes, fe_stream_t stream);
int fe_prefill_paged_window_bf16(const void* q, void* out, const void* k_pool,
                                 const void* v_pool, int num_blocks, const int32_t* block_tables,
                                 int table_stride, const int32_t* q_offsets,
                                 const int32_t* context_lens, int num_seqs, int total_q,
                                 int num_q_heads, int kv_heads, int head_dim, int block_size,
                                 float scale, int window, int sinks, void* workspace,
                                 size_t workspace_bytes, fe_stream_t stream);
int fe_prefill_paged_window_f32(const void* q, void* out, const void* k_pool, const void* v_pool,
                                int num_blocks, const int32_t* block_tables, int table_stride,
                                const int32_t* q_offsets, const int32_t* context_lens,
                                int num_seqs, int total_q, int num_q_heads, int kv_heads,
                                int head_dim, int block_size, float scale, int window, int sinks,
                                void* workspace, size_t workspace_bytes, fe_stream_t stream);

/* The same over 4-bit pools (q and out in fp16 or bfloat16; window 0: all keys). */
int fe_prefill_paged_kv4(const void* q, void* out, const void* k_codes, const void* k_scales,
                         const void* v_codes, const void* v_scales, int num_blocks,
                         const int32_t* block_tables, int table_stride, const int32_t* q_offsets,
                         const int32_t* context_lens, int num_seqs, int total_q, int num_q_heads,
                         int kv_heads, int head_dim, int block_size, float scale, int window,
                         int sinks, void* workspace, size_t workspace_bytes, fe_stream_t stream);
int fe_prefill_paged_kv4_bf16(const void* q, void* out, const void* k_codes,
                              const void* k_scales, const void* v_codes, const void* v_scales,
                              int num_blocks, const int32_t* block_tables, int table_stride,
                              const int32_t* q_offsets, const int32_t* context_lens, int num_seqs,
                              int total_q, int num_q_heads, int kv_heads, int head_dim,
                              int block_size, float scale, int window, int sinks, void* workspace,
                              size_t workspace_bytes, fe_stream_t stream);

/*
 * The forms above of 4-bit pools with strides of their own (null: those forms).  Reads cost least
 * where the rows of a head are side by side, as in the layout above: at head_dim 128 two rows of
 * neighbouring heads that are side by side share a cache line that both heads' reads fetch.
 */
int fe_write_kv4_strided(const void* k_new, const void* v_new, int64_t new_token_stride,
                         void* k_codes, void* k_scales, void* v_codes, void* v_scales,
                         const fe_kv4_strides* strides, int num_blocks, const int32_t* slot_block,
                         const int32_t* slot_offset, int num_tokens, int kv_heads, int head_dim,
                         int block_size, fe_stream_t stream);
int fe_write_kv4_strided_bf16(const void* k_new, const void* v_new, int64_t new_token_stride,
                              void* k_codes, void* k_scales, void* v_codes, void* v_scales,
                              const fe_kv4_strides* strides, int num_blocks,
                              const int32_t* slot_block, const int32_t* slot_offset, int num_tokens,
                              int kv_heads, int head_dim, int block_size, fe_stream_t stream);
int fe_write_kv4_decode_strided(const void* k_new, const void* v_new, int64_t new_batch_stride,
                                void* k_codes, void* k_scales, void* v_codes, void* v_scales,
                                const fe_kv4_strides* strides, int num_blocks,
                                const int32_t* block_tables, int table_stride,
                                const int32_t* context_lens, int batch, int kv_heads, int head_dim,
                                int block_size, fe_stream_t stream);
int fe_write_kv4_decode_strided_bf16(const void* k_new, const void* v_new, int64_t new_batch_stride,
                                     void* k_codes, void* k_scales, void* v_codes, void* v_scales,
                                     const fe_kv4_strides* strides, int num_blocks,
                                     const int32_t* block_tables, int table_stride,
                                     const int32_t* context_lens, int batch, int kv_heads,
                                     int head_dim, int block_size, fe_stream_t stream);
int fe_write_kv4_ragged_strided(const void* k_new, const void* v_new, int64_t new_token_stride,
                                void* k_codes, void* k_scales, void* v_codes, void* v_scales,
                                const fe_kv4_strides* strides, int num_blocks,
                                const int32_t* block_tables, int table_stride,
                                const int32_t* q_offsets, const int32_t* context_lens, int num_seqs,
                                int total_tokens, int kv_heads, int head_dim, int block_size,
                                fe_stream_t stream);
int fe_write_kv4_ragged_strided_bf16(const void* k_new, const void* v_new, int64_t new_token_stride,
                                     void* k_codes, void* k_scales, void* v_codes, void* v_scales,
                                     const fe_kv4_strides* strides, int num_blocks,
                                     const int32_t* block_tables, int table_stride,
                                     const int32_t* q_offsets, const int32_t* context_lens,
                                     int num_seqs, int total_tokens, int kv_heads, int head_dim,
                                     int block_size, fe_stream_t stream);
int fe_gather_kv4_strided(const void* k_codes, const void* k_scales, const void* v_codes,
                          const void* v_scales, const fe_kv4_strides* strides, int num_blocks,
                          const int32_t* block_tables, int table_stride,
                          const int32_t* context_lens, const int32_t* out_offsets, void* k_out,
                          void* v_out, int batch, int total_tokens, int kv_heads, int head_dim,
                          int block_size, fe_stream_t stream);
int fe_gather_kv4_strided_bf16(const void* k_codes, const void* k_scales, const void* v_codes,
                               const void* v_scales, const fe_kv4_strides* strides, int num_blocks,
                               const int32_t* block_tables, int table_stride,
                               const int32_t* context_lens, const int32_t* out_offsets, void* k_out,
                               void* v_out, int batch, int total_tokens, int kv_heads, int head_dim,
                               int block_size, fe_stream_t stream);
int fe_paged_decode_kv4_strided(const void* q, int64_t q_batch_stride, void* out, const void* k_new,
                                const void* v_new, int64_t new_batch_stride, void* k_codes,
                                void* k_scales, void* v_codes, void* v_scales,
                                const fe_kv4_strides* strides, int num_blocks,
                                const int32_t* block_tables, int table_stride,
                                const int32_t* context_lens, void* workspace,
                                size_t workspace_bytes, int batch, int num_q_heads, int kv_heads,
                                int head_dim, int block_size, float scale, int window, int sinks,
                                int target_splits, fe_stream_t stream);
int fe_paged_decode_kv4_strided_bf16(const void* q, int64_t q_batch_stride, void* out,
                                     const void* k_new, const void* v_new, int64_t new_batch_stride,
                                     void* k_codes, void* k_scales, void* v_codes, void* v_scales,
                                     const fe_kv4_strides* strides, int num_blocks,
                                     const int32_t* block_tables, int table_stride,
                                     const int32_t* context_lens, void* workspace,
                                     size_t workspace_bytes, int batch, int num_q_heads,
                                     int kv_heads, int head_dim, int block_size, float scale,
                                     int window, int sinks, int target_splits, fe_stream_t stream);
int fe_prefill_paged_kv4_strided(const void* q, void* out, const void* k_codes,
                                 const void* k_scales, const void* v_codes, const void* v_scales,
                                 const fe_kv4_strides* strides, int num_blocks,
                                 const int32_t* block_tables, int table_stride,
                                 const int32_t* q_offsets, const int32_t* context_lens,
                                 int num_seqs, int total_q, int num_q_heads, int kv_heads,
                                 int head_dim, int block_size, float scale, int window, int sinks,
                                 void* workspace, size_t workspace_bytes, fe_stream_t stream);
int fe_prefill_paged_kv4_strided_bf16(const void* q, void* out, const void* k_codes,
                                      const void* k_scales, const void* v_codes,
                                      const void* v_scales, const fe_kv4_strides* strides,
                                      int num_blocks, const int32_t* block_tables, int table_stride,
                                      const int32_t* q_offsets, const int32_t* context_lens,
                                      int num_seqs, int total_q, int num_q_heads, int kv_heads,
                                      int head_dim, int block_size, float scale, int window,
                                      int sinks, void* workspace, size_t workspace_bytes,
                                      fe_stream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* FLEXENGINE_AMD_SPAN_H */
