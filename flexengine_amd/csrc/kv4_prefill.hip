// Ragged prefill over 4-bit pools, with or without a window.
#include "span_prefill.h"

using namespace fe;

#define FE_KV4_PREFILL(SUFFIX, E, STRIDES_PARAM, STRIDES)                                         \
  extern "C" int fe_prefill_paged_kv4##SUFFIX(                                                    \
      const void* q, void* out, const void* k_codes, const void* k_scales, const void* v_codes,   \
      const void* v_scales, STRIDES_PARAM int num_blocks, const int32_t* block_tables,            \
      int table_stride, const int32_t* q_offsets, const int32_t* context_lens, int num_seqs,      \
      int total_q, int num_q_heads, int kv_heads, int head_dim, int block_size, float scale,      \
      int window, int sinks, void* workspace, size_t workspace_bytes, fe_stream_t stream) {       \
    return span_prefill<E, true>(q, out, k_codes, k_scales, v_codes, v_scales, STRIDES,           \
                                 num_blocks, block_tables, table_stride, q_offsets, context_lens, \
                                 num_seqs, total_q, num_q_heads, kv_heads, head_dim, block_size,  \
                                 scale, window, sinks, workspace, workspace_bytes, stream);       \
  }
#define FE_STRIDES_PARAM const fe_kv4_strides *strides,
FE_KV4_PREFILL(, Fp16, , nullptr)
FE_KV4_PREFILL(_bf16, Bf16, , nullptr)
FE_KV4_PREFILL(_strided, Fp16, FE_STRIDES_PARAM, strides)
FE_KV4_PREFILL(_strided_bf16, Bf16, FE_STRIDES_PARAM, strides)
