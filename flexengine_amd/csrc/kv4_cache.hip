// Page writes into 4-bit pools and the gather back to 16 bits (format and layout: kv4.h).
//
// A thread takes 8 dims of one (token, KV head) row of K and of V: one 16-byte load each, the
// block's largest magnitude over the four threads of its 32 dims (two DPP steps on the
// magnitudes' bits), four conversions, one 4-byte store; the block's first thread stores the
// scale.  The gather is the reverse.  Bound: HBM bandwidth of the 16-bit rows.
#include "kv4.h"
#include "flexengine_amd_span.h"

using namespace fe;

namespace {

struct Q4Pools {
  uint8_t* k_codes;
  uint8_t* k_scales;
  uint8_t* v_codes;
  uint8_t* v_scales;
};

// Where a new token's row goes (block < 0: nowhere).
struct Slot {
  int block;
  int offset;
};
struct SlotArrays {  // explicit (block, offset) pairs
  const int32_t* block;
  const int32_t* offset;
  __device__ Slot at(int t, int nb, int bs) const {
    const int b = block[t], o = offset[t];
    return b < 0 || b >= nb || o < 0 || o >= bs ? Slot{-1, 0} : Slot{b, o};
  }
};
struct SlotDecode {  // row t is position ctx[t] - 1 of sequence t
  const int32_t* tables;
  const int32_t* ctx;
  int W, bs_log2;
  __device__ Slot at(int t, int nb, int bs) const {
    const int pos = ctx[t] - 1;
    const int page = pos >> bs_log2;
    if (pos < 0 || page >= W) return Slot{-1, 0};
    const int b = tables[(int64_t)t * W + page];
    return b < 0 || b >= nb ? Slot{-1, 0} : Slot{b, pos & (bs - 1)};
  }
};
// last s in [0, n) with off[s] <= t (0 if none)
__device__ __forceinline__ int find_row(const int32_t* off, int n, int t) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (off[mid] <= t) lo = mid; else hi = mid - 1;
  }
  return lo;
}
struct SlotRagged {  // rows q_off[s] .. q_off[s + 1] - 1 are the last positions of sequence s
  const int32_t* tables;
  const int32_t* q_off;
  const int32_t* ctx;
  int S, W, bs_log2;
  __device__ Slot at(int t, int nb, int bs) const {
    const int s = find_row(q_off, S, t);
    const int first = q_off[s], end = q_off[s + 1];
    if (t < first || t >= end) return Slot{-1, 0};
    const int pos = ctx[s] - (end - first) + (t - first);
    const int page = pos >> bs_log2;
    if (pos < 0 || page >= W) return Slot{-1, 0};
    const int b = tables[(int64_t)s * W + page];
    return b < 0 || b >= nb ? Slot{-1, 0} : Slot{b, pos & (bs - 1)};
  }
};

// codes and scale byte of the 8 dims of this thread, whose block is the quad of lanes
template <class E>
__device__ __forceinline__ uint32_t q4_quad(const f16* src, uint32_t& s) {
  const f16x8 h = ld16(src);
  float x[8];
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    x[i] = from16<E>(h[i]);
    top = max(top, abs_bits(x[i]));
  }
  top = max(top, (uint32_t)dpp::mov<dpp::kQuadXor1>((int)top));
  top = max(top, (uint32_t)dpp::mov<dpp::kQuadXor2>((int)top));
  s = q4_scale<E>(top);
  return q4_pack8(x, q4_scale_value(s));
}

template <class E, class Slots>
__global__ __launch_bounds__(256) void write_kv4_kernel(const f16* __restrict__ k_new,
                                                        const f16* __restrict__ v_new,
                                                        int64_t src_stride, Q4Pools p, int nb,
                                                        Slots slots, int T, int Hkv, int D, int BS) {
  const int cpr = D >> 3;  // a multiple of 4: a quad of lanes is one block of one row
  const int per_tok = Hkv * cpr;
  const int64_t total = (int64_t)T * per_tok;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total;
       i += (int64_t)gridDim.x * blockDim.x) {
    const int t = (int)(i / per_tok);
    const int r = (int)(i - (int64_t)t * per_tok);
    const int h = r / cpr;
    const int c = r - h * cpr;
    const Slot sl = slots.at(t, nb, BS);
    if (sl.block < 0) continue;
    const int64_t src = (int64_t)t * src_stride + (int64_t)r * 8;
    const int64_t row = ((int64_t)sl.block * Hkv + h) * BS + sl.offset;
    uint32_t ks, vs;
    const uint32_t kc = q4_quad<E>(k_new + src, ks);
    const uint32_t vc = q4_quad<E>(v_new + src, vs);
    *reinterpret_cast<uint32_t*>(p.k_codes + row * (D / 2) + c * 4) = kc;
    *reinterpret_cast<uint32_t*>(p.v_codes + row * (D / 2) + c * 4) = vc;
    if ((c & 3) == 0) {
      p.k_scales[row * (D / kQ4Block) + (c >> 2)] = (uint8_t)ks;
      p.v_scales[row * (D / kQ4Block) + (c >> 2)] = (uint8_t)vs;
    }
  }
}

template <class E>
__global__ __launch_bounds__(256) void gather_kv4_kernel(Q4Pools p, int nb,
                                                         const int32_t* __restrict__ tables, int W,
                                                         const int32_t* __restrict__ ctx,
                                                         const int32_t* __restrict__ out_off,
                                                         f16* __restrict__ k_out,
                                                         f16* __restrict__ v_out, int B,
                                                         int total_tokens, int Hkv, int D, int BS,
                                                         int bs_log2) {
  const int cpr = D >> 3;
  const int per_tok = Hkv * cpr;
  const int64_t total = (int64_t)total_tokens * per_tok;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total;
       i += (int64_t)gridDim.x * blockDim.x) {
    const int tok = (int)(i / per_tok);
    const int r = (int)(i - (int64_t)tok * per_tok);
    const int b = find_row(out_off, B, tok);
    const int t = tok - out_off[b];
    if (t < 0 || t >= ctx[b]) continue;
    int page = t >> bs_log2;
    page = page < W ? page : W - 1;
    const int blk = clamp_block(tables[(int64_t)b * W + page], nb);
    const int h = r / cpr;
    const int c = r - h * cpr;
    const int64_t row = ((int64_t)blk * Hkv + h) * BS + (t & (BS - 1));
    const uint32_t kc = *reinterpret_cast<const uint32_t*>(p.k_codes + row * (D / 2) + c * 4);
    const uint32_t vc = *reinterpret_cast<const uint32_t*>(p.v_codes + row * (D / 2) + c * 4);
    const float ks = q4_scale_value(p.k_scales[row * (D / kQ4Block) + (c >> 2)]);
    const float vs = q4_scale_value(p.v_scales[row * (D / kQ4Block) + (c >> 2)]);
    const int64_t dst = (int64_t)tok * per_tok * 8 + (int64_t)r * 8;
    st16(k_out + dst, q4_unpack8<E>(kc, ks));
    st16(v_out + dst, q4_unpack8<E>(vc, vs));
  }
}

bool aligned_to(const void* p, size_t n) { return (reinterpret_cast<uintptr_t>(p) % n) == 0; }
inline int log2_exact(int x) {
  if (x <= 0 || (x & (x - 1))) return -1;
  int l = 0;
  while ((1 << l) < x) ++l;
  return l;
}
inline dim3 grid_for(int64_t work) {
  const int64_t g = (work + 255) / 256;
  return dim3((unsigned)(g < 1 ? 1 : (g > 65536 ? 65536 : g)));
}

// Checks the writers share; what stays is each form's own arrays.
int check_rows(int rows, int64_t stride, int num_blocks, int kv_heads, int head_dim,
               int block_size) {
  FE_CHECK_ARG(rows >= 0 && num_blocks > 0 && kv_heads > 0 && head_dim > 0 && block_size > 0);
  if (head_dim % kQ4Block != 0 || log2_exact(block_size) < 0) return FE_ERR_UNSUPPORTED;
  FE_CHECK_ARG(stride % 8 == 0 && stride >= (int64_t)kv_heads * head_dim);
  return FE_OK;
}
int check_pools(const Q4Pools& p) {
  FE_CHECK_ARG(p.k_codes && p.k_scales && p.v_codes && p.v_scales);
  FE_CHECK_ARG(aligned_to(p.k_codes, 16) && aligned_to(p.v_codes, 16));
  return FE_OK;
}

template <class E, class Slots>
int write_rows(const void* k_new, const void* v_new, int64_t stride, const Q4Pools& p,
               int num_blocks, const Slots& slots, int rows, int kv_heads, int head_dim,
               int block_size, fe_stream_t stream) {
  if (int rc = check_pools(p)) return rc;
  FE_CHECK_ARG(k_new && v_new && aligned_to(k_new, 16) && aligned_to(v_new, 16));
  hipLaunchKernelGGL((write_kv4_kernel<E, Slots>),
                     grid_for((int64_t)rows * kv_heads * (head_dim / 8)), dim3(256), 0,
                     (hipStream_t)stream, (const f16*)k_new, (const f16*)v_new, stride, p,
                     num_blocks, slots, rows, kv_heads, head_dim, block_size);
  return FE_LAUNCH_STATUS();
}

inline Q4Pools pools(const void* kc, const void* ks, const void* vc, const void* vs) {
  return Q4Pools{(uint8_t*)kc, (uint8_t*)ks, (uint8_t*)vc, (uint8_t*)vs};
}

template <class E>
int write_slots(const void* k_new, const void* v_new, int64_t stride, const Q4Pools& p,
                int num_blocks, const int32_t* slot_block, const int32_t* slot_offset, int rows,
                int kv_heads, int head_dim, int block_size, fe_stream_t stream) {
  if (int rc = check_rows(rows, stride, num_blocks, kv_heads, head_dim, block_size)) return rc;
  if (rows == 0) return FE_OK;
  FE_CHECK_ARG(slot_block && slot_offset);
  return write_rows<E>(k_new, v_new, stride, p, num_blocks, SlotArrays{slot_block, slot_offset},
                       rows, kv_heads, head_dim, block_size, stream);
}

template <class E>
int write_decode(const void* k_new, const void* v_new, int64_t stride, const Q4Pools& p,
                 int num_blocks, const int32_t* tables, int table_stride, const int32_t* ctx,
                 int batch, int kv_heads, int head_dim, int block_size, fe_stream_t stream) {
  if (int rc = check_rows(batch, stride, num_blocks, kv_heads, head_dim, block_size)) return rc;
  FE_CHECK_ARG(table_stride > 0);
  if (batch == 0) return FE_OK;
  FE_CHECK_ARG(tables && ctx);
  return write_rows<E>(k_new, v_new, stride, p, num_blocks,
                       SlotDecode{tables, ctx, table_stride, log2_exact(block_size)}, batch,
                       kv_heads, head_dim, block_size, stream);
}

template <class E>
int write_ragged(const void* k_new, const void* v_new, int64_t stride, const Q4Pools& p,
                 int num_blocks, const int32_t* tables, int table_stride, const int32_t* q_off,
                 const int32_t* ctx, int num_seqs, int total, int kv_heads, int head_dim,
                 int block_size, fe_stream_t stream) {
  if (int rc = check_rows(total, stride, num_blocks, kv_heads, head_dim, block_size)) return rc;
  FE_CHECK_ARG(num_seqs >= 0 && table_stride > 0);
  if (num_seqs == 0 || total == 0) return FE_OK;
  FE_CHECK_ARG(tables && q_off && ctx);
  return write_rows<E>(k_new, v_new, stride, p, num_blocks,
                       SlotRagged{tables, q_off, ctx, num_seqs, table_stride, log2_exact(block_size)},
                       total, kv_heads, head_dim, block_size, stream);
}

template <class E>
int gather(const Q4Pools& p, int num_blocks, const int32_t* tables, int table_stride,
           const int32_t* ctx, const int32_t* out_offsets, void* k_out, void* v_out, int batch,
           int total, int kv_heads, int head_dim, int block_size, fe_stream_t stream) {
  if (int rc = check_rows(total, (int64_t)kv_heads * head_dim, num_blocks, kv_heads, head_dim,
                          block_size))
    return rc;
  FE_CHECK_ARG(batch >= 0 && table_stride > 0);
  if (batch == 0 || total == 0) return FE_OK;
  if (int rc = check_pools(p)) return rc;
  FE_CHECK_ARG(tables && ctx && out_offsets && k_out && v_out && aligned_to(k_out, 16) &&
               aligned_to(v_out, 16));
  hipLaunchKernelGGL(gather_kv4_kernel<E>, grid_for((int64_t)total * kv_heads * (head_dim / 8)),
                     dim3(256), 0, (hipStream_t)stream, p, num_blocks, tables, table_stride, ctx,
                     out_offsets, (f16*)k_out, (f16*)v_out, batch, total, kv_heads, head_dim,
                     block_size, log2_exact(block_size));
  return FE_LAUNCH_STATUS();
}

}  // namespace

// The fp16 form and its bf16 twin of each entry point.
#define FE_KV4_FORMS(SUFFIX, E)                                                                    \
  extern "C" int fe_write_kv4##SUFFIX(                                                             \
      const void* k_new, const void* v_new, int64_t new_token_stride, void* k_codes,               \
      void* k_scales, void* v_codes, void* v_scales, int num_blocks, const int32_t* slot_block,    \
      const int32_t* slot_offset, int num_tokens, int kv_heads, int head_dim, int block_size,      \
      fe_stream_t stream) {                                                                        \
    return write_slots<E>(k_new, v_new, new_token_stride,                                          \
                          pools(k_codes, k_scales, v_codes, v_scales), num_blocks, slot_block,     \
                          slot_offset, num_tokens, kv_heads, head_dim, block_size, stream);        \
  }                                                                                                \
  extern "C" int fe_write_kv4_decode##SUFFIX(                                                      \
      const void* k_new, const void* v_new, int64_t new_batch_stride, void* k_codes,               \
      void* k_scales, void* v_codes, void* v_scales, int num_blocks, const int32_t* block_tables,  \
      int table_stride, const int32_t* context_lens, int batch, int kv_heads, int head_dim,        \
      int block_size, fe_stream_t stream) {                                                        \
    return write_decode<E>(k_new, v_new, new_batch_stride,                                         \
                           pools(k_codes, k_scales, v_codes, v_scales), num_blocks, block_tables,  \
                           table_stride, context_lens, batch, kv_heads, head_dim, block_size,      \
                           stream);                                                                \
  }                                                                                                \
  extern "C" int fe_write_kv4_ragged##SUFFIX(                                                      \
      const void* k_new, const void* v_new, int64_t new_token_stride, void* k_codes,               \
      void* k_scales, void* v_codes, void* v_scales, int num_blocks, const int32_t* block_tables,  \
      int table_stride, const int32_t* q_offsets, const int32_t* context_lens, int num_seqs,       \
      int total_tokens, int kv_heads, int head_dim, int block_size, fe_stream_t stream) {          \
    return write_ragged<E>(k_new, v_new, new_token_stride,                                         \
                           pools(k_codes, k_scales, v_codes, v_scales), num_blocks, block_tables,  \
                           table_stride, q_offsets, context_lens, num_seqs, total_tokens,          \
                           kv_heads, head_dim, block_size, stream);                                \
  }                                                                                                \
  extern "C" int fe_gather_kv4##SUFFIX(                                                            \
      const void* k_codes, const void* k_scales, const void* v_codes, const void* v_scales,        \
      int num_blocks, const int32_t* block_tables, int table_stride, const int32_t* context_lens,  \
      const int32_t* out_offsets, void* k_out, void* v_out, int batch, int total_tokens,           \
      int kv_heads, int head_dim, int block_size, fe_stream_t stream) {                            \
    return gather<E>(pools(k_codes, k_scales, v_codes, v_scales), num_blocks, block_tables,        \
                     table_stride, context_lens, out_offsets, k_out, v_out, batch, total_tokens,   \
                     kv_heads, head_dim, block_size, stream);                                      \
  }
FE_KV4_FORMS(, Fp16)
FE_KV4_FORMS(_bf16, Bf16)
