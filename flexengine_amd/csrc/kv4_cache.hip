// Page writes into 4-bit pools and the gather back to 16 bits (format and layout: kv4.h).
//
// A thread takes 8 dims of one (token, KV head) row of K and of V at a time: one 16-byte load
// each, the block's largest magnitude over the four threads of its 32 dims (two DPP steps on
// the magnitudes' bits), four conversions, one 4-byte store; the block's first thread stores
// the scale.  The gather is the reverse.  A workgroup takes a run of tokens of kChunks such
// chunks and looks their slots up first, one thread a token, over offsets and lengths in LDS:
// looked up by every thread the chain of dependent loads was the kernels' length.  6468 tokens
// of 8 heads of 128, 33.5 MB moved by each: write 10.8 -> 9.1 us, gather 10.1 -> 8.4 (of 6.6 at
// the rate of a large copy; 2048 chunks a workgroup 12.2 and 10.9).
#include "kv4.h"
#include "flexengine_amd_span.h"

using namespace fe;

namespace {

struct Q4Pools {
  uint8_t* k_codes;
  uint8_t* k_scales;
  uint8_t* v_codes;
  uint8_t* v_scales;
  Q4Layout rows;
};

constexpr int kThreads = 256;
constexpr int kChunks = 512;     // chunks of a workgroup
constexpr int kMaxTokens = 256;  // tokens of a workgroup at most (one looked up by a thread)
constexpr int kMaxSeqs = 512;    // sequences whose offsets and lengths are searched in LDS

// Where a token's row is (block < 0: nowhere).
struct Slot {
  int block;
  int offset;
};
// Row offsets and context lengths of the sequences, in LDS where they fit
struct SeqLds {
  int off[kMaxSeqs + 1];
  int ctx[kMaxSeqs];
};
struct Seq {
  int s, first, end, ctx;
};
__device__ __forceinline__ void load_seqs(const int32_t* off, const int32_t* ctx, int S, SeqLds& l) {
  if (S > kMaxSeqs) return;
  for (int i = threadIdx.x; i <= S; i += kThreads) {
    l.off[i] = off[i];
    if (i < S) l.ctx[i] = ctx[i];
  }
}
// the last sequence s with off[s] <= t (0 if none)
__device__ __forceinline__ Seq find_seq(const int32_t* off, const int32_t* ctx, int S, int t,
                                        const SeqLds& l) {
  int lo = 0, hi = S - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if ((S > kMaxSeqs ? off[mid] : l.off[mid]) <= t) lo = mid; else hi = mid - 1;
  }
  if (S > kMaxSeqs) return Seq{lo, off[lo], off[lo + 1], ctx[lo]};
  return Seq{lo, l.off[lo], l.off[lo + 1], l.ctx[lo]};
}

// Slot maps of the writes: load() before a barrier, at() after it
struct SlotArrays {  // explicit (block, offset) pairs
  const int32_t* block;
  const int32_t* offset;
  __device__ void load(SeqLds&) const {}
  __device__ Slot at(int t, int nb, int bs, const SeqLds&) const {
    const int b = block[t], o = offset[t];
    return b < 0 || b >= nb || o < 0 || o >= bs ? Slot{-1, 0} : Slot{b, o};
  }
};
struct SlotDecode {  // row t is position ctx[t] - 1 of sequence t
  const int32_t* tables;
  const int32_t* ctx;
  int W, bs_log2;
  __device__ void load(SeqLds&) const {}
  __device__ Slot at(int t, int nb, int bs, const SeqLds&) const {
    const int pos = ctx[t] - 1;
    const int page = pos >> bs_log2;
    if (pos < 0 || page >= W) return Slot{-1, 0};
    const int b = tables[(int64_t)t * W + page];
    return b < 0 || b >= nb ? Slot{-1, 0} : Slot{b, pos & (bs - 1)};
  }
};
struct SlotRagged {  // rows q_off[s] .. q_off[s + 1] - 1 are the last positions of sequence s
  const int32_t* tables;
  const int32_t* q_off;
  const int32_t* ctx;
  int S, W, bs_log2;
  __device__ void load(SeqLds& l) const { load_seqs(q_off, ctx, S, l); }
  __device__ Slot at(int t, int nb, int bs, const SeqLds& l) const {
    const Seq q = find_seq(q_off, ctx, S, t, l);
    if (t < q.first || t >= q.end) return Slot{-1, 0};
    const int pos = q.ctx - (q.end - q.first) + (t - q.first);
    const int page = pos >> bs_log2;
    if (pos < 0 || page >= W) return Slot{-1, 0};
    const int b = tables[(int64_t)q.s * W + page];
    return b < 0 || b >= nb ? Slot{-1, 0} : Slot{b, pos & (bs - 1)};
  }
};

// codes and scale byte of the 8 dims of this thread, whose block is the quad of lanes
template <class E>
__device__ __forceinline__ uint32_t q4_quad(f16x8 h, uint32_t& s) {
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

// Tokens of a workgroup
inline int tokens_per_wg(int per_tok) {
  const int n = kChunks / per_tok;
  return n < 1 ? 1 : (n > kMaxTokens ? kMaxTokens : n);
}

// Chunk i of a workgroup of n tokens: chunk c of KV head h of token t, head by head, so that
// neighbouring tokens, whose 4-bit rows of a head lie side by side, are written together.
// (A quad of lanes is one block of one row: cpr and with it every count is a multiple of 4.)
struct Chunk {
  uint32_t t, h, c;
  bool on;
  __device__ __forceinline__ Chunk(uint32_t i, uint32_t n, uint32_t total, uint32_t cpr) {
    const uint32_t row = i / cpr;
    c = i - row * cpr;
    h = row / n;
    t = row - h * n;
    on = i < total;
  }
  // of the token's chunks
  __device__ __forceinline__ uint32_t of_token(uint32_t cpr) const { return h * cpr + c; }
};

// byte offsets of a chunk's codes and of its block's scale
__device__ __forceinline__ int64_t code_at(const Q4Layout& l, const Slot& s, const Chunk& ch) {
  return (int64_t)l.code_row(s.block, s.offset) + l.code_offset(ch.h) + ch.c * 4;
}
__device__ __forceinline__ int64_t scale_at(const Q4Layout& l, const Slot& s, const Chunk& ch) {
  return (int64_t)l.scale_row(s.block, s.offset) + l.scale_offset(ch.h) + (ch.c >> 2);
}

template <class E, class Slots>
__global__ __launch_bounds__(kThreads) void write_kv4_kernel(const f16* __restrict__ k_new,
                                                             const f16* __restrict__ v_new,
                                                             int64_t src_stride, Q4Pools p, int nb,
                                                             Slots slots, int T, int per_wg,
                                                             int Hkv, int D, int BS) {
  __shared__ Slot at[kMaxTokens];
  __shared__ SeqLds seqs;
  const int t0 = (int)blockIdx.x * per_wg;
  const int n = min(per_wg, T - t0);
  const uint32_t cpr = D >> 3, per_tok = Hkv * cpr, total = n * per_tok;
  slots.load(seqs);
  for (uint32_t base = 0; base < total; base += kThreads) {  // workgroup-uniform
    const Chunk ch(base + threadIdx.x, n, total, cpr);
    f16x8 k = {}, v = {};
    if (ch.on) {
      const int64_t src = (int64_t)(t0 + ch.t) * src_stride + ch.of_token(cpr) * 8;
      k = ld16(k_new + src);
      v = ld16(v_new + src);
    }
    if (base == 0) {  // the first rows do not wait for their slots
      __syncthreads();
      if ((int)threadIdx.x < n) at[threadIdx.x] = slots.at(t0 + threadIdx.x, nb, BS, seqs);
      __syncthreads();
    }
    if (!ch.on) continue;
    const Slot sl = at[ch.t];
    if (sl.block < 0) continue;
    uint32_t ks, vs;
    const uint32_t kc = q4_quad<E>(k, ks), vc = q4_quad<E>(v, vs);
    const int64_t co = code_at(p.rows, sl, ch), so = scale_at(p.rows, sl, ch);
    *reinterpret_cast<uint32_t*>(p.k_codes + co) = kc;
    *reinterpret_cast<uint32_t*>(p.v_codes + co) = vc;
    if ((ch.c & 3) == 0) {
      p.k_scales[so] = (uint8_t)ks;
      p.v_scales[so] = (uint8_t)vs;
    }
  }
}

template <class E>
__global__ __launch_bounds__(kThreads) void gather_kv4_kernel(
    Q4Pools p, int nb, const int32_t* __restrict__ tables, int W, const int32_t* __restrict__ ctx,
    const int32_t* __restrict__ out_off, f16* __restrict__ k_out, f16* __restrict__ v_out, int B,
    int total_tokens, int per_wg, int Hkv, int D, int BS, int bs_log2) {
  __shared__ Slot at[kMaxTokens];
  __shared__ SeqLds seqs;
  const int t0 = (int)blockIdx.x * per_wg;
  const int n = min(per_wg, total_tokens - t0);
  const uint32_t cpr = D >> 3, per_tok = Hkv * cpr, total = n * per_tok;
  load_seqs(out_off, ctx, B, seqs);
  __syncthreads();
  if ((int)threadIdx.x < n) {
    const int tok = t0 + threadIdx.x;
    const Seq q = find_seq(out_off, ctx, B, tok, seqs);
    const int t = tok - q.first;
    Slot sl{-1, 0};
    if (t >= 0 && t < q.ctx) {
      int page = t >> bs_log2;
      page = page < W ? page : W - 1;
      sl = Slot{clamp_block(tables[(int64_t)q.s * W + page], nb), t & (BS - 1)};
    }
    at[threadIdx.x] = sl;
  }
  __syncthreads();
  for (uint32_t i = threadIdx.x; i < total; i += kThreads) {
    const Chunk ch(i, n, total, cpr);
    const Slot sl = at[ch.t];
    if (sl.block < 0) continue;
    const int64_t co = code_at(p.rows, sl, ch), so = scale_at(p.rows, sl, ch);
    const uint32_t kc = *reinterpret_cast<const uint32_t*>(p.k_codes + co);
    const uint32_t vc = *reinterpret_cast<const uint32_t*>(p.v_codes + co);
    const uint32_t ks = p.k_scales[so];
    const uint32_t vs = p.v_scales[so];
    const int64_t dst = ((int64_t)(t0 + ch.t) * per_tok + ch.of_token(cpr)) * 8;
    st16(k_out + dst, q4_unpack8<E>(kc, q4_scale_value(ks)));
    st16(v_out + dst, q4_unpack8<E>(vc, q4_scale_value(vs)));
  }
}

bool aligned_to(const void* p, size_t n) { return (reinterpret_cast<uintptr_t>(p) % n) == 0; }
inline int log2_exact(int x) {
  if (x <= 0 || (x & (x - 1))) return -1;
  int l = 0;
  while ((1 << l) < x) ++l;
  return l;
}
// Checks the writers share; what stays is each form's own arrays.
int check_rows(int rows, int64_t stride, int num_blocks, int kv_heads, int head_dim,
               int block_size) {
  FE_CHECK_ARG(rows >= 0 && num_blocks > 0 && kv_heads > 0 && head_dim > 0 && block_size > 0);
  if (head_dim % kQ4Block != 0 || log2_exact(block_size) < 0) return FE_ERR_UNSUPPORTED;
  // a token's chunks are counted in 32 bits
  if ((int64_t)kv_heads * head_dim >= ((int64_t)1 << 25) || rows > (1 << 30))
    return FE_ERR_UNSUPPORTED;
  FE_CHECK_ARG(stride % 8 == 0 && stride >= (int64_t)kv_heads * head_dim);
  return FE_OK;
}
// The pools as a caller gives them (strides null: dense), and as the kernels take them
struct PoolArgs {
  const void *k_codes, *k_scales, *v_codes, *v_scales;
  const fe_kv4_strides* strides;
};
int check_pools(const PoolArgs& a, int num_blocks, int kv_heads, int head_dim, int block_size,
                Q4Pools& p) {
  p = Q4Pools{(uint8_t*)a.k_codes, (uint8_t*)a.k_scales, (uint8_t*)a.v_codes,
              (uint8_t*)a.v_scales, {}};
  FE_CHECK_ARG(p.k_codes && p.k_scales && p.v_codes && p.v_scales);
  FE_CHECK_ARG(aligned_to(p.k_codes, 16) && aligned_to(p.v_codes, 16));
  return q4_layout(a.strides, num_blocks, kv_heads, head_dim, block_size, p.rows);
}

template <class E, class Slots>
int write_rows(const void* k_new, const void* v_new, int64_t stride, const PoolArgs& args,
               int num_blocks, const Slots& slots, int rows, int kv_heads, int head_dim,
               int block_size, fe_stream_t stream) {
  Q4Pools p;
  if (int rc = check_pools(args, num_blocks, kv_heads, head_dim, block_size, p)) return rc;
  FE_CHECK_ARG(k_new && v_new && aligned_to(k_new, 16) && aligned_to(v_new, 16));
  const int per_wg = tokens_per_wg(kv_heads * (head_dim / 8));
  hipLaunchKernelGGL((write_kv4_kernel<E, Slots>), dim3((rows + per_wg - 1) / per_wg),
                     dim3(kThreads), 0, (hipStream_t)stream, (const f16*)k_new,
                     (const f16*)v_new, stride, p, num_blocks, slots, rows, per_wg, kv_heads,
                     head_dim, block_size);
  return FE_LAUNCH_STATUS();
}

template <class E>
int write_slots(const void* k_new, const void* v_new, int64_t stride, const PoolArgs& args,
                int num_blocks, const int32_t* slot_block, const int32_t* slot_offset, int rows,
                int kv_heads, int head_dim, int block_size, fe_stream_t stream) {
  if (int rc = check_rows(rows, stride, num_blocks, kv_heads, head_dim, block_size)) return rc;
  if (rows == 0) return FE_OK;
  FE_CHECK_ARG(slot_block && slot_offset);
  return write_rows<E>(k_new, v_new, stride, args, num_blocks, SlotArrays{slot_block, slot_offset},
                       rows, kv_heads, head_dim, block_size, stream);
}

template <class E>
int write_decode(const void* k_new, const void* v_new, int64_t stride, const PoolArgs& args,
                 int num_blocks, const int32_t* tables, int table_stride, const int32_t* ctx,
                 int batch, int kv_heads, int head_dim, int block_size, fe_stream_t stream) {
  if (int rc = check_rows(batch, stride, num_blocks, kv_heads, head_dim, block_size)) return rc;
  FE_CHECK_ARG(table_stride > 0);
  if (batch == 0) return FE_OK;
  FE_CHECK_ARG(tables && ctx);
  return write_rows<E>(k_new, v_new, stride, args, num_blocks,
                       SlotDecode{tables, ctx, table_stride, log2_exact(block_size)}, batch,
                       kv_heads, head_dim, block_size, stream);
}

template <class E>
int write_ragged(const void* k_new, const void* v_new, int64_t stride, const PoolArgs& args,
                 int num_blocks, const int32_t* tables, int table_stride, const int32_t* q_off,
                 const int32_t* ctx, int num_seqs, int total, int kv_heads, int head_dim,
                 int block_size, fe_stream_t stream) {
  if (int rc = check_rows(total, stride, num_blocks, kv_heads, head_dim, block_size)) return rc;
  FE_CHECK_ARG(num_seqs >= 0 && table_stride > 0);
  if (num_seqs == 0 || total == 0) return FE_OK;
  FE_CHECK_ARG(tables && q_off && ctx);
  return write_rows<E>(k_new, v_new, stride, args, num_blocks,
                       SlotRagged{tables, q_off, ctx, num_seqs, table_stride, log2_exact(block_size)},
                       total, kv_heads, head_dim, block_size, stream);
}

template <class E>
int gather(const PoolArgs& args, int num_blocks, const int32_t* tables, int table_stride,
           const int32_t* ctx, const int32_t* out_offsets, void* k_out, void* v_out, int batch,
           int total, int kv_heads, int head_dim, int block_size, fe_stream_t stream) {
  if (int rc = check_rows(total, (int64_t)kv_heads * head_dim, num_blocks, kv_heads, head_dim,
                          block_size))
    return rc;
  FE_CHECK_ARG(batch >= 0 && table_stride > 0);
  if (batch == 0 || total == 0) return FE_OK;
  Q4Pools p;
  if (int rc = check_pools(args, num_blocks, kv_heads, head_dim, block_size, p)) return rc;
  FE_CHECK_ARG(tables && ctx && out_offsets && k_out && v_out && aligned_to(k_out, 16) &&
               aligned_to(v_out, 16));
  const int per_wg = tokens_per_wg(kv_heads * (head_dim / 8));
  hipLaunchKernelGGL(gather_kv4_kernel<E>, dim3((total + per_wg - 1) / per_wg), dim3(kThreads), 0,
                     (hipStream_t)stream, p, num_blocks, tables, table_stride, ctx, out_offsets,
                     (f16*)k_out, (f16*)v_out, batch, total, per_wg, kv_heads, head_dim,
                     block_size, log2_exact(block_size));
  return FE_LAUNCH_STATUS();
}

}  // namespace

// The fp16 form and its bf16 twin of each entry point, and the forms that take strides.
#define FE_KV4_FORMS(STRIDED, SUFFIX, E, STRIDES_PARAM, STRIDES)                                   \
  extern "C" int fe_write_kv4##STRIDED##SUFFIX(                                                    \
      const void* k_new, const void* v_new, int64_t new_token_stride, void* k_codes,               \
      void* k_scales, void* v_codes, void* v_scales, STRIDES_PARAM int num_blocks,                 \
      const int32_t* slot_block, const int32_t* slot_offset, int num_tokens, int kv_heads,         \
      int head_dim, int block_size, fe_stream_t stream) {                                          \
    return write_slots<E>(k_new, v_new, new_token_stride,                                          \
                          PoolArgs{k_codes, k_scales, v_codes, v_scales, STRIDES}, num_blocks,     \
                          slot_block, slot_offset, num_tokens, kv_heads, head_dim, block_size,     \
                          stream);                                                                 \
  }                                                                                                \
  extern "C" int fe_write_kv4_decode##STRIDED##SUFFIX(                                             \
      const void* k_new, const void* v_new, int64_t new_batch_stride, void* k_codes,               \
      void* k_scales, void* v_codes, void* v_scales, STRIDES_PARAM int num_blocks,                 \
      const int32_t* block_tables, int table_stride, const int32_t* context_lens, int batch,       \
      int kv_heads, int head_dim, int block_size, fe_stream_t stream) {                            \
    return write_decode<E>(k_new, v_new, new_batch_stride,                                         \
                           PoolArgs{k_codes, k_scales, v_codes, v_scales, STRIDES}, num_blocks,    \
                           block_tables, table_stride, context_lens, batch, kv_heads, head_dim,    \
                           block_size, stream);                                                    \
  }                                                                                                \
  extern "C" int fe_write_kv4_ragged##STRIDED##SUFFIX(                                             \
      const void* k_new, const void* v_new, int64_t new_token_stride, void* k_codes,               \
      void* k_scales, void* v_codes, void* v_scales, STRIDES_PARAM int num_blocks,                 \
      const int32_t* block_tables, int table_stride, const int32_t* q_offsets,                     \
      const int32_t* context_lens, int num_seqs, int total_tokens, int kv_heads, int head_dim,     \
      int block_size, fe_stream_t stream) {                                                        \
    return write_ragged<E>(k_new, v_new, new_token_stride,                                         \
                           PoolArgs{k_codes, k_scales, v_codes, v_scales, STRIDES}, num_blocks,    \
                           block_tables, table_stride, q_offsets, context_lens, num_seqs,          \
                           total_tokens, kv_heads, head_dim, block_size, stream);                  \
  }                                                                                                \
  extern "C" int fe_gather_kv4##STRIDED##SUFFIX(                                                   \
      const void* k_codes, const void* k_scales, const void* v_codes, const void* v_scales,        \
      STRIDES_PARAM int num_blocks, const int32_t* block_tables, int table_stride,                 \
      const int32_t* context_lens, const int32_t* out_offsets, void* k_out, void* v_out,           \
      int batch, int total_tokens, int kv_heads, int head_dim, int block_size,                     \
      fe_stream_t stream) {                                                                        \
    return gather<E>(PoolArgs{k_codes, k_scales, v_codes, v_scales, STRIDES}, num_blocks,          \
                     block_tables, table_stride, context_lens, out_offsets, k_out, v_out, batch,   \
                     total_tokens, kv_heads, head_dim, block_size, stream);                        \
  }
#define FE_STRIDES_PARAM const fe_kv4_strides *strides,
FE_KV4_FORMS(, , Fp16, , nullptr)
FE_KV4_FORMS(, _bf16, Bf16, , nullptr)
FE_KV4_FORMS(_strided, , Fp16, FE_STRIDES_PARAM, strides)
FE_KV4_FORMS(_strided, _bf16, Bf16, FE_STRIDES_PARAM, strides)
