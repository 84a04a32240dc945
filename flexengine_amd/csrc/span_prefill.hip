// Ragged prefill under a window with sinks over fp16, bf16 and fp32 pools.
#include "span_prefill.h"

using namespace fe;

namespace {

// ---- fp32 pools ---------------------------------------------------------------------------
// The plain fp32 prefill's organisation on the same engine (F32Core, attn_core.h): a workgroup
// takes 16 rows of a sequence and KV head, its four waves the row block's 16-key tiles in turn
// -- the tiles of the sinks and those from the first row's window start on -- and the waves'
// states are joined in LDS.  Bound by the fp32 MFMAs (154 TFLOP/s in a large product): three
// chunks of 100-700 tokens of 12/2 heads under a window of 512 40.9 us, 65 TFLOP/s, half the
// chip in its second round.  32 rows a workgroup, which halve the reads of K and V: 49.1 us,
// and four chunks of 500 under 1024 120 -> 145 (as two waves a 16-row tile 49.8 and 118.5);
// eight waves 50.5.  Units too few for the chip share their keys out over splits, as the 16-bit
// kernel's do (span_prefill.h): 50 tokens over up to 3000 under a window of 2000 38.3 -> 15.7 us,
// four chunks of 10-20 over up to 8000 under 4000 92.6 -> 35.8 (four chunks of 500 at head_dim 96,
// not split, 128.5 -> 132: that padded form spills 15 registers, 64 bytes of scratch a lane).
constexpr int kF32Waves = 4;
constexpr int kF32Slots = 768;  // workgroups that run at once: three on each of 256 CUs

template <int D>
struct SpanF32Lds {
  static constexpr int NX = D / 16;
  static constexpr size_t park = 0;  // [kF32Waves][NX][64] x 16 bytes
  static constexpr size_t park_m = park + (size_t)kF32Waves * NX * kWave * 16;
  static constexpr size_t park_l = park_m + (size_t)kF32Waves * kWave * sizeof(float);
  static constexpr size_t last = park_l + (size_t)kF32Waves * kWave * sizeof(float);
  static constexpr size_t bytes = last + sizeof(int);
};

template <int D, bool PAD>
__global__ __launch_bounds__(kF32Waves* kWave) __attribute__((amdgpu_waves_per_eu(3, 8)))
void span_prefill_f32_kernel(const SpanPrefill a) {
  using Core = F32Core<D, true, PAD, 1, true>;
  using Lds = SpanF32Lds<D>;
  constexpr int ROWS = kTile;
  constexpr int NX = Core::NX;
  extern __shared__ __align__(16) unsigned char smem[];
  const int DR = PAD ? a.dr : D;
  // by split, then the later units, which see more keys, first
  const int at = (int)blockIdx.x / a.Hkv;
  const int h = (int)blockIdx.x - at * a.Hkv;
  const int item = a.units - 1 - at;
  const int ks = blockIdx.y;
  SpanUnit u;
  SpanWork work;
  if (!find_unit<ROWS>(a, item, u, work)) return;
  const int G = a.G;
  const int lane = lane_id();
  const int g = lane >> 4;
  const int n = lane & 15;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int ctx = min(u.ctx, a.W * a.BS);
  const int total_rows = u.n * G;
  const int cached = ctx >= u.n ? ctx - u.n : 0;
  const int r0 = u.block * ROWS;
  const int r_last = min(r0 + ROWS, total_rows) - 1;
  const int row = r0 + n;
  const bool valid = row < total_rows;
  const int rc = valid ? row : r_last;

  Core core;
  core.k_pool = (const float*)a.k_pool;
  core.v_pool = (const float*)a.v_pool;
  core.k_pool_w = nullptr;
  core.v_pool_w = nullptr;
  core.trow = a.tables + (int64_t)u.s * a.W;
  core.rs = (int64_t)a.Hkv * DR;
  core.hoff = h * DR;
  core.dr = DR;
  core.W = a.W;
  core.NB = a.NB;
  core.BS = a.BS;
  core.bs_log2 = a.bs_log2;
  core.scale_log2 = a.scale_log2;
  core.knew_row = nullptr;
  core.vnew_row = nullptr;
  core.new_pos = -1;
  const UnitRows rows(a, u, r0, h);
  SpanWalk wk;
  wk.init(a.span, cached + rows.q, cached + rows.token(r_last - r0));
  core.tok_end = wk.key_end;
  core.sinks = wk.sinks;
  core.wmin = wk.ws;
  core.span_head = wk.head;
  core.span_skip = wk.skip;
  const int pos = cached + rows.token(rc - r0);
  core.limit[0] = valid ? pos + 1 : 0;
  core.wlo[0] = window_start(a.span, pos);
  const int nt = (wk.key_end + kTile - 1) / kTile - wk.skip;
  const int splits = span_splits(a, work, wk.blocks(), kF32Slots);
  if (ks >= splits) return;
  const int ntiles = core.begin(nt * ks / splits + w, kF32Waves, nt * (ks + 1) / splits);
  const float* qrow = (const float*)a.q + rows(rc - r0) * DR;
#pragma unroll
  for (int c = 0; c < Core::NC; ++c) {
    core.qv[0][c] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (!PAD || 16 * c + 4 * g < DR)
      core.qv[0][c] = *reinterpret_cast<const f32x4*>(qrow + 16 * c + 4 * g);
  }
  core.init_acc();
  core.run_single(ntiles);

  f32x4* park = reinterpret_cast<f32x4*>(smem + Lds::park);
  float* park_m = reinterpret_cast<float*>(smem + Lds::park_m);
  float* park_l = reinterpret_cast<float*>(smem + Lds::park_l);
#pragma unroll
  for (int x = 0; x < NX; ++x) park[(w * NX + x) * kWave + lane] = core.o[0][x];
  park_m[w * kWave + lane] = core.m_run[0];
  park_l[w * kWave + lane] = core.l_total();
  __syncthreads();
  float M = kNegInf, den = 0.f, sc[kF32Waves];
#pragma unroll
  for (int v = 0; v < kF32Waves; ++v) M = fmaxf(M, park_m[v * kWave + lane]);
#pragma unroll
  for (int v = 0; v < kF32Waves; ++v) {
    const float mv = park_m[v * kWave + lane];
    sc[v] = mv == kNegInf ? 0.f : exp2f(mv - M);
    den += sc[v] * park_l[v * kWave + lane];
  }
  const float inv = den > 0.f ? 1.f / den : 0.f;
  constexpr int C = NX / kF32Waves;
  f32x4 o[C];
#pragma unroll
  for (int i = 0; i < C; ++i) {
    const int x = w + kF32Waves * i;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int v = 0; v < kF32Waves; ++v)
      // tile x as the 16 dims from 16 x (a lane parked its 4 dims from f32_dim0)
      acc += sc[v] * park[(v * NX + (x & ~3) + g) * kWave + 16 * (x & 3) + n];
    o[i] = acc * inv;
  }
  if (splits > 1) {
    const SplitParts<C, kF32Waves * kWave> part(a, item, h);
    if (valid) part.store(ks, o, den > 0.f ? M + log2f(den) : kNegInf);
    int* const last = reinterpret_cast<int*>(smem + Lds::last);
    if (!last_split(a.tickets + item * a.Hkv + h, splits, last)) return;
    part.join(splits, o);
  }
  if (!valid) return;
  const int64_t orow = rows(row - r0) * DR;
#pragma unroll
  for (int i = 0; i < C; ++i) {
    const int d0 = 16 * (w + kF32Waves * i) + 4 * g;
    if (!PAD || d0 < DR) store_out4<F32>(a.out, orow + d0, o[i]);
  }
}

template <int D, bool PAD>
int launch_f32(const SpanPrefill& a, hipStream_t s) {
  hipLaunchKernelGGL((span_prefill_f32_kernel<D, PAD>),
                     dim3((unsigned)(a.units * a.Hkv), (unsigned)a.KS), dim3(kF32Waves * kWave),
                     SpanF32Lds<D>::bytes, s, a);
  return FE_LAUNCH_STATUS();
}

int span_prefill_f32(const void* q, void* out, const void* k_pool, const void* v_pool,
                     int num_blocks, const int32_t* tables, int table_stride, const int32_t* q_off,
                     const int32_t* ctx, int num_seqs, int total_q, int hq, int hkv, int d, int bs,
                     float scale, int window, int sinks, void* workspace, size_t workspace_bytes,
                     fe_stream_t stream) {
  FE_CHECK_ARG(num_seqs >= 0 && total_q >= 0 && hq > 0 && hkv > 0 && d > 0 && num_blocks > 0 &&
               table_stride > 0 && window > 0 && sinks >= 0 && hq % hkv == 0 && scale > 0.f);
  const int bs_log2 = span_log2(bs);
  if (bs_log2 < 0 || bs % kTile != 0 || d > 128 || d % 8 != 0) return FE_ERR_UNSUPPORTED;
  if ((int64_t)table_stride * bs >= ((int64_t)1 << 30) || hq / hkv > (1 << 20) ||
      (int64_t)num_blocks * bs >= ((int64_t)1 << 31) || (int64_t)hkv * d >= ((int64_t)1 << 25) ||
      (int64_t)total_q * (hq / hkv) >= ((int64_t)1 << 30))
    return FE_ERR_UNSUPPORTED;
  if (num_seqs == 0 || total_q == 0) return FE_OK;
  FE_CHECK_ARG(q && out && k_pool && v_pool && tables && q_off && ctx);
  const auto aligned = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; };
  FE_CHECK_ARG(aligned(q) && aligned(out) && aligned(k_pool) && aligned(v_pool));
  const SpanShape p = span_shape(num_seqs, total_q, hq, hkv, d, window, false, kTile, kF32Slots);
  // (a grid's threads are counted in 32 bits)
  if (p.units * hkv >= ((int64_t)1 << 23)) return FE_ERR_UNSUPPORTED;
  if (workspace == nullptr || workspace_bytes < p.bytes || !aligned(workspace))
    return FE_ERR_WORKSPACE;
  SpanPrefill a{};
  a.tickets = (int*)workspace;
  a.parts = (unsigned char*)workspace + kSpanTicketBytes;
  a.q = (const f16*)q;
  a.out = (f16*)out;
  a.k_pool = k_pool;
  a.v_pool = v_pool;
  a.tables = tables;
  a.q_off = q_off;
  a.ctx = ctx;
  a.W = table_stride;
  a.S = num_seqs;
  a.total_q = total_q;
  a.Hq = hq;
  a.Hkv = hkv;
  a.G = hq / hkv;
  a.BS = bs;
  a.bs_log2 = bs_log2;
  a.NB = num_blocks;
  a.KS = p.ks;
  a.units = (int)p.units;
  a.dr = d;
  a.scale_log2 = scale * kLog2e;
  a.span = Span{window, sinks};
  const hipStream_t s = (hipStream_t)stream;
  if (d == 64) return launch_f32<64, false>(a, s);
  if (d == 128) return launch_f32<128, false>(a, s);
  return d < 64 ? launch_f32<64, true>(a, s) : launch_f32<128, true>(a, s);
}

}  // namespace

extern "C" size_t fe_span_prefill_workspace_size(int num_seqs, int total_q, int num_q_heads,
                                                 int kv_heads, int head_dim) {
  if (num_seqs < 0 || total_q < 0 || num_q_heads <= 0 || kv_heads <= 0 || head_dim <= 0 ||
      num_q_heads % kv_heads)
    return 0;
  // (the form of eight waves takes no more)
  const size_t b16 = span_shape(num_seqs, total_q, num_q_heads, kv_heads, head_dim, 1, false).bytes;
  const size_t b32 = span_shape(num_seqs, total_q, num_q_heads, kv_heads, head_dim, 1, false, kTile,
                                kF32Slots).bytes;
  return b16 > b32 ? b16 : b32;
}

extern "C" int fe_span_prefill_rows(int num_seqs, int total_q, int num_q_heads, int kv_heads,
                                    int head_dim, int window, int kv4, int elem_bytes) {
  FE_CHECK_ARG(num_seqs > 0 && total_q > 0 && num_q_heads > 0 && kv_heads > 0 && head_dim > 0 &&
               window >= 0 && num_q_heads % kv_heads == 0);
  FE_CHECK_ARG(kv4 ? elem_bytes == 2 : (window > 0 && (elem_bytes == 2 || elem_bytes == 4)));
  if (elem_bytes == 4) return kTile;
  return 32 * span_waves(num_seqs, total_q, num_q_heads, kv_heads, head_dim, window, kv4 != 0);
}

#define FE_WINDOW_PREFILL(SUFFIX, E)                                                              \
  extern "C" int fe_prefill_paged_window##SUFFIX(                                                 \
      const void* q, void* out, const void* k_pool, const void* v_pool, int num_blocks,           \
      const int32_t* block_tables, int table_stride, const int32_t* q_offsets,                    \
      const int32_t* context_lens, int num_seqs, int total_q, int num_q_heads, int kv_heads,      \
      int head_dim, int block_size, float scale, int window, int sinks, void* workspace,          \
      size_t workspace_bytes, fe_stream_t stream) {                                               \
    return span_prefill<E, false>(q, out, k_pool, nullptr, v_pool, nullptr, nullptr, num_blocks,  \
                                  block_tables, table_stride, q_offsets, context_lens, num_seqs,  \
                                  total_q, num_q_heads, kv_heads, head_dim, block_size, scale,    \
                                  window, sinks, workspace, workspace_bytes, stream);             \
  }
FE_WINDOW_PREFILL(, Fp16)
FE_WINDOW_PREFILL(_bf16, Bf16)

extern "C" int fe_prefill_paged_window_f32(const void* q, void* out, const void* k_pool,
                                           const void* v_pool, int num_blocks,
                                           const int32_t* block_tables, int table_stride,
                                           const int32_t* q_offsets, const int32_t* context_lens,
                                           int num_seqs, int total_q, int num_q_heads,
                                           int kv_heads, int head_dim, int block_size, float scale,
                                           int window, int sinks, void* workspace,
                                           size_t workspace_bytes, fe_stream_t stream) {
  return span_prefill_f32(q, out, k_pool, v_pool, num_blocks, block_tables, table_stride,
                          q_offsets, context_lens, num_seqs, total_q, num_q_heads, kv_heads,
                          head_dim, block_size, scale, window, sinks, workspace, workspace_bytes,
                          stream);
}
