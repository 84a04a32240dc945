// Single-token paged decode over a window with sinks, and over 4-bit pools, for gfx950.
//
// A row at position p = L - 1 attends the keys j of its sequence with p - j < window and those
// with j < sinks (all keys without a window).  Pools are fp16, bf16 or fp32 in the plain
// decode's layout, or 4-bit rows (kv4.h).
//
// Work split: the plain decode's (fe_common.h): the keys that are walked -- 16-key tiles from
// the first to the sinks' last, then those from the one that holds the window's first key on,
// numbered through -- are cut into pieces of 64-key quads, about `target` per KV head over the
// whole batch; one 256-thread workgroup per (piece, KV head), wave w taking the piece's tiles
// w, w + 4, ...  Nothing is read of the pages between the sinks and the window, nor of their
// table entries.  The G query heads of a KV head are the 16 MFMA columns, so K and V are read
// once.  Pieces of one row are joined in the launch: each writes its normalised fp32 output
// and base-2 log-sum-exp with device-coherent stores, waits for them and draws a ticket; the
// last one merges and sets the ticket back to zero.
//
// One tile (lane l = 16g + n): S^T[16 keys x 16 heads] = K . Q^T, base-2 online softmax, O^T +=
// V^T . P^T as in attn_core.h.  4-bit rows: lane (g, n) loads dims g D/4 .. +D/4 of key n, for
// K and V alike -- at D = 128 one 16-byte chunk, whose 32 codes are exactly one block with one
// scale -- and converts them to 16 bits (16 conversions a lane for 32 values), K for the MFMA
// operand itself (any order of the dims does, if q is loaded in the same), V into the row-major
// LDS tile.
#include <type_traits>

#include "kv4.h"
#include "flexengine_amd_span.h"

using namespace fe;

namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;
constexpr int kMaxGroup = 16;
constexpr int kMaxTickets = 65536;
constexpr size_t kTicketBytes = kMaxTickets * sizeof(int);
constexpr int kMaxContext = 262144;  // kMaxPieces pieces of 64 quads
// Working workgroups in all that the default split aims at
constexpr int kDefaultWorkgroups = 512;
// A row of few keys is cut into at most this many short pieces: joining one costs about a
// quarter of what computing a quad does.  One row of 16384 tokens in 4 bits (12/2 heads of 128)
// with 64 / 32 / 16: 14.8 / 12.6 / 14.1 us; of 100000, whose pieces are long, 24.6.
constexpr int kFewPieces = 32;
// Tiles of a wave from which a 4-bit walk takes them two at a time, which has the matrix
// instructions with V take 32 keys and one round of the softmax serve both, but computes an odd
// last tile twice over: 37 rows of 2048-16384 tokens (32/8 heads of 128) one / two at a time
// 70.3 / 67.4 us (the loads alone 63), 64 rows of 128-4096 (12/2 heads) 11.5 / 12.6.
constexpr int kPairTiles = 16;

struct SpanArgs {
  const f16* q;
  f16* out;
  const f16* k_new;
  const f16* v_new;
  void* k_pool;   // 4-bit: codes
  void* v_pool;
  uint8_t* k_scales;
  uint8_t* v_scales;
  const int32_t* tables;
  const int32_t* ctx;
  float* ws_o;    // [pieces, Hq, D]
  float* ws_lse;  // [pieces, Hq] (base 2)
  int* tickets;   // [B, Hkv], zero between calls
  int64_t q_stride;
  int64_t new_stride;
  // Hkv: KV heads as the kernel sees them, hdiv of them per pool head (a group of more than 16
  // query heads is cut into hdiv groups of G that each read the pool head's K and V)
  int W, B, Hq, Hkv, G, BS, bs_log2, NB, target, hdiv;
  int dr;         // the real head_dim (PAD: below D)
  int max_len;
  float scale_log2;
  Span span;
  Q4Layout rows4;  // 4-bit pools
};

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
constexpr int kSc1 = 16;  // buffer-instruction cache policy: sc1 (device-coherent)
constexpr uint32_t kPastEnd = 0x7ffffff0u;  // an offset past every buffer: loads give zeros

__device__ __forceinline__ void store_coherent(float* p, float v) {
  __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float load_coherent(const float* p) {
  return __hip_atomic_load(const_cast<float*>(p), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void wait_stores() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

__device__ __forceinline__ __amdgpu_buffer_rsrc_t uniform_rsrc(const void* base, int bytes) {
  const uint64_t addr = reinterpret_cast<uint64_t>(base);
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)addr);
  const uint32_t hi = __builtin_amdgcn_readfirstlane((uint32_t)(addr >> 32));
  return __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void*>(((uint64_t)hi << 32) | lo), 0,
                                           __builtin_amdgcn_readfirstlane(bytes), 0x00020000);
}

// ---- rows of a tile in registers ---------------------------------------------------------

// 16-bit pools: K of lane (g, n) chunks 4s + g of key n, V in 16-byte chunks row by row
template <int D, class E, bool PAD>
struct Rows16 {
  using C = TileCfg<D>;
  struct Tile {
    f16x8 k[C::NK], v[C::NK];
  };
  struct NewRow {
    f16x8 k[C::NK], v;
  };
  const f16* k_pool;
  const f16* v_pool;
  int rs, hoff, dr;  // elements per pool row, offset of the head, real head_dim

  __device__ __forceinline__ void init(const SpanArgs& a, int hp) {
    k_pool = (const f16*)a.k_pool;
    v_pool = (const f16*)a.v_pool;
    rs = (a.Hkv / a.hdiv) * a.dr;
    hoff = hp * a.dr;
    dr = a.dr;
  }
  static __device__ __forceinline__ int q_dim(int s) { return (4 * s + (lane_id() >> 4)) * 8; }
  static __device__ __forceinline__ int pool_row(const SpanArgs& a, int blk, int off) {
    return blk * a.BS + off;
  }
  __device__ __forceinline__ void load(int row, int rows, Tile& t) const {
    const int64_t base = (int64_t)row * rs + hoff;
    const int bytes = rows > 0 ? ((rows - 1) * rs + dr) * 2 : 0;
    const __amdgpu_buffer_rsrc_t kr = uniform_rsrc(k_pool + base, bytes);
    const __amdgpu_buffer_rsrc_t vr = uniform_rsrc(v_pool + base, bytes);
    const int lane = lane_id();
    const uint32_t ko = (uint32_t)(((lane & 15) * rs + (lane >> 4) * 8) * 2);
    const uint32_t vo = (uint32_t)(((lane / C::CPR) * rs + (lane % C::CPR) * 8) * 2);
#pragma unroll
    for (int s = 0; s < C::NK; ++s) {
      t.k[s] = f16x8{};
      if (!PAD || q_dim(s) < dr) t.k[s] = ld(kr, ko + s * 64);
    }
#pragma unroll
    for (int j = 0; j < C::NK; ++j) {
      t.v[j] = f16x8{};
      if (!PAD || (lane % C::CPR) * 8 < dr) t.v[j] = ld(vr, vo + (uint32_t)(j * C::RPI * rs * 2));
    }
  }
  static __device__ __forceinline__ f16x8 ld(__amdgpu_buffer_rsrc_t r, uint32_t off) {
    return __builtin_bit_cast(f16x8, __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, kPagePolicy));
  }
  __device__ __forceinline__ void load_new(const f16* kr, const f16* vr, NewRow& nr) const {
    const int c = (lane_id() % C::CPR) * 8;
#pragma unroll
    for (int s = 0; s < C::NK; ++s)
      nr.k[s] = !PAD || q_dim(s) < dr ? ld16(kr + q_dim(s)) : f16x8{};
    nr.v = !PAD || c < dr ? ld16(vr + c) : f16x8{};
  }
  __device__ __forceinline__ void put_new(const NewRow& nr, int r, Tile& t) const {
    const int lane = lane_id();
#pragma unroll
    for (int s = 0; s < C::NK; ++s) t.k[s] = (lane & 15) == r ? nr.k[s] : t.k[s];
#pragma unroll
    for (int j = 0; j < C::NK; ++j) t.v[j] = j * C::RPI + lane / C::CPR == r ? nr.v : t.v[j];
  }
  // V of the keys that see() refuses as zeros
  template <class See>
  __device__ __forceinline__ void hide(Tile& t, See see) const {
#pragma unroll
    for (int j = 0; j < C::NK; ++j)
      if (!see(j * C::RPI + lane_id() / C::CPR)) t.v[j] = f16x8{};
  }
  __device__ __forceinline__ f16x8 key(const Tile& t, int s) const { return t.k[s]; }
  __device__ __forceinline__ void stage_v(const Tile& t, unsigned char* stage) const {
    const int lane = lane_id();
#pragma unroll
    for (int j = 0; j < C::NK; ++j)
      *reinterpret_cast<f16x8*>(stage + (j * C::RPI + lane / C::CPR) * C::ROWB +
                                (lane % C::CPR) * 16) = t.v[j];
  }
  __device__ __forceinline__ void store_new(const SpanArgs& a, const NewRow& nr, int row, int r) const {
    const int lane = lane_id();
    const int64_t base = (int64_t)(row + r) * rs + hoff;
    if ((lane & 15) == r)
#pragma unroll
      for (int s = 0; s < C::NK; ++s)
        if (!PAD || q_dim(s) < dr) st16((f16*)a.k_pool + base + q_dim(s), nr.k[s]);
    const int c = (lane % C::CPR) * 8;
    if (lane < C::CPR && (!PAD || c < dr)) st16((f16*)a.v_pool + base + c, nr.v);
  }
};

// 4-bit pools: dims g D/4 .. +D/4 of key n, K and V
template <int D, class E, bool PAD>
struct Rows4 {
  using C = TileCfg<D>;
  static constexpr int NW = D / 32;          // dwords of codes per lane and matrix
  static constexpr int NS = D > 128 ? 2 : 1;  // scales per lane and matrix
  struct Half {
    uint32_t c[NW];
    uint32_t s[NS];
  };
  struct Tile {
    Half k, v;
  };
  using NewRow = Tile;
  const uint8_t* kc;
  const uint8_t* vc;
  const uint8_t* ks;
  const uint8_t* vs;  // of the head
  Q4Layout at;
  int dr, bs_log2;

  __device__ __forceinline__ void init(const SpanArgs& a, int hp) {
    at = a.rows4;
    kc = (const uint8_t*)a.k_pool + at.code_offset(hp);
    vc = (const uint8_t*)a.v_pool + at.code_offset(hp);
    ks = a.k_scales + at.scale_offset(hp);
    vs = a.v_scales + at.scale_offset(hp);
    dr = a.dr;
    bs_log2 = a.bs_log2;
  }
  static __device__ __forceinline__ int dim0() { return (lane_id() >> 4) * (D / 4); }
  static __device__ __forceinline__ int q_dim(int s) { return dim0() + 8 * s; }
  static __device__ __forceinline__ int pool_row(const SpanArgs& a, int blk, int off) {
    return blk * a.BS + off;
  }
  __device__ __forceinline__ int block_of(int row) const { return row >> bs_log2; }
  __device__ __forceinline__ int offset_of(int row) const { return row & ((1 << bs_log2) - 1); }
  __device__ __forceinline__ void load_half(const uint8_t* codes, const uint8_t* scales, int row,
                                            int rows, Half& t) const {
    // from the first row to the end of the last one, nothing without rows (0 <= rows <= 16);
    // between them may be other heads' rows
    const int cs = (int)at.code_token * 16, ss = (int)at.scale_token;
    const int blk = block_of(row), off = offset_of(row);
    const __amdgpu_buffer_rsrc_t cr =
        uniform_rsrc(codes + at.code_row(blk, off), max(rows * cs - (cs - dr / 2), 0));
    const __amdgpu_buffer_rsrc_t sr = uniform_rsrc(
        scales + at.scale_row(blk, off), max(rows * ss - (ss - dr / kQ4Block), 0));
    const int n = lane_id() & 15;
    const uint32_t co = (uint32_t)(n * cs + dim0() / 2);
    const uint32_t so = (uint32_t)(n * ss + dim0() / kQ4Block);
    // (blocks past the real row come from past the descriptor's end: zeros)
    if constexpr (D == 64) {
      const bool on = !PAD || dim0() < dr;
      const u32x2 x = __builtin_bit_cast(
          u32x2, __builtin_amdgcn_raw_buffer_load_b64(cr, on ? co : kPastEnd, 0, kPagePolicy));
      t.c[0] = x[0];
      t.c[1] = x[1];
      t.s[0] = (uint8_t)__builtin_amdgcn_raw_buffer_load_b8(sr, on ? so : kPastEnd, 0, kPagePolicy);
    } else {
#pragma unroll
      for (int j = 0; j < NS; ++j) {
        const bool on = !PAD || dim0() + 32 * j < dr;
        const u32x4 x = __builtin_bit_cast(
            u32x4, __builtin_amdgcn_raw_buffer_load_b128(cr, on ? co + 16 * j : kPastEnd, 0,
                                                         kPagePolicy));
#pragma unroll
        for (int i = 0; i < 4; ++i) t.c[4 * j + i] = x[i];
        t.s[j] = (uint8_t)__builtin_amdgcn_raw_buffer_load_b8(sr, on ? so + j : kPastEnd, 0,
                                                              kPagePolicy);
      }
    }
  }
  __device__ __forceinline__ void load(int row, int rows, Tile& t) const {
    load_half(kc, ks, row, rows, t.k);
    load_half(vc, vs, row, rows, t.v);
  }
  // codes and scales of a 16-bit row, as the page write stores them
  __device__ __forceinline__ void pack(const f16* src, Half& t) const {
    float x[NW][8];
    uint32_t top[NS];
#pragma unroll
    for (int j = 0; j < NS; ++j) top[j] = 0;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const int d = dim0() + 8 * w;
      const f16x8 h = !PAD || d < dr ? ld16(src + d) : f16x8{};
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        x[w][i] = from16<E>(h[i]);
        top[w / 4] = max(top[w / 4], abs_bits(x[w][i]));
      }
    }
    // D = 64: a block spans the lanes g = 0, 1 or g = 2, 3
    if constexpr (D == 64) top[0] = max(top[0], (uint32_t)__shfl_xor((int)top[0], 16, kWave));
#pragma unroll
    for (int j = 0; j < NS; ++j) t.s[j] = q4_scale<E>(top[j]);
#pragma unroll
    for (int w = 0; w < NW; ++w) t.c[w] = q4_pack8(x[w], q4_scale_value(t.s[w / 4]));
  }
  __device__ __forceinline__ void load_new(const f16* kr, const f16* vr, NewRow& nr) const {
    pack(kr, nr.k);
    pack(vr, nr.v);
  }
  __device__ __forceinline__ void put_new(const NewRow& nr, int r, Tile& t) const {
    const bool mine = (lane_id() & 15) == r;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      t.k.c[w] = mine ? nr.k.c[w] : t.k.c[w];
      t.v.c[w] = mine ? nr.v.c[w] : t.v.c[w];
    }
#pragma unroll
    for (int j = 0; j < NS; ++j) {
      t.k.s[j] = mine ? nr.k.s[j] : t.k.s[j];
      t.v.s[j] = mine ? nr.v.s[j] : t.v.s[j];
    }
  }
  template <class See>
  __device__ __forceinline__ void hide(Tile& t, See see) const {
    if (see(lane_id() & 15)) return;
#pragma unroll
    for (int w = 0; w < NW; ++w) t.v.c[w] = 0;
#pragma unroll
    for (int j = 0; j < NS; ++j) t.v.s[j] = kQ4ScaleLow;
  }
  __device__ __forceinline__ f16x8 key(const Tile& t, int s) const {
    return q4_unpack8<E>(t.k.c[s], q4_scale_value(t.k.s[s / 4]));
  }
  __device__ __forceinline__ void stage_v(const Tile& t, unsigned char* stage) const {
    unsigned char* dst = stage + (lane_id() & 15) * C::ROWB + dim0() * 2;
#pragma unroll
    for (int w = 0; w < NW; ++w)
      *reinterpret_cast<f16x8*>(dst + 16 * w) =
          q4_unpack8<E>(t.v.c[w], q4_scale_value(t.v.s[w / 4]));
  }
  __device__ __forceinline__ void store_new(const SpanArgs& a, const NewRow& nr, int row, int r) const {
    if ((lane_id() & 15) != r) return;
    const int blk = block_of(row), off = offset_of(row) + r;  // (a tile lies in one page)
    const uint64_t co = at.code_row(blk, off) + dim0() / 2;
    const uint64_t so = at.scale_row(blk, off) + dim0() / kQ4Block;
#pragma unroll
    for (int w = 0; w < NW; ++w)
      if (!PAD || dim0() + 8 * w < dr) {
        *reinterpret_cast<uint32_t*>(const_cast<uint8_t*>(kc) + co + 4 * w) = nr.k.c[w];
        *reinterpret_cast<uint32_t*>(const_cast<uint8_t*>(vc) + co + 4 * w) = nr.v.c[w];
      }
#pragma unroll
    for (int j = 0; j < NS; ++j)
      if ((!PAD || dim0() + 32 * j < dr) && dim0() % kQ4Block == 0) {
        const_cast<uint8_t*>(ks)[so + j] = (uint8_t)nr.k.s[j];
        const_cast<uint8_t*>(vs)[so + j] = (uint8_t)nr.v.s[j];
      }
  }
};

// ---- the walk of one wave ----------------------------------------------------------------

__device__ __forceinline__ float vmax(float a, float b) { return __builtin_elementwise_maximum(a, b); }
// Maximum over the four lanes of a column (n, n + 16, n + 32, n + 48): permlane swaps, both
// halves of which are used, in the place of two LDS round trips
__device__ __forceinline__ float max_of_column(float x) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = vmax(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return vmax(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

// A wave's tiles, NT of them (1 or 2) at a time
template <int D, class E, class Rows>
struct SpanCore {
  using C = TileCfg<D>;
  using Tile = typename Rows::Tile;
  Rows rows;
  int L;          // context length
  int sinks, ws;  // keys below sinks and from ws on are seen
  float scale_log2;
  unsigned char* stage;
  int ntiles;     // tiles of this wave (<= 64)
  int row_vec;    // lane k < ntiles: pool row of tile k's first key
  int tok_vec;    // lane k < ntiles: its position
  int new_tile, new_row;  // the tile (-1: none) and key of it that is the decoded token
  typename Rows::NewRow fresh;
  f16x8 qv[C::NK];
  float m_run, l_run;
  f32x4 o[C::NX];

  // position of tile k's first key (L past the list: no key of it is seen)
  __device__ __forceinline__ int tile_tok(int k) const {
    const int t = __builtin_amdgcn_readlane(tok_vec, k & (kWave - 1));
    return k < ntiles ? t : L;
  }
  template <int NT>
  __device__ __forceinline__ void load(int k0, Tile (&t)[NT]) const {
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      // keys past the context read as zeros, tiles past the list are not read
      const int left = L - tile_tok(k0 + i);
      rows.load(__builtin_amdgcn_readlane(row_vec, (k0 + i) & (kWave - 1)),
                left < kTile ? left : kTile, t[i]);
    }
  }
  __device__ __forceinline__ bool sees(int tok) const {
    return tok < L && (tok < sinks || tok >= ws);
  }
  template <int NT>
  __device__ __forceinline__ void compute(int k0, Tile (&t)[NT]) {
    const int lane = lane_id();
    const int g = lane >> 4;
    const int n = lane & 15;
    if (new_tile >= k0 && new_tile < k0 + NT)
#pragma unroll
      for (int i = 0; i < NT; ++i)
        if (k0 + i == new_tile) rows.put_new(fresh, new_row, t[i]);
    float sv[NT][4];
    f32x4 sacc[NT];
#pragma unroll
    for (int i = 0; i < NT; ++i) sacc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < C::NK; ++s)
#pragma unroll
      for (int i = 0; i < NT; ++i) sacc[i] = mma32<E>(rows.key(t[i], s), qv[s], sacc[i]);
    float mx = kNegInf;
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      const int t0 = tile_tok(k0 + i);
#pragma unroll
      for (int j = 0; j < 4; ++j) sv[i][j] = sacc[i][j] * scale_log2;
      // whole tiles need no mask
      if (!(t0 + kTile <= L && (t0 >= ws || t0 + kTile <= sinks))) {
        rows.hide(t[i], [&](int r) { return sees(t0 + r); });
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (!sees(t0 + 4 * g + j)) sv[i][j] = kNegInf;
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) mx = vmax(mx, sv[i][j]);
    }
    mx = max_of_column(mx);
    if (__ballot(mx > m_run + kRescaleSlack)) {  // wave-uniform
      const float m_new = fmaxf(m_run, mx);
      const float alpha = m_new == kNegInf ? 1.f : exp2_fast(m_run - m_new);
      l_run *= alpha;
#pragma unroll
      for (int x = 0; x < C::NX; ++x) o[x] *= alpha;
      m_run = m_new;
    }
    const float m_use = m_run == kNegInf ? 0.f : m_run;
    // probabilities in 16 bits for the matrix instruction (at most 2^kRescaleSlack)
    f16x4 pb[NT];
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      float p[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) p[j] = exp2_fast(sv[i][j] - m_use);
      pb[i] = to16x4<E>(p[0], p[1], p[2], p[3]);
      // the sum takes the rounded ones: what multiplies V adds up to one
      l_run = sum4<E>(pb[i], l_run);
    }
    const unsigned char* vb = stage + (4 * g + (n >> 2)) * C::ROWB + (n & 3) * 8;
    auto vfrag = [&](const unsigned char* at) __attribute__((always_inline)) {
      return __builtin_bit_cast(f16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                           (__attribute__((address_space(3))) s16x4*)at));
    };
    compiler_fence();
#pragma unroll
    for (int i = 0; i < NT; ++i) rows.stage_v(t[i], stage + i * C::STAGE);
    compiler_fence();
#pragma unroll
    for (int x = 0; x < C::NX; ++x) {
      const f16x4 a = vfrag(vb + 32 * x);
      if constexpr (NT == 2) {
        const f16x4 b = vfrag(vb + C::STAGE + 32 * x);
        o[x] = mma32<E>(f16x8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]},
                        f16x8{pb[0][0], pb[0][1], pb[0][2], pb[0][3], pb[1][0], pb[1][1], pb[1][2],
                              pb[1][3]},
                        o[x]);
      } else {
        o[x] = mma16<E>(a, pb[0], o[x]);
      }
    }
    compiler_fence();
  }
  // two sets of tiles in registers: while one is computed, the loads of the next are in flight
  template <int NT>
  __device__ __forceinline__ void run_by() {
    Tile ta[NT], tb[NT];
    load(0, ta);
    for (int k = 0;; k += 2 * NT) {
      load(k + NT, tb);
      if (k >= ntiles) break;
      compute(k, ta);
      load(k + 2 * NT, ta);
      if (k + NT >= ntiles) break;
      compute(k + NT, tb);
    }
  }
  template <int MAX>
  __device__ __forceinline__ void run() {
    m_run = kNegInf;
    l_run = 0.f;
#pragma unroll
    for (int x = 0; x < C::NX; ++x) o[x] = f32x4{0.f, 0.f, 0.f, 0.f};
    if constexpr (MAX == 2) {
      if (ntiles >= kPairTiles) return run_by<2>();
    }
    run_by<1>();
  }
  __device__ __forceinline__ float l_total() const {
    float l = l_run + shfl_xor_f(l_run, 16);
    return l + shfl_xor_f(l, 32);
  }
};

// ---- the join of a row's pieces ------------------------------------------------------------

// Pieces read in one round trip (16 hold the walk to 2 or 3 waves a SIMD instead of 4: 16-bit
// windows of 1024, 64 rows of 32/8 heads of 128, 65.2 / 61.1 us)
constexpr int kMergeBatch = 8;

// out = sum_s 2^(lse_s - M) o_s / sum_s 2^(lse_s - M) over the ns pieces from slot `first` on;
// a thread takes 4 dims of a query head
template <int D, class E, bool PAD>
__device__ __forceinline__ void merge_pieces(const SpanArgs& a, int b, int h, int first, int ns) {
  const int G = a.G;
  const int o_step = a.Hq * D;
  const float* lse_base = a.ws_lse + (int64_t)first * a.Hq + h * G;
  // one descriptor over the ns slots (the host keeps the partials under 2 GiB)
  const __amdgpu_buffer_rsrc_t ro = __builtin_amdgcn_make_buffer_rsrc(
      a.ws_o + ((int64_t)first * a.Hq + h * G) * D, 0, ns * o_step * (int)sizeof(float),
      0x00020000);
  for (int e4 = threadIdx.x; e4 < G * D / 4; e4 += kThreads) {
    const int hh = e4 * 4 / D;
    float M = kNegInf, den = 0.f;
    f32x4 num = {0.f, 0.f, 0.f, 0.f};
    for (int s0 = 0; s0 < ns; s0 += kMergeBatch) {
      const int nb = ns - s0 < kMergeBatch ? ns - s0 : kMergeBatch;  // wave-uniform
      float lv[kMergeBatch];
      f32x4 ov[kMergeBatch];
#pragma unroll
      for (int u = 0; u < kMergeBatch; ++u) {
        lv[u] = kNegInf;
        ov[u] = f32x4{0.f, 0.f, 0.f, 0.f};
        if (u < nb) {
          lv[u] = load_coherent(lse_base + (int64_t)(s0 + u) * a.Hq + hh);
          ov[u] = __builtin_bit_cast(
              f32x4, __builtin_amdgcn_raw_buffer_load_b128(
                         ro, (uint32_t)(((s0 + u) * o_step + e4 * 4) * sizeof(float)), 0, kSc1));
        }
      }
      float bm = M;
#pragma unroll
      for (int u = 0; u < kMergeBatch; ++u) bm = fmaxf(bm, lv[u]);
      const float alpha = M == kNegInf ? 0.f : exp2f(M - bm);
      num *= alpha;
      den *= alpha;
#pragma unroll
      for (int u = 0; u < kMergeBatch; ++u) {
        const float wv = lv[u] == kNegInf ? 0.f : exp2f(lv[u] - bm);
        num += wv * ov[u];
        den += wv;
      }
      M = bm;
    }
    const int d = e4 * 4 - hh * D;  // the partials keep D's layout
    if (!PAD || d < a.dr)
      store_out4<E>(a.out, ((int64_t)b * a.Hq + h * G + hh) * (PAD ? a.dr : D) + d,
                    num * (den > 0.f ? 1.f / den : 0.f));
  }
}

// Tiles that a wave computes at a time, at most
// (16-bit tiles two at a time: 61.1 -> 65.1 us)
template <bool Q4>
constexpr int kTilesAtOnce = Q4 ? 2 : 1;

// LDS: the waves' V tiles, and in their place after the walk the waves' states (o, m, l) for
// the combine; a flag
template <int D, int NT>
struct SpanLds {
  static constexpr size_t per_wave = (NT > 1 ? 2 : 1) * TileCfg<D>::STAGE;
  static constexpr size_t park_m = (size_t)kWaves * TileCfg<D>::NX * kWave * 16;
  static constexpr size_t park_l = park_m + (size_t)kWaves * kWave * sizeof(float);
  static constexpr size_t parked = park_l + (size_t)kWaves * kWave * sizeof(float);
  static constexpr size_t flag = parked > kWaves * per_wave ? parked : kWaves * per_wave;
  static constexpr size_t bytes = flag + sizeof(int);
};

template <int D, class E, bool Q4, bool PAD>
__global__ __launch_bounds__(kThreads)
// (D = 256: one wave per SIMD, as the plain decode.  4-bit: four waves a SIMD against the
// latency of a tile's chain, 74 -> 67 us for the long rows above; the padded form spills there)
__attribute__((amdgpu_waves_per_eu(D > 128 ? 1 : (Q4 ? (PAD ? 3 : 4) : 2), 8)))
void span_decode_kernel(const SpanArgs a) {
  using C = TileCfg<D>;
  constexpr int NT = kTilesAtOnce<Q4>;
  using Lds = SpanLds<D, NT>;
  extern __shared__ __align__(16) unsigned char smem[];
  const int DR = PAD ? a.dr : D;
  const int h = blockIdx.x % a.Hkv;
  const int item = blockIdx.x / a.Hkv;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = lane_id();
  const int g = lane >> 4;
  const int n = lane & 15;
  const int G = a.G;
  const int span_head = (int)(((unsigned)a.span.sinks + kTile - 1) / kTile);

  Piece pc;
  int total = 0;
  const auto walk = [&](int L) __attribute__((always_inline)) {
    return L - kTile * span_skip(a.span, window_start(a.span, L - 1), kTile);
  };
  if (!find_piece(a.ctx, nullptr, a.B, a.max_len, a.target, item, pc, total, walk,
                  kFewPieces)) {
    // past the last piece: zero rows of empty sequences
    const int b = item - total;
    if (b < a.B && seq_len(a.ctx, b, a.max_len) == 0)
      for (int e = threadIdx.x; e < G * DR; e += kThreads)
        store_out1<E>(a.out, ((int64_t)b * a.Hq + h * G) * DR + e, 0.f);
    return;
  }
  const int b = pc.b;
  const int hp = h / a.hdiv;
  const int ws = window_start(a.span, pc.L - 1);
  const int skip = span_skip(a.span, ws, kTile);
  const int t_first = pc.tok_begin / kTile + w;
  const int t_end = (pc.tok_end + kTile - 1) / kTile;
  const int hq = h * G + (n < G ? n : G - 1);
  const int64_t q_row = (int64_t)b * a.q_stride + (int64_t)hq * DR;
  const int64_t new_row = (int64_t)b * a.new_stride + (int64_t)hp * DR;

  float m_run, l_tot;
  f32x4 o[C::NX];
  if constexpr (kIsF32<E>) {
    using Core = F32Core<D, true, PAD, 1, true>;
    Core core;
    core.k_pool = (const float*)a.k_pool;
    core.v_pool = (const float*)a.v_pool;
    core.k_pool_w = (float*)a.k_pool;
    core.v_pool_w = (float*)a.v_pool;
    core.trow = a.tables + (int64_t)b * a.W;
    core.rs = (a.Hkv / a.hdiv) * DR;
    core.hoff = hp * DR;
    core.dr = DR;
    core.W = a.W;
    core.NB = a.NB;
    core.BS = a.BS;
    core.bs_log2 = a.bs_log2;
    core.tok_end = pc.L;
    core.limit[0] = pc.L;
    core.scale_log2 = a.scale_log2;
    core.span_head = span_head;
    core.span_skip = skip;
    core.sinks = a.span.sinks;
    core.wmin = ws;
    core.wlo[0] = ws;
    core.new_pos = -1;
    core.knew_row = nullptr;
    core.vnew_row = nullptr;
    if (a.k_new != nullptr) {
      core.knew_row = (const float*)a.k_new + new_row;
      core.vnew_row = (const float*)a.v_new + new_row;
      const int blk = core.trow[(pc.L - 1) >> a.bs_log2];
      if (blk >= 0 && blk < a.NB) core.new_pos = pc.L - 1;
    }
    const float* qr = (const float*)a.q + q_row;
#pragma unroll
    for (int c = 0; c < Core::NC; ++c) {
      f32x4 v = {0.f, 0.f, 0.f, 0.f};
      if (n < G && (!PAD || 16 * c + 4 * g < DR)) v = *reinterpret_cast<const f32x4*>(qr + 16 * c + 4 * g);
      core.qv[0][c] = v;
    }
    core.init_acc();
    core.run(t_first, kWaves, t_end);
    m_run = core.m_run[0];
    l_tot = core.l_total();
#pragma unroll
    for (int x = 0; x < C::NX; ++x) o[x] = core.o[0][x];
  } else {
    using Rows = std::conditional_t<Q4, Rows4<D, E, PAD>, Rows16<D, E, PAD>>;
    SpanCore<D, E, Rows> core;
    core.rows.init(a, hp);
    core.L = pc.L;
    core.sinks = a.span.sinks;
    core.ws = ws;
    core.scale_log2 = a.scale_log2;
    core.stage = smem + w * Lds::per_wave;
    core.ntiles = t_first < t_end ? (t_end - t_first + kWaves - 1) / kWaves : 0;
    int blk = 0, tok = 0;
    if (lane < core.ntiles) {
      const int t = t_first + lane * kWaves;
      tok = (t < span_head ? t : t + skip) * kTile;
      blk = a.tables[(int64_t)b * a.W + (tok >> a.bs_log2)];
    }
    core.tok_vec = tok;
    core.row_vec = Rows::pool_row(a, clamp_block(blk, a.NB), tok & (a.BS - 1));
#pragma unroll
    for (int s = 0; s < C::NK; ++s) {
      const int d = Rows::q_dim(s);
      core.qv[s] = n < G && (!PAD || d < DR) ? ld16(a.q + q_row + d) : f16x8{};
    }
    // the decoded token's row comes from k_new / v_new where this wave has its tile
    core.new_tile = -1;
    core.new_row = (pc.L - 1) & (kTile - 1);
    if (a.k_new != nullptr) {
      const unsigned long long hit =
          __ballot(lane < core.ntiles && pc.L - 1 >= tok && pc.L - 1 < tok + kTile);
      if (hit) {
        core.new_tile = __builtin_ctzll(hit);
        core.rows.load_new(a.k_new + new_row, a.v_new + new_row, core.fresh);
      }
    }
    core.template run<NT>();
    if (core.new_tile >= 0) {
      // (no page write through a table entry that is not a block)
      const int id = __builtin_amdgcn_readlane(blk, core.new_tile);
      if (id >= 0 && id < a.NB)
        core.rows.store_new(a, core.fresh, __builtin_amdgcn_readlane(core.row_vec, core.new_tile),
                            core.new_row);
    }
    m_run = core.m_run;
    l_tot = core.l_total();
#pragma unroll
    for (int x = 0; x < C::NX; ++x) o[x] = core.o[x];
  }

  // ---- combine the four waves through LDS: wave w takes output tiles w XW .. +XW ----
  __syncthreads();  // the V tiles are done with
  f32x4* park = reinterpret_cast<f32x4*>(smem);  // [4][NX][64]
  float* park_m = reinterpret_cast<float*>(smem + Lds::park_m);
  float* park_l = reinterpret_cast<float*>(smem + Lds::park_l);
  int* flag = reinterpret_cast<int*>(smem + Lds::flag);
  constexpr int XW = C::NX / kWaves;
  const auto dim0 = [g](int x) { return kIsF32<E> ? f32_dim0(x, g) : 16 * x + 4 * g; };
#pragma unroll
  for (int x = 0; x < C::NX; ++x) park[(w * C::NX + x) * kWave + lane] = o[x];
  park_m[w * kWave + lane] = m_run;
  park_l[w * kWave + lane] = l_tot;
  __syncthreads();
  float M = kNegInf, den = 0.f, sc[kWaves];
#pragma unroll
  for (int v = 0; v < kWaves; ++v) M = fmaxf(M, park_m[v * kWave + lane]);
#pragma unroll
  for (int v = 0; v < kWaves; ++v) {
    const float mv = park_m[v * kWave + lane];
    sc[v] = mv == kNegInf ? 0.f : exp2f(mv - M);
    den += sc[v] * park_l[v * kWave + lane];
  }
  // (a piece of the last keys before a window may see none of its own: it adds nothing)
  const float inv = den > 0.f ? 1.f / den : 0.f;
  f32x4 ox[XW];
#pragma unroll
  for (int xi = 0; xi < XW; ++xi) {
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int v = 0; v < kWaves; ++v)
      acc += sc[v] * park[(v * C::NX + w * XW + xi) * kWave + lane];
    ox[xi] = acc * inv;
  }
  if (pc.nsplit == 1) {
    if (n < G) {
      const int64_t orow = ((int64_t)b * a.Hq + hq) * DR;
#pragma unroll
      for (int xi = 0; xi < XW; ++xi)
        if (!PAD || dim0(w * XW + xi) < DR)
          store_out4<E>(a.out, orow + dim0(w * XW + xi), ox[xi]);
    }
    return;
  }
  if (n < G) {
    const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(
        a.ws_o + ((int64_t)pc.id * a.Hq + h * G) * D, 0, G * D * (int)sizeof(float), 0x00020000);
#pragma unroll
    for (int xi = 0; xi < XW; ++xi)
      __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, ox[xi]), r,
                                             (n * D + dim0(w * XW + xi)) * (uint32_t)sizeof(float),
                                             0, kSc1);
    if (w == 0 && g == 0)
      store_coherent(a.ws_lse + (int64_t)pc.id * a.Hq + hq,
                     den > 0.f ? M + log2f(den) : kNegInf);
  }
  int* const ticket = a.tickets + b * a.Hkv + h;
  wait_stores();  // this wave's partials are complete at the device-coherent level
  __syncthreads();
  if (threadIdx.x == 0)
    *flag = __hip_atomic_fetch_add(ticket, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) ==
            pc.nsplit - 1;
  __syncthreads();
  if (!*flag) return;
  if (threadIdx.x == 0) __hip_atomic_store(ticket, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  merge_pieces<D, E, PAD>(a, b, h, pc.id - pc.split, pc.nsplit);
}

// ---- host ------------------------------------------------------------------------------------

inline size_t align256(size_t x) { return (x + 255) & ~size_t(255); }
inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
inline int log2_exact(int x) {
  if (x <= 0 || (x & (x - 1))) return -1;
  int l = 0;
  while ((1 << l) < x) ++l;
  return l;
}
inline int computed_dim(int d) { return d <= 64 ? 64 : (d <= 128 ? 128 : 256); }

// Query heads of a KV head are at most 16 MFMA columns: the smallest divisor of the group that
// leaves no more
inline int head_split(int group) {
  int v = (group + kMaxGroup - 1) / kMaxGroup;
  while (group % v) ++v;
  return v;
}

// Split target that keeps a piece within 64 quads (64 tiles per wave) for any lengths
inline int split_target(int batch, int kv_heads, int max_len, int target_splits) {
  int t = target_splits > 0 ? target_splits
                            : (kDefaultWorkgroups > kv_heads ? kDefaultWorkgroups / kv_heads : 1);
  const int64_t quads = ((int64_t)max_len + 63) / 64;
  const int64_t need = ((int64_t)batch * quads + 63) / 64;
  return need > t ? (int)need : t;
}

struct SpanWorkspace {
  size_t o, lse, bytes;  // offsets of the partials and the LSEs
};
inline SpanWorkspace workspace_of(int batch, int hq, int d, int target) {
  SpanWorkspace w;
  const size_t slots = (size_t)target + batch;
  w.o = kTicketBytes;
  w.lse = w.o + align256(slots * hq * computed_dim(d) * sizeof(float));
  w.bytes = w.lse + align256(slots * hq * sizeof(float));
  return w;
}

template <int D, class E, bool Q4, bool PAD>
int launch(const SpanArgs& a, hipStream_t s) {
  hipLaunchKernelGGL((span_decode_kernel<D, E, Q4, PAD>), dim3((a.target + 2 * a.B) * a.Hkv),
                     dim3(kThreads), (SpanLds<D, kTilesAtOnce<Q4>>::bytes), s, a);
  return FE_LAUNCH_STATUS();
}
template <class E, bool Q4>
int launch_dim(const SpanArgs& a, hipStream_t s) {
  if (a.dr == 64) return launch<64, E, Q4, false>(a, s);
  if (a.dr == 128) return launch<128, E, Q4, false>(a, s);
  if (a.dr < 64) return launch<64, E, Q4, true>(a, s);
  if (a.dr < 128) return launch<128, E, Q4, true>(a, s);
  if constexpr (!kIsF32<E>) {
    if (a.dr == 256) return launch<256, E, Q4, false>(a, s);
    return launch<256, E, Q4, true>(a, s);
  }
  return FE_ERR_UNSUPPORTED;
}

template <class E, bool Q4>
int span_decode(const void* q, int64_t q_stride, void* out, const void* k_new, const void* v_new,
                int64_t new_stride, void* k_pool, void* k_scales, void* v_pool, void* v_scales,
                const fe_kv4_strides* strides, int num_blocks, const int32_t* tables, int table_stride, const int32_t* ctx,
                void* workspace, size_t workspace_bytes, int batch, int hq, int hkv, int d, int bs,
                float scale, int window, int sinks, int target_splits, fe_stream_t stream) {
  FE_CHECK_ARG(batch >= 0 && hq > 0 && hkv > 0 && d > 0 && num_blocks > 0 && table_stride > 0 &&
               target_splits >= 0 && window >= 0 && sinks >= 0);
  FE_CHECK_ARG(hq % hkv == 0);
  FE_CHECK_ARG(Q4 || window > 0);
  const int bs_log2 = log2_exact(bs);
  if (bs_log2 < 0 || bs % kTile != 0) return FE_ERR_UNSUPPORTED;
  if (Q4 ? (d % kQ4Block != 0 || d > 256) : (d % 8 != 0 || d > (kIsF32<E> ? 128 : 256)))
    return FE_ERR_UNSUPPORTED;
  const int hdiv = head_split(hq / hkv);
  const int hkv_v = hkv * hdiv;
  if ((int64_t)batch * hkv_v > kMaxTickets) return FE_ERR_UNSUPPORTED;
  if ((int64_t)table_stride * bs > kMaxContext) return FE_ERR_UNSUPPORTED;
  // pool rows are 32-bit in the kernels, and so are the offsets within a tile's 16 rows
  if ((int64_t)num_blocks * bs >= ((int64_t)1 << 31) ||
      (int64_t)hkv * d >= ((int64_t)1 << 25))
    return FE_ERR_UNSUPPORTED;
  const int max_len = table_stride * bs;
  const int target = split_target(batch, hkv_v, max_len, target_splits);
  if (((int64_t)target + batch) * hq * computed_dim(d) * (int64_t)sizeof(float) >= ((int64_t)1 << 31) ||
      ((int64_t)target + 2 * (int64_t)batch) * hkv_v >= ((int64_t)1 << 31))
    return FE_ERR_UNSUPPORTED;
  if (batch == 0) return FE_OK;
  FE_CHECK_ARG(q && out && k_pool && v_pool && tables && ctx);
  FE_CHECK_ARG((k_new == nullptr) == (v_new == nullptr));
  // 16-byte loads of q and of the new rows
  const int per16 = kIsF32<E> ? 4 : 8;
  FE_CHECK_ARG(q_stride % per16 == 0 && q_stride >= (int64_t)hq * d);
  FE_CHECK_ARG(aligned16(q) && aligned16(out) && aligned16(k_pool) && aligned16(v_pool));
  Q4Layout rows4{};
  if (Q4) {
    FE_CHECK_ARG(k_scales && v_scales);
    if (int rc = q4_layout(strides, num_blocks, hkv, d, bs, rows4)) return rc;
  }
  if (k_new)
    FE_CHECK_ARG(aligned16(k_new) && aligned16(v_new) && new_stride % per16 == 0 &&
                 new_stride >= (int64_t)hkv * d);
  const SpanWorkspace w = workspace_of(batch, hq, d, target);
  if (workspace == nullptr || workspace_bytes < w.bytes || !aligned16(workspace))
    return FE_ERR_WORKSPACE;
  SpanArgs a{};
  a.q = (const f16*)q;
  a.out = (f16*)out;
  a.k_new = (const f16*)k_new;
  a.v_new = (const f16*)v_new;
  a.k_pool = k_pool;
  a.v_pool = v_pool;
  a.k_scales = (uint8_t*)k_scales;
  a.v_scales = (uint8_t*)v_scales;
  a.tables = tables;
  a.ctx = ctx;
  a.tickets = (int*)workspace;
  a.ws_o = (float*)((char*)workspace + w.o);
  a.ws_lse = (float*)((char*)workspace + w.lse);
  a.q_stride = q_stride;
  a.new_stride = new_stride;
  a.W = table_stride;
  a.B = batch;
  a.Hq = hq;
  a.Hkv = hkv_v;
  a.G = hq / hkv_v;
  a.BS = bs;
  a.bs_log2 = bs_log2;
  a.NB = num_blocks;
  a.target = target;
  a.hdiv = hdiv;
  a.dr = d;
  a.max_len = max_len;
  a.scale_log2 = scale * kLog2e;
  a.span = Span{window, window > 0 ? sinks : 0};
  a.rows4 = rows4;
  return launch_dim<E, Q4>(a, (hipStream_t)stream);
}

}  // namespace

extern "C" size_t fe_span_decode_workspace_size(int batch, int num_q_heads, int kv_heads,
                                                int head_dim, int max_context, int target_splits) {
  if (batch < 0 || num_q_heads <= 0 || kv_heads <= 0 || num_q_heads % kv_heads || head_dim <= 0 ||
      max_context < 0 || target_splits < 0)
    return 0;
  const int hkv_v = kv_heads * head_split(num_q_heads / kv_heads);
  return workspace_of(batch, num_q_heads, head_dim,
                      split_target(batch, hkv_v, max_context, target_splits))
      .bytes;
}

#define FE_WINDOW_DECODE(SUFFIX, E)                                                               \
  extern "C" int fe_paged_decode_window##SUFFIX(                                                  \
      const void* q, int64_t q_batch_stride, void* out, const void* k_new, const void* v_new,     \
      int64_t new_batch_stride, void* k_pool, void* v_pool, int num_blocks,                       \
      const int32_t* block_tables, int table_stride, const int32_t* context_lens,                 \
      void* workspace, size_t workspace_bytes, int batch, int num_q_heads, int kv_heads,          \
      int head_dim, int block_size, float scale, int window, int sinks, int target_splits,        \
      fe_stream_t stream) {                                                                       \
    return span_decode<E, false>(q, q_batch_stride, out, k_new, v_new, new_batch_stride, k_pool,  \
                                 nullptr, v_pool, nullptr, nullptr, num_blocks, block_tables,     \
                                 table_stride, context_lens, workspace, workspace_bytes, batch,   \
                                 num_q_heads, kv_heads, head_dim, block_size, scale, window,      \
                                 sinks, target_splits, stream);                                   \
  }
FE_WINDOW_DECODE(, Fp16)
FE_WINDOW_DECODE(_bf16, Bf16)
FE_WINDOW_DECODE(_f32, F32)

#define FE_KV4_DECODE(SUFFIX, E, STRIDES_PARAM, STRIDES)                                          \
  extern "C" int fe_paged_decode_kv4##SUFFIX(                                                     \
      const void* q, int64_t q_batch_stride, void* out, const void* k_new, const void* v_new,     \
      int64_t new_batch_stride, void* k_codes, void* k_scales, void* v_codes, void* v_scales,     \
      STRIDES_PARAM int num_blocks, const int32_t* block_tables, int table_stride,                \
      const int32_t* context_lens, void* workspace, size_t workspace_bytes, int batch,            \
      int num_q_heads, int kv_heads, int head_dim, int block_size, float scale, int window,       \
      int sinks, int target_splits, fe_stream_t stream) {                                         \
    return span_decode<E, true>(q, q_batch_stride, out, k_new, v_new, new_batch_stride, k_codes,  \
                                k_scales, v_codes, v_scales, STRIDES, num_blocks, block_tables,   \
                                table_stride, context_lens, workspace, workspace_bytes, batch,    \
                                num_q_heads, kv_heads, head_dim, block_size, scale, window,       \
                                sinks, target_splits, stream);                                    \
  }
#define FE_STRIDES_PARAM const fe_kv4_strides *strides,
FE_KV4_DECODE(, Fp16, , nullptr)
FE_KV4_DECODE(_bf16, Bf16, , nullptr)
FE_KV4_DECODE(_strided, Fp16, FE_STRIDES_PARAM, strides)
FE_KV4_DECODE(_strided_bf16, Bf16, FE_STRIDES_PARAM, strides)
