// Ragged causal prefill under a window with sinks, and over 4-bit pools, for gfx950.
//
// Sequence s contributes the query rows q_off[s] .. q_off[s + 1] - 1, the last n_s positions of
// its context; a query at position p sees the keys j <= p with p - j < window and those with
// j < sinks (without a window every j <= p).
//
// Work split: for one KV head the rows of a sequence are the pairs (position, query head of the
// group), position-major (row r: position r / G), so the G heads share what is read of K and V.
// A unit is 32 * NW such rows of one sequence and KV head, one workgroup of NW waves of 32 rows
// each; it walks the 16-key tiles from the first to the sinks' last and then from the one that
// holds its first row's window start to its last row's position, four at a time.  Tiles between
// are not read, keys that no row of the unit sees are taken as zeros (their pages may hold
// anything).  Where the units are too few for the chip, up to KS workgroups share one, each an
// equal run of its blocks: each writes its normalised fp32 state and base-2 log-sum-exps with
// device-coherent stores, waits for them and draws a ticket; the last one joins them and sets the
// ticket back to zero.
//
// One block of four tiles (lane (hf, n) = (lane / 32, lane % 32) holds row n of its wave), both
// products on v_mfma_f32_32x32x16:
//   S^T[32 keys x 32 rows] = K.Q^T, two key tiles; register i holds the score of key 8 (i / 4)
//     + 4 hf + i % 4 of the tile, so a row's maximum takes one exchange between the halves;
//   base-2 online softmax with the lazy rescale, masks only on blocks at an edge of some row;
//   O^T[32 dims x 32 rows] += V^T.P^T: the probabilities are the B operand as they stand, two
//     transposing LDS reads give the A operand the same keys.
//
// K and V of a block sit in LDS as 16-bit rows whose 16-byte chunks are XOR-swizzled (all 64
// banks busy in both reads), two stages: while one block is computed the next arrives.  16-bit
// pools come by LDS DMA (buffer_load ... lds), one 8- or 16-key run a wave.  4-bit pools come
// through registers: a thread loads 16-byte chunks -- 32 codes, one block with one scale --
// two blocks ahead, and converts them (16 conversions and four 16-byte LDS writes a chunk) one
// block ahead; at D = 128 and NW = 8 that is one chunk a thread and block, beside the 32 matrix
// instructions of its wave.
#pragma once

#include "kv4.h"
#include "flexengine_amd_span.h"

namespace fe {
namespace {

constexpr int kSpanKeys = 64;      // keys per staged block
// Workgroups that run at once (two of four waves on each of 256 CUs)
constexpr int kSpanSlots = 512;
// Key splits have at least kSpanShare blocks, fewer down to kSpanShareLow where that leaves no
// more than half the workgroups that run at once (two on a CU take nearly twice as long each), and
// a unit is split into two such at least.  12/2 heads of 128 in 4 bits, six blocks at least / fewer
// by that rule / four always: 500 fresh tokens 19.2, 17.9, 17.8 us; 500 over 600 cached 21.8, 18.9,
// 18.8; 50 over 2000 21.6, 20.4, 20.3; 16 over 4000 22.0, 22.6, 22.4; four chunks of 400 over up to
// 500 25.2, 25.3, 25.9; eight of 64 over up to 4000 33.5, 33.7, 42.1 (eight blocks at least: 34.1).
constexpr int kSpanShare = 6;
constexpr int kSpanShareLow = 4;
constexpr int kSpanMaxSplits = 16;
typedef uint32_t span_u32x4 __attribute__((ext_vector_type(4)));
constexpr int kSpanTickets = 65536;
constexpr size_t kSpanTicketBytes = kSpanTickets * sizeof(int);
constexpr int64_t kSpanPartBytes = (int64_t)1 << 28;  // of all split states: fewer splits past it
constexpr int kSpanSc1 = 16;       // buffer-instruction cache policy: sc1 (device-coherent)
// Blocks of a walk over which the reference of the softmax follows every block's maximum in
// either direction (the probabilities' rounding is then relative to the block's own largest);
// after them it lags by up to kRescaleSlack.  4095 tokens over a 4-bit cache, 8191 under a
// window of 1024 (bf16): 142 and 164 us, 2.0e-3 and 2.1e-3 from 64 bits (the output's rounding
// alone is 1.6e-3); with a slack of 2, as the wide 16-bit prefill has, 148 and 168 us, 1.9e-3
// and 2.0e-3.
constexpr int kSpanFollow = 2;

struct SpanPrefill {
  const f16* q;
  f16* out;
  const void* k_pool;  // 4-bit: codes
  const void* v_pool;
  const uint8_t* k_scales;
  const uint8_t* v_scales;
  const int32_t* tables;
  const int32_t* q_off;
  const int32_t* ctx;
  unsigned char* parts;  // [units][Hkv][KS] split states
  int* tickets;     // [units bound][Hkv], zero between calls
  int W, S, total_q, Hq, Hkv, G, BS, bs_log2, NB, KS, units;
  int dr;            // the real head_dim (PAD: below D)
  float scale_log2;
  Span span;
  Q4Layout rows4;  // 4-bit pools
};

// The 16-key tiles that a run of query rows walks: those of the sinks, then those from the one
// that holds the first row's window start to the last row's position
struct SpanWalk {
  int head, skip;  // tiles head, head + 1, ... of the walk are `skip` tiles further on
  int key_end, ws, sinks;
  __device__ __forceinline__ void init(const Span& sp, int first_pos, int last_pos) {
    key_end = last_pos + 1;
    sinks = sp.sinks;
    ws = window_start(sp, first_pos);
    head = (int)(((unsigned)sp.sinks + kTile - 1) / kTile);
    skip = span_skip(sp, ws, kTile);
  }
  // 64-key blocks of four tiles
  __device__ __forceinline__ int blocks() const {
    return ((key_end + kTile - 1) / kTile - skip + 3) / 4;
  }
  // first key of tile t (past the last one: keys past key_end)
  __device__ __forceinline__ int key(int t) const { return (t < head ? t : t + skip) * kTile; }
  __device__ __forceinline__ bool sees(int k) const {
    return k < key_end && (k < sinks || k >= ws);
  }
};

// A unit of work: rows r0 .. r0 + ROWS - 1 (fewer at the end) of sequence s
struct SpanUnit {
  int s, block, n, q0, ctx;
};
// All units of one KV head: how many, and about how many key blocks they walk (each sequence's
// mean of its first and last unit's)
struct SpanWork {
  int units, blocks;
};
// Finds unit `item`, and with key splits counts the work.
template <int ROWS>
__device__ __forceinline__ bool find_unit(const SpanPrefill& a, int item, SpanUnit& u,
                                          SpanWork& work) {
  const int lane = lane_id();
  int carry = 0;
  bool found = false;
  work = SpanWork{0, 0};
  for (int base = 0; base < a.S; base += kWave) {
    const int s = base + lane < a.S ? base + lane : a.S - 1;
    const int e0 = a.q_off[s], e1 = a.q_off[s + 1], cx = clamp_len(a.ctx[s]);
    // rows outside [0, total_q) are dropped
    const int q0 = min(max(e0, 0), a.total_q);
    const int n = base + lane < a.S ? max(min(e1, a.total_q) - q0, 0) : 0;
    const int nb = (int)(((int64_t)n * a.G + ROWS - 1) / ROWS);
    if (a.KS > 1) {
      const int ctx = min(cx, a.W * a.BS), cached = ctx >= n ? ctx - n : 0;
      const int step = min(n, (ROWS + a.G - 1) / a.G);
      SpanWalk f, l;
      f.init(a.span, cached, cached + step - 1);
      l.init(a.span, cached + n - step, cached + n - 1);
      const int64_t walked = (int64_t)(f.blocks() + l.blocks()) * nb / 2;
      // (bounded: split units are few, and KS bounds their splits)
      work.blocks += wave_sum_i(n > 0 ? (int)min(walked, (int64_t)1 << 20) : 0);
    }
    const int incl = wave_scan_incl_i(nb) + carry;
    const unsigned long long hit = __ballot(item >= incl - nb && item < incl);
    if (hit) {
      const int src = __builtin_ctzll(hit);
      u.s = base + src;
      u.block = item - readlane_i(incl - nb, src);
      u.n = readlane_i(n, src);
      u.q0 = readlane_i(q0, src);
      u.ctx = readlane_i(cx, src);
      found = true;
      if (a.KS == 1) return true;
    }
    carry = readlane_i(incl, kWave - 1);
  }
  work.units = carry;
  return found;
}

__device__ __forceinline__ __amdgpu_buffer_rsrc_t span_rsrc(const void* base, uint32_t bytes) {
  const uint64_t addr = reinterpret_cast<uint64_t>(base);
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)addr);
  const uint32_t hi = __builtin_amdgcn_readfirstlane((uint32_t)(addr >> 32));
  return __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void*>(((uint64_t)hi << 32) | lo), 0,
                                           (int)__builtin_amdgcn_readfirstlane(bytes), 0x00020000);
}

// ---- key splits -----------------------------------------------------------------------------

// Splits of a unit of nb key blocks
__device__ __forceinline__ int span_splits(const SpanPrefill& a, const SpanWork& work, int nb,
                                           int chip) {
  if (a.KS == 1 || nb < 2 * kSpanShareLow) return 1;
  // equal shares of the work, so that all splits fit the chip at once: the units' last ones are
  // short, half a workgroup more a unit on average (counted as 5/8: two chunks of 1000 over up
  // to 4000 cached 71 us, as a whole one 78.5, as 1/2 72.8)
  const int ends = (int)((int64_t)work.units * a.Hkv * 5 / 8);
  if (chip <= ends) return 1;
  const float all = (float)work.blocks * (float)a.Hkv;
  const int share = (int)ceilf(all / (float)(chip - ends));
  const int spread = chip / 2 > ends ? (int)fminf(ceilf(all / (float)(chip / 2 - ends)), kSpanShare)
                                     : kSpanShare;
  const int least = max(spread, kSpanShareLow);
  if (nb < 2 * least) return 1;
  const int blocks = max(share, least);
  return min((nb + blocks - 1) / blocks, a.KS);
}

// The splits' states of a unit, [KS] jobs of C chunks of 16 bytes and a base-2 log-sum-exp for
// each of T threads: normalised fp32 outputs as the threads hold them, so that a wave's access is
// one run of memory and nothing is rearranged.  Device-coherent.  Four chunks of 256-500 over up
// to 3000 cached 37.5 us; as output rows, joined row by row with weights in LDS, 42.5.
template <int C, int T>
struct SplitParts {
  static constexpr int kLse = C * T * 16;
  static constexpr int kBytes = kLse + T * 4;
  __amdgpu_buffer_rsrc_t r;
  __device__ __forceinline__ SplitParts(const SpanPrefill& a, int item, int h) {
    r = span_rsrc(a.parts + (int64_t)(item * a.Hkv + h) * a.KS * kBytes, a.KS * kBytes);
  }
  __device__ __forceinline__ void store(int s, const f32x4 (&v)[C], float lse) const {
#pragma unroll
    for (int c = 0; c < C; ++c)
      __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(span_u32x4, v[c]), r,
                                             s * kBytes + (c * T + threadIdx.x) * 16, 0, kSpanSc1);
    __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(uint32_t, lse), r,
                                          s * kBytes + kLse + threadIdx.x * 4, 0, kSpanSc1);
  }
  struct State {
    f32x4 v[C];
    float lse;
  };
  __device__ __forceinline__ void load(int s, State& x) const {
    x.lse = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(
                                          r, s * kBytes + kLse + threadIdx.x * 4, 0, kSpanSc1));
#pragma unroll
    for (int c = 0; c < C; ++c)
      x.v[c] = __builtin_bit_cast(
          f32x4, __builtin_amdgcn_raw_buffer_load_b128(
                     r, s * kBytes + (c * T + threadIdx.x) * 16, 0, kSpanSc1));
  }
  // The join of the splits' states in their order, the next one's loads in flight meanwhile (the
  // last one's once more at the end: without a branch around the loads the wait for one state
  // leaves the next one's running).
  __device__ __forceinline__ void join(int splits, f32x4 (&num)[C]) const {
    float M = kNegInf, den = 0.f;
#pragma unroll
    for (int c = 0; c < C; ++c) num[c] = f32x4{0.f, 0.f, 0.f, 0.f};
    const auto add = [&](const State& x) __attribute__((always_inline)) {
      const float m = fmaxf(M, x.lse);
      const float alpha = M == kNegInf ? 0.f : exp2f(M - m);
      const float w = x.lse == kNegInf ? 0.f : exp2f(x.lse - m);
      den = den * alpha + w;
#pragma unroll
      for (int c = 0; c < C; ++c) num[c] = num[c] * alpha + w * x.v[c];
      M = m;
    };
    State x, y;
    load(0, x);
    for (int s = 0;; s += 2) {  // workgroup-uniform
      load(min(s + 1, splits - 1), y);
      add(x);
      if (s + 1 >= splits) break;
      load(min(s + 2, splits - 1), x);
      add(y);
      if (s + 2 >= splits) break;
    }
    const float inv = den > 0.f ? 1.f / den : 0.f;
#pragma unroll
    for (int c = 0; c < C; ++c) num[c] *= inv;
  }
};

// Positions and output rows (token * Hq + head) of a unit's rows, without integer divisions: row
// r0 + r is x = r0 % G + r rows on from r0 - r0 % G, and x / G is exact by float: x < G + 256 is at
// least half a row from the next multiple of G, 0.5 / G of a quotient below 256 / G + 1
// (G <= 2^20).
struct UnitRows {
  int64_t base;
  int q, rem, step;
  float inv;
  __device__ __forceinline__ UnitRows(const SpanPrefill& a, const SpanUnit& u, int r0, int h) {
    q = r0 / a.G;
    rem = r0 - q * a.G;
    base = (int64_t)(u.q0 + q) * a.Hq + h * a.G;
    step = a.Hq - a.G;
    inv = 1.f / (float)a.G;
  }
  // token of row r0 + r within the sequence's new ones
  __device__ __forceinline__ int token(int r) const {
    return q + (int)(((float)(rem + r) + 0.5f) * inv);
  }
  __device__ __forceinline__ int64_t operator()(int r) const {
    const int x = rem + r;
    return base + x + (int64_t)(int)(((float)x + 0.5f) * inv) * step;
  }
};

// Whether this workgroup is the unit's last: its rows are complete before its ticket is drawn,
// and the last one sets the ticket back to zero.
__device__ __forceinline__ bool last_split(int* ticket, int splits, int* last) {
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // this wave's rows are complete
  __syncthreads();
  if (threadIdx.x == 0)
    *last = __hip_atomic_fetch_add(ticket, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) ==
            splits - 1;
  __syncthreads();
  if (!*last) return false;
  if (threadIdx.x == 0) __hip_atomic_store(ticket, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  return true;
}

template <int D, bool Q4>
struct SpanCfg {
  static constexpr int ROWB = D * 2;                // LDS bytes per staged key row
  static constexpr int MAT = kSpanKeys * ROWB;
  static constexpr int CPR = D / 8;                 // 16-byte chunks per row
  static constexpr int RPI = kWave / CPR;           // rows per DMA instruction
  // Chunk swizzles of row r.  Reads: K 32 rows, one chunk each; V 4 rows x 64 bytes, so V's
  // quads of chunks move together.  Writes of 4-bit rows: 4 (D = 64: 8) rows, one chunk of each
  // quad, so V's chunks move within their quads too (4095 tokens of 32/8 heads 179 -> 173 us;
  // the DMA of 16-bit rows is slower for it, 165 -> 169 us under a window of 1024).
  static __device__ __forceinline__ int swz_k(int r) { return D >= 128 ? (r & 15) : ((r >> 1) & 7); }
  static __device__ __forceinline__ int swz_v(int r) {
    const int quad = D >= 128 ? (r & 3) : ((r >> 1) & 1);
    return quad << 2 | (Q4 ? (D >= 128 ? r & 3 : (r >> 1) & 3) : 0);
  }
};

__device__ __forceinline__ float span_max(float a, float b) { return __builtin_elementwise_maximum(a, b); }
__device__ __forceinline__ float other_half(float x, int hf) {
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(hf ? b[0] : b[1]);
}

typedef __attribute__((address_space(3))) void span_lds_void;
typedef __attribute__((address_space(3))) s16x4 span_lds_s16x4;

// The state of a wave's 32 rows
template <int D>
struct SpanRows {
  f16x8 qv[D / 16];
  int pos, lo;  // the lane's row sees keys lo .. pos (and those below the sinks)
  float m, l;   // running reference (base 2) and this lane's part of the sum
  f32x16 o[D / 32];
};

// One staged block, tiles t .. t + 3 of the walk.  mask: some row does not see all of it.
template <int D, class E, bool Q4>
__device__ __forceinline__ void span_block(const SpanWalk& wk, int t, const unsigned char* kst,
                                           const unsigned char* vst, bool mask, float scale_log2,
                                           bool follow, SpanRows<D>& r) {
  using C = SpanCfg<D, Q4>;
  constexpr int NC = D / 16, NT = D / 32;
  const int lane = lane_id();
  const int hf = lane >> 5;
  const int n = lane & 31;
  f16x8 kf[2][NC];
#pragma unroll
  for (int kt = 0; kt < 2; ++kt)
#pragma unroll
    for (int c = 0; c < NC; ++c)
      kf[kt][c] = *reinterpret_cast<const f16x8*>(kst + (32 * kt + n) * C::ROWB +
                                                  (((2 * c + hf) ^ C::swz_k(n)) * 16));
  f32x16 st[2];
#pragma unroll
  for (int kt = 0; kt < 2; ++kt) st[kt] = f32x16{};
#pragma unroll
  for (int c = 0; c < NC; ++c)
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) st[kt] = mma32x32<E>(kf[kt][c], r.qv[c], st[kt]);
  const int l16 = lane & 15;
  const int vrow = 4 * hf + (l16 >> 2);
  const int vchunk = 2 * ((lane >> 4) & 1) + ((l16 & 3) >> 1);
  const int vswz = C::swz_v(vrow);
  auto vfrag = [&](int s, int x) __attribute__((always_inline)) {
    const unsigned char* vb = vst + (16 * s + vrow) * C::ROWB + (l16 & 1) * 8;
    const int slot = ((4 * x + vchunk) ^ vswz) * 16;
    const f16x4 a = __builtin_bit_cast(
        f16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((span_lds_s16x4*)(vb + slot)));
    const f16x4 b = __builtin_bit_cast(
        f16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((span_lds_s16x4*)(vb + 8 * C::ROWB + slot)));
    return f16x8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
  };
  // the first 32 keys' V fragments are read before the softmax, which hides their latency (16
  // keys' at D = 256, for registers)
  constexpr int VS = D > 128 ? 1 : 2;
  f16x8 vf[VS][NT];
#pragma unroll
  for (int s = 0; s < VS; ++s)
#pragma unroll
    for (int x = 0; x < NT; ++x) vf[s][x] = vfrag(s, x);

  if (mask) {  // wave-uniform
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int k0 = wk.key(t + 2 * kt + half) + 4 * hf;  // the lane's first key of the tile
        int past = r.pos - k0, before = r.lo - k0, sink = wk.sinks - k0;
        // (defined here as far as the compiler knows: otherwise it hoists the comparisons out
        // of the branch)
        asm volatile("" : "+v"(past), "+v"(before), "+v"(sink));
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int key = 8 * (i / 4) + i % 4;
          if (key > past || (key < before && key >= sink)) st[kt][8 * half + i] = kNegInf;
        }
      }
  }
  float mx = span_max(st[0][0], st[1][0]), my = span_max(st[0][1], st[1][1]);
#pragma unroll
  for (int i = 2; i < 16; i += 2) {
    mx = span_max(span_max(mx, st[0][i]), st[1][i]);
    my = span_max(span_max(my, st[0][i + 1]), st[1][i + 1]);
  }
  mx = span_max(mx, my);
  mx = span_max(mx, other_half(mx, hf)) * scale_log2;
  if (__ballot(mx > r.m + (follow ? kNegInf : kRescaleSlack))) {  // wave-uniform
    float m_new = fmaxf(r.m, mx);
    if (follow) {
      // down to the block's maximum too, as long as the sum stays below 2^16 of its largest
      const float l = r.l + other_half(r.l, hf);
      m_new = fmaxf(mx, r.m - fmaxf(16.f - __builtin_amdgcn_logf(l), 0.f));
    }
    const float alpha = m_new == kNegInf ? 1.f : exp2_fast(r.m - m_new);
    r.l *= alpha;
#pragma unroll
    for (int x = 0; x < NT; ++x) r.o[x] *= alpha;
    r.m = m_new;
  }
  const float neg_m = r.m == kNegInf ? 0.f : -r.m;
  f16x8 pb[4];
#pragma unroll
  for (int s = 0; s < 4; ++s) {
    // probabilities in 16 bits for the matrix instruction; the sum takes the rounded ones
#pragma unroll
    for (int j = 0; j < 8; ++j)
      pb[s][j] = to16<E>(exp2_fast(__builtin_fmaf(st[s / 2][8 * (s % 2) + j], scale_log2, neg_m)));
    r.l = sum8<E>(pb[s], r.l);
  }
#pragma unroll
  for (int s = 0; s < 4; ++s)
#pragma unroll
    for (int x = 0; x < NT; ++x) {
      const f16x8 va = vf[s % VS][x];
      // in flight during the products before its own
      if (s + VS < 4) vf[s % VS][x] = vfrag(s + VS, x);
      r.o[x] = mma32x32<E>(va, pb[s], r.o[x]);
    }
}

// 16-bit pools: wave w brings keys RUN w .. +RUN of a block by LDS DMA
template <int D, bool PAD, int NW>
struct Stage16 {
  using C = SpanCfg<D, false>;
  static constexpr int RUN = kSpanKeys / NW;
  static constexpr int NI = RUN / C::RPI;
  static_assert(RUN <= 16 && NI >= 1, "a run lies in one page");
  int w, id_base;
  int idv;              // lane j: pool block of this wave's run of walk block id_base + j
  uint32_t vk[NI], vv[NI];  // lane offsets of the DMA, the swizzles applied

  // first key of this wave's run of walk block j
  __device__ __forceinline__ int run_key(const SpanWalk& wk, int j) const {
    return wk.key(4 * j + RUN * w / kTile) + (RUN * w) % kTile;
  }

  __device__ __forceinline__ void load_ids(const SpanPrefill& a, const SpanWalk& wk,
                                           const int32_t* trow, int base) {
    id_base = base;
    int page = run_key(wk, base + lane_id()) >> a.bs_log2;
    page = page < a.W ? page : a.W - 1;
    idv = trow[page];
  }
  __device__ __forceinline__ void init(const SpanPrefill& a, const SpanWalk& wk,
                                       const int32_t* trow, int h, int j0) {
    w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    load_ids(a, wk, trow, j0);
    const int rs = a.Hkv * a.dr * 2;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int rr = C::RPI * i + lane_id() / C::CPR;
      const int sl = lane_id() % C::CPR;
      const int ck = sl ^ C::swz_k(RUN * w + rr), cv = sl ^ C::swz_v(RUN * w + rr);
      // chunks past the real row come from past the descriptor's end: zeros
      vk[i] = !PAD || ck * 8 < a.dr ? (uint32_t)(rr * rs + ck * 16) : 0x7ffffff0u;
      vv[i] = !PAD || cv * 8 < a.dr ? (uint32_t)(rr * rs + cv * 16) : 0x7ffffff0u;
    }
  }
  __device__ __forceinline__ void fetch(const SpanPrefill& a, const SpanWalk& wk,
                                        const int32_t* trow, int h, int j, unsigned char* kst,
                                        unsigned char* vst) {
    if (j - id_base >= kWave) {  // wave-uniform
      load_ids(a, wk, trow, j);
      __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0)
    }
    const int t0 = run_key(wk, j);
    const int id = clamp_block(__builtin_amdgcn_readlane(idv, j - id_base), a.NB);
    const int rs = a.Hkv * a.dr * 2;
    int nv = wk.key_end - t0;
    nv = nv < 0 ? 0 : (nv > RUN ? RUN : nv);
    const uint32_t bytes = nv > 0 ? (uint32_t)((nv - 1) * rs + a.dr * 2) : 0u;
    const int64_t off =
        (((int64_t)id * a.BS + (t0 & (a.BS - 1))) * a.Hkv + h) * (int64_t)a.dr;
    const __amdgpu_buffer_rsrc_t rk = span_rsrc((const f16*)a.k_pool + off, bytes);
    const __amdgpu_buffer_rsrc_t rv = span_rsrc((const f16*)a.v_pool + off, bytes);
    const bool edge = !(t0 >= wk.ws || t0 + RUN <= wk.sinks);  // wave-uniform
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      uint32_t ok = vk[i], ov = vv[i];
      if (edge && !wk.sees(t0 + C::RPI * i + lane_id() / C::CPR)) ok = ov = 0x7ffffff0u;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          rk, (span_lds_void*)(kst + (RUN * w + i * C::RPI) * C::ROWB), 16, ok, 0, 0, 0);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          rv, (span_lds_void*)(vst + (RUN * w + i * C::RPI) * C::ROWB), 16, ov, 0, 0, 0);
    }
  }
};

// 4-bit pools: a thread's chunks of a block, loaded into registers and converted into LDS
template <int D, class E, bool PAD, int NW>
struct Stage4 {
  using C = SpanCfg<D, true>;
  static constexpr int T = NW * kWave;
  static constexpr int BPR = D / kQ4Block;                 // chunks (32 dims) per row
  static constexpr int CHUNKS = 2 * kSpanKeys * BPR;       // of a block: K's, then V's
  static constexpr int NI = (CHUNKS + T - 1) / T;
  span_u32x4 codes[NI];
  uint32_t scale[NI];
  int id[NI];

  static __device__ __forceinline__ int chunk(int i) { return threadIdx.x + i * T; }
  static __device__ __forceinline__ int key_of(int i) { return chunk(i) / BPR % kSpanKeys; }
  // position of the key of chunk i of walk block j
  static __device__ __forceinline__ int key_at(const SpanWalk& wk, int j, int i) {
    return wk.key(4 * j + key_of(i) / kTile) + key_of(i) % kTile;
  }
  __device__ __forceinline__ void load_ids(const SpanPrefill& a, const SpanWalk& wk,
                                           const int32_t* trow, int j) {
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      int page = key_at(wk, j, i) >> a.bs_log2;
      page = page < a.W ? page : a.W - 1;
      id[i] = trow[page];
    }
  }
  __device__ __forceinline__ void load(const SpanPrefill& a, const SpanWalk& wk, int h, int j) {
    const Q4Layout& at = a.rows4;
    const int sb = a.dr / kQ4Block;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int c = chunk(i), key = key_at(wk, j, i), blk = c % BPR;
      const bool is_v = c >= kSpanKeys * BPR;
      codes[i] = span_u32x4{0, 0, 0, 0};
      scale[i] = kQ4ScaleLow;
      if (c < CHUNKS && (!PAD || blk < sb) && wk.sees(key)) {
        const int page = clamp_block(id[i], a.NB), off = key & (a.BS - 1);
        const uint8_t* cp = (const uint8_t*)(is_v ? a.v_pool : a.k_pool) + at.code_offset(h);
        const uint8_t* sp = (is_v ? a.v_scales : a.k_scales) + at.scale_offset(h);
        codes[i] = *reinterpret_cast<const span_u32x4*>(cp + at.code_row(page, off) + blk * 16);
        scale[i] = sp[at.scale_row(page, off) + blk];
      }
    }
  }
  __device__ __forceinline__ void put(unsigned char* kst, unsigned char* vst) const {
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int c = chunk(i), key = key_of(i), blk = c % BPR;
      if (CHUNKS % T != 0 && c >= CHUNKS) continue;
      const bool is_v = c >= kSpanKeys * BPR;
      unsigned char* row = (is_v ? vst : kst) + key * C::ROWB;
      const int swz = is_v ? C::swz_v(key) : C::swz_k(key);
      const float s = q4_scale_value(scale[i]);
#pragma unroll
      for (int q = 0; q < 4; ++q)
        *reinterpret_cast<f16x8*>(row + ((4 * blk + q) ^ swz) * 16) = q4_unpack8<E>(codes[i][q], s);
    }
  }
};

template <int D, class E, bool Q4, bool PAD, int NW>
__global__ __launch_bounds__(NW* kWave)
__attribute__((amdgpu_waves_per_eu(D > 128 ? 1 : 2, D > 128 ? 1 : 2)))
void span_prefill_kernel(const SpanPrefill a) {
  using C = SpanCfg<D, Q4>;
  constexpr int ROWS = 32 * NW;
  // one LDS object per stage and matrix: the compiler's wait for an LDS DMA before an LDS read
  // is then limited to reads of the object it fills
  __shared__ __align__(16) unsigned char k0[C::MAT];
  __shared__ __align__(16) unsigned char v0[C::MAT];
  __shared__ __align__(16) unsigned char k1[C::MAT];
  __shared__ __align__(16) unsigned char v1[C::MAT];
  __shared__ int last;
  // Workgroups in the order of their split, within it the later units, which see more keys,
  // first: those without work (a unit has as many splits as its keys are worth) come last
  const int at = (int)blockIdx.x / a.Hkv;
  const int h = (int)blockIdx.x - at * a.Hkv;
  const int item = a.units - 1 - at;
  const int ks = blockIdx.y;
  SpanUnit u;
  SpanWork work;
  if (!find_unit<ROWS>(a, item, u, work)) return;
  const int G = a.G;
  const int DR = PAD ? a.dr : D;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = lane_id();
  const int hf = lane >> 5;
  const int n = lane & 31;
  const int ctx = min(u.ctx, a.W * a.BS);
  const int total_rows = u.n * G;
  const int cached = ctx >= u.n ? ctx - u.n : 0;
  const int r0 = u.block * ROWS;
  const int r_last = min(r0 + ROWS, total_rows) - 1;

  const UnitRows rows(a, u, r0, h);
  SpanWalk wk;
  wk.init(a.span, cached + rows.q, cached + rows.token(r_last - r0));
  const int nb = wk.blocks();
  const int splits = span_splits(a, work, nb, kSpanSlots);
  if (ks >= splits) return;
  const int j0 = nb * ks / splits, j1 = nb * (ks + 1) / splits;  // (nb < 2^24)

  const int wr0 = r0 + 32 * w;
  const bool has_rows = wr0 <= r_last;
  // positions of the wave's first and last row, and where their windows start
  const int p_first = cached + rows.token(min(wr0, r_last) - r0);
  const int p_last = cached + rows.token(min(wr0 + 31, r_last) - r0);
  const int lo_first = window_start(a.span, p_first), lo_last = window_start(a.span, p_last);
  const int row = wr0 + n;
  const bool valid = row < total_rows;
  const int rc = valid ? row : r_last;
  const int32_t* trow = a.tables + (int64_t)u.s * a.W;
  SpanRows<D> r;
  r.pos = cached + rows.token(rc - r0);
  r.lo = window_start(a.span, r.pos);
  r.m = kNegInf;
  r.l = 0.f;
#pragma unroll
  for (int x = 0; x < D / 32; ++x) r.o[x] = f32x16{};
  {
    const f16* qrow = a.q + rows(rc - r0) * DR + 8 * hf;
#pragma unroll
    for (int c = 0; c < D / 16; ++c)
      r.qv[c] = valid && (!PAD || 16 * c + 8 * hf < DR) ? ld16(qrow + 16 * c) : f16x8{};
  }
  auto compute = [&](int j, const unsigned char* kst, const unsigned char* vst)
                     __attribute__((always_inline)) {
    // first and last key of the block (a block with both sinks and window keys has a gap)
    const int k0 = wk.key(4 * j), k1 = wk.key(4 * j + 3) + kTile - 1;
    if (!has_rows || k0 > p_last || (k1 < lo_first && k0 >= wk.sinks)) return;
    const bool mask = k1 > p_first || (k0 < lo_last && k1 >= wk.sinks);
    span_block<D, E, Q4>(wk, 4 * j, kst, vst, mask, a.scale_log2, j - j0 < kSpanFollow, r);
  };

  if constexpr (Q4) {
    Stage4<D, E, PAD, NW> st;
    st.load_ids(a, wk, trow, j0);
    st.load(a, wk, h, j0);
    if (j0 + 1 < j1) st.load_ids(a, wk, trow, j0 + 1);
    st.put(k0, v0);
    if (j0 + 1 < j1) st.load(a, wk, h, j0 + 1);
    if (j0 + 2 < j1) st.load_ids(a, wk, trow, j0 + 2);
    // step j: block j is staged once every wave has passed the barrier, and no wave reads block
    // j - 1 any more, whose stage block j + 1 goes into
    auto step = [&](int j, unsigned char* kc, unsigned char* vc, unsigned char* kn,
                    unsigned char* vn) __attribute__((always_inline)) {
      __syncthreads();
      if (j + 1 < j1) st.put(kn, vn);
      if (j + 2 < j1) st.load(a, wk, h, j + 2);
      if (j + 3 < j1) st.load_ids(a, wk, trow, j + 3);
      compute(j, kc, vc);
    };
    for (int j = j0; j < j1; j += 2) {
      step(j, k0, v0, k1, v1);
      if (j + 1 < j1) step(j + 1, k1, v1, k0, v0);
    }
  } else {
    Stage16<D, PAD, NW> st;
    st.init(a, wk, trow, h, j0);
    st.fetch(a, wk, trow, h, j0, k0, v0);
    auto step = [&](int j, unsigned char* kc, unsigned char* vc, unsigned char* kn,
                    unsigned char* vn) __attribute__((always_inline)) {
      __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0): this wave's run of block j is in LDS
      __syncthreads();
      if (j + 1 < j1) st.fetch(a, wk, trow, h, j + 1, kn, vn);
      compute(j, kc, vc);
    };
    for (int j = j0; j < j1; j += 2) {
      step(j, k0, v0, k1, v1);
      if (j + 1 < j1) step(j + 1, k1, v1, k0, v0);
    }
  }

  const float l = r.l + other_half(r.l, hf);
  const float inv = l > 0.f ? 1.f / l : 0.f;
  f32x4 o[D / 8];  // chunk 4 x + i: dims 32 x + 8 i + 4 hf .. +3
#pragma unroll
  for (int x = 0; x < D / 32; ++x)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      o[4 * x + i] =
          f32x4{r.o[x][4 * i], r.o[x][4 * i + 1], r.o[x][4 * i + 2], r.o[x][4 * i + 3]} * inv;
  if (splits > 1) {
    const SplitParts<D / 8, NW * kWave> part(a, item, h);
    if (valid) part.store(ks, o, l > 0.f ? r.m + log2f(l) : kNegInf);
    if (!last_split(a.tickets + item * a.Hkv + h, splits, &last)) return;
    if (has_rows) part.join(splits, o);
  }
  if (!valid) return;
  f16* orow = a.out + rows(row - r0) * DR + 4 * hf;
#pragma unroll
  for (int c = 0; c < D / 8; ++c)
    if (!PAD || 8 * c + 4 * hf < DR) *reinterpret_cast<f16x4*>(orow + 8 * c) = to16x4<E>(o[c]);
}

// ---- host -----------------------------------------------------------------------------------

inline size_t span_align(size_t x) { return (x + 255) & ~size_t(255); }
inline int span_log2(int x) {
  if (x <= 0 || (x & (x - 1))) return -1;
  int l = 0;
  while ((1 << l) < x) ++l;
  return l;
}
inline int span_dim(int d) { return d <= 64 ? 64 : (d <= 128 ? 128 : 256); }

// Launch shape, from what the host knows
struct SpanShape {
  int waves;  // per workgroup
  int64_t units;
  int ks;
  size_t bytes;  // workspace: tickets, split states
};
// Eight waves a workgroup halve what a row block converts, but leave one workgroup a CU, whose
// start and end nothing hides: for long prompts over 4-bit pools that fill the chip either way.
// Four / eight waves, fp16, 32/8 heads of 128: 1000 fresh tokens 38 / 39 us, 2000 64 / 70, 4095
// (bf16) 173 / 148, 6000 338 / 325 (under a window of 2000 209 / 215, of 4000 302 / 282), four
// of 1000 67 / 71; four of 2000 of 12/2 heads 97 / 94.  16-bit rows: 8191 tokens under a window
// of 1024 165 / 189, 6000 under 4000 289 / 289.
inline int span_waves(int num_seqs, int total_q, int hq, int hkv, int d, int window, bool q4) {
  const int64_t wgs = ((int64_t)total_q * (hq / hkv) + 255) / 256 * hkv;
  return q4 && d == 128 && (window == 0 || window >= 4000) && wgs >= 384 &&
                 total_q / num_seqs >= 2000
             ? 8
             : 4;
}
// rows of a unit (0: 32 a wave) and workgroups that run at once: the 16-bit kernel's, unless given
inline SpanShape span_shape(int num_seqs, int total_q, int hq, int hkv, int d, int window, bool q4,
                            int unit_rows = 0, int chip = kSpanSlots) {
  SpanShape p;
  const int64_t rows = (int64_t)total_q * (hq / hkv);
  p.waves = span_waves(num_seqs, total_q, hq, hkv, d, window, q4);
  if (unit_rows == 0) unit_rows = 32 * p.waves;
  p.units = (rows + unit_rows - 1) / unit_rows + num_seqs;
  // key splits of a unit at most: twice the slots over the units, for those with more keys
  // than the others
  const int64_t wgs = ((rows + unit_rows - 1) / unit_rows) * hkv;
  int64_t ks = wgs > 0 ? 2 * chip / wgs : 1;
  ks = ks < 1 ? 1 : (ks > kSpanMaxSplits ? kSpanMaxSplits : ks);
  if (p.waves != 4 || p.units * hkv > kSpanTickets) ks = 1;
  // a split's rows and its threads' log-sum-exps (SplitParts)
  const int64_t job = (int64_t)unit_rows * span_dim(d) * (int64_t)sizeof(float) +
                      4 * kWave * (int64_t)sizeof(float);
  while (ks > 1 && ks * p.units * hkv * job > kSpanPartBytes) --ks;
  p.ks = (int)ks;
  p.bytes = kSpanTicketBytes + (ks > 1 ? (size_t)(ks * p.units * hkv * job) : 0);
  return p;
}

template <int D, class E, bool Q4, bool PAD>
int span_launch(const SpanPrefill& a, const SpanShape& p, hipStream_t s) {
  const dim3 grid((unsigned)(p.units * a.Hkv), (unsigned)a.KS);
  if constexpr (D == 128 && Q4 && !PAD) {
    if (p.waves == 8) {
      hipLaunchKernelGGL((span_prefill_kernel<D, E, Q4, PAD, 8>), grid, dim3(8 * kWave), 0, s, a);
      return FE_LAUNCH_STATUS();
    }
  }
  hipLaunchKernelGGL((span_prefill_kernel<D, E, Q4, PAD, 4>), grid, dim3(4 * kWave), 0, s, a);
  return FE_LAUNCH_STATUS();
}

// Checks and launch that the 16-bit and the 4-bit forms share
template <class E, bool Q4>
int span_prefill(const void* q, void* out, const void* k_pool, const void* k_scales,
                 const void* v_pool, const void* v_scales, const fe_kv4_strides* strides,
                 int num_blocks, const int32_t* tables,
                 int table_stride, const int32_t* q_off, const int32_t* ctx, int num_seqs,
                 int total_q, int hq, int hkv, int d, int bs, float scale, int window, int sinks,
                 void* workspace, size_t workspace_bytes, fe_stream_t stream) {
  FE_CHECK_ARG(num_seqs >= 0 && total_q >= 0 && hq > 0 && hkv > 0 && d > 0 && num_blocks > 0 &&
               table_stride > 0 && window >= 0 && sinks >= 0 && hq % hkv == 0);
  FE_CHECK_ARG(Q4 || window > 0);
  FE_CHECK_ARG(scale > 0.f);  // the row maxima are taken on unscaled scores
  const int bs_log2 = span_log2(bs);
  if (bs_log2 < 0 || bs % kTile != 0) return FE_ERR_UNSUPPORTED;
  if (d > 256 || d % (Q4 ? kQ4Block : 8) != 0) return FE_ERR_UNSUPPORTED;
  // key positions, pool rows and the offsets within a run of keys are 32-bit in the kernel
  if ((int64_t)table_stride * bs >= ((int64_t)1 << 30) || hq / hkv > (1 << 20) ||
      (int64_t)num_blocks * bs >= ((int64_t)1 << 31) || (int64_t)hkv * d >= ((int64_t)1 << 25) ||
      (int64_t)total_q * (hq / hkv) >= ((int64_t)1 << 30))
    return FE_ERR_UNSUPPORTED;
  if (num_seqs == 0 || total_q == 0) return FE_OK;
  FE_CHECK_ARG(q && out && k_pool && v_pool && tables && q_off && ctx);
  Q4Layout rows4{};
  if (Q4) {
    FE_CHECK_ARG(k_scales && v_scales);
    if (int rc = q4_layout(strides, num_blocks, hkv, d, bs, rows4)) return rc;
  }
  const auto aligned = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; };
  FE_CHECK_ARG(aligned(q) && aligned(out) && aligned(k_pool) && aligned(v_pool));
  const SpanShape p = span_shape(num_seqs, total_q, hq, hkv, d, window, Q4);
  // (a grid's threads are counted in 32 bits)
  if (p.units * hkv >= ((int64_t)1 << 23)) return FE_ERR_UNSUPPORTED;
  if (workspace == nullptr || workspace_bytes < p.bytes || !aligned(workspace))
    return FE_ERR_WORKSPACE;
  SpanPrefill a{};
  a.q = (const f16*)q;
  a.out = (f16*)out;
  a.k_pool = k_pool;
  a.v_pool = v_pool;
  a.k_scales = (const uint8_t*)k_scales;
  a.v_scales = (const uint8_t*)v_scales;
  a.tables = tables;
  a.q_off = q_off;
  a.ctx = ctx;
  a.tickets = (int*)workspace;
  a.parts = (unsigned char*)workspace + kSpanTicketBytes;
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
  a.span = Span{window, window > 0 ? sinks : 0};
  a.rows4 = rows4;
  const hipStream_t s = (hipStream_t)stream;
  if (d == 64) return span_launch<64, E, Q4, false>(a, p, s);
  if (d == 128) return span_launch<128, E, Q4, false>(a, p, s);
  if (d < 64) return span_launch<64, E, Q4, true>(a, p, s);
  if (d < 128) return span_launch<128, E, Q4, true>(a, p, s);
  return span_launch<256, E, Q4, true>(a, p, s);
}

}  // namespace
}  // namespace fe
