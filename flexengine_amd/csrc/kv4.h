// The 4-bit row format of the KV pools (fe_write_kv4 and the kernels that read it).
//
// A K or V row of one token and KV head is cut into blocks of 32 dims.  A block is 32 e2m1
// codes (sign, 2 exponent and 1 mantissa bits: 0, 0.5, 1, 1.5, 2, 3, 4, 6) and one e8m0 scale
// byte s, its values code * 2^(s - 127) -- the microscaling fp4 format of the OCP MX
// specification, which gfx950 converts to and from in one instruction per pair
// (v_cvt_scalef32_pk_*): with a power-of-two scale the 16-bit values are exact, so they feed
// the 16-bit matrix instructions without a rounding of their own.
//
// Scale of a block: the smallest power of two 2^e with max|x| <= 7 * 2^e.  7 is half a step
// past the largest code, so no value is further from its code's than half the distance between
// the codes around it, and a block's range is never more than 2x wider than it needs.
// e >= -23, so that every value is a multiple of 2^-24 (exact in fp16, subnormals included;
// bf16 rows have the same bound: a block below 2^-21 has fewer codes, one up to 2^-25 is zeros), and e <= 13 for fp16 rows, 125 for bf16 (the values
// stay finite; an fp16 magnitude above 49152 is held as 49152).  A block with an infinity or
// NaN has s = 255, which the conversion turns into NaN for all 32 values.
//
// Rounding to nearest, ties to the even code, as the conversion instruction does it.
//
// Layout: codes [num_blocks, kv_heads, block_size, head_dim / 2] bytes (the even dim in a
// byte's low half), scales [num_blocks, kv_heads, block_size, head_dim / 32].  The head stands
// before the token, unlike in the 16-bit pools: a 4-bit row is 64 bytes at head_dim 128, half
// a cache line, and heads run on different XCDs, whose L2s would each fetch the whole line.
// The _strided forms take the same dims in any order and with gaps (Q4Layout): 37 rows of
// 2048-16384 tokens of 8 heads, the token before the head, 104 us where the layout above takes 68.
#pragma once

#include "attn_core.h"
#include "flexengine_amd_span.h"

namespace fe {

constexpr int kQ4Block = 32;            // dims that share a scale
constexpr uint32_t kQ4ScaleLow = 127 - 23;
template <class E>
constexpr uint32_t kQ4ScaleHigh = __is_same(E, Bf16) ? 127 + 125 : 127 + 13;
constexpr uint32_t kQ4ScaleNan = 255;

// ---- where the rows are -------------------------------------------------------------------
// Distances between blocks, heads and tokens, of the codes in units of 16 bytes (a block of 32
// dims), of the scales in bytes.  A page and a position in it are 32-bit, what they are
// multiplied by too: one multiply-add each into a 64-bit offset.
struct Q4Layout {
  uint32_t code_block, code_token, scale_block, scale_token;
  int64_t code_head, scale_head;
  // byte offsets of a row of head 0
  __device__ __forceinline__ uint64_t code_row(int blk, int off) const {
    return ((uint64_t)(uint32_t)blk * code_block + (uint64_t)(uint32_t)off * code_token) * 16;
  }
  __device__ __forceinline__ uint64_t scale_row(int blk, int off) const {
    return (uint64_t)(uint32_t)blk * scale_block + (uint64_t)(uint32_t)off * scale_token;
  }
  __device__ __forceinline__ int64_t code_offset(int h) const { return h * code_head * 16; }
  __device__ __forceinline__ int64_t scale_offset(int h) const { return h * scale_head; }
};

// Whether rows of `row` bytes at these strides (blocks, heads, tokens; those of a size of 1
// count for nothing) lie apart from each other: each stride past all that the smaller ones span
inline bool q4_rows_apart(const int64_t (&stride)[3], const int64_t (&size)[3], int64_t row) {
  int order[3] = {0, 1, 2};
  for (int i = 0; i < 2; ++i)
    for (int j = i + 1; j < 3; ++j)
      if (stride[order[j]] < stride[order[i]]) {
        const int t = order[i];
        order[i] = order[j];
        order[j] = t;
      }
  int64_t extent = row;
  for (int i = 0; i < 3; ++i) {
    const int k = order[i];
    if (size[k] == 1) continue;
    int64_t span;
    if (stride[k] < extent || __builtin_mul_overflow(stride[k], size[k] - 1, &span) ||
        __builtin_add_overflow(extent, span, &extent))
      return false;
  }
  return true;
}

// The layout of pools of these sizes: the dense one, or what `s` says
inline int q4_layout(const fe_kv4_strides* s, int nb, int hkv, int d, int bs, Q4Layout& l) {
  const int64_t size[3] = {nb, hkv, bs};
  const int64_t sb = d / kQ4Block;
  int64_t g[3] = {size[1] * size[2] * sb, size[2] * sb, sb}, c[3] = {g[0] * 16, g[1] * 16, sb * 16};
  if (s != nullptr)
    for (int i = 0; i < 3; ++i) {
      c[i] = s->codes[i];
      g[i] = s->scales[i];
    }
  for (int i = 0; i < 3; ++i) {
    if (size[i] == 1) c[i] = g[i] = 0;
    FE_CHECK_ARG(c[i] >= 0 && g[i] >= 0 && c[i] % 16 == 0);
  }
  FE_CHECK_ARG(q4_rows_apart(c, size, sb * 16) && q4_rows_apart(g, size, sb));
  // block strides are 32-bit units, and 16 tokens of a tile are within a 32-bit offset
  if (c[0] >> 36 || g[0] >> 32 || c[2] >> 26 || g[2] >> 26) return FE_ERR_UNSUPPORTED;
  l = Q4Layout{(uint32_t)(c[0] / 16), (uint32_t)(c[2] / 16), (uint32_t)g[0], (uint32_t)g[2],
               c[1] / 16, g[1]};
  return FE_OK;
}

template <class E>
__device__ __forceinline__ float from16(f16 x) {
  if constexpr (__is_same(E, Bf16))
    return (float)__builtin_bit_cast(__bf16, x);
  else
    return (float)x;
}
// |x| as an integer: ordered like the magnitude, infinities and NaN above every finite one
__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// scale byte of a block whose largest magnitude has the bits `top`
template <class E>
__device__ __forceinline__ uint32_t q4_scale(uint32_t top) {
  // exponent of top, one more past 1.75 (7 / 4); less 2, for the code 4 is 2^2
  const int e = (int)((top + 0x1fffffu) >> 23) - 2;
  const int lo = (int)kQ4ScaleLow, hi = (int)kQ4ScaleHigh<E>;
  return top >= 0x7f800000u ? kQ4ScaleNan : (uint32_t)(e < lo ? lo : (e > hi ? hi : e));
}
__device__ __forceinline__ float q4_scale_value(uint32_t s) { return __uint_as_float(s << 23); }

// the codes of 8 values
__device__ __forceinline__ uint32_t q4_pack8(const float (&x)[8], float scale) {
  uint32_t r = 0;
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, x[0], x[1], scale, 0);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, x[2], x[3], scale, 1);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, x[4], x[5], scale, 2);
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, x[6], x[7], scale, 3);
}
// the 8 values of a dword of codes, in the 16-bit type E
template <class E>
__device__ __forceinline__ f16x8 q4_unpack8(uint32_t c, float scale) {
  if constexpr (__is_same(E, Bf16)) {
    bf16x8_t r;
    const bf16x2_t a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, 0);
    const bf16x2_t b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, 1);
    const bf16x2_t d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, 2);
    const bf16x2_t e = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, 3);
    r = bf16x8_t{a[0], a[1], b[0], b[1], d[0], d[1], e[0], e[1]};
    return __builtin_bit_cast(f16x8, r);
  } else {
    const f16x2_t a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c, scale, 0);
    const f16x2_t b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c, scale, 1);
    const f16x2_t d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c, scale, 2);
    const f16x2_t e = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c, scale, 3);
    return f16x8{a[0], a[1], b[0], b[1], d[0], d[1], e[0], e[1]};
  }
}

// ---- visible keys of a window with sinks --------------------------------------------------
// A query at position p sees the keys j <= p with p - j < window (all of them if window is 0)
// and the keys j < sinks.  Kernels walk the keys in units of `unit` keys and leave out the
// units between the sinks and the first window: units 0 .. sink_units - 1 and then those from
// the one that holds the window's first key on.  `skip` units are left out.
struct Span {
  int window;  // 0: no window
  int sinks;
};
// first key in the window of position p
__device__ __forceinline__ int window_start(const Span& s, int p) {
  return s.window > 0 && p >= s.window ? p - s.window + 1 : 0;
}
// units left out for queries whose windows start at key ws or later
__device__ __forceinline__ int span_skip(const Span& s, int ws, int unit) {
  const int su = (int)(((unsigned)s.sinks + unit - 1) / unit);
  const int k = ws / unit - su;
  return k > 0 ? k : 0;
}

}  // namespace fe
