// The 4-bit paged KV cache (--kv-cache-dtype mxfp4): OCP microscaling FP4. A value is an e2m1 number (sign and one of 0, 0.5,
// 1, 1.5, 2, 3, 4, 6) times 2^(b - 127), the byte b shared by 32 neighbouring dims of one token and head: 4.25 bits a value.
// gfx950 converts between such numbers and bf16 in hardware and multiplies them by e4m3 numbers on the matrix cores as they are.
//
// Per block and kv head, 17 D block_size / 32 bytes (codes, then scales; two codes a byte, the even dim in the low half):
//   keys    codes [block_size][D / 2]: a lane's 32 dims of a key are one 16-byte load and one operand of the scaled product
//           scales [D / 32][block_size], token o of a run of 16 at 4 (o % 4) + o / 4: the four tokens that a lane of the decode
//           kernel takes from a run (o, o + 4, ...) lie in one 32-bit word, whose bytes the products select
//   values  codes [D / 2][block_size]: 16 tokens of two dims are one 16-byte load; a byte is one token's, so writers of
//           different tokens never share one
//           scales [D / 32][block_size], in order
#pragma once
#include "hipserve/common.h"
#include "hipserve/kernels.h"

namespace hipserve {

constexpr int kKv4Group = 32;  // dims that share a scale
constexpr int kKv4Nan = 255;   // scale byte of a group that held a NaN or an infinity: the whole group reads as NaN
constexpr float kLog2E = 1.4426950408889634f;

typedef int i32x8 __attribute__((ext_vector_type(8)));

// bytes of one (block, kv head), of its codes, and where a token's key scale stands among its group's
HS_HOST_DEVICE int kv4_head_bytes(int bs, int D) { return bs * D / 32 * 17; }
HS_HOST_DEVICE int kv4_code_bytes(int bs, int D) { return bs * D / 2; }
HS_HOST_DEVICE int kv4_key_scale_at(int off) { return (off & ~15) | ((off & 3) << 2) | ((off >> 2) & 3); }

// Scale byte of a group whose largest magnitude has these bf16 bits (NaN and infinities above all finite ones): the power of two
// under which it is at most 7, so within a sixth of the largest level 6. Never below 2^-119 (no value subnormal) or
// above 2^125 (no value above bf16's range).
HS_DEVICE int kv4_scale_byte(unsigned amax_bits) {
  if (amax_bits >= 0x7f80u) return kKv4Nan;
  return min(max((int)((amax_bits + 31u) >> 7) - 2, 8), 252);
}
// the scale as a float; the conversions below use its exponent alone
HS_DEVICE float kv4_scale(int byte) { return __uint_as_float((unsigned)byte << 23); }

// largest magnitude's bits among 8 bf16 values
HS_DEVICE unsigned kv4_amax8(const u16x8 v) {
  unsigned m = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) m = max(m, (unsigned)v[j] & 0x7fffu);
  return m;
}

// 8 bf16 values as 8 codes: nearest level, ties to the even code, magnitudes above 6 to 6 (the conversion's own rounding);
// zeros for a group of scale byte kKv4Nan
HS_DEVICE unsigned kv4_quantise8(const u16x8 v, int byte) {
  if (byte == kKv4Nan) return 0;
  const float s = kv4_scale(byte);
  unsigned r = 0;
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, bf16_to_f32(v[0]), bf16_to_f32(v[1]), s, 0);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, bf16_to_f32(v[2]), bf16_to_f32(v[3]), s, 1);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, bf16_to_f32(v[4]), bf16_to_f32(v[5]), s, 2);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, bf16_to_f32(v[6]), bf16_to_f32(v[7]), s, 3);
  return r;
}

// the two values of byte kByte of w under scale s (its exponent), as two bf16: exact
template <int kByte>
HS_DEVICE unsigned kv4_widen2(unsigned w, float s) {
  return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, kByte));
}

// 8 bf16 values over scale (its exponent) as e4m3 numbers hi + lo / 16: the upper four of their eight significant bits (cut: bf16's
// largest values would round up out of 32 bits' range), and the rest. The rest is taken from hi as it was converted: where hi is subnormal
// (below 2^-6) it has fewer than four bits, and lo holds what they lack down to 2^-13.
HS_DEVICE void kv4_split8(const u16x8 v, float scale, float scale16, u32x2& hi, u32x2& lo) {
  typedef short i16x2 __attribute__((ext_vector_type(2)));
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    float x[4], h[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      x[j] = bf16_to_f32(v[4 * w + j]);
      h[j] = __uint_as_float(__float_as_uint(x[j]) & 0xfff00000u);
    }
    i16x2 hp = {0, 0}, lp = {0, 0};
    hp = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(hp, h[0], h[1], scale, false);
    hp = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(hp, h[2], h[3], scale, true);
    hi[w] = __builtin_bit_cast(unsigned, hp);
    const auto h0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(hi[w], scale, false);
    const auto h1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(hi[w], scale, true);
    lp = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(lp, x[0] - h0[0], x[1] - h0[1], scale16, false);
    lp = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(lp, x[2] - h1[0], x[3] - h1[1], scale16, true);
    lo[w] = __builtin_bit_cast(unsigned, lp);
  }
}

// Scale bytes of the two parts of a query's 32 dims (the keys' groups: what is small in q may meet what is large in a key), hi in byte 0,
// lo in byte 1, from their largest magnitude's bits: that value comes to [128, 256) of e4m3's 448, so values down to 2^-13 of it are exact
// and smaller ones within 2^-21 of it. Of dims that hold a NaN or an infinity both are 255: the query's scores are NaN.
HS_DEVICE int kv4_query_scales(unsigned amax_bits) {
  if (amax_bits >= 0x7f80u) return 0xffff;
  const int e = max((int)(amax_bits >> 7), 16);
  return (e - 7) | (e - 11) << 8;
}
// scores to base 2; never 0, as a hidden key's -inf has to stay one
HS_DEVICE float kv4_score_scale(float scale) { return fmaxf(scale * kLog2E, 1.17549435e-38f); }
constexpr float kKv4Least = -3.4028235e38f;  // where a running maximum begins
// exp2(score * scale - maximum) takes the product unrounded, the maximum is a rounded one: what is between them is a factor of the whole row,
// and no more than 2 up to here. Rows beyond round their products first.
HS_DEVICE bool kv4_far(float m) { return m != kKv4Least && fabsf(m) > 16777216.f; }

// Blocks' ids of a sequence come from its block table. One outside of the cache is no page: its keys are not visible.
HS_DEVICE int kv4_page(int id, long blocks) { return (unsigned)id < (unsigned long)blocks ? id : -1; }

// Whether key j is seen from position pos: not after it, and within the window or among the first tokens that stay visible
HS_DEVICE bool kv4_sees(int j, int pos, int window, int sinks) {
  return j <= pos && (window <= 0 || j > pos - window || j < sinks);
}

}  // namespace hipserve
