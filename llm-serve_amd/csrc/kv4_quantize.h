// Rows quantized on their way into the 4-bit key/value cache, in registers.
#pragma once

#include "kv4_common.h"

namespace w4a16 {

// Maximum over the LANES neighbouring lanes (4, 8 or 16) of a row, every lane getting it.
template <int LANES>
__device__ __forceinline__ float lanes_max(float v) {
  v = fmaxf(v, dpp_f32<0xB1>(v));
  v = fmaxf(v, dpp_f32<0x4E>(v));
  if (LANES >= 8) v = fmaxf(v, dpp_f32<0x141>(v));
  if (LANES == 16) v = fmaxf(v, dpp_f32<0x140>(v));
  return v;
}

// x / s rounded to a multiple of 2^-11 (|x / s| < 16), by the reciprocal: enough to round it to a
// code as the exact quotient would be.  x and s have at most 8 significant bits: where x / s lies
// near a border k + 1/2 between two codes, |x| > s / 4 makes 2 x - (2 k + 1) s a multiple of s's
// last place, so x / s is the border itself or at least 1 / 510 away.  The product is off by 2^-18
// at most, and the sum with 1.5 * 2^12, whose last place is 2^-11, then returns a border as it is
// and moves nothing across one.
__device__ __forceinline__ float near_quotient(float x, float inverse) { return (x * inverse + 6144.0f) - 6144.0f; }

// One row's channels in LANES neighbouring lanes, WORDS eights of them in each -> their code words; returns
// the row's meta word.  All lanes of a row must be active.  The range takes in zero, so z is in
// 0..15 and a row of one sign keeps its far end.  The scale is rounded to bf16 (the cache's type)
// before the codes are formed, so codes are right for the scale that readers multiply by.  A row
// with a NaN or infinity becomes NaN as a whole; a range beyond fp32 is formed a sixteenth at a
// time; scales too small for the reciprocal take the division.
template <int LANES, int WORDS>
__device__ __forceinline__ uint32_t quantize_row(const uint4 (&raw)[WORDS], int lane, uint32_t (&words)[WORDS]) {
  typedef uint16_t u16x2_t __attribute__((ext_vector_type(2)));
  float x[WORDS][8];
  u16x2_t top = {0, 0};
  float hi = 0.0f, lo = 0.0f;
#pragma unroll
  for (int j = 0; j < WORDS; ++j) {
    unpack_bf16x8(raw[j], x[j]);
    const uint32_t w[4] = {raw[j].x, raw[j].y, raw[j].z, raw[j].w};
#pragma unroll
    for (int i = 0; i < 4; ++i) top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2_t, w[i] & 0x7FFF7FFFu));
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      hi = fmaxf(hi, x[j][i]);
      lo = fminf(lo, x[j][i]);
    }
    words[j] = 0;
  }
  const bool bad = top[0] >= 0x7F80 || top[1] >= 0x7F80;
  hi = lanes_max<LANES>(hi);
  lo = -lanes_max<LANES>(-lo);
  constexpr uint64_t kRow = (1ull << LANES) - 1;
  if (__ballot(bad) >> (lane & ~(LANES - 1)) & kRow) return 0x7FC04300u;
  const float range = hi - lo;
  const float exact = __builtin_isinf(range) ? (hi * 0.0625f - lo * 0.0625f) / 15.0f * 16.0f : range / 15.0f;
  const float s = bf16_bits_to_f32(pack_bf16x2(exact, 0.0f) & 0xFFFFu);
  if (!(s > 0.0f)) return 0x00004300u;  // all zeros, or below the smallest scale
  float t[WORDS][8], z;
  if (s < 0x1p-100f || s > 0x1p100f) {
    z = rintf(-lo / s);
#pragma unroll
    for (int j = 0; j < WORDS; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i) t[j][i] = x[j][i] / s;
  } else {
    const float inverse = __builtin_amdgcn_rcpf(s);
    z = rintf(near_quotient(-lo, inverse));
#pragma unroll
    for (int j = 0; j < WORDS; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i) t[j][i] = near_quotient(x[j][i], inverse);
  }
  z = fminf(z, 15.0f);
#pragma unroll
  for (int j = 0; j < WORDS; ++j) {
    uint32_t c[8];  // the code in the low bits of 2^23 + code
#pragma unroll
    for (int i = 0; i < 8; ++i)
      c[i] = __float_as_uint(__builtin_amdgcn_fmed3f(rintf(t[j][i]), -z, 15.0f - z) + (z + 8388608.0f));
    const uint32_t p0 = __builtin_amdgcn_perm(c[1], c[0], 0x05040100u), p1 = __builtin_amdgcn_perm(c[3], c[2], 0x05040100u);
    const uint32_t p2 = __builtin_amdgcn_perm(c[5], c[4], 0x05040100u), p3 = __builtin_amdgcn_perm(c[7], c[6], 0x05040100u);
    words[j] = p0 | (p1 << 4) | (p2 << 8) | (p3 << 12);
  }
  return kv_meta(s, static_cast<int>(z));
}

}  // namespace w4a16
