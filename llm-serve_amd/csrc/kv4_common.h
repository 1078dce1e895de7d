// The 4-bit key/value cache: its layout, and the device helpers its kernels share.
//
// Cache: bytes [num_blocks, kv_heads, page], page = block_size * (D + 8), one page per (block,
// kv head).  A row (one token, one kv head) of D channels is held as codes c in 0..15 with one
// scale s and one zero point z, and channel x stands for s (c - z).  Inside a page:
//   K codes  block_size rows of D / 8 words
//   V codes  [token / 4][word][token % 4]: the words of four tokens interleaved
//   K meta, V meta  one word a token each: bf16(s) in the high half, bf16(128 + z) in the low
// Channel c = 0..7 of a word sits at bit awq_shift(c), AutoAWQ's nibble order, so that the four
// words ((w >> 4 i) & 0x000F000F) | 0x43004300 are its channels in order, as exact bf16 pairs
// (128 + code): a matrix operand without a multiplication.  128 + z has the same form, which
// makes the zero point an operand too.
//
// Why V is interleaved: the values' operand has eight *tokens* of one channel in a lane.  A lane
// of the attention kernels takes one 16-byte load, the same word of four tokens, and one
// v_perm_b32 per four channels pairs two tokens' nibbles; rows in K's order would cost eight
// 4-byte loads.  A token still owns whole words, so rows are stored without read-modify-write.
#pragma once

#include "w4a16_common.h"

namespace w4a16 {

// Blocks are a power of two of at least 16 tokens, so a 16-token matrix tile never leaves its page.
template <int D>
__device__ __forceinline__ size_t kv_page_bytes(int log2_block) {
  return static_cast<size_t>(D + 8) << log2_block;
}

// Word offset of a token's V word w inside the V part of its page.
template <int D>
__device__ __forceinline__ int kv_v_word(int token, int w) {
  return ((token >> 2) * (D / 8) + w) * 4 + (token & 3);
}

__device__ __forceinline__ uint32_t kv_meta(float scale, int zero) {
  return (pack_bf16x2(scale, 0.0f) << 16) | 0x4300u | static_cast<uint32_t>(zero);
}

__device__ __forceinline__ float kv_meta_scale(uint32_t meta) { return __uint_as_float(meta & 0xFFFF0000u); }
// 128 + zero point.
__device__ __forceinline__ float kv_meta_zero128(uint32_t meta) { return __uint_as_float(meta << 16); }

// Sum / maximum of a value over the four lanes l % 16, l % 16 + 16, + 32, + 48 (the lanes that
// hold one column of a 16x16 accumulator), every lane getting the same bits.  v_permlane16_swap
// and v_permlane32_swap exchange whole rows of 16 lanes and halves in registers.
__device__ __forceinline__ float column_max(float v) {
  const u32x2_t a = __builtin_bit_cast(
      u32x2_t, __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false));
  v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const u32x2_t b = __builtin_bit_cast(
      u32x2_t, __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false));
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

__device__ __forceinline__ float column_sum(float v) {
  const u32x2_t a = __builtin_bit_cast(
      u32x2_t, __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false));
  v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  const u32x2_t b = __builtin_bit_cast(
      u32x2_t, __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false));
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// Eight codes of a word -> eight exact bf16 values (128 + code), in channel order.
__device__ __forceinline__ bf16x8_t unpack_codes(uint32_t w, const NibbleConsts& k) {
  u32x4_t r;
  r[0] = (w & k.mask) | k.bias;
  r[1] = ((w >> 4) & k.mask) | k.bias;
  r[2] = ((w >> 8) & k.mask) | k.bias;
  r[3] = ((w >> 12) & k.mask) | k.bias;
  return __builtin_bit_cast(bf16x8_t, r);
}

}  // namespace w4a16
