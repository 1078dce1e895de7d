// What the kernels of long queries share: workgroups of WAVES waves with 32 rows each, whose output O^T lies in
// accumulators of 32 x 32 -- a lane has one row, lane % 32, and of each 32 channels those of its half of
// the wave, lane / 32 -- and goes to the output, or to a part of it that is joined with others.
#pragma once

#include "kv4_attention.h"

namespace w4a16 {

typedef float f32x16_t __attribute__((ext_vector_type(16)));

__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

constexpr int kKeyTileCost = 16;  // cost units of a tile of 64 keys

// Cost of a request's row tiles: tile j of a head costs first + step j, its keys growing with its last
// token (all keys under a tree mask), plus its set-up.  Host checks keep all sums below 2^31.
struct KvTileCosts {
  int tiles, first, step;
  __device__ __forceinline__ int before(int j) const {
    return j * first + static_cast<int>(static_cast<unsigned>(step) * static_cast<unsigned>(j) * static_cast<unsigned>(j - 1) / 2u);
  }
  __device__ __forceinline__ int of(int j) const { return first + step * j; }
};

// Sum / maximum of a value over a lane and the one of the wave's other half.
__device__ __forceinline__ u32x2_t halves(float v) {
  return __builtin_bit_cast(u32x2_t, __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false));
}
__device__ __forceinline__ float halves_sum(float v) {
  const u32x2_t b = halves(v);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}
__device__ __forceinline__ float halves_max(float v) {
  const u32x2_t b = halves(v);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

// l 2^d, also where 2^d alone lies below fp32's range.
__device__ __forceinline__ float scaled(float l, float d) {
  const float h = __builtin_amdgcn_exp2f(0.5f * d);
  return l * h * h;
}

// Byte offset of a lane's fragment f (four channels: 32 (f / 4) + 8 (f % 4) + 4 (lane / 32) ..) of
// its wave's 32 rows in slot `slot`: whole waves of 16 bytes a lane, in the accumulators' layout.
template <int D, int WAVES>
__device__ __forceinline__ uint32_t part_offset(int slot, int wave, int f, int lane) {
  return ((static_cast<uint32_t>(slot) * WAVES + wave) * (D / 8) + f) * 1024u + lane * 16u;
}

// Two fragments of a lane -- channels 4 h .. of eights b and b + 1 -- times inv, rounded: the halves of the
// wave exchange theirs, so that a lane has one eight's 16 bytes, b + lane / 32.
__device__ __forceinline__ u32x4_t row_pair(float inv, const f32x4_t& x, const f32x4_t& y) {
  const u32x2_t lo = __builtin_bit_cast(u32x2_t, __builtin_amdgcn_permlane32_swap(pack_bf16x2(x[0] * inv, x[1] * inv),
                                                                                  pack_bf16x2(y[0] * inv, y[1] * inv), false, false));
  const u32x2_t hi = __builtin_bit_cast(u32x2_t, __builtin_amdgcn_permlane32_swap(pack_bf16x2(x[2] * inv, x[3] * inv),
                                                                                  pack_bf16x2(y[2] * inv, y[3] * inv), false, false));
  return u32x4_t{lo[0], hi[0], lo[1], hi[1]};
}

// Writes a wave's rows, o / sum (rows that saw nothing are zero), to out [T, H, D] of the kernel's arguments.
template <int D, class Args>
__device__ __forceinline__ void write_rows(const Args& a, bool live, int row, int head, int lane, float sum,
                                           const f32x4_t (&o)[D / 8]) {
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
  for (int f = 0; f < D / 8; f += 2) {
    const u32x4_t w = row_pair(inv, o[f], o[f + 1]);
    if (live) *reinterpret_cast<u32x4_t*>(a.out + (static_cast<size_t>(row) * a.H + head) * D + 8 * (f + (lane >> 5))) = w;
  }
}

// Joins a tile's `count` parts, from worker `first` on, into `own` (channels) and `own_sum`; part `mine` is
// this workgroup's own, in these registers.  Parts are taken in order, one at a time: there are registers for
// one part's fragments beside the sums, so each part's loads are waited for before the next one's are sent.
template <int D, int WAVES>
__device__ __forceinline__ void join_parts(const KvPartials& part, int first, int count, int mine, int wave, int lane,
                                           bool live, float own_top, float& own_sum, f32x4_t (&own)[D / 8]) {
  constexpr int kFrags = D / 8;
  const __amdgpu_buffer_rsrc_t ro = make_buffer(part.out, part.out_bytes), rs = make_buffer(part.stats, part.stats_bytes);
  float top = -INFINITY, sum = 0.0f;
  f32x4_t acc[kFrags], v[kFrags];
#pragma unroll
  for (int f = 0; f < kFrags; ++f) acc[f] = f32x4_t{0, 0, 0, 0};
  for (int i = 0; i < count; ++i) {
    float m = own_top, l = own_sum;
    if (i == mine) {
#pragma unroll
      for (int f = 0; f < kFrags; ++f) v[f] = own[f];
    } else {
      const int slot = i == 0 ? 2 * first + 1 : 2 * (first + i);
      const uint32_t row = static_cast<uint32_t>(slot) * (32 * WAVES) + 32 * wave + (lane & 31);
      const u32x2_t st = __builtin_bit_cast(
          u32x2_t, __builtin_amdgcn_raw_buffer_load_b64(rs, live ? row * 8 : kOutOfRange, 0, kCoherentPolicy));
      const uint32_t mb = st[0], lb = st[1];
      m = __uint_as_float(mb), l = __uint_as_float(lb);
#pragma unroll
      for (int f = 0; f < kFrags; ++f) v[f] = load_fragment(ro, live ? part_offset<D, WAVES>(slot, wave, f, lane) : kOutOfRange);
    }
    const float next = fmaxf(top, m), ref = next == -INFINITY ? 0.0f : next;
    const float x = __builtin_amdgcn_exp2f(top - ref), y = __builtin_amdgcn_exp2f(m - ref);
    sum = scaled(sum, top - ref) + scaled(l, m - ref);
    top = next;
#pragma unroll
    for (int f = 0; f < kFrags; ++f)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[f][j] = acc[f][j] * x + v[f][j] * y;
  }
  own_sum = sum;
#pragma unroll
  for (int f = 0; f < kFrags; ++f) own[f] = acc[f];
}

}  // namespace w4a16
