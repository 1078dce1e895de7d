// Per-head norm and position rotation of queries and keys, in one pass from the QKV projection's
// output, and on the way into the 4-bit cache.
//
// A row x (one token, one head) of D channels becomes, with r = 1 / sqrt(mean(x^2) + eps), weight w
// and the cosines and sines of its token's position,
//   y = x r w,   z[i] = y[i] cos[i] - y[i + R/2] sin[i],   z[i + R/2] = y[i + R/2] cos[i] + y[i] sin[i]
// for i < R / 2; channels from R on are y.  z is rounded to bf16 once.  All of it is fp32 in this
// order, each product and sum rounded by itself; the sum of squares is fp64.  Keys are quantized
// behind it, and a last bit may move a key across the border between two codes: with the order of
// the arithmetic pinned, a key gets the same code whichever entry point forms it, and any program
// of the formulas' plain operations gives the same bits.
//
// Bytes bound it: each row is read and written once, the table's row of a token is read once for all of
// the token's heads that a wave takes.  16384 tokens of 32 + 8 heads of 128 channels move 335 MB in 68 us
// (4.9 TB/s, where a large copy reaches 5.2), with the store into the cache behind it, keys written too, 387 MB in
// 80 us; few tokens take the 3 us of a launch whose loads wait for each other twice (position, then table).
#include "kv4_launch.h"
#include "kv4_quantize.h"

namespace w4a16 {
namespace {

// A lane's part of the token's rotation: channels lo .. lo + 7 turn with hi .. hi + 7.
struct Turn {
  float cos[8], sin[8];
  bool rotates, inside;  // inside: the table has the token's position
};

template <int CTRL>
__device__ __forceinline__ double add_dpp(double v) {
  const u32x2_t w = __builtin_bit_cast(u32x2_t, v);
  u32x2_t u;
  u[0] = __builtin_amdgcn_update_dpp(0, static_cast<int>(w[0]), CTRL, 0xF, 0xF, false);
  u[1] = __builtin_amdgcn_update_dpp(0, static_cast<int>(w[1]), CTRL, 0xF, 0xF, false);
  return v + __builtin_bit_cast(double, u);
}

// Sum over the LANES neighbouring lanes (4 or 8) of a row, every lane getting the same bits.
template <int LANES>
__device__ __forceinline__ double lanes_sum(double v) {
  v = add_dpp<0xB1>(v);
  v = add_dpp<0x4E>(v);
  if (LANES == 8) v = add_dpp<0x141>(v);
  return v;
}

// The lane's two eights of a row, normed (with a weight) and rotated.
template <int D>
__device__ __forceinline__ void turn_row(uint4 (&x)[2], bool norm, const uint4 (&weight)[2], float eps, const Turn& t) {
#pragma clang fp contract(off)
  float y[2][8];
  unpack_bf16x8(x[0], y[0]);
  unpack_bf16x8(x[1], y[1]);
  if (norm) {
    double sum = 0.0;
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const double d = static_cast<double>(y[j][i]);
        sum = __builtin_fma(d, d, sum);
      }
    const float r = rsqrt_rn(static_cast<float>(lanes_sum<D / 16>(sum) * (1.0 / D)) + eps);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      float w[8];
      unpack_bf16x8(weight[j], w);
#pragma unroll
      for (int i = 0; i < 8; ++i) y[j][i] = y[j][i] * r * w[i];
    }
  }
  if (t.rotates) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float a = y[0][i], b = y[1][i];
      const float ac = a * t.cos[i], bs = b * t.sin[i], bc = b * t.cos[i], as = a * t.sin[i];
      y[0][i] = ac - bs;
      y[1][i] = bc + as;
    }
  }
  x[0] = pack_bf16x8(y[0]);
  x[1] = pack_bf16x8(y[1]);
  if (!t.inside) x[0] = x[1] = make_uint4(0x7FC07FC0u, 0x7FC07FC0u, 0x7FC07FC0u, 0x7FC07FC0u);
}

// A wave takes one token and a share of its rows -- the heads of q, then k, then v -- D / 16 lanes a row
// with 16 channels each, so that a rotating pair lies in one lane, and HEADS groups of 64 / (D / 16)
// rows at a time, all loaded before the first is used.
//
// While there are few tokens, waves that take all of a token's rows, three groups at a time, are too few to hide
// what they wait for (2048 of them are two a SIMD), and each group of rows has a wave of its own (HEADS 1, a
// grid of groups): 3.0 us instead of 5.3 for 8 tokens of 32 + 8 heads of 128 channels, 6.0 instead of 6.8 for
// 1024, 9.8 instead of 10.2 for 2048.  With more tokens, reading weights and table once for all of a token's
// rows wins: 15.4 us instead of 16.4 for 4096, 66 instead of 81 for 16384.  So the border is a number of tokens,
// whatever the heads.  Of 256 to 16384 tokens, with and without the store, one form is ahead up to 2048 and the
// other from 4096 on, but for a few sizes in which they are within 6 %, in 64 + 8 and 8 + 2 heads of 128 (2048:
// 15.5 and 15.9, 4.8 and 4.8; 16384: 152 and 127, 23 and 19) and in 16 + 16 and 14 + 2 of 64 (2048 with the store: 6.6
// and 6.9, 6.3 and 7.0; 16384: 37 and 32, 30 and 27); at 3000 they are within 6 % of each other.  One group at a
// time instead of three takes 3 % longer there with the store, four take 4 % longer.
template <int D, int HEADS>
__global__ __launch_bounds__(256) void qk_rope_kernel(QkRopeArgs a) {
  constexpr int kLanes = D / 16, kRows = 64 / kLanes;
  const int lane = threadIdx.x & 63, p = lane % kLanes, r = lane / kLanes;
  // Workgroups go to the 8 XCDs in turn; each XCD takes neighbouring tokens, whose words in the cache
  // share lines.
  const int blocks = (a.T + 3) / 4, per_xcd = (blocks + 7) / 8;
  const int block = static_cast<int>(blockIdx.x & 7) * per_xcd + static_cast<int>(blockIdx.x >> 3);
  const int token = block * 4 + wave_id();
  if (static_cast<int>(blockIdx.x >> 3) >= per_xcd || token >= a.T) return;

  const int half = a.rotary / 2;
  const int position = a.positions[token];
  Turn t;
  t.inside = static_cast<unsigned>(position) < static_cast<unsigned>(a.table_rows);
  t.rotates = 8 * p < half;
  const int lo = t.rotates ? 8 * p : 16 * p, hi = t.rotates ? lo + half : lo + 8;
  if (t.rotates & t.inside) {
    const float* row = a.table + static_cast<int64_t>(position) * a.rotary + lo;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float4 c = reinterpret_cast<const float4*>(row)[i], s = reinterpret_cast<const float4*>(row + half)[i];
      t.cos[4 * i] = c.x, t.cos[4 * i + 1] = c.y, t.cos[4 * i + 2] = c.z, t.cos[4 * i + 3] = c.w;
      t.sin[4 * i] = s.x, t.sin[4 * i + 1] = s.y, t.sin[4 * i + 2] = s.z, t.sin[4 * i + 3] = s.w;
    }
  }
  uint4 q_weight[2] = {}, k_weight[2] = {};
  if (a.q_weight) {
    q_weight[0] = *reinterpret_cast<const uint4*>(a.q_weight + lo);
    q_weight[1] = *reinterpret_cast<const uint4*>(a.q_weight + hi);
  }
  if (a.k_weight) {
    k_weight[0] = *reinterpret_cast<const uint4*>(a.k_weight + lo);
    k_weight[1] = *reinterpret_cast<const uint4*>(a.k_weight + hi);
  }
  const int slot = a.cache ? a.slots[token] : -1, id = slot >> a.log2_block;
  const bool stored = slot >= 0 && id < a.num_blocks;
  const int in_page = slot & ((1 << a.log2_block) - 1);

  const int heads = a.H + a.KV, rows = heads + (a.cache ? a.KV : 0);
  const int64_t at = token;
  for (int row0 = blockIdx.y * kRows * HEADS; row0 < rows; row0 += gridDim.y * kRows * HEADS) {
    uint4 x[HEADS][2];
#pragma unroll
    for (int i = 0; i < HEADS; ++i) {
      const int row = row0 + i * kRows + r;
      x[i][0] = x[i][1] = make_uint4(0, 0, 0, 0);
      if (row < rows) {
        const uint16_t* src = row < a.H   ? a.q + at * a.q_stride_t + row * a.q_stride_h
                              : row < heads ? a.k + at * a.k_stride_t + (row - a.H) * a.k_stride_h
                                            : a.v + at * a.v_stride_t + (row - heads) * a.v_stride_h;
        x[i][0] = *reinterpret_cast<const uint4*>(src + lo);
        x[i][1] = *reinterpret_cast<const uint4*>(src + hi);
      }
    }
#pragma unroll
    for (int i = 0; i < HEADS; ++i) {
      const int row = row0 + i * kRows + r;
      if (row < a.H) {
        turn_row<D>(x[i], a.q_weight != nullptr, q_weight, a.eps, t);
        uint16_t* out = a.q_out + (at * a.H + row) * D;
        *reinterpret_cast<uint4*>(out + lo) = x[i][0];
        *reinterpret_cast<uint4*>(out + hi) = x[i][1];
      } else if (row < rows) {
        const bool is_k = row < heads;
        const int head = row - (is_k ? a.H : heads);
        if (is_k) {
          turn_row<D>(x[i], a.k_weight != nullptr, k_weight, a.eps, t);
          if (a.k_out) {
            uint16_t* out = a.k_out + (at * a.KV + head) * D;
            *reinterpret_cast<uint4*>(out + lo) = x[i][0];
            *reinterpret_cast<uint4*>(out + hi) = x[i][1];
          }
        }
        if (stored) {
          uint32_t words[2];
          const uint32_t meta = quantize_row<kLanes>(x[i], lane, words);
          uint32_t* page = reinterpret_cast<uint32_t*>(
              a.cache + (static_cast<size_t>(id) * a.KV + head) * kv_page_bytes<D>(a.log2_block));
          const int part = (D / 8) << a.log2_block;  // words of the K or V codes
          const int w0 = lo / 8, w1 = hi / 8;
          page[is_k ? in_page * (D / 8) + w0 : part + kv_v_word<D>(in_page, w0)] = words[0];
          page[is_k ? in_page * (D / 8) + w1 : part + kv_v_word<D>(in_page, w1)] = words[1];
          if (p == 0) page[2 * part + (is_k ? 0 : 1 << a.log2_block) + in_page] = meta;
        }
      }
    }
  }
}

template <int D>
hipError_t launch(const QkRopeArgs& a, hipStream_t stream) {
  constexpr int kRows = 1024 / D;
  const int rows = a.H + a.KV + (a.cache ? a.KV : 0), groups = (rows + kRows - 1) / kRows;
  const unsigned blocks = static_cast<unsigned>((a.T + 3) / 4 + 7) / 8 * 8;
  if (a.T <= kQkRopeFewTokens)
    qk_rope_kernel<D, 1><<<dim3(blocks, groups), 256, 0, stream>>>(a);
  else
    qk_rope_kernel<D, 3><<<dim3(blocks, 1), 256, 0, stream>>>(a);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_qk_rope(const QkRopeArgs& a, hipStream_t stream) {
  return a.D == 64 ? launch<64>(a, stream) : launch<128>(a, stream);
}

}  // namespace w4a16
