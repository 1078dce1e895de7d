// What the attention kernels over the 4-bit cache share: requests, shares of work, partial
// results and the output's rounding.
#pragma once

#include "kv4_common.h"
#include "kv4_launch.h"

namespace w4a16 {

// What a combine needs to join one row tile's partial results.  A workgroup's share of the work is
// contiguous, so it holds at most one tile that began before it (its result goes to slot 2 w) and
// one that ends behind it (slot 2 w + 1); the workgroup where a tile begins describes it.
struct KvSplit {
  int request, head, tile;
  int count;        // partial results (0: this entry joins nothing)
  int first, next;  // slot of the first one, and of the second; the others lie 2 apart from there
};

struct KvPartials {
  float* out;      // [slots][rows][D], unnormalized
  float* stats;    // [slots][rows][2]: maximum (raw score) and sum
  KvSplit* split;  // one a worker
};

// Prompt kernel: rows of a tile, and its grid (a workgroup a CU).
constexpr int kKvPromptRows = 256;
constexpr int kKvPromptWorkers = 256;
// A call goes to the split kernel alone up to this many rows a request (longest query x heads of a
// group); beyond, requests of at most kKvMixedMaxRows rows go to it, the others to the prompt kernel.
constexpr int kKvSplitMaxRows = 64;
constexpr int kKvMixedMaxRows = 32;

hipError_t launch_kv_prompt(const KvAttentionArgs& a, const KvPartials& part, int workers, hipStream_t stream);

// One request as the kernels see it, all lengths safe whatever the tensors hold.
struct KvRequest {
  int row;     // its first packed row
  int n;       // its packed rows
  int cached;  // sequence length before them
  int keys;    // keys that its block table can hold of the sequence
};

__device__ __forceinline__ KvRequest kv_request(const KvAttentionArgs& a, int r) {
  KvRequest q;
  const int lo = a.cu_query_lens[r], hi = a.cu_query_lens[r + 1];
  q.row = min(max(lo, 0), a.T);
  q.n = max(min(hi, a.T) - q.row, 0);
  const int seq = max(a.seq_lens[r], 0);
  q.cached = seq - (hi - lo);
  const int64_t room = static_cast<int64_t>(a.width) << a.log2_block;
  q.keys = seq < room ? seq : static_cast<int>(room);
  return q;
}

// Inclusive sum over the lanes up to this one: DPP moves within rows of 16, then the row totals.
__device__ __forceinline__ int wave_scan(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);  // row 0 -> 1, row 2 -> 3
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);  // lane 31 -> rows 2, 3
  return v;
}

// Equal contiguous shares of `total` units for `workers` workgroups: the first `rest` take one
// more than the others.
struct KvShares {
  int each, rest;
  __device__ __forceinline__ int begin(int w) const { return w * each + min(w, rest); }
  __device__ __forceinline__ int owner(int unit) const {
    const int head = rest * (each + 1);
    return unit < head ? unit / (each + 1) : rest + (unit - head) / each;
  }
};

// out[row, h, ch ..] = o / sum, rounded; a row that saw nothing (or only scores of -inf) is zero.
template <int N>
__device__ __forceinline__ void kv_write(const KvAttentionArgs& a, int row, int h, int ch, float sum, const float (&o)[N]) {
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
  uint16_t* p = a.out + (static_cast<size_t>(row) * a.H + h) * a.D + ch;
  if constexpr (N == 8) {
    *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16x2(o[0] * inv, o[1] * inv), pack_bf16x2(o[2] * inv, o[3] * inv),
                                              pack_bf16x2(o[4] * inv, o[5] * inv), pack_bf16x2(o[6] * inv, o[7] * inv));
  } else if constexpr (N == 4) {
    *reinterpret_cast<uint2*>(p) = make_uint2(pack_bf16x2(o[0] * inv, o[1] * inv), pack_bf16x2(o[2] * inv, o[3] * inv));
  } else if constexpr (N == 2) {
    *reinterpret_cast<uint32_t*>(p) = pack_bf16x2(o[0] * inv, o[1] * inv);
  } else {
    *p = f32_to_bf16_bits(o[0] * inv);
  }
}

}  // namespace w4a16
