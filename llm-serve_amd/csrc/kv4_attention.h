// What the attention kernels over the 4-bit cache share: requests, shares of work, partial
// results and the output's rounding.
#pragma once

#include "kv4_common.h"
#include "kv4_launch.h"

namespace w4a16 {

// Partial results.  A workgroup's share of the work is contiguous, so it covers at most one tile
// that began before it (its part goes to slot 2 w) and one that ends behind it (slot 2 w + 1).
// The workgroups of a tile count their arrivals at the counter of the one where it begins; the
// last to arrive joins the parts in the workgroups' order, so the result does not depend on which
// one that is, and leaves the counter at zero.  Parts travel with the coherent policy of the
// split-K exchange (w4a16_common.h).
struct KvPartials {
  float* out;      // [slots][tile rows][D], unnormalized
  float* stats;    // [slots][tile rows][2]: reference (a raw score; the prompt kernel: its base-2 exponent) and sum
  int* counters;   // [workers]
  uint32_t out_bytes, stats_bytes;
};

inline size_t align256(size_t n) { return (n + 255) / 256 * 256; }

// A kernel's part of the workspace: partial results of 2 tiles of `rows` rows a worker.
inline size_t partials_bytes(int workers, int rows, int D) {
  const size_t n = static_cast<size_t>(2) * workers * rows;
  return align256(n * D * sizeof(float)) + align256(n * 2 * sizeof(float));
}

inline KvPartials partials_at(char* ws, int* counters, int workers, int rows, int D) {
  const size_t n = static_cast<size_t>(2) * workers * rows;
  KvPartials part;
  part.out = reinterpret_cast<float*>(ws);
  part.stats = reinterpret_cast<float*>(ws + align256(n * D * sizeof(float)));
  part.out_bytes = static_cast<uint32_t>(n * D * sizeof(float));
  part.stats_bytes = static_cast<uint32_t>(n * 2 * sizeof(float));
  part.counters = counters;
  return part;
}

// Prompt kernel: rows of a tile, and its grid (a workgroup a CU).
constexpr int kKvPromptRows = 256;
constexpr int kKvPromptWorkers = 256;
// The split kernel's largest grid: three workgroups a CU.
constexpr int kKvSplitWorkers = 768;
static_assert(kKvSplitWorkers + kKvPromptWorkers == kKvAttentionCounters, "a counter a worker");
// Rows a request (tokens x heads of a group) up to which the split kernel takes it.  Below the border it
// is the faster one.  Above it, given longer requests (a caller's hint of 1), it still is for a while: 20
// tokens x 4 heads behind 500, 12000 and 131000 take 14, 27 and 131 us where the prompt kernel takes 26,
// 46 and 263; 64 x 4 take 30, 48 and 355 (31, 62 and 371).  The prompt kernel is the faster one from some
// 400 rows on: 128 x 4 behind 2000 and 12000 take 41 and 71 us there (47 and 80), 256 x 4 42 and 87 (91
// and 137).
constexpr int kKvSplitMaxRows = 64;

hipError_t launch_kv_prompt(const KvAttentionArgs& a, const KvPartials& part, int workers, hipStream_t stream);

// One request as the kernels see it, all lengths safe whatever the tensors hold.
struct KvRequest {
  int row;     // its first packed row
  int n;       // its packed rows
  int cached;  // sequence length before them
  int keys;    // keys that its block table can hold of the sequence
};

// The lists that no kernel here writes, read through the scalar cache where the index is uniform.
typedef const __attribute__((address_space(4))) int32_t* ConstInts;
__device__ __forceinline__ ConstInts const_ints(const int32_t* p) { return (ConstInts)p; }

__device__ __forceinline__ KvRequest kv_request(const KvAttentionArgs& a, int r) {
  KvRequest q;
  const int lo = const_ints(a.cu_query_lens)[r], hi = const_ints(a.cu_query_lens)[r + 1];
  const int seq = max(const_ints(a.seq_lens)[r], 0);
  q.row = min(max(lo, 0), a.T);
  q.n = max(min(hi, a.T) - q.row, 0);
  q.cached = seq - (hi - lo);
  q.keys = min(seq, a.width << a.log2_block);
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

// The largest of the lanes' values, none of them negative.
__device__ __forceinline__ int wave_max(int v) {
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, true));
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, true));
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, true));
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, true));
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false));
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false));
  return __builtin_amdgcn_readlane(v, 63);
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

// out[row, h, ch .. ch + 7] = o / sum, rounded; a row that saw nothing (or only scores of -inf) is zero.
__device__ __forceinline__ void kv_write(const KvAttentionArgs& a, int row, int h, int ch, float sum, const float (&o)[8]) {
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
  float t[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) t[i] = o[i] * inv;
  *reinterpret_cast<uint4*>(a.out + (static_cast<size_t>(row) * a.H + h) * a.D + ch) = pack_bf16x8(t);
}

// Whether request r's offsets decrease.  Offsets that never do give requests of at most T rows in
// all, which bounds every count of work; with others the kernels do none.
__device__ __forceinline__ bool kv_decreases(const KvAttentionArgs& a, int r) {
  return const_ints(a.cu_query_lens)[r + 1] < const_ints(a.cu_query_lens)[r];
}

// Zeros for the output rows of no request: those before the first one's and behind the last one's
// (all rows if there is no work).
template <class Args>
__device__ __forceinline__ void kv_zero_unowned(const Args& a, bool all) {
  const int first = all ? 0 : min(max(const_ints(a.cu_query_lens)[0], 0), a.T);
  const int end = all ? 0 : min(max(const_ints(a.cu_query_lens)[a.R], 0), a.T);
  const int unowned = first + a.T - end, chunks = a.H * a.D / 8;
  for (int i = blockIdx.x; i < unowned; i += gridDim.x) {
    const int row = i < first ? i : end + i - first;
    for (int c = threadIdx.x; c < chunks; c += blockDim.x)
      reinterpret_cast<uint4*>(a.out)[static_cast<size_t>(row) * chunks + c] = make_uint4(0, 0, 0, 0);
  }
}

// One part of a tile row's result: eight channels, or the row's statistics.
__device__ __forceinline__ void store_part(__amdgpu_buffer_rsrc_t r, uint32_t offset, const float (&o)[8]) {
  store_fragment(r, offset, f32x4_t{o[0], o[1], o[2], o[3]});
  store_fragment(r, offset + 16, f32x4_t{o[4], o[5], o[6], o[7]});
}

__device__ __forceinline__ void store_stats(__amdgpu_buffer_rsrc_t r, uint32_t offset, float top, float sum) {
  const u32x2_t v = {__float_as_uint(top), __float_as_uint(sum)};
  __builtin_amdgcn_raw_buffer_store_b64(v, r, offset, 0, kCoherentPolicy);
}

// Whether all other workgroups of a tile of `count` parts have arrived: then this one need not
// store its own.  All threads call it; `flag` is LDS.
__device__ __forceinline__ bool kv_is_last(int* counter, int count, int* flag) {
  if (threadIdx.x == 0)
    *flag = __hip_atomic_load(counter, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == count - 1;
  __syncthreads();
  return *flag != 0;
}

// Counts this workgroup's arrival, its part stored; whether it is the last of `count`.  All
// threads call it; `flag` is LDS.
__device__ __forceinline__ bool kv_arrive(int* counter, int count, int* flag) {
  __builtin_amdgcn_s_waitcnt(0);  // this wave's part has reached memory
  __syncthreads();
  if (threadIdx.x == 0) {
    const bool last = arrive(counter) == count - 1;
    if (last) rearm(counter);
    *flag = last;
  }
  __syncthreads();
  return *flag != 0;
}

// Joins a tile's `count` parts, from worker `first` on, into the output: a thread takes eight
// channels of a row; where a tile has fewer of them than the workgroup has threads, groups of
// threads take every group-th part each and are joined through `scratch` (LDS, 10 floats a thread).
template <int D, int THREADS>
__device__ __forceinline__ void kv_join(const KvAttentionArgs& a, const KvPartials& part, int tile_rows, int first,
                                        int count, const KvRequest& q, int head, int row0, int rows, float* scratch) {
  constexpr int kChunks = D / 8, kBatch = 4;
  const int group = a.H / a.KV, tid = threadIdx.x;
  const int items = rows * kChunks, groups = items < THREADS ? THREADS / items : 1;
  const __amdgpu_buffer_rsrc_t ro = make_buffer(part.out, part.out_bytes), rs = make_buffer(part.stats, part.stats_bytes);
  for (int e0 = 0; e0 < items; e0 += THREADS) {
    const int mine = groups > 1 ? tid / items : 0;
    const int e = groups > 1 ? tid - mine * items : e0 + tid;
    const bool live = e < items && mine < groups;
    const int row = e / kChunks, ch = e % kChunks * 8;
    float top = -INFINITY, sum = 0.0f, o[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    for (int i0 = mine; i0 < count && live; i0 += kBatch * groups) {
      f32x4_t lo[kBatch], hi[kBatch];
      u32x2_t st[kBatch];
#pragma unroll
      for (int b = 0; b < kBatch; ++b) {
        const int i = i0 + b * groups;
        const uint32_t at = static_cast<uint32_t>(i == 0 ? 2 * first + 1 : 2 * (first + i)) * tile_rows + row;
        const bool in = i < count;  // loads beyond the last part touch nothing and give zeros
        st[b] = __builtin_bit_cast(u32x2_t, __builtin_amdgcn_raw_buffer_load_b64(rs, in ? at * 8 : kOutOfRange, 0, kCoherentPolicy));
        lo[b] = load_fragment(ro, in ? (at * D + ch) * 4 : kOutOfRange);
        hi[b] = load_fragment(ro, in ? (at * D + ch) * 4 + 16 : kOutOfRange);
      }
#pragma unroll
      for (int b = 0; b < kBatch; ++b) {
        const uint32_t mb = st[b][0], lb = st[b][1];
        const float m = i0 + b * groups < count ? __uint_as_float(mb) : -INFINITY;
        const float next = fmaxf(top, m), ref = next == -INFINITY ? 0.0f : next;
        const float f = __builtin_amdgcn_exp2f((top - ref) * a.scale_log2e);
        const float g = __builtin_amdgcn_exp2f((m - ref) * a.scale_log2e);
        top = next;
        sum = sum * f + __uint_as_float(lb) * g;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          o[j] = o[j] * f + lo[b][j] * g;
          o[4 + j] = o[4 + j] * f + hi[b][j] * g;
        }
      }
    }
    if (groups > 1) {
      if (live) {
        float* s = scratch + tid * 10;
        s[0] = top;
        s[1] = sum;
#pragma unroll
        for (int j = 0; j < 8; ++j) s[2 + j] = o[j];
      }
      __syncthreads();
      if (mine > 0) return;
      for (int k = 1; k < groups; ++k) {
        const float* s = scratch + (tid + k * items) * 10;
        const float next = fmaxf(top, s[0]), ref = next == -INFINITY ? 0.0f : next;
        const float f = __builtin_amdgcn_exp2f((top - ref) * a.scale_log2e);
        const float g = __builtin_amdgcn_exp2f((s[0] - ref) * a.scale_log2e);
        top = next;
        sum = sum * f + s[1] * g;
#pragma unroll
        for (int j = 0; j < 8; ++j) o[j] = o[j] * f + s[2 + j] * g;
      }
    }
    if (live) {
      const int token = (row0 + row) / group;
      kv_write(a, q.row + token, head * group + row0 + row - token * group, ch, sum, o);
    }
  }
}

}  // namespace w4a16
