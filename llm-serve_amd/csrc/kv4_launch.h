// Host-side launchers of the 4-bit key/value cache kernels (kv4_cache.hip, kv4_attention.hip), of the
// norm and rotation in front of them (qk_rope.hip) and of prompt attention in bf16 (prompt_attention.hip).
// Arguments are checked by the callers (w4a16_api.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace w4a16 {

// Requests of one step: the kernel keeps three ints of each in LDS.
constexpr int kKvStepMaxRequests = 4096;
// Packed rows of one step; with kKvStepMaxRequests lengths clamped to it, sums stay below 2^31.
constexpr int kKvStepMaxTokens = 1 << 18;

// Tokens that a block table's row may reach.  A sequence's keys rounded up to the kernels' tiles, and
// a step's tokens behind it, then stay below 2^31.
constexpr int64_t kKvMaxReach = 0x7FFFFFFF - (1 << 19);

struct KvStepArgs {
  const int32_t* query_lens;    // [R]
  const int32_t* context_lens;  // [R]
  int32_t* tables;              // [R, width], row stride table_stride
  const int32_t* free_blocks;   // [num_free]
  int32_t* cu_query_lens;       // [R + 1]
  int32_t* seq_lens;            // [R]
  int32_t* positions;           // [T]
  int32_t* slots;               // [T]
  int32_t* blocks_used;         // [1]
  int64_t table_stride;
  int R, width, num_free, log2_block, T;
};
hipError_t launch_kv_step(const KvStepArgs& a, hipStream_t stream);

struct KvRowsArgs {
  uint16_t* k;  // [T, KV, D], rows of D contiguous channels at the strides below (elements)
  uint16_t* v;
  int64_t k_stride_t, k_stride_h, v_stride_t, v_stride_h;
  uint8_t* cache;
  const int32_t* slots;  // [T]
  int T, KV, D, num_blocks, log2_block;
};
hipError_t launch_kv_store(const KvRowsArgs& a, hipStream_t stream);
hipError_t launch_kv_load(const KvRowsArgs& a, hipStream_t stream);

// Up to this many tokens a wave of the norm-and-rotation kernel takes one group of heads, whatever the heads
// (qk_rope.hip has both sides measured).
constexpr int kQkRopeFewTokens = 2048;

struct QkRopeArgs {
  const uint16_t *q, *k, *v;  // [T, H or KV, D] at strides (elements); v only with a cache
  int64_t q_stride_t, q_stride_h, k_stride_t, k_stride_h, v_stride_t, v_stride_h;
  const int32_t* positions;  // [T]
  const float* table;        // [table_rows, rotary]: cosines, then sines
  const uint16_t *q_weight, *k_weight;  // [D], or null: no norm
  uint16_t* q_out;           // [T, H, D]
  uint16_t* k_out;           // [T, KV, D], or null with a cache
  uint8_t* cache;            // or null: keys and values are not stored
  const int32_t* slots;      // [T]
  float eps;
  int T, H, KV, D, table_rows, rotary, num_blocks, log2_block;
};
hipError_t launch_qk_rope(const QkRopeArgs& a, hipStream_t stream);

struct KvAttentionArgs {
  const uint16_t* q;  // [T, H, D] at strides (elements)
  int64_t q_stride_t, q_stride_h;
  const uint8_t* cache;
  const int32_t* tables;
  int64_t table_stride;
  const int32_t* seq_lens;
  const int32_t* cu_query_lens;
  const uint64_t* tree_mask;  // [T] or null
  uint16_t* out;              // [T, H, D] contiguous
  float scale_log2e;
  int T, R, H, KV, D, num_blocks, log2_block, width;
  int max_query_len;
  int split_rows;  // requests of more rows (tokens x heads of a group) are the prompt kernel's
  bool zero_tail;
};
size_t kv_attention_workspace(const KvAttentionArgs& a);
// counters: kKvAttentionCounters ints, zero before and after the call's kernels.
constexpr int kKvAttentionCounters = 1024;
hipError_t launch_kv_attention(const KvAttentionArgs& a, void* workspace, int* counters, hipStream_t stream);

struct PromptArgs {
  const uint16_t *q, *k, *v;  // [T, H or KV, D] at strides (elements)
  int64_t q_stride_t, q_stride_h, k_stride_t, k_stride_h, v_stride_t, v_stride_h;
  const int32_t* cu_query_lens;
  uint16_t* out;  // [T, H, D] contiguous
  float scale_log2e;
  int T, R, H, KV, D;
  int group;              // H / KV, and x / group = x * group_inverse >> group_shift for 0 <= x < 2^31
  uint32_t group_inverse;
  int group_shift;
  bool zero_tail;
  int tile_rows, cost_shift, part_workers;  // plan_prompt_attention's
};
// Steps of up to this many rows (the most that w4a16_kv_step makes) are planned whatever their number of requests.
constexpr int kPromptStepRows = 1 << 18;
// The rows (tokens x heads of a group) of a row tile, the unit that work is counted in and the workers that may hand
// over parts of row tiles, for a call of these sizes (T, R, H, KV, D); false: its work may pass 32 bits.
bool plan_prompt_attention(PromptArgs* a);
size_t prompt_attention_workspace(const PromptArgs& a);
// counters: kKvAttentionCounters ints, zero before and after the call's kernel.
hipError_t launch_prompt_attention(const PromptArgs& a, void* workspace, int* counters, hipStream_t stream);

}  // namespace w4a16
