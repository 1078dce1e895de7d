// The 4-bit key/value cache's bookkeeping and rows: the step's slots and block tables from the
// request lengths, quantizing rows into the cache, and reading rows back.
#include "kv4_common.h"
#include "kv4_launch.h"

namespace w4a16 {
namespace {

constexpr int kStepThreads = 256;

// Inclusive scan of v over the workgroup's 256 threads; `part` is 4 ints of LDS.
__device__ __forceinline__ int block_scan(int v, int* part, int* total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int u = __shfl_up(v, d);
    if (lane >= d) v += u;
  }
  if (lane == 63) part[wave] = v;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kStepThreads / 64; ++w) {
    if (w < wave) before += part[w];
    all += part[w];
  }
  *total = all;
  return v + before;
}

// One launch, no exchange between workgroups: each scans all request lengths (they fit its
// registers and LDS and come from L2), then places its own 256 packed rows by a binary search
// of the row offsets.  The block of a row's position is the table's where the request had it
// before this step, and else the free list's at the request's offset -- so nothing that another
// workgroup writes is read.  A row that opens a block enters it in the table; rows cover all
// positions of a request, so each new block is entered exactly once.  Where the lengths count more
// rows than there are, the blocks that rows behind the last one would open are entered by request,
// so that every block counted in blocks_used is in its table.  Latency bounds it: two
// dependent loads, a scan, and the search.  2.5 us for 8 decode requests, 4.3 us for 512 rows of
// requests with chunks among them.
__global__ __launch_bounds__(kStepThreads) void kv_step_kernel(KvStepArgs a) {
  __shared__ int s_first_row[kKvStepMaxRequests + 1];
  __shared__ int s_first_block[kKvStepMaxRequests];
  __shared__ int s_context[kKvStepMaxRequests];
  __shared__ int part[2][kStepThreads / 64];
  const int tid = threadIdx.x;
  const int per = (a.R + kStepThreads - 1) / kStepThreads;
  const int r0 = tid * per, r1 = min(a.R, r0 + per);
  const int block = 1 << a.log2_block;
  const int max_context = a.width << a.log2_block;  // no cached token lies behind the table; sums stay in range
  int rows = 0, blocks = 0;
  for (int r = r0; r < r1; ++r) {
    const int n = min(max(a.query_lens[r], 0), kKvStepMaxTokens);
    const int c = min(max(a.context_lens[r], 0), max_context);
    s_context[r] = c;
    s_first_row[r] = n;
    rows += n;
    blocks += ((c + n + block - 1) >> a.log2_block) - ((c + block - 1) >> a.log2_block);
  }
  int total_rows, total_blocks;
  int row = block_scan(rows, part[0], &total_rows) - rows;
  int at = block_scan(blocks, part[1], &total_blocks) - blocks;
  const bool first = blockIdx.x == 0;
  for (int r = r0; r < r1; ++r) {
    const int n = s_first_row[r], c = s_context[r];
    s_first_row[r] = row;
    s_first_block[r] = at;
    if (first) {
      a.cu_query_lens[r] = row;
      a.seq_lens[r] = c + n;
    }
    row += n;
    at += ((c + n + block - 1) >> a.log2_block) - ((c + block - 1) >> a.log2_block);
  }
  if (tid == 0) {
    s_first_row[a.R] = total_rows;
    if (first) {
      a.cu_query_lens[a.R] = total_rows;
      a.blocks_used[0] = total_blocks;
    }
  }
  __syncthreads();
  const int t = blockIdx.x * kStepThreads + tid;
  if (total_rows > a.T) {
    for (int r = t; r < a.R; r += gridDim.x * kStepThreads) {
      const int c = s_context[r], n = s_first_row[r + 1] - s_first_row[r];
      const int have = (c + block - 1) >> a.log2_block, need = min((c + n + block - 1) >> a.log2_block, a.width);
      const int there = min(max(a.T - s_first_row[r], 0), n);  // the request's rows that exist
      for (int i = max((c + there + block - 1) >> a.log2_block, have); i < need; ++i) {
        const int f = s_first_block[r] + i - have;
        a.tables[static_cast<int64_t>(r) * a.table_stride + i] = f < a.num_free ? a.free_blocks[f] : -1;
      }
    }
  }
  if (t >= a.T) return;
  int position = 0, slot = -1;
  if (t < total_rows) {
    int lo = 0, hi = a.R;  // the last request that begins at or before row t (empty ones before it share its offset)
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (s_first_row[mid] <= t) lo = mid; else hi = mid;
    }
    const int c = s_context[lo];
    position = c + t - s_first_row[lo];
    const int index = position >> a.log2_block;
    const int have = (c + block - 1) >> a.log2_block;
    if (index < a.width) {
      int32_t* entry = a.tables + static_cast<int64_t>(lo) * a.table_stride + index;
      int id;
      if (index < have) {
        id = *entry;
      } else {
        const int f = s_first_block[lo] + index - have;
        id = f < a.num_free ? a.free_blocks[f] : -1;
        if ((position & (block - 1)) == 0) *entry = id;
      }
      const int64_t s = (static_cast<int64_t>(id) << a.log2_block) | (position & (block - 1));
      if (id >= 0 && s <= 0x7FFFFFFF) slot = static_cast<int>(s);
    }
  }
  a.positions[t] = position;
  a.slots[t] = slot;
}

// Maximum over the LANES neighbouring lanes (8 or 16) of a row, every lane getting it.
template <int LANES>
__device__ __forceinline__ float lanes_max(float v) {
  v = fmaxf(v, dpp_f32<0xB1>(v));
  v = fmaxf(v, dpp_f32<0x4E>(v));
  v = fmaxf(v, dpp_f32<0x141>(v));
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

// One row's eight channels in a lane -> its code word and the row's meta word.  The range takes
// in zero, so z is in 0..15 and a row of one sign keeps its far end.  The scale is rounded to
// bf16 (the cache's type) before the codes are formed, so codes are right for the scale that
// readers multiply by.  A row with a NaN or infinity becomes NaN as a whole; a range beyond fp32
// is formed a sixteenth at a time; scales too small for the reciprocal take the division.
template <int LANES>
__device__ __forceinline__ uint32_t quantize_row(uint4 raw, int lane, uint32_t* meta) {
  typedef uint16_t u16x2_t __attribute__((ext_vector_type(2)));
  float x[8];
  unpack_bf16x8(raw, x);
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
  u16x2_t top = {0, 0};
#pragma unroll
  for (int i = 0; i < 4; ++i) top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2_t, w[i] & 0x7FFF7FFFu));
  const bool bad = top[0] >= 0x7F80 || top[1] >= 0x7F80;
  float hi = 0.0f, lo = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    hi = fmaxf(hi, x[i]);
    lo = fminf(lo, x[i]);
  }
  hi = lanes_max<LANES>(hi);
  lo = -lanes_max<LANES>(-lo);
  constexpr uint64_t kRow = LANES == 16 ? 0xFFFFull : 0xFFull;
  if (__ballot(bad) >> (lane & ~(LANES - 1)) & kRow) {
    *meta = 0x7FC04300u;
    return 0;
  }
  const float range = hi - lo;
  const float exact = __builtin_isinf(range) ? (hi * 0.0625f - lo * 0.0625f) / 15.0f * 16.0f : range / 15.0f;
  const float s = bf16_bits_to_f32(pack_bf16x2(exact, 0.0f) & 0xFFFFu);
  if (!(s > 0.0f)) {  // all zeros, or below the smallest scale
    *meta = 0x00004300u;
    return 0;
  }
  float t[8], z;
  if (s < 0x1p-100f || s > 0x1p100f) {
    z = rintf(-lo / s);
#pragma unroll
    for (int i = 0; i < 8; ++i) t[i] = x[i] / s;
  } else {
    const float inverse = __builtin_amdgcn_rcpf(s);
    z = rintf(near_quotient(-lo, inverse));
#pragma unroll
    for (int i = 0; i < 8; ++i) t[i] = near_quotient(x[i], inverse);
  }
  z = fminf(z, 15.0f);
  uint32_t c[8];  // the code in the low bits of 2^23 + code
#pragma unroll
  for (int i = 0; i < 8; ++i)
    c[i] = __float_as_uint(__builtin_amdgcn_fmed3f(rintf(t[i]), -z, 15.0f - z) + (z + 8388608.0f));
  *meta = kv_meta(s, static_cast<int>(z));
  const uint32_t p0 = __builtin_amdgcn_perm(c[1], c[0], 0x05040100u), p1 = __builtin_amdgcn_perm(c[3], c[2], 0x05040100u);
  const uint32_t p2 = __builtin_amdgcn_perm(c[5], c[4], 0x05040100u), p3 = __builtin_amdgcn_perm(c[7], c[6], 0x05040100u);
  return p0 | (p1 << 4) | (p2 << 8) | (p3 << 12);
}

// A wave takes 64 / (D / 8) consecutive tokens of one kv head, K and V: D / 8 lanes a row, 16
// bytes a lane.  Consecutive tokens usually follow each other in a page, where the wave's words
// are then whole lines.  Reads and writes bound it: 16384 tokens of 8 heads (85 MB) take 20.8 us,
// 4.1 TB/s of a large copy's 5.2; 61 scattered decode rows take 3.3 us, a launch.  With a division a
// code in place of near_quotient the vector instructions bound it.
template <int D>
__global__ __launch_bounds__(256) void kv_store_kernel(KvRowsArgs a) {
  constexpr int kLanes = D / 8, kTokens = 64 / kLanes;
  const int lane = threadIdx.x & 63, w = lane % kLanes;
  const int item = blockIdx.x * 4 + wave_id();
  const int head = item % a.KV;
  const int t = item / a.KV * kTokens + lane / kLanes;
  const bool live = t < a.T;
  const int slot = live ? a.slots[t] : -1;
  uint4 k = make_uint4(0, 0, 0, 0), v = k;
  if (live) {
    k = *reinterpret_cast<const uint4*>(a.k + t * a.k_stride_t + head * a.k_stride_h + w * 8);
    v = *reinterpret_cast<const uint4*>(a.v + t * a.v_stride_t + head * a.v_stride_h + w * 8);
  }
  uint32_t k_meta, v_meta;
  const uint32_t kw = quantize_row<kLanes>(k, lane, &k_meta);
  const uint32_t vw = quantize_row<kLanes>(v, lane, &v_meta);
  const int id = slot >> a.log2_block;
  if (slot < 0 || id >= a.num_blocks) return;
  const int token = slot & ((1 << a.log2_block) - 1);
  uint32_t* page = reinterpret_cast<uint32_t*>(
      a.cache + (static_cast<size_t>(id) * a.KV + head) * kv_page_bytes<D>(a.log2_block));
  const int part = kLanes << a.log2_block;  // words of the K or V codes
  page[token * kLanes + w] = kw;
  page[part + kv_v_word<D>(token, w)] = vw;
  if (w == 0) {
    page[2 * part + token] = k_meta;
    page[2 * part + (1 << a.log2_block) + token] = v_meta;
  }
}

// bf16(s (c - z)), the product exact in fp32.
__device__ __forceinline__ uint4 dequantize_row(uint32_t word, uint32_t meta) {
  const float s = kv_meta_scale(meta), z = kv_meta_zero128(meta) - 128.0f;
  float x[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = s * (static_cast<float>((word >> awq_shift(i)) & 15u) - z);
  return pack_bf16x8(x);
}

// The rows that kv_store_kernel writes, read back; a slot outside the cache gives zeros.  Writes
// bound it: 16384 tokens of 8 heads take 16 us, 5.3 TB/s.
template <int D>
__global__ __launch_bounds__(256) void kv_load_kernel(KvRowsArgs a) {
  constexpr int kLanes = D / 8, kTokens = 64 / kLanes;
  const int lane = threadIdx.x & 63, w = lane % kLanes;
  const int item = blockIdx.x * 4 + wave_id();
  const int head = item % a.KV;
  const int t = item / a.KV * kTokens + lane / kLanes;
  if (t >= a.T) return;
  const int slot = a.slots[t];
  const int id = slot >> a.log2_block;
  uint4 k = make_uint4(0, 0, 0, 0), v = k;
  if (slot >= 0 && id < a.num_blocks) {
    const int token = slot & ((1 << a.log2_block) - 1);
    const uint32_t* page = reinterpret_cast<const uint32_t*>(
        a.cache + (static_cast<size_t>(id) * a.KV + head) * kv_page_bytes<D>(a.log2_block));
    const int part = kLanes << a.log2_block;
    k = dequantize_row(page[token * kLanes + w], page[2 * part + token]);
    v = dequantize_row(page[part + kv_v_word<D>(token, w)], page[2 * part + (1 << a.log2_block) + token]);
  }
  *reinterpret_cast<uint4*>(a.k + t * a.k_stride_t + head * a.k_stride_h + w * 8) = k;
  *reinterpret_cast<uint4*>(a.v + t * a.v_stride_t + head * a.v_stride_h + w * 8) = v;
}

int rows_grid(const KvRowsArgs& a) {
  const int tokens = 512 / a.D;
  const long long items = static_cast<long long>((a.T + tokens - 1) / tokens) * a.KV;
  return static_cast<int>((items + 3) / 4);
}

}  // namespace

hipError_t launch_kv_step(const KvStepArgs& a, hipStream_t stream) {
  const int grid = a.T > 0 ? (a.T + kStepThreads - 1) / kStepThreads : 1;
  kv_step_kernel<<<grid, kStepThreads, 0, stream>>>(a);
  return hipGetLastError();
}

hipError_t launch_kv_store(const KvRowsArgs& a, hipStream_t stream) {
  if (a.D == 64)
    kv_store_kernel<64><<<rows_grid(a), 256, 0, stream>>>(a);
  else
    kv_store_kernel<128><<<rows_grid(a), 256, 0, stream>>>(a);
  return hipGetLastError();
}

hipError_t launch_kv_load(const KvRowsArgs& a, hipStream_t stream) {
  if (a.D == 64)
    kv_load_kernel<64><<<rows_grid(a), 256, 0, stream>>>(a);
  else
    kv_load_kernel<128><<<rows_grid(a), 256, 0, stream>>>(a);
  return hipGetLastError();
}

}  // namespace w4a16
