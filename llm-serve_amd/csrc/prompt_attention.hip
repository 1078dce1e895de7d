// Causal attention of whole prompts over their own keys and values in bf16: packed sequences of any
// lengths, query heads sharing key heads in groups.
//
// For row t of a sequence, o = sum_j p_j v_j / sum_j p_j over j <= t with p_j = 2^(c s_j - m), s_j = q k_j
// and c = scale log2(e), in one pass over the keys with a running reference m, which follows the largest
// c s_j where that leads it by more than 8.  All heads of a kv head share its tiles: a row tile holds the
// (token, head of the group) pairs of one kv head.
//
// Scores are formed turned over, S^T = K Q^T, in tiles of 64 keys and 32 rows a wave (v_mfma_f32_32x32x16):
// a lane then holds 32 keys' scores of one row, its maximum and sum need one exchange with the other half of
// the wave, and the weights, rounded to bf16, are in place as the second operand of O^T = V^T P^T.  V is read
// by rows and turned over by ds_read_b64_tr_b16.  Weights are rounded to bf16 because the matrix cores multiply
// bf16; their sum is of the fp32 values.  Errors of different weights average out in the quotient (0.0021 of the output
// against 64 bits, where a computation in fp32 with one rounding at the end has 0.0016), those of equal ones do not: such a
// row may be off by a rounding of bf16 besides the output's own.  Weights in two bf16 terms, with a second product
// each, give 0.0016 and cost 10 % of short prompts' time (24 of up to 120 rows 12.7 us instead of 11.6) and a
// third of long ones' (2039 rows 63 instead of 51, 16384 rows 2935 instead of 2189): not taken.
//
// Keys and values go to LDS by loads that pass no register, a tile ahead (two stages); queries and outputs
// go through LDS too, so that memory is read and written in whole rows.  A row's channels lie in LDS in an order
// of their own (swizzle), in which no read has a bank conflict.
//
// One prompt of 16384 rows, 32 + 8 heads of 128 channels (2.2 TFLOP): 2.1 to 2.25 ms, 980 to 1040 TFLOP/s.  On one box
// and in turn with it, library products of 8192 x 8192 x 8192 reach 1395 TFLOP/s and this 973, 70 % of them (of five
// boxes the library's range is 1227 to 1414).  What bounds it there is power: the core clock is 1.9 to 2.0 GHz in the
// loop, and 2.4 with zeros in place of the data (1150 TFLOP/s).  A wave needs 1024 cycles of matrix instructions for a
// tile and takes 2000 of a SIMD; loops that overlap one tile's products with another's softmax within a wave need a
// sixth fewer cycles, at a lower clock: 3 % less time, which they lose again at both ends of a row tile in prompts of
// a few thousand rows.  Nor is anything gained by waves half a tile apart, by wave priorities, or by a next row tile's
// first loads beside the present one's last tile (0 to 4 % slower).
// Short prompts are bound by a chain of latencies: 1 us to find the part, 2 for queries and first tile, 0.7 to 1.2 a
// tile, 1.2 to write.
#include <algorithm>

#include "attention_rows.h"

namespace w4a16 {
namespace {

constexpr int kKeys = 64;  // keys of a tile
// Whether a row's reference lies beyond the border from which c s is rounded as m is.  The weights' exponents c s - m
// are formed without rounding c s, and m is a rounded c s: weights are larger by half of m's last place at most, which
// is 2^-5 below the border, but 2^7 and more from scores of 2^31 on and takes the row's largest weight out of fp32.
// Looked for in one branch with references that grow: a comparison a tile, 0 to 1.5 % of a call.
__device__ __forceinline__ bool is_far(float m) { return (fabsf(m) > 0x1p20f) & (m != -INFINITY); }
// Of a row tile besides its keys: finding it, queries, output take as long as four tiles of keys (with half of
// that in the shares, nine prompts of up to 2500 rows take 313 us instead of 305).
constexpr int kSetupCost = 4 * kKeyTileCost;
// The share that workers are counted by where there is little work, and the number of parts of the longest row tile
// where there is much: joining parts costs some 3 us, and more with each.  Neither is a bound: the number of workers
// is rounded up, so that a share may be little more than half of kMinShare, and a tile that begins inside a
// share has a part more than kMaxParts.
constexpr int kMinShare = 3 * kKeyTileCost;
// Workgroups beyond two waves a SIMD work from this share on: below it more joins cost what they gain (3 prompts of up
// to 1500, 16 + 16 heads of 64, 33 us instead of 30), and a number in between leaves CUs unevenly filled (43).
constexpr int kFullShare = 12 * kKeyTileCost;
constexpr int kMaxParts = 12;
// Row tiles of up to four tiles of keys are dealt out whole, as many to each worker: no share of them saves what
// its join costs (64 prompts of up to 60 rows, 32 + 8 heads, 16.2 us instead of 23.5, 128 of up to 100 32 instead
// of 41, 32 of up to 250 29.0 instead of 33.0; with up to eight, 32 of up to 500 take 70 instead of 61).
constexpr int kWholeCost = kSetupCost + 4 * kKeyTileCost;
// Where each finds a workgroup of its own, row tiles of up to this cost are taken whole too: 700 rows of 32 + 8
// heads take 21 us in whole tiles and 28 in shares.
constexpr int kShortCost = kSetupCost + 12 * kKeyTileCost;

typedef __attribute__((address_space(3))) uint8_t lds_u8_t;
typedef __attribute__((address_space(3))) s16x4_t lds_s16x4_t;
typedef __attribute__((address_space(3))) bf16x8_t lds_bf16x8_t;
typedef __attribute__((address_space(3))) u32x4_t lds_u32x4_t;
typedef __attribute__((address_space(3))) f32x4_t lds_f32x4_t;

__device__ __forceinline__ f32x16_t mfma32(bf16x8_t a, bf16x8_t b, f32x16_t c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

// x / group, 0 <= x < 2^31.
__device__ __forceinline__ int by_group(const PromptArgs& a, int x) {
  return static_cast<int>(static_cast<uint64_t>(static_cast<uint32_t>(x)) * a.group_inverse >> a.group_shift);
}

// One sequence, safe whatever the offsets hold.
struct Sequence {
  int row, n;  // first packed row, length
  bool decreases;
};

__device__ __forceinline__ Sequence sequence(const PromptArgs& a, int r) {
  const int lo = const_ints(a.cu_query_lens)[r], hi = const_ints(a.cu_query_lens)[r + 1];
  Sequence s;
  s.row = min(max(lo, 0), a.T);
  s.n = max(min(hi, a.T) - s.row, 0);
  s.decreases = hi < lo;
  return s;
}

template <int ROWS>
__device__ __forceinline__ KvTileCosts tile_costs(const PromptArgs& a, const Sequence& s, bool whole) {
  KvTileCosts c;
  c.tiles = (s.n * a.group + ROWS - 1) / ROWS;
  c.step = by_group(a, (ROWS / (kKeys / kKeyTileCost) >> a.cost_shift) + a.group - 1);
  c.first = c.step + (kSetupCost >> a.cost_shift);
  if (whole) c.first = 1, c.step = 0;
  return c;
}

// A barrier and nothing else: no wait for loads on their way.
__device__ __forceinline__ void barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// Waves that a SIMD holds: heads of 64 channels need 128 registers a wave, of 128 channels 222.  Four waves overlap
// their products with each other's softmax, which is the longer part there: one prompt of 8000 rows of 16 + 16 heads of 64
// 163 us instead of 176 with two, 6 of up to 2500 71 instead of 80, 64 of up to 100 10.9 instead of 14.1.
template <int D>
constexpr int kWavesPerSimd = D == 64 ? 4 : 2;

// Which 16-byte chunk of a row lies where: chunk c of row r is stored at c ^ swizzle(r).  Sixteen
// neighbouring rows' same chunk (the first product's operand) and four rows' same 64 bytes (the
// second's) then lie in different banks.
template <int D>
__device__ __forceinline__ int swizzle(int row) {
  return D == 128 ? ((row & 3) << 2) | ((row >> 2) & 3) : ((row & 2) << 1) | ((row >> 2) & 3);
}

// 16 bytes a lane from base + offset to LDS at byte `to` + 16 lane.  Written as an instruction because the
// compiler, which does not know that a load's stage is not the one being read, would wait for it in front of
// every LDS read.  Its caller waits (wait_loads) before the barrier that hands the bytes over.  The wait states
// are those of a scalar register that a vector instruction wrote, and of m0.
__device__ __forceinline__ void load_to_lds(const void* base, uint32_t offset, uint32_t to) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 4\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(offset), "s"(base), "s"(to) : "m0", "memory");
}
__device__ __forceinline__ void wait_loads() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// A value that is no number would reach rows that do not see its key (0 * NaN in the second product).  Where a
// tile is masked, each wave looks through its loads' part of the values (`found` in its flag) ...
template <int BYTES, int WAVES>
__device__ __forceinline__ void look_through(const uint8_t* tile, int (&flags)[WAVES], int wave, int lane) {
  typedef uint16_t u16x2_t __attribute__((ext_vector_type(2)));
  u16x2_t top = {0, 0};
#pragma unroll
  for (int j = 0; j < BYTES / WAVES / 1024; ++j) {
    const uint4 v = *reinterpret_cast<const uint4*>(&tile[(wave * (BYTES / WAVES / 1024) + j) * 1024 + lane * 16]);
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2_t, w[i] & 0x7FFF7FFFu));
  }
  const bool found = __any((top[0] >= 0x7F80) | (top[1] >= 0x7F80));
  if (lane == 0) flags[wave] = found;
}

// ... and if any wave found one, they become zeros, and the kernel adds them to the rows that see them.  All
// threads call it, behind a barrier that follows look_through.
template <int BYTES, int WAVES>
__device__ __forceinline__ bool clean_values(uint8_t* tile, const int (&flags)[WAVES], int wave, int lane) {
  int any = 0;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) any |= flags[w];
  if (__builtin_expect(uniform(any) == 0, 1)) return false;
  for (int j = 0; j < BYTES / WAVES / 1024; ++j) {
    uint32_t* p = reinterpret_cast<uint32_t*>(&tile[(wave * (BYTES / WAVES / 1024) + j) * 1024 + lane * 16]);
    for (int i = 0; i < 4; ++i) {
      const uint32_t w = p[i];
      p[i] = ((w & 0x7F80u) == 0x7F80u ? 0 : w & 0xFFFFu) | ((w & 0x7F800000u) == 0x7F800000u ? 0 : w & 0xFFFF0000u);
    }
  }
  __syncthreads();
  return true;
}

// The lane's number, formed anew: what depends on it is then formed where it is used, and takes no registers
// in the loop, which has none to spare.
__device__ __forceinline__ int lane_again() {
  int lane = threadIdx.x & 63;
  asm volatile("" : "+v"(lane));
  return lane;
}

// WAVES waves of 32 rows each, or, with SPLIT 2, half as many rows, each with two waves that take half of every
// tile's keys and are joined in LDS.
//
// Work is dealt out by cost, not by row tile: workers (workgroups, as many as the chip holds at once) take equal
// shares of all row tiles' costs, in order, those of one XCD neighbouring ones; a row tile that a border cuts is
// joined by the last of its workers to arrive, in the workers' order, so that results do not depend on it.
template <int D, int WAVES, int SPLIT>
__global__ __launch_bounds__(64 * WAVES, kWavesPerSimd<D>) void prompt_attention_kernel(PromptArgs a, KvPartials out) {
  constexpr int kPitch = 2 * D, kTileBytes = kKeys * kPitch;  // bytes
  // Operand fragments in flight between LDS and matrix instructions; 5 or 8 make no difference that shows with 128
  // channels, 5 spill registers with 64.
  constexpr int kRing = D == 64 ? 4 : 6;
  constexpr int kRowWaves = WAVES / SPLIT, kRows = 32 * kRowWaves, kMine = kKeys / SPLIT, kSteps = D / 16, kTiles = D / 32, kLoads = kTileBytes / WAVES / 1024;
  // Two stages of a tile of keys and one of values.
  __shared__ __align__(1024) uint8_t s_tiles[2][2][kTileBytes];
  // Queries on their way in and the output on its way out: whole rows in memory, a lane each in the products.
  // Eight waves have a part of LDS for them, four take the stage that is idle at that time.
  constexpr bool kOwnRows = WAVES * 32 * kPitch > 2 * kTileBytes;
  __shared__ __align__(1024) uint8_t s_rows[kOwnRows ? WAVES * 32 * kPitch : 16];
  __shared__ float2 s_join[SPLIT > 1 ? 32 * kRowWaves : 1];
  __shared__ __align__(16) int s_bad[WAVES];
  __shared__ int s_last;

  const int tid = threadIdx.x, lane = tid & 63, wave = wave_id();
  const int row_wave = wave % kRowWaves, key_part = wave / kRowWaves;
  const int group = a.group;
  // Each lane has a sequence of the first 64; more are gone through in turn.
  const Sequence mine = sequence(a, min(lane, a.R - 1));
  KvTileCosts my_costs = tile_costs<kRows>(a, mine, false);
  bool bad = mine.decreases;
  int sum = lane < a.R ? my_costs.before(my_costs.tiles) * a.KV : 0, tiles = lane < a.R ? my_costs.tiles * a.KV : 0;
  int longest = my_costs.tiles > 0 ? my_costs.of(my_costs.tiles - 1) : 0;
  for (int r = 64 + lane; r < a.R; r += 64) {
    const Sequence s = sequence(a, r);
    bad |= s.decreases;
    const KvTileCosts c = tile_costs<kRows>(a, s, false);
    sum += c.before(c.tiles) * a.KV;
    tiles += c.tiles * a.KV;
    if (c.tiles > 0) longest = max(longest, c.of(c.tiles - 1));
  }
  bad = __any(bad);
  int total = __builtin_amdgcn_readlane(wave_scan(sum), 63);
  const int all_tiles = __builtin_amdgcn_readlane(wave_scan(tiles), 63);
  longest = wave_max(longest);
  const bool whole = (longest <= kWholeCost >> a.cost_shift) |
                     ((longest <= kShortCost >> a.cost_shift) & (all_tiles <= static_cast<int>(gridDim.x)));
  if (whole) {
    total = all_tiles;
    my_costs.first = 1, my_costs.step = 0;
  }
  int workers = min(total, static_cast<int>(gridDim.x));
  if (!whole) {
    workers = total > 0 ? min(workers, (total - 1) / max(kMinShare >> a.cost_shift, longest / kMaxParts) + 1) : 0;
    if (D == 64 && total / (kFullShare >> a.cost_shift) < static_cast<int>(gridDim.x)) workers = min(workers, static_cast<int>(gridDim.x / 2));
  }
  const int per_xcd = (workers + 7) / 8, turn = static_cast<int>(blockIdx.x >> 3);
  const int me = static_cast<int>(blockIdx.x & 7) * per_xcd + turn;
  if (bad | (turn >= per_xcd) | (me >= workers)) {
    if (a.zero_tail) kv_zero_unowned(a, bad);
    return;
  }
  const KvShares shares{uniform(total / workers), uniform(total % workers)};
  const int begin = shares.begin(me), end = shares.begin(me + 1);
  // The sequence that the share begins in, and the units before it.
  int r = 0, base = 0;
  Sequence q;
  int cost_here = lane < a.R ? my_costs.before(my_costs.tiles) * a.KV : 0;
  Sequence here = mine;
  for (;; r += 64) {
    if (r > 0) {
      here = sequence(a, min(r + lane, a.R - 1));
      const KvTileCosts c = tile_costs<kRows>(a, here, whole);
      cost_here = r + lane < a.R ? c.before(c.tiles) * a.KV : 0;
    }
    const int upto = wave_scan(cost_here);
    const uint64_t past = __ballot(base + upto > begin);
    if (past || r + 64 >= a.R) {
      const int first = past ? __builtin_ctzll(past) : 0;
      base += __builtin_amdgcn_readlane(upto - cost_here, first);
      q.row = __builtin_amdgcn_readlane(here.row, first);
      q.n = __builtin_amdgcn_readlane(here.n, first);
      r += first;
      break;
    }
    base += __builtin_amdgcn_readlane(upto, 63);
  }
  r = uniform(r);
  base = uniform(base);

  const int col = lane & 31, h = lane >> 5;
  const uint32_t tiles_lds = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((lds_u8_t*)&s_tiles[0][0][0]));
  const uint32_t k_lds = tiles_lds + wave * kLoads * 1024, v_lds = k_lds + kTileBytes;
  auto rows_at = [&](int kt) {  // of this wave, where tile kt's stage is idle
    const uint32_t rows_lds = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((lds_u8_t*)&s_rows[0]));
    return (kOwnRows ? rows_lds : tiles_lds + (kt & 1) * 2 * kTileBytes) + row_wave * 32 * kPitch;
  };
  // This lane's operands in a tile: of the keys, row col and chunk h, the others by exclusive or with 32 a
  // step of 16 channels; of the values, its four rows' 8 bytes, the others by exclusive or with 64 a step of
  // 32 channels and with 32 for the second four rows, which are 8 rows further.
  const int v_row = 4 * h + ((lane >> 2) & 3);
  const uint32_t k_read = tiles_lds + (key_part * kMine + col) * kPitch + (h ^ swizzle<D>(col)) * 16;
  const uint32_t v_read = tiles_lds + kTileBytes + (key_part * kMine + v_row) * kPitch + ((((lane >> 3) & 2) | ((lane >> 1) & 1)) ^ swizzle<D>(v_row)) * 16 + (lane & 1) * 8;
  const float scale = a.scale_log2e;

  for (int u = begin; u < end;) {
    KvTileCosts costs = tile_costs<kRows>(a, q, whole);
    int a_head = costs.before(costs.tiles);
    while (u >= base + a_head * a.KV) {
      base += a_head * a.KV;
      ++r;
      q = sequence(a, r);
      costs = tile_costs<kRows>(a, q, whole);
      a_head = costs.before(costs.tiles);
    }
    const int head = uniform((u - base) / a_head);
    const int x = u - base - head * a_head;
    int tile = 0, over = costs.tiles;  // the last tile that begins at or before x
    while (over - tile > 1) {
      const int mid = (tile + over) >> 1;
      if (costs.before(mid) <= x) tile = mid; else over = mid;
    }
    const int cost = costs.of(tile), x0 = x - costs.before(tile);
    const int x1 = min(cost, x0 + end - u);
    const int row0 = tile * kRows, rows = min(kRows, q.n * group - row0);
    const int key_end = uniform(by_group(a, row0 + rows - 1)) + 1;
    const int key_tiles = (key_end + kKeys - 1) / kKeys;
    // The share's part of the tile's keys, in proportion to the cost; both sides of a border
    // evaluate the same expression, which is below the tiles' number below the whole cost.
    const bool complete = x0 == 0 && x1 == cost;
    int t0 = 0, t1 = key_tiles;
    if (!complete) {
      const double per_unit = key_tiles * __builtin_amdgcn_rcp(static_cast<double>(cost));
      t0 = uniform(static_cast<int>(x0 * per_unit));
      if (x1 < cost) t1 = uniform(static_cast<int>(x1 * per_unit));
    }

    const uint16_t* k_base = a.k + q.row * a.k_stride_t + head * a.k_stride_h;
    const uint16_t* v_base = a.v + q.row * a.v_stride_t + head * a.v_stride_h;
    // The loads of tile kt.  Rows behind the sequence's last one repeat it; no row sees them.
    auto issue = [&](const uint16_t* rows_base, int64_t stride, uint32_t lds, int kt) {
      const int key0 = kt * kKeys, last = q.n - 1 - key0, lane = lane_again();
      const void* first = rows_base + key0 * stride;
      const uint32_t to = lds + (kt & 1) * 2 * kTileBytes;
#pragma unroll
      for (int j = 0; j < kLoads; ++j) {
        const int row = (wave * kLoads + j) * (1024 / kPitch) + lane / (kPitch / 16);
        const uint32_t chunk = (lane % (kPitch / 16)) ^ swizzle<D>(row);
        load_to_lds(first, min(row, last) * static_cast<uint32_t>(2 * stride) + chunk * 16, to + j * 1024);
      }
    };
    auto issue_k = [&](int kt) { if (kt < t1) issue(k_base, a.k_stride_t, k_lds, kt); };
    auto issue_v = [&](int kt) { if (kt < t1) issue(v_base, a.v_stride_t, v_lds, kt); };

    issue_k(t0);
    issue_v(t0);
    // The wave's 32 rows: queries as the second operand, and what they see.
    const int first_row = row0 + 32 * row_wave;
    // The wave's rows as whole memory rows: a lane's 16 bytes of row j kEach + lane / (chunks of a row), and where
    // that row lies, a token and a head of the group, from the tile's first token and head on.
    constexpr int kEach = 1024 / kPitch, kChunks = kPitch / 16;
    const int token0 = uniform(by_group(a, row0)), last_row = row0 + rows - 1;
    const int skip = uniform(by_group(a, kEach)), skip_heads = kEach - skip * group;
    struct Place {
      int row, token, head;
    };
    auto first_place = [&](int lane) {
      const int row = first_row + lane / kChunks, token = by_group(a, row);
      return Place{row, token - token0, row - token * group};
    };
    auto next_place = [&](Place& p) {
      p.row += kEach;
      p.token += skip;
      p.head += skip_heads;
      if (p.head >= group) p.head -= group, ++p.token;
    };
    {
      const uint32_t by_token = 2 * a.q_stride_t, by_head = 2 * a.q_stride_h;
      const uint16_t* from = a.q + (q.row + token0) * a.q_stride_t + head * group * a.q_stride_h;
      const int last_token = by_group(a, last_row);
      const uint32_t last = (last_token - token0) * by_token + (last_row - last_token * group) * by_head;
      const int lane = lane_again();
      constexpr int kMyRows = 32 / SPLIT;  // two waves of the same rows load half of them each
      Place p = first_place(lane + key_part * (kMyRows * kChunks));
#pragma unroll
      for (int j = 0; j < kMyRows / kEach; ++j) {
        const uint32_t chunk = (lane % kChunks) ^ ((key_part * kMyRows + lane / kChunks + j * kEach) & (kChunks - 1));
        const uint32_t at = p.row <= last_row ? p.token * by_token + p.head * by_head : last;
        load_to_lds(from, at + chunk * 16, rows_at(t0 + 1) + (key_part * (kMyRows / kEach) + j) * 1024);
        next_place(p);
      }
    }
    // keys that this lane's row sees (none where there is no row)
    auto sees = [&]() {
      const int c = lane_again() & 31;
      return 32 * row_wave + c < rows ? by_group(a, first_row + c) + 1 : 0;
    };
    // keys that all rows of the wave see, and that some row may; keys that all rows of the tile see
    const int all_see = uniform(by_group(a, first_row)) + 1;
    const int any_sees = 32 * row_wave >= rows ? 0 : uniform(by_group(a, row0 + min(32 * row_wave + 32, rows) - 1)) + 1;
    const int tile_sees = uniform(by_group(a, row0)) + 1;


    f32x16_t acc[kTiles];
#pragma unroll
    for (int c = 0; c < kTiles; ++c)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[c][i] = 0.0f;
    float row_max = -INFINITY, row_sum = 0.0f;

    // Fragments of a tile: of its keys, number i (half i / kSteps of the keys, step i % kSteps of 16 channels);
    // of its values, step i / kTiles of 16 keys, channels 32 (i % kTiles) ..
    auto read_k = [&](uint32_t at, int i) {
      return *(const lds_bf16x8_t*)static_cast<uintptr_t>((at ^ (32 * (i % kSteps))) + 32 * (i / kSteps) * kPitch);
    };
    auto read_v = [&](uint32_t at, int i) {
      const int s = i / kTiles, c = i % kTiles;
      const u32x2_t lo = __builtin_bit_cast(u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          (lds_s16x4_t*)static_cast<uintptr_t>((at ^ (64 * c)) + 16 * s * kPitch)));
      const u32x2_t hi = __builtin_bit_cast(u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          (lds_s16x4_t*)static_cast<uintptr_t>((at ^ (64 * c + 32)) + (16 * s + 8) * kPitch)));
      return __builtin_bit_cast(bf16x8_t, u32x4_t{lo[0], lo[1], hi[0], hi[1]});
    };

    bf16x8_t qf[kSteps];
    wait_loads();
    if (SPLIT > 1) barrier();
    {
      const int lane = lane_again(), c = lane & 31;
      const uint32_t at = rows_at(t0 + 1) + c * kPitch + ((lane >> 5) ^ (c & (kPitch / 16 - 1))) * 16;
#pragma unroll
      for (int i = 0; i < kSteps; ++i) qf[i] = *(const lds_bf16x8_t*)static_cast<uintptr_t>(at ^ (32 * i));
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // read before the stage is another tile's

    for (int kt = t0; kt < t1; ++kt) {
      const int key0 = kt * kKeys;
      wait_loads();
      barrier();
      issue_k(kt + 1);
      issue_v(kt + 1);
      const bool masked = key0 + kKeys > tile_sees;
      if (masked) look_through<kTileBytes, WAVES>(s_tiles[kt & 1][1], s_bad, wave, lane);
      const int my_key0 = key0 + key_part * kMine;
      if (my_key0 >= any_sees) {
        if (masked) {
          __syncthreads();
          clean_values<kTileBytes, WAVES>(s_tiles[kt & 1][1], s_bad, wave, lane);
        }
        continue;
      }
      const uint32_t k_at = k_read + (kt & 1) * 2 * kTileBytes, v_at = v_read + (kt & 1) * 2 * kTileBytes;
      bf16x8_t ring[kRing];
      constexpr int kHalves = kMine / 32;
      f32x16_t sc[kHalves];
#pragma unroll
      for (int n = 0; n < kHalves; ++n)
#pragma unroll
        for (int i = 0; i < 16; ++i) sc[n][i] = 0.0f;
#pragma unroll
      for (int i = 0; i < kRing - 1; ++i) ring[i] = read_k(k_at, i);
#pragma unroll
      for (int i = 0; i < kHalves * kSteps; ++i) {
        if (i + kRing - 1 < kHalves * kSteps) ring[(i + kRing - 1) % kRing] = read_k(k_at, i + kRing - 1);
        __builtin_amdgcn_sched_barrier(0);
        sc[i / kSteps] = mfma32(ring[i % kRing], qf[i % kSteps], sc[i / kSteps]);
      }
      bool broken = false;
      if (masked) {
        __syncthreads();
        broken = clean_values<kTileBytes, WAVES>(s_tiles[kt & 1][1], s_bad, wave, lane);
      }
      // the values' first fragments are read beside the softmax
#pragma unroll
      for (int i = 0; i < kRing - 1; ++i) ring[i] = read_v(v_at, i);
      __builtin_amdgcn_sched_barrier(0);
      if (__builtin_expect(my_key0 + kMine > all_see, 0)) {
        const int lead = sees() - my_key0 - 4 * (lane_again() >> 5);
#pragma unroll
        for (int n = 0; n < kHalves; ++n)
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const float y = sc[n][i];
            sc[n][i] = 32 * n + 8 * (i >> 2) + (i & 3) < lead ? y : -INFINITY;
          }
#pragma unroll
        for (int n = 0; n < kHalves; ++n) asm volatile("" : "+v"(sc[n]));
      }
      // The scores as whole accumulators on both sides of the branch's end: taken apart, they would be
      // copied on the path that masks nothing.
#pragma unroll
      for (int n = 0; n < kHalves; ++n) asm volatile("" : "+v"(sc[n]));
      float top = sc[0][0];
#pragma unroll
      for (int n = 0; n < kHalves; ++n)
#pragma unroll
        for (int i = 0; i < 16; ++i) top = fmaxf(top, sc[n][i]);
      top = halves_max(top) * scale;
      // The reference follows the maximum where that leads it by more than 8: weights stay below 2^8.
      const bool grew = top - row_max > 8.0f;
      bool far = false;
      if (__any(grew | is_far(row_max))) {
        const float f = grew ? __builtin_amdgcn_exp2f(row_max - top) : 1.0f;
        row_max = grew ? top : row_max;
        row_sum *= f;
#pragma unroll
        for (int c = 0; c < kTiles; ++c)
#pragma unroll
          for (int i = 0; i < 16; ++i) acc[c][i] *= f;
        far = __any(is_far(row_max));
        if (__builtin_expect(far, 0)) {  // the exponents themselves, of each row as its own reference asks
          if (is_far(row_max)) {
#pragma unroll
            for (int n = 0; n < kHalves; ++n)
#pragma unroll
              for (int i = 0; i < 16; ++i) sc[n][i] *= scale;
#pragma unroll
            for (int n = 0; n < kHalves; ++n) asm volatile("" : "+v"(sc[n]));
#pragma unroll
            for (int n = 0; n < kHalves; ++n)
#pragma unroll
              for (int i = 0; i < 16; ++i) sc[n][i] -= row_max;
          } else {
            const float from = row_max == -INFINITY ? 0.0f : -row_max;
#pragma unroll
            for (int n = 0; n < kHalves; ++n)
#pragma unroll
              for (int i = 0; i < 16; ++i) sc[n][i] = __builtin_fmaf(sc[n][i], scale, from);
          }
#pragma unroll
          for (int n = 0; n < kHalves; ++n) asm volatile("" : "+v"(sc[n]));
        }
#pragma unroll
        for (int n = 0; n < kHalves; ++n) asm volatile("" : "+v"(sc[n]));
      }
#pragma unroll
      for (int n = 0; n < kHalves; ++n) asm volatile("" : "+v"(sc[n]));
      const float factor = far ? 1.0f : scale, from = (far | (row_max == -INFINITY)) ? 0.0f : -row_max;
      // Weights of 16 keys at a time, beside the products of the 16 before them.
      constexpr int kPv = 2 * kHalves * kTiles, kPairs = 4 / kTiles;  // matrix instructions; pairs of weights beside one
      u32x4_t now, next;
      // Summed for the tile first: single weights added to the sum of all tiles would all be rounded at its last
      // place, equal ones the same way (350000 rows of weights of 0.7 were off by 0.0026).
      float tile_sum = 0.0f;
      auto pair = [&](int i, u32x4_t& w) {  // weights 2 i and 2 i + 1 of a lane's 32
        float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[i >> 3][2 * (i & 7)], factor, from));
        float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[i >> 3][2 * (i & 7) + 1], factor, from));
        tile_sum += p0;
        tile_sum += p1;
        w[i & 3] = pack_bf16x2(p0, p1);
      };
#pragma unroll
      for (int i = 0; i < 4; ++i) pair(i, now);
#pragma unroll
      for (int i = 0; i < kPv; ++i) {
        const int s = i / kTiles, c = i % kTiles;
        if (i + kRing - 1 < kPv) ring[(i + kRing - 1) % kRing] = read_v(v_at, i + kRing - 1);
        __builtin_amdgcn_sched_barrier(0);
        acc[c] = mfma32(ring[i % kRing], __builtin_bit_cast(bf16x8_t, now), acc[c]);
        __builtin_amdgcn_sched_barrier(0);
        if (s < 2 * kHalves - 1) {
#pragma unroll
          for (int j = 0; j < kPairs; ++j) pair(4 * (s + 1) + c * kPairs + j, next);
        }
        if (c == kTiles - 1) now = next;
      }
      row_sum += tile_sum;
      if (__builtin_expect(broken, 0)) {
        const int see = sees();
        for (int key = my_key0; key < min(my_key0 + kMine, any_sees); ++key) {
          const uint16_t* v = v_base + key * a.v_stride_t + 4 * h;
          if (key < see) {
#pragma unroll
            for (int c = 0; c < kTiles; ++c)
#pragma unroll
              for (int i = 0; i < 16; ++i) {
                const uint32_t bits = v[32 * c + 8 * (i >> 2) + (i & 3)];
                if ((bits & 0x7F80u) == 0x7F80u) acc[c][i] += bf16_bits_to_f32(bits);
              }
          }
        }
      }
    }

    row_sum = halves_sum(row_sum);
    f32x4_t own[D / 8];
#pragma unroll
    for (int f = 0; f < D / 8; ++f)
#pragma unroll
      for (int j = 0; j < 4; ++j) own[f][j] = acc[f >> 2][4 * (f & 3) + j];
    if (SPLIT > 1) {  // the waves of the tiles' second half hand over what they have, through the idle stage
      const uint32_t at = tiles_lds + (t1 & 1) * 2 * kTileBytes + row_wave * 64 * kPitch + lane_again() * 16;
      const int of_row = 32 * row_wave + (lane_again() & 31);
      if (key_part) {
#pragma unroll
        for (int f = 0; f < D / 8; ++f) *(lds_f32x4_t*)static_cast<uintptr_t>(at + f * 1024) = own[f];
        s_join[of_row] = make_float2(row_max, row_sum);
      }
      __syncthreads();
      if (!key_part) {
        const float2 with = s_join[of_row];
        const float top = fmaxf(row_max, with.x), ref = top == -INFINITY ? 0.0f : top;
        const float x = __builtin_amdgcn_exp2f(row_max - ref), y = __builtin_amdgcn_exp2f(with.x - ref);
        row_sum = scaled(row_sum, row_max - ref) + scaled(with.y, with.x - ref);
        row_max = top;
#pragma unroll
        for (int f = 0; f < D / 8; ++f) own[f] = own[f] * x + *(const lds_f32x4_t*)static_cast<uintptr_t>(at + f * 1024) * y;
      }
    }
    bool last = true;
    if (!complete) {
      const int lane = lane_again();
      const bool live = key_part == 0 && 32 * row_wave + (lane & 31) < rows;
      const int first = shares.owner(u - x0), count = shares.owner(u - x0 + cost - 1) - first + 1;
      // A tile's other parts stand at the beginning of their workgroups' shares and are rarely the last to be done.
      last = x0 == 0 && kv_is_last(out.counters + first, count, &s_last);
      if (!last) {
        const int slot = 2 * me + (x0 == 0);
        const __amdgpu_buffer_rsrc_t ro = make_buffer(out.out, out.out_bytes), rs = make_buffer(out.stats, out.stats_bytes);
        if (live) {
#pragma unroll
          for (int f = 0; f < D / 8; ++f) store_fragment(ro, part_offset<D, kRowWaves>(slot, row_wave, f, lane), own[f]);
          if (lane < 32) store_stats(rs, (static_cast<uint32_t>(slot) * kRows + 32 * row_wave + lane) * 8, row_max, row_sum);
        }
        last = kv_arrive(out.counters + first, count, &s_last);
      } else if (tid == 0) {
        rearm(out.counters + first);
      }
      if (last) join_parts<D, kRowWaves>(out, first, count, me - first, row_wave, lane, live, row_max, row_sum, own);
    }
    if (last && key_part == 0) {
      const float inv = row_sum == 0.0f ? 0.0f : 1.0f / row_sum;
      const int lane = lane_again(), c = lane & 31;
      const uint32_t rows_lds = rows_at(t1) + row_wave * (SPLIT - 1) * 32 * kPitch, at = rows_lds + c * kPitch + ((lane >> 5) ^ (c & (kPitch / 16 - 1))) * 16;
#pragma unroll
      for (int f = 0; f < D / 8; f += 2) *(lds_u32x4_t*)static_cast<uintptr_t>(at ^ (16 * f)) = row_pair(inv, own[f], own[f + 1]);
      char* to = reinterpret_cast<char*>(a.out + (static_cast<int64_t>(q.row + token0) * a.H + head * group) * D);
      Place p = first_place(lane);
#pragma unroll
      for (int j = 0; j < 32 / kEach; ++j) {
        const u32x4_t w = *(const lds_u32x4_t*)static_cast<uintptr_t>(rows_lds + j * 1024 + lane * 16);
        const uint32_t chunk = (lane % kChunks) ^ ((lane / kChunks + j * kEach) & (kChunks - 1));
        if (p.row <= last_row) *reinterpret_cast<u32x4_t*>(to + (static_cast<uint32_t>(p.token * a.H + p.head) * kPitch + chunk * 16)) = w;
        next_place(p);
      }
    }
    __syncthreads();  // all are done with this tile's LDS
    u += x1 - x0;
  }
  wait_loads();  // none may land when the workgroup's LDS is another's
  if (a.zero_tail) kv_zero_unowned(a, false);
}

// Workgroups of a form: row tiles of 256 rows have eight waves, others four.
constexpr int workers(int D, int tile_rows) {
  return 256 * 4 * (D == 64 ? kWavesPerSimd<64> : kWavesPerSimd<128>) / (tile_rows == 256 ? 8 : 4);
}

template <int D, int WAVES, int SPLIT>
hipError_t launch(const PromptArgs& a, void* workspace, int* counters, hipStream_t stream) {
  constexpr int kWorkers = workers(D, 32 * WAVES / SPLIT);
  static_assert(kWorkers == 256 * 4 * kWavesPerSimd<D> / WAVES, "as many workgroups as the chip holds");
  const KvPartials part = partials_at(static_cast<char*>(workspace), counters, a.part_workers, 32 * WAVES / SPLIT, D);
  prompt_attention_kernel<D, WAVES, SPLIT><<<kWorkers, 64 * WAVES, 0, stream>>>(a, part);
  return hipGetLastError();
}

template <int D>
hipError_t launch_for(const PromptArgs& a, void* workspace, int* counters, hipStream_t stream) {
  switch (a.tile_rows) {
    case 64: return launch<D, 4, 2>(a, workspace, counters, stream);
    case 128: return launch<D, 4, 1>(a, workspace, counters, stream);
    default: return launch<D, 8, 1>(a, workspace, counters, stream);
  }
}

// The most row tiles of n rows that a call may have, what the longest of them may cost, and what all may.  With
// rows / n = y, sequences have at most y + R tiles together, tile j of each costs first + step j (tile_costs), and the
// sum of all j is largest, below (y + 1) y / 2, where one sequence has all rows; x is y rounded down.
struct MostWork {
  int64_t tiles, longest, total;
};
MostWork most_work(const PromptArgs& a, int n, int shift) {
  const int64_t group = a.H / a.KV, rows = a.T * group, x = rows / n;
  const int64_t step = ((n / (kKeys / kKeyTileCost) >> shift) + group - 1) / group, first = step + (kSetupCost >> shift);
  const int64_t tiles = x + (a.R < rows ? a.R : rows);
  return {a.KV * tiles, first + step * x, a.KV * (tiles * first + step * ((x + 1) * (x + 2) / 2))};
}

// The most workers that a call may have where row tiles are cut, by the kernel's own rule; 0 where none can be.
int part_workers(const PromptArgs& a, const MostWork& most) {
  const int grid = workers(a.D, a.tile_rows);
  if (most.longest <= kWholeCost >> a.cost_shift || (most.longest <= kShortCost >> a.cost_shift && most.tiles <= grid)) return 0;
  const int64_t n = (most.total - 1) / (kMinShare >> a.cost_shift) + 1;
  return n < grid ? static_cast<int>(n) : grid;
}

// While row tiles of 64 find a CU each, the longest of them is what takes time: with its keys split between
// two waves, one prompt of 511 rows (32 + 8 heads of 128) takes 14.4 us instead of 16.5, one of 700 rows of 16
// heads of 64 12.6 instead of 14.9.  With more tiles than CUs it loses (four prompts of up to 250 rows 12.8
// instead of 11.7), and with many requests (128 of 4 rows 20 instead of 18).
//
// Of the others, long prompts take eight waves: a tile of keys and values is loaded for twice the rows (16384
// rows 2118 us instead of 2348, 2039 rows 49 instead of 52).  Four waves, two workgroups a CU, waste less on
// short row tiles and have more of them (24 prompts of up to 120 rows 13 us instead of 23, 128 of up to 100 43
// instead of 48, 32 of up to 200 in 16 heads of 64 19 instead of 22); about 500 rows a request are the border.
//
// (T counts rows of no request too and R empty places, so that a request's mean length may be larger than T / R.)
constexpr int kSplitRows = 256 * 64, kSplitTiles = 256, kLongRows = 200 * 256;
int tile_rows(const PromptArgs& a) {
  const int64_t rows = static_cast<int64_t>(a.T) * a.H;
  if (rows <= kSplitRows && static_cast<int64_t>(a.R) * a.KV <= kSplitTiles) return 64;
  return rows >= kLongRows && a.T / 512 >= a.R ? 256 : 128;
}

}  // namespace

// The kernel counts work in 32 bits.  A step of many requests may be one long prompt and empty places, which the
// host cannot tell from their number: where its work might pass 32 bits, it takes the form with fewer row tiles, and
// units of up to a whole tile of keys (shares of so many are even whatever the unit).  262144 rows of 64 + 8 heads,
// one prompt, count 2.155e9 sixteenths of a tile of keys.
bool plan_prompt_attention(PromptArgs* a) {
  constexpr int64_t kMost = 0x7FFFFFFF;
  static_assert(kKeyTileCost == 16, "a tile of keys in units of cost_shift 4 is one");
  a->tile_rows = tile_rows(*a), a->cost_shift = 0;
  MostWork most = most_work(*a, a->tile_rows, 0);
  if (most.total > kMost) {
    if (a->T > kPromptStepRows) return false;
    a->tile_rows = 256;
    while ((most = most_work(*a, 256, a->cost_shift)).total > kMost)
      if (++a->cost_shift > 4) return false;
  }
  a->part_workers = part_workers(*a, most);
  return true;
}

// The most that a call of these sizes or of fewer rows or requests needs, in any form that one of them takes.
// (Never nothing: zero bytes would read as a refusal.)
size_t prompt_attention_workspace(const PromptArgs& a) {
  size_t most = 256;
  const auto form = [&](int n, int T, int R) {
    PromptArgs b = a;
    b.T = T, b.R = R, b.tile_rows = n, b.cost_shift = 0;
    if (const int workers = part_workers(b, most_work(b, n, 0))) most = std::max(most, partials_bytes(workers, n, b.D));
  };
  const int64_t rows = static_cast<int64_t>(a.T) * a.H, tiles = static_cast<int64_t>(a.R) * a.KV;
  form(64, std::min(a.T, kSplitRows / a.H), std::min(a.R, kSplitTiles / a.KV));
  if (rows > kSplitRows || tiles > kSplitTiles) form(128, a.T, a.R);
  if (rows >= kLongRows) form(256, a.T, a.R);
  return most;
}

hipError_t launch_prompt_attention(const PromptArgs& a, void* workspace, int* counters, hipStream_t stream) {
  return a.D == 64 ? launch_for<64>(a, workspace, counters, stream) : launch_for<128>(a, workspace, counters, stream);
}

}  // namespace w4a16
