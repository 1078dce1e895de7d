// Causal attention of whole prompts over their own keys and values in bf16: packed sequences of any
// lengths, query heads sharing key heads in groups.
//
// For row t of a sequence, o = sum_j p_j v_j / sum_j p_j over j <= t with p_j = 2^(c s_j - m), s_j = q k_j
// and c = scale log2(e), in one pass over the keys with a running reference m.
#include "attention_rows.h"

namespace w4a16 {
namespace {

constexpr int kKeys = 64;        // keys of a tile
constexpr int kSetupCost = 64;   // of a row tile besides its keys
constexpr int kRing = 6;         // operand fragments in flight
constexpr int kMinShare = 3 * kKeyTileCost;
constexpr int kMaxParts = 12;
constexpr int kShortCost = kSetupCost + 12 * kKeyTileCost;

typedef __attribute__((address_space(3))) uint8_t lds_u8_t;
typedef __attribute__((address_space(3))) s16x4_t lds_s16x4_t;
typedef __attribute__((address_space(3))) bf16x8_t lds_bf16x8_t;
typedef __attribute__((address_space(3))) u32x4_t lds_u32x4_t;

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
  c.step = by_group(a, ROWS / (kKeys / kKeyTileCost) + a.group - 1);
  c.first = c.step + kSetupCost;
  if (whole) c.first = 1, c.step = 0;
  return c;
}

// Which 16-byte chunk of a row lies where: chunk c of row r is stored at c ^ swizzle(r).  Sixteen
// neighbouring rows' same chunk (the first product's operand) and four rows' same 64 bytes (the
// second's) then lie in different banks.
// A barrier and nothing else: no wait for loads on their way.
__device__ __forceinline__ void barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

template <int D>
__device__ __forceinline__ int swizzle(int row) {
  return D == 128 ? ((row & 3) << 2) | ((row >> 2) & 3) : ((row & 2) << 1) | ((row >> 2) & 3);
}

// 16 bytes a lane from base + offset to LDS at byte `to` + 16 lane.  Written as an instruction because the
// compiler, which does not know that a load's stage is not the one being read, would wait for it in front of
// every LDS read.  Its caller waits (wait_loads) before the barrier that hands the bytes over.  The wait states
// are those of a scalar register that a vector instruction wrote, and of m0.
__device__ __forceinline__ void load_to_lds(const void* base, uint32_t offset, uint32_t to) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 4\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(offset), "s"(base), "s"(to) : "memory");
}
template <int LATER>
__device__ __forceinline__ void wait_loads() {  // but for the last LATER ones; loads to LDS complete in order
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(LATER) : "memory");
}

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

template <int D, int WAVES>
__global__ __launch_bounds__(64 * WAVES, 2) void prompt_attention_kernel(PromptArgs a, KvPartials out) {
  constexpr int kPitch = 2 * D, kTileBytes = kKeys * kPitch;  // bytes
  constexpr int kRows = 32 * WAVES, kSteps = D / 16, kTiles = D / 32, kLoads = kTileBytes / WAVES / 1024;
  // Two stages of a tile of keys and one of values.
  __shared__ __align__(1024) uint8_t s_tiles[2][2][kTileBytes];
  // Queries on their way in and the output on its way out: whole rows in memory, a lane each in the products.
  // Eight waves have a part of LDS for them, four take the stage that is idle at that time.
  constexpr bool kOwnRows = kRows * kPitch > 2 * kTileBytes;
  __shared__ __align__(1024) uint8_t s_rows[kOwnRows ? kRows * kPitch : 16];
  __shared__ __align__(16) int s_bad[WAVES];
  __shared__ int s_last;

  const int tid = threadIdx.x, lane = tid & 63, wave = wave_id();
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
  const bool whole = (longest <= kShortCost) & (all_tiles <= static_cast<int>(gridDim.x));
  if (whole) {
    total = all_tiles;
    my_costs.first = 1, my_costs.step = 0;
  }
  int workers = total;
  if (!whole) workers = total > 0 ? min(static_cast<int>(gridDim.x), (total - 1) / max(kMinShare, longest / kMaxParts) + 1) : 0;
  const int per_xcd = (workers + 7) / 8, turn = static_cast<int>(blockIdx.x >> 3);
  const int me = static_cast<int>(blockIdx.x & 7) * per_xcd + turn;
  if (bad | (turn >= per_xcd) | (me >= workers)) {
    if (a.zero_tail) kv_zero_unowned(a, bad);
    return;
  }
  KvShares shares{1, 0};
  if (!whole) shares = KvShares{uniform(total / workers), uniform(total % workers)};
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
    return (kOwnRows ? rows_lds : tiles_lds + (kt & 1) * 2 * kTileBytes) + wave * 32 * kPitch;
  };
  // This lane's operands in a tile: of the keys, row col and chunk h, the others by exclusive or with 32 a
  // step of 16 channels; of the values, its four rows' 8 bytes, the others by exclusive or with 64 a step of
  // 32 channels and with 32 for the second four rows, which are 8 rows further.
  const int v_row = 4 * h + ((lane >> 2) & 3);
  const uint32_t k_read = tiles_lds + col * kPitch + (h ^ swizzle<D>(col)) * 16;
  const uint32_t v_read = tiles_lds + kTileBytes + v_row * kPitch + ((((lane >> 3) & 2) | ((lane >> 1) & 1)) ^ swizzle<D>(v_row)) * 16 + (lane & 1) * 8;
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
    const int first_row = row0 + 32 * wave;
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
      Place p = first_place(lane);
#pragma unroll
      for (int j = 0; j < 32 / kEach; ++j) {
        const uint32_t chunk = (lane % kChunks) ^ ((lane / kChunks + j * kEach) & (kChunks - 1));
        const uint32_t at = p.row <= last_row ? p.token * by_token + p.head * by_head : last;
        load_to_lds(from, at + chunk * 16, rows_at(t0 + 1) + j * 1024);
        next_place(p);
      }
    }
    // keys that this lane's row sees (none where there is no row)
    auto sees = [&]() {
      const int c = lane_again() & 31;
      return 32 * wave + c < rows ? by_group(a, first_row + c) + 1 : 0;
    };
    // keys that all rows of the wave see, and that some row may; keys that all rows of the tile see
    const int all_see = uniform(by_group(a, first_row)) + 1;
    const int any_sees = 32 * wave >= rows ? 0 : uniform(by_group(a, row0 + min(32 * wave + 32, rows) - 1)) + 1;
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
    wait_loads<0>();
    {
      const int lane = lane_again(), c = lane & 31;
      const uint32_t at = rows_at(t0 + 1) + c * kPitch + ((lane >> 5) ^ (c & (kPitch / 16 - 1))) * 16;
#pragma unroll
      for (int i = 0; i < kSteps; ++i) qf[i] = *(const lds_bf16x8_t*)static_cast<uintptr_t>(at ^ (32 * i));
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // read before the stage is another tile's

    for (int kt = t0; kt < t1; ++kt) {
      const int key0 = kt * kKeys;
      wait_loads<0>();
      barrier();
      issue_k(kt + 1);
      issue_v(kt + 1);
      const bool masked = key0 + kKeys > tile_sees;
      if (masked) look_through<kTileBytes, WAVES>(s_tiles[kt & 1][1], s_bad, wave, lane);
      if (key0 >= any_sees) {
        if (masked) {
          __syncthreads();
          clean_values<kTileBytes, WAVES>(s_tiles[kt & 1][1], s_bad, wave, lane);
        }
        continue;
      }
      const uint32_t k_at = k_read + (kt & 1) * 2 * kTileBytes, v_at = v_read + (kt & 1) * 2 * kTileBytes;
      bf16x8_t ring[kRing];
      f32x16_t sc[2];
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int i = 0; i < 16; ++i) sc[n][i] = 0.0f;
#pragma unroll
      for (int i = 0; i < kRing - 1; ++i) ring[i] = read_k(k_at, i);
#pragma unroll
      for (int i = 0; i < 2 * kSteps; ++i) {
        if (i + kRing - 1 < 2 * kSteps) ring[(i + kRing - 1) % kRing] = read_k(k_at, i + kRing - 1);
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
      if (__builtin_expect(key0 + kKeys > all_see, 0)) {
        const int lead = sees() - key0 - 4 * (lane_again() >> 5);
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const float y = sc[n][i];
            sc[n][i] = 32 * n + 8 * (i >> 2) + (i & 3) < lead ? y : -INFINITY;
          }
#pragma unroll
        for (int n = 0; n < 2; ++n) asm volatile("" : "+v"(sc[n]));
      }
      // The scores as whole accumulators on both sides of the branch's end: taken apart, they would be
      // copied on the path that masks nothing.
#pragma unroll
      for (int n = 0; n < 2; ++n) asm volatile("" : "+v"(sc[n]));
      float top = sc[0][0];
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int i = 0; i < 16; ++i) top = fmaxf(top, sc[n][i]);
      top = halves_max(top) * scale;
      // The reference follows the maximum where that leads it by more than 8: weights stay below 2^8.
      const bool grew = top - row_max > 8.0f;
      if (__any(grew)) {
        const float f = grew ? __builtin_amdgcn_exp2f(row_max - top) : 1.0f;
        row_max = grew ? top : row_max;
        row_sum *= f;
#pragma unroll
        for (int c = 0; c < kTiles; ++c)
#pragma unroll
          for (int i = 0; i < 16; ++i) acc[c][i] *= f;
      }
      const float from = row_max == -INFINITY ? 0.0f : -row_max;
      // Weights of 16 keys at a time, beside the products of the 16 before them.
      constexpr int kPv = 4 * kTiles, kPairs = 4 / kTiles;  // matrix instructions; pairs of weights beside one
      u32x4_t now, next;
      auto pair = [&](int i, u32x4_t& w) {  // weights 2 i and 2 i + 1 of a lane's 32
        float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[i >> 3][2 * (i & 7)], scale, from));
        float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[i >> 3][2 * (i & 7) + 1], scale, from));
        row_sum += p0;
        row_sum += p1;
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
        if (s < 3) {
#pragma unroll
          for (int j = 0; j < kPairs; ++j) pair(4 * (s + 1) + c * kPairs + j, next);
        }
        if (c == kTiles - 1) now = next;
      }
      if (__builtin_expect(broken, 0)) {
        const int see = sees();
        for (int key = key0; key < min(key0 + kKeys, any_sees); ++key) {
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
    bool last = true;
    if (!complete) {
      const int lane = lane_again();
      const bool live = 32 * wave + (lane & 31) < rows;
      const int first = shares.owner(u - x0), count = shares.owner(u - x0 + cost - 1) - first + 1;
      // A tile's other parts stand at the beginning of their workgroups' shares and are rarely the last to be done.
      last = x0 == 0 && kv_is_last(out.counters + first, count, &s_last);
      if (!last) {
        const int slot = 2 * me + (x0 == 0);
        const __amdgpu_buffer_rsrc_t ro = make_buffer(out.out, out.out_bytes), rs = make_buffer(out.stats, out.stats_bytes);
        if (live) {
#pragma unroll
          for (int f = 0; f < D / 8; ++f) store_fragment(ro, part_offset<D, WAVES>(slot, wave, f, lane), own[f]);
          if (lane < 32) store_stats(rs, (static_cast<uint32_t>(slot) * kRows + 32 * wave + lane) * 8, row_max, row_sum);
        }
        last = kv_arrive(out.counters + first, count, &s_last);
      } else if (tid == 0) {
        rearm(out.counters + first);
      }
      if (last) join_parts<D, WAVES>(out, first, count, me - first, wave, lane, live, row_max, row_sum, own);
    }
    if (last) {
      const float inv = row_sum == 0.0f ? 0.0f : 1.0f / row_sum;
      const int lane = lane_again(), c = lane & 31;
      const uint32_t rows_lds = rows_at(t1), at = rows_lds + c * kPitch + ((lane >> 5) ^ (c & (kPitch / 16 - 1))) * 16;
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
  wait_loads<0>();  // none may land when the workgroup's LDS is another's
  if (a.zero_tail) kv_zero_unowned(a, false);
}

template <int D, int WAVES>
hipError_t launch(const PromptArgs& a, void* workspace, int* counters, hipStream_t stream) {
  constexpr int kWorkers = kKvPromptWorkers * 8 / WAVES;
  const KvPartials part = partials_at(static_cast<char*>(workspace), counters, kWorkers, 32 * WAVES, D);
  prompt_attention_kernel<D, WAVES><<<kWorkers, 64 * WAVES, 0, stream>>>(a, part);
  return hipGetLastError();
}

}  // namespace

size_t prompt_attention_workspace(const PromptArgs& a) { return partials_bytes(kKvPromptWorkers, kKvPromptRows, a.D); }

hipError_t launch_prompt_attention(const PromptArgs& a, void* workspace, int* counters, hipStream_t stream) {
  const bool many = static_cast<int64_t>(a.T) * a.H >= 200 * 256 && a.T / 512 >= a.R;
  if (a.D == 64) return many ? launch<64, 8>(a, workspace, counters, stream) : launch<64, 4>(a, workspace, counters, stream);
  return many ? launch<128, 8>(a, workspace, counters, stream) : launch<128, 4>(a, workspace, counters, stream);
}

}  // namespace w4a16
