// Causal attention of whole prompts over their own keys and values in bf16: packed sequences of any
// lengths, query heads sharing key heads in groups.
//
// For row t of a sequence, o = sum_j p_j v_j / sum_j p_j over j <= t with p_j = 2^(c s_j - m), s_j = q k_j
// and c = scale log2(e), in one pass over the keys with a running reference m.
#include "attention_rows.h"

namespace w4a16 {
namespace {

constexpr int kThreads = 512;
constexpr int kKeys = 64;        // keys of a tile
constexpr int kSetupCost = 32;   // of a row tile besides its keys
constexpr int kMinShare = 3 * kKeyTileCost;
constexpr int kMaxParts = 12;
constexpr int kShortCost = kSetupCost + 8 * kKeyTileCost;

typedef __attribute__((address_space(3))) uint8_t lds_u8_t;
typedef __attribute__((address_space(3))) s16x4_t lds_s16x4_t;

__device__ __forceinline__ f32x16_t mfma32(bf16x8_t a, bf16x8_t b, f32x16_t c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

// One sequence, safe whatever the offsets hold.
struct Sequence {
  int row, n;  // first packed row, length
};

__device__ __forceinline__ Sequence sequence(const PromptArgs& a, int r) {
  const int lo = const_ints(a.cu_query_lens)[r], hi = const_ints(a.cu_query_lens)[r + 1];
  Sequence s;
  s.row = min(max(lo, 0), a.T);
  s.n = max(min(hi, a.T) - s.row, 0);
  return s;
}

__device__ __forceinline__ KvTileCosts tile_costs(const Sequence& s, int group, bool whole) {
  KvTileCosts c;
  c.tiles = (s.n * group + kKvPromptRows - 1) / kKvPromptRows;
  c.step = (kKvPromptRows / (kKeys / kKeyTileCost) + group - 1) / group;
  c.first = c.step + kSetupCost;
  if (whole) c.first = 1, c.step = 0;
  return c;
}

// Which 16-byte chunk of a row lies where: chunk c of row r is stored at c ^ swizzle(r).  Sixteen
// neighbouring rows' same chunk (the first product's operand) and four rows' same 64 bytes (the
// second's) then lie in different banks.
template <int D>
__device__ __forceinline__ int swizzle(int row) {
  return D == 128 ? ((row & 3) << 2) | ((row >> 2) & 3) : ((row & 2) << 1) | ((row >> 2) & 3);
}

// 16 bytes a lane from base + offset to LDS at byte `to` + 16 lane.  The LDS address is a number, so the
// compiler orders these loads with no LDS read: their caller waits for them (wait_loads) before the barrier
// that hands the bytes over.
__device__ __forceinline__ void load_to_lds(const void* base, uint32_t offset, uint32_t to) {
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(static_cast<const char*>(base) + offset),
                                   (__attribute__((address_space(3))) void*)static_cast<uintptr_t>(to), 16, 0, 0);
}
__device__ __forceinline__ void wait_loads() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

template <int D>
__global__ __launch_bounds__(kThreads, 2) void prompt_attention_kernel(PromptArgs a, KvPartials out) {
  constexpr int kPitch = 2 * D, kTileBytes = kKeys * kPitch;  // bytes
  constexpr int kSteps = D / 16, kTiles = D / 32, kLoads = D / 64;
  __shared__ __align__(1024) uint8_t s_k[2][kTileBytes];
  __shared__ __align__(1024) uint8_t s_v[2][kTileBytes];
  __shared__ __align__(16) int s_bad[8];
  __shared__ int s_last;

  const int tid = threadIdx.x, lane = tid & 63, wave = wave_id();
  const int group = a.H / a.KV;
  int sum = 0, tiles = 0, longest = 0;
  bool bad = false;
  for (int r = lane; r < a.R; r += 64) {
    bad |= kv_decreases(a, r);
    const KvTileCosts c = tile_costs(sequence(a, r), group, false);
    sum += c.before(c.tiles) * a.KV;
    tiles += c.tiles * a.KV;
    if (c.tiles > 0) longest = max(longest, c.of(c.tiles - 1));
  }
  bad = __any(bad);
  if (a.zero_tail) kv_zero_unowned(a, bad);
  int total = __builtin_amdgcn_readlane(wave_scan(sum), 63);
  const int all_tiles = __builtin_amdgcn_readlane(wave_scan(tiles), 63);
  longest = wave_max(longest);
  const bool whole = (longest <= kShortCost) & (all_tiles <= static_cast<int>(gridDim.x));
  if (whole) total = all_tiles;
  const int least = whole ? 1 : max(kMinShare, longest / kMaxParts);
  const int workers = total > 0 ? min(static_cast<int>(gridDim.x), (total - 1) / least + 1) : 0;
  const int per_xcd = (workers + 7) / 8, turn = static_cast<int>(blockIdx.x >> 3);
  const int me = static_cast<int>(blockIdx.x & 7) * per_xcd + turn;
  if (bad | (turn >= per_xcd) | (me >= workers)) return;
  const KvShares shares{uniform(total / workers), uniform(total % workers)};
  const int begin = shares.begin(me), end = shares.begin(me + 1);
  int r = 0, base = 0;
  for (;; r += 64) {
    const KvTileCosts c = tile_costs(sequence(a, min(r + lane, a.R - 1)), group, whole);
    const int cost = r + lane < a.R ? c.before(c.tiles) * a.KV : 0;
    const int upto = wave_scan(cost);
    const uint64_t past = __ballot(base + upto > begin);
    if (past || r + 64 >= a.R) {
      const int first = past ? __builtin_ctzll(past) : 0;
      base += __builtin_amdgcn_readlane(upto - cost, first);
      r += first;
      break;
    }
    base += __builtin_amdgcn_readlane(upto, 63);
  }
  r = uniform(r);
  base = uniform(base);
  Sequence q = sequence(a, r);

  const int col = lane & 31, h = lane >> 5;
  // This lane's 16 bytes of each of the wave's loads of a tile: a row, and the chunk that belongs there.
  int load_row[kLoads], load_chunk[kLoads];
#pragma unroll
  for (int j = 0; j < kLoads; ++j) {
    const int at = (wave * kLoads + j) * 1024 + lane * 16;
    load_row[j] = at / kPitch;
    load_chunk[j] = (at % kPitch / 16) ^ swizzle<D>(load_row[j]);
  }
  const uint32_t k_lds = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((lds_u8_t*)&s_k[0][0])) + wave * kLoads * 1024;
  const uint32_t v_lds = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((lds_u8_t*)&s_v[0][0])) + wave * kLoads * 1024;
  // Byte offsets of this lane's operands in a tile: of the keys, row col and chunk h, the others by exclusive
  // or with 32 a step of 16 channels; of the values, its four rows' 8 bytes, the others by exclusive or with
  // 64 a step of 32 channels and with 32 for the second four rows, whose offset is 8 rows.
  const int k_at = col * kPitch + (h ^ swizzle<D>(col)) * 16;
  const int v_row = 4 * h + ((lane >> 2) & 3);
  const int v_at = v_row * kPitch + ((((lane >> 3) & 2) | ((lane >> 1) & 1)) ^ swizzle<D>(v_row)) * 16 + (lane & 1) * 8;
  const float scale = a.scale_log2e;

  for (int u = begin; u < end;) {
    KvTileCosts costs = tile_costs(q, group, whole);
    int a_head = costs.before(costs.tiles);
    while (u >= base + a_head * a.KV) {
      base += a_head * a.KV;
      ++r;
      q = sequence(a, r);
      costs = tile_costs(q, group, whole);
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
    const int row0 = tile * kKvPromptRows, rows = min(kKvPromptRows, q.n * group - row0);
    const int key_end = uniform((row0 + rows - 1) / group) + 1;
    const int key_tiles = (key_end + kKeys - 1) / kKeys;
    // The share's part of the tile's keys, in proportion to the cost; both sides of a border
    // evaluate the same expression, exact at 0 and at the whole cost.
    const double per_unit = static_cast<double>(key_tiles);
    const int t0 = uniform(static_cast<int>(x0 * per_unit / cost)), t1 = uniform(static_cast<int>(x1 * per_unit / cost));
    const bool complete = x0 == 0 && x1 == cost;

    const uint16_t* k_base = a.k + q.row * a.k_stride_t + head * a.k_stride_h;
    const uint16_t* v_base = a.v + q.row * a.v_stride_t + head * a.v_stride_h;
    // Rows behind the sequence's last one repeat it; no row sees them.
    auto issue = [&](int kt) {
      const int key0 = kt * kKeys, buf = kt & 1;
      const void* k_tile = k_base + key0 * a.k_stride_t;
      const void* v_tile = v_base + key0 * a.v_stride_t;
#pragma unroll
      for (int j = 0; j < kLoads; ++j) {
        const uint32_t row = min(load_row[j], q.n - 1 - key0);
        load_to_lds(k_tile, row * static_cast<uint32_t>(2 * a.k_stride_t) + load_chunk[j] * 16, k_lds + buf * kTileBytes + j * 1024);
        load_to_lds(v_tile, row * static_cast<uint32_t>(2 * a.v_stride_t) + load_chunk[j] * 16, v_lds + buf * kTileBytes + j * 1024);
      }
    };

    if (t0 < t1) issue(t0);
    // The wave's 32 rows: queries as the second operand, and what they see.
    const int first_row = row0 + 32 * wave;
    const int row = first_row + col;
    const int token = row / group, qh = head * group + row - token * group;
    const bool live = 32 * wave + col < rows;
    bf16x8_t qf[kSteps];
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      uint4 w = make_uint4(0, 0, 0, 0);
      if (live)
        w = *reinterpret_cast<const uint4*>(a.q + (q.row + token) * a.q_stride_t + qh * a.q_stride_h + 16 * i + 8 * h);
      qf[i] = __builtin_bit_cast(bf16x8_t, w);
    }
    const int sees = live ? token + 1 : 0;
    // keys that all rows of the wave see, and that some row may; keys that all rows of the tile see
    const int all_see = uniform(first_row / group) + 1;
    const int any_sees = 32 * wave >= rows ? 0 : uniform((row0 + min(32 * wave + 32, rows) - 1) / group) + 1;
    const int tile_sees = uniform(row0 / group) + 1;

    f32x16_t acc[kTiles];
#pragma unroll
    for (int c = 0; c < kTiles; ++c)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[c][i] = 0.0f;
    float row_max = -INFINITY, row_sum = 0.0f;

    for (int kt = t0; kt < t1; ++kt) {
      const int buf = kt & 1, key0 = kt * kKeys;
      wait_loads();
      __syncthreads();
      if (kt + 1 < t1) issue(kt + 1);
      // A value that is no number would reach rows that do not see its key (0 * NaN in the second product).
      // Where a tile is masked, each thread makes such values of its 32 bytes zeros, and they are added to
      // the rows that see them below.
      bool broken = false;
      if (key0 + kKeys > tile_sees) {
        bool found = false;
#pragma unroll
        for (int j = 0; j < kLoads; ++j) {
          uint4* p = reinterpret_cast<uint4*>(&s_v[buf][(wave * kLoads + j) * 1024 + lane * 16]);
          const uint4 v = *p;
          uint32_t w[4] = {v.x, v.y, v.z, v.w};
          bool here = false;
#pragma unroll
          for (int i = 0; i < 4; ++i) here |= ((w[i] & 0x7F80u) == 0x7F80u) | ((w[i] & 0x7F800000u) == 0x7F800000u);
          if (here) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              if ((w[i] & 0x7F80u) == 0x7F80u) w[i] &= 0xFFFF0000u;
              if ((w[i] & 0x7F800000u) == 0x7F800000u) w[i] &= 0xFFFFu;
            }
            *p = make_uint4(w[0], w[1], w[2], w[3]);
          }
          found |= here;
        }
        found = __any(found);
        if (lane == 0) s_bad[wave] = found;
        __syncthreads();
        int any = 0;
#pragma unroll
        for (int w = 0; w < 8; ++w) any |= s_bad[w];
        broken = uniform(any) != 0;
      }
      if (key0 < any_sees) {
        f32x16_t sc[2];
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int i = 0; i < 16; ++i) sc[n][i] = 0.0f;
        const lds_u8_t* k_tile = (const lds_u8_t*)&s_k[buf][0];
        lds_u8_t* v_tile = (lds_u8_t*)&s_v[buf][0];
#pragma unroll
        for (int i = 0; i < kSteps; ++i)
#pragma unroll
          for (int n = 0; n < 2; ++n) {
            const bf16x8_t f = *reinterpret_cast<const __attribute__((address_space(3))) bf16x8_t*>(
                k_tile + ((k_at ^ (32 * i)) + 32 * n * kPitch));
            sc[n] = mfma32(f, qf[i], sc[n]);
          }
        if (key0 + kKeys > all_see) {
          const int lead = sees - key0 - 4 * h;
#pragma unroll
          for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int i = 0; i < 16; ++i) sc[n][i] = 32 * n + 8 * (i >> 2) + (i & 3) < lead ? sc[n][i] : -INFINITY;
        }
        float top = sc[0][0];
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int i = 0; i < 16; ++i) top = fmaxf(top, sc[n][i]);
        top = halves_max(top) * scale;
        // The reference follows the maximum where that leads it by more than 8: weights stay below 2^8.
        const bool grew = top > row_max && top - row_max > 8.0f;
        if (__any(grew)) {
          const float next = grew ? top : row_max, f = __builtin_amdgcn_exp2f(row_max - (next == -INFINITY ? 0.0f : next));
          row_max = next;
          row_sum *= f;
#pragma unroll
          for (int c = 0; c < kTiles; ++c)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[c][i] *= f;
        }
        const float from = row_max == -INFINITY ? 0.0f : -row_max;
#pragma unroll
        for (int s = 0; s < 4; ++s) {
          u32x4_t w;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[s >> 1][8 * (s & 1) + 2 * i], scale, from));
            const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[s >> 1][8 * (s & 1) + 2 * i + 1], scale, from));
            row_sum += p0;
            row_sum += p1;
            w[i] = pack_bf16x2(p0, p1);
          }
          const bf16x8_t pf = __builtin_bit_cast(bf16x8_t, w);
#pragma unroll
          for (int c = 0; c < kTiles; ++c) {
            const u32x2_t lo = __builtin_bit_cast(u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (lds_s16x4_t*)(v_tile + ((v_at ^ (64 * c)) + 16 * s * kPitch))));
            const u32x2_t hi = __builtin_bit_cast(u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (lds_s16x4_t*)(v_tile + ((v_at ^ (64 * c + 32)) + (16 * s + 8) * kPitch))));
            acc[c] = mfma32(__builtin_bit_cast(bf16x8_t, u32x4_t{lo[0], lo[1], hi[0], hi[1]}), pf, acc[c]);
          }
        }
        if (broken) {
          for (int key = key0; key < min(key0 + kKeys, any_sees); ++key) {
            const uint16_t* v = v_base + key * a.v_stride_t + 4 * h;
            if (key < sees) {
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
    }

    row_sum = halves_sum(row_sum);
    f32x4_t own[D / 8];
#pragma unroll
    for (int f = 0; f < D / 8; ++f)
#pragma unroll
      for (int j = 0; j < 4; ++j) own[f][j] = acc[f >> 2][4 * (f & 3) + j];
    if (complete) {
      write_rows<D>(a, live, q.row + token, qh, lane, row_sum, own);
    } else {
      const int first = shares.owner(u - x0), count = shares.owner(u - x0 + cost - 1) - first + 1;
      bool last = kv_is_last(out.counters + first, count, &s_last);
      if (!last) {
        const int slot = 2 * me + (x0 == 0);
        const __amdgpu_buffer_rsrc_t ro = make_buffer(out.out, out.out_bytes), rs = make_buffer(out.stats, out.stats_bytes);
        if (live) {
#pragma unroll
          for (int f = 0; f < D / 8; ++f) store_fragment(ro, part_offset<D>(slot, wave, f, lane), own[f]);
          if (h == 0) store_stats(rs, (static_cast<uint32_t>(slot) * kKvPromptRows + 32 * wave + col) * 8, row_max, row_sum);
        }
        last = kv_arrive(out.counters + first, count, &s_last);
      } else if (tid == 0) {
        rearm(out.counters + first);
      }
      if (last)
        join_parts<D>(a, out, first, count, me - first, wave, lane, live, q.row + token, qh, row_max, row_sum, own);
    }
    __syncthreads();  // all are done with this tile's LDS
    u += x1 - x0;
  }
}

}  // namespace

size_t prompt_attention_workspace(const PromptArgs& a) { return partials_bytes(kKvPromptWorkers, kKvPromptRows, a.D); }

hipError_t launch_prompt_attention(const PromptArgs& a, void* workspace, int* counters, hipStream_t stream) {
  const KvPartials part = partials_at(static_cast<char*>(workspace), counters, kKvPromptWorkers, kKvPromptRows, a.D);
  if (a.D == 64)
    prompt_attention_kernel<64><<<kKvPromptWorkers, kThreads, 0, stream>>>(a, part);
  else
    prompt_attention_kernel<128><<<kKvPromptWorkers, kThreads, 0, stream>>>(a, part);
  return hipGetLastError();
}

}  // namespace w4a16
