// Attention over the 4-bit paged cache.
//
// For a row q of a kv head and its visible keys t,
//   S_t = scale s_k (q . (c_k - z_k)),  P = softmax(S),  out = sum_t P_t s_v (c_v - z_v).
// Codes and zero points enter the matrix instructions as they are: (128 + c) is an exact bf16
// value (kv4_common.h), and
//   q . (c - z)          = q . (128 + c) - (128 + z) sum(q)
//   sum P' (c - z)       = sum P' (128 + c) - sum P' (128 + z),   P' = P s_v,
// so no code is ever scaled: the key's offset is the accumulator's initial value and its scale
// one multiplication a score, and the values' offset is one more matrix tile whose operand is
// the meta words' low halves.  Scores, statistics and sums are fp32; the one rounding is P' to
// the sum of two bf16 values (16 bits), the codes' operand type, each with a matrix instruction of
// its own: outputs are then as far from 64 bits as their own rounding, 0.0017.  One bf16 value gave
// 0.0020 and took 131 us instead of 134 for 128 sequences of up to 8192 keys; fp16's range does not
// hold P s_v.
#include "kv4_attention.h"

namespace w4a16 {
namespace {

constexpr int kUnit = 128;      // keys of one work unit: 32 a wave
constexpr int kWaves = 4;
constexpr int kRows = 16;       // rows of a tile
constexpr int kThreads = 64 * kWaves;

// Units of one row tile (a tile whose rows see nothing still has its zeros to write).
__device__ __forceinline__ int kv_span(const KvRequest& q) { return max((q.keys + kUnit - 1) / kUnit, 1); }

// Units of a request (none if the prompt kernel takes it).
__device__ __forceinline__ int kv_units(const KvAttentionArgs& a, const KvRequest& q, int group) {
  if (q.n * group > a.split_rows) return 0;
  return (q.n * group + kRows - 1) / kRows * a.KV * kv_span(q);
}

// One slice of 32 keys of a wave, in registers: two 16-key tiles, each inside one page.
template <int D>
struct KvSlice {
  uint32_t k[2][D / 32];        // K words of key lane % 16: D / 4 channels from (D / 4) (lane / 16)
  uint32_t v[2][4];             // one V word of four keys 4 (lane / 16) ..
  uint32_t km[2][4], vm[2][4];  // those keys' meta words
};

// Where a slice's tiles are: a descriptor of each tile's page (wave-uniform), and its first token.
struct KvPlace {
  __amdgpu_buffer_rsrc_t page[2];
  int token[2];
  bool ok[2];  // the page is in the cache (else the first page's rows are read, and masked)
};

// Lane offsets into a page, in bytes.
struct KvLane {
  uint32_t k, v, meta;
};

template <int D>
__device__ __forceinline__ KvPlace kv_place(const KvAttentionArgs& a, const int (&id)[2], int head, int key) {
  KvPlace p;
  const uint32_t bytes = static_cast<uint32_t>(kv_page_bytes<D>(a.log2_block));
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    p.ok[t] = static_cast<unsigned>(id[t]) < static_cast<unsigned>(a.num_blocks);
    p.token[t] = (key + 16 * t) & ((1 << a.log2_block) - 1);
    const uint32_t index = static_cast<uint32_t>((p.ok[t] ? id[t] : 0) * a.KV + head);
    p.page[t] = make_buffer(a.cache + static_cast<uint64_t>(index) * bytes, bytes);
  }
  return p;
}

template <int D>
__device__ __forceinline__ void load_keys(KvSlice<D>& s, const KvPlace& p, const KvLane& o, int log2_block) {
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    if constexpr (D == 128) {
      const u32x4_t w = __builtin_bit_cast(u32x4_t, __builtin_amdgcn_raw_buffer_load_b128(p.page[t], o.k, p.token[t] * (D / 2), 0));
#pragma unroll
      for (int i = 0; i < 4; ++i) s.k[t][i] = w[i];
    } else {
      const u32x2_t w = __builtin_bit_cast(u32x2_t, __builtin_amdgcn_raw_buffer_load_b64(p.page[t], o.k, p.token[t] * (D / 2), 0));
      s.k[t][0] = w[0], s.k[t][1] = w[1];
    }
    const u32x4_t m = __builtin_bit_cast(
        u32x4_t, __builtin_amdgcn_raw_buffer_load_b128(p.page[t], o.meta, (D << log2_block) + p.token[t] * 4, 0));
#pragma unroll
    for (int i = 0; i < 4; ++i) s.km[t][i] = m[i];
  }
}

template <int D>
__device__ __forceinline__ void load_values(KvSlice<D>& s, const KvPlace& p, const KvLane& o, int log2_block) {
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const u32x4_t w = __builtin_bit_cast(
        u32x4_t, __builtin_amdgcn_raw_buffer_load_b128(p.page[t], o.v, ((D / 2) << log2_block) + p.token[t] * (D / 2), 0));
    const u32x4_t m = __builtin_bit_cast(
        u32x4_t, __builtin_amdgcn_raw_buffer_load_b128(p.page[t], o.meta, ((D + 4) << log2_block) + p.token[t] * 4, 0));
#pragma unroll
    for (int i = 0; i < 4; ++i) s.v[t][i] = w[i], s.vm[t][i] = m[i];
  }
}

// The page ids of the tiles at key and key + 16; keys behind the last one repeat its page.
__device__ __forceinline__ void kv_ids(int (&id)[2], ConstInts table, int key, int last, int log2_block) {
#pragma unroll
  for (int t = 0; t < 2; ++t)
    id[t] = table[min(key + 16 * t, last) >> log2_block];
}

// Split attention.  A row tile is up to 16 rows (tokens x heads of the group) of one request
// and kv head; its keys are cut into units of 128.  All units of all tiles, in order, are dealt
// to the grid's workgroups in equal contiguous shares, so that a batch of any lengths loads them
// alike; a share that covers a tile's keys only in part leaves a partial result (KvPartials).
// Inside a unit each of the 4 waves takes 32 keys and keeps its own running maximum and sum; the
// waves are joined through LDS at the end of a tile.  More rows than 16 take several tiles, which
// read the keys again, mostly from L2: 24 requests of 8 drafts (32 rows) took 24 us so when weights
// were one operand (24.6 with two), and 26 us with 32 rows a tile, whose registers leave room for two
// waves a SIMD.
//
// The next slice's keys are loaded into the registers that the scores have just consumed, and
// its values into those that the second product has, so a wave has loads in flight throughout
// without a second set of registers, and three waves fit a SIMD.  A fourth would cost spills
// inside the loop: 128 sequences of up to 8192 keys took 255 us with four, 149 us with three.
//
// 128 sequences of up to 8192 keys take 133 us, 4.6 TB/s of the cache's bytes (a large copy:
// 5.1 to 5.2 TB/s); 2 of 131000 take 62 us.  Short calls are bound by latency: some 4 us to the first
// keys, 2 us to join and write, and a tail of a few us between the first and the last workgroup.
template <int D>
__global__ __launch_bounds__(kThreads, 3) void kv_attention_kernel(KvAttentionArgs a, KvPartials out) {
  constexpr int kSteps = D / 32, kTiles = D / 16, kPitch = D + 4;
  __shared__ __align__(16) float s_out[kWaves][kRows][kPitch];
  __shared__ float s_max[kWaves][kRows], s_sum[kWaves][kRows];
  __shared__ int s_last;

  const int tid = threadIdx.x, lane = tid & 63, wave = wave_id();
  const int group = a.H / a.KV;

  // This workgroup's share.  Every wave sums the requests' units (64 requests at a time, a lane
  // each), then scans them to the request where the share begins.
  const bool few = a.R <= 64;
  KvRequest mine{0, 0, 0, 0};
  int my_units = 0, sum = 0;
  bool bad = false;
  for (int i = lane; i < a.R; i += 64) {
    bad |= kv_decreases(a, i);
    mine = kv_request(a, i);
    my_units = kv_units(a, mine, group);
    sum += my_units;
  }
  int upto = wave_scan(sum);
  const int total = __builtin_amdgcn_readlane(upto, 63);
  const int workers = min(total, static_cast<int>(gridDim.x));
  const int me = blockIdx.x;

  bad = __any(bad);
  if (a.zero_tail) kv_zero_unowned(a, bad);
  if (bad | (me >= workers)) return;
  const KvShares shares{total / workers, total % workers};
  const int begin = shares.begin(me), end = shares.begin(me + 1);
  int r = 0, base = 0, units;  // the share's first request, the units before it, and its own
  KvRequest q;
  if (few) {
    r = __builtin_ctzll(__ballot(upto > begin));
    base = __builtin_amdgcn_readlane(upto - my_units, r);
    units = __builtin_amdgcn_readlane(my_units, r);
    q = KvRequest{__builtin_amdgcn_readlane(mine.row, r), __builtin_amdgcn_readlane(mine.n, r),
                  __builtin_amdgcn_readlane(mine.cached, r), __builtin_amdgcn_readlane(mine.keys, r)};
  } else {
    for (;; r += 64) {
      my_units = r + lane < a.R ? kv_units(a, kv_request(a, r + lane), group) : 0;
      upto = wave_scan(my_units);
      const uint64_t past = __ballot(base + upto > begin);
      if (past || r + 64 >= a.R) {
        const int first = past ? __builtin_ctzll(past) : 0;
        base += __builtin_amdgcn_readlane(upto - my_units, first);
        r += first;
        break;
      }
      base += __builtin_amdgcn_readlane(upto, 63);
    }
    q = kv_request(a, r);
    units = kv_units(a, q, group);
  }

  const NibbleConsts nc = nibble_consts();
  const int col = lane & 15, g = lane >> 4;
  const float scale = a.scale_log2e;
  const KvLane offset{static_cast<uint32_t>(col * (D / 2) + g * (D / 8)),
                      static_cast<uint32_t>((g * (D / 8) + col % (D / 8)) * 16), static_cast<uint32_t>(g * 16)};

  for (int u = begin; u < end;) {
    while (u >= base + units) {
      base += units;
      ++r;
      q = kv_request(a, r);
      units = kv_units(a, q, group);
    }
    const int tiles = (q.n * group + kRows - 1) / kRows, span = kv_span(q);
    const int seg = (u - base) / span, k0 = u - base - seg * span;
    const int head = seg / tiles, tile = seg - head * tiles;
    const int n = min(span - k0, end - u);
    const int row0 = tile * kRows, rows = min(kRows, q.n * group - row0);
    const ConstInts table = const_ints(a.tables + static_cast<int64_t>(r) * a.table_stride);

    const int key_end = min((k0 + n) * kUnit, q.keys);
    int key = k0 * kUnit + 32 * wave;
    KvSlice<D> s;
    KvPlace place;
    int id[2];
    if (key < key_end) {
      kv_ids(id, table, key, key_end - 1, a.log2_block);
      place = kv_place<D>(a, id, head, key);
      load_keys<D>(s, place, offset, a.log2_block);
      load_values<D>(s, place, offset, a.log2_block);
      if (key + kUnit < key_end) kv_ids(id, table, key + kUnit, key_end - 1, a.log2_block);
    }

    // The queries as the second operand: column = row of the tile, channels as K's words have them.
    bf16x8_t qf[kSteps];
    const int row = row0 + col;
    const int token = row / group, h = head * group + row - token * group;
    const bool live = col < rows;
    float total_q = 0.0f;
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      uint4 w = make_uint4(0, 0, 0, 0);
      if (live)
        w = *reinterpret_cast<const uint4*>(a.q + (q.row + token) * a.q_stride_t + h * a.q_stride_h + (D / 4) * g +
                                            8 * i);
      float f[8];
      unpack_bf16x8(w, f);
#pragma unroll
      for (int j = 0; j < 8; ++j) total_q += f[j];
      qf[i] = __builtin_bit_cast(bf16x8_t, w);
    }
    const float neg_sum = -column_sum(total_q);
    const bool tree = a.tree_mask != nullptr;
    // Leading keys that the lane's row sees, and which of the request's new ones behind them.
    const uint64_t bits = tree && live ? a.tree_mask[q.row + token] : 0;
    const int sees = live ? min(tree ? q.cached : q.cached + token + 1, q.keys) : 0;
    const int all_see = min(a.tree_mask ? q.cached : q.cached + row0 / group + 1, q.keys);

    f32x4_t acc_o[kTiles], acc_z = {0, 0, 0, 0};
    float row_max = -INFINITY, row_sum = 0.0f;
#pragma unroll
    for (int c = 0; c < kTiles; ++c) acc_o[c] = f32x4_t{0, 0, 0, 0};

    // A SIMD issues its oldest wave first, so of equal shares the first workgroup's on a CU would end
    // a quarter sooner than the third's (96 against 126 us of 128 sequences up to 8192 keys).  The
    // waves take turns in priority instead.
    int turn = static_cast<int>(blockIdx.x >> 8) % 3;
    for (; key < key_end; key += kUnit) {
      if (turn == 0) {
        __builtin_amdgcn_s_setprio(0);
      } else if (turn == 1) {
        __builtin_amdgcn_s_setprio(1);
      } else {
        __builtin_amdgcn_s_setprio(2);
      }
      turn = turn == 2 ? 0 : turn + 1;
      const bool more = key + kUnit < key_end;
      const bool whole = key + 32 <= all_see && place.ok[0] && place.ok[1];
      const bool ok[2] = {place.ok[0], place.ok[1]};

      f32x4_t sc[2];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
#pragma unroll
        for (int i = 0; i < 4; ++i) sc[t][i] = kv_meta_zero128(s.km[t][i]) * neg_sum;
#pragma unroll
        for (int i = 0; i < kSteps; ++i) sc[t] = mfma16(unpack_codes(s.k[t][i], nc), qf[i], sc[t]);
#pragma unroll
        for (int i = 0; i < 4; ++i) sc[t][i] *= kv_meta_scale(s.km[t][i]);
      }
      if (more) {
        place = kv_place<D>(a, id, head, key + kUnit);
        load_keys<D>(s, place, offset, a.log2_block);
        if (key + 2 * kUnit < key_end) kv_ids(id, table, key + 2 * kUnit, key_end - 1, a.log2_block);
      }

      float vs[2][4];  // the values' scales as the rows see them
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) vs[t][i] = kv_meta_scale(s.vm[t][i]);
      if (!whole) {
        // A lane's keys are 16 t + 4 g + i.  Keys outside the sequence, or on no page, hold
        // anything: their score becomes -inf, their scale 0 and their zero point 0.  Keys that
        // only this row does not see keep their zero point (the offset tile's operand serves
        // all rows), and their scale is taken as 0 for this row.
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int k = key + 16 * t + 4 * g + i;
            // selections, not branches, one scalar at a time
            const bool held = ok[t] & (k < q.keys);
            const unsigned fresh = static_cast<unsigned>(k - q.cached);
            s.vm[t][i] = held ? s.vm[t][i] : 0x00004300u;
            const uint32_t word = fresh & 32u ? static_cast<uint32_t>(bits >> 32) : static_cast<uint32_t>(bits);
            const uint32_t named = fresh < 64u ? word >> (fresh & 31u) : 0u;
            const bool visible = held & ((k < sees) | ((named & 1u) != 0));
            const float x = sc[t][i];
            sc[t][i] = visible ? x : -INFINITY;
            vs[t][i] = visible ? vs[t][i] : 0.0f;
          }
      }
      u32x4_t zf;  // the keys' 128 + z as the first operand of the offset tile
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 2; ++i)
          zf[2 * t + i] = __builtin_amdgcn_perm(s.vm[t][2 * i + 1], s.vm[t][2 * i], 0x05040100u);
      const float mx = fmaxf(fmaxf(fmaxf(sc[0][0], sc[0][1]), fmaxf(sc[0][2], sc[0][3])),
                             fmaxf(fmaxf(sc[1][0], sc[1][1]), fmaxf(sc[1][2], sc[1][3])));
      const float top = fmaxf(row_max, column_max(mx));
      if (__any(top > row_max)) {
        const float ref = top == -INFINITY ? 0.0f : top;
        const float f = __builtin_amdgcn_exp2f((row_max - ref) * scale);
        row_max = top;
        row_sum *= f;
#pragma unroll
        for (int c = 0; c < kTiles; ++c)
#pragma unroll
          for (int i = 0; i < 4; ++i) acc_o[c][i] *= f;
#pragma unroll
        for (int i = 0; i < 4; ++i) acc_z[i] *= f;
      }
      const float ref = (row_max == -INFINITY ? 0.0f : row_max) * scale;
      u32x4_t w, rest;
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        float p[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          p[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[t][i], scale, -ref));
          row_sum += p[i];
          p[i] *= vs[t][i];
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint32_t high = pack_bf16x2(p[2 * i], p[2 * i + 1]);
          w[2 * t + i] = high;
          rest[2 * t + i] =
              pack_bf16x2(p[2 * i] - __uint_as_float(high << 16), p[2 * i + 1] - __uint_as_float(high & 0xFFFF0000u));
        }
      }
      const bf16x8_t pf = __builtin_bit_cast(bf16x8_t, w), pr = __builtin_bit_cast(bf16x8_t, rest);
      acc_z = mfma16(__builtin_bit_cast(bf16x8_t, zf), pf, acc_z);
      acc_z = mfma16(__builtin_bit_cast(bf16x8_t, zf), pr, acc_z);

      // V: words of tokens paired into halves with 4 channels each (even ones, then odd ones);
      // nibble i of the halves is one channel of two tokens.  A 64-channel row has 8 words, and
      // lanes 8 .. 15 of a row of 16 take the same words' odd channels.
#pragma unroll
      for (int half = 0; half < (D == 128 ? 2 : 1); ++half) {
        uint32_t pair[4];
        const uint32_t select = (D == 128 ? half != 0 : (col & 8) != 0) ? 0x07060302u : 0x05040100u;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int i = 0; i < 2; ++i)
            pair[2 * t + i] = __builtin_amdgcn_perm(s.v[t][2 * i + 1], s.v[t][2 * i], select);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          u32x4_t f;
#pragma unroll
          for (int i = 0; i < 4; ++i) f[i] = ((pair[i] >> (4 * c)) & nc.mask) | nc.bias;
          const int ch = D == 128 ? 2 * c + half : c;
          acc_o[ch] = mfma16(__builtin_bit_cast(bf16x8_t, f), pf, acc_o[ch]);
          acc_o[ch] = mfma16(__builtin_bit_cast(bf16x8_t, f), pr, acc_o[ch]);
        }
      }
      if (more) load_values<D>(s, place, offset, a.log2_block);
    }

    // Join the waves.  Accumulator register i of a lane is operand row 4 g + i: the word (D =
    // 128) or word and half (D = 64) whose channels the tiles c count.
    const float row_total = column_sum(row_sum);
    if (g == 0) {
      s_max[wave][col] = row_max;
      s_sum[wave][col] = row_total;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float* o = s_out[wave][col];
      if constexpr (D == 128) {
#pragma unroll
        for (int c = 0; c < 8; c += 4) {
          const f32x4_t v = {acc_o[c][i] - acc_z[i], acc_o[c + 1][i] - acc_z[i],
                             acc_o[c + 2][i] - acc_z[i], acc_o[c + 3][i] - acc_z[i]};
          *reinterpret_cast<f32x4_t*>(o + 8 * (4 * g + i) + c) = v;
        }
      } else {
        const int word = (4 * g + i) & 7, odd = g >> 1;
#pragma unroll
        for (int c = 0; c < 4; ++c) o[8 * word + 2 * c + odd] = acc_o[c][i] - acc_z[i];
      }
    }
    __syncthreads();
    const bool complete = k0 == 0 && n == span;
    const uint32_t slot = 2 * me + (k0 == 0);
    const __amdgpu_buffer_rsrc_t ro = make_buffer(out.out, out.out_bytes), rs = make_buffer(out.stats, out.stats_bytes);
    constexpr int kChunks = D / 8;
    for (int e = tid; e < rows * kChunks; e += kThreads) {
      const int row = e / kChunks, ch = e % kChunks * 8;
      float high = s_max[0][row];
#pragma unroll
      for (int w = 1; w < kWaves; ++w) high = fmaxf(high, s_max[w][row]);
      const float ref = high == -INFINITY ? 0.0f : high;
      float all = 0.0f, o[8] = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        const float f = __builtin_amdgcn_exp2f((s_max[w][row] - ref) * scale);
        all += f * s_sum[w][row];
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i] += f * s_out[w][row][ch + i];
      }
      if (complete) {
        const int token = (row0 + row) / group;
        kv_write(a, q.row + token, head * group + row0 + row - token * group, ch, all, o);
      } else {
        const uint32_t at = slot * kRows + row;
        store_part(ro, (at * D + ch) * 4, o);
        if (ch == 0) store_stats(rs, at * 8, high, all);
      }
    }
    if (!complete) {
      const int first = shares.owner(u - k0), count = shares.owner(u - k0 + span - 1) - first + 1;
      if (kv_arrive(out.counters + first, count, &s_last))
        kv_join<D, kThreads>(a, out, kRows, first, count, q, head, row0, rows, &s_out[0][0][0]);
    }
    u += n;
    if (u < end) __syncthreads();
  }
}

// Kernels and grids of a call, by sizes alone (lengths are on the device, and every choice is
// right for any).  Requests of at most split_rows rows (tokens x heads of a group) go to the
// split kernel, longer ones to the prompt kernel, which is launched only if the longest query
// may be that long.
struct KvPlan {
  int split_workers;   // the split kernel's grid (0: not launched)
  int split_rows;
  int prompt_workers;  // the prompt kernel's grid (0: not launched)
};

KvPlan kv_plan(const KvAttentionArgs& a) {
  KvPlan p;
  const int64_t longest = static_cast<int64_t>(a.max_query_len) * (a.H / a.KV);
  const bool prompts = longest > kKvSplitMaxRows;
  const bool alone = prompts && a.R == 1;  // a prompt by itself: one launch
  p.split_rows = alone ? 0 : prompts ? kKvSplitMaxRows : 0x7FFFFFFF;
  const int64_t tiles = ((prompts ? kKvSplitMaxRows : longest) + kRows - 1) / kRows;
  const int64_t units = ((static_cast<int64_t>(a.width) << a.log2_block) + kUnit - 1) / kUnit;
  const int64_t most = tiles * a.R * a.KV * (units > 0 ? units : 1);
  p.split_workers = alone ? 0 : static_cast<int>(most < kKvSplitWorkers ? most : kKvSplitWorkers);
  p.prompt_workers = prompts ? kKvPromptWorkers : 0;
  return p;
}

size_t align256(size_t n) { return (n + 255) / 256 * 256; }

// A kernel's part of the workspace: partial results of 2 tiles of `rows` rows a worker.
size_t partials_bytes(int workers, int rows, int D) {
  const size_t n = static_cast<size_t>(2) * workers * rows;
  return align256(n * D * sizeof(float)) + align256(n * 2 * sizeof(float));
}

KvPartials partials_at(char* ws, int* counters, int workers, int rows, int D) {
  const size_t n = static_cast<size_t>(2) * workers * rows;
  KvPartials part;
  part.out = reinterpret_cast<float*>(ws);
  part.stats = reinterpret_cast<float*>(ws + align256(n * D * sizeof(float)));
  part.out_bytes = static_cast<uint32_t>(n * D * sizeof(float));
  part.stats_bytes = static_cast<uint32_t>(n * 2 * sizeof(float));
  part.counters = counters;
  return part;
}

template <int D>
hipError_t launch(const KvAttentionArgs& a, const KvPlan& p, char* ws, int* counters, hipStream_t stream) {
  const KvPartials split = partials_at(ws, counters, p.split_workers, kRows, D);
  if (p.split_workers) {
    kv_attention_kernel<D><<<p.split_workers, kThreads, 0, stream>>>(a, split);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || p.prompt_workers == 0) return e;
  }
  const KvPartials prompt = partials_at(ws + partials_bytes(p.split_workers, kRows, D), counters + kKvSplitWorkers,
                                        p.prompt_workers, kKvPromptRows, D);
  return launch_kv_prompt(a, prompt, p.prompt_workers, stream);
}

}  // namespace

size_t kv_attention_workspace(const KvAttentionArgs& a) {
  const KvPlan p = kv_plan(a);
  return partials_bytes(p.split_workers, kRows, a.D) +
         (p.prompt_workers ? partials_bytes(p.prompt_workers, kKvPromptRows, a.D) : 0);
}

hipError_t launch_kv_attention(const KvAttentionArgs& args, void* workspace, int* counters, hipStream_t stream) {
  const KvPlan p = kv_plan(args);
  KvAttentionArgs a = args;
  a.split_rows = p.split_rows;
  char* ws = static_cast<char*>(workspace);
  return a.D == 64 ? launch<64>(a, p, ws, counters, stream) : launch<128>(a, p, ws, counters, stream);
}

}  // namespace w4a16
