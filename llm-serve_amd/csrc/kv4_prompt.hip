// Attention of long queries over the 4-bit paged cache: prompts, and chunks of them.
//
// The same mathematics as kv4_attention.hip in the shape of a matrix kernel.  A workgroup takes
// 256 rows (tokens x heads of a kv head's group) of a request, 32 a wave, and walks their keys in
// tiles of 64.  Eight waves would each have to unpack the same codes, and unpacking costs more
// vector instructions than the softmax, so a tile is dequantized once for all of them: the first
// four waves turn the K codes of the next tile into rows in LDS while the other four turn the V
// codes into columns, into the buffer that is not being read.
//
// Operands are fp16, whose 11 bits hold s (c - z) to half a unit in 2^-11: an error an eighth of
// bf16's, below the output's rounding.  (As bf16, keys and values moved outputs by 0.0036 of 64-bit
// ones against 0.0017 for the rounding alone; codes as exact bf16 128 + c and scales applied to
// scores and weights took 20 % longer, and lost as much in long sums of 128 P.)  fp16's range is
// met by powers of two: one out of each 16 keys' scales and each row of queries.  Those of keys and
// queries join the softmax's scale in the exponent's multiplier, those of values are its addend.  The 16
// keys share it whether a row sees them or not.
//
// Scores are formed transposed, S^T = K Q^T, so that a lane holds 16 keys' scores of one row in
// the accumulator layout, and P^T is the second product's operand as it stands: its 16 contraction
// slots 8 h + j of a lane half h are the keys 16 s + 4 h + j (j < 4) and 16 s + 8 + 4 h + j - 4,
// and V's columns are written in that order.  The output is O^T = V^T P^T: every statistic of a
// row sits in the two lanes that hold it.
//
// What bounds it: a tile of 64 keys costs a SIMD (two waves) some 2000 cycles of matrix
// instructions and 3000 of vector instructions (softmax, conversion).  The two waves are in the same
// phase, every tile ends in a barrier, and little of it overlaps: for 4096 rows behind 12288 cached
// tokens (1.00 to 1.03 ms, 935 to 960 TFLOP/s; a large matrix product of the library reaches 1250 to
// 1266) matrix instructions fill 41 % of the cycles and vector instructions 61 %.  A row tile costs 4 to
// 5 us besides its keys (queries, the first keys, writing or joining), which is what short prompts pay:
// 2039 tokens take 59 to 62 us, 550 to 580 TFLOP/s.  Workgroups take equal shares of the cost of all row tiles,
// so a share may end inside a tile's keys; tiles as units would leave a causal prompt's last rows to
// few workgroups.  Measured and not taken, with bf16 operands: a conversion interleaved with the same
// wave's first product (4096 rows 3 % faster, 2039 rows 3 % slower: both converters' loops are then
// apart, twice the code to fetch), and with it waves half a tile apart over three value buffers
// (registers spill; 5 and 20 % slower).
#include "attention_rows.h"

namespace w4a16 {
namespace {

typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));

constexpr int kPromptThreads = 512;
constexpr int kKeys = 64;      // keys of a tile
constexpr int kTileCost = kKeyTileCost;
constexpr int kSetupCost = 32;  // of a row tile besides its keys
// Shares.  A part costs some 5 us besides its keys (set-up, its way through memory, its turn in the
// join), so shares are no smaller than 3 key tiles and a row tile has at most some 12 parts: 40
// tokens x 5 heads behind 2172 take 32 us (8 key tiles at least: 42), 20 x 4 behind 12000 46 us (as
// many parts as workgroups: 56).  Where no row tile has more than 8 key tiles and there is a
// workgroup for each, they are not split: 2 x 34 tokens x 8 heads 16 us (27 split), 400 x 4 23 (29).
// The bound on parts was measured at those two contexts and costs more behind longer ones, where the
// join is small beside a part's keys: 20 x 4 take 85 us behind 32000 and 262 behind 131000 (the split
// kernel 44 and 131, see kKvSplitMaxRows).
constexpr int kMinShare = 3 * kTileCost;
constexpr int kMaxParts = 12;
constexpr int kShortCost = kSetupCost + 8 * kTileCost;
constexpr uint32_t kZeroMeta = 0x00004300u, kNanMeta = 0x7FC04300u;  // rows of zeros, of NaN

// Exponents.  fp16 has the codes' products with a scale to 11 bits, but not bf16's range, so a power
// of two is taken out of each group of 16 keys' scales (the largest is brought to 2^10 .. 2^11) and of
// each row of queries (2^14 .. 2^15), as fields of fp32 exponents.  What lies 2^-24 below its group's
// largest loses bits: it is that much smaller in the sums.  Fields are held in range: groups whose
// scales are all below 2^-63 keep that exponent and lose bits below 2^-87.
constexpr int kGroupFactor = 264, kRowFactor = 268;

// A weight carries its values' power of two, 2^(field - 137), and the sum of weights takes it out
// again.  Beside values of a very large power, the weights of keys with small ones, or with zeros, would
// leave fp32's range below although they are large by themselves.  So once a workgroup has met a field
// above this border (scales of 2^15 and more, which are rare), it forms sums of weights without that
// power, an exponential more a score.  Below the border fields lie between 64 and 142, and a weight that
// is lost, 133 powers under the reference's maximum, is 2^-55 of the row's largest at most.
constexpr int kLargeField = 142;

__device__ __forceinline__ f32x16_t mfma32(f16x8_t a, f16x8_t b, f32x16_t c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}

__device__ __forceinline__ KvTileCosts kv_costs(const KvAttentionArgs& a, const KvRequest& q, int group, bool whole) {
  KvTileCosts c;
  const int rows = q.n * group;
  c.tiles = rows > a.split_rows ? (rows + kKvPromptRows - 1) / kKvPromptRows : 0;
  c.step = a.tree_mask ? 0 : (kKvPromptRows / 4 + group - 1) / group;
  c.first = min(a.tree_mask ? q.keys : max(q.cached, 0), q.keys) / (kKeys / kTileCost) + c.step + kSetupCost;
  if (whole) c.first = 1, c.step = 0;
  return c;
}

__device__ __forceinline__ uint32_t pack_f16x2(float x, float y) {
  return __builtin_bit_cast(uint32_t, f16x2_t{static_cast<_Float16>(x), static_cast<_Float16>(y)});
}

// 2^(field - 127).
__device__ __forceinline__ float power(int field) { return __uint_as_float(static_cast<uint32_t>(field) << 23); }

// Nibbles of a pair of keys or channels -> fp16 (c - z) s, rounded once: 1024 + c is exact with c in an
// fp16's low bits, and so is the difference from 1024 + z.
__device__ __forceinline__ uint32_t pair_value(uint32_t biased, uint32_t zero, uint32_t scale) {
  return __builtin_bit_cast(uint32_t, (__builtin_bit_cast(f16x2_t, biased) - __builtin_bit_cast(f16x2_t, zero)) *
                                          __builtin_bit_cast(f16x2_t, scale));
}

// The masks in SGPRs and the biases in VGPRs, hidden from constant folding, so that each and-or is
// one v_and_or_b32 (see NibbleConsts).  In bits 4 .. 7 of an fp16 64.0 a nibble is 64 + c.
struct HalfConsts {
  uint32_t mask_low, mask_high, bias_low, bias_high;
};

__device__ __forceinline__ HalfConsts half_consts() {
  HalfConsts k{0x000F000Fu, 0x00F000F0u, 0x64006400u, 0x54005400u};
  asm volatile("" : "+s"(k.mask_low), "+s"(k.mask_high));
  asm volatile("" : "+v"(k.bias_low), "+v"(k.bias_high));
  return k;
}

// The largest of a wave's values where four neighbouring lanes have the same.
__device__ __forceinline__ uint32_t group_max(uint32_t v) {
  v = max(v, static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(v), 0x124, 0xF, 0xF, true)));
  v = max(v, static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(v), 0x128, 0xF, 0xF, true)));
  const u32x2_t a = __builtin_bit_cast(u32x2_t, __builtin_amdgcn_permlane16_swap(v, v, false, false));
  v = max(a[0], a[1]);
  const u32x2_t b = __builtin_bit_cast(u32x2_t, __builtin_amdgcn_permlane32_swap(v, v, false, false));
  return max(b[0], b[1]);
}

// The exponent field of a group, from the bits of its largest scale.
__device__ __forceinline__ int group_field(uint32_t top) { return min(max(static_cast<int>(top >> 23), 64), 254); }

template <int D>
__global__ __launch_bounds__(kPromptThreads, 2) void kv_prompt_kernel(KvAttentionArgs a, KvPartials out) {
  constexpr int kPitchK = D + 8, kPitchV = kKeys + 8;  // fp16 elements; 16-byte reads of 16 lanes meet all banks
  constexpr int kSteps = D / 16, kTiles = D / 32;
  __shared__ __align__(16) uint16_t s_k[2][kKeys][kPitchK];
  __shared__ __align__(16) uint16_t s_v[2][D][kPitchV];
  // A group of 16 keys: what a raw score is multiplied by, the values' power of two, and what takes it out
  // of a sum of weights (0: these sums are formed without it).
  __shared__ __align__(16) float s_score[2][4], s_log[2][4], s_part[2][4];
  __shared__ int s_last;
  __shared__ uint64_t s_held[2][4];  // 4 bits a key: whether it is in the sequence and on a page

  const int tid = threadIdx.x, lane = tid & 63, wave = wave_id();
  const int group = a.H / a.KV;
  int sum = 0, tiles = 0;
  int longest = 0;
  bool bad = false;
  for (int r = lane; r < a.R; r += 64) {
    bad |= kv_decreases(a, r);
    const KvTileCosts c = kv_costs(a, kv_request(a, r), group, false);
    sum += c.before(c.tiles) * a.KV;
    tiles += c.tiles * a.KV;
    if (c.tiles > 0) longest = max(longest, c.of(c.tiles - 1));
  }
  bad = __any(bad);
  if (a.split_rows == 0 && a.zero_tail) kv_zero_unowned(a, bad);  // no split kernel in this call
  int total = __builtin_amdgcn_readlane(wave_scan(sum), 63);
  const int all_tiles = __builtin_amdgcn_readlane(wave_scan(tiles), 63);
  // Short tiles go to a workgroup each, if there are enough: parts of them would wait for each other.
  longest = wave_max(longest);
  const bool whole = (longest <= kShortCost) & (all_tiles <= static_cast<int>(gridDim.x));
  if (whole) total = all_tiles;
  const int least = whole ? 1 : max(kMinShare, longest / kMaxParts);
  const int workers = total > 0 ? min(static_cast<int>(gridDim.x), (total - 1) / least + 1) : 0;
  // Workers of one XCD (workgroups go to the 8 XCDs in turn) take neighbouring shares, mostly of
  // the same kv heads, whose pages then stay in that XCD's L2.
  const int per_xcd = (workers + 7) / 8, turn = static_cast<int>(blockIdx.x >> 3);
  const int me = static_cast<int>(blockIdx.x & 7) * per_xcd + turn;
  if (bad | (turn >= per_xcd) | (me >= workers)) return;
  const KvShares shares{uniform(total / workers), uniform(total % workers)};
  const int begin = shares.begin(me), end = shares.begin(me + 1);
  int r = 0, base = 0;
  for (;; r += 64) {
    const KvTileCosts c = kv_costs(a, kv_request(a, min(r + lane, a.R - 1)), group, whole);
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
  KvRequest q = kv_request(a, r);

  const HalfConsts hc = half_consts();
  const int col = lane & 31, h = lane >> 5;
  const float scale = a.scale_log2e;
  bool large = false;  // a converter of values has met a field above the border

  for (int u = begin; u < end;) {
    KvTileCosts costs = kv_costs(a, q, group, whole);
    int a_head = costs.before(costs.tiles);
    while (u >= base + a_head * a.KV) {
      base += a_head * a.KV;
      ++r;
      q = kv_request(a, r);
      costs = kv_costs(a, q, group, whole);
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
    const int key_end = a.tree_mask ? q.keys : max(min(q.cached + uniform((row0 + rows - 1) / group) + 1, q.keys), 0);
    const int key_tiles = (key_end + kKeys - 1) / kKeys;
    // The share's part of the tile's keys, in proportion to the cost; both sides of a border
    // evaluate the same expression, exact at 0 and at the whole cost.
    const double per_unit = static_cast<double>(key_tiles);
    const int t0 = uniform(static_cast<int>(x0 * per_unit / cost)), t1 = uniform(static_cast<int>(x1 * per_unit / cost));
    const bool complete = x0 == 0 && x1 == cost;
    const ConstInts table = const_ints(a.tables + static_cast<int64_t>(r) * a.table_stride);

    // This thread's part of a key tile.  K (waves 0 .. 3): D / 4 channels of one key.  V (waves 4
    // .. 7): D / 32 channels of the 8 keys of one lane half and contraction step, two quads.
    const bool converts_v = wave >= 4;
    const int t = tid & 255;
    const int chunk = t & 3;                       // K: channels (D / 4) chunk ..
    const int vgroup = t & 7, word = (t >> 3) & (D / 8 - 1), part = t / D;  // V: keys, word, bytes of it
    const int quad = 4 * (vgroup >> 1) + (vgroup & 1);
    const int my_key = converts_v ? 4 * quad : t >> 2;
    const int last_key = max(key_end - 1, 0);
    int id = 0;
    uint32_t raw[8], meta[8];
    bool held = false;
    auto fetch_id = [&](int key_tile) { id = table[min(key_tile * kKeys + my_key, last_key) >> a.log2_block]; };
    auto fetch = [&](int key_tile) {
      const int key = key_tile * kKeys + my_key;
      const bool page_ok = static_cast<unsigned>(id) < static_cast<unsigned>(a.num_blocks);
      const uint32_t index = static_cast<uint32_t>(page_ok ? id : 0) * static_cast<uint32_t>(a.KV) + head;
      const char* page = reinterpret_cast<const char*>(a.cache) +
                         static_cast<uint64_t>(index) * static_cast<uint32_t>(kv_page_bytes<D>(a.log2_block));
      const uint32_t token = key & ((1 << a.log2_block) - 1);
      held = page_ok;
      if (converts_v) {
        const char* v = page + (((D / 2u) << a.log2_block) + token * (D / 2) + word * 16);
        const char* m = page + (((D + 4u) << a.log2_block) + token * 4);
        const uint4 v0 = *reinterpret_cast<const uint4*>(v), v1 = *reinterpret_cast<const uint4*>(v + 4 * D);
        const uint4 m0 = *reinterpret_cast<const uint4*>(m), m1 = *reinterpret_cast<const uint4*>(m + 32);
        raw[0] = v0.x, raw[1] = v0.y, raw[2] = v0.z, raw[3] = v0.w;
        raw[4] = v1.x, raw[5] = v1.y, raw[6] = v1.z, raw[7] = v1.w;
        meta[0] = m0.x, meta[1] = m0.y, meta[2] = m0.z, meta[3] = m0.w;
        meta[4] = m1.x, meta[5] = m1.y, meta[6] = m1.z, meta[7] = m1.w;
      } else {
        const char* k = page + (token * (D / 2) + chunk * (D / 8));
        if constexpr (D == 128) {
          const uint4 w = *reinterpret_cast<const uint4*>(k);
          raw[0] = w.x, raw[1] = w.y, raw[2] = w.z, raw[3] = w.w;
        } else {
          const uint2 w = *reinterpret_cast<const uint2*>(k);
          raw[0] = w.x, raw[1] = w.y;
        }
        const char* m = page + ((static_cast<uint32_t>(D) << a.log2_block) + token * 4);
        meta[0] = *reinterpret_cast<const uint32_t*>(m);
        meta[1] = *reinterpret_cast<const uint32_t*>(m + (4u << a.log2_block));
      }
    };
    // Fetched codes -> fp16 in LDS.  Keys outside the sequence or on no page become zeros (they hold
    // anything) and are masked by s_held.  A key whose value row is NaN would reach rows that do not
    // see it (0 * NaN in the second product): its values become zeros and its scores NaN, which masks
    // hide from those rows, and which make every row that sees it NaN.
    auto convert = [&](int key_tile, int buf) {
      const int key = key_tile * kKeys + my_key;
      if (converts_v) {
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) top = max(top, meta[i] & 0x7FFFFFFFu);
        if (__any(!held | (key + 12 > q.keys) | (top >= 0x7F800000u))) {
          top = 0;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const bool use = held & (key + (i < 4 ? i : i + 4) < q.keys) & (fabsf(kv_meta_scale(meta[i])) < INFINITY);
            meta[i] = use ? meta[i] : kZeroMeta;
            top = max(top, meta[i] & 0x7FFFFFFFu);
          }
        }
        // the next lane has the other half of the 16 keys
        const int field = group_field(max(top, static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(top), 0xB1, 0xF, 0xF, true))));
        const float factor = power(kGroupFactor - field);
        large |= __any(field > kLargeField) != 0;
        if (t < 8 && !(t & 1)) {
          s_log[buf][vgroup >> 1] = static_cast<float>(field - (kGroupFactor - 127));
          s_part[buf][vgroup >> 1] = large ? 0.0f : factor;
        }
        // A half of a word is its even or its odd channels, nibble i being channel 2 i or 2 i + 1: the
        // halves of two keys side by side, then a nibble of each.  A thread takes the 4 channels of a
        // half (D = 128), or 2 of them (D = 64).
        const int half = part & 1, nibble = D == 128 ? 0 : 2 * (part >> 1);
        const uint32_t select = half ? 0x07060302u : 0x05040100u;
        uint32_t w[D / 32][4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t pair = __builtin_amdgcn_perm(raw[2 * i + 1], raw[2 * i], select) >> (4 * nibble);
          const uint32_t zero =
              (__builtin_amdgcn_perm(meta[2 * i + 1], meta[2 * i], 0x05040100u) & hc.mask_low) | hc.bias_low;
          const uint32_t scales = pack_f16x2(kv_meta_scale(meta[2 * i]) * factor, kv_meta_scale(meta[2 * i + 1]) * factor);
#pragma unroll
          for (int c = 0; c < D / 32; ++c) w[c][i] = pair_value(((pair >> (4 * c)) & hc.mask_low) | hc.bias_low, zero, scales);
        }
#pragma unroll
        for (int c = 0; c < D / 32; ++c)
          *reinterpret_cast<uint4*>(&s_v[buf][8 * word + 2 * (nibble + c) + half][8 * vgroup]) =
              make_uint4(w[c][0], w[c][1], w[c][2], w[c][3]);
      } else {
        const bool use = held & (key < q.keys);
        const uint64_t all = __ballot(use);
        if (lane == 0) s_held[buf][wave] = all;
        uint32_t m = fabsf(kv_meta_scale(meta[1])) < INFINITY ? meta[0] : kNanMeta;
        m = use ? m : kZeroMeta;
        // a wave has the 16 keys of one group, a key in four lanes
        const uint32_t bits = m & 0x7FFFFFFFu;
        const int field = group_field(group_max(bits < 0x7F800000u ? bits : 0u));
        if (lane == 0) s_score[buf][wave] = power(field - (kGroupFactor - 254)) * scale;
        const float s = kv_meta_scale(m) * power(kGroupFactor - field);
        const uint32_t scales = pack_f16x2(s, s), z = m & 15u;
        const uint32_t zero_low = (0x6400u | z) * 0x00010001u, zero_high = (0x5400u | (z << 4)) * 0x00010001u;
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
          const uint32_t lo = raw[i], hi = raw[i] >> 8;
          *reinterpret_cast<uint4*>(&s_k[buf][t >> 2][(D / 4) * chunk + 8 * i]) =
              make_uint4(pair_value((lo & hc.mask_low) | hc.bias_low, zero_low, scales),
                         pair_value((lo & hc.mask_high) | hc.bias_high, zero_high, scales),
                         pair_value((hi & hc.mask_low) | hc.bias_low, zero_low, scales),
                         pair_value((hi & hc.mask_high) | hc.bias_high, zero_high, scales));
        }
      }
    };

    if (t0 < t1) {
      fetch_id(t0);
      fetch(t0);
      fetch_id(min(t0 + 1, t1 - 1));
    }

    // The wave's 32 rows: queries as the second operand, and what they see.
    const int first_row = row0 + 32 * wave;
    const int row = first_row + col;
    const int token = row / group, qh = head * group + row - token * group;
    const bool live = 32 * wave + col < rows;
    f16x8_t qf[kSteps];
    float row_power;  // what a row's raw scores are multiplied by
    {
      typedef uint16_t u16x2_t __attribute__((ext_vector_type(2)));
      uint4 raw_q[kSteps];
      u16x2_t top = {0, 0};
#pragma unroll
      for (int i = 0; i < kSteps; ++i) {
        raw_q[i] = make_uint4(0, 0, 0, 0);
        if (live)
          raw_q[i] = *reinterpret_cast<const uint4*>(a.q + (q.row + token) * a.q_stride_t + qh * a.q_stride_h + 16 * i + 8 * h);
        const uint32_t w[4] = {raw_q[i].x, raw_q[i].y, raw_q[i].z, raw_q[i].w};
#pragma unroll
        for (int j = 0; j < 4; ++j) top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2_t, w[j] & 0x7FFF7FFFu));
      }
      const uint16_t t0 = top[0], t1 = top[1];
      const float most = halves_max(__uint_as_float(static_cast<uint32_t>(t0 > t1 ? t0 : t1) >> 7 << 23));
      const int field = min(max(static_cast<int>(__float_as_uint(most) >> 23), 27), 254);
      const float factor = power(kRowFactor - field);
      row_power = power(field - (kRowFactor - 254));
#pragma unroll
      for (int i = 0; i < kSteps; ++i) {
        float f[8];
        unpack_bf16x8(raw_q[i], f);
        u32x4_t w;
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = pack_f16x2(f[2 * j] * factor, f[2 * j + 1] * factor);
        qf[i] = __builtin_bit_cast(f16x8_t, w);
      }
    }
    const bool tree = a.tree_mask != nullptr;
    const uint64_t bits = tree && live ? a.tree_mask[q.row + token] : 0;
    const int sees = live ? min(tree ? q.cached : q.cached + token + 1, q.keys) : 0;
    // keys that all rows of the wave see, and that some row may
    const int all_see = min(tree ? q.cached : q.cached + first_row / group + 1, q.keys);
    const int last_row = row0 + min(32 * wave + 32, rows) - 1;
    const int any_sees = 32 * wave >= rows ? 0 : tree ? q.keys : min(q.cached + last_row / group + 1, q.keys);

    f32x16_t acc[kTiles];
#pragma unroll
    for (int c = 0; c < kTiles; ++c)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[c][i] = 0.0f;
    float row_max = -INFINITY, row_sum = 0.0f;

    if (t0 < t1) {
      convert(t0, 0);
      if (t0 + 1 < t1) {
        fetch(t0 + 1);
        fetch_id(min(t0 + 2, t1 - 1));
      }
    }
    __syncthreads();

    for (int kt = t0; kt < t1; ++kt) {
      const int buf = (kt - t0) & 1;
      // The two waves of a SIMD are a K and a V converter: one converts the next tile before its
      // products, the other after, so that one's vector instructions run beside the other's
      // matrix instructions.
      auto next_tile = [&]() {
        if (kt + 1 < t1) {
          convert(kt + 1, buf ^ 1);
          if (kt + 2 < t1) {
            fetch(kt + 2);
            fetch_id(min(kt + 3, t1 - 1));
          }
        }
      };
      if (!converts_v) next_tile();
      const int key0 = kt * kKeys;
      if (key0 < any_sees) {
        f32x16_t sc[2];
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int i = 0; i < 16; ++i) sc[n][i] = 0.0f;
        // LDS reads run ahead of the matrix instructions by one group of four fragments (two steps
        // of K, one of V); V's first group is read ahead of the softmax.  Left to itself the
        // compiler reads each fragment just before its use.
        f16x8_t frag[2][4];
        auto read_k = [&](int group_of, f16x8_t (&f)[4]) {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            f[j] = *reinterpret_cast<const f16x8_t*>(&s_k[buf][32 * (j & 1) + col][16 * (2 * group_of + (j >> 1)) + 8 * h]);
        };
        auto read_v = [&](int step, f16x8_t (&f)[4]) {
#pragma unroll
          for (int c = 0; c < kTiles; ++c)
            f[c] = *reinterpret_cast<const f16x8_t*>(&s_v[buf][32 * c + col][8 * (2 * step + h)]);
        };
        read_k(0, frag[0]);
#pragma unroll
        for (int i = 0; i < kSteps / 2; ++i) {
          if (i + 1 < kSteps / 2) read_k(i + 1, frag[(i + 1) & 1]);
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int j = 0; j < 4; ++j) sc[j & 1] = mfma32(frag[i & 1][j], qf[2 * i + (j >> 1)], sc[j & 1]);
          __builtin_amdgcn_sched_barrier(0);
        }
        read_v(0, frag[0]);
        __builtin_amdgcn_sched_barrier(0);
        const uint64_t held_keys[4] = {s_held[buf][0], s_held[buf][1], s_held[buf][2], s_held[buf][3]};
        const bool all_held = (held_keys[0] & held_keys[1] & held_keys[2] & held_keys[3]) == ~0ull;
        if (__builtin_expect(!(key0 + kKeys <= all_see && all_held), 0)) {
          if (all_held && !tree) {
            const int lead = sees - key0 - 4 * h;
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
              for (int i = 0; i < 16; ++i) {
                const float y = sc[n][i];
                sc[n][i] = 32 * n + 8 * (i >> 2) + (i & 3) < lead ? y : -INFINITY;
              }
          } else {
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
              for (int i = 0; i < 16; ++i) {
                const int k = key0 + 32 * n + 8 * (i >> 2) + 4 * h + (i & 3);
                const uint64_t on = held_keys[2 * n + (i >> 3)] >> (16 * h);
                const unsigned fresh = static_cast<unsigned>(k - q.cached);
                const uint32_t half = fresh & 32u ? static_cast<uint32_t>(bits >> 32) : static_cast<uint32_t>(bits);
                const uint32_t named = fresh < 64u ? half >> (fresh & 31u) : 0u;
                const bool visible = ((on >> (4 * (8 * ((i >> 2) & 1) + (i & 3)))) & 1) & ((k < sees) | ((named & 1u) != 0));
                const float y = sc[n][i];
                sc[n][i] = visible ? y : -INFINITY;
              }
          }
#pragma unroll
          for (int n = 0; n < 2; ++n) asm volatile("" : "+v"(sc[n]));
        }
        // The scores as whole accumulators on both sides of the branch's end: taken apart, they would be
        // copied on the path that masks nothing (32 instructions a tile, 4 % of a long chunk's time).
#pragma unroll
        for (int n = 0; n < 2; ++n) asm volatile("" : "+v"(sc[n]));
        // A weight is 2^(score + the values' power - reference): the powers of two of keys, values and
        // queries are one multiplier and one addend a group.
        const f32x4_t of_score = *reinterpret_cast<const f32x4_t*>(s_score[buf]), of_value = *reinterpret_cast<const f32x4_t*>(s_log[buf]);
        const f32x4_t of_sum = *reinterpret_cast<const f32x4_t*>(s_part[buf]);
        float by[4], top = -INFINITY;
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int s = 0; s < 2; ++s) {
            by[2 * n + s] = __builtin_amdgcn_fmed3f(of_score[2 * n + s] * row_power, 0x1p-126f, 0x1p127f);
            float most = sc[n][8 * s];
#pragma unroll
            for (int i = 1; i < 8; ++i) most = fmaxf(most, sc[n][8 * s + i]);
            top = fmaxf(top, __builtin_fmaf(most, by[2 * n + s], of_value[2 * n + s]));
          }
        top = halves_max(top);
        // The reference is 7 below the maximum where it was set, and follows when that leads it by
        // more than 15: weights stay below 2^15 as fp16, keep 11 bits down to 2^-21 of the row's
        // largest at least, and sums are rescaled rarely.
        const bool grew = top > row_max && top - row_max > 15.0f, large_values = of_sum[0] == 0.0f;
        if (__any(grew | large_values)) {
          const float next = grew ? top - 7.0f : row_max, change = row_max - (next == -INFINITY ? 0.0f : next);
          const float f = __builtin_amdgcn_exp2f(change);
          row_max = next;
          row_sum = scaled(row_sum, change);
#pragma unroll
          for (int c = 0; c < kTiles; ++c)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[c][i] *= f;
          if (large_values) {
            const float from = next == -INFINITY ? 0.0f : -next;
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
              for (int i = 0; i < 16; ++i)
                row_sum += __builtin_amdgcn_exp2f(__builtin_fmaf(sc[n][i], by[2 * n + (i >> 3)], from));
          }
        }
        const float ref = row_max == -INFINITY ? 0.0f : row_max;
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int s = 0; s < 2; ++s) {
            if (2 * n + s < 3) read_v(2 * n + s + 1, frag[(s + 1) & 1]);
            u32x4_t w;
            const float from = of_value[2 * n + s] - ref;
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[n][8 * s + 2 * i], by[2 * n + s], from));
              const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[n][8 * s + 2 * i + 1], by[2 * n + s], from));
              sum += p0;
              sum += p1;
              w[i] = pack_f16x2(p0, p1);
            }
            row_sum = __builtin_fmaf(sum, of_sum[2 * n + s], row_sum);
            const f16x8_t pf = __builtin_bit_cast(f16x8_t, w);
#pragma unroll
            for (int c = 0; c < kTiles; ++c) acc[c] = mfma32(frag[s & 1][c], pf, acc[c]);
          }
      }
      if (converts_v) next_tile();
      __syncthreads();
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
          for (int f = 0; f < D / 8; ++f) store_fragment(ro, part_offset<D, kPromptThreads / 64>(slot, wave, f, lane), own[f]);
          if (h == 0) store_stats(rs, (static_cast<uint32_t>(slot) * kKvPromptRows + 32 * wave + col) * 8, row_max, row_sum);
        }
        last = kv_arrive(out.counters + first, count, &s_last);
      } else if (tid == 0) {
        rearm(out.counters + first);
      }
      if (last) {
        join_parts<D, kPromptThreads / 64>(out, first, count, me - first, wave, lane, live, row_max, row_sum, own);
        write_rows<D>(a, live, q.row + token, qh, lane, row_sum, own);
      }
      __syncthreads();  // s_last is read by all before the next tile writes it
    }
    u += x1 - x0;
  }
}

}  // namespace

hipError_t launch_kv_prompt(const KvAttentionArgs& a, const KvPartials& part, int workers, hipStream_t stream) {
  if (a.D == 64)
    kv_prompt_kernel<64><<<workers, kPromptThreads, 0, stream>>>(a, part);
  else
    kv_prompt_kernel<128><<<workers, kPromptThreads, 0, stream>>>(a, part);
  return hipGetLastError();
}

}  // namespace w4a16
