// paged_prefill_int4.cu — paged prefill / chunked-prefill attention over a 4-bit
// cache (format in kv_int4.cuh) on tcgen05 + TMEM.
//
// Row (token, q head) i of a sequence at position x attends to tokens t <= x:
//   o_i = sum_t p_it v_t / sum_t p_it,  p_it = exp2(c q_i . k_t - m_i)
// with k_t, v_t = s (code - 8) and c = scale log2(e).
//
// Bound: the MMAs (4 x 128 operations per row and token) and, right behind
// them, an exp2 per row and token; the cache is 3.6 times smaller than in 16
// bits and never bounds. What does is a tile's chain: S, its softmax and PV of a Q
// tile follow one another, as P lies over S, and one softmax warp a scheduler and Q
// tile walks through it. 2048 rows on 8k tokens: the MMA pipe is 40 % active, 52 % of
// the issue slots are used, and of the 7.2 cycles between two instructions of a warp
// 2.0 wait for tensor memory and barriers, 1.7 for fixed latencies, 0.9 for
// instructions. The converters' instructions (3 to 4 per pair of values next to the
// softmax's 7 per pair of scores) are in that chain's way, so both are kept short, and
// their loops small: at 14 KB of hot code more than a third of the fetches missed the
// instruction cache (1.8 ms for 2048 rows on 32k tokens, 1.3 once they were short).
//
// Work. A unit is (sequence, block of 256 packed rows, KV head): the (token, q
// head of the group) rows of 256 / group query tokens, two UMMA M = 128 tiles A
// and B that share every K and V tile of 128 tokens. Its cost is the tiles it
// streams plus kUnitCost for its start and end. One CTA per SM; every CTA derives
// its work from the lengths by itself, so the host needs none of them:
//   * Units all below a third of a share, or shares below kSplitShare and no unit
//     much above one: units whole, back and forth through the costliest-first order
//     (at most kOrder sequence blocks, ranked by each CTA).
//   * Otherwise the sum of all costs is cut into equal shares, in unit order, one
//     a CTA. A cut inside a unit leaves parts, whose sums (O, m, l in fp32) go to
//     the workspace and are joined in part order by a second kernel; a cut within
//     kMinPart tiles of a unit's end moves there. Without a workspace cuts move to
//     the nearest end.
// Measured (32 q heads, 8 KV heads, bf16; us, whole and cut): 2048 rows on 32k tokens,
// 256 equal units on 148 SMs, 1280 and 1241 (1204 in short runs: 0.89 PFLOP/s); on 8k,
// 307 and 300; 64 rows on 8k, 8 units, 170 and 45, eight of them 176 and 104; four
// chunks of 512 on 512 to 2560 tokens, 76 and 97; two prompts of 2048, 120 and 138; one
// of 8192, 684 and 734. The rule looks at the longest unit and the share only and not
// at how whole units fall on the SMs, so near its edges it can take the slower: three
// chunks of 512 on 512 to 2560 tokens 67 and 80, and cut; a prompt of 4096 184 and 214,
// cut; 19 x 64 rows on 2048 tokens, 152 equal units, 106 and 82, and whole.
//
// A CTA's 16 warps:
//   0-3, 4-7  softmax of tile A, B: thread = row = TMEM lane. A row's 128 scores
//             stay in registers between the maximum and the exponentials.
//   8         one thread issues all MMAs: PV_A(j) S_A(j+1) PV_B(j) S_B(j+1) ...,
//             across units, so the tensor core works on one tile while the other
//             tile's warps run their softmax
//   9-15      converters, 32 rows of a tile each in turn, K0 K1 V0 K2 V1 ..., across
//             units: codes and scales from the cache to registers, one item ahead,
//             and as T to the swizzled layouts the MMAs read. (16-token boxes by TMA
//             took 150 to 200 cycles each to issue, 32 a tile, more than the tile.)
// setmaxnreg moves registers from the last two warpgroups (80) to the softmax
// ones (176), which hold a row's 128 scores.
//
// Order of columns. A word of 8 codes gives the pairs (e0 e4) (e1 e5) (e2 e6)
// (e3 e7) with one mask each, so K and V tiles hold each 8 columns in the order
// 0 4 1 5 2 6 3 7. Q is staged in the same order, and O is put back in order
// when it leaves; both are rare next to the tiles.
//
// Roundings. The MMAs run in fp16 for bf16 calls too: s (c - 8) has up to 11 bits
// and is exact there, and p loses 3 bits less (against the 64-bit result 0.0017 of
// the output's norm, all of it the output's own rounding, where bf16 operands gave
// 0.0032). bf16 queries become fp16 exactly, each row times a power of two. p is
// rounded to the operands' type while l sums it unrounded.
//
// A unit with a scale that fp16 does not hold is run a second time, before the CTA's
// next units; its first results are overwritten. Weights and values are bf16 then (2^-8
// each). Keys stay exact in fp16, times a power of two of the unit, while their scales
// lie within 2^25; beyond that they, and the queries, are bf16 as well. fp16
// calls need it as well: the cache has no type, and a value that overflows is 0 times
// infinity in every row that does not see it. A converter warp looks closer where a
// scale lies outside the octaves that it has met in the unit, so this costs a vote and
// some ten instructions an item (chunks of 512 on 0 to 2048 tokens: 75.6 us without it,
// 76.6 with it).
#include <cuda_runtime.h>
#include <math.h>

#include <type_traits>

#include "common.cuh"
#include "kv_int4.cuh"
#include "paged_decode.cuh"
#include "tcgen05.cuh"

namespace b200 {
namespace {

constexpr int kRows = 128;  // UMMA M
constexpr int kTokens = 128;  // KV tokens of a tile
constexpr int kThreads = 512;
constexpr int kMmaWarp = 8, kConvWarp = 9, kConvs = 7;
constexpr int kListWarp = 12;  // warps 12-15 also deal and list the units
constexpr int kSoftmaxRegs = 176, kOtherRegs = 80;
static_assert(256 * kSoftmaxRegs + 256 * kOtherRegs <= kThreads * 128, "registers at launch");

constexpr int kHalfBytes = kRows * 128;      // [128 rows x 64 columns]
constexpr int kTileBytes = 2 * kHalfBytes;
constexpr int kUnits = 15;  // of a CTA's list (as there is room for); longer lists run in rounds
constexpr int kOutBytes = 32 * 128;  // 32 rows x 64 columns of output on their way, a warp
// shared memory: Q A, B | K x 2 | V x 2 | output x 8 | list | barriers
constexpr int kQ0 = 0;
constexpr int kK0 = 2 * kTileBytes;
constexpr int kV0 = kK0 + 2 * kTileBytes;
constexpr int kOut0 = kV0 + 2 * kTileBytes;
constexpr int kList0 = kOut0 + 8 * kOutBytes;

constexpr int kOrder = 256;  // sequence blocks that are ranked: of 128 sequences at most

// One unit, or part of one, of a CTA.
struct Unit {
  int seq, kvh;
  int row0;      // first query token (row of q)
  int ntok;      // query tokens
  int pos0;      // position of the first
  int seq_len;
  int t0, t1;    // KV tiles [t0, t1)
  int lim[2];    // tiles that A, B need: [0, lim)
  int rec;       // record of a part, or -1: the whole unit
  int nan[4];    // first token whose value group g has no finite scale
  // 0, 1 when a scale is found that fp16 operands do not hold; the second run: 2 with
  // weights and values in bf16, 3 with keys and queries as well
  int wide;
  uint32_t k_ranges;      // of the key scales, the ends: bit i from 2^(5 i - 80) on, 0 and 31 also beyond
  uint32_t v_octaves[4];  // of value group g's scales, the ends: bit i from 2^(i - 18) on, 0 also below
};

struct Shared {
  Unit units[kUnits];
  uint64_t k_full[2], k_empty[2], v_full[2], v_empty[2];
  uint64_t s_full[2], p_lo[2], p_hi[2], o_done[2], q_full[2];
  uint64_t drain;
  // the walk over the units, kept between rounds by the thread that lists them
  int64_t share, base;          // base: position of the next unit
  int64_t scan[4];
  int2 scan_pairs[4];
  int seq, block, kvh;          // the next unit
  int whole;                    // units are dealt whole, from `order`
  uint16_t order[kOrder];       // (sequence << 9 | block) pairs, costliest first
  int count, tiles;             // of the list
  int dead;                     // a wait ran out
  uint32_t tmem;
};
constexpr int kSmemBytes = 1024 + kList0 + sizeof(Shared);
static_assert(kSmemBytes <= 227 * 1024, "shared memory budget");

constexpr int kUnitCost = 3;  // of a unit besides its tiles, in tiles (2: 20000 rows 12 % slower)
constexpr int kMinPart = kInt4PrefillMinPart;
constexpr int kSplitShare = 64;  // shares from here on are always cut
constexpr float kRescale = 8.f;  // log2
// fp16 weights are multiplied by 2^7 (2^15 at most, by kRescale): those down to 2^-21 of
// a row's largest are normal numbers there. bf16 ones stay at or below 1, so that sums of
// the largest values are finite.
constexpr float kWeightLift = 7.f;

__device__ __forceinline__ void bar_sync(int id, int threads) {
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}

// Tiles of query tokens [.., last] of a sequence: keys up to position pos.
__device__ __forceinline__ int tiles_to(int seq_len, int pos) {
  return seq_len <= 0 ? 0 : (min(seq_len, max(1, pos + 1)) + kTokens - 1) / kTokens;
}

// Where a cut at offset o of a unit goes: 0, the unit's cost, or a tile.
__device__ __forceinline__ int cut(int o, int tiles, bool split) {
  const int cost = tiles + kUnitCost;
  if (o <= 0) return 0;
  if (o >= cost) return cost;
  if (!split || tiles < 2 * kMinPart) return 2 * o < cost ? 0 : cost;
  return o < kMinPart ? 0 : o > tiles - kMinPart ? cost : (int)o;
}

struct SeqInfo {
  int row0, q_len, len;
  __device__ __forceinline__ int blocks(int per) const { return q_len > 0 ? (q_len - 1) / per + 1 : 0; }
  __device__ __forceinline__ int tiles(int block, int per) const {
    return tiles_to(len, len - q_len + min(q_len, (block + 1) * per) - 1);
  }
};
__device__ __forceinline__ SeqInfo seq_info(const Int4PrefillParams& p, int s) {
  const int r = p.query_start_loc[s];
  return {r, p.query_start_loc[s + 1] - r, p.seq_lens[s]};
}

// The share of each CTA, and the unit this CTA's begins in. 128 threads.
__device__ void find_share(const Int4PrefillParams& p, Shared* sh, int* scratch, int i) {
  const int per = 256 / p.group;
  const int chunk = (p.num_seqs + 127) / 128;
  const int s0 = min(p.num_seqs, i * chunk), s1 = min(p.num_seqs, s0 + chunk);
  int64_t sum = 0;
  int pairs = 0, most = 0;
  for (int s = s0; s < s1; ++s) {
    const SeqInfo q = seq_info(p, s);
    const int n = q.blocks(per);
    for (int b = 0; b < n; ++b) sum += q.tiles(b, per) + kUnitCost;
    pairs += n;
    if (n > 0) most = max(most, q.tiles(n - 1, per) + kUnitCost);
  }
  sum *= p.cache.num_kv_heads;
  int64_t incl = sum;
  int incl_pairs = pairs;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int64_t v = __shfl_up_sync(0xffffffffu, incl, d);
    const int n = __shfl_up_sync(0xffffffffu, incl_pairs, d);
    if ((i & 31) >= d) {
      incl += v;
      incl_pairs += n;
    }
  }
  most = __reduce_max_sync(0xffffffffu, most);
  if ((i & 31) == 31) {
    sh->scan[i >> 5] = incl;
    sh->scan_pairs[i >> 5] = make_int2(incl_pairs, most);
  }
  bar_sync(2, 128);
  int64_t before = incl - sum, total = 0;
  int first_pair = incl_pairs - pairs, total_pairs = 0;
  for (int w = 0; w < 4; ++w) {
    if (w < (i >> 5)) {
      before += sh->scan[w];
      first_pair += sh->scan_pairs[w].x;
    }
    total += sh->scan[w];
    total_pairs += sh->scan_pairs[w].x;
    most = max(most, sh->scan_pairs[w].y);
  }
  int64_t share = (total + gridDim.x - 1) / gridDim.x;
  if (share < kMinPart + kUnitCost - 1) share = kMinPart + kUnitCost - 1;
  const bool whole =
      total_pairs <= kOrder && p.num_seqs <= 128 &&
      (p.records == nullptr || 3 * most <= share || (share < kSplitShare && 4 * most <= 5 * share));
  if (i == 0) sh->whole = whole;
  if (whole) {
    int id = first_pair;
    for (int s = s0; s < s1; ++s) {
      const SeqInfo q = seq_info(p, s);
      const int n = q.blocks(per);
      for (int b = 0; b < n; ++b, ++id) {
        scratch[id] = q.tiles(b, per) + kUnitCost;
        scratch[kOrder + id] = s << 9 | b;
      }
    }
    bar_sync(2, 128);
    for (int at = i; at < total_pairs; at += 128) {
      const int cost = scratch[at];
      int rank = 0;
      for (int k = 0; k < total_pairs; ++k)
        rank += scratch[k] > cost || (scratch[k] == cost && k < at);
      sh->order[rank] = (uint16_t)scratch[kOrder + at];
    }
    if (i == 0) {
      sh->base = 0;
      sh->seq = total_pairs;
    }
    return;
  }
  const int64_t lo = share * blockIdx.x;
  if (i == 0) {
    sh->share = share;
    if (lo >= total) sh->seq = p.num_seqs;
  }
  if (lo >= before && lo < before + sum) {
    int64_t at = before;
    for (int s = s0; s < s1; ++s) {
      const SeqInfo q = seq_info(p, s);
      const int n = q.blocks(per);
      for (int b = 0; b < n; ++b) {
        const int cost = q.tiles(b, per) + kUnitCost;
        if (lo < at + (int64_t)cost * p.cache.num_kv_heads) {
          const int h = (int)((lo - at) / cost);
          sh->seq = s;
          sh->block = b;
          sh->kvh = h;
          sh->base = at + (int64_t)h * cost;
          return;
        }
        at += (int64_t)cost * p.cache.num_kv_heads;
      }
    }
  }
}

__device__ void put_unit(const Int4PrefillParams& p, Unit& u, const SeqInfo& q, int s, int b, int h,
                         int t0, int t1, int tiles) {
  const int per = 256 / p.group;
  u.seq = s;
  u.kvh = h;
  u.row0 = q.row0 + b * per;
  u.ntok = min(per, q.q_len - b * per);
  u.pos0 = q.len - q.q_len + b * per;
  u.seq_len = q.len;
  u.t0 = t0;
  u.t1 = t1;
  // tile A's last valid row; B's is the unit's
  const int rows = u.ntok * p.group;
  u.lim[0] = tiles_to(q.len, u.pos0 + (min(kRows, rows) - 1) / p.group);
  u.lim[1] = rows > kRows ? tiles : 0;
  u.rec = t0 > 0 ? 2 * (int)blockIdx.x : t1 < tiles ? 2 * (int)blockIdx.x + 1 : -1;
  u.wide = 0;
  u.k_ranges = 0;
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    u.nan[g] = 0x7fffffff;
    u.v_octaves[g] = 0;
  }
}

// The next units of this CTA's share, by one thread.
__device__ void list_units(const Int4PrefillParams& p, Shared* sh, bool first) {
  const int per = 256 / p.group;
  const bool split = p.records != nullptr;
  if (first && split) p.joins[blockIdx.x] = make_int4(0, 0, 0, 0);
  if (sh->whole) {
    // unit k of this CTA: back and forth through the order, so that a CTA with a
    // costly unit in one round has a cheap one in the next
    const int grid = gridDim.x, units = sh->seq * p.cache.num_kv_heads;
    int k = (int)sh->base, n = 0, total = 0;
    for (; n < kUnits; ++k) {
      const int64_t at = (int64_t)k * grid + (k & 1 ? grid - 1 - blockIdx.x : blockIdx.x);
      if (at >= units) break;
      const int pair = sh->order[(int)at / p.cache.num_kv_heads];
      const SeqInfo q = seq_info(p, pair >> 9);
      const int b = pair & 511, tiles = q.tiles(b, per);
      put_unit(p, sh->units[n++], q, pair >> 9, b, (int)at % p.cache.num_kv_heads, 0, tiles, tiles);
      total += tiles;
    }
    sh->base = k;
    sh->count = n;
    sh->tiles = total;
    return;
  }
  const int64_t share = sh->share;
  const int64_t lo = share * blockIdx.x;
  const int len = (int)share;
  int base = (int)(sh->base - lo);
  int s = sh->seq, b = sh->block, h = sh->kvh, n = 0, total = 0;
  SeqInfo q{};
  if (s < p.num_seqs) q = seq_info(p, s);
  while (n < kUnits && s < p.num_seqs && base < len) {
    const int tiles = q.tiles(b, per);
    const int cost = tiles + kUnitCost;
    const int o0 = cut(-base, tiles, split), o1 = cut(len - base, tiles, split);
    if (o1 > o0) {
      Unit& u = sh->units[n++];
      put_unit(p, u, q, s, b, h, min(o0, tiles), min(o1, tiles), tiles);
      total += u.t1 - u.t0;
      if (u.t0 == 0 && u.t1 < tiles) {
        int parts = 2;
        for (int c = 2 * len; cut(c - base, tiles, split) < cost; c += len) ++parts;
        p.joins[blockIdx.x] = make_int4(parts, u.row0, u.ntok, h);
      }
    }
    base += cost;
    if (++h == p.cache.num_kv_heads) {
      h = 0;
      if (++b >= q.blocks(per)) {
        b = 0;
        do {
          if (++s >= p.num_seqs) break;
          q = seq_info(p, s);
        } while (q.q_len <= 0);
      }
    }
  }
  sh->base = lo + base;
  sh->seq = s;
  sh->block = b;
  sh->kvh = h;
  sh->count = n;
  sh->tiles = total;
}

// Key scales by fives of octaves. Where six of them hold all keys of a unit, a power of
// two brings its scales to [2^-17, 2^13), where fp16 holds s (c - 8) exactly.
__device__ __forceinline__ uint32_t key_range(uint32_t bits) {
  return 1u << min(max((static_cast<int>(bits >> 7) - 47) / 5, 0), 31);
}
__device__ __forceinline__ bool keys_shifted(uint32_t ranges) {
  return 32 - __clz(ranges) - __ffs(ranges) <= 5 && !(ranges & 0x80000001u);
}
__device__ __forceinline__ int key_shift(uint32_t ranges) {  // its exponent
  return ranges == 0 ? 0 : 88 - 5 * (31 - __clz(ranges));
}

// The units of the list that have to run again; true if there are any.
__device__ bool list_wide(Shared* sh) {
  int n = 0, total = 0;
  for (int e = 0; e < sh->count; ++e) {
    if (sh->units[e].wide != 1) continue;
    Unit& u = sh->units[n++];
    u = sh->units[e];
    u.wide = keys_shifted(u.k_ranges) ? 2 : 3;
#pragma unroll
    for (int g = 0; g < 4; ++g) u.nan[g] = 0x7fffffff;
    total += u.t1 - u.t0;
  }
  if (n == 0) return false;
  sh->count = n;
  sh->tiles = total;
  return true;
}

// A walk over the tiles of the list.
struct Cursor {
  int e = 0, t = 0;
  __device__ __forceinline__ void seek(const Shared* sh) {
    while (e < sh->count && sh->units[e].t0 >= sh->units[e].t1) ++e;
    if (e < sh->count) t = sh->units[e].t0;
  }
  __device__ __forceinline__ void next(const Shared* sh) {
    if (++t >= sh->units[e].t1) {
      ++e;
      seek(sh);
    }
  }
};

// Items of a list of n / 2 tiles: K0 K1 V0 K2 V1 ... V(n/2 - 2) V(n/2 - 1).
__device__ __forceinline__ bool item_is_v(int i, int n) {
  return i >= 2 ? (i & 1) == 0 || i == n - 1 : i == n - 1;
}

// 8 codes -> 8 values of T in the order 0 4 1 5 2 6 3 7, each rn(s (c - 8)).
struct ConvertBf16 {
  uint32_t mul;
  __device__ __forceinline__ explicit ConvertBf16(uint32_t bits) : mul(bits | (bits << 16)) {}
  __device__ __forceinline__ uint32_t pair(uint32_t w) const {
    uint32_t v = (w & 0x000f000fu) | 0x43004300u;  // 128 + c
    asm("add.rn.bf16x2 %0, %0, %1;" : "+r"(v) : "r"(0xc308c308u));  // - 136
    asm("mul.rn.bf16x2 %0, %0, %1;" : "+r"(v) : "r"(mul));
    return v;
  }
  __device__ __forceinline__ uint4 operator()(uint32_t w) const {
    return make_uint4(pair(w), pair(w >> 4), pair(w >> 8), pair(w >> 12));
  }
};
// fp16: both nibbles of a byte fit the mantissa, 1024 + c and 1024 + 16 c, and one
// add or fma makes either c - 8 (the published way of turning small integers into
// floating point: as the low bits of a number whose last place is 1). kSmall: scales below 2^-14, subnormal in fp16, are
// multiplied in as 256 s, exact down to 2^-22, and the last product, by 2^-8, rounds.
template <bool kSmall>
struct ConvertHalf {
  uint32_t mul;
  uint32_t post = 0x3c003c00u;
  __device__ __forceinline__ explicit ConvertHalf(float s) {
    if (kSmall && s < 6.103515625e-5f) {
      s *= 256.f;
      post = 0x1c001c00u;
    }
    mul = Elem<__half>::pack(s, s);
  }
  __device__ __forceinline__ uint32_t scaled(uint32_t v) const {
    asm("mul.rn.f16x2 %0, %0, %1;" : "+r"(v) : "r"(mul));
    if (kSmall) asm("mul.rn.f16x2 %0, %0, %1;" : "+r"(v) : "r"(post));
    return v;
  }
  __device__ __forceinline__ uint32_t low(uint32_t w) const {
    uint32_t v = (w & 0x000f000fu) | 0x64006400u;
    asm("add.rn.f16x2 %0, %0, %1;" : "+r"(v) : "r"(0xe408e408u));  // - 1032
    return scaled(v);
  }
  __device__ __forceinline__ uint32_t high(uint32_t w) const {
    uint32_t v = (w & 0x00f000f0u) | 0x64006400u;
    asm("fma.rn.f16x2 %0, %0, %1, %2;" : "+r"(v) : "r"(0x2c002c00u), "r"(0xd480d480u));  // / 16 - 72
    return scaled(v);
  }
  __device__ __forceinline__ uint4 operator()(uint32_t w) const {
    const uint32_t t = w >> 8;
    return make_uint4(low(w), high(w), low(t), high(t));
  }
};

// Whether fp16 holds s (c - 8) for scales from `low` (bf16 bits less one) to `top`. bf16
// calls: from 2^13 on 7 s overflows, and below 2^-16 a rounding of s and one of the
// product pass 2^-9 of the value each. fp16 calls: rows appended in fp16 have 9344 at
// most; small values are as exact as the output is.
template <bool kHalf>
__device__ __forceinline__ bool fp16_holds(uint32_t low, uint32_t top) {
  return kHalf ? top <= 0x4612u : top < 0x4600u && low >= 0x377fu;
}
// Weights below 2^-21 of a row's largest are multiples of 2^-32 of it, which is less
// than the roundings of the others while the values of a group lie within 2^18.
constexpr int kApart = 18;
__device__ __forceinline__ uint32_t octave(uint32_t bits) {
  return 1u << min(max(static_cast<int>(bits >> 7) - (127 - 18), 0), 31);
}
// The ends of a scale's octave (so that not each new extreme is one), within what fp16
// holds; 0 is none.
template <bool kHalf>
__device__ __forceinline__ uint32_t octave_top(uint32_t bits) {
  return bits == 0 ? 0u : kHalf && bits <= 0x4612u ? min(bits | 0x7fu, 0x4612u) : bits | 0x7fu;
}
__device__ __forceinline__ uint32_t octave_low(uint32_t less_one) {
  return ((less_one + 1u) & ~0x7fu) - 1u;
}
// One lane's 32 codes -> four 16-byte chunks at shared addresses dst[j] + kOff.
template <int kOff, typename C>
__device__ __forceinline__ void convert32(const C& f, const uint4& w, const uint32_t (&dst)[4]) {
  const uint32_t words[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint4 v = f(words[j]);
    asm volatile("st.shared.v4.b32 [%0 + %1], {%2, %3, %4, %5};" ::"r"(dst[j]), "n"(kOff), "r"(v.x),
                 "r"(v.y), "r"(v.z), "r"(v.w)
                 : "memory");
  }
}

// One lane of a converged warp. The MMA loop runs under this predicate, not under
// lane == 0: the compiler then keeps descriptors in uniform registers (9 cycles a
// small MMA against 45, which the loop needs 32 times a tile next to three busy
// warps on its sub-partition).
__device__ __forceinline__ bool elect_one() {
  uint32_t on;
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b32 r;\n\telect.sync r|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(on));
  return on != 0;
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

__device__ __forceinline__ void tmem_ld16(uint32_t addr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, "
      "%12, %13, %14, %15}, [%16];\n\ttcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15])
      : "r"(addr)
      : "memory");
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool on) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src),
               "r"(on ? 16 : 0)
               : "memory");
}

// A record: [130][128 rows] floats, 128 columns of O (in tile order), their base 2^m and l.
__device__ __forceinline__ float* record(float* records, int rec, int x) {
  return records + ((int64_t)rec * 2 + x) * (130 * kRows);
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 1)
    int4_prefill_kernel(const Int4PrefillParams p) {
  constexpr bool kHalf = Elem<T>::kDtype == B200_DTYPE_FLOAT16;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  Shared* sh = reinterpret_cast<Shared*>(smem + kList0);
  const uint32_t sbase = smem_u32(smem);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&sh->k_full[i]), 4);
      mbar_init(smem_u32(&sh->k_empty[i]), 1);
      mbar_init(smem_u32(&sh->v_full[i]), 4);
      mbar_init(smem_u32(&sh->v_empty[i]), 1);
      mbar_init(smem_u32(&sh->s_full[i]), 1);
      mbar_init(smem_u32(&sh->p_lo[i]), kRows);
      mbar_init(smem_u32(&sh->p_hi[i]), kRows);
      mbar_init(smem_u32(&sh->o_done[i]), 1);
      mbar_init(smem_u32(&sh->q_full[i]), kRows);
    }
    mbar_init(smem_u32(&sh->drain), 1);
    sh->dead = 0;
    mbar_init_fence();
  }
  if (warp == kMmaWarp) {
    tmem_alloc(smem_u32(&sh->tmem), 512);
    tmem_relinquish();
  }
  pdl_launch_dependents();
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_base = sh->tmem;

  // Each role: wait for the list, work through it, and meet again. A role whose
  // wait ran out reports it and sets `dead`, which ends every role's next round.
  auto give_up = [&] {
    report_status(p.status, B200_STATUS_WAIT_TIMEOUT);
    atomicExch(&sh->dead, 1);
  };

  // one instruction for the whole of each warpgroup
  if (warp < 8)
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
  else
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));

  if (warp < 8) {
    // -------------------------------------------------------------- softmax --
    const int x = warp >> 2;          // Q tile
    const int t = threadIdx.x & 127;  // row of it
    const int tl = (x * kRows + t) / p.group;
    const uint32_t tS = tmem_base + x * 256 + ((uint32_t)((warp & 3) * 32) << 16);
    const uint32_t tO = tS + 128;
    uint8_t* qtile = smem + kQ0 + x * kTileBytes;
    auto limit = [&](int e) { return min(sh->units[e].t1, sh->units[e].lim[x]); };
    // Q of unit e into the tile, this warp's 32 rows: 16 lanes copy a row, so that
    // a copy touches 2 rows and not 32. Each lane then orders the chunks it copied.
    const int qr = (warp & 3) * 32 + (lane >> 4), qc = lane & 15;
    const uint32_t qdst = smem_u32(qtile) + (qc >> 3) * kHalfBytes;
    auto stage_q = [&](int e) {
      const Unit& u = sh->units[e];
      const T* src = reinterpret_cast<const T*>(p.q) + (int64_t)u.row0 * p.q_token_stride +
                     (int64_t)(u.kvh * p.group) * p.q_head_stride + qc * 8;
#pragma unroll 4
      for (int i = 0; i < 32; i += 2) {
        const int r = x * kRows + qr + i, tok = r * p.inv_group >> 16;
        const bool on = tok < u.ntok;
        cp_async16(qdst + swz128(qr + i, qc & 7),
                   src + (on ? tok * p.q_token_stride + (r - tok * p.group) * p.q_head_stride : 0),
                   on);
      }
    };
    // in the tiles' order of columns; bf16 rows as fp16, each times a power of two
    // that puts its largest element into [2^14, 2^15), which the row's scale undoes
    float scale = p.scale_log2;  // of this thread's row in the unit whose Q is ordered
    auto order_q = [&](int e) {
      asm volatile("cp.async.wait_all;" ::: "memory");
      const int wide = sh->units[e].wide;
      int shift = 0;
#pragma unroll 2
      for (int i = 0; i < 32; i += 2) {
        uint4* ptr = reinterpret_cast<uint4*>(qtile + (qc >> 3) * kHalfBytes + swz128(qr + i, qc & 7));
        uint4 v = *ptr;
        if (kHalf && wide == 3) {
          auto brain = [&](uint32_t w) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
            return Elem<__nv_bfloat16>::pack(f.x, f.y);
          };
          v = make_uint4(brain(v.x), brain(v.y), brain(v.z), brain(v.w));
        }
        if (!kHalf && wide != 3) {
          uint32_t most = __vmaxu2(__vmaxu2(v.x & 0x7fff7fffu, v.y & 0x7fff7fffu),
                                   __vmaxu2(v.z & 0x7fff7fffu, v.w & 0x7fff7fffu));
          most = max(most & 0xffffu, most >> 16);
#pragma unroll
          for (int d = 1; d < 16; d <<= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, d));
          // no more than 2^126; rows with an infinity or a NaN as they are
          const int k = most >= 0x7f80u ? 0 : min(126, 127 + 14 - (int)(most >> 7));
          const float f = __uint_as_float((uint32_t)(127 + k) << 23);
          auto half = [&](uint32_t w) {
            return Elem<__half>::pack(__uint_as_float(w << 16) * f,
                                      __uint_as_float(w & 0xffff0000u) * f);
          };
          v = make_uint4(half(v.x), half(v.y), half(v.z), half(v.w));
          const int of_row = __shfl_sync(0xffffffffu, k, (lane & 1) * 16);
          if ((lane & 30) == i) shift = of_row;
        }
        *ptr = make_uint4(__byte_perm(v.x, v.z, 0x5410), __byte_perm(v.x, v.z, 0x7632),
                          __byte_perm(v.y, v.w, 0x5410), __byte_perm(v.y, v.w, 0x7632));
      }
      if (wide == 2) shift += key_shift(sh->units[e].k_ranges);
      // never 0: masked scores are -inf, and stay so
      scale = fmaxf(ldexpf(p.scale_log2, -shift), 1.1754944e-38f);
      fence_proxy_async_smem();
      mbar_arrive(smem_u32(&sh->q_full[x]));
    };
    auto next_unit = [&](int e) {  // with tiles for this Q tile
      while (e < sh->count && limit(e) <= sh->units[e].t0) ++e;
      return e;
    };
    int done = 0, units = 0;  // tiles and units behind this warpgroup
    while (true) {
      bar_sync(1, kThreads);
      if (sh->dead || sh->count == 0) break;
      bool ok = true;
      const int first = next_unit(0);
      if (first < sh->count) {
        stage_q(first);
        order_q(first);
      }
      for (int e = 0; e < sh->count && ok; ++e) {
        const Unit& u = sh->units[e];
        const int t0 = u.t0, end = limit(e);
        const int qpos = tl < u.ntok ? u.pos0 + tl : -1;
        const int seen = min(qpos + 1, u.seq_len);  // tokens this row sees
        float m = -INFINITY, l = 0.f;
        const float row_scale = scale;
        const bool wide = u.wide >= 2;
        const float weight_lift = wide ? -kRescale : kWeightLift;
        for (int j = t0; j < end; ++j) {
          const bool got = mbar_wait(smem_u32(&sh->s_full[x]), done & 1);
          if (!__all_sync(0xffffffffu, got)) {
            ok = false;
            break;
          }
          ++done;
          tc_fence_after_sync();
          // S_X(j) done implies PV_X(j-1) done (in-order MMAs): O_X is stable
          // and the P_X(j-1) columns may be overwritten
          // scores this row does not see become -inf where they lie: a loop that few
          // tiles enter, against 256 predicated instructions in every tile if the
          // registers were masked
          const int lim = seen - j * kTokens;
          if (__any_sync(0xffffffffu, lim < kTokens)) {
#pragma unroll 1
            for (int c = 0; c < kTokens; c += 32) {
              float v[32];
              tmem_ld32(tS + c, v);
#pragma unroll
              for (int i = 0; i < 32; ++i)
                if (c + i >= lim) v[i] = -INFINITY;
              tmem_st32(tS + c, v);
            }
            tmem_wait_st();
          }
          float sv[2][64];
          tmem_ld64(tS, sv[0]);
          tmem_ld64(tS + 64, sv[1]);
          if (j + 1 == end) {  // the Q tile is free: fetch the next unit's
            const int n = next_unit(e + 1);
            if (n < sh->count) stage_q(n);
          }
          float mk[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int i = 0; i < 64; ++i)
            mk[i & 3] = max3(mk[i & 3], sv[i >> 5][(2 * i) & 63], sv[i >> 5][(2 * i + 1) & 63]);
          const float m_tile = max3(fmaxf(mk[0], mk[1]), mk[2], mk[3]) * row_scale;
          float alpha = 1.f;
          if (m_tile > m + kRescale) {
            alpha = fast_exp2(m - m_tile);
            m = m_tile;
          }
          if (j > t0 && __any_sync(0xffffffffu, alpha != 1.f)) {
#pragma unroll 1
            for (int c = 0; c < 8; ++c) {
              uint32_t o[16];
              tmem_ld16(tO + c * 16, o);
#pragma unroll
              for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
              tmem_st16(tO + c * 16, o);
            }
          }
          const float base = m == -INFINITY ? 0.f : weight_lift - m;
          const uint64_t scale2 = f2(row_scale, row_scale), base2 = f2(base, base);
          uint64_t sum2[2] = {f2(0.f, 0.f), f2(0.f, 0.f)};
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            float* pc = sv[c >> 1] + (c & 1) * 32;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              float x0, x1;
              f2_split(f2_fma(f2(pc[2 * i], pc[2 * i + 1]), scale2, base2), x0, x1);
              pc[2 * i] = ex2_approx(x0);
              pc[2 * i + 1] = ex2_approx(x1);
              sum2[i & 1] = f2_add(sum2[i & 1], f2(pc[2 * i], pc[2 * i + 1]));
            }
            uint32_t pk[16];
            if (wide) {
#pragma unroll
              for (int i = 0; i < 16; ++i) pk[i] = Elem<__nv_bfloat16>::pack(pc[2 * i], pc[2 * i + 1]);
            } else {
#pragma unroll
              for (int i = 0; i < 16; ++i) pk[i] = Elem<__half>::pack(pc[2 * i], pc[2 * i + 1]);
            }
            tmem_st16(tS + c * 16, pk);
            if (c & 1) {
              tmem_wait_st();
              tc_fence_before_sync();
              mbar_arrive(smem_u32(c == 1 ? &sh->p_lo[x] : &sh->p_hi[x]));
            }
          }
          float s0, s1, s2, s3;
          f2_split(sum2[0], s0, s1);
          f2_split(sum2[1], s2, s3);
          l = l * alpha + ((s0 + s1) + (s2 + s3));
          if (j + 1 == end) {
            const int n = next_unit(e + 1);
            if (n < sh->count) order_q(n);
          }
        }
        if (ok && end > t0) {
          const bool got = mbar_wait(smem_u32(&sh->o_done[x]), units & 1);
          ok = __all_sync(0xffffffffu, got);
          ++units;
          tc_fence_after_sync();
        }
        if (!ok) break;
        // O leaves in order of its columns, 64 at a time through shared memory so that
        // a store writes 4 rows' whole lines and not 32 pieces; or as a record
        const float inv = l != 0.f ? 1.f / l : 0.f;
        float* rec = u.rec >= 0 ? record(p.records, u.rec, x) + t : nullptr;
        T* out = reinterpret_cast<T*>(p.out) + (int64_t)u.row0 * p.out_token_stride +
                 (int64_t)(u.kvh * p.group) * p.out_head_stride;
        uint8_t* stage = smem + kOut0 + warp * kOutBytes;
#pragma unroll 1
        for (int h = 0; h < 2; ++h) {
          float o[64];
          if (end > t0) {
            tmem_ld64(tO + h * 64, o);
          } else {
#pragma unroll
            for (int i = 0; i < 64; ++i) o[i] = 0.f;
          }
          float f[2];
#pragma unroll
          for (int g = 0; g < 2; ++g) {
            f[g] = rec ? 1.f : inv;
            if (qpos >= u.nan[2 * h + g]) f[g] = __uint_as_float(0x7fc00000u);
          }
#pragma unroll
          for (int i = 0; i < 64; ++i) o[i] *= f[i >> 5];
          if (rec) {
#pragma unroll
            for (int i = 0; i < 64; ++i) rec[(h * 64 + i) * kRows] = o[i];
            continue;
          }
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const float* v = o + 8 * k;
            *reinterpret_cast<uint4*>(stage + swz128(lane, k)) =
                make_uint4(Elem<T>::pack(v[0], v[2]), Elem<T>::pack(v[4], v[6]),
                           Elem<T>::pack(v[1], v[3]), Elem<T>::pack(v[5], v[7]));
          }
          __syncwarp();
#pragma unroll 4
          for (int i = 0; i < 32; i += 4) {
            const int sr = i + (lane >> 3), r = x * kRows + (warp & 3) * 32 + sr;
            const int tok = r * p.inv_group >> 16;
            const uint4 w = *reinterpret_cast<const uint4*>(stage + swz128(sr, lane & 7));
            if (tok < u.ntok)
              *reinterpret_cast<uint4*>(out + tok * p.out_token_stride +
                                        (r - tok * p.group) * p.out_head_stride + h * 64 +
                                        (lane & 7) * 8) = w;
          }
          __syncwarp();
        }
        if (rec) {
          rec[128 * kRows] = m - weight_lift;  // what O and l are relative to
          rec[129 * kRows] = l;
        }
      }
      if (!ok && lane == 0) give_up();
      bar_sync(1, kThreads);
    }
  } else if (warp >= kConvWarp) {
    // ----------------------------------------------------- list, converters --
    const int i0 = threadIdx.x - kListWarp * 32;
    if (warp >= kListWarp) {
      find_share(p, sh, reinterpret_cast<int*>(smem + kOut0), i0);
      bar_sync(2, 128);
    }
    // Warp m takes items m, m + 7, ..., 8 rows at a time: lane l holds the 32 codes
    // of group l / 8 of row l % 8, and writes 64 bytes of T as four chunks (no bank
    // conflicts). Its codes and scales come straight from the cache: the registers
    // are loaded for the next item as soon as this item is converted, and that
    // item's page ids one item earlier still.
    const int c = lane >> 3;
    const uint32_t code_lane = (lane & 7) * kInt4CodeBytes + c * 16;
    const uint32_t scale_lane = p.cache.num_kv_heads * p.cache.block_size * kInt4CodeBytes +
                                (lane & 7) * kInt4ScaleBytes + c * 2;
    uint32_t at[4];  // where this lane's chunks go in the first 8 rows of a tile
#pragma unroll
    for (int j = 0; j < 4; ++j)
      at[j] = sbase + (c >> 1) * kHalfBytes + swz128(lane & 7, (c & 1) * 4 + j);
    int turn = warp - kConvWarp;  // items until this warp's next
    int tiles = 0;                // of all rounds
    for (bool fresh = true;; fresh = false) {
      if (i0 == 0 && (fresh || !list_wide(sh))) list_units(p, sh, fresh);
      bar_sync(1, kThreads);
      if (sh->dead || sh->count == 0) break;
      bool ok = true;
      struct Item {
        int e = -1, t, quarter, g;  // unit (-1: none left), tile, 32 rows of it, tile of all
        bool is_v;
        int page[2], row[2];  // of its two runs of 16 tokens: page, kvh * block_size + slot
      };
      const int n_items = 2 * sh->tiles;
      int i = 0, kn = tiles, vn = tiles;
      Cursor kc, vc;
      kc.seek(sh);
      vc = kc;
      auto first_token = [&](const Item& x) { return x.t * kTokens + x.quarter * 32; };
      auto take = [&](Item& x) {  // this warp's next item, and its page ids
        x.e = -1;
        while (i < n_items && x.e < 0) {
          const bool is_v = item_is_v(i, n_items);
          Cursor& cur = is_v ? vc : kc;
          if (turn < 4) {
            x.e = cur.e;
            x.t = cur.t;
            x.quarter = turn;
            x.g = is_v ? vn : kn;
            x.is_v = is_v;
            turn += kConvs;
          }
          turn -= 4;
          cur.next(sh);
          if (is_v) ++vn; else ++kn;
          ++i;
        }
        if (x.e < 0) return;
        const Unit& u = sh->units[x.e];
        const int32_t* table = p.block_tables + (int64_t)u.seq * p.block_table_stride;
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const int tok = first_token(x) + r * kTileTokens;
          const int col = (int)(__umulhi(tok, p.div_mul) >> p.div_shift);
          // past the end any page will do: K's scores there are masked, V's scales dropped
          x.page[r] = tok >= u.seq_len ? 0 : col < p.max_blocks ? __ldg(table + col) : -1;
          x.row[r] = (u.kvh - col) * p.cache.block_size + tok;
        }
      };
      uint4 w[4];
      uint32_t bits[4];
      const uint8_t *codes, *scales;
      int bad = 0;  // runs of the loaded item outside the table or the pool
      // bits of the scales met so far in unit `met`, of keys and of this lane's value group:
      // the largest, and the smallest but 0 less one; whether any is below 2^-14
      int met = -1;
      uint32_t k_top = 0, k_low = 0, v_top = 0, v_low = 0;
      bool k_small = false, v_small = false;
      // rows 8 k + l % 8 of the item, k = 2 r and 2 r + 1: run r
      auto load = [&](const Item& x, int k) {
        if ((k & 1) == 0) {
          const int r = k >> 1;
          const bool in = (uint32_t)x.page[r] < (uint32_t)p.cache.num_blocks;
          bad = (r ? bad : 0) | (in ? 0 : 1 << r);
          const uint8_t* base = (x.is_v ? p.cache.v : p.cache.k) +
                                ((uint64_t)(uint32_t)(in ? x.page[r] : 0) * p.stride128 << 7);
          codes = base + (uint32_t)(x.row[r] * kInt4CodeBytes) + code_lane;
          scales = base + (uint32_t)(x.row[r] * kInt4ScaleBytes) + scale_lane;
        }
        // read once by this SM: past L1, of which shared memory leaves little (4 % less
        // time), and behind the conversions, not between them (1 %)
        asm volatile("ld.global.nc.L1::no_allocate.v4.b32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(w[k].x), "=r"(w[k].y), "=r"(w[k].z), "=r"(w[k].w)
                     : "l"(codes + (k & 1) * (8 * kInt4CodeBytes)));
        bits[k] = *reinterpret_cast<const uint16_t*>(scales + (k & 1) * (8 * kInt4ScaleBytes));
      };
      Item now, next;
      take(now);
      if (now.e >= 0) {
#pragma unroll
        for (int k = 0; k < 4; ++k) load(now, k);
        take(next);
      }
      while (now.e >= 0) {
        const int st = now.g & 1;
        if (now.g >= 2) {
          const bool got =
              mbar_wait(smem_u32(now.is_v ? &sh->v_empty[st] : &sh->k_empty[st]), ((now.g >> 1) - 1) & 1);
          if (!__all_sync(0xffffffffu, got)) {
            ok = false;
            break;
          }
        }
        const uint32_t tile = (now.is_v ? kV0 : kK0) + st * kTileBytes + now.quarter * (32 * 128);
        const uint32_t dst[4] = {at[0] + tile, at[1] + tile, at[2] + tile, at[3] + tile};
        if (bad) {  // rows of zeros, and a report
          if (lane == 0) report_status(p.status, B200_STATUS_PAGE_OUT_OF_RANGE);
          if (bad & 1) bits[0] = bits[1] = 0;
          if (bad & 2) bits[2] = bits[3] = 0;
        }
        const bool more = next.e >= 0;
        Unit& u = sh->units[now.e];
        const int wide = u.wide;
        if (met != now.e) {
          met = now.e;
          k_top = v_top = 0;
          k_low = v_low = 0xffffffffu;
          k_small = v_small = false;
        }
        const int tok0 = first_token(now) + (lane & 7);
        auto ends = [&](uint32_t& top, uint32_t& low) {
          top = max(max(bits[0], bits[1]), max(bits[2], bits[3]));
          low = min(min(bits[0] - 1u, bits[1] - 1u), min(bits[2] - 1u, bits[3] - 1u));
        };
        uint32_t top, low;
        ends(top, low);
        if (now.is_v) {
          if (__any_sync(0xffffffffu, top > v_top || low < v_low || tok0 + 24 >= u.seq_len)) {
            // a row past the end counts as zeros (its slot may hold anything), and so
            // does a group without a finite scale, whose token is remembered: rows
            // that see it get NaN when O leaves, rows before it do not
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              if (tok0 + k * 8 >= u.seq_len) {
                bits[k] = 0;
              } else if (bits[k] >= 0x7f80u) {
                atomicMin(&u.nan[c], tok0 + k * 8);
                bits[k] = 0;
              }
            }
            ends(top, low);
            v_top = max(v_top, octave_top<kHalf>(top));
            v_low = min(v_low, octave_low(low));
            v_small = __any_sync(0xffffffffu, v_low < 0x387fu);
            if (wide < 2 && v_top != 0) {
              const uint32_t mine = octave(v_top) | octave(v_low + 1u);
              const uint32_t all = atomicOr(&u.v_octaves[c], mine) | mine;
              if (!fp16_holds<kHalf>(v_low, v_top) || 32 - __clz(all) - __ffs(all) > kApart)
                u.wide = 1;
            }
          }
        } else if (__any_sync(0xffffffffu, top > k_top || low < k_low)) {
          // past the end slots hold anything, and a scale that is no number spoils its
          // rows in any type
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (tok0 + 8 * k < u.seq_len && bits[k] < 0x7f80u) {
              k_top = max(k_top, octave_top<kHalf>(bits[k]));
              k_low = min(k_low, octave_low(bits[k] - 1u));
            }
          k_top = __reduce_max_sync(0xffffffffu, k_top);
          k_low = __reduce_min_sync(0xffffffffu, k_low);
          k_small = k_low < 0x387fu;
          if (wide < 2 && k_top != 0) {
            const uint32_t mine = key_range(k_top) | key_range(k_low + 1u);
            const uint32_t all = atomicOr(&u.k_ranges, mine) | mine;
            // fp16 calls: keys below 2^-17 only count if all are below 2^-10
            if (!fp16_holds<kHalf>(k_low, k_top) || (kHalf && k_low < 0x36ffu && all < 1u << 14))
              u.wide = 1;
          }
        }
        auto rows = [&](auto of) {
          auto row8 = [&](auto step) {
            constexpr int k = decltype(step)::value;
            convert32<k * 1024>(of(bits[k]), w[k], dst);
          };
          row8(std::integral_constant<int, 0>());
          row8(std::integral_constant<int, 1>());
          row8(std::integral_constant<int, 2>());
          row8(std::integral_constant<int, 3>());
        };
        if (wide >= 2) {
          if (now.is_v || wide == 3) {
            rows([](uint32_t b) { return ConvertBf16(b); });
          } else {
            const int shift = key_shift(u.k_ranges);
            const float f0 = ldexpf(1.f, shift / 2), f1 = ldexpf(1.f, shift - shift / 2);
            rows([&](uint32_t b) { return ConvertHalf<true>(__uint_as_float(b << 16) * f0 * f1); });
          }
        } else if (kHalf && (now.is_v ? v_small : k_small)) {
          rows([](uint32_t b) { return ConvertHalf<true>(__uint_as_float(b << 16)); });
        } else {
          rows([](uint32_t b) { return ConvertHalf<false>(__uint_as_float(b << 16)); });
        }
        if (more) {
#pragma unroll
          for (int k = 0; k < 4; ++k) load(next, k);
        }
        // generic writes of the tile -> the MMAs' async proxy
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(now.is_v ? &sh->v_full[st] : &sh->k_full[st]));
        now = next;
        if (more) take(next);
      }
      tiles += sh->tiles;
      if (!ok && lane == 0) give_up();
      bar_sync(1, kThreads);
    }
  } else {
    // ---------------------------------------------------------------- MMAs --
    int pv0 = 0, pv1 = 0, qn0 = 0, qn1 = 0;  // tiles and units issued per Q tile
    int tiles = 0;
    while (true) {
      bar_sync(1, kThreads);
      if (sh->dead || sh->count == 0) break;
      const int n_tiles = sh->tiles;
      if (elect_one()) {
        bool ok = true;
        uint32_t idesc_s = 0;  // of the unit that S is in
        // n = -1 only begins tile 0's S
        Cursor cur, nxt;
        nxt.seek(sh);
#pragma unroll 1
        for (int n = -1; n < n_tiles && ok; ++n) {
          const int g = tiles + n;
          const bool more = n + 1 < n_tiles;
          if (n >= 0) {
            cur = nxt;
            if (more) nxt.next(sh);
          }
#pragma unroll 1
          for (int x = 0; x < 2 && ok; ++x) {
            const uint32_t acc = tmem_base + x * 256;
            if (n >= 0 && cur.t < sh->units[cur.e].lim[x]) {  // PV of tile g
              const Unit& u = sh->units[cur.e];
              const uint64_t vd = smem_desc(sbase + kV0 + (g & 1) * kTileBytes, kHalfBytes, 1024);
              const uint32_t par = (x ? pv1 : pv0) & 1;
              const uint32_t idesc_pv = f16_instr_desc(kRows, kHeadDim, u.wide >= 2, true);
              ok = mbar_wait(smem_u32(&sh->p_lo[x]), par) &&
                   mbar_wait(smem_u32(&sh->v_full[g & 1]), (g >> 1) & 1);
              if (!ok) break;
              tc_fence_after_sync();
#pragma unroll
              for (int k = 0; k < 8; ++k) {
                if (k == 4) {  // the second 64 tokens of P
                  ok = mbar_wait(smem_u32(&sh->p_hi[x]), par);
                  if (!ok) break;
                  tc_fence_after_sync();
                }
                umma_f16_ts(acc + 128, acc + k * 8, vd + k * (16 * 128 / 16), idesc_pv,
                            (cur.t > u.t0 || k > 0) ? 1u : 0u);
              }
              if (!ok) break;
              if (x) ++pv1; else ++pv0;
              if (cur.t + 1 >= min(u.t1, u.lim[x])) umma_commit(smem_u32(&sh->o_done[x]));
            }
            if (more && nxt.t < sh->units[nxt.e].lim[x]) {  // S of tile g + 1
              if (nxt.t == sh->units[nxt.e].t0) {
                idesc_s = f16_instr_desc(kRows, kTokens, sh->units[nxt.e].wide == 3, false);
                ok = mbar_wait(smem_u32(&sh->q_full[x]), (x ? qn1 : qn0) & 1);
                if (!ok) break;
                if (x) ++qn1; else ++qn0;
              }
              ok = mbar_wait(smem_u32(&sh->k_full[(g + 1) & 1]), ((g + 1) >> 1) & 1);
              if (!ok) break;
              const uint64_t qd = smem_desc(sbase + kQ0 + x * kTileBytes, 16, 1024);
              const uint64_t kd = smem_desc(sbase + kK0 + ((g + 1) & 1) * kTileBytes, 16, 1024);
#pragma unroll
              for (int k = 0; k < 8; ++k) {
                const int off = ((k >> 2) * kHalfBytes + (k & 3) * 32) / 16;
                umma_f16(acc, qd + off, kd + off, idesc_s, k > 0 ? 1u : 0u);
              }
              umma_commit(smem_u32(&sh->s_full[x]));
            }
          }
          if (!ok) break;
          if (n >= 0) umma_commit(smem_u32(&sh->v_empty[g & 1]));       // every PV of tile g
          if (more) umma_commit(smem_u32(&sh->k_empty[(g + 1) & 1]));   // every S of g + 1
        }
        if (!ok) give_up();
      }
      tiles += n_tiles;
      __syncwarp();
      bar_sync(1, kThreads);
    }
    // every MMA issued has completed before TMEM is freed
    if (elect_one()) {  // the lane that issued them
      umma_commit(smem_u32(&sh->drain));
      mbar_wait(smem_u32(&sh->drain), 0);
    }
    __syncwarp();
  }
  tc_fence_before_sync();
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after_sync();
    tmem_dealloc(tmem_base, 512);
  }
}

// Joins the parts of the unit that CTA blockIdx.x began and did not end, in
// part order; block y takes 16 columns of Q tile y / 8, a thread a row. It reads
// what the parts wrote, 66 KB for each Q tile of each, from L2; two parts at a
// time are in flight and few registers used, so that the blocks of a whole batch
// of cuts (148 x 16) are resident in two rounds.
constexpr int kJoinColumns = 16, kJoinParts = 2;
template <typename T>
__global__ void __launch_bounds__(kRows) int4_prefill_join_kernel(const Int4PrefillParams p) {
  pdl_wait();
  const int4 join = p.joins[blockIdx.x];
  const int parts = join.x;
  constexpr int kBlocks = kHeadDim / kJoinColumns;
  const int x = blockIdx.y / kBlocks, c0 = blockIdx.y % kBlocks * kJoinColumns, t = threadIdx.x;
  const int tl = (x * kRows + t) / p.group;
  if (parts == 0 || tl >= join.z) return;
  float top = -INFINITY, l = 0.f, o[kJoinColumns];
#pragma unroll
  for (int i = 0; i < kJoinColumns; ++i) o[i] = 0.f;
  for (int k0 = 0; k0 < parts; k0 += kJoinParts) {
    float v[kJoinParts][kJoinColumns], m[kJoinParts], lk[kJoinParts];
#pragma unroll
    for (int u = 0; u < kJoinParts; ++u) {
      m[u] = -INFINITY;
      lk[u] = 0.f;
      const int k = k0 + u;
      if (k < parts) {
        // part 0 is this CTA's second record, the others the next CTAs' first
        const float* r = record(p.records, 2 * (blockIdx.x + k) + (k == 0 ? 1 : 0), x) + t;
        m[u] = r[128 * kRows];
        lk[u] = r[129 * kRows];
#pragma unroll
        for (int i = 0; i < kJoinColumns; ++i) v[u][i] = r[(c0 + i) * kRows];
      }
    }
    const float next = fmaxf(top, fmaxf(m[0], m[1]));
    if (next > top) {
      const float f = fast_exp2(top - next);
      l *= f;
#pragma unroll
      for (int i = 0; i < kJoinColumns; ++i) o[i] *= f;
      top = next;
    }
#pragma unroll
    for (int u = 0; u < kJoinParts; ++u) {
      if (lk[u] == 0.f) continue;  // the part sees nothing (NaN is not 0)
      const float f = fast_exp2(m[u] - top);
      l += f * lk[u];
#pragma unroll
      for (int i = 0; i < kJoinColumns; ++i) o[i] += f * v[u][i];
    }
  }
  const float inv = l != 0.f ? 1.f / l : 0.f;
  T* row = reinterpret_cast<T*>(p.out) + (int64_t)(join.y + tl) * p.out_token_stride +
           (int64_t)(join.w * p.group + x * kRows + t - tl * p.group) * p.out_head_stride + c0;
#pragma unroll
  for (int i = 0; i < kJoinColumns; ++i) o[i] *= inv;
#pragma unroll
  for (int i = 0; i < kJoinColumns; i += 8)
    *reinterpret_cast<uint4*>(row + i) =
        make_uint4(Elem<T>::pack(o[i], o[i + 2]), Elem<T>::pack(o[i + 4], o[i + 6]),
                   Elem<T>::pack(o[i + 1], o[i + 3]), Elem<T>::pack(o[i + 5], o[i + 7]));
}

template <typename T>
cudaError_t launch_typed(const Int4PrefillParams& p, cudaStream_t stream) {
  auto kernel = int4_prefill_kernel<T>;
  cudaError_t e = ensure_smem_attr(reinterpret_cast<const void*>(kernel), kSmemBytes);
  if (e != cudaSuccess) return e;
  kernel<<<p.num_ctas, kThreads, kSmemBytes, stream>>>(p);
  if ((e = cudaGetLastError()) != cudaSuccess || p.records == nullptr) return e;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(p.num_ctas, 2 * kHeadDim / kJoinColumns);
  cfg.blockDim = dim3(kRows);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, int4_prefill_join_kernel<T>, p);
}

}  // namespace

cudaError_t launch_paged_prefill_int4(const Int4PrefillParams& p, int dtype, cudaStream_t stream) {
  return dtype == B200_DTYPE_BFLOAT16 ? launch_typed<__nv_bfloat16>(p, stream)
                                      : launch_typed<__half>(p, stream);
}

}  // namespace b200
