// paged_decode_int4.cu — paged GQA decode attention over a 4-bit KV cache.
//
//   out[b, h] = sum_t p_t V'_t,  p = softmax_t(scale q[b, h] . K'_t),  t < len_b
// where K'_t and V'_t stand for s (c - 8) per group of 32 (kv_int4.cuh).
//
// Mathematics. Neither K' nor V' is ever formed: with g the groups of head_dim,
//   score_t = sum_g ks_g(t) (sum_{d in g} c_d q_d - 8 sum_{d in g} q_d)
//   O_d     = sum_t w_t c_d(t) - 8 sum_t w_t,   w_t = p_t vs_g(t), g the group of d
// so the matrix instructions multiply the codes themselves. A code in the low
// bits of a 16-bit lane IS the fp16 subnormal c 2^-24, in the next four bits
// c 2^-20, and a whole byte is (c + 16 c') 2^-24: a mask per two values makes an
// operand, no conversion. For K the odd nibbles' factor of 16 is taken out of q
// beforehand; for V the rows of bytes are taken apart at the end, as o' = (O of
// bytes - O of low nibbles) / 16. The 2^-24 goes into the softmax scale.
// Products and sums are fp32. -8 sum_g ks_g sum q is one bf16 MMA over (group,
// digit): the scales are bf16 as they are, the four sums of q are split into
// three bf16 digits. 8 sum w adds up the weights as they were rounded, by additions
// of fp16 to fp32. Roundings to 16 bits: q (exact: each head is scaled to [2^14,
// 2^15) by a power of two first) and the weights w (fp16, 2^-11). The weights are
// kept in fp16's range by a power of two of each (head, group), which follows the
// largest w seen, so that neither another group's scales nor a token that the head
// hardly sees cost it bits; the softmax's maximum follows the scores alone. (One
// power of two for a warp, over the scales, lost a group whose scales lay 2^24 below
// another's. The multiplications and the check cost 1 to 6 %: 128 to 8192 tokens of
// 124 sequences 142.4 to 144.1 us, one head of 512 rows 77.8 to 82.4.)
//
// Work split: the batch's 32-token tiles, in the order (sequence, KV head, tile),
// are dealt to the CTAs in equal consecutive shares, whatever the sequences'
// lengths: a share is a run of segments, each the whole of a (sequence, KV
// head) or a part of it. Parts are joined by a second kernel. (One CTA per
// partition of a sequence left SMs idle in the last wave and waited 3 to 4 us at
// its start: 4 x 32768 tokens of 8 KV heads 44.5 us against 34.9, one head of 512
// rows of 1024 to 8192 tokens 86.6 us against 77.4, at the time.) Short sequences that one wave of
// CTAs takes whole are not cut and not joined. The 4 warps take a quarter of a
// segment each, with its own ring of two stages (2 KiB of K codes, 2 KiB of V
// codes, 256 bytes of K and of V scales) that it fills itself with 16-byte
// asynchronous copies: nine instructions a tile, all lanes on consecutive bytes.
// (TMA boxes, of which a tile of 16-token pages takes eight, cost 180 more
// instructions a tile: 284 against 218 us on 256 x 4096 tokens at the time.) Codes
// land swizzled, 16-byte chunk c of row r at chunk c ^ ((r >> 1) & 3), for ldmatrix
// without bank conflicts. The KV tile is the A operand (M = 16 tokens, or 16 values
// of d), up to 8 heads of the GQA group are the columns; larger groups are two
// units that read the same tiles. A K row's 16-byte chunk and a V chunk's 8 columns
// of 16 bits are both one scale group.
//
// What bounds it is the chain of a tile, not HBM and no single pipe: time times the
// SM clock stays the same while the clock varies (256 x 4096 tokens, 32/8 heads: 215 to
// 218 us at 1965 MHz, 240 at 1732 under the power cap, 242 cycles a tile and SM both
// times), so memory does not set the pace, at 0.77 to 0.86 of its measured rate; and
// of the issue slots 54 % are used, of the MMA pipe 30 %. A warp spends 487
// instructions on a tile of 4608 bytes (231 of them on the ALU pipe), and with three
// warps a scheduler 4.7 cycles pass between two of a warp's: 1.1 on fixed latencies, 0.7
// not chosen, 0.7 on memory, 0.6 on busy pipes, 0.3 on shared memory. 64 x 4096: 63.4 us,
// 4.8 TB/s; one head of 512 rows 82.9 us, 4.1 TB/s (both 1965 MHz; 581 instructions a
// tile with 8 heads). Tried and not kept: four CTAs per SM (registers spill: 70 against
// 65 us), a third stage (64.4 against 61.6), e4m3 operands for K (their MMAs are taken
// apart into fp16 ones: 69).
#include <cuda_runtime.h>
#include <math.h>

#include <type_traits>

#include "common.cuh"
#include "kv_int4.cuh"
#include "paged_decode.cuh"

namespace b200 {
namespace {

constexpr int kWarps = 4;
constexpr int kTile = 32;                        // tokens of a tile
constexpr int kCodeTile = kTile * kInt4CodeBytes;    // 2 KiB
constexpr int kScaleTile = kTile * kInt4ScaleBytes;  // 256 B
constexpr int kVCodes = kCodeTile, kKScales = 2 * kCodeTile, kVScales = kKScales + kScaleTile;
constexpr int kStageBytes = 2 * (kCodeTile + kScaleTile);
constexpr int kTableTiles = 16;  // tiles whose places a warp looks up at once
constexpr int kCtasPerSm = 3;
// Shared memory by blocks of 4 heads: rings | tables | merge area (sums, then rows
// of O^T per warp) | q's B operands (per group of d, lane by lane).
template <int kBlocks>
struct Layout {
  static constexpr int kHeads = 4 * kBlocks;
  static constexpr int kTable = kWarps * 2 * kStageBytes;
  static constexpr int kMerge = kTable + kWarps * 2 * kTableTiles * 16;
  static constexpr int kQuery = kMerge + kWarps * (2 * kHeads + kHeads * kMergeStride) * 4;
  static constexpr int kBytes = kQuery + 4 * 32 * 16;
  static_assert(kCtasPerSm * (kBytes + 1024 + 192) <= 228 * 1024, "CTAs per SM");
};
// Places in a cache tensor are counted in units of 128 bytes: a tile's codes and
// scales start at such, and 32 bits reach 512 GiB.
constexpr int kPlaceUnit = 128;
constexpr uint32_t kNoPlace = 0xffffffffu;
// A CTA takes at least so many tiles: fewer, and joining the parts costs more.
constexpr int kMinTiles = 4;
// Sequences of up to so many tiles are not cut where one wave of CTAs holds them.
// us, whole and cut, with 16/8 heads: 1 x 512 tokens 6.0 and 7.6, 1 x 1024 8.3 and 7.8,
// 1 x 2048 12.8 and 8.7; 24 x 512 7.7 and 13.5, 24 x 1024 11.0 and 15.8, 24 x 2048 18.7
// and 20.6; 55 x 1 to 2048 21 and 44. So one sequence could go whole to 768 tokens, and
// many to 2048 and past it; the edge stands where whole is the faster for all.
constexpr int kWholeTiles = 16;

// Weights of a (head, group) may grow past kMostWeight before their power of two is
// lowered; the largest one is about 2^kHeadroom when it is, so fp16's normal range
// reaches 2^-14 / 2^kHeadroom below it.
constexpr int kHeadroom = 6;
constexpr uint32_t kMostWeight = 0x78007800;  // 2^15 twice, in fp16
constexpr int kMostLift = 126;                // of the power of two
// The softmax's base moves before a lane's sum of a tile passes this (fp32 holds
// them all, so it moves for the first tile and hardly ever again).
constexpr float kMostSum = 1152921504606846976.f;  // 2^60

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                        uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, "
      "{%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// The same from zero.
__device__ __forceinline__ void mma_f16_first(float (&d)[4], uint32_t a0, uint32_t a1,
                                              uint32_t a2, uint32_t a3, uint32_t b0,
                                              uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, "
      "{%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ void mma_bf16_first(float (&d)[4], uint32_t a0, uint32_t a1,
                                               uint32_t a2, uint32_t a3, uint32_t b0,
                                               uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, "
      "{%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}

// 16 bytes from global to shared memory (`bytes` 0 writes zeros and reads nothing).
template <int kTo, int kFrom>
__device__ __forceinline__ void copy16(uint32_t dst, const uint8_t* src) {
  asm volatile("cp.async.cg.shared.global [%0 + %1], [%2 + %3], 16;" ::"r"(dst), "n"(kTo), "l"(src),
               "n"(kFrom)
               : "memory");
}
__device__ __forceinline__ void copy16(uint32_t dst, const uint8_t* src, uint32_t bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes)
               : "memory");
}
__device__ __forceinline__ const uint8_t* place(const uint8_t* base, uint32_t at) {
  return base + static_cast<uint64_t>(at) * kPlaceUnit;
}
__device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// sum += the low or high half of a pair of fp16 (one mixed-precision addition)
__device__ __forceinline__ void add_low(float& sum, uint32_t pair) {
  asm("{\n .reg .b16 l, h;\n mov.b32 {l, h}, %1;\n add.rn.f32.f16 %0, l, %0;\n}" : "+f"(sum) : "r"(pair));
}
__device__ __forceinline__ void add_high(float& sum, uint32_t pair) {
  asm("{\n .reg .b16 l, h;\n mov.b32 {l, h}, %1;\n add.rn.f32.f16 %0, h, %0;\n}" : "+f"(sum) : "r"(pair));
}

__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

template <int kOffset>
__device__ __forceinline__ uint2 lds64(uint32_t addr) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2 + %3];" : "=r"(v.x), "=r"(v.y) : "r"(addr), "n"(kOffset));
  return v;
}
template <int kOffset>
__device__ __forceinline__ uint4 lds128(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4 + %5];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr), "n"(kOffset));
  return v;
}
template <int kOffset>
__device__ __forceinline__ uint32_t lds32(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1 + %2];" : "=r"(v) : "r"(addr), "n"(kOffset));
  return v;
}
template <int kOffset>
__device__ __forceinline__ void load_k(uint32_t addr, uint32_t* r) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4 + %5];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr), "n"(kOffset));
}
template <int kOffset>
__device__ __forceinline__ void load_v(uint32_t addr, uint32_t* r) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4 + %5];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr), "n"(kOffset));
}

// Bytes 0 and 2, or 1 and 3, of a word as two fp16 subnormals (c + 16 c') 2^-24,
// and the low nibbles of such a pair.
__device__ __forceinline__ uint32_t low_bytes(uint32_t w) { return w & 0x00ff00ffu; }
__device__ __forceinline__ uint32_t high_bytes(uint32_t w) { return __byte_perm(w, 0, 0x4341); }
__device__ __forceinline__ uint32_t even_codes(uint32_t w) { return w & 0x000f000fu; }
__device__ __forceinline__ uint32_t odd_codes(uint32_t w) { return w & 0x00f000f0u; }
// high nibbles of a pair of bytes, by an exact subtraction: it goes to another
// pipe than the masks, of which this kernel has the most
__device__ __forceinline__ uint32_t rest_codes(uint32_t bytes, uint32_t even) {
  uint32_t r;
  asm("sub.f16x2 %0, %1, %2;" : "=r"(r) : "r"(bytes), "r"(even));
  return r;
}
// 2^n; 0 below the normal range.
__device__ __forceinline__ float pow2(int n) {
  return n < -126 ? 0.f : __uint_as_float(static_cast<uint32_t>(min(n, 127) + 127) << 23);
}
__device__ __forceinline__ float lo_scale(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float hi_scale(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }

template <typename T>
__device__ __forceinline__ float2 widen(uint32_t w);
template <>
__device__ __forceinline__ float2 widen<__nv_bfloat16>(uint32_t w) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <>
__device__ __forceinline__ float2 widen<__half>(uint32_t w) {
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}

// One run of tiles of a (sequence, unit).
struct Segment {
  int b, unit;     // unit: KV head, or half of its q heads
  int len;         // tokens of the sequence
  int begin, end;  // tiles
};

__device__ __forceinline__ int tiles_of(int len) { return (max(len, 0) + kTile - 1) / kTile; }

// The segment after `s` in a share with `left` tiles to go after it; left 0: none.
__device__ __forceinline__ void next_segment(const Int4DecodeParams& p, Segment& s, int left) {
  if (left <= 0) return;
  if (++s.unit == p.num_units) {
    s.unit = 0;
    do s.len = p.seq_lens[++s.b];
    while (s.len <= 0);
  }
  s.begin = 0;
  s.end = min(tiles_of(s.len), left);
}

// kBlocks: blocks of 4 heads. Column 2i of the MMAs is head i, column 2i + 1 head 4 +
// i, so lane tq has the scores of heads tq and 4 + tq; with one block it is 0.
template <typename T, int kBlocks>
__global__ void __launch_bounds__(kWarps * 32, kCtasPerSm)
    paged_decode_int4_kernel(const Int4DecodeParams p) {
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int scan[kWarps];
  __shared__ Segment start;
  using L = Layout<kBlocks>;
  constexpr int kHeads = L::kHeads;

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  // per 16 tokens of this warp's next tiles: the places of their codes and scales,
  // in two runs of up to 16 tiles, the one in use and the one after it
  uint2* table = reinterpret_cast<uint2*>(smem + L::kTable) + warp * kTableTiles * 4;

  // Launched as a programmatic dependent of the append (or whatever ran
  // before): nothing that kernel may have written is read above this line, and
  // nothing of it by the read-only path below.
  pdl_wait();

  // ---- this CTA's share [t0, t1) of the tiles, and the segment it starts in ----
  int64_t t0 = 0, t1, total;
  int ctas = 1;
  if (p.whole) {  // a CTA for each (sequence, unit)
    Segment s;
    s.b = static_cast<int>(blockIdx.x / static_cast<unsigned>(p.num_units));
    s.unit = static_cast<int>(blockIdx.x - (unsigned)s.b * (unsigned)p.num_units);
    s.len = p.seq_lens[s.b];
    s.begin = 0;
    s.end = tiles_of(s.len);
    t1 = total = s.end;
    if (threadIdx.x == 0) start = s;
    __syncthreads();
  } else {
    const int per = (p.num_seqs + kWarps * 32 - 1) / (kWarps * 32);
    const int first = threadIdx.x * per, last = min(first + per, p.num_seqs);
    int sum = 0;
    for (int i = first; i < last; ++i) sum += tiles_of(p.seq_lens[i]);
    int incl = sum;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, incl, d);
      if (lane >= d) incl += v;
    }
    if (lane == 31) scan[warp] = incl;
    __syncthreads();
    int before = incl - sum, all = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      before += w < warp ? scan[w] : 0;
      all += scan[w];
    }
    total = (int64_t)all * p.num_units;
    const int64_t worth = max(total / kMinTiles, (int64_t)1);
    ctas = static_cast<int>(min((int64_t)p.num_parts, worth));
    if (blockIdx.x >= ctas || total == 0) return;
    t0 = blockIdx.x * total / ctas;
    t1 = (blockIdx.x + 1) * total / ctas;
    int64_t at = (int64_t)before * p.num_units;
    if (t0 >= at && t0 < at + (int64_t)sum * p.num_units) {
      Segment s;
      for (s.b = first;; ++s.b) {
        s.len = p.seq_lens[s.b];
        const int64_t n = (int64_t)tiles_of(s.len) * p.num_units;
        if (t0 < at + n) break;
        at += n;
      }
      const int n = tiles_of(s.len), r = static_cast<int>(t0 - at);
      s.unit = r / n;
      s.begin = r - s.unit * n;
      s.end = static_cast<int>(min((int64_t)n, s.begin + (t1 - t0)));
      start = s;
    }
    __syncthreads();
  }
  Segment seg = start;
  if (p.whole && seg.len <= 0) {  // no tokens: zeros
    const int kvh = seg.unit / p.splits;
    const int head0 = kvh * p.group + (seg.unit - kvh * p.splits) * p.heads;
    const int heads = min(p.heads, (kvh + 1) * p.group - head0);
    T* ob = static_cast<T*>(p.out) + (int64_t)seg.b * p.out_seq_stride +
            (int64_t)head0 * p.out_head_stride;
    for (int i = threadIdx.x; i < heads * kHeadDim; i += blockDim.x)
      ob[(i >> 7) * p.out_head_stride + (i & 127)] = Elem<T>::from_float(0.f);
    return;
  }
  int left = static_cast<int>(t1 - t0) - (seg.end - seg.begin);  // tiles after this segment

  const int gr = lane >> 2;
  const int tq = lane & 3;
  const uint32_t ring = smem_u32(smem) + warp * 2 * kStageBytes;
  // this lane's 16 bytes of a copy of 8 rows of codes, and of the copy of the scales
  const uint32_t copy_to = ring + gr * 64 + ((tq ^ ((gr >> 1) & 3)) << 4);
  const uint8_t* k_from = p.cache.k + lane * 16;
  const uint8_t* v_from = p.cache.v + lane * 16;
  const uint8_t* s_from = (lane < 16 ? p.cache.k : p.cache.v) + (lane & 7) * 16;

  // q of the first segment: its loads run beside the tables'
  uint32_t qw[16];
  auto load_q = [&]() {
    const int kvh = seg.unit / p.splits;
    const int head0 = kvh * p.group + (seg.unit - kvh * p.splits) * p.heads;
    const int heads = min(p.heads, (kvh + 1) * p.group - head0);
    const int h = (gr & 1) * 4 + (gr >> 1);
    const bool mine = h < heads;
    const T* qb = static_cast<const T*>(p.q) + (int64_t)seg.b * p.q_seq_stride +
                  (int64_t)(head0 + (mine ? h : 0)) * p.q_head_stride + tq * 8;
#pragma unroll
    for (int i = 0; i < 16; ++i)
      qw[i] = mine ? *reinterpret_cast<const uint32_t*>(qb + (i >> 2) * 32 + (i & 3) * 2) : 0u;
  };
  load_q();

  // ---- the warp's runs of tiles: up to 16 of one segment ----
  Segment far = seg;  // of the next run
  int far_left = left;
  int fx = far.begin + (far.end - far.begin) * warp / kWarps;
  int fe = far.begin + (far.end - far.begin) * (warp + 1) / kWarps;

  // Looks up the next run and leaves its places in half `h` of the table; where
  // there is none, the place of any bytes of the pool (fetched, never used). True:
  // some page of the run is none of the pool's.
  auto look_up = [&](int h) {
    while (fx >= fe && far_left > 0) {
      next_segment(p, far, far_left);
      far_left -= far.end - far.begin;
      fx = far.begin + (far.end - far.begin) * warp / kWarps;
      fe = far.begin + (far.end - far.begin) * (warp + 1) / kWarps;
    }
    const int n = max(min(fe - fx, kTableTiles), 0);
    const int tok = (fx * 2 + lane) * 16;
    fx += n;
    uint2 at = make_uint2(0, 0);  // past the end too
    bool none = false;
    if (lane < n * 2 && tok < far.len) {
      const int kvh = far.unit / p.splits;
      const int col = tok / p.block_size;
      const int64_t row = (int64_t)kvh * p.block_size + (tok - col * p.block_size);
      const int page = col < p.max_blocks
                           ? p.block_tables[(int64_t)far.b * p.block_table_stride + col] : -1;
      none = page < 0 || page >= p.cache.num_blocks;
      const int64_t base = page * p.cache.block_stride;
      at.x = static_cast<uint32_t>((base + row * kInt4CodeBytes) / kPlaceUnit);
      at.y = static_cast<uint32_t>((base + row * kInt4ScaleBytes +
                                    (int64_t)p.cache.num_kv_heads * p.block_size * kInt4CodeBytes) /
                                   kPlaceUnit);
      if (none) {
        report_status(p.status, B200_STATUS_PAGE_OUT_OF_RANGE);
        at = make_uint2(kNoPlace, 0);
      }
    }
    __syncwarp();
    table[h * kTableTiles * 2 + lane] = at;
    __syncwarp();
    return __any_sync(0xffffffffu, none);
  };
  // Copies the tile whose places are at `entry` into the stage at `into`.
  auto fetch = [&](uint32_t entry, uint32_t into, bool lost) {
    const uint4 at = lds128<0>(entry);
    const uint32_t to = copy_to + into;
    const uint32_t s_to = ring + into + lane * 16 + kKScales;
    const uint32_t s_at = (lane & 8) ? at.w : at.y;
    if (!lost) {
      const uint8_t* k0 = place(k_from, at.x);
      const uint8_t* v0 = place(v_from, at.x);
      const uint8_t* k1 = place(k_from, at.z);
      const uint8_t* v1 = place(v_from, at.z);
      copy16<0, 0>(to, k0);
      copy16<512, 512>(to, k0);
      copy16<1024, 0>(to, k1);
      copy16<1536, 512>(to, k1);
      copy16<kVCodes, 0>(to, v0);
      copy16<kVCodes + 512, 512>(to, v0);
      copy16<kVCodes + 1024, 0>(to, v1);
      copy16<kVCodes + 1536, 512>(to, v1);
      copy16<0, 0>(s_to, place(s_from, s_at));
    } else {  // a page that is none counts as rows of zeros
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint32_t c = i ? at.z : at.x;
        const uint32_t bytes = c == kNoPlace ? 0 : 16;
        const uint32_t from = c == kNoPlace ? 0 : c;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          copy16(to + i * 1024 + h * 512, place(k_from, from) + h * 512, bytes);
          copy16(to + kVCodes + i * 1024 + h * 512, place(v_from, from) + h * 512, bytes);
        }
      }
      copy16(s_to, place(s_from, s_at), ((lane & 8) ? at.z : at.x) == kNoPlace ? 0 : 16);
    }
  };
  const uint32_t entries = smem_u32(table);
  uint32_t half = 0;   // of the table, in use
  uint32_t stage = 0;  // byte offset of the stage in use
  bool lost = look_up(0);
  fetch(entries, 0, lost);

  // ldmatrix row addresses: matrices are (tokens 0-7 | 8-15) x (chunks 2i | 2i + 1)
  const int lrow = (lane & 7) + ((lane >> 3) & 1) * 8;
  const uint32_t load0 = ring + lrow * 64 + (((lane >> 4) ^ ((lrow >> 1) & 3)) << 4);
  const uint32_t load1 = load0 ^ 32;
  const uint32_t scales = ring + gr * 8;
  const float kNegInf = -INFINITY;
  uint4* queries = reinterpret_cast<uint4*>(smem + L::kQuery);
  const uint32_t query = smem_u32(queries + lane);
  const uint32_t first_half = (gr & 1) ? 0u : 0xffffffffu;

  while (true) {
    const int kvh = seg.unit / p.splits;
    const int head0 = kvh * p.group + (seg.unit - kvh * p.splits) * p.heads;
    const int heads = min(p.heads, (kvh + 1) * p.group - head0);

    // ---- q: B operands (k = the 8 codes of a K word, n = column), fp16 ----
    uint32_t qz[2];       // -8 2^-24 sum_{d in g} q in three bf16 digits, k = 4 digit + g
    float fac[kBlocks];   // raw score of head 4 block + tq -> log2 units
    {
      float x[4][8];
      float amax = 0.f;
#pragma unroll
      for (int g = 0; g < 4; ++g)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 v = widen<T>(qw[g * 4 + j]);
          x[g][2 * j] = v.x;
          x[g][2 * j + 1] = v.y;
          amax = fmaxf(amax, fmaxf(fabsf(v.x), fabsf(v.y)));
        }
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
      // 2^(14 - floor(log2 amax)), and back with the codes' 2^24
      const int e = max(static_cast<int>(__float_as_uint(amax) >> 23), 14);
      const float up = __uint_as_float(static_cast<uint32_t>(268 - e) << 23);
      // never 0: masked scores are -inf, and stay so
      const float down =
          fmaxf(__uint_as_float(static_cast<uint32_t>(e) << 23) * 1024.f * p.scale_log2, 1e-45f);
#pragma unroll
      for (int c = 0; c < kBlocks; ++c) fac[c] = __shfl_sync(0xffffffffu, down, tq * 8 + c * 4);
      float own[4];
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          x[g][j] *= up;
          sum += x[g][j];
        }
        // MMA k pairs: nibbles (0, 4) and (1, 5) of the word, then (2, 6) and (3, 7)
        if (warp == g)
          queries[g * 32 + lane] =
              make_uint4(Elem<__half>::pack(x[g][0], x[g][4]),
                         Elem<__half>::pack(x[g][1] * 0.0625f, x[g][5] * 0.0625f),
                         Elem<__half>::pack(x[g][2], x[g][6]),
                         Elem<__half>::pack(x[g][3] * 0.0625f, x[g][7] * 0.0625f));
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        own[g] = sum * (-8.f * 5.9604644775390625e-8f);
      }
      // lane tq: k = 2 tq, 2 tq + 1 are groups (0, 1) for even tq and (2, 3) for odd
      // tq, digit tq / 2; k + 8 the last digit, in the lanes of digit 0 only
      const float z[2] = {(tq & 1) ? own[2] : own[0], (tq & 1) ? own[3] : own[1]};
      float d0[2], d1[2], d2[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        d0[i] = __bfloat162float(__float2bfloat16_rn(z[i]));
        d1[i] = __bfloat162float(__float2bfloat16_rn(z[i] - d0[i]));
        d2[i] = z[i] - d0[i] - d1[i];
      }
      qz[0] = tq < 2 ? Elem<__nv_bfloat16>::pack(d0[0], d0[1])
                     : Elem<__nv_bfloat16>::pack(d1[0], d1[1]);
      qz[1] = tq < 2 ? Elem<__nv_bfloat16>::pack(d2[0], d2[1]) : 0u;
    }
    __syncthreads();  // the queries (and the merge area is free again)

    float base[kBlocks], l_run[kBlocks];  // base: whole numbers, so that rescaling is exact
    uint64_t lift[4];  // 2^e of each group, of the lane's heads (one head: twice the same)
#pragma unroll
    for (int c = 0; c < kBlocks; ++c) {
      base[c] = kNegInf;
      l_run[c] = 0.f;
    }
    // ws: sums of the weights by column of the lane's pair, as o has them
    float o[8][4], ws[2][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      lift[i] = f2(pow2(kMostLift), pow2(kMostLift));
      ws[0][i] = ws[1][i] = 0.f;
#pragma unroll
      for (int mt = 0; mt < 8; ++mt) o[mt][i] = 0.f;
    }
    float most = -1.f;  // the first tile sets the base and the lifts

    const int first = seg.begin + (seg.end - seg.begin) * warp / kWarps;
    const int last = seg.begin + (seg.end - seg.begin) * (warp + 1) / kWarps;
    int valid = seg.len - first * kTile;  // tokens from the tile's first one on
    bool fold = false;  // every second run of tiles
    for (int todo = last - first, n; todo > 0; todo -= n) {
      n = min(todo, kTableTiles);
      const bool lost_next = look_up(half ^ 1);
      uint32_t entry = entries + half * (kTableTiles * 16);
      half ^= 1;
      for (int i = n; i > 0; --i) {
        copy_wait();
        __syncwarp();  // the tile has landed for every lane, and every lane is done with the one before
        const uint32_t at = stage;
        stage = kStageBytes - stage;
        entry = i == 1 ? entries + half * (kTableTiles * 16) : entry + 16;
        fetch(entry, stage, i == 1 ? lost_next : lost);

        // ---- raw scores of 32 tokens: sc[block][st][token g | g + 8], head tq ----
        float sc[kBlocks][2][2];
        const uint32_t sa = scales + at;
        {
          const uint32_t za = sa + (tq & 1) * 4;
          const uint32_t z[4] = {lds32<kKScales>(za), lds32<kKScales + 64>(za),
                                 lds32<kKScales + 128>(za), lds32<kKScales + 192>(za)};
#pragma unroll
          for (int st = 0; st < 2; ++st) {
            float acc[4];
            mma_bf16_first(acc, z[2 * st], z[2 * st + 1], z[2 * st], z[2 * st + 1], qz[0], qz[1]);
#pragma unroll
            for (int blk = 0; blk < kBlocks; ++blk) {
              sc[blk][st][0] = acc[blk];
              sc[blk][st][1] = acc[2 + blk];
            }
          }
        }
        const uint2 ks[2][2] = {{lds64<kKScales>(sa), lds64<kKScales + 64>(sa)},
                                {lds64<kKScales + 128>(sa), lds64<kKScales + 192>(sa)}};
        auto keys = [&](auto part) {  // chunks 2h and 2h + 1 of the rows: two groups
          constexpr int h = decltype(part)::value;
          uint32_t kw[2][4];
          load_k<0>((h ? load1 : load0) + at, kw[0]);
          load_k<1024>((h ? load1 : load0) + at, kw[1]);
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const uint4 qf = i ? lds128<(2 * h + 1) * 512>(query) : lds128<2 * h * 512>(query);
#pragma unroll
            for (int st = 0; st < 2; ++st) {
              const uint32_t w0 = kw[st][2 * i], w1 = kw[st][2 * i + 1];
              const uint32_t v0 = high_bytes(w0), v1 = high_bytes(w1);
              const uint32_t e0 = even_codes(v0), e1 = even_codes(v1);
              float acc[4];
              mma_f16_first(acc, even_codes(w0), even_codes(w1), odd_codes(w0), odd_codes(w1), qf.x,
                            qf.y);
              mma_f16(acc, e0, e1, rest_codes(v0, e0), rest_codes(v1, e1), qf.z, qf.w);
              const uint32_t s0 = h ? ks[st][0].y : ks[st][0].x, s1 = h ? ks[st][1].y : ks[st][1].x;
              const float f0 = i ? hi_scale(s0) : lo_scale(s0);
              const float f1 = i ? hi_scale(s1) : lo_scale(s1);
#pragma unroll
              for (int blk = 0; blk < kBlocks; ++blk) {
                sc[blk][st][0] = fmaf(f0, acc[blk], sc[blk][st][0]);
                sc[blk][st][1] = fmaf(f1, acc[2 + blk], sc[blk][st][1]);
              }
            }
          }
        };
        keys(std::integral_constant<int, 0>());
        keys(std::integral_constant<int, 1>());

        // ---- value scales of this lane's tokens, masked past the end ----
        uint2 vs[2][2];
        auto load_scales = [&]() {
          vs[0][0] = lds64<kVScales>(sa);
          vs[0][1] = lds64<kVScales + 64>(sa);
          vs[1][0] = lds64<kVScales + 128>(sa);
          vs[1][1] = lds64<kVScales + 192>(sa);
          if (valid < kTile) {
            // rows past the end may be any bytes; their codes are finite whatever they
            // are, so a weight of exactly 0 needs the scale cleared
#pragma unroll
            for (int st = 0; st < 2; ++st)
#pragma unroll
              for (int i = 0; i < 2; ++i)
                if (st * 16 + i * 8 + gr >= valid) {
                  vs[st][i] = make_uint2(0, 0);
#pragma unroll
                  for (int blk = 0; blk < kBlocks; ++blk) sc[blk][st][i] = kNegInf;
                }
          }
        };
        load_scales();

        // ---- weights: p in fp32, then p vs 2^e in fp16 ----
        // wt[st][g]: tokens g and g + 8 of head tq (one block), or heads tq and 4 + tq
        // of token g, then of token g + 8
        float sum[kBlocks];
        uint32_t wt[2][4][kBlocks];
        uint32_t top;  // the larger halves of all, and kMostWeight
        auto weigh = [&]() {
          float pr[kBlocks][2][2];
#pragma unroll
          for (int blk = 0; blk < kBlocks; ++blk) {
#pragma unroll
            for (int st = 0; st < 2; ++st)
#pragma unroll
              for (int i = 0; i < 2; ++i)
                pr[blk][st][i] = ex2_approx(fmaf(sc[blk][st][i], fac[blk], -base[blk]));
            sum[blk] = (pr[blk][0][0] + pr[blk][0][1]) + (pr[blk][1][0] + pr[blk][1][1]);
          }
          top = kMostWeight;
#pragma unroll
          for (int st = 0; st < 2; ++st) {
            const uint2 v0 = vs[st][0], v1 = vs[st][1];
#pragma unroll
            for (int g = 0; g < 4; ++g) {
              const uint32_t s0 = g < 2 ? v0.x : v0.y, s1 = g < 2 ? v1.x : v1.y;
              const float f0 = (g & 1) ? hi_scale(s0) : lo_scale(s0);
              const float f1 = (g & 1) ? hi_scale(s1) : lo_scale(s1);
              float a, b;
              if constexpr (kBlocks == 1) {
                f2_split(f2_mul(f2_mul(f2(pr[0][st][0], pr[0][st][1]), f2(f0, f1)), lift[g]), a, b);
                wt[st][g][0] = Elem<__half>::pack(a, b);
              } else {
                f2_split(f2_mul(f2_mul(f2(pr[0][st][0], pr[kBlocks - 1][st][0]), f2(f0, f0)), lift[g]),
                         a, b);
                wt[st][g][0] = Elem<__half>::pack(a, b);
                f2_split(f2_mul(f2_mul(f2(pr[0][st][1], pr[kBlocks - 1][st][1]), f2(f1, f1)), lift[g]),
                         a, b);
                wt[st][g][kBlocks - 1] = Elem<__half>::pack(a, b);
              }
            }
          }
#pragma unroll
          for (int g = 0; g < 4; ++g)
#pragma unroll
            for (int c = 0; c < kBlocks; ++c) top = __vimax3_u16x2(top, wt[0][g][c], wt[1][g][c]);
        };
        weigh();
        if (__any_sync(0xffffffffu, top != kMostWeight || !(sum[0] <= most) ||
                                        !(sum[kBlocks - 1] <= most))) {
          load_scales();  // again: they are not kept for this
          // the base follows the scores alone
          int up[kBlocks];  // by how much
#pragma unroll
          for (int c = 0; c < kBlocks; ++c) {
            float m = fmaxf(fmaxf(sc[c][0][0], sc[c][0][1]), fmaxf(sc[c][1][0], sc[c][1][1])) * fac[c];
            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 4));
            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 8));
            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
            // (scores of -inf alone leave it below every score)
            const float next = fmaxf(fmaxf(base[c], floorf(m)), -3.4e38f);
            up[c] = most < 0.f ? 0 : static_cast<int>(fminf(next - base[c], 512.f));
            base[c] = next;
            l_run[c] *= pow2(-up[c]);
          }
          most = kMostSum;
          // each (head, group)'s power of two follows its largest p vs: one that stands
          // far above the rest costs them their bits only where it is all that counts. A
          // scale that is no number spoils its own group's sums and is not followed
          uint32_t high[kBlocks][2];  // exponents of p vs: groups 2 w | 2 w + 1 << 16
#pragma unroll
          for (int c = 0; c < kBlocks; ++c) {
            float x[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int st = 0; st < 2; ++st)
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                // below 2, so that a product with a finite scale is finite
                const float pr = ex2_approx(fmaf(sc[c][st][i], fac[c], -base[c]));
                x[0] = fmaxf(x[0], pr * lo_scale(vs[st][i].x));
                x[1] = fmaxf(x[1], pr * hi_scale(vs[st][i].x));
                x[2] = fmaxf(x[2], pr * lo_scale(vs[st][i].y));
                x[3] = fmaxf(x[3], pr * hi_scale(vs[st][i].y));
              }
#pragma unroll
            for (int w = 0; w < 2; ++w) {
              uint32_t e = __float_as_uint(x[2 * w]) >> 23 | (__float_as_uint(x[2 * w + 1]) >> 23) << 16;
              e = __vmaxu2(e, __shfl_xor_sync(0xffffffffu, e, 4));
              e = __vmaxu2(e, __shfl_xor_sync(0xffffffffu, e, 8));
              high[c][w] = __vmaxu2(e, __shfl_xor_sync(0xffffffffu, e, 16));
            }
          }
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            float held[2], factor[2];
            f2_split(lift[g], held[0], held[1]);
#pragma unroll
            for (int c = 0; c < kBlocks; ++c) {
              const int x = static_cast<int>(high[c][g >> 1] >> (g & 1) * 16 & 0xffffu);
              const int old = static_cast<int>(__float_as_uint(held[c]) >> 23);
              // (each + 127.) A higher base alone leaves p vs 2^e as it was; p vs < 2^(x - 126)
              int e = min(old + up[c], kMostLift + 127);
              if (e + x > 15 + 126 + 127 && x < 255) e = kHeadroom + 126 + 127 - x;
              held[c] = __uint_as_float(static_cast<uint32_t>(e) << 23);
              factor[c] = pow2(e - old - up[c]);
            }
            lift[g] = kBlocks == 1 ? f2(held[0], held[0]) : f2(held[0], held[1]);
            if (kBlocks == 1) factor[1] = factor[0];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              o[2 * g][i] *= factor[i & 1];
              o[2 * g + 1][i] *= factor[i & 1];
              if (i < 2) ws[i][g] *= factor[i];
            }
          }
          weigh();
        }
#pragma unroll
        for (int c = 0; c < kBlocks; ++c) l_run[c] += sum[c];

        // ---- O^T += V^T w^T ----
        auto values = [&](auto part) {
          constexpr int st = decltype(part)::value;
          uint32_t vw[8];
          load_v<kVCodes + st * 1024>(load0 + at, vw);
          load_v<kVCodes + st * 1024>(load1 + at, vw + 4);
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const uint32_t w0 = vw[2 * g], w1 = vw[2 * g + 1];  // tokens 0-7 | 8-15
            const uint32_t v0 = high_bytes(w0), v1 = high_bytes(w1);
            uint32_t b0, b1;
            if constexpr (kBlocks == 1) {
              // tokens g and g + 8 of head tq as columns 2 tq and 2 tq + 1: the even
              // columns sum over the first 8 tokens, the odd ones over the others
              add_low(ws[0][g], wt[st][g][0]);
              add_high(ws[1][g], wt[st][g][0]);
              const uint32_t w = movmatrix_trans(wt[st][g][0]);
              b0 = w & first_half;
              b1 = w & ~first_half;
            } else {
#pragma unroll
              for (int i = 0; i < kBlocks; ++i) {
                add_low(ws[0][g], wt[st][g][i]);
                add_high(ws[1][g], wt[st][g][i]);
              }
              b0 = movmatrix_trans(wt[st][g][0]);
              b1 = movmatrix_trans(wt[st][g][kBlocks - 1]);
            }
            mma_f16(o[2 * g], even_codes(w0), low_bytes(w0), even_codes(w1), low_bytes(w1), b0, b1);
            mma_f16(o[2 * g + 1], even_codes(v0), v0, even_codes(v1), v1, b0, b1);
          }
        };
        values(std::integral_constant<int, 0>());
        values(std::integral_constant<int, 1>());
        valid -= kTile;
      }
      lost = lost_next;
      fold = !fold;
      if (fold && todo > n) continue;

      // ---- 8 sum w off the sums of codes, 136 of them off the sums of bytes ----
      // The MMAs cut their sums off, so each adds a bias of up to 2^-23 of what it
      // holds, and most of that are these offsets: off after every 32 tiles, the bias
      // stays below 2^-16 of the values' scale whatever the length. (Off at the
      // segment's end alone, 32768 tokens of equal weights in one CTA were 0.9 % off.)
#pragma unroll
      for (int g = 0; g < 4; ++g)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float w = ws[c][g];
          ws[c][g] = 0.f;
          w += __shfl_xor_sync(0xffffffffu, w, 4);
          w += __shfl_xor_sync(0xffffffffu, w, 8);
          w += __shfl_xor_sync(0xffffffffu, w, 16);
          constexpr float kUnit = 5.9604644775390625e-8f;  // 2^-24, of a code
#pragma unroll
          for (int mt = 2 * g; mt < 2 * g + 2; ++mt) {
            o[mt][c] = fmaf(w, -8.f * kUnit, o[mt][c]);
            o[mt][2 + c] = fmaf(w, -136.f * kUnit, o[mt][2 + c]);
          }
        }
    }

    // ---- merge the warps ----
    float* ml = reinterpret_cast<float*>(smem + L::kMerge);  // [warp][base | sum]
    float* mo = ml + kWarps * 2 * kHeads;                                   // [warp][head][stride]
#pragma unroll
    for (int c = 0; c < kBlocks; ++c) {
      l_run[c] += __shfl_xor_sync(0xffffffffu, l_run[c], 4);
      l_run[c] += __shfl_xor_sync(0xffffffffu, l_run[c], 8);
      l_run[c] += __shfl_xor_sync(0xffffffffu, l_run[c], 16);
      const int head = c * 4 + tq;
      if (head < heads) {
        constexpr float kUnit = 16777216.f, kUnit16 = 1048576.f;
        float* row = &mo[(warp * kHeads + head) * kMergeStride + gr * 4];
        auto total = [&](const float (&x)[4], int i) {
          return kBlocks == 1 ? x[2 * i] + x[2 * i + 1] : x[2 * i + c];
        };
        // the warp's own result, which stays in range; scores of -inf alone have none
        const float own = l_run[c] == 0.f ? 0.f : 1.f / l_run[c];
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          float mine, other;
          f2_split(lift[g], mine, other);
          // 2^-e; a power of two, so nothing is rounded
          const float down = __uint_as_float(0x7f000000u - __float_as_uint(c ? other : mine));
          const float f = kUnit * own, f16 = kUnit16 * own;
          const float x0 = total(o[2 * g], 0), x2 = total(o[2 * g + 1], 0);
          *reinterpret_cast<float4*>(row + g * 32) =
              make_float4(x0 * f * down, (total(o[2 * g], 1) - x0) * f16 * down, x2 * f * down,
                          (total(o[2 * g + 1], 1) - x2) * f16 * down);
        }
        if (gr == 0) {
          ml[warp * 2 * kHeads + head] = base[c];
          ml[warp * 2 * kHeads + kHeads + head] = l_run[c];
        }
      }
    }
    __syncthreads();

    const int tiles = tiles_of(seg.len);
    const bool whole = seg.begin == 0 && seg.end == tiles;
    // a CTA has at most two parts: the segment it starts with and the one it ends with
    const bool starts = left + (seg.end - seg.begin) == t1 - t0;
    const int slot = blockIdx.x * 2 + (starts ? 0 : 1);
    for (int idx = threadIdx.x; idx < heads * (kHeadDim / 4); idx += blockDim.x) {
      const int head = idx >> 5;
      const int d = (idx & 31) * 4;
      float m = kNegInf, l = 0.f, f[kWarps];
#pragma unroll
      for (int w = 0; w < kWarps; ++w) m = fmaxf(m, ml[w * 2 * kHeads + head]);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float mw = ml[w * 2 * kHeads + head];
        f[w] = mw == kNegInf ? 0.f  // a warp without tiles
                             : ml[w * 2 * kHeads + kHeads + head] * fast_exp2(mw - m);
        l += f[w];
      }
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
      // a part with scores of -inf alone is nothing; a whole sequence of them has no result
      const float inv = l == 0.f && !whole ? 0.f : 1.f / l;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        if (ml[w * 2 * kHeads + head] == kNegInf) continue;
        const float fw = f[w] * inv;
        const float4 v = *reinterpret_cast<const float4*>(&mo[(w * kHeads + head) * kMergeStride + d]);
        acc.x += v.x * fw;
        acc.y += v.y * fw;
        acc.z += v.z * fw;
        acc.w += v.w * fw;
      }
      if (whole) {
        uint32_t* ob = reinterpret_cast<uint32_t*>(
            static_cast<T*>(p.out) + (int64_t)seg.b * p.out_seq_stride +
            (int64_t)(head0 + head) * p.out_head_stride + d);
        ob[0] = Elem<T>::pack(acc.x, acc.y);
        ob[1] = Elem<T>::pack(acc.z, acc.w);
      } else {
        const int64_t to = (int64_t)slot * p.heads + head;
        *reinterpret_cast<float4*>(p.part_o + to * kHeadDim + d) = acc;
        if (d == 0) p.part_lse[to] = m + log2f(l);
      }
    }
    // the CTA with the last tile knows who had the others: CTA c starts at tile
    // c * total / ctas, and has its first part in slot 2c, its last in 2c + 1
    if (threadIdx.x == 0 && seg.end == tiles && !p.whole) {
      int4 parts = make_int4(0, 0, 0, 0);
      if (!whole) {
        const int64_t from = t1 - left - seg.end;  // the first tile of this (sequence, unit)
        const int c = static_cast<int>(((from + 1) * ctas - 1) / total);
        parts = make_int4(c * 2 + (c * total / ctas == from ? 0 : 1), (c + 1) * 2,
                          blockIdx.x - c + 1, 0);
      }
      p.parts[(int64_t)seg.b * p.num_units + seg.unit] = parts;
    }
    if (left == 0) {
      copy_wait();  // the last copy, of no tile
      return;
    }
    next_segment(p, seg, left);
    left -= seg.end - seg.begin;
    load_q();
  }
}

// Joins the parts of one (sequence, q head) per CTA, where it has any: lane i of
// each warp owns 4 values, the warps take the parts in turn. parts: first slot,
// second slot (then every other one), number of parts.
template <typename T>
__global__ void __launch_bounds__(kWarps * 32) int4_join_kernel(const Int4DecodeParams p) {
  __shared__ float4 acc_s[kWarps][32];
  __shared__ float m_s[kWarps], l_s[kWarps];
  pdl_wait();
  const int b = static_cast<int>(blockIdx.x / static_cast<unsigned>(p.num_q_heads));
  const int head = static_cast<int>(blockIdx.x - (unsigned)b * (unsigned)p.num_q_heads);
  const int kvh = head / p.group, in_group = head - kvh * p.group;
  const int half = in_group / p.heads;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int4 parts = make_int4(0, 0, 0, 0);
  const bool empty = p.seq_lens[b] <= 0;
  if (!empty) parts = __ldcg(p.parts + (int64_t)b * p.num_units + kvh * p.splits + half);
  const int n = parts.z;
  if (!empty && n == 0) return;  // the whole of it is in place
  float m = -3.4e38f, l = 0.f;  // (a part with scores of -inf alone has -inf)
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  constexpr int kAtOnce = 4;  // parts in flight per warp
  for (int i0 = warp; i0 < n; i0 += kWarps * kAtOnce) {
    float lse[kAtOnce];
    float4 x[kAtOnce];
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j) {
      const int i = min(i0 + j * kWarps, n - 1);
      const int64_t at = (int64_t)(i == 0 ? parts.x : parts.y + 2 * (i - 1)) * p.heads +
                         (in_group - half * p.heads);
      lse[j] = __ldcg(p.part_lse + at);
      x[j] = __ldcg(reinterpret_cast<const float4*>(p.part_o + at * kHeadDim) + lane);
    }
    float next = m;
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j) {
      if (i0 + j * kWarps >= n) lse[j] = -INFINITY;
      next = fmaxf(next, lse[j]);
    }
    const float keep = fast_exp2(m - next);
    m = next;
    l *= keep;
    acc = make_float4(acc.x * keep, acc.y * keep, acc.z * keep, acc.w * keep);
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j) {
      const float w = fast_exp2(lse[j] - next);
      if (i0 + j * kWarps >= n) break;  // (its row is some other part's: 0 times it is not 0)
      l += w;
      acc.x += x[j].x * w;
      acc.y += x[j].y * w;
      acc.z += x[j].z * w;
      acc.w += x[j].w * w;
    }
  }
  acc_s[warp][lane] = acc;
  if (lane == 0) {
    m_s[warp] = m;
    l_s[warp] = l;
  }
  __syncthreads();
  if (warp != 0) return;
#pragma unroll
  for (int w = 1; w < kWarps; ++w) {
    if (w >= n) break;
    const float4 x = acc_s[w][lane];
    const float next = fmaxf(m, m_s[w]);
    const float keep = fast_exp2(m - next), f = fast_exp2(m_s[w] - next);
    m = next;
    l = l * keep + l_s[w] * f;
    acc.x = acc.x * keep + x.x * f;
    acc.y = acc.y * keep + x.y * f;
    acc.z = acc.z * keep + x.z * f;
    acc.w = acc.w * keep + x.w * f;
  }
  const float inv = n > 0 ? 1.f / l : 0.f;
  uint32_t* ob = reinterpret_cast<uint32_t*>(static_cast<T*>(p.out) + (int64_t)b * p.out_seq_stride +
                                             (int64_t)head * p.out_head_stride + lane * 4);
  ob[0] = Elem<T>::pack(acc.x * inv, acc.y * inv);
  ob[1] = Elem<T>::pack(acc.z * inv, acc.w * inv);
}

template <typename... Args>
cudaError_t launch_dependent(void (*kernel)(Args...), unsigned grid, int smem, cudaStream_t stream,
                             Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(kWarps * 32);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

template <typename T>
cudaError_t launch_typed(const Int4DecodeParams& p, cudaStream_t stream) {
  const bool two = p.heads > 4;
  auto kernel = two ? paged_decode_int4_kernel<T, 2> : paged_decode_int4_kernel<T, 1>;
  const int smem = two ? Layout<2>::kBytes : Layout<1>::kBytes;
  cudaError_t e = ensure_smem_attr(reinterpret_cast<const void*>(kernel), smem);
  if (e != cudaSuccess) return e;
  const unsigned grid = (unsigned)(p.whole ? p.num_seqs * p.num_units : p.num_parts);
  e = launch_dependent(kernel, grid, smem, stream, p);
  if (e != cudaSuccess || p.whole) return e;
  return launch_dependent(int4_join_kernel<T>, (unsigned)p.num_seqs * (unsigned)p.num_q_heads, 0,
                          stream, p);
}

}  // namespace

// Short sequences that one wave of CTAs takes whole: no joining, and a CTA's
// start does not wait for every length.
bool int4_decode_whole(int64_t units, int64_t max_tiles, int sms) {
  return units <= (int64_t)sms * kCtasPerSm && max_tiles <= kWholeTiles;
}

int64_t int4_decode_ctas(int64_t tiles, int sms) {
  const int64_t most = (int64_t)sms * kCtasPerSm, worth = tiles / kMinTiles;
  return worth < 1 ? 1 : worth < most ? worth : most;
}

cudaError_t launch_paged_decode_int4(const Int4DecodeParams& p, int dtype, cudaStream_t stream) {
  if ((int64_t)p.num_seqs * p.num_q_heads > 0x7fffffff ||
      (int64_t)p.num_seqs * p.num_units > 0x7fffffff)
    return cudaErrorInvalidConfiguration;
  return dtype == B200_DTYPE_BFLOAT16 ? launch_typed<__nv_bfloat16>(p, stream)
                                      : launch_typed<__half>(p, stream);
}

}  // namespace b200
