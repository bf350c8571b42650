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
// c 2^-20: one AND per two values makes an operand, no conversion. The odd
// nibbles' factor of 16 is taken out of q beforehand, and out of O's rows
// afterwards; the 2^-24 goes into the softmax scale. Products and sums are
// fp32. -8 sum_g ks_g sum q is one bf16 MMA over (group, digit): the scales are
// bf16 as they are, the four sums of q are split into three bf16 digits. 8 sum
// w comes from one MMA per group whose A operand is the constant 8, so both
// sums see the same rounded weights. Roundings to 16 bits: q (exact: each head is
// scaled to [2^14, 2^15) by a power of two first) and the weights w (fp16,
// 2^-11). The weights' range is kept in fp16 by a running power of two over
// the value scales, which takes part in the softmax's running maximum.
//
// Work split: one CTA per (sequence, KV head, KV partition), its 4 warps take
// the partition's 32-token tiles in turn, each with its own ring of stages (2
// KiB of K codes, 2 KiB of V codes, 256 bytes of K and of V scales) that it
// fills itself with 16-byte asynchronous copies: nine instructions a tile, all
// lanes on consecutive bytes. (TMA boxes, of which a tile of 16-token pages
// takes eight, cost more issue slots than they saved: 295 us against XX.) Codes
// land swizzled, 16-byte chunk c of row r at chunk c ^ ((r >> 1) & 3), for
// ldmatrix without bank conflicts. The KV tile is the A operand (M = 16 tokens,
// or 16 values of d), the GQA group's heads are the columns. A K row's 16-byte
// chunk and a V chunk's 8 columns of 16 bits are both one scale group.
#include <cuda_runtime.h>
#include <math.h>

#include "common.cuh"
#include "kv_int4.cuh"
#include "paged_decode.cuh"

namespace b200 {
namespace {

constexpr int kWarps = 4;
constexpr int kTile = 32;                        // tokens of a tile
constexpr int kStages = 2;
constexpr int kCodeTile = kTile * kInt4CodeBytes;    // 2 KiB
constexpr int kScaleTile = kTile * kInt4ScaleBytes;  // 256 B
constexpr int kVCodes = kCodeTile, kKScales = 2 * kCodeTile, kVScales = kKScales + kScaleTile;
constexpr int kStageBytes = 2 * (kCodeTile + kScaleTile);
constexpr int kRingBytes = kWarps * kStages * kStageBytes;
constexpr int kMaxSubTiles = kMaxPartTokens / 16 + 1;  // a partition may end in half a tile
constexpr int kSmemBytes = kRingBytes + kMaxSubTiles * 16;
static_assert(kWarps * (32 + 16 * kMergeStride) * 4 <= kRingBytes, "merge area in the ring");

// Scores may exceed the running maximum by 2^kSlack before O is rescaled; a
// weight is then at most 2^(kSlack + kHead) and fp16's normal range still
// reaches 2^-14 / 2^kHead below the largest one.
constexpr float kSlack = 8.f;
constexpr float kHeadroom = 6.f;
constexpr int kMinScaleExp = 36;  // value scales below 2^-91 are not followed

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

// 16 bytes from global to shared memory; `bytes` 0 writes zeros and reads nothing.
__device__ __forceinline__ void copy16(uint32_t dst, const uint8_t* src, uint32_t bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes)
               : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kPending>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(kPending) : "memory");
}

__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

__device__ __forceinline__ uint2 lds64(uint32_t addr) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr));
  return v;
}

// Nibbles 0 and 4 (even = true) or 1 and 5 of a word as two fp16 subnormals.
__device__ __forceinline__ uint32_t even_codes(uint32_t w) { return w & 0x000f000fu; }
__device__ __forceinline__ uint32_t odd_codes(uint32_t w) { return w & 0x00f000f0u; }
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

// NT: 8-head column tiles (2 for groups of more than 8 q heads).
template <typename T, int NT>
__global__ void __launch_bounds__(kWarps * 32, NT == 1 ? 4 : 3)
    paged_decode_int4_kernel(const Int4DecodeParams p) {
  extern __shared__ __align__(128) uint8_t smem[];
  // per 16 tokens of the partition: byte offsets of their codes and of their
  // scales in a cache tensor; codes < 0: no such page, or past the end
  longlong2* subtiles = reinterpret_cast<longlong2*>(smem + kRingBytes);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const unsigned parts = static_cast<unsigned>(p.num_parts);
  const unsigned unit = blockIdx.x / parts;
  const int part = static_cast<int>(blockIdx.x - unit * parts);
  const int b = static_cast<int>(unit / static_cast<unsigned>(p.num_kv_heads));
  const int kvh = static_cast<int>(unit - (unsigned)b * (unsigned)p.num_kv_heads);

  // Launched as a programmatic dependent of the append (or whatever ran
  // before): nothing that kernel may have written is read above this line.
  pdl_wait();

  const int seq_len = __ldg(p.seq_lens + b);
  const int tok_begin = part * p.part_tokens;
  const int tokens = min(seq_len - tok_begin, p.part_tokens);
  {
    const int32_t* bt = p.block_tables + (int64_t)b * p.block_table_stride;
    for (int i = threadIdx.x; i <= p.part_tokens / 16; i += blockDim.x) {
      const int tok = tok_begin + i * 16;
      const int col = tok / p.block_size;
      const int row = kvh * p.block_size + (tok - col * p.block_size);
      const int page = col < p.max_blocks ? __ldg(bt + col) : -1;
      longlong2 at = make_longlong2(-1, 0);
      if (i * 16 < tokens) {
        if (page >= 0 && page < p.cache.num_blocks) {
          at.x = page * p.cache.block_stride;
          at.y = at.x + (int64_t)p.num_kv_heads * p.block_size * kInt4CodeBytes +
                 row * kInt4ScaleBytes;
          at.x += row * kInt4CodeBytes;
        } else {
          report_status(p.status, B200_STATUS_PAGE_OUT_OF_RANGE);
        }
      }
      subtiles[i] = at;
    }
  }
  if (tokens <= 0) {
    // partitions past the end are ignored by the reduce; a sequence without
    // tokens gives zeros
    if (part == 0 && p.num_parts == 1) {
      T* ob = static_cast<T*>(p.out) + (int64_t)b * p.out_seq_stride +
              (int64_t)(kvh * p.group) * p.out_head_stride;
      for (int i = threadIdx.x; i < p.group * kHeadDim; i += blockDim.x)
        ob[(i >> 7) * p.out_head_stride + (i & 127)] = Elem<T>::from_float(0.f);
    }
    return;
  }
  if (part == p.num_parts - 1 && seq_len - tok_begin > p.part_tokens && threadIdx.x == 0)
    report_status(p.status, B200_STATUS_PLAN_EXCEEDED);
  const int ntiles = (tokens + kTile - 1) / kTile;
  const int my_tiles = ntiles > warp ? (ntiles - warp + kWarps - 1) / kWarps : 0;

  const int gr = lane >> 2;
  const int tq = lane & 3;
  const uint32_t ring = smem_u32(smem) + warp * kStages * kStageBytes;
  // this lane's place in a copy of 8 rows of codes, and in the copy of the scales
  const uint32_t copy_to = gr * 64 + ((tq ^ ((gr >> 1) & 3)) << 4);
  const int64_t lane16 = lane * 16;
  const uint8_t* scale_from = (lane < 16 ? p.cache.k : p.cache.v) + (lane & 7) * 16;

  auto issue = [&](int j) {
    const uint32_t dst = ring + (j % kStages) * kStageBytes;
    const longlong2* at = subtiles + (warp + j * kWarps) * 2;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int64_t from = at[i].x;
      const uint32_t bytes = from < 0 ? 0 : 16;
      const int64_t off = (from < 0 ? 0 : from) + lane16;
      copy16(dst + i * 1024 + copy_to, p.cache.k + off, bytes);
      copy16(dst + i * 1024 + 512 + copy_to, p.cache.k + off + 512, bytes);
      copy16(dst + kVCodes + i * 1024 + copy_to, p.cache.v + off, bytes);
      copy16(dst + kVCodes + i * 1024 + 512 + copy_to, p.cache.v + off + 512, bytes);
    }
    const longlong2 mine = at[(lane >> 3) & 1];
    copy16(dst + kKScales + lane * 16, scale_from + mine.y, mine.x < 0 ? 0 : 16);
  };
  __syncthreads();  // the table
#pragma unroll
  for (int j = 0; j < kStages - 1; ++j) {
    if (j < my_tiles) issue(j);
    copy_commit();
  }

  // ---- q: B operands (k = the 8 codes of a K word, n = head), fp16 ----
  uint32_t qf[NT][8][2];
  uint32_t qz[NT][2];   // -8 2^-24 sum_{d in g} q in three bf16 digits, k = 4 digit + g
  float fac[NT][2];     // raw score -> log2 units, per column
  const float sign = p.scale_log2 < 0.f ? -1.f : 1.f;  // the factor itself stays positive
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int h = nt * 8 + gr;
    const bool mine = h < p.group;
    const T* qb = static_cast<const T*>(p.q) + (int64_t)b * p.q_seq_stride +
                  (int64_t)(kvh * p.group + (mine ? h : 0)) * p.q_head_stride + tq * 8;
    float x[4][8];
    float amax = 0.f;
#pragma unroll
    for (int g = 0; g < 4; ++g)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t w = mine ? __ldg(reinterpret_cast<const uint32_t*>(qb + g * 32 + j * 2)) : 0u;
        const float2 v = widen<T>(w);
        x[g][2 * j] = v.x;
        x[g][2 * j + 1] = v.y;
        amax = fmaxf(amax, fmaxf(fabsf(v.x), fabsf(v.y)));
      }
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
    // 2^(14 - floor(log2 amax)), and back with the codes' 2^24
    const int e = max(static_cast<int>(__float_as_uint(amax) >> 23), 14);
    const float up = __uint_as_float(static_cast<uint32_t>(268 - e) << 23) * sign;
    const float down =
        __uint_as_float(static_cast<uint32_t>(e) << 23) * 1024.f * fabsf(p.scale_log2);
    float sums[4];
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      float sum = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        x[g][j] *= up;
        sum += x[g][j];
      }
      // MMA k pairs: nibbles (0, 4) and (1, 5) of the word, then (2, 6) and (3, 7)
      qf[nt][2 * g][0] = Elem<__half>::pack(x[g][0], x[g][4]);
      qf[nt][2 * g][1] = Elem<__half>::pack(x[g][1] * 0.0625f, x[g][5] * 0.0625f);
      qf[nt][2 * g + 1][0] = Elem<__half>::pack(x[g][2], x[g][6]);
      qf[nt][2 * g + 1][1] = Elem<__half>::pack(x[g][3] * 0.0625f, x[g][7] * 0.0625f);
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      sum += __shfl_xor_sync(0xffffffffu, sum, 2);
      sums[g] = sum * (-8.f * 5.9604644775390625e-8f);
    }
    // lane tq: k = 2 tq, 2 tq + 1 are groups (0, 1) for even tq and (2, 3) for odd
    // tq, digit tq / 2; k + 8 the last digit, in the lanes of digit 0 only
    float z[2] = {(tq & 1) ? sums[2] : sums[0], (tq & 1) ? sums[3] : sums[1]};
    float d0[2], d1[2], d2[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      d0[i] = __bfloat162float(__float2bfloat16_rn(z[i]));
      d1[i] = __bfloat162float(__float2bfloat16_rn(z[i] - d0[i]));
      d2[i] = z[i] - d0[i] - d1[i];
    }
    qz[nt][0] = tq < 2 ? Elem<__nv_bfloat16>::pack(d0[0], d0[1])
                       : Elem<__nv_bfloat16>::pack(d1[0], d1[1]);
    qz[nt][1] = tq < 2 ? Elem<__nv_bfloat16>::pack(d2[0], d2[1]) : 0u;
    fac[nt][0] = __shfl_sync(0xffffffffu, down, tq * 8);
    fac[nt][1] = __shfl_sync(0xffffffffu, down, tq * 8 + 4);
  }

  // ldmatrix row addresses: matrices are (tokens 0-7 | 8-15) x (chunks 2i | 2i + 1)
  const int lrow = (lane & 7) + ((lane >> 3) & 1) * 8;
  const uint32_t loff0 = lrow * 64 + (((lane >> 4) ^ ((lrow >> 1) & 3)) << 4);
  const uint32_t loff1 = loff0 ^ 32;
  const float kNegInf = -INFINITY;
  constexpr uint32_t kEight = 0x48004800u;

  float m_run[NT][2], base[NT][2], l_run[NT][2];
  float o[NT][8][4], oz[NT][4][4];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    m_run[nt][0] = m_run[nt][1] = kNegInf;
    base[nt][0] = base[nt][1] = kNegInf;
    l_run[nt][0] = l_run[nt][1] = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
      for (int g = 0; g < 4; ++g) oz[nt][g][i] = 0.f;
#pragma unroll
      for (int mt = 0; mt < 8; ++mt) o[nt][mt][i] = 0.f;
    }
  }
  uint32_t ref = (kMinScaleExp << 7) | 0x7f;  // bf16 bits: the value scales stay at or below

  for (int j = 0; j < my_tiles; ++j) {
    copy_wait<kStages - 2>();
    __syncwarp();  // tile j has landed for every lane, and every lane is done with j - 1
    if (j + kStages - 1 < my_tiles) issue(j + kStages - 1);
    copy_commit();
    const uint32_t kb = ring + (j % kStages) * kStageBytes;
    const int valid = tokens - (warp + j * kWarps) * kTile;

    // ---- raw scores of 32 tokens: sc[nt][st] = (token g | g + 8) x 2 columns ----
    float sc[NT][2][4];
#pragma unroll
    for (int st = 0; st < 2; ++st) {
      uint32_t kw[8];
      ldmatrix_x4(kb + st * 1024 + loff0, kw[0], kw[1], kw[2], kw[3]);
      ldmatrix_x4(kb + st * 1024 + loff1, kw[4], kw[5], kw[6], kw[7]);
      const uint2 s_lo = lds64(kb + kKScales + (st * 16 + gr) * 8);
      const uint2 s_hi = lds64(kb + kKScales + (st * 16 + gr + 8) * 8);
      const uint32_t z_lo = (tq & 1) ? s_lo.y : s_lo.x, z_hi = (tq & 1) ? s_hi.y : s_hi.x;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
        mma_bf16_first(sc[nt][st], z_lo, z_hi, z_lo, z_hi, qz[nt][0], qz[nt][1]);
      const float ks[4][2] = {{lo_scale(s_lo.x), lo_scale(s_hi.x)},
                              {hi_scale(s_lo.x), hi_scale(s_hi.x)},
                              {lo_scale(s_lo.y), lo_scale(s_hi.y)},
                              {hi_scale(s_lo.y), hi_scale(s_hi.y)}};
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const uint32_t w0 = kw[2 * g], w1 = kw[2 * g + 1];
        const uint32_t v0 = w0 >> 8, v1 = w1 >> 8;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float acc[4];
          mma_f16_first(acc, even_codes(w0), even_codes(w1), odd_codes(w0), odd_codes(w1),
                        qf[nt][2 * g][0], qf[nt][2 * g][1]);
          mma_f16(acc, even_codes(v0), even_codes(v1), odd_codes(v0), odd_codes(v1),
                  qf[nt][2 * g + 1][0], qf[nt][2 * g + 1][1]);
#pragma unroll
          for (int i = 0; i < 4; ++i) sc[nt][st][i] = fmaf(ks[g][i >> 1], acc[i], sc[nt][st][i]);
        }
      }
    }

    // ---- value scales of this lane's tokens, masked past the end ----
    uint2 vs[2][2];
#pragma unroll
    for (int st = 0; st < 2; ++st)
#pragma unroll
      for (int i = 0; i < 2; ++i) vs[st][i] = lds64(kb + kVScales + (st * 16 + i * 8 + gr) * 8);
    // the four lanes of a token look at one each of its row's four tokens
    uint2 look = lds64(kb + kVScales + (tq * 8 + gr) * 8);
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
            for (int nt = 0; nt < NT; ++nt) sc[nt][st][2 * i] = sc[nt][st][2 * i + 1] = kNegInf;
          }
      if (tq * 8 + gr >= valid) look = make_uint2(0, 0);
    }

    // ---- running maximum and value exponent; both move rarely ----
    const uint32_t vmax2 = __vmaxu2(look.x, look.y);
    uint32_t vmax = max(vmax2 & 0xffffu, vmax2 >> 16);
    bool moved = vmax > ref || j == 0;
    float mx[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        mx[nt][c] = fmaxf(fmaxf(sc[nt][0][c], sc[nt][0][2 + c]),
                          fmaxf(sc[nt][1][c], sc[nt][1][2 + c]));
        moved |= fmaf(mx[nt][c], fac[nt][c], -kSlack) > m_run[nt][c];
      }
    if (__any_sync(0xffffffffu, moved)) {
      // a scale that is no number spoils its own group's sums only: it is not followed
      uint32_t top = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t w = i < 2 ? look.x : look.y;
        const uint32_t s = (i & 1) ? w >> 16 : w & 0xffffu;
        if (s < 0x7f80u) top = max(top, s);
      }
      ref = max(ref, __reduce_max_sync(0xffffffffu, top) | 0x7fu);
      const float lift = static_cast<float>(static_cast<int>(ref >> 7) - 126) - kHeadroom;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float alpha[2];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float m = mx[nt][c] * fac[nt][c];
          m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 4));
          m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 8));
          m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
          m_run[nt][c] = fmaxf(m_run[nt][c], m);
          const float next = (m_run[nt][c] == kNegInf ? 0.f : m_run[nt][c]) + lift;
          alpha[c] = fminf(fast_exp2(base[nt][c] - next), 1.f);
          base[nt][c] = next;
          l_run[nt][c] *= alpha[c];
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
#pragma unroll
          for (int g = 0; g < 4; ++g) oz[nt][g][i] *= alpha[i & 1];
#pragma unroll
          for (int mt = 0; mt < 8; ++mt) o[nt][mt][i] *= alpha[i & 1];
        }
      }
    }

    // ---- weights and O^T += V^T w^T ----
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int st = 0; st < 2; ++st)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          sc[nt][st][i] = ex2_approx(fmaf(sc[nt][st][i], fac[nt][i & 1], -base[nt][i & 1]));
          l_run[nt][i & 1] += sc[nt][st][i];
        }
#pragma unroll
    for (int st = 0; st < 2; ++st) {
      uint32_t vw[8];
      ldmatrix_x4_trans(kb + kVCodes + st * 1024 + loff0, vw[0], vw[1], vw[2], vw[3]);
      ldmatrix_x4_trans(kb + kVCodes + st * 1024 + loff1, vw[4], vw[5], vw[6], vw[7]);
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const uint32_t w0 = vw[2 * g], w1 = vw[2 * g + 1];  // tokens 0-7 | 8-15
        const uint32_t v0 = w0 >> 8, v1 = w1 >> 8;
        const uint32_t s0 = g < 2 ? vs[st][0].x : vs[st][0].y;
        const uint32_t s1 = g < 2 ? vs[st][1].x : vs[st][1].y;
        const float f0 = (g & 1) ? hi_scale(s0) : lo_scale(s0);
        const float f1 = (g & 1) ? hi_scale(s1) : lo_scale(s1);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const float* pr = sc[nt][st];
          const uint32_t b0 = movmatrix_trans(Elem<__half>::pack(pr[0] * f0, pr[1] * f0));
          const uint32_t b1 = movmatrix_trans(Elem<__half>::pack(pr[2] * f1, pr[3] * f1));
          mma_f16(o[nt][2 * g], even_codes(w0), odd_codes(w0), even_codes(w1), odd_codes(w1), b0,
                  b1);
          mma_f16(o[nt][2 * g + 1], even_codes(v0), odd_codes(v0), even_codes(v1), odd_codes(v1),
                  b0, b1);
          mma_f16(oz[nt][g], kEight, kEight, kEight, kEight, b0, b1);
        }
      }
    }
  }

  // ---- merge the warps ----
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      l_run[nt][c] += __shfl_xor_sync(0xffffffffu, l_run[nt][c], 4);
      l_run[nt][c] += __shfl_xor_sync(0xffffffffu, l_run[nt][c], 8);
      l_run[nt][c] += __shfl_xor_sync(0xffffffffu, l_run[nt][c], 16);
    }
  __syncthreads();  // every warp is done with the ring

  float* ml = reinterpret_cast<float*>(smem);     // [warp][base 16 | sum 16]
  float* mo = ml + kWarps * 32;                   // [warp][16][kMergeStride]
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int head = nt * 8 + tq * 2 + c;
        const float z = oz[nt][g][c];
        if (head < p.group) {
          const float4 row = make_float4(o[nt][2 * g][c] * 16777216.f - z,
                                         o[nt][2 * g][2 + c] * 1048576.f - z,
                                         o[nt][2 * g + 1][c] * 16777216.f - z,
                                         o[nt][2 * g + 1][2 + c] * 1048576.f - z);
          *reinterpret_cast<float4*>(&mo[(warp * 16 + head) * kMergeStride + g * 32 + gr * 4]) = row;
          if (g == 0 && gr == 0) {
            ml[warp * 32 + head] = base[nt][c];
            ml[warp * 32 + 16 + head] = l_run[nt][c];
          }
        }
      }
    }
  __syncthreads();

  for (int idx = threadIdx.x; idx < p.group * (kHeadDim / 4); idx += blockDim.x) {
    const int row = idx >> 5;
    const int d = (idx & 31) * 4;
    float m = kNegInf;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) m = fmaxf(m, ml[w * 32 + row]);
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    float l = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float mw = ml[w * 32 + row];
      if (mw == kNegInf) continue;  // a warp without tiles
      const float f = fast_exp2(mw - m);
      const float4 x = *reinterpret_cast<const float4*>(&mo[(w * 16 + row) * kMergeStride + d]);
      acc.x += x.x * f;
      acc.y += x.y * f;
      acc.z += x.z * f;
      acc.w += x.w * f;
      l += ml[w * 32 + 16 + row] * f;
    }
    const float inv = 1.f / l;
    acc = make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
    const int head = kvh * p.group + row;
    if (p.num_parts == 1) {
      uint32_t* ob = reinterpret_cast<uint32_t*>(static_cast<T*>(p.out) +
                                                 (int64_t)b * p.out_seq_stride +
                                                 (int64_t)head * p.out_head_stride + d);
      ob[0] = Elem<T>::pack(acc.x, acc.y);
      ob[1] = Elem<T>::pack(acc.z, acc.w);
    } else {
      const int64_t slot = ((int64_t)b * p.num_q_heads + head) * p.num_parts + part;
      *reinterpret_cast<float4*>(p.part_o + slot * kHeadDim + d) = acc;
      if (d == 0) p.part_lse[slot] = m + log2f(l);
    }
  }
}

// Joins the partitions of one (sequence, q head) per CTA: lane i of each warp
// owns 4 values, the warps take the partitions in turn.
template <typename T>
__global__ void __launch_bounds__(kWarps * 32) int4_reduce_kernel(const Int4DecodeParams p) {
  __shared__ float4 acc_s[kWarps][32];
  __shared__ float m_s[kWarps], l_s[kWarps];
  pdl_wait();
  const int b = static_cast<int>(blockIdx.x / static_cast<unsigned>(p.num_q_heads));
  const int head = static_cast<int>(blockIdx.x - (unsigned)b * (unsigned)p.num_q_heads);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int seq_len = max(__ldg(p.seq_lens + b), 0);
  const int n = min((seq_len + p.part_tokens - 1) / p.part_tokens, p.num_parts);
  const int64_t at = ((int64_t)b * p.num_q_heads + head) * p.num_parts;
  float m = -INFINITY, l = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int i = warp; i < n; i += kWarps) {
    const float lse = __ldcg(p.part_lse + at + i);
    const float4 x = __ldcg(reinterpret_cast<const float4*>(p.part_o + (at + i) * kHeadDim) + lane);
    const float next = fmaxf(m, lse);
    const float keep = fast_exp2(m - next), w = fast_exp2(lse - next);
    m = next;
    l = l * keep + w;
    acc.x = acc.x * keep + x.x * w;
    acc.y = acc.y * keep + x.y * w;
    acc.z = acc.z * keep + x.z * w;
    acc.w = acc.w * keep + x.w * w;
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

template <typename T, int NT>
cudaError_t launch_typed(const Int4DecodeParams& p, unsigned grid,
                         cudaStream_t stream) {
  auto kernel = paged_decode_int4_kernel<T, NT>;
  cudaError_t e = ensure_smem_attr(reinterpret_cast<const void*>(kernel), kSmemBytes);
  if (e != cudaSuccess) return e;
  e = launch_dependent(kernel, grid, kSmemBytes, stream, p);
  if (e != cudaSuccess || p.num_parts == 1) return e;
  return launch_dependent(int4_reduce_kernel<T>, (unsigned)p.num_seqs * (unsigned)p.num_q_heads, 0,
                          stream, p);
}

}  // namespace

cudaError_t launch_paged_decode_int4(const Int4DecodeParams& p, int dtype, cudaStream_t stream) {
  const int64_t grid = (int64_t)p.num_seqs * p.num_kv_heads * p.num_parts;
  if (grid > 0x7fffffff || (int64_t)p.num_seqs * p.num_q_heads > 0x7fffffff)
    return cudaErrorInvalidConfiguration;
  const bool wide = p.group > 8;
  if (dtype == B200_DTYPE_BFLOAT16)
    return wide ? launch_typed<__nv_bfloat16, 2>(p, (unsigned)grid, stream)
                : launch_typed<__nv_bfloat16, 1>(p, (unsigned)grid, stream);
  return wide ? launch_typed<__half, 2>(p, (unsigned)grid, stream)
              : launch_typed<__half, 1>(p, (unsigned)grid, stream);
}

}  // namespace b200
