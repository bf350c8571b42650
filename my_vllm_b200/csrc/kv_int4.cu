// kv_int4.cu — the 4-bit KV cache's append (quantise and scatter) and read-back
// (gather and dequantise). Format and page layout: kv_int4.cuh.
//
// Both are HBM traffic: 256 bytes of a 16-bit row one way, 72 bytes of the
// 4-bit row the other. Eight lanes own the K row and the V row of one (token,
// head): lane i holds elements [16i, 16i + 16), 32 bytes of the 16-bit row and
// 8 bytes of codes, so two lanes share a group and the scale, the dearest part
// of the arithmetic, is computed once per 16 elements (with 16 lanes a row and
// an IEEE division the append was bound by issue slots: 89 us, now 59 us, for
// 64k tokens of 8 heads in consecutive slots, 5.8 TB/s of 6.5 measured). A
// block takes 32 consecutive tokens of one head: neighbouring blocks read
// neighbouring 256-byte pieces of the same rows, and tokens in consecutive
// slots write consecutive bytes of the head-major page. More tokens a thread,
// with their loads issued together, were no faster (2: the same, 4: 72 us);
// the read-back slows down with them (59 us, 68, 83). What bounds both is DRAM.
// 128k tokens of 8 heads, us of the append and of the read-back: slots in order 111
// and 110, whole pages in random order 113 and 112 (6.1 TB/s, 0.93 of the measured
// rate), slots in random order 148 and 149 (4.6 TB/s); the size of the pages, 16 to
// 256, changes each by 3 % at most. At random slots the read-back takes 354 MB from
// DRAM where 151 are the cache's (in order 152), 1.33 times the bytes in all and 1.31
// times the time: an 8-byte scale brings a hundred bytes with it. The append's bytes
// grow by 8 % within the kernel, the rest of its 1.26 is not accounted for. Pools that L2
// holds lose less (32k tokens 1.1 times), larger ones more (256k 1.5 times).
#include <cuda_runtime.h>

#include "common.cuh"
#include "kv_int4.cuh"

namespace b200 {
namespace {

constexpr int kLanes = 8;           // of a row
constexpr int kThreads = 256;
constexpr int kRows = kThreads / kLanes;  // of a block

template <typename T>
struct Row16;
template <>
struct Row16<__nv_bfloat16> {
  static constexpr uint32_t kInf = 0x7f80;
  __device__ __forceinline__ static float bits(uint32_t b) { return __uint_as_float(b << 16); }
  __device__ __forceinline__ static float2 widen(uint32_t w) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  }
};
template <>
struct Row16<__half> {
  static constexpr uint32_t kInf = 0x7c00;
  __device__ __forceinline__ static float bits(uint32_t b) {
    return __half2float(__ushort_as_half(static_cast<unsigned short>(b)));
  }
  __device__ __forceinline__ static float2 widen(uint32_t w) {
    return __half22float2(*reinterpret_cast<const __half2*>(&w));
  }
};

// Scale of a group whose largest |x| has the 16-bit pattern `amax` (patterns of
// one sign order like their values, infinity and NaN above all of them):
// bf16 bits, and the reciprocal the codes are taken with (0: all codes 8).
// Both quotients are rounded correctly by one Newton step on an estimate: the
// residual of each is exact in one fma (divisors of 3 and 8 bits), so the
// corrected value differs from the quotient by under 2^-44 of it, and no
// quotient by such a divisor lies that near the middle of two fp32 numbers.
template <typename T>
__device__ __forceinline__ uint32_t group_scale(uint32_t amax, float& r) {
  const float a = Row16<T>::bits(amax);
  const float seventh = 0.142857142857142857f;
  const float q = a * seventh;
  float s = __bfloat162float(__float2bfloat16_rn(fmaf(fmaf(-7.f, q, a), seventh, q)));
  if (Elem<T>::kDtype == B200_DTYPE_FLOAT16) s = fminf(s, 9344.f);
  float e;
  asm("rcp.approx.f32 %0, %1;" : "=f"(e) : "f"(s));
  e = fmaf(e, fmaf(-s, e, 1.f), e);
  const bool fine = amax < Row16<T>::kInf;
  const bool used = fine && s >= 1.17549435e-38f;  // 2^-126
  r = used ? e : 0.f;
  return used ? __float_as_uint(s) >> 16 : fine ? 0u : 0x7fc0u;
}

// 16 elements of a row (with the neighbouring lane's 16 a whole group): their
// codes, and the group's scale.
template <typename T>
__device__ __forceinline__ uint2 quantise16(const uint4 (&x)[2], uint32_t& scale) {
  const uint32_t w[8] = {x[0].x, x[0].y, x[0].z, x[0].w, x[1].x, x[1].y, x[1].z, x[1].w};
  uint32_t m = w[0] & 0x7fff7fffu;
#pragma unroll
  for (int i = 1; i < 8; ++i) m = __vmaxu2(m, w[i] & 0x7fff7fffu);
  m = __vmaxu2(m, __shfl_xor_sync(0xffffffffu, m, 1));
  m = max(m & 0xffffu, m >> 16);
  float r;
  scale = group_scale<T>(m, r);
  // 12582920 = 1.5 * 2^23 + 8: the sum's last place is 1 and its parity that of
  // the rounded product, so the addition rounds half to even and leaves the
  // code in the low bits; the constant upper bits cancel in the packed sum. The
  // product is two scalar ones: a packed product into a packed sum comes out
  // fused, and one rounding instead of two breaks the ties of the definition
  const uint64_t magic2 = f2(12582920.f, 12582920.f);
  uint32_t packed[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    packed[h] = 0u - 0x4b400000u * 0x11111111u;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 v = Row16<T>::widen(w[4 * h + i]);
      float lo, hi;
      f2_split(f2_add(f2(__fmul_rn(v.x, r), __fmul_rn(v.y, r)), magic2), lo, hi);
      packed[h] += (__float_as_uint(lo) << (8 * i)) + (__float_as_uint(hi) << (8 * i + 4));
    }
  }
  // (a product with an element that is no number is no number either)
  return m < Row16<T>::kInf ? make_uint2(packed[0], packed[1])
                            : make_uint2(0x88888888u, 0x88888888u);
}

// Codes of 8 elements -> one 16-byte piece of T, each rn(s * (c - 8)).
template <typename T>
__device__ __forceinline__ uint4 dequantise8(uint32_t codes, float s) {
  const uint64_t s2 = f2(s, s), zero2 = f2(-8388616.f, -8388616.f);
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float lo = __uint_as_float(0x4b000000u | ((codes >> (8 * i)) & 15u));
    const float hi = __uint_as_float(0x4b000000u | ((codes >> (8 * i + 4)) & 15u));
    float x, y;
    f2_split(f2_mul(f2_add(f2(lo, hi), zero2), s2), x, y);
    w[i] = Elem<T>::pack(x, y);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// Byte offsets of a slot's row of one head inside a cache tensor.
struct RowAt {
  int64_t codes, scales;
};
__device__ __forceinline__ RowAt row_at(const Int4Cache& c, int64_t slot, int head) {
  int64_t page;
  int row;
  if (slot < (int64_t(1) << 32)) {
    const uint32_t p = static_cast<uint32_t>(slot) / static_cast<uint32_t>(c.block_size);
    page = p;
    row = static_cast<int>(static_cast<uint32_t>(slot) - p * static_cast<uint32_t>(c.block_size));
  } else {
    page = slot / c.block_size;
    row = static_cast<int>(slot - page * c.block_size);
  }
  const int64_t base = page * c.block_stride;
  const int64_t hr = (int64_t)head * c.block_size + row;
  return {base + hr * kInt4CodeBytes,
          base + (int64_t)c.num_kv_heads * c.block_size * kInt4CodeBytes + hr * kInt4ScaleBytes};
}

// The slot of a token; -1: none, or out of range (reported by one lane).
template <typename SlotT>
__device__ __forceinline__ int64_t slot_of(const SlotT* slots, int64_t token, const Int4Cache& c,
                                           bool reports, int32_t* status) {
  const int64_t slot = static_cast<int64_t>(__ldg(slots + token));
  if (slot >= 0 && slot < c.num_blocks * c.block_size) return slot;
  if (slot != -1 && reports) report_status(status, B200_STATUS_SLOT_OUT_OF_RANGE);
  return -1;
}

// The token and head of this thread's row; false past the last token.
__device__ __forceinline__ bool my_row(int num_kv_heads, int64_t num_tokens, int64_t& token,
                                       int& head) {
  const uint32_t tile = blockIdx.x / static_cast<uint32_t>(num_kv_heads);
  head = static_cast<int>(blockIdx.x - tile * static_cast<uint32_t>(num_kv_heads));
  token = (int64_t)tile * kRows + threadIdx.x / kLanes;
  return token < num_tokens;
}

template <typename T, typename SlotT>
__global__ void __launch_bounds__(kThreads)
    store_int4_kernel(const T* __restrict__ key, int64_t key_row_stride,
                      const T* __restrict__ value, int64_t value_row_stride, const Int4Cache c,
                      const SlotT* __restrict__ slots, int64_t num_tokens, int32_t* status) {
  // a decode launched as this kernel's programmatic dependent may start now; it
  // waits for this grid to complete before it reads anything
  pdl_launch_dependents();
  const int i = threadIdx.x & (kLanes - 1);
  int64_t token, slot = -1;
  int head;
  uint4 k[2] = {}, v[2] = {};
  if (my_row(c.num_kv_heads, num_tokens, token, head)) {
    const int64_t col = (int64_t)head * 128 + i * 16;
    const uint4* ks = reinterpret_cast<const uint4*>(key + token * key_row_stride + col);
    const uint4* vs = reinterpret_cast<const uint4*>(value + token * value_row_stride + col);
    k[0] = __ldg(ks);
    k[1] = __ldg(ks + 1);
    v[0] = __ldg(vs);
    v[1] = __ldg(vs + 1);
    slot = slot_of(slots, token, c, head == 0 && i == 0, status);
  }
  uint32_t ks, vs;
  const uint2 kc = quantise16<T>(k, ks);
  const uint2 vc = quantise16<T>(v, vs);
  if (slot < 0) return;
  const RowAt at = row_at(c, slot, head);
  *reinterpret_cast<uint2*>(c.k + at.codes + i * 8) = kc;
  *reinterpret_cast<uint2*>(c.v + at.codes + i * 8) = vc;
  // even lanes write the K scale, odd lanes the V scale of their group
  *reinterpret_cast<uint16_t*>(((i & 1) ? c.v : c.k) + at.scales + (i >> 1) * 2) =
      static_cast<uint16_t>((i & 1) ? vs : ks);
}

// kSector: the 16-bit rows are 32-byte aligned, and a thread's 32 bytes leave in
// one store. Two 16-byte stores write every sector in halves, which costs a
// fifth (128k tokens of 8 heads in order: 140 us, 113 us with one).
template <typename T, typename SlotT, bool kSector>
__global__ void __launch_bounds__(kThreads)
    load_int4_kernel(const Int4Cache c, const SlotT* __restrict__ slots, int64_t num_tokens,
                     T* __restrict__ key, int64_t key_row_stride, T* __restrict__ value,
                     int64_t value_row_stride, int32_t* status) {
  const int i = threadIdx.x & (kLanes - 1);
  int64_t token;
  int head;
  if (!my_row(c.num_kv_heads, num_tokens, token, head)) return;
  const int64_t slot = slot_of(slots, token, c, head == 0 && i == 0, status);
  if (slot < 0) return;
  const RowAt at = row_at(c, slot, head);
  const uint2 kc = *reinterpret_cast<const uint2*>(c.k + at.codes + i * 8);
  const uint2 vc = *reinterpret_cast<const uint2*>(c.v + at.codes + i * 8);
  const uint32_t ks = *reinterpret_cast<const uint16_t*>(c.k + at.scales + (i >> 1) * 2);
  const uint32_t vs = *reinterpret_cast<const uint16_t*>(c.v + at.scales + (i >> 1) * 2);
  const int64_t col = (int64_t)head * 128 + i * 16;
  uint4* kd = reinterpret_cast<uint4*>(key + token * key_row_stride + col);
  uint4* vd = reinterpret_cast<uint4*>(value + token * value_row_stride + col);
  const float sk = __uint_as_float(ks << 16), sv = __uint_as_float(vs << 16);
  const uint4 k0 = dequantise8<T>(kc.x, sk), k1 = dequantise8<T>(kc.y, sk);
  const uint4 v0 = dequantise8<T>(vc.x, sv), v1 = dequantise8<T>(vc.y, sv);
  if constexpr (kSector) {
    st_global_v8(kd, k0, k1);
    st_global_v8(vd, v0, v1);
  } else {
    kd[0] = k0;
    kd[1] = k1;
    vd[0] = v0;
    vd[1] = v1;
  }
}

cudaError_t grid_of(int64_t num_tokens, int num_kv_heads, unsigned* grid) {
  const int64_t blocks = (num_tokens + kRows - 1) / kRows * num_kv_heads;
  if (blocks > 0x7fffffff) return cudaErrorInvalidConfiguration;
  *grid = static_cast<unsigned>(blocks);
  return cudaSuccess;
}

template <typename T, typename SlotT>
cudaError_t store_typed(const void* key, int64_t ks, const void* value, int64_t vs,
                        const Int4Cache& c, const void* slots, int64_t n, int32_t* status,
                        cudaStream_t stream) {
  unsigned grid;
  const cudaError_t e = grid_of(n, c.num_kv_heads, &grid);
  if (e != cudaSuccess) return e;
  store_int4_kernel<T, SlotT><<<grid, kThreads, 0, stream>>>(
      static_cast<const T*>(key), ks, static_cast<const T*>(value), vs, c,
      static_cast<const SlotT*>(slots), n, status);
  return cudaGetLastError();
}

template <typename T, typename SlotT>
cudaError_t load_typed(const Int4Cache& c, const void* slots, int64_t n, void* key, int64_t ks,
                       void* value, int64_t vs, int32_t* status, cudaStream_t stream) {
  unsigned grid;
  const cudaError_t e = grid_of(n, c.num_kv_heads, &grid);
  if (e != cudaSuccess) return e;
  const bool sector = ((reinterpret_cast<uintptr_t>(key) | reinterpret_cast<uintptr_t>(value)) &
                       31) == 0 && ((ks | vs) & 15) == 0;
  auto kernel = sector ? load_int4_kernel<T, SlotT, true> : load_int4_kernel<T, SlotT, false>;
  kernel<<<grid, kThreads, 0, stream>>>(c, static_cast<const SlotT*>(slots), n,
                                        static_cast<T*>(key), ks, static_cast<T*>(value), vs,
                                        status);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_store_kvcache_int4(const void* key, int64_t ks, const void* value, int64_t vs,
                                      int dtype, const Int4Cache& c, const void* slots,
                                      bool slot64, int64_t n, int32_t* status,
                                      cudaStream_t stream) {
  if (dtype == B200_DTYPE_BFLOAT16)
    return slot64 ? store_typed<__nv_bfloat16, int64_t>(key, ks, value, vs, c, slots, n, status,
                                                        stream)
                  : store_typed<__nv_bfloat16, int32_t>(key, ks, value, vs, c, slots, n, status,
                                                        stream);
  return slot64 ? store_typed<__half, int64_t>(key, ks, value, vs, c, slots, n, status, stream)
                : store_typed<__half, int32_t>(key, ks, value, vs, c, slots, n, status, stream);
}

cudaError_t launch_load_kvcache_int4(const Int4Cache& c, const void* slots, bool slot64, int64_t n,
                                     void* key, int64_t ks, void* value, int64_t vs, int dtype,
                                     int32_t* status, cudaStream_t stream) {
  if (dtype == B200_DTYPE_BFLOAT16)
    return slot64 ? load_typed<__nv_bfloat16, int64_t>(c, slots, n, key, ks, value, vs, status,
                                                       stream)
                  : load_typed<__nv_bfloat16, int32_t>(c, slots, n, key, ks, value, vs, status,
                                                       stream);
  return slot64 ? load_typed<__half, int64_t>(c, slots, n, key, ks, value, vs, status, stream)
                : load_typed<__half, int32_t>(c, slots, n, key, ks, value, vs, status, stream);
}

}  // namespace b200
