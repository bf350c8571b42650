// kv_int4.cu — the 4-bit KV cache's append (quantise and scatter) and read-back
// (gather and dequantise). Format and page layout: kv_int4.cuh.
//
// Both are HBM traffic: 256 bytes of a 16-bit row one way, 72 bytes of the
// 4-bit row the other. A half-warp owns the K row and the V row of one (token,
// head): lane i holds elements [8i, 8i + 8), 16 bytes of the 16-bit row and 4
// bytes of codes, so a group's maximum takes two shuffles over its 4 lanes and
// every access is a full-width coalesced one. A block takes 16 consecutive
// tokens of one head: neighbouring blocks read neighbouring 256-byte pieces of
// the same rows, and tokens in consecutive slots write consecutive bytes of
// the head-major page.
#include <cuda_runtime.h>

#include "common.cuh"
#include "kv_int4.cuh"

namespace b200 {
namespace {

constexpr int kRowsPerBlock = 16;
constexpr int kThreads = kRowsPerBlock * 16;

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
template <typename T>
__device__ __forceinline__ uint32_t group_scale(uint32_t amax, float& r) {
  r = 0.f;
  if (amax >= Row16<T>::kInf) return 0x7fc0u;
  __nv_bfloat16 s = __float2bfloat16_rn(__fdiv_rn(Row16<T>::bits(amax), 7.f));
  float f = __bfloat162float(s);
  if (Elem<T>::kDtype == B200_DTYPE_FLOAT16 && f > 9344.f) f = 9344.f;
  if (f < 1.17549435e-38f) return 0u;  // 2^-126
  r = __frcp_rn(f);
  return __float_as_uint(f) >> 16;
}

// One 16-byte piece of a row: its 8 codes and, via its group's lanes, the scale.
template <typename T>
__device__ __forceinline__ uint32_t quantise8(const uint4& x, uint32_t& scale) {
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) m = __vmaxu2(m, w[i] & 0x7fff7fffu);
  m = max(m & 0xffffu, m >> 16);
  m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
  m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
  float r;
  scale = group_scale<T>(m, r);
  // 12582920 = 1.5 * 2^23 + 8: the sum's last place is 1 and its parity that of
  // the rounded product, so the addition rounds half to even and leaves the
  // code in the low bits; the constant upper bits cancel in the packed sum
  constexpr uint32_t kMagic = 0x4b400000u;
  uint32_t packed = 0u - kMagic * 0x11111111u;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 v = Row16<T>::widen(w[i]);
    const uint32_t lo = __float_as_uint(__fadd_rn(__fmul_rn(v.x, r), 12582920.f));
    const uint32_t hi = __float_as_uint(__fadd_rn(__fmul_rn(v.y, r), 12582920.f));
    packed += (lo << (8 * i)) + (hi << (8 * i + 4));
  }
  return m >= Row16<T>::kInf ? 0x88888888u : packed;
}

// Codes of 8 elements -> one 16-byte piece of T, each rn(s * (c - 8)).
template <typename T>
__device__ __forceinline__ uint4 dequantise8(uint32_t codes, float s) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float lo = __uint_as_float(0x4b000000u | ((codes >> (8 * i)) & 15u)) - 8388616.f;
    const float hi = __uint_as_float(0x4b000000u | ((codes >> (8 * i + 4)) & 15u)) - 8388616.f;
    w[i] = Elem<T>::pack(__fmul_rn(lo, s), __fmul_rn(hi, s));
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

// The token and head of this half-warp; false past the last token.
__device__ __forceinline__ bool my_row(int num_kv_heads, int64_t num_tokens, int64_t& token,
                                       int& head) {
  const uint32_t tile = blockIdx.x / static_cast<uint32_t>(num_kv_heads);
  head = static_cast<int>(blockIdx.x - tile * static_cast<uint32_t>(num_kv_heads));
  token = (int64_t)tile * kRowsPerBlock + (threadIdx.x >> 4);
  return token < num_tokens;
}

template <typename SlotT>
__device__ __forceinline__ int64_t my_slot(const SlotT* slots, int64_t token, const Int4Cache& c,
                                           int head, int32_t* status) {
  const int64_t slot = static_cast<int64_t>(__ldg(slots + token));
  if (slot == -1) return -1;
  if (slot < 0 || slot >= c.num_blocks * c.block_size) {
    if (head == 0 && (threadIdx.x & 15) == 0) report_status(status, B200_STATUS_SLOT_OUT_OF_RANGE);
    return -1;
  }
  return slot;
}

template <typename T, typename SlotT>
__global__ void __launch_bounds__(kThreads)
    store_int4_kernel(const T* __restrict__ key, int64_t key_row_stride,
                      const T* __restrict__ value, int64_t value_row_stride, const Int4Cache c,
                      const SlotT* __restrict__ slots, int64_t num_tokens, int32_t* status) {
  // a decode launched as this kernel's programmatic dependent may start now; it
  // waits for this grid to complete before it reads anything
  pdl_launch_dependents();
  const int i = threadIdx.x & 15;
  int64_t token;
  int head;
  const bool live = my_row(c.num_kv_heads, num_tokens, token, head);
  uint4 k = make_uint4(0, 0, 0, 0), v = k;
  int64_t slot = -1;
  if (live) {
    const int64_t col = (int64_t)head * 128 + i * 8;
    k = __ldg(reinterpret_cast<const uint4*>(key + token * key_row_stride + col));
    v = __ldg(reinterpret_cast<const uint4*>(value + token * value_row_stride + col));
    slot = my_slot(slots, token, c, head, status);
  }
  uint32_t ks, vs;
  const uint32_t kc = quantise8<T>(k, ks);
  const uint32_t vc = quantise8<T>(v, vs);
  if (slot < 0) return;
  const RowAt at = row_at(c, slot, head);
  *reinterpret_cast<uint32_t*>(c.k + at.codes + i * 4) = kc;
  *reinterpret_cast<uint32_t*>(c.v + at.codes + i * 4) = vc;
  if ((i & 3) == 0) {
    *reinterpret_cast<uint16_t*>(c.k + at.scales + (i >> 1)) = static_cast<uint16_t>(ks);
    *reinterpret_cast<uint16_t*>(c.v + at.scales + (i >> 1)) = static_cast<uint16_t>(vs);
  }
}

template <typename T, typename SlotT>
__global__ void __launch_bounds__(kThreads)
    load_int4_kernel(const Int4Cache c, const SlotT* __restrict__ slots, int64_t num_tokens,
                     T* __restrict__ key, int64_t key_row_stride, T* __restrict__ value,
                     int64_t value_row_stride, int32_t* status) {
  const int i = threadIdx.x & 15;
  int64_t token;
  int head;
  if (!my_row(c.num_kv_heads, num_tokens, token, head)) return;
  const int64_t slot = my_slot(slots, token, c, head, status);
  if (slot < 0) return;
  const RowAt at = row_at(c, slot, head);
  const uint32_t kc = *reinterpret_cast<const uint32_t*>(c.k + at.codes + i * 4);
  const uint32_t vc = *reinterpret_cast<const uint32_t*>(c.v + at.codes + i * 4);
  const uint32_t ks = *reinterpret_cast<const uint16_t*>(c.k + at.scales + (i >> 2) * 2);
  const uint32_t vs = *reinterpret_cast<const uint16_t*>(c.v + at.scales + (i >> 2) * 2);
  const int64_t col = (int64_t)head * 128 + i * 8;
  *reinterpret_cast<uint4*>(key + token * key_row_stride + col) =
      dequantise8<T>(kc, __uint_as_float(ks << 16));
  *reinterpret_cast<uint4*>(value + token * value_row_stride + col) =
      dequantise8<T>(vc, __uint_as_float(vs << 16));
}

cudaError_t grid_of(int64_t num_tokens, int num_kv_heads, unsigned* grid) {
  const int64_t blocks = (num_tokens + kRowsPerBlock - 1) / kRowsPerBlock * num_kv_heads;
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
  load_int4_kernel<T, SlotT><<<grid, kThreads, 0, stream>>>(
      c, static_cast<const SlotT*>(slots), n, static_cast<T*>(key), ks, static_cast<T*>(value), vs,
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
