// paged_int4.cu — attention over a 4-bit paged KV cache, one warp per (query
// row, q head): lane i owns elements [4i, 4i + 4) of the head, keys are visited
// one after the other with the running maximum and sum of the softmax in fp32.
#include <cuda_runtime.h>
#include <math.h>

#include "common.cuh"
#include "kv_int4.cuh"

namespace b200 {
namespace {

constexpr int kWarps = 4;

__device__ __forceinline__ void dequant4(uint32_t c, float s, float (&x)[4]) {
#pragma unroll
  for (int j = 0; j < 4; ++j)
    x[j] = s * (static_cast<float>((c >> (4 * j)) & 15u) - 8.f);
}

template <typename T>
__device__ __forceinline__ float to_float(T x);
template <>
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
template <>
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }

template <typename T>
__global__ void __launch_bounds__(kWarps * 32)
    int4_attention_kernel(const Int4Cache c, const Int4AttnParams p) {
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int head = blockIdx.y * kWarps + (threadIdx.x >> 5);
  if (head >= p.num_q_heads) return;
  const int row = blockIdx.x;
  int s = row, limit;
  if (p.query_start_loc != nullptr) {
    if (row < p.query_start_loc[0] || row >= p.query_start_loc[p.num_seqs]) return;
    int lo = 0, hi = p.num_seqs - 1;  // the last sequence that starts at or before the row
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (p.query_start_loc[mid] <= row) lo = mid;
      else hi = mid - 1;
    }
    s = lo;
    const int q0 = p.query_start_loc[s], q_len = p.query_start_loc[s + 1] - q0;
    limit = p.seq_lens[s] - q_len + (row - q0) + 1;
  } else {
    limit = p.seq_lens[s];
    if (limit > p.plan_tokens) {
      limit = static_cast<int>(p.plan_tokens);
      if (lane == 0) report_status(p.status, B200_STATUS_PLAN_EXCEEDED);
    }
  }
  const int kvh = head / p.group;
  const T* q = static_cast<const T*>(p.q) + row * p.q_token_stride + head * p.q_head_stride;
  float qv[4], acc[4] = {0.f, 0.f, 0.f, 0.f}, m = -INFINITY, l = 0.f;
#pragma unroll
  for (int j = 0; j < 4; ++j) qv[j] = to_float(q[lane * 4 + j]) * p.scale_log2;
  for (int t = 0; t < limit; ++t) {
    const int col = t / c.block_size, r = t - col * c.block_size;
    int page = col < p.max_blocks ? p.block_tables[s * p.block_table_stride + col] : -1;
    float k[4] = {0.f, 0.f, 0.f, 0.f}, v[4] = {0.f, 0.f, 0.f, 0.f};
    if (page < 0 || page >= c.num_blocks) {
      if (lane == 0) report_status(p.status, B200_STATUS_PAGE_OUT_OF_RANGE);
    } else {
      const int64_t hr = (int64_t)kvh * c.block_size + r;
      const int64_t base = page * c.block_stride;
      const int64_t cat = base + hr * kInt4CodeBytes + lane * 2;
      const int64_t sat = base + (int64_t)c.num_kv_heads * c.block_size * kInt4CodeBytes +
                          hr * kInt4ScaleBytes + (lane >> 3) * 2;
      const uint32_t ks = *reinterpret_cast<const uint16_t*>(c.k + sat);
      const uint32_t vs = *reinterpret_cast<const uint16_t*>(c.v + sat);
      dequant4(*reinterpret_cast<const uint16_t*>(c.k + cat), __uint_as_float(ks << 16), k);
      dequant4(*reinterpret_cast<const uint16_t*>(c.v + cat), __uint_as_float(vs << 16), v);
    }
    float d = (qv[0] * k[0] + qv[1] * k[1]) + (qv[2] * k[2] + qv[3] * k[3]);
#pragma unroll
    for (int o = 16; o; o >>= 1) d += __shfl_xor_sync(0xffffffffu, d, o);
    const float mn = fmaxf(m, d);
    const float base = mn == -INFINITY ? 0.f : mn;
    const float alpha = exp2f(m - base), pr = exp2f(d - base);
    m = mn;
    l = l * alpha + pr;
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[j] = acc[j] * alpha + pr * v[j];
  }
  T* out = static_cast<T*>(p.out) + row * p.out_token_stride + head * p.out_head_stride;
#pragma unroll
  for (int j = 0; j < 4; ++j) out[lane * 4 + j] = Elem<T>::from_float(limit > 0 ? acc[j] / l : 0.f);
}

}  // namespace

cudaError_t launch_int4_attention(const Int4Cache& c, const Int4AttnParams& p, int dtype,
                                  cudaStream_t stream) {
  const dim3 grid(p.num_q_tokens, (p.num_q_heads + kWarps - 1) / kWarps);
  if (dtype == B200_DTYPE_BFLOAT16)
    int4_attention_kernel<__nv_bfloat16><<<grid, kWarps * 32, 0, stream>>>(c, p);
  else
    int4_attention_kernel<__half><<<grid, kWarps * 32, 0, stream>>>(c, p);
  return cudaGetLastError();
}

}  // namespace b200
