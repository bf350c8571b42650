// kv_int4.cuh — the 4-bit KV cache: row format, page layout and the launch
// functions of the kernels that write it, read it back and attend over it.
//
// A row is the 128 values of one (slot, KV head) of K or V in four groups of
// 32 along head_dim. Per group, with a = max |x|:
//   s = bf16(a / 7) (nearest even; fp16 rows at most 9344, so 7 s is finite in
//       fp16), 0 below 2^-126, NaN where a is not finite
//   c = 8 + rne(fl32(x * fl32(1 / s))), 1..15 (8 where s is 0 or NaN)
// and the group stands for s * (c - 8). A row takes 64 bytes of codes (even
// elements in the low nibble) and 8 bytes of scales: 4.5 bits per value.
//
// A page of block_size slots holds, per tensor, all codes and then all scales,
// both head-major:
//   codes  [num_kv_heads][block_size][64 bytes]
//   scales [num_kv_heads][block_size][4] bf16
// so that the 16 rows of one (tile, head) are 1 KiB of codes and 128 bytes of
// scales, each contiguous, whatever the number of heads.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace b200 {

constexpr int kInt4GroupElems = 32;
constexpr int kInt4CodeBytes = 64;   // of a row
constexpr int kInt4ScaleBytes = 8;   // of a row
constexpr int kInt4RowBytes = kInt4CodeBytes + kInt4ScaleBytes;

struct Int4Cache {
  uint8_t* k;
  uint8_t* v;
  int64_t block_stride;  // bytes between consecutive pages, a multiple of 128
  int64_t num_blocks;
  int block_size;
  int num_kv_heads;
};

cudaError_t launch_store_kvcache_int4(const void* key, int64_t key_row_stride, const void* value,
                                      int64_t value_row_stride, int dtype, const Int4Cache& cache,
                                      const void* slots, bool slot64, int64_t num_tokens,
                                      int32_t* status, cudaStream_t stream);

cudaError_t launch_load_kvcache_int4(const Int4Cache& cache, const void* slots, bool slot64,
                                     int64_t num_tokens, void* key, int64_t key_row_stride,
                                     void* value, int64_t value_row_stride, int dtype,
                                     int32_t* status, cudaStream_t stream);

struct Int4DecodeParams {
  const void* q;
  int64_t q_seq_stride;
  int64_t q_head_stride;
  const int32_t* block_tables;
  int64_t block_table_stride;
  int max_blocks;
  const int32_t* seq_lens;
  void* out;
  int64_t out_seq_stride;
  int64_t out_head_stride;
  float* part_o;    // [2 num_parts, heads, head_dim]
  float* part_lse;  // [2 num_parts, heads], log2 domain
  int4* parts;      // [num_seqs, num_units]: where the parts of each are
  int num_parts;    // CTAs that share the batch
  int whole;        // instead a CTA for each (sequence, unit), nothing to join
  int block_size;
  int num_seqs;
  int num_q_heads;
  int group;      // q heads per KV head
  int splits;     // units of a KV head: 1, or 2 for groups of more than 8 heads
  int heads;      // q heads of a unit (the second may have one less)
  int num_units;  // num_kv_heads * splits
  Int4Cache cache;
  float scale_log2;
  int32_t* status;
};

cudaError_t launch_paged_decode_int4(const Int4DecodeParams& p, int dtype, cudaStream_t stream);
constexpr int kInt4DecodeTile = 32;   // tokens
constexpr int kInt4DecodeHeads = 8;   // q heads of a unit at most
int64_t int4_decode_ctas(int64_t tiles, int sms);  // that so many tiles are worth
bool int4_decode_whole(int64_t units, int64_t max_tiles, int sms);

struct Int4PrefillParams {
  const void* q;
  int64_t q_token_stride;
  int64_t q_head_stride;
  const int32_t* block_tables;
  int64_t block_table_stride;
  int max_blocks;  // valid columns of block_tables
  const int32_t* seq_lens;
  const int32_t* query_start_loc;
  int num_seqs;
  void* out;
  int64_t out_token_stride;
  int64_t out_head_stride;
  int group;       // q heads per KV head
  int inv_group;   // r / group = r * inv_group >> 16, r < 256
  int num_ctas;
  Int4Cache cache;
  uint32_t stride128;           // cache.block_stride / 128
  uint32_t div_mul, div_shift;  // t / block_size = umulhi(t, div_mul) >> div_shift, t < 2^31
  float scale_log2;
  int4* joins;     // [num_ctas]; with records: parts, first query row, rows, KV head
  float* records;  // [2 num_ctas], or nullptr: no unit is split
  int32_t* status;
};
constexpr int kInt4PrefillMinPart = 4;  // 128-token tiles of a part of a split unit at least
constexpr int kInt4PrefillCtas = 148;  // at most: one for each SM
constexpr int64_t kInt4PrefillRecordBytes = 2 * 130 * 128 * 4;
constexpr int64_t kInt4PrefillJoinBytes = (kInt4PrefillCtas * 16 + 255) / 256 * 256;
constexpr int64_t kInt4PrefillWorkspaceBytes =
    kInt4PrefillJoinBytes + 2 * kInt4PrefillCtas * kInt4PrefillRecordBytes;
cudaError_t launch_paged_prefill_int4(const Int4PrefillParams& p, int dtype, cudaStream_t stream);

}  // namespace b200
