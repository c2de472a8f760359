// What the two paths of attention over the paged 8-bit cache share: arguments, the rule that parts them, conversions.
#pragma once

#include "host.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace krnb {

constexpr int kErrDeviceIndex = 6;  // mirrors KRN_B200_ERR_DEVICE_INDEX in include/krn_b200.h

enum CacheAttnSite { kSitePage = 51, kSiteRows = 52, kSiteTile = 53, kSiteKeys = 54, kSiteValues = 55,
                     kSiteScores = 57, kSiteWeights = 58, kSiteOutput = 59, kSiteRoom = 60, kSiteRead = 61 };

struct PoolSide {
  const uint8_t* pages;
  const float* scale;  // [num_pages, kv_heads]
  long long page_pitch, token_pitch, head_pitch;
};

struct CacheAttnParams {
  const uint16_t* q;
  uint16_t* o;
  long long q_row, q_head, o_row, o_head, table_pitch;
  PoolSide k, v;
  const int32_t* page_table;
  const int32_t* context_len;
  const int32_t* row_start;
  int batch, rows, q_heads, kv_heads, group, page_shift, num_pages, max_new, max_context;
  uint32_t group_inverse;  // ceil(2^16 / group)
  int few;  // a request with at most this many rows (new tokens x q heads of a kv head) is streamed, one with more is tiled
  float scale_log2;
};

// Row `row` of a (request, kv head) is new token row / group, q head row % group of the kv head; for rows below 2^9 and
// groups up to 2^7, (row * ceil(2^16 / group)) >> 16 is that quotient.
struct RowAt {
  int token, head;
};

__device__ __forceinline__ RowAt row_at(const CacheAttnParams& a, int row) {
  const int token = int(uint32_t(row) * a.group_inverse >> 16);
  return {token, row - token * a.group};
}

// Whether request b's n rows can be computed: some, no more than announced, and all of them rows of q.
__device__ __forceinline__ bool rows_ok(const CacheAttnParams& a, int b, int n) {
  const int first = a.row_start[b];
  return n > 0 && n <= a.max_new && first >= 0 && first <= a.rows - n;
}

// Requests that have rows and cannot be computed are left out and reported.
__device__ __forceinline__ void report_rows(const CacheAttnParams& a, int b, DeviceStatus* status) {
  const int n = a.row_start[b + 1] - a.row_start[b];
  if (n > 0 && !rows_ok(a, b, n)) report_failure(status, kErrDeviceIndex, kSiteRows, uint32_t(n));
}

template <bool BF16>
__device__ __forceinline__ float2 unpack(uint32_t w) {
  if constexpr (BF16) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  } else {
    return __half22float2(*reinterpret_cast<const __half2*>(&w));
  }
}

// Two e4m3 codes in the low 16 bits, as f16.
__device__ __forceinline__ uint32_t halves_of(uint32_t codes) {
  uint32_t h2;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h2) : "h"(uint16_t(codes)));
  return h2;
}

// Boxes of `tokens` rows of one head.
inline int encode_pool(CUtensorMap* map, const PoolSide& side, int64_t d, int64_t kv_heads, int64_t page_size, int64_t num_pages,
                       uint32_t tokens, Swizzle swizzle) {
  uint64_t dims[4] = {uint64_t(d), uint64_t(kv_heads), uint64_t(page_size), uint64_t(num_pages)};
  uint64_t strides[3] = {uint64_t(side.head_pitch), uint64_t(side.token_pitch), uint64_t(side.page_pitch)};
  uint32_t box[4] = {uint32_t(d), 1, tokens, 1};
  return encode_tensor_map(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, side.pages, dims, strides, box, swizzle);
}

// Requests with many rows (cache_attn_tile.cu). `partial` holds tile_workspace() bytes. tile_blocks() bounds the blocks of
// query rows that they can have: with none there is nothing to launch.
int64_t tile_blocks(int64_t batch, int64_t rows, int64_t group, int64_t few);
int64_t tile_workspace(int64_t rows, int64_t q_heads, int64_t d, int64_t max_context);
int launch_tiles(const DeviceContext* ctx, const CacheAttnParams& a, bool bf16, int64_t d, int64_t page_size, float* partial,
                 cudaStream_t stream);
// Joins what launch_tiles() split over the keys, behind the kernels that were launched since.
int launch_tile_join(const CacheAttnParams& a, bool bf16, int64_t d, float* partial, cudaStream_t stream);

}  // namespace krnb
