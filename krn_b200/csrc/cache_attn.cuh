// What the two paths of attention over the paged 8-bit cache share: arguments and the rule that parts them.
#pragma once

#include "cache.cuh"

namespace krnb {

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

__device__ __forceinline__ uint4 ld_shared_16(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
  return v;
}

// Boxes of `tokens` rows of one head.
inline int encode_pool(CUtensorMap* map, const PoolSide& side, int64_t d, int64_t kv_heads, int64_t page_size, int64_t num_pages,
                       uint32_t tokens, Swizzle swizzle) {
  uint64_t dims[4] = {uint64_t(d), uint64_t(kv_heads), uint64_t(page_size), uint64_t(num_pages)};
  uint64_t strides[3] = {uint64_t(side.head_pitch), uint64_t(side.token_pitch), uint64_t(side.page_pitch)};
  uint32_t box[4] = {uint32_t(d), 1, tokens, 1};
  return encode_tensor_map(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, side.pages, dims, strides, box, swizzle);
}

// ---- requests with many rows (cache_attn_tile.cu)

constexpr int kTileQ = 128;        // rows of a query tile; a block has two
constexpr int kSMs = 148;          // blocks that run at once: fewer may be split over the keys
constexpr float kNone = -3.0e38f;  // reference maximum of a row that has seen no key

// What the join has to know of the split blocks.
struct SplitHeader {
  int2 split;            // shares of each block's keys, blocks x kv heads
  int2 block[kSMs / 2];  // request and first token of each
};
constexpr int kHeaderBytes = (sizeof(SplitHeader) + 15) / 16 * 16;

struct TileShares {
  SplitHeader* header;  // null: nothing is split
  float* partial;       // [shares, blocks, 2 * kTileQ rows, d + 4]: m, l, two unused, the unnormalised output
  int tokens;           // tokens of a query tile: 128 / group
};

// kRows rows a warp at a time: their loads hide each other's latency.
template <int D, bool BF16, int kRows>
__device__ __forceinline__ void join_rows(const CacheAttnParams& a, const TileShares& p, int shares, int units, int warp, int warps) {
  constexpr int kCols = D / 32, kLanes = 32 / kRows;  // a lane's columns; lanes that look for a row's maximum
  const int lane = int(lane_id());
  const long long stride = (long long)units * 2 * kTileQ * (D + 4);
  for (int i = warp * kRows; i < units * 2 * kTileQ; i += warps * kRows) {
    const int unit = i / (2 * kTileQ), first = i % (2 * kTileQ);
    const int2 block = p.header->block[unit];
    const float* from = p.partial + (long long)i * (D + 4);
    float high = kNone;
    for (int s = lane % kLanes; s < shares; s += kLanes) high = fmaxf(high, from[s * stride + lane / kLanes * (D + 4)]);
#pragma unroll
    for (int o = 1; o < kLanes; o <<= 1) high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, o));
    float m[kRows], l[kRows], acc[kRows][kCols];
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      m[r] = __shfl_sync(0xffffffffu, high, r * kLanes);
      l[r] = 0.f;
#pragma unroll
      for (int c = 0; c < kCols; ++c) acc[r][c] = 0.f;
    }
#pragma unroll(8 / kRows)
    for (int s = 0; s < shares; ++s) {
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        const float* at = from + s * stride + r * (D + 4);
        const float2 ml = *reinterpret_cast<const float2*>(at);
        float x[kCols];
        if constexpr (D == 128) {
          const float4 v = *reinterpret_cast<const float4*>(at + 4 + lane * 4);
          x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
        } else {
          const float2 v = *reinterpret_cast<const float2*>(at + 4 + lane * 2);
          x[0] = v.x, x[1] = v.y;
        }
        const bool seen = ml.y != 0.f;  // some key of this share
        const float by = ex2_approx(ml.x - m[r]);
        l[r] += seen ? ml.y * by : 0.f;
#pragma unroll
        for (int c = 0; c < kCols; ++c) acc[r][c] += seen ? x[c] * by : 0.f;
      }
    }
    const int row0 = a.row_start[block.x], n = a.row_start[block.x + 1] - row0;
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      const RowAt where = row_at(a, (first + r) % kTileQ);
      const int token = block.y + (first + r) / kTileQ * p.tokens + where.token;
      if (where.token >= p.tokens || token >= n) continue;  // no row: nothing was written of it
      const float by = l[r] == 0.f ? 0.f : 1.0f / l[r];
      uint32_t w[kCols / 2];
#pragma unroll
      for (int c = 0; c < kCols / 2; ++c) {
        const float x = acc[r][2 * c] * by, y = acc[r][2 * c + 1] * by;
        w[c] = BF16 ? pack_bf16x2(x, y) : pack_f16x2(x, y);
      }
      uint16_t* out = a.o + (long long)(row0 + token) * a.o_row + (long long)(unit % a.kv_heads * a.group + where.head) * a.o_head + lane * kCols;
      if constexpr (D == 128) *reinterpret_cast<uint2*>(out) = make_uint2(w[0], w[1]);
      else *reinterpret_cast<uint32_t*>(out) = w[0];
    }
  }
}

// Joins the shares of split blocks, by block `part` of `parts`, `split` being the first two words of the header: a row a warp
// where there are warps enough (few blocks have many shares), else four. What was not split, and rows behind the last request, are not touched.
template <int D, bool BF16>
__device__ __forceinline__ void join_shares(const CacheAttnParams& a, const TileShares& p, int2 split, int part, int parts) {
  const int shares = split.x, units = split.y;
  if (shares == 1) return;
  const int each = int(blockDim.x) >> 5, warp = part * each + int(threadIdx.x >> 5), warps = parts * each;
  if (units * 2 * kTileQ <= warps) join_rows<D, BF16, 1>(a, p, shares, units, warp, warps);
  else join_rows<D, BF16, 4>(a, p, shares, units, warp, warps);
}

// tile_blocks() bounds the blocks of query rows: with none there is nothing to launch. `workspace` holds tile_workspace()
// bytes. The shares of what was split are joined behind the kernels that were launched since, by launch_tile_join() or a
// kernel that calls join_shares().
int64_t tile_blocks(int64_t batch, int64_t rows, int64_t group, int64_t few);
int64_t tile_workspace(int64_t batch, int64_t rows, int64_t q_heads, int64_t kv_heads, int64_t d, int64_t few, int64_t max_context);
TileShares tile_shares(const CacheAttnParams& a, void* workspace);
int launch_tiles(const DeviceContext* ctx, const CacheAttnParams& a, const TileShares& shares, bool bf16, int64_t d, int64_t page_size,
                 cudaStream_t stream);
int launch_tile_join(const CacheAttnParams& a, const TileShares& shares, bool bf16, int64_t d, cudaStream_t stream);

}  // namespace krnb
