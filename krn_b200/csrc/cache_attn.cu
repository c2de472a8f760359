// Attention over the paged 8-bit cache with one scale per (page, kv head): rows of q packed by request, row i of a request
// with n rows and a context of c tokens stands at position c - n + i and sees the keys up to it.
//
// One warp per (row, q head): each lane holds d / 32 columns, a key's score is a shuffle sum, one pass over the keys with a
// running maximum and sum.
#include "host.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cmath>

namespace krnb {
namespace {

constexpr int kErrDeviceIndex = 6;  // mirrors KRN_B200_ERR_DEVICE_INDEX in include/krn_b200.h

enum Site { kSitePage = 51, kSiteRows = 52 };

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
  float scale_log2;
};

template <bool BF16>
__device__ __forceinline__ float widen(uint16_t w) {
  if constexpr (BF16) return __uint_as_float(uint32_t(w) << 16);
  return __half2float(__ushort_as_half(w));
}

__device__ __forceinline__ float from_e4m3(uint32_t code) {
  uint32_t h2;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h2) : "h"(uint16_t(code)));
  return __half2float(__ushort_as_half(uint16_t(h2 & 0xffffu)));
}

template <int D, bool BF16>
__global__ void __launch_bounds__(128) cache_attn_kernel(CacheAttnParams p, DeviceStatus* status) {
  constexpr int kCols = D / 32;
  const int lane = int(lane_id());
  const int row = blockIdx.x, h = blockIdx.y * 4 + (threadIdx.x >> 5);
  if (h >= p.q_heads) return;
  int b = 0;
  while (b < p.batch && p.row_start[b + 1] <= row) ++b;
  if (b >= p.batch || p.row_start[b] > row) return;  // behind the last request
  const int n = p.row_start[b + 1] - p.row_start[b];
  const int context = max(0, min(p.context_len[b], p.max_context));
  if (n > p.max_new) {
    report_failure(status, kErrDeviceIndex, kSiteRows, uint32_t(n));
    return;
  }
  const int visible = context - n + (row - p.row_start[b]) + 1;
  const int g = h / p.group;
  float q[kCols], acc[kCols];
  for (int c = 0; c < kCols; ++c) {
    q[c] = widen<BF16>(p.q[row * p.q_row + h * p.q_head + lane * kCols + c]) * p.scale_log2;
    acc[c] = 0.f;
  }
  float m = -INFINITY, l = 0.f;
  for (int j = 0; j < visible; ++j) {
    const int page = p.page_table[b * p.table_pitch + (j >> p.page_shift)];
    const bool good = uint32_t(page) < uint32_t(p.num_pages);
    if (!good) report_failure(status, kErrDeviceIndex, kSitePage, uint32_t(page) & 0x7fffffffu);
    const int at = j & ((1 << p.page_shift) - 1);
    float s = 0.f;
    const uint8_t* key = p.k.pages + page * p.k.page_pitch + at * p.k.token_pitch + g * p.k.head_pitch + lane * kCols;
    const uint8_t* val = p.v.pages + page * p.v.page_pitch + at * p.v.token_pitch + g * p.v.head_pitch + lane * kCols;
    for (int c = 0; c < kCols; ++c) s += good ? q[c] * from_e4m3(key[c]) : 0.f;
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (good) s *= p.k.scale[(long long)page * p.kv_heads + g];
    const float m_new = fmaxf(m, s), corr = exp2f(m - m_new), w = exp2f(s - m_new);
    m = m_new;
    l = l * corr + w;
    const float wv = good ? w * p.v.scale[(long long)page * p.kv_heads + g] : 0.f;
    for (int c = 0; c < kCols; ++c) acc[c] = acc[c] * corr + (good ? wv * from_e4m3(val[c]) : 0.f);
  }
  for (int c = 0; c < kCols; ++c) {
    const float y = l > 0.f ? acc[c] / l : 0.f;
    p.o[row * p.o_row + h * p.o_head + lane * kCols + c] =
        BF16 ? uint16_t(pack_bf16x2(y, 0.f) & 0xffffu) : uint16_t(pack_f16x2(y, 0.f) & 0xffffu);
  }
}

template <int D, bool BF16>
int launch(const CacheAttnParams& p, DeviceStatus* status, cudaStream_t stream) {
  cache_attn_kernel<D, BF16><<<dim3(unsigned(p.rows), unsigned((p.q_heads + 3) / 4)), 128, 0, stream>>>(p, status);
  KRNB_CUDA(cudaGetLastError());
  return KRN_B200_OK;
}

}  // namespace
}  // namespace krnb

extern "C" int64_t krn_b200_cache_attn_workspace_bytes(int64_t batch, int64_t rows, int64_t q_heads, int64_t kv_heads, int64_t d,
                                                       int64_t max_new, int64_t max_context) {
  (void)batch, (void)rows, (void)q_heads, (void)kv_heads, (void)d, (void)max_new, (void)max_context;
  return 16;
}

extern "C" int krn_b200_cache_attn(int type, const void* q, const void* k_pages, const void* v_pages, const float* k_scale,
                                   const float* v_scale, const int32_t* page_table, const int32_t* context_len,
                                   const int32_t* row_start, void* o, int64_t batch, int64_t rows, int64_t q_heads,
                                   int64_t kv_heads, int64_t d, int64_t page_size, int64_t num_pages, int64_t max_pages,
                                   int64_t table_pitch, int64_t max_new, int64_t max_context, const int64_t* q_strides,
                                   const int64_t* o_strides, const int64_t* k_page_strides, const int64_t* v_page_strides,
                                   float scale_log2, void* workspace, int64_t workspace_bytes, void* stream_handle) {
  using namespace krnb;
  if (type != KRN_B200_BF16 && type != KRN_B200_F16) {
    return fail(KRN_B200_ERR_UNSUPPORTED, "attention element type %d is not available on sm_100a: queries come in 16 bits. "
                "Instead: pass bf16 or f16 tensors", type);
  }
  if (d != 64 && d != 128) {
    return fail(KRN_B200_ERR_UNSUPPORTED, "head dimension %lld is not available on sm_100a: tiles are built from 64- or 128-byte "
                "rows. Instead: use d = 64 or d = 128", (long long)d);
  }
  if (page_size < 16 || page_size > 256 || (page_size & (page_size - 1)) != 0) {
    return fail(KRN_B200_ERR_UNSUPPORTED, "page size %lld is not available on sm_100a: pages are 16, 32, 64, 128 or 256 tokens. "
                "Instead: use one of them", (long long)page_size);
  }
  if (batch < 0 || rows < 0 || q_heads <= 0 || kv_heads <= 0 || q_heads % kv_heads != 0 || num_pages <= 0 || max_pages <= 0 ||
      table_pitch < max_pages || max_new <= 0 || max_context <= 0) {
    return fail(KRN_B200_ERR_INVALID_ARGUMENT, "bad extents (batch %lld, %lld rows, %lld / %lld heads, %lld pages, table of %lld, "
                "max_new %lld, max_context %lld)", (long long)batch, (long long)rows, (long long)q_heads, (long long)kv_heads,
                (long long)num_pages, (long long)max_pages, (long long)max_new, (long long)max_context);
  }
  if (q_heads / kv_heads > 128) {
    return fail(KRN_B200_ERR_UNSUPPORTED, "%lld q heads per kv head is not available: a tile holds 128 rows. Instead: repeat the "
                "kv heads", (long long)(q_heads / kv_heads));
  }
  if (max_context > max_pages * page_size) {
    return fail(KRN_B200_ERR_INVALID_ARGUMENT, "max_context %lld does not fit %lld pages per sequence", (long long)max_context,
                (long long)max_pages);
  }
  if (batch == 0 || rows == 0) return KRN_B200_OK;
  if (batch > 65535 || kv_heads > 65535 || rows > INT32_MAX / 256 || rows * q_heads > INT32_MAX / 2 ||
      max_context > INT32_MAX / 2 || num_pages >= INT32_MAX) {
    return fail(KRN_B200_ERR_UNSUPPORTED, "extents too large for this kernel's 32-bit indices");
  }
  if (q == nullptr || k_pages == nullptr || v_pages == nullptr || k_scale == nullptr || v_scale == nullptr ||
      page_table == nullptr || context_len == nullptr || row_start == nullptr || o == nullptr || q_strides == nullptr ||
      o_strides == nullptr || k_page_strides == nullptr || v_page_strides == nullptr) {
    return fail(KRN_B200_ERR_INVALID_ARGUMENT, "null tensor address");
  }
  if (!aligned16(q) || !aligned16(o) || !aligned16(k_pages) || !aligned16(v_pages) || q_strides[0] % 8 || q_strides[1] % 8 ||
      o_strides[0] % 8 || o_strides[1] % 8) {
    return fail(KRN_B200_ERR_INVALID_ARGUMENT, "addresses and the strides of q and o must be multiples of 16 bytes");
  }
  for (int i = 0; i < 3; ++i) {
    if (k_page_strides[i] % 16 || v_page_strides[i] % 16 || k_page_strides[i] <= 0 || v_page_strides[i] <= 0) {
      return fail(KRN_B200_ERR_INVALID_ARGUMENT, "the strides of a page pool must be positive multiples of 16 bytes");
    }
  }
  const int64_t need = krn_b200_cache_attn_workspace_bytes(batch, rows, q_heads, kv_heads, d, max_new, max_context);
  if (workspace == nullptr || workspace_bytes < need) {
    return fail(KRN_B200_ERR_WORKSPACE, "workspace of %lld bytes is too small: %lld needed", (long long)workspace_bytes,
                (long long)need);
  }
  if (!aligned16(workspace)) return fail(KRN_B200_ERR_INVALID_ARGUMENT, "the workspace must be 16-byte aligned");
  DeviceContext* ctx = current_context();
  if (ctx == nullptr) return KRN_B200_ERR_CUDA;
  if (int rc = require_sm100(ctx)) return rc;
  CacheAttnParams p;
  p.q = static_cast<const uint16_t*>(q);
  p.o = static_cast<uint16_t*>(o);
  p.q_row = q_strides[0];
  p.q_head = q_strides[1];
  p.o_row = o_strides[0];
  p.o_head = o_strides[1];
  p.table_pitch = table_pitch;
  p.k = {static_cast<const uint8_t*>(k_pages), k_scale, k_page_strides[0], k_page_strides[1], k_page_strides[2]};
  p.v = {static_cast<const uint8_t*>(v_pages), v_scale, v_page_strides[0], v_page_strides[1], v_page_strides[2]};
  p.page_table = page_table;
  p.context_len = context_len;
  p.row_start = row_start;
  p.batch = int(batch);
  p.rows = int(rows);
  p.q_heads = int(q_heads);
  p.kv_heads = int(kv_heads);
  p.group = int(q_heads / kv_heads);
  p.page_shift = 0;
  while ((int64_t(1) << p.page_shift) < page_size) ++p.page_shift;
  p.num_pages = int(num_pages);
  p.max_new = int(max_new);
  p.max_context = int(max_context);
  p.scale_log2 = scale_log2;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_handle);
  const bool bf16 = type == KRN_B200_BF16;
  if (d == 128) return bf16 ? launch<128, true>(p, ctx->status_dev, stream) : launch<128, false>(p, ctx->status_dev, stream);
  return bf16 ? launch<64, true>(p, ctx->status_dev, stream) : launch<64, false>(p, ctx->status_dev, stream);
}
