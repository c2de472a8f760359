// Attention of many query rows (prompts, chunks of prompts) over the paged 8-bit cache: tensor-core tiles.
//
// A block owns two tiles of 128 query rows of one (request, kv head): 128 / group consecutive tokens of each q head that
// shares the kv head, so K and V are fetched once for the whole group. It runs over the keys in tiles of 128:
//
//   warp 0        issues S = Q_t K^T (kind::f8f6f4) on the cache's bytes as they are;
//   warp 1        issues O_t += P_t V (kind::f16);
//   warp 2        issues the copies (TMA): K codes into a ring of kKStages tiles, V codes into a ring of two;
//   warps 4..7    turn a V tile into f16, times its pages' scales: a 16-bit P needs a 16-bit V;
//   warps 8..15   softmax of the two query tiles, a thread per row; then the output.
//
// Q is split into 8-bit parts, each the rounded remainder of the ones before (a power-of-two factor puts the row's largest
// magnitude into [128, 256)): e4m3, the last one e5m2, whose three significant bits are what is left of a value by then and whose
// range goes seven octaves further down. Two parts hold bf16's 8 significant bits exactly down to 2^-13 of the row's largest
// magnitude, three hold f16's 11 down to 2^-10; below, the remainder is at most 2^-21 of it (2^-17 with an e4m3 part in the last
// place). S is the sum over the parts, and two 8-bit products take the tensor cores as long as one of 16 bits, so K needs no
// conversion at all.
//
// A page's key scale multiplies its columns of S in f32, before the maximum. Its value scale multiplies V, relative to the
// largest one that this block meets and times 2^7 (448 * 2^7 is within f16): for scales that are powers of two V stays
// exact down to 2^-22 of the largest; any other scale costs two roundings of at most 2^-11, small beside bf16's 2^-8. f16
// outputs would show them: there only the power of two in the scale goes to V, and the rest of it to P before its rounding.
//
// Weights are f16 in P, relative to a reference that the row's maximum may pass by 8 octaves before O is rescaled, and lifted by
// 2^7 (f16 outputs 2^6), which l carries too, so that it leaves with the division: a weight has eleven bits down to 2^-21 (2^-20)
// of the row's largest and vanishes at 2^-32 (2^-31). Without the lift, outputs made of small weights lost them: 2 % of a result
// where one key of 8192 lies 21.7 octaves above the others and has a value of zero, 7 % with 131072 keys and 23.2 octaves. A
// rescale at 7 / 6 / 5 octaves with a lift of 8 / 9 / 10 takes 1 / 2 / 4 % more time for a prompt of 8192 tokens.
//
// Tensor memory (512 columns): S (128) | P0 (64) | P1 (64) | O0 (128) | O1 (128). The two query tiles take turns in one S:
// a softmax warp reads its scores into registers at once, so S is free for the other tile's scores long before the
// exponentials are done, and each tile finds its next scores ready when it has handed over its weights. Two warps issue,
// because one sets the pace: it spends over a hundred cycles on each wait and about 80 on each product, 2030 cycles a query
// and key tile in a trace, of which the tensor cores work 1024.
//
// A step of both query tiles takes 3170 cycles in a trace, of which the exponentials need 2048 (16 a cycle) and the products about
// 2580 from issue to end, 2048 by arithmetic; counters have tensor cores and special-function units busy for 60 % of the active
// cycles each, the set-up of a block included. That the products wait for shared memory, which they read beside the conversion's
// traffic, is a guess. A prompt of 8192 tokens, 8 kv heads of 128, group 4: 465 to 545 us by the box = 1180 to 1010 TFLOP/s under the
// power limit; f16, with a product and a half for the scores: 510 to 550; d = 64: 410 to 460. Two threads a query row (16 softmax
// warps of 104 registers) shorten the chain of a query tile and not the step: 72 against 69 us for four chunks of 512 over 4096.
#include "cache_attn.cuh"

namespace krnb {
namespace {

constexpr int kTileKV = 128;
constexpr int kThreads = 512;
constexpr int kRegsFew = 40, kRegsMany = 216;  // warps 0..7 / 8..15, of the 128 that each thread is launched with
constexpr int kShortest = 4;              // key tiles of a share, at least
constexpr float kStreamWork = 0.5f;       // a streamed request's 128 keys, in steps of a block: 25 us on all SMs for 36 requests
                                          // of 4096 tokens and 4 kv heads of 128, at 1.7 us a step
constexpr float kRescaleThreshold = 8.0f;           // octaves by which a row's maximum may pass its reference
constexpr float kLift = 15.0f - kRescaleThreshold;  // octaves that weights are lifted by: the largest stay below f16's 2^16

struct TileParams {
  CacheAttnParams a;
  TileShares shares;
  int room;  // shares that the workspace holds
};

template <int D, int Parts>
struct Layout {
  static constexpr int kKStages = D == 128 && Parts == 3 ? 2 : 3;
  static constexpr int kPerRow = 128 / D;                               // parts in a 128-byte row of Q
  static constexpr int kQBlocks = (Parts + kPerRow - 1) / kPerRow;
  static constexpr int kQBytes = kQBlocks * kTileQ * 128;               // one query tile
  static constexpr int kRawBytes = kTileKV * D;                         // a tile of codes
  static constexpr int kHalfBytes = kTileKV * D * 2;                    // a tile of V in f16
  static constexpr int kBlockBytes = 128 * 128;                         // [128 rows x 128 bytes]
  static constexpr int kOffK = 2 * kQBytes;
  static constexpr int kOffRaw = kOffK + kKStages * kRawBytes;
  static constexpr int kOffHalf = kOffRaw + 2 * kRawBytes;
  static constexpr int kOffTail = kOffHalf + 2 * kHalfBytes;
  static constexpr int kSmemBytes = kOffTail + 528 + 2 * kTileQ * 4 + 1024;
};

__device__ __forceinline__ void tie(uint32_t (&r)[32]) {
  asm volatile("" : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
                   "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]),
                   "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
               :: "memory");
}

// K-major operand rows of 64 bytes, 64-byte swizzle (what TMA writes with that mode): 8-row groups are 512 bytes apart.
__device__ __forceinline__ uint64_t desc_kmajor_sw64(uint32_t smem_addr) {
  uint64_t desc = 0;
  desc |= static_cast<uint64_t>((smem_addr & 0x3FFFFu) >> 4);
  desc |= static_cast<uint64_t>(1) << 16;
  desc |= static_cast<uint64_t>(512 >> 4) << 32;
  desc |= static_cast<uint64_t>(1) << 46;
  desc |= static_cast<uint64_t>(4) << 61;
  return desc;
}

__device__ __forceinline__ void st_shared_16(uint32_t addr, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}

// One lane polls, the warp follows. (For a warp that has others of its kind to wait with, polling with every lane is faster:
// 3170 against 3450 cycles a key tile for the softmax warps.)
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag, DeviceStatus* status, int site) {
  bool ok = true;
  if (lane_id() == 0) ok = mbar_wait(bar, parity, abort_flag, status, site);
  return __all_sync(0xffffffffu, ok);
}

__device__ __forceinline__ uint32_t times(uint32_t a, uint32_t b) {  // f16x2
  uint32_t r;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

// Blocks of two query tiles that request b has on this path.
__device__ __forceinline__ int blocks_of(const TileParams& p, int b) {
  const int n = p.a.row_start[b + 1] - p.a.row_start[b];
  if (!rows_ok(p.a, b, n) || (long long)n * p.a.group <= p.a.few) return 0;
  return (n + 2 * p.shares.tokens - 1) / (2 * p.shares.tokens);
}

// The scales of the 16-token groups of key tiles, one group per lane of 8 (a warp may have two of them). Page ids are fetched two tiles ahead and scales
// one, by a call placed where a tile's long work follows. Groups without a page in the pool have the scale `none`.
struct ScaleAhead {
  const int32_t* table;
  const float* scale;
  int shift, pages, num_pages, heads, head, lane;
  float none;
  int id;
  float next;
  __device__ __forceinline__ int id_at(int tile) const {
    const int at = (tile * kTileKV + (lane & 7) * 16) >> shift;
    return at < pages ? table[at] : -1;
  }
  __device__ __forceinline__ float scale_at(int page) const {
    return uint32_t(page) < uint32_t(num_pages) ? scale[(long long)page * heads + head] : none;
  }
  __device__ __forceinline__ void start(int tile) {
    next = scale_at(id_at(tile));
    id = id_at(tile + 1);
  }
  // `next` is the scale of `tile` before the call and that of tile + 1, on its way, after it.
  __device__ __forceinline__ void fetch(int tile) {
    next = scale_at(id);
    id = id_at(tile + 2);
  }
};

template <int D, bool BF16, int Groups>
__global__ void __launch_bounds__(kThreads, 1)
cache_tile_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, TileParams p,
                  DeviceStatus* status) {
  constexpr int Parts = BF16 ? 2 : 3, kGroup = kTileKV / Groups;  // keys of a scale
  using L = Layout<D, Parts>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  uint8_t* smem = smem_raw + (base - raw);
  const CacheAttnParams& a = p.a;

  const uint32_t q_addr = base, k_addr = base + L::kOffK, raw_addr = base + L::kOffRaw, half_addr = base + L::kOffHalf;
  uint8_t* tail = smem + L::kOffTail;
  const uint32_t bars = smem_u32(tail);
  const uint32_t k_full = bars + 8, k_empty = bars + 32, raw_full = bars + 56, raw_empty = bars + 72;
  const uint32_t v_full = bars + 88, v_empty = bars + 104, s_full = bars + 120, p_full = bars + 136, o_full = bars + 152;
  const uint32_t s_read = bars + 168;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tail + 176);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tail + 180);
  int32_t* found = reinterpret_cast<int32_t*>(tail + 184);  // request, block of it, blocks of it
  int4* sums = reinterpret_cast<int4*>(tail + 208);         // [kThreads / 32]
  float* tops = reinterpret_cast<float*>(tail + 464);       // [kThreads / 32]
  float* row_scales = reinterpret_cast<float*>(tail + 528); // [2 * kTileQ]

  const int warp = threadIdx.x >> 5;
  const int lane = int(lane_id());

  wait_for_kernel_before();
  launch_dependents();  // what comes beside needs what came before
  // ---- the batch's blocks and their work
  if (threadIdx.x == 0) {
    found[0] = -1;
    *abort_flag = 0;
  }
  int blocks = 0, start = 0, own = 0, longest = 0;
  float work = 0.f;  // key tiles of this path's blocks, and what the stream has to do in that measure
  const auto count_blocks = [&](int first) {  // requests first, ..., one a thread: `blocks` goes on, `start` is the request's own
    const int b = first + int(threadIdx.x);
    own = b < a.batch ? blocks_of(p, b) : 0;
    int v = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int below = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v += below;
    }
    const int steps = b < a.batch ? (max(0, min(a.context_len[b], a.max_context)) + kTileKV - 1) / kTileKV : 0;
    float mine = own > 0 ? float(own) * float(steps) : kStreamWork * float(steps);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
    const int high = __reduce_max_sync(0xffffffffu, own > 0 ? steps : 0);
    __syncthreads();
    if (lane == 31) sums[warp] = make_int4(v, high, __float_as_int(mine), 0);
    __syncthreads();
    start = blocks + v - own;
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) {
      const int4 s = sums[w];
      if (w < warp) start += s.x;
      blocks += s.x;
      longest = max(longest, s.y);
      work += __int_as_float(s.z);
    }
  };
  for (int first = 0; first < a.batch; first += kThreads) {
    count_blocks(first);
    if (blockIdx.x == 0 && first + int(threadIdx.x) < a.batch) report_rows(a, first + int(threadIdx.x), status);
  }
  // ---- shares of the keys: so many that the longest block takes little longer than all work spread over the GPU. The kernel
  // decides, which knows the lengths: the host's bounds are loose where rows are padded or decode requests are among them.
  // One request of 40 new tokens, 4 kv heads of 128, over 2000 / 8000 / 60000 tokens: 23 / 26 / 55 us, 42 / 138 / 968 with
  // one share; 512 new tokens over 8000 / 60000: 51 / 237, 110 / 765 with one; 64 new tokens in 4096 padded rows over 8192
  // tokens, 8 kv heads: 31, 114 with one; beside 36 decode requests, all over 32768 tokens, 4 kv heads: 351, 452 with one.
  // With more shares than this, 2 x 512 new tokens beside 36 decode requests over 4096: 73 -> 89 us (nothing runs beside).
  const int units = blocks * a.kv_heads;
  const float even = fmaxf(work * float(a.kv_heads) * (1.0f / kSMs), float(kShortest));
  const int splits = units == 0 ? 1 : max(1, min(p.room / units, int(float(longest) / even + 0.75f)));
  if (blockIdx.x == 0 && threadIdx.x == 0 && p.shares.header != nullptr) {
    p.shares.header->split = make_int2(splits, units);
  }
  // ---- whose block this is: requests in order, the last (longest) block of a request first
  if (int(blockIdx.x) >= units * splits) return;  // the whole block: the grid is sized by a bound
  const int split = int(blockIdx.x) / units, unit = int(blockIdx.x) - split * units;
  const int g = unit % a.kv_heads, wanted = unit / a.kv_heads;
  if (a.batch > kThreads) blocks = 0;
  for (int first = 0; first < a.batch; first += kThreads) {
    if (a.batch > kThreads) count_blocks(first);
    if (wanted >= start && wanted < start + own) {
      found[0] = first + int(threadIdx.x);
      found[1] = own - 1 - (wanted - start);
    }
    if (blocks > wanted) break;
  }
  __syncthreads();
  const int b = found[0];
  if (b < 0) return;
  const int row0 = a.row_start[b], n = a.row_start[b + 1] - row0;
  const int context = max(0, min(a.context_len[b], a.max_context));
  const int token0 = found[1] * 2 * p.shares.tokens;  // first token of query tile 0
  if (splits > 1 && split == 0 && threadIdx.x == 0) p.shares.header->block[unit] = make_int2(b, token0);
  const int32_t* table = a.page_table + b * a.table_pitch;
  const int pages = (context + (1 << a.page_shift) - 1) >> a.page_shift;

  // ---- key tiles: up to the position of a query tile's last token, this split's share of them
  int counts[2];
  int most = 0;
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const int last = min(n, token0 + (t + 1) * p.shares.tokens) - 1;  // last token of the tile
    const int keys = token0 + t * p.shares.tokens < n ? max(0, min(context, context - n + last + 1)) : 0;
    counts[t] = (keys + kTileKV - 1) / kTileKV;
    most = max(most, counts[t]);
  }
  const int j0 = int((long long)most * split / splits), j1 = int((long long)most * (split + 1) / splits);
  const int n0 = max(0, min(counts[0], j1) - j0), n1 = max(0, min(counts[1], j1) - j0);
  const int count = max(n0, n1);

  // ---- the pages of these keys, one a thread, and behind them the largest value scale: their loads come around the others'
  const int first_page = (j0 * kTileKV) >> a.page_shift, end_page = min(pages, (((j0 + count) * kTileKV - 1) >> a.page_shift) + 1);
  int scan_page = first_page + int(threadIdx.x) < end_page ? table[first_page + int(threadIdx.x)] : 0;
  auto scan = [&](int at, int page) -> float {  // ids outside the pool are reported
    if (at >= end_page) return 0.f;
    if (uint32_t(page) < uint32_t(a.num_pages)) return fabsf(a.v.scale[(long long)page * a.kv_heads + g]);
    report_failure(status, kErrDeviceIndex, kSitePage, uint32_t(page) & 0x7fffffffu);
    return 0.f;
  };

  // ---- Q: every thread takes 16 bytes of some rows; what it loads arrives while the rest is set up
  constexpr int kQLanes = D / 8, kQRows = kThreads / kQLanes, kQPasses = 2 * kTileQ / kQRows;
  const int q_lane = int(threadIdx.x) % kQLanes, q_row = int(threadIdx.x) / kQLanes;
  uint4 q_words[kQPasses];
#pragma unroll
  for (int i = 0; i < kQPasses; ++i) {
    const int row = i * kQRows + q_row, in_tile = row % kTileQ;
    const RowAt at = row_at(a, in_tile);
    const int token = token0 + (row / kTileQ) * p.shares.tokens + at.token;
    const bool live = at.token < p.shares.tokens && token < n && row0 + token < a.rows;
    const uint16_t* src = a.q + (long long)(row0 + token) * a.q_row + (long long)(g * a.group + at.head) * a.q_head + q_lane * 8;
    q_words[i] = live ? *reinterpret_cast<const uint4*>(src) : make_uint4(0, 0, 0, 0);
  }

  // Copies of K and V tile j, a lane each, by warp 2; page ids come 32 at a time.
  const int box = min(kTileKV, 1 << a.page_shift), copies = kTileKV / box;
  int ids = 0, ids_first = -64;
  auto copy = [&](const CUtensorMap* map, int j, uint32_t dst, uint32_t bar) {
    const int token = (j0 + j) * kTileKV, first_page = token >> a.page_shift;
    if (first_page < ids_first || first_page + copies > ids_first + 32) {
      ids_first = first_page;
      ids = first_page + lane < pages ? table[first_page + lane] : 0;
    }
    int page = __shfl_sync(0xffffffffu, ids, (first_page + lane - ids_first) & 31);
    if (uint32_t(page) >= uint32_t(a.num_pages)) page = a.num_pages;  // one past the pool: TMA fills zeros
    const int there = min(copies, pages - first_page);
    if (lane == 0) mbar_arrive_expect_tx(bar, uint32_t(there) * uint32_t(box) * D);
    __syncwarp();
    if (lane < there) tma_load_4d(dst + lane * box * D, map, 0, g, token & ((1 << a.page_shift) - 1), page, bar);
  };
  auto copy_k = [&](int j) { copy(&map_k, j, k_addr + (j % L::kKStages) * L::kRawBytes, k_full + 8 * (j % L::kKStages)); };
  auto copy_v = [&](int j) { copy(&map_v, j, raw_addr + (j & 1) * L::kRawBytes, raw_full + 8 * (j & 1)); };
  if (warp == 2) {
    if (lane == 0) {
      mbar_init(s_read, 4);
      for (int i = 0; i < 3; ++i) {
        mbar_init(k_full + 8 * i, 1);
        mbar_init(k_empty + 8 * i, 1);
      }
      for (int i = 0; i < 2; ++i) {
        mbar_init(raw_full + 8 * i, 1);
        mbar_init(raw_empty + 8 * i, 4);
        mbar_init(v_full + 8 * i, 4);
        mbar_init(v_empty + 8 * i, 1);
        mbar_init(s_full + 8 * i, 1);
        mbar_init(p_full + 8 * i, 4);
        mbar_init(o_full + 8 * i, 1);
      }
      fence_mbar_init();
    }
    __syncwarp();
    for (int j = 0; j < min(count, 2); ++j) {  // both rings have room for two
      copy_k(j);
      copy_v(j);
    }
  }
  if (warp == 1) {
    tmem_alloc<1>(smem_u32(tmem_slot), 512);
    tmem_relinquish<1>();
  }
  float top = scan(first_page + int(threadIdx.x), scan_page);

  // ---- Q as 8-bit parts
#pragma unroll
  for (int i = 0; i < kQPasses; ++i) {
    const int row = i * kQRows + q_row, in_tile = row % kTileQ;
    const uint32_t words[4] = {q_words[i].x, q_words[i].y, q_words[i].z, q_words[i].w};
    float2 v[4];
    float size = 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      v[e] = unpack<BF16>(words[e]);
      size = fmaxf(size, fmaxf(fabsf(v[e].x), fabsf(v[e].y)));
    }
#pragma unroll
    for (int o = 1; o < kQLanes; o <<= 1) size = fmaxf(size, __shfl_xor_sync(0xffffffffu, size, o));
    const int up = max(-120, min(126, 7 - (int(__float_as_uint(size) >> 23) - 127)));
    const float by = copysignf(__uint_as_float(uint32_t(up + 127) << 23), a.scale_log2);
    if (q_lane == 0) {
      const float back = __uint_as_float(uint32_t(127 - up) << 23) * fabsf(a.scale_log2);
      row_scales[row] = size > 3.4028234663852886e38f ? __int_as_float(0x7fffffff) : back;  // no factor brings an infinity back
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = __fmul2_rn(v[e], make_float2(by, by));
    const uint32_t row_addr = q_addr + (row / kTileQ) * L::kQBytes + in_tile * 128 + (q_lane & 1) * 8;
#pragma unroll
    for (int part = 0; part < Parts; ++part) {
      uint32_t code[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        uint16_t two;
        if (part + 1 == Parts) {
          asm("cvt.rn.satfinite.e5m2x2.f32 %0, %1, %2;" : "=h"(two) : "f"(v[e].y), "f"(v[e].x));
          code[e] = two;
        } else {
          asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(two) : "f"(v[e].y), "f"(v[e].x));
          code[e] = two;
          const uint32_t h = halves_of(two);
          const float2 back = __half22float2(*reinterpret_cast<const __half2*>(&h));
          v[e].x -= back.x;
          v[e].y -= back.y;
        }
      }
      const uint32_t chunk = uint32_t((part % L::kPerRow) * (D / 16) + (q_lane >> 1));
      const uint32_t at = row_addr + (part / L::kPerRow) * L::kBlockBytes + ((chunk ^ (uint32_t(in_tile) & 7u)) << 4);
      asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(at), "r"(code[0] | code[1] << 16), "r"(code[2] | code[3] << 16) : "memory");
    }
  }
  for (int at = first_page + int(threadIdx.x) + kThreads; at < end_page; at += kThreads) top = fmaxf(top, scan(at, table[at]));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (lane == 0) tops[warp] = top;
  fence_async_smem();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  top = 0x1p-110f;  // smaller value scales are held against it
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) top = fmaxf(top, tops[w]);

  if (warp < 8) reg_dealloc<kRegsFew>();
  if (warp < 2) {
    // ---------------------------------------------------------------- MMA issuers: warp 0 the scores, warp 1 P V
    const bool leader = elect_one();
    const int nt[2] = {n0, n1};
    auto wait = [&](uint32_t bar, uint32_t parity, int site) {
      return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, status, site)) != 0;
    };
    bool ok = true;
    if (warp == 0) {
      constexpr uint32_t kIdesc = umma_idesc(kFmtE4M3, kFmtE4M3, kTileQ, kTileKV, 0, 0);
      constexpr uint32_t kIdescLast = umma_idesc(kFmtE5M2, kFmtE4M3, kTileQ, kTileKV, 0, 0);  // Q's last part
      const uint64_t q_desc = umma_desc_kmajor_sw128(0);
      const uint64_t k_desc = D == 128 ? umma_desc_kmajor_sw128(0) : desc_kmajor_sw64(0);
      const uint32_t q_hi = uint32_t(q_desc >> 32), k_hi = uint32_t(k_desc >> 32);
      const uint32_t q_lo = uint32_t(q_desc) + (q_addr >> 4), k_lo = uint32_t(k_desc) + (k_addr >> 4);
      int stage = 0;
      uint32_t phase = 0, reads = 0;  // reads: score tiles issued so far, each of which a softmax reads once
      for (int j = 0; j < count && ok; ++j) {
        ok = wait(k_full + 8 * stage, phase, kSiteKeys);
        for (int t = 0; t < 2 && ok; ++t) {
          if (j >= nt[t]) continue;
          if (reads > 0 && !wait(s_read, (reads - 1) & 1, kSiteRead)) {
            ok = false;
            break;
          }
          ++reads;
          tc_fence_after();
          // S = sum over Q's parts: D / 32 instructions of K = 32 columns each
          const uint32_t qa = q_lo + t * (L::kQBytes >> 4), ka = k_lo + stage * (L::kRawBytes >> 4);
          if (leader) {
#pragma unroll
            for (int part = 0; part < Parts; ++part) {
#pragma unroll
              for (int ks = 0; ks < D / 32; ++ks) {
                const uint32_t off = ((part / L::kPerRow) * L::kBlockBytes + (part % L::kPerRow) * D + ks * 32) >> 4;
                umma_ss_halves<1, true>(tmem_base, qa + off, q_hi, ka + ks * 2, k_hi, part + 1 == Parts ? kIdescLast : kIdesc,
                                        part + ks > 0 ? 1u : 0u);
              }
            }
            umma_commit(s_full + 8 * t);
          }
          __syncwarp();
        }
        if (ok && leader) umma_commit(k_empty + 8 * stage);
        __syncwarp();
        if (++stage == L::kKStages) {
          stage = 0;
          phase ^= 1u;
        }
      }
    } else {
      const uint32_t idesc = umma_idesc(kFmtF16, kFmtF16, kTileQ, D, 0, 1);
      const uint64_t v_desc = umma_desc_mnmajor_sw128(0, L::kBlockBytes, 1024);
      const uint32_t v_hi = uint32_t(v_desc >> 32), v_lo = uint32_t(v_desc) + (half_addr >> 4);
      for (int j = 0; j < count && ok; ++j) {
        const int stage = j & 1;
        ok = wait(v_full + 8 * stage, (j >> 1) & 1, kSiteValues);
        for (int t = 0; t < 2 && ok; ++t) {
          if (j >= nt[t]) continue;
          if (!wait(p_full + 8 * t, j & 1, kSiteWeights)) {
            ok = false;
            break;
          }
          tc_fence_after();
          // O_t += P_t V: 8 instructions of K = 16 keys; P_t from tensor memory, V with d contiguous in 64-column blocks
          const uint32_t va = v_lo + stage * (L::kHalfBytes >> 4);
          if (leader) {
#pragma unroll
            for (int ks = 0; ks < kTileKV / 16; ++ks) {
              umma_ts_f16_halves(tmem_base + 256 + t * 128, tmem_base + 128 + t * 64 + ks * 8, va + ks * (2048 >> 4), v_hi, idesc,
                                 (j > 0 || ks > 0) ? 1u : 0u);
            }
            umma_commit(o_full + 8 * t);
          }
          __syncwarp();
        }
        if (ok && leader) umma_commit(v_empty + 8 * stage);
        __syncwarp();
      }
    }
  } else if (warp == 2) {
    // ---------------------------------------------------------------- copies behind the first two
    for (int j = 2; j < count; ++j) {
      const int stage = j % L::kKStages;
      if (!warp_wait(k_empty + 8 * stage, ((j / L::kKStages) & 1) ^ 1u, abort_flag, status, kSiteKeys)) break;
      copy_k(j);
      if (!warp_wait(raw_empty + 8 * (j & 1), ((j >> 1) & 1) ^ 1u, abort_flag, status, kSiteValues)) break;
      copy_v(j);
    }
  } else if (warp >= 4 && warp < 8) {
    // ---------------------------------------------------------------- V to f16
    constexpr int kLanes = D / 16;               // threads per row, 16 codes each
    constexpr int kRows = 128 / kLanes;          // rows per pass of the four warps
    const int tid = int(threadIdx.x) - 128;
    const int row_of = tid / kLanes, c = tid % kLanes;
    ScaleAhead scales = {table, a.v.scale, a.page_shift, pages, a.num_pages, a.kv_heads, g, lane, 0.f, 0, 0.f};
    if (count > 0) scales.start(j0);
    const float unit = 128.0f / top;
    // a thread's two stores, in an order that spreads a row over all banks
    const uint32_t turn = uint32_t(c >> 2) & 1u, even = uint32_t(2 * c) & 7u;
    for (int j = 0; j < count; ++j) {
      const int stage = j & 1;
      float factor = scales.next * unit;
      if (!BF16) factor = __uint_as_float(__float_as_uint(factor) & 0x7f800000u);
      scales.fetch(j0 + j);
      const uint32_t mine = pack_f16x2(factor, factor);
      const bool ok = mbar_wait(raw_full + 8 * stage, (j >> 1) & 1, abort_flag, status, kSiteValues) &&
                      mbar_wait(v_empty + 8 * stage, ((j >> 1) & 1) ^ 1u, abort_flag, status, kSiteRoom);
      if (!__all_sync(0xffffffffu, ok)) break;
      const int valid = context - (j0 + j) * kTileKV;  // rows behind the context may hold any bits
      const uint32_t from = raw_addr + stage * L::kRawBytes + c * 16;
      const uint32_t to = half_addr + stage * L::kHalfBytes + (c >> 2) * L::kBlockBytes;
#pragma unroll 4
      for (int i = 0; i < kTileKV / kRows; ++i) {
        const int row = i * kRows + row_of;
        uint4 w = ld_shared_16(from + row * D);
        if (row >= valid) w = make_uint4(0, 0, 0, 0);
        const uint32_t by = __shfl_sync(0xffffffffu, mine, row >> 4);
        if (turn) w = make_uint4(w.z, w.w, w.x, w.y);
        const uint32_t at = to + row * 128, x7 = uint32_t(row & 7);
        st_shared_16(at + (((even + turn) ^ x7) << 4), times(halves_of(w.x), by), times(halves_of(w.x >> 16), by),
                     times(halves_of(w.y), by), times(halves_of(w.y >> 16), by));
        st_shared_16(at + (((even + 1 - turn) ^ x7) << 4), times(halves_of(w.z), by), times(halves_of(w.z >> 16), by),
                     times(halves_of(w.w), by), times(halves_of(w.w >> 16), by));
      }
      fence_async_smem();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(v_full + 8 * stage);
        mbar_arrive(raw_empty + 8 * stage);
      }
    }
  } else if (warp >= 8) {
    // ---------------------------------------------------------------- Q, softmax, output
    reg_alloc<kRegsMany>();
    const int t = (warp - 8) >> 2;
    const int quarter = warp & 3;
    const int nt = t == 0 ? n0 : n1;
    const int row_in_tile = quarter * 32 + lane;
    const RowAt where = row_at(a, row_in_tile);
    const int token = token0 + t * p.shares.tokens + where.token, head = g * a.group + where.head;
    const bool live = where.token < p.shares.tokens && token < n && row0 + token < a.rows;
    const float row_scale = row_scales[t * kTileQ + row_in_tile];
    const uint32_t lane_base = tmem_base + (uint32_t(quarter * 32) << 16);
    const uint32_t s_tmem = lane_base, p_tmem = lane_base + 128 + t * 64;
    const uint32_t o_tmem = lane_base + 256 + t * 128;
    const int sees = live ? max(0, min(context, context - n + token + 1)) : 0;  // keys of this row
    // lanes 0..7 hold K's scales; f16: lanes 8..15 V's
    const bool for_v = !BF16 && (lane & 8) != 0;
    ScaleAhead scales = {table, for_v ? a.v.scale : a.k.scale, a.page_shift, pages, a.num_pages, a.kv_heads, g, lane, 1.f, 0, 0.f};
    const float unit_v = 128.0f / top;
    if (nt > 0) scales.start(j0);
    float m_ref = kNone, l = 0.f;
    bool ok = true;

    for (int j = 0; j < nt; ++j) {
      float scale[Groups], rest[Groups];  // rest: V's scale without its power of two
      if (!BF16) {
        const float mine = __uint_as_float((__float_as_uint(scales.next * unit_v) & 0x7fffffu) | 0x3f800000u);
#pragma unroll
        for (int i = 0; i < Groups; ++i) rest[i] = __shfl_sync(0xffffffffu, mine, 8 + i * (8 / Groups));
      }
#pragma unroll
      for (int i = 0; i < Groups; ++i) {
        const float x = __shfl_sync(0xffffffffu, scales.next, i * (8 / Groups)) * row_scale;
        scale[i] = x < 0x1p-126f ? 0x1p-126f : x;  // never 0: a masked score is -inf times this
      }
      if (!__all_sync(0xffffffffu, mbar_wait(s_full + 8 * t, j & 1, abort_flag, status, kSiteScores))) {
        ok = false;
        break;
      }
      tc_fence_after();
      uint32_t s[4][32];
#pragma unroll
      for (int c = 0; c < 4; ++c) tmem_ld_32x32(s_tmem + c * 32, s[c]);
      tmem_ld_wait(s[0]);
      tie(s[1]);
      tie(s[2]);
      tie(s[3]);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(s_read);
      scales.fetch(j0 + j);

      const int visible = sees - (j0 + j) * kTileKV;
      if (visible < kTileKV) {
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          if (i >= visible) s[0][i] = 0xff800000u;
          if (32 + i >= visible) s[1][i] = 0xff800000u;
          if (64 + i >= visible) s[2][i] = 0xff800000u;
          if (96 + i >= visible) s[3][i] = 0xff800000u;
        }
#pragma unroll
        for (int c = 0; c < Groups; ++c) {
          if (c * kGroup >= visible) scale[c] = 1.f;  // whatever the page holds, nothing of it is seen
        }
      }
      float m_new = m_ref;
#pragma unroll
      for (int c = 0; c < Groups; ++c) {
        // sixteen short chains over the tile: one long one waits for itself
        constexpr int kChains = 16 / Groups, kLength = kGroup / kChains;
        float mx[kChains];
#pragma unroll
        for (int i = 0; i < kLength; i += 2) {
#pragma unroll
          for (int x = 0; x < kChains; ++x) {
            const int at = c * kGroup + x * kLength + i;
            const float pair = fmaxf(__uint_as_float(s[at / 32][at % 32]), __uint_as_float(s[at / 32][at % 32 + 1]));
            mx[x] = i == 0 ? pair : fmaxf(mx[x], pair);
          }
        }
#pragma unroll
        for (int x = 1; x < kChains; ++x) mx[0] = fmaxf(mx[0], mx[x]);
        m_new = fmaxf(m_new, mx[0] * scale[c]);
      }
      if (j == 0) {
        m_ref = m_new;
      } else {
        const bool moved = m_new - m_ref > kRescaleThreshold;
        if (__any_sync(0xffffffffu, moved)) {
          // O_t is idle from the end of P_t(j - 1) V(j - 1) until p_full is signalled
          if (!__all_sync(0xffffffffu, mbar_wait(o_full + 8 * t, (j - 1) & 1, abort_flag, status, kSiteOutput))) {
            ok = false;
            break;
          }
          tc_fence_after();
          const float corr = moved ? ex2_approx(m_ref - m_new) : 1.0f;
          l *= corr;
          if (moved) m_ref = m_new;
#pragma unroll
          for (int c = 0; c < D / 32; ++c) {
            uint32_t o[32];
            tmem_ld_32x32(o_tmem + c * 32, o);
            tmem_ld_wait(o);
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * corr);
            tmem_st_32x32(o_tmem + c * 32, o);
          }
        }
      }
      // p = 2^lift exp2(s * scale - m_ref), summed in f32 before the rounding to f16
      constexpr float kOwnLift = BF16 ? kLift : kLift - 1.0f;  // f16: `rest` doubles a weight at most
      const float2 shift2 = make_float2(kOwnLift - m_ref, kOwnLift - m_ref);
      float2 sum[4];
      uint32_t packed[2][32];
#pragma unroll
      for (int c = 0; c < 4; ++c) sum[c] = make_float2(0.f, 0.f);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const float by = scale[(c * 32 + 2 * i) / kGroup];
          const float2 x = __ffma2_rn(make_float2(__uint_as_float(s[c][2 * i]), __uint_as_float(s[c][2 * i + 1])),
                                      make_float2(by, by), shift2);
          const float2 e = make_float2(ex2_approx(x.x), ex2_approx(x.y));
          sum[c] = __fadd2_rn(sum[c], e);
          const float2 w = BF16 ? e : __fmul2_rn(e, make_float2(rest[(c * 32 + 2 * i) / kGroup], rest[(c * 32 + 2 * i) / kGroup]));
          packed[c >> 1][(c & 1) * 16 + i] = pack_f16x2(w.x, w.y);
        }
      }
      const float2 all = __fadd2_rn(__fadd2_rn(sum[0], sum[1]), __fadd2_rn(sum[2], sum[3]));
      l += all.x + all.y;
      // P_t is free when P_t(j - 1) V(j - 1) has read it
      if (j > 0 && !__all_sync(0xffffffffu, mbar_wait(o_full + 8 * t, (j - 1) & 1, abort_flag, status, kSiteOutput))) {
        ok = false;
        break;
      }
      tc_fence_after();
      tmem_st_32x32(p_tmem, packed[0]);       // keys 0..63  -> columns 0..31
      tmem_st_32x32(p_tmem + 32, packed[1]);  // keys 64..127 -> columns 32..63
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(p_full + 8 * t);
    }

    // ---- O_t over l, or a split's share of it
    if (nt > 0 && ok) ok = __all_sync(0xffffffffu, mbar_wait(o_full + 8 * t, (nt - 1) & 1, abort_flag, status, kSiteOutput));
    if (ok) {
      tc_fence_after();
      const float unit = top * (1.0f / 128.0f);
      if (splits > 1) {
        float* share = p.shares.partial + ((long long)blockIdx.x * 2 * kTileQ + t * kTileQ + row_in_tile) * (D + 4);
        if (live) *reinterpret_cast<float2*>(share) = make_float2(nt > 0 ? m_ref : kNone, l);
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {
          uint32_t o[32];
          __syncwarp();
          if (nt > 0) {
            tmem_ld_32x32(o_tmem + c * 32, o);
            tmem_ld_wait(o);
          } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = 0;
          }
          if (live) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              *reinterpret_cast<float4*>(share + 4 + c * 32 + i * 4) =
                  make_float4(__uint_as_float(o[4 * i]) * unit, __uint_as_float(o[4 * i + 1]) * unit,
                              __uint_as_float(o[4 * i + 2]) * unit, __uint_as_float(o[4 * i + 3]) * unit);
            }
          }
        }
      } else {
        // through this tile's Q, which no product reads any more, so that a row's bytes go out side by side
        constexpr int kLanes = D / 8;  // threads per row, 16 bytes each
        const float by = l == 0.f ? 0.f : unit / l;
        const uint32_t stage = q_addr + t * L::kQBytes + quarter * 32 * D * 2;
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {
          uint32_t o[32];
          __syncwarp();
          if (nt > 0) {
            tmem_ld_32x32(o_tmem + c * 32, o);
            tmem_ld_wait(o);
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint32_t w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float x = l == 0.f ? 0.f : __uint_as_float(o[8 * i + 2 * e]) * by;
              const float y = l == 0.f ? 0.f : __uint_as_float(o[8 * i + 2 * e + 1]) * by;
              w[e] = BF16 ? pack_bf16x2(x, y) : pack_f16x2(x, y);
            }
            const uint32_t chunk = uint32_t(c * 4 + i);
            st_shared_16(stage + lane * D * 2 + ((chunk ^ (uint32_t(lane) & 7u)) << 4), w[0], w[1], w[2], w[3]);
          }
        }
        __syncwarp();
        const long long mine = live ? (long long)(row0 + token) * a.o_row + (long long)head * a.o_head : -1;
#pragma unroll 4
        for (int i = 0; i < kLanes; ++i) {  // 32 / kLanes rows at a time
          const int row = i * (32 / kLanes) + lane / kLanes;
          const long long at = __shfl_sync(0xffffffffu, mine, row);
          const uint4 w = ld_shared_16(stage + row * D * 2 + ((uint32_t(lane % kLanes) ^ (uint32_t(row) & 7u)) << 4));
          if (at >= 0) *reinterpret_cast<uint4*>(a.o + at + (lane % kLanes) * 8) = w;
        }
      }
    }
  }

  // ------------------------------------------------------------------ teardown
  if (*abort_flag != 0) {
    for (int i = 0; i < 1000; ++i) __nanosleep(1000);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc<1>(tmem_base, 512);
  }
}

// Where no stream kernel and no join of its pieces follow.
template <int D, bool BF16>
__global__ void __launch_bounds__(256) cache_tile_join_kernel(TileParams p) {
  wait_for_kernel_before();
  join_shares<D, BF16>(p.a, p.shares, p.shares.header->split, blockIdx.x, gridDim.x);
}

template <int D, bool BF16, int Groups>
int launch(const DeviceContext* ctx, const TileParams& p, int64_t page_size, int64_t blocks, cudaStream_t stream) {
  const CacheAttnParams& a = p.a;
  using L = Layout<D, BF16 ? 2 : 3>;
  CUtensorMap map_k, map_v;
  const uint32_t box = uint32_t(page_size < kTileKV ? page_size : kTileKV);
  const Swizzle swizzle = D == 128 ? Swizzle::k128B : Swizzle::k64B;
  if (int rc = encode_pool(&map_k, a.k, D, a.kv_heads, page_size, a.num_pages, box, swizzle)) return rc;
  if (int rc = encode_pool(&map_v, a.v, D, a.kv_heads, page_size, a.num_pages, box, Swizzle::kNone)) return rc;
  auto kernel = cache_tile_kernel<D, BF16, Groups>;
  static OncePerDevice ready;
  if (int rc = ready(ctx->device, [&] {
        KRNB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kSmemBytes));
        // setmaxnreg.inc blocks until the registers that the other warps let go cover it
        cudaFuncAttributes attributes;
        KRNB_CUDA(cudaFuncGetAttributes(&attributes, kernel));
        if (2 * attributes.numRegs < kRegsFew + kRegsMany || attributes.numRegs < kRegsFew) {
          return fail(KRN_B200_ERR_UNSUPPORTED, "cache attention kernel was built with %d registers per thread; the register "
                      "re-partitioning needs %d", attributes.numRegs, (kRegsFew + kRegsMany) / 2);
        }
        return KRN_B200_OK;
      })) {
    return rc;
  }
  return launch_dependent(kernel, dim3(unsigned(blocks)), kThreads, L::kSmemBytes, stream, map_k, map_v,
                          p, ctx->status_dev);
}

// A key tile has two scales at most where pages are 64 tokens or more, up to eight where they are smaller. Eight would do for
// both: 178 us against 174 for four prompts of 2048 tokens, 8 kv heads of 128, group 4, within 2 % elsewhere.
template <int D, bool BF16>
int launch_pages(const DeviceContext* ctx, const TileParams& p, int64_t page_size, int64_t blocks, cudaStream_t stream) {
  return page_size >= 64 ? launch<D, BF16, 2>(ctx, p, page_size, blocks, stream) : launch<D, BF16, 8>(ctx, p, page_size, blocks, stream);
}

// Shares of a block's keys, at most: none is shorter than kShortest key tiles.
int64_t most_shares(int64_t max_context) { return (max_context + kShortest * kTileKV - 1) / (kShortest * kTileKV); }

}  // namespace

// Every tiled request has more than `few` rows, so there are not many of them.
int64_t tile_blocks(int64_t batch, int64_t rows, int64_t group, int64_t few) {
  const int64_t least = few / group + 1, tokens = 2 * (kTileQ / group);
  const int64_t requests = rows / least < batch ? rows / least : batch;
  return requests > 0 ? rows / tokens + requests : 0;
}

bool tiles_split(int64_t max_context) { return most_shares(max_context) > 1; }

namespace {

// As many as run at once, at most.
int64_t share_room(int64_t blocks, int64_t max_context) {
  const int64_t most = most_shares(max_context);
  return most <= 1 ? 0 : blocks >= kSMs || most >= kSMs || blocks * most >= kSMs ? kSMs : blocks * most;
}

}  // namespace

TileShares tile_shares(const CacheAttnParams& a, void* workspace) {
  uint8_t* at = static_cast<uint8_t*>(workspace);
  return {tiles_split(a.max_context) ? reinterpret_cast<SplitHeader*>(at) : nullptr, reinterpret_cast<float*>(at + kHeaderBytes),
          kTileQ / a.group};
}

int64_t tile_workspace(int64_t batch, int64_t rows, int64_t q_heads, int64_t kv_heads, int64_t d, int64_t few, int64_t max_context) {
  if (!tiles_split(max_context)) return 0;
  const int64_t blocks = tile_blocks(batch, rows, q_heads / kv_heads, few) * kv_heads;
  return kHeaderBytes + share_room(blocks, max_context) * 2 * kTileQ * (d + 4) * 4;
}

int launch_tiles(const DeviceContext* ctx, const CacheAttnParams& a, const TileShares& shares, bool bf16, int64_t d, int64_t page_size,
                 cudaStream_t stream) {
  const int64_t bound = tile_blocks(a.batch, a.rows, a.group, a.few) * a.kv_heads, room = share_room(bound, a.max_context);
  const TileParams p = {a, shares, int(room)};
  const int64_t blocks = bound < room ? room : bound;
  if (d == 128) return bf16 ? launch_pages<128, true>(ctx, p, page_size, blocks, stream) : launch_pages<128, false>(ctx, p, page_size, blocks, stream);
  return bf16 ? launch_pages<64, true>(ctx, p, page_size, blocks, stream) : launch_pages<64, false>(ctx, p, page_size, blocks, stream);
}

int launch_tile_join(const CacheAttnParams& a, const TileShares& shares, bool bf16, int64_t d, cudaStream_t stream) {
  if (shares.header == nullptr) return KRN_B200_OK;
  const TileParams p = {a, shares, 0};
  const dim3 grid(3 * kSMs);
  if (d == 128) return launch_dependent(bf16 ? cache_tile_join_kernel<128, true> : cache_tile_join_kernel<128, false>, grid, 256, 0, stream, p);
  return launch_dependent(bf16 ? cache_tile_join_kernel<64, true> : cache_tile_join_kernel<64, false>, grid, 256, 0, stream, p);
}

}  // namespace krnb
