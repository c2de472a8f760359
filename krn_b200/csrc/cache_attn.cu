// Attention over the paged 8-bit cache with one scale per (page, kv head): rows of q packed by request, row i of a request
// with n rows and a context of c tokens stands at position c - n + i and sees the keys up to it.
//
// Two paths: requests with few rows (new tokens x q heads of a kv head) are streamed, a warp per stretch of keys, here;
// prompts and chunks of prompts go to tensor-core tiles (cache_attn_tile.cu).
#include "cache_attn.cuh"

#include <cmath>

namespace krnb {
namespace {

// ---- few rows: a stream of keys per warp ---------------------------------------------------------------------------------

constexpr int kTile = 32;          // tokens a warp takes at a time
constexpr int kMaxWarps = 12;      // of a block
constexpr int kMaxBlocks = 160;    // bounds the workspace; a B200 has 148 SMs
constexpr int kMaxBatch = 8192;    // tile counts of the batch sit in shared memory
constexpr int kMaxGroup = kTileQ;  // q heads of a kv head: a query tile holds a token's rows whole
constexpr float kLeastScale = 0x1p-110f;  // value scales below it are held against it

// Partial results of the pieces of split segments, d + 4 floats (m, l, two unused, the unnormalised output) for each row.
struct StreamParams {
  CacheAttnParams a;
  int4* pieces;      // [batch] first and last stretch of each request, whether its first piece is a warp's second; for the join
  float* partial;
  int row_blocks;    // warps that share a stretch and kv head, each with its own NT * 8 rows of every request
  int beside;        // launched beside the tile kernel, which waited for what came before
  TileShares tiles;  // what the tile kernel may have split, for the join
};

__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t transposed(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

__device__ __forceinline__ uint2 ld_shared_8(uint32_t addr) {
  uint2 v;
  asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr));
  return v;
}

__device__ __forceinline__ float ld_shared_f32(uint32_t addr) {
  float v;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(addr));
  return v;
}

// 4 bytes global -> shared that complete on `bar` with one arrival; zeros when `take` is false.
__device__ __forceinline__ void copy_scale(uint32_t dst, const float* src, bool take, uint32_t bar) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(take ? 4 : 0) : "memory");
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}

// Tiles of one (request, kv head): none for a request without rows or with more than this path takes, at least one
// otherwise, so that rows that see no key get their zeros.
__device__ __forceinline__ int tiles_of(const StreamParams& p, int b) {
  const int n = p.a.row_start[b + 1] - p.a.row_start[b];
  if (!rows_ok(p.a, b, n) || (long long)n * p.a.group > p.a.few) return 0;
  const int context = max(0, min(p.a.context_len[b], p.a.max_context));
  return max(1, (context + kTile - 1) / kTile);
}

// The line of the batch's tiles, dealt evenly and in order to `parts` stretches: the first tile of stretch `part`.
__device__ __forceinline__ int first_tile(int part, int parts, int total) { return int((long long)part * total / parts); }

// The stretch that holds tile `at`.
__device__ __forceinline__ int stretch_of(int at, int parts, int total) { return int(((long long)(at + 1) * parts - 1) / total); }

// Stretches: one warp for each, kv head and block of rows, one tile at least.
__device__ __forceinline__ int stretches(int total, int warps, int sharers) { return max(1, min(warps / sharers, total)); }

// Where a warp stands in the line.
struct Spot {
  int b, tile, tiles;  // request, tile of it, tiles it has
};

__device__ __forceinline__ Spot spot_at(const int32_t* tiles, int batch, int at) {
  int low = 0, high = batch;
  while (high - low > 1) {
    const int mid = (low + high) >> 1;
    if (tiles[mid] <= at) low = mid; else high = mid;
  }
  return {low, at - tiles[low], tiles[low + 1] - tiles[low]};
}

__device__ __forceinline__ void step(Spot& s, const int32_t* tiles, int batch) {
  if (++s.tile < s.tiles) return;
  s.tile = 0;
  do {
    ++s.b;
  } while (s.b < batch && tiles[s.b + 1] == tiles[s.b]);
  if (s.b < batch) s.tiles = tiles[s.b + 1] - tiles[s.b];
}

// Warps of a block and their rings. Rows of 128 columns: 8 warps with 3 tiles of 8 KB each, 105 us on the 64-sequence mix of
// 1024 to 8192 tokens (10 warps with 2: 105.4, 12 with 2: 109, 9 with 2: 111). Rows of 64: tiles of 4 KB leave room for 12
// warps, 30.5 us against 34.5 with 8 (64 sequences of 2048 to 4096 tokens, 4 kv heads; 16 with 3: 29.8, but 19.5 against
// 17.6 us for one sequence of 60000), with 16 rows a warp 38.9 against 40.6 (11.1 against 9.8 for one request of 4096).
template <int D>
struct StreamLayout {
  static constexpr int kWarps = D == 64 ? 12 : 8;
  static constexpr int kStages = 3;                       // tiles a warp has in flight or in work
  static constexpr int kSide = kTile * D;                 // one of K and V, bytes
  static constexpr int kStage = 2 * kSide;
  static constexpr int kRing = kWarps * kStages * kStage;
  static constexpr int kScales = kWarps * kStages * 16;   // ks, ks, vs, vs of a tile's two 16-token groups
  static constexpr int kBars = kWarps * kStages * 8;
  static int bytes(int batch) { return 1024 + kRing + kScales + kBars + 16 + 4 * (batch + 1 + kWarps); }
};

// Few query rows against many keys: bound by HBM. The contexts of the batch, cut into tiles of 32 tokens, form one line;
// it is dealt in equal stretches, and a warp takes one stretch for one kv head and works alone, with a ring of TMA tiles of
// its own, no block barrier after the start. Neighbouring warps take the kv heads of one stretch, so that a token's heads,
// which lie side by side in a page, are fetched at about the same time. NT * 8 rows (a request's new tokens x the q heads
// of the kv head) share a tile:
//   S^T[token, row] = K Q^T   (M = 16 tokens, N = 8 rows, K = 16 columns of d; K's codes become f16 exactly, q is f16 with a
//                              power-of-two factor per row)
//   running maximum and sum per row in f32; P^T = exp2(S - m) times the page's value scale, f16
//   O^T[d, row] += V^T P^T    (M = 16 columns of d, K = 16 tokens; P^T turns from accumulator to operand by movmatrix)
// Value scales enter P relative to the largest seen so far, R, and P carries 2^15: a weight keeps f16's eleven bits down to
// 2^-29 of the largest one. A warp whose stretch covers a whole segment writes its output; pieces of split segments go to
// the workspace and cache_join_kernel joins them. 64 sequences of 1024 to 8192 tokens, 8 kv heads of 128, one new token each:
// 605 MB in 100 us = 6.06 TB/s.
template <int D, bool BF16, int NT>
__global__ void __launch_bounds__(StreamLayout<D>::kWarps * 32, 1)
cache_stream_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, StreamParams p,
                    DeviceStatus* status) {
  using L = StreamLayout<D>;
  constexpr int kWarps = L::kWarps, kStages = L::kStages;
  constexpr int kSteps = D / 16;       // MMA steps over d
  constexpr int kWords = D / 16;       // 32-bit words of a K row that a thread holds
  constexpr int kSlotRows = NT * 8;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  uint8_t* smem = smem_raw + (base - raw);
  const CacheAttnParams& a = p.a;
  const int warp = threadIdx.x >> 5;
  const int lane = int(lane_id());
  const int r = lane >> 2, q4 = lane & 3;
  const uint32_t ring = base + warp * kStages * L::kStage;
  const uint32_t scales = base + L::kRing + warp * kStages * 16;
  const uint32_t bars = base + L::kRing + L::kScales + warp * kStages * 8;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::kRing + L::kScales + L::kBars);
  int32_t* tiles = reinterpret_cast<int32_t*>(smem + L::kRing + L::kScales + L::kBars + 16);
  int32_t* sums = tiles + a.batch + 1;

  if (lane == 0) {
    for (int s = 0; s < kStages; ++s) mbar_init(bars + 8 * s, 5);  // the TMA bytes' arrival and four scales
    fence_mbar_init();
  }
  if (threadIdx.x == 0) {
    *abort_flag = 0;
    prefetch_tensormap(&map_k);
    prefetch_tensormap(&map_v);
  }
  if (!p.beside) wait_for_kernel_before();
  launch_dependents();
  // ---- every block counts the batch's tiles for itself
  int carry = 0;
  for (int first = 0; first < a.batch; first += kWarps * 32) {
    const int b = first + int(threadIdx.x);
    int v = b < a.batch ? tiles_of(p, b) : 0;
    const int own = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int below = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v += below;
    }
    if (lane == 31) sums[warp] = v;
    __syncthreads();
    int before = carry, total = carry;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const int s = sums[w];
      if (w < warp) before += s;
      total += s;
    }
    if (b < a.batch) tiles[b] = before + v - own;
    carry = total;
    __syncthreads();
  }
  if (threadIdx.x == 0) tiles[a.batch] = carry;
  __syncthreads();
  const int total = carry, grid_warps = int(gridDim.x) * kWarps;
  const int sharers = a.kv_heads * p.row_blocks, parts = stretches(total, grid_warps, sharers);
  if (blockIdx.x == 0) {
    for (int b = threadIdx.x; b < a.batch; b += kWarps * 32) {
      const int first = tiles[b], last = tiles[b + 1] - 1;
      const int p0 = last >= first ? stretch_of(first, parts, total) : 0, p1 = last >= first ? stretch_of(last, parts, total) : 0;
      p.pieces[b] = make_int4(p0, p1, first > first_tile(p0, parts, total) ? 1 : 0, 0);
      report_rows(a, b, status);
    }
  }
  // Beside the tile kernel this grid must not end before it, which one block sees to: the others leave their SMs to the next.
  const auto leave = [&] {
    if (blockIdx.x + 1 == gridDim.x) wait_for_kernel_before();
  };
  if (total == 0) {
    leave();
    return;
  }

  const int page_mask = (1 << a.page_shift) - 1;
  const int box = min(kTile, page_mask + 1);  // tokens of one copy
  int bad_page = 0;

  bool ok = true;
  int done = 0;  // tiles of earlier units: the ring goes on
  for (int unit = int(blockIdx.x) * kWarps + warp; unit < parts * sharers && ok; unit += grid_warps) {
    const int part = unit / sharers, g = (unit - part * sharers) / p.row_blocks;
    const int row_base = (unit % p.row_blocks) * kSlotRows;  // first row of each request that is this warp's
    const int begin = first_tile(part, parts, total), count = first_tile(part + 1, parts, total) - begin;

    // ---- the stretch's tiles in order: page ids come 32 at a time, one per lane
    Spot ahead = spot_at(tiles, a.batch, begin);
    int ids = 0, ids_b = -1, ids_first = 0, ahead_pages = 0;
    auto issue = [&](int number) {  // tile `number` of the stretch into its stage
      const int stage = (done + number) % kStages;
      const uint32_t bar = bars + 8 * stage, dst = ring + stage * L::kStage;
      const int token = ahead.tile * kTile;
      const int first_page = token >> a.page_shift;
      if (ahead.b != ids_b || first_page < ids_first || first_page + 1 >= ids_first + 32) {
        ids_b = ahead.b;
        ids_first = first_page;
        const int context = max(0, min(a.context_len[ahead.b], a.max_context));
        const bool mine = (a.row_start[ahead.b + 1] - a.row_start[ahead.b]) * a.group > row_base;  // else nothing is fetched
        ahead_pages = mine ? (context + page_mask) >> a.page_shift : 0;
        ids = first_page + lane < ahead_pages ? a.page_table[ahead.b * a.table_pitch + first_page + lane] : 0;
      }
      // sub-tile 0 / 1: tokens 0..15 / 16..31 for 16-token pages; else one copy of 32 tokens
      const int sub = box == kTile ? 0 : (lane & 1);
      int page = __shfl_sync(0xffffffffu, ids, first_page + sub - ids_first);
      const bool there = first_page + sub < ahead_pages;
      const bool good = there && uint32_t(page) < uint32_t(a.num_pages);
      if (there && !good) {
        bad_page = page | int(0x80000000);
        page = a.num_pages;  // one past the pool: TMA fills zeros
      }
      const int copies = kTile / box;
      const int there_parts = min(copies, ahead_pages - first_page);
      if (lane == 0) mbar_arrive_expect_tx(bar, uint32_t(max(0, there_parts)) * 2u * uint32_t(box) * D);
      __syncwarp();
      if (lane < 4) {
        const bool keys = lane < 2;
        if (there && (lane & 1) < copies) {
          tma_load_4d(dst + (keys ? 0 : L::kSide) + sub * box * D, keys ? &map_k : &map_v, 0, g, token & page_mask, page, bar);
        }
        const float* source = keys ? a.k.scale : a.v.scale;
        copy_scale(scales + stage * 16 + lane * 4, source + (good ? (long long)page * a.kv_heads + g : 0), good, bar);
      }
      step(ahead, tiles, a.batch);
    };
    for (int i = 0; i < min(count, kStages); ++i) issue(i);

    Spot at = spot_at(tiles, a.batch, begin);
    float acc[kSteps][NT][4], m[NT][2];
    float2 l[NT], row_scale[NT];
    uint32_t query[NT][kSteps][2];
    int limit[NT][2], context = 0, rows = 0, row0 = 0, nearest = 0;
    float top = kLeastScale, from_top = 0.f;
    int piece = 0;  // first tile of the current piece within its request

    for (int i = 0; i < count; ++i) {
      if (i == 0 || at.tile == 0) {
        // ---- a new piece: its rows of q as f16 with a power-of-two factor, and how far each row sees
        piece = at.tile;
        row0 = a.row_start[at.b];
        const int n = a.row_start[at.b + 1] - row0;
        rows = n * a.group;
        context = max(0, min(a.context_len[at.b], a.max_context));
        nearest = context - n + 1;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          const int mine = row_base + t * 8 + r;
          uint4 w[D / 32];
          float size = 0.f;
          const RowAt row = row_at(a, mine);
          const bool live = mine < rows && row0 + row.token < a.rows;
          const uint16_t* src = a.q + (long long)(row0 + row.token) * a.q_row + (long long)(g * a.group + row.head) * a.q_head + q4 * (D / 4);
#pragma unroll
          for (int c = 0; c < D / 32; ++c) {
            w[c] = live ? *reinterpret_cast<const uint4*>(src + c * 8) : make_uint4(0, 0, 0, 0);
            const uint32_t words[4] = {w[c].x, w[c].y, w[c].z, w[c].w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float2 v = unpack<BF16>(words[e]);
              size = fmaxf(size, fmaxf(fabsf(v.x), fabsf(v.y)));
            }
          }
          size = fmaxf(size, __shfl_xor_sync(0xffffffffu, size, 1));
          size = fmaxf(size, __shfl_xor_sync(0xffffffffu, size, 2));
          // the row's largest magnitude comes to lie in [2^14, 2^15)
          const int up = max(-113, min(126, 14 - (int(__float_as_uint(size) >> 23) - 127)));
          const float by = copysignf(__uint_as_float(uint32_t(up + 127) << 23), a.scale_log2);
#pragma unroll
          for (int c = 0; c < D / 32; ++c) {
            const uint32_t words[4] = {w[c].x, w[c].y, w[c].z, w[c].w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float2 v = unpack<BF16>(words[e]);
              query[t][c * 2 + e / 2][e & 1] = pack_f16x2(v.x * by, v.y * by);
            }
          }
          const float back = __uint_as_float(uint32_t(127 - up) << 23) * fabsf(a.scale_log2);
          // of the rows whose scores this thread holds
          row_scale[t] = make_float2(__shfl_sync(0xffffffffu, back, q4 * 8), __shfl_sync(0xffffffffu, back, q4 * 8 + 4));
          l[t] = make_float2(0.f, 0.f);
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int at_row = row_base + t * 8 + 2 * q4 + e;
            limit[t][e] = at_row < rows ? nearest + row_at(a, at_row).token : context;
            m[t][e] = kNone;
          }
        }
#pragma unroll
        for (int c = 0; c < kSteps; ++c)
#pragma unroll
          for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[c][t][e] = 0.f;
        top = kLeastScale;
        from_top = 32768.0f / kLeastScale;
      }

      const int stage = (done + i) % kStages;
      const uint32_t keys = ring + stage * L::kStage, values = keys + L::kSide;
      if (!__all_sync(0xffffffffu, mbar_wait(bars + 8 * stage, ((done + i) / kStages) & 1, abort_flag, status, kSiteTile))) {
        ok = false;
        break;
      }
      if (rows <= row_base) {  // a request with fewer rows than others
        if (i + kStages < count) issue(i + kStages);
        step(at, tiles, a.batch);
        continue;
      }
      const int token0 = at.tile * kTile;

      // ---- scores: a thread's words of K are 32 (d = 64: 16) consecutive bytes of rows r and r + 8; q holds the same columns
      float s[2][NT][4];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        uint32_t ka[kWords], kb[kWords];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const int row = u * 16 + half * 8 + r;
          uint32_t(&k)[kWords] = half == 0 ? ka : kb;
          if constexpr (D == 128) {
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              const uint4 v = ld_shared_16(keys + row * 128 + (((q4 * 2 + c) ^ (row & 7)) << 4));
              k[c * 4] = v.x, k[c * 4 + 1] = v.y, k[c * 4 + 2] = v.z, k[c * 4 + 3] = v.w;
            }
          } else {
            const uint4 v = ld_shared_16(keys + row * 64 + ((q4 ^ ((row >> 1) & 3)) << 4));
            k[0] = v.x, k[1] = v.y, k[2] = v.z, k[3] = v.w;
          }
        }
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[u][t][e] = 0.f;
#pragma unroll
        for (int c = 0; c < kSteps; ++c) {
          const uint32_t a0 = halves_of(ka[c]), a2 = halves_of(ka[c] >> 16), a1 = halves_of(kb[c]), a3 = halves_of(kb[c] >> 16);
#pragma unroll
          for (int t = 0; t < NT; ++t) mma_f16(s[u][t], a0, a1, a2, a3, query[t][c][0], query[t][c][1]);
        }
      }

      // ---- softmax: the thread's tokens are u * 16 + r and + 8, its rows 2 * q4 and + 1 of each eight. Arithmetic goes two
      // rows at a time; the maximum is taken of the raw scores, whose factors are positive
      if (token0 + kTile > nearest) {  // some row does not see all of the tile
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              if (token0 + u * 16 + r + (e >> 1) * 8 >= limit[t][e & 1]) s[u][t][e] = -INFINITY;
            }
      }
      const float ks0 = ld_shared_f32(scales + stage * 16), vs0 = ld_shared_f32(scales + stage * 16 + 8);
      const float ks1 = box == kTile ? ks0 : ld_shared_f32(scales + stage * 16 + 4);
      const float vs1 = box == kTile ? vs0 : ld_shared_f32(scales + stage * 16 + 12);
      auto factor = [&](int u, int t) {  // never 0: a masked score is -inf times it
        const float ks = u == 0 ? ks0 : ks1;
        const float2 f = __fmul2_rn(row_scale[t], make_float2(ks, ks));
        return make_float2(f.x < 0x1p-126f ? 0x1p-126f : f.x, f.y < 0x1p-126f ? 0x1p-126f : f.y);
      };
      const float new_top = fmaxf(top, fmaxf(fabsf(vs0), fabsf(vs1)));
      bool moved = new_top != top;
      float m_new[NT][2];
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const float2 f0 = factor(0, t), f1 = factor(1, t);
        float high[2] = {fmaxf(fmaxf(s[0][t][0], s[0][t][2]) * f0.x, fmaxf(s[1][t][0], s[1][t][2]) * f1.x),
                         fmaxf(fmaxf(s[0][t][1], s[0][t][3]) * f0.y, fmaxf(s[1][t][1], s[1][t][3]) * f1.y)};
#pragma unroll
        for (int e = 0; e < 2; ++e) {
#pragma unroll
          for (int o = 4; o < 32; o <<= 1) high[e] = fmaxf(high[e], __shfl_xor_sync(0xffffffffu, high[e], o));
          m_new[t][e] = fmaxf(m[t][e], high[e]);
          moved |= m_new[t][e] != m[t][e];
        }
      }
      if (__any_sync(0xffffffffu, moved)) {
        const float shrink = top / new_top;
        top = new_top;
        from_top = 32768.0f / new_top;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          float2 corr;
          corr.x = ex2_approx(m[t][0] - m_new[t][0]);
          corr.y = ex2_approx(m[t][1] - m_new[t][1]);
          m[t][0] = m_new[t][0];
          m[t][1] = m_new[t][1];
          l[t] = __fmul2_rn(l[t], corr);
          corr = __fmul2_rn(corr, make_float2(shrink, shrink));
#pragma unroll
          for (int c = 0; c < kSteps; ++c)
#pragma unroll
            for (int e = 0; e < 4; e += 2) {
              const float2 x = __fmul2_rn(make_float2(acc[c][t][e], acc[c][t][e + 1]), corr);
              acc[c][t][e] = x.x;
              acc[c][t][e + 1] = x.y;
            }
        }
      }
      uint32_t weight[2][NT][2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const float vs = (u == 0 ? vs0 : vs1) * from_top;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          const float2 f = factor(u, t), shift = make_float2(-m[t][0], -m[t][1]);
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float2 x = __ffma2_rn(make_float2(s[u][t][2 * e], s[u][t][2 * e + 1]), f, shift);
            const float2 w = make_float2(ex2_approx(x.x), ex2_approx(x.y));
            l[t] = __fadd2_rn(l[t], w);
            const float2 y = __fmul2_rn(w, make_float2(vs, vs));
            weight[u][t][e] = transposed(pack_f16x2(y.x, y.y));
          }
        }
      }

      // ---- output: a thread's columns of V are 16 (d = 64: 8) consecutive ones of tokens 2 * q4, + 1, + 8, + 9
      const bool tail = token0 + kTile > context;  // what lies behind the context may be any bits
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        uint32_t v[4][D / 32];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int row = u * 16 + 2 * q4 + (e & 1) + (e >> 1) * 8;
          if constexpr (D == 128) {
            const uint4 x = ld_shared_16(values + row * 128 + ((r ^ (row & 7)) << 4));
            v[e][0] = x.x, v[e][1] = x.y, v[e][2] = x.z, v[e][3] = x.w;
          } else {
            const uint2 x = ld_shared_8(values + row * 64 + (((r >> 1) ^ ((row >> 1) & 3)) << 4) + (r & 1) * 8);
            v[e][0] = x.x, v[e][1] = x.y;
          }
          if (tail && token0 + row >= context) {
#pragma unroll
            for (int c = 0; c < D / 32; ++c) v[e][c] = 0;
          }
        }
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {
          const uint32_t x0 = __byte_perm(v[0][c], v[1][c], 0x5140), x1 = __byte_perm(v[0][c], v[1][c], 0x7362);
          const uint32_t y0 = __byte_perm(v[2][c], v[3][c], 0x5140), y1 = __byte_perm(v[2][c], v[3][c], 0x7362);
          const uint32_t a0 = halves_of(x0), a1 = halves_of(x0 >> 16), a2 = halves_of(y0), a3 = halves_of(y0 >> 16);
          const uint32_t b0 = halves_of(x1), b1 = halves_of(x1 >> 16), b2 = halves_of(y1), b3 = halves_of(y1 >> 16);
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            mma_f16(acc[2 * c][t], a0, a1, a2, a3, weight[u][t][0], weight[u][t][1]);
            mma_f16(acc[2 * c + 1][t], b0, b1, b2, b3, weight[u][t][0], weight[u][t][1]);
          }
        }
      }
      __syncwarp();
      if (i + kStages < count) issue(i + kStages);

      // ---- the end of a piece
      if (at.tile + 1 == at.tiles || i + 1 == count) {
        const bool whole = piece == 0 && at.tile + 1 == at.tiles;
        const int slot = 2 * unit + (i - (at.tile - piece) == 0 ? 0 : 1);
        const float value = top * (1.0f / 32768.0f);
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float sum = e == 0 ? l[t].x : l[t].y;
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            const int in_slot = t * 8 + 2 * q4 + e, row = row_base + in_slot;
            const RowAt at_row = row_at(a, row);
            if (row >= rows || row0 + at_row.token >= a.rows) continue;
            if (whole) {
              const float by = sum == 0.f ? 0.f : value / sum;
              uint16_t* out = a.o + (long long)(row0 + at_row.token) * a.o_row + (long long)(g * a.group + at_row.head) * a.o_head + r * (D / 8);
#pragma unroll
              for (int c = 0; c < D / 64; ++c) {
                uint32_t w[4];
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                  const float y0 = acc[c * 4 + x][t][e] * by, y1 = acc[c * 4 + x][t][2 + e] * by;
                  w[x] = BF16 ? pack_bf16x2(y0, y1) : pack_f16x2(y0, y1);
                }
                *reinterpret_cast<uint4*>(out + c * 8) = make_uint4(w[0], w[1], w[2], w[3]);
              }
            } else {
              float* out = p.partial + ((long long)slot * kSlotRows + in_slot) * (D + 4);
              if (r == 0) *reinterpret_cast<float2*>(out) = make_float2(m[t][e], sum);
#pragma unroll
              for (int c = 0; c < D / 32; ++c) {
                *reinterpret_cast<float4*>(out + 4 + r * (D / 8) + c * 4) =
                    make_float4(acc[c * 2][t][e] * value, acc[c * 2][t][2 + e] * value, acc[c * 2 + 1][t][e] * value,
                                acc[c * 2 + 1][t][2 + e] * value);
              }
            }
          }
      }
      step(at, tiles, a.batch);
    }
    done += count;
  }
  if (bad_page != 0) report_failure(status, kErrDeviceIndex, kSitePage, uint32_t(bad_page) & 0x7fffffffu);
  if (!ok) {  // let this warp's own copies land before the block's memory goes
    for (int i = 0; i < 1000; ++i) __nanosleep(1000);
  }
  leave();
}

// Joins the pieces of split segments,
//   o = sum 2^(m_i - M) acc_i / sum 2^(m_i - M) l_i.
// A block takes `slots` rows of one (request, kv head); kGroups / slots groups of threads, four columns a thread, share a
// row's pieces, eight of them in flight at a time, and meet in shared memory. Bound by latency: one load of what the stream
// kernel says about the request, one round of pieces: 4 us after the stream kernel, as whose programmatic dependent it is
// launched: its blocks are resident when that ends.
template <int D, bool BF16, int Threads>
__device__ __forceinline__ void join_pieces(const StreamParams& p, int slot_rows, int slots) {
  constexpr int kLanes = D / 4, kGroups = Threads / kLanes;
  __shared__ float4 shared_acc[kGroups][kLanes];
  __shared__ float2 shared_ml[kGroups];
  const CacheAttnParams& a = p.a;
  const int b = blockIdx.x / a.kv_heads, g = blockIdx.x % a.kv_heads;
  const int group = threadIdx.x / kLanes, lane = threadIdx.x % kLanes;
  const int row = blockIdx.y * slots + group % slots, share = group / slots, shares = kGroups / slots;
  const int row0 = a.row_start[b], rows = (a.row_start[b + 1] - row0) * a.group;
  const RowAt where = row_at(a, row);
  const int at = row0 + where.token;
  const int4 piece = p.pieces[b];
  if (piece.x == piece.y) return;  // no split: the rows are written, or belong to the other path
  const bool live = row < rows && at < a.rows;
  float m = kNone, l = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  if (live) {
    const long long pitch = (long long)slot_rows * (D + 4);  // of a slot; every warp of a stretch has two
    const int sharers = a.kv_heads * p.row_blocks, block = row / slot_rows;
    const float* from = p.partial + 2 * (g * p.row_blocks + block) * pitch + (long long)(row - block * slot_rows) * (D + 4);
#pragma unroll 1
    for (int first = piece.x + share; first <= piece.y; first += 8 * shares) {
      float2 ml[8];
      float4 x[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int part = first + k * shares;
        const bool there = part <= piece.y;
        const float* at_piece = from + (2ll * (there ? part : piece.x) * sharers + (part == piece.x ? piece.z : 0)) * pitch;
        ml[k] = there ? *reinterpret_cast<const float2*>(at_piece) : make_float2(kNone, 0.f);
        x[k] = there ? *reinterpret_cast<const float4*>(at_piece + 4 + lane * 4) : make_float4(0.f, 0.f, 0.f, 0.f);
      }
      float high = m;
#pragma unroll
      for (int k = 0; k < 8; ++k) high = fmaxf(high, ml[k].x);
      const float old = ex2_approx(m - high);
      m = high;
      l *= old;
      acc.x *= old, acc.y *= old, acc.z *= old, acc.w *= old;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float by = ex2_approx(ml[k].x - high);
        l += by * ml[k].y;
        acc.x += by * x[k].x, acc.y += by * x[k].y, acc.z += by * x[k].z, acc.w += by * x[k].w;
      }
    }
  }
  if (shares > 1) {
    shared_acc[group][lane] = acc;
    if (lane == 0) shared_ml[group] = make_float2(m, l);
    __syncthreads();
    if (share > 0) return;
    float high = m;
    for (int k = 1; k < shares; ++k) high = fmaxf(high, shared_ml[group + k * slots].x);
    const float own = ex2_approx(m - high);
    l *= own;
    acc.x *= own, acc.y *= own, acc.z *= own, acc.w *= own;
    for (int k = 1; k < shares; ++k) {
      const float2 ml = shared_ml[group + k * slots];
      const float4 x = shared_acc[group + k * slots][lane];
      const float by = ex2_approx(ml.x - high);
      l += by * ml.y;
      acc.x += by * x.x, acc.y += by * x.y, acc.z += by * x.z, acc.w += by * x.w;
    }
  }
  if (!live) return;
  const float by = l == 0.f ? 0.f : 1.0f / l;
  uint2 w;
  w.x = BF16 ? pack_bf16x2(acc.x * by, acc.y * by) : pack_f16x2(acc.x * by, acc.y * by);
  w.y = BF16 ? pack_bf16x2(acc.z * by, acc.w * by) : pack_f16x2(acc.z * by, acc.w * by);
  *reinterpret_cast<uint2*>(a.o + (long long)at * a.o_row + (long long)(g * a.group + where.head) * a.o_head + lane * 4) = w;
}

template <int D, bool BF16, int Threads>
__global__ void __launch_bounds__(Threads) cache_join_kernel(StreamParams p, int slot_rows, int slots) {
  wait_for_kernel_before();
  const int2 split = p.tiles.header != nullptr ? p.tiles.header->split : make_int2(1, 0);
  if (int(blockIdx.y) * slots < p.a.few) join_pieces<D, BF16, Threads>(p, slot_rows, slots);
  join_shares<D, BF16>(p.a, p.tiles, split, blockIdx.y * gridDim.x + blockIdx.x, gridDim.x * gridDim.y);
}

template <int D, bool BF16, int NT>
int launch_stream(const DeviceContext* ctx, const StreamParams& p, int64_t page_size, cudaStream_t stream) {
  const CacheAttnParams& a = p.a;
  CUtensorMap map_k, map_v;
  const uint32_t box = uint32_t(page_size < kTile ? page_size : kTile);
  const Swizzle swizzle = D == 128 ? Swizzle::k128B : Swizzle::k64B;
  if (int rc = encode_pool(&map_k, a.k, D, a.kv_heads, page_size, a.num_pages, box, swizzle)) return rc;
  if (int rc = encode_pool(&map_v, a.v, D, a.kv_heads, page_size, a.num_pages, box, swizzle)) return rc;
  auto kernel = cache_stream_kernel<D, BF16, NT>;
  static OncePerDevice ready;
  if (int rc = ready(ctx->device, [&] {
        KRNB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, StreamLayout<D>::bytes(kMaxBatch)));
        return KRN_B200_OK;
      })) {
    return rc;
  }
  constexpr int kWarps = StreamLayout<D>::kWarps;
  // no more blocks than the contexts could give warps work
  const int64_t sharers = int64_t(a.kv_heads) * p.row_blocks;
  const int64_t wanted = (int64_t(a.batch) * sharers * ((a.max_context + kTile - 1) / kTile) + kWarps - 1) / kWarps;
  const int most = ctx->sm_count < kMaxBlocks ? ctx->sm_count : kMaxBlocks;
  const int blocks = int(wanted < most ? wanted : most);
  if (int rc = launch_dependent(kernel, dim3(unsigned(blocks)), kWarps * 32, StreamLayout<D>::bytes(a.batch), stream, map_k, map_v, p,
                                ctx->status_dev)) {
    return rc;
  }
  // Rows of a block: as many as leave each group of threads no more than eight pieces, as the batch is split on average. One
  // sequence of 60000 tokens: 25.1 us (stream and join) with one row a block, 48.5 with eight; 64 sequences of up to 4 rows
  // over 1024 to 8192 tokens: 83 us with one, 69.6 with eight.
  constexpr int kGroups = 256 * 4 / D;
  const int64_t pieces = int64_t(blocks) * kWarps / sharers / a.batch + 2;
  int slots = kGroups;
  while (slots > 1 && (slots / 2 >= a.few || pieces > 8 * (kGroups / slots))) slots /= 2;
  unsigned depth = unsigned((a.few + slots - 1) / slots);
  const unsigned width = unsigned(a.batch) * unsigned(a.kv_heads);
  if (p.tiles.header != nullptr && width * depth < 3 * kSMs) depth = (3 * kSMs + width - 1) / width;  // blocks for what was split
  const dim3 grid(width, depth);
  // Many pieces, which takes few sequences, are worth twice the groups: one sequence of 60000 tokens 25.2 -> 20.5 us, eight of
  // 4096 13.5 -> 12.7; 64 of 8192 would go from 60 to 62. Not where the blocks, one to an SM, come in several waves (four
  // sequences of 4096 with 32 rows each: 20.7 -> 25.6), nor beside the tile kernel, where the batch is not what these are of.
  if (!p.beside && pieces > 4 * kGroups && width * depth <= unsigned(ctx->sm_count)) return launch_dependent(cache_join_kernel<D, BF16, 512>, grid, 512, 0, stream, p, NT * 8, slots);
  return launch_dependent(cache_join_kernel<D, BF16, 256>, grid, 256, 0, stream, p, NT * 8, slots);
}

// Rows that count as few: 32 of 128 columns, 64 of 64. With 4 kv heads and a group of 4, streamed and tiled: 32 rows of 128
// columns 12.4 and 21.3 us (1 request of up to 4096 tokens), 44 and 70 (24 of them), 91 and 118 (64), 31 and 44 (1 of 60000);
// 64 rows: 16.1 and 21.6, 70 and 71, 163 and 119, 49 and 45. 64 rows of 64 columns: 12.1 and 19.4, 47 and 64, 106 and 110, 33
// and 36.
int64_t few_limit(int64_t d) { return d == 128 ? 32 : 64; }

// Rows of a streamed request: all of them where every request has few; where some have many, those with one new token
// (or the few that fit beside it) are streamed and the rest is tiled. The host knows bounds only, and a warp that is made for more
// rows costs a request that has one token as much as one that has them. Beside 2 prompts of 512 new tokens, up to 4096 tokens, 4 kv
// heads of 128, group 4, with 8 / 16 / 32 rows: 24 requests of one token 56 / 61 / 73 us, 60 of them 65 / 76 / 110, 4 beside one
// prompt 39 / 47 / 49; of four drafted tokens, which are tiled with 8: 24 requests 80 / 67 / 76 us, 60 120 / 82 / 116; of eight 79 /
// 79 / 78. Rows of 64 columns: 45 / 47 / 56, 49 / 54 / 81, 32 / 35 / 37; 76 / 49 / 57, 111 / 59 / 84; 75 / 75 / 58. Single tokens are
// what most requests bring beside a prompt.
int64_t few_rows(int64_t d, int64_t max_new, int64_t group) {
  if (max_new * group <= few_limit(d)) return max_new * group;
  return group <= 8 ? 8 : group <= 16 ? 16 : group <= 32 ? 32 : 0;
}

int64_t pieces_bytes(int64_t batch) { return batch * 16; }

// Rows of a warp: 8 or 16, as registers hold them (32 rows of 128 columns spilled: 58 us against 44 for two warps of 16 rows
// each, 24 requests of 8 x 4 rows over 4096 tokens; 32 of 64 columns leave room for 8 warps a block, not 12: 31.4 us against
// 30.0, 18.4 against 14.8 with 4 requests, 55 against 60 with 64). Where a request may have more, several warps share a stretch.
int64_t warp_rows(int64_t few) { return few <= 8 ? 8 : 16; }

int64_t row_blocks(int64_t few) { return (few + warp_rows(few) - 1) / warp_rows(few); }

// Of any smaller call too: `few` is the most rows that a call with up to max_new rows a request streams.
int64_t stream_workspace(int64_t batch, int64_t kv_heads, int64_t d, int64_t max_new, int64_t group) {
  const int64_t limit = few_limit(d), few = group > limit ? 0 : max_new * group < limit ? max_new * group : limit;
  const int64_t warps = int64_t(kMaxBlocks) * kMaxWarps, sharers = kv_heads * row_blocks(few);
  const int64_t units = warps > sharers ? warps : sharers;
  return pieces_bytes(batch) + 2 * units * warp_rows(few) * (d + 4) * 4;
}

template <int D, bool BF16>
int launch_stream_rows(const DeviceContext* ctx, const StreamParams& p, int64_t page_size, cudaStream_t stream) {
  return warp_rows(p.a.few) == 8 ? launch_stream<D, BF16, 1>(ctx, p, page_size, stream) : launch_stream<D, BF16, 2>(ctx, p, page_size, stream);
}

}  // namespace
}  // namespace krnb

extern "C" int64_t krn_b200_cache_attn_workspace_bytes(int64_t batch, int64_t rows, int64_t q_heads, int64_t kv_heads, int64_t d,
                                                       int64_t max_new, int64_t max_context) {
  using namespace krnb;
  if (batch <= 0 || rows <= 0 || q_heads <= 0 || kv_heads <= 0 || q_heads % kv_heads != 0 || d <= 0 || max_new <= 0) return 16;
  const int64_t group = q_heads / kv_heads, most = max_new < rows ? max_new : rows;  // no request has more rows than there are
  if (group > kMaxGroup) return 16;  // refused by the call
  return stream_workspace(batch, kv_heads, d, most, group) +
         (most * group <= few_limit(d) ? 0 : tile_workspace(batch, rows, q_heads, kv_heads, d, few_rows(d, most, group), max_context));
}

extern "C" int krn_b200_cache_attn(int type, const void* q, const void* k_pages, const void* v_pages, const float* k_scale,
                                   const float* v_scale, const int32_t* page_table, const int32_t* context_len,
                                   const int32_t* row_start, void* o, int64_t batch, int64_t rows, int64_t q_heads,
                                   int64_t kv_heads, int64_t d, int64_t page_size, int64_t num_pages, int64_t max_pages,
                                   int64_t table_pitch, int64_t max_new, int64_t max_context, const int64_t* strides,
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
  if (int rc = check_page_size(page_size)) return rc;
  if (batch < 0 || rows < 0 || q_heads <= 0 || kv_heads <= 0 || q_heads % kv_heads != 0 || num_pages <= 0 || max_pages <= 0 ||
      table_pitch < max_pages || max_new <= 0 || max_context <= 0) {
    return fail(KRN_B200_ERR_INVALID_ARGUMENT, "bad extents (batch %lld, %lld rows, %lld / %lld heads, %lld pages, table of %lld, "
                "max_new %lld, max_context %lld)", (long long)batch, (long long)rows, (long long)q_heads, (long long)kv_heads,
                (long long)num_pages, (long long)max_pages, (long long)max_new, (long long)max_context);
  }
  if (q_heads / kv_heads > kMaxGroup) {
    return fail(KRN_B200_ERR_UNSUPPORTED, "%lld q heads per kv head is not available: a tile holds %d rows. Instead: repeat the "
                "kv heads", (long long)(q_heads / kv_heads), kMaxGroup);
  }
  if (max_context > max_pages * page_size) {
    return fail(KRN_B200_ERR_INVALID_ARGUMENT, "max_context %lld does not fit %lld pages per sequence", (long long)max_context,
                (long long)max_pages);
  }
  if (batch == 0 || rows == 0) return KRN_B200_OK;
  if (batch > kMaxBatch) {
    return fail(KRN_B200_ERR_UNSUPPORTED, "a batch of %lld requests is not available: their tile counts sit in shared memory, at "
                "most %d fit. Instead: split the batch", (long long)batch, kMaxBatch);
  }
  if (batch * kv_heads * ((max_context + kTile - 1) / kTile) > INT32_MAX / 2 || q_heads > 65535 || rows > INT32_MAX / 256 || rows * q_heads > INT32_MAX / 2 ||
      max_context > INT32_MAX / 2 || num_pages >= INT32_MAX) {
    return fail(KRN_B200_ERR_UNSUPPORTED, "extents too large for this kernel's 32-bit indices");
  }
  if (q == nullptr || k_pages == nullptr || v_pages == nullptr || k_scale == nullptr || v_scale == nullptr ||
      page_table == nullptr || context_len == nullptr || row_start == nullptr || o == nullptr || strides == nullptr) {
    return fail(KRN_B200_ERR_INVALID_ARGUMENT, "null tensor address");
  }
  const int64_t *q_strides = strides, *o_strides = strides + 2, *k_page_strides = strides + 4, *v_page_strides = strides + 7;
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
  p.group_inverse = uint32_t((65536 + p.group - 1) / p.group);
  p.page_shift = shift_of(page_size);
  p.num_pages = int(num_pages);
  p.max_new = int(max_new < rows ? max_new : rows);
  p.max_context = int(max_context);
  p.scale_log2 = scale_log2;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_handle);
  const bool bf16 = type == KRN_B200_BF16;
  StreamParams sp;
  p.few = int(few_rows(d, p.max_new, p.group));
  sp.a = p;
  sp.pieces = static_cast<int4*>(workspace);
  sp.partial = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + pieces_bytes(batch));
  sp.row_blocks = int(row_blocks(p.few));
  // The two paths run side by side: the tile kernel first, whose blocks take longest, and the stream on the SMs that it
  // leaves free.
  const bool tiled = int64_t(p.max_new) * p.group > p.few && tile_blocks(batch, rows, p.group, p.few) > 0;
  void* split = static_cast<uint8_t*>(workspace) + stream_workspace(batch, kv_heads, d, p.max_new, p.group);
  sp.tiles = tiled ? tile_shares(p, split) : TileShares{nullptr, nullptr, 0};
  if (tiled) {
    if (int rc = launch_tiles(ctx, p, sp.tiles, bf16, d, page_size, stream)) return rc;
  }
  if (p.few > 0) {
    sp.beside = tiled;
    if (d == 128) return bf16 ? launch_stream_rows<128, true>(ctx, sp, page_size, stream) : launch_stream_rows<128, false>(ctx, sp, page_size, stream);
    return bf16 ? launch_stream_rows<64, true>(ctx, sp, page_size, stream) : launch_stream_rows<64, false>(ctx, sp, page_size, stream);
  }
  return tiled ? launch_tile_join(p, sp.tiles, bf16, d, stream) : KRN_B200_OK;
}
