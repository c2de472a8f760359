// The paged 8-bit cache: the step's plan (block tables and slot maps from request lengths) and the append that quantises
// new keys and values into pages with one power-of-two scale per (page, kv head).
//
// A pool is codes e4m3 [num_pages, page_size, kv_heads, d] for K and for V and f32 scales [num_pages, kv_heads] for each;
// value = code * scale. A token's slot is page * page_size + offset in the page.
//
// The reference has neither (its roadmap lists paged attention); the rounding to e4m3 is its narrowing rule, nearest even
// and saturating (src/krn/compiler/narrow.py:94-105).
#include "cache.cuh"

namespace krnb {
namespace {

enum Site { kSitePlanPage = 41, kSiteAppendSlot = 42 };

// ---- plan ----------------------------------------------------------------------------------------------------------

constexpr int kPlanThreads = 512;
constexpr int kPlanWarps = kPlanThreads / 32;
constexpr int kMaxBatch = 8192;             // four prefixes of the batch sit in shared memory
constexpr uint32_t kSaturated = 1u << 30;   // sums stop here: above every bound they are compared with

struct PlanParams {
  const int32_t* context_len;  // [batch]
  const int32_t* new_len;      // [batch], < 0: finished
  int32_t* page_table;         // [batch, max_pages], new entries are written
  int32_t* free_pages;         // ring [capacity], pages of finished requests are written
  const int64_t* pool_state;   // taken, given, -
  int32_t* context_out;        // [batch]
  int32_t* row_start;          // [batch + 1]
  int64_t* slot_map;           // [rows]
  int32_t* runs;               // [runs_len]
  int64_t* state_out;          // taken, given, refused
  int64_t table_pitch;
  int batch, max_pages, page_shift, rows, runs_len, num_pages, capacity;
};

__device__ __forceinline__ uint32_t add_saturated(uint32_t a, uint32_t b) { return min(a + b, kSaturated); }

// What one request asks of the step.
struct Request {
  int context, rows;         // tokens it holds, rows it brings
  int have;                  // pages it holds
  uint32_t need, lead, back; // pages it takes, page runs of its rows, pages it gives back
  bool wide;                 // its pages would not fit its row of the table
};

__device__ __forceinline__ Request request_at(const PlanParams& p, int i) {
  Request r;
  const int brings = p.new_len[i];
  const long long most = (long long)p.max_pages << p.page_shift;
  r.context = int(min((long long)max(p.context_len[i], 0), most));
  r.rows = min(max(brings, 0), p.rows + 1);  // one more than there is room for is refused all the same
  const int page = 1 << p.page_shift;
  const long long length = (long long)r.context + r.rows;
  const int after = int((length + page - 1) >> p.page_shift);
  r.have = (r.context + page - 1) >> p.page_shift;
  r.need = uint32_t(after - r.have);
  r.lead = r.rows > 0 ? uint32_t(((length - 1) >> p.page_shift) - (r.context >> p.page_shift) + 1) : 0u;
  r.back = brings < 0 ? uint32_t(r.have) : 0u;
  r.wide = after > p.max_pages;
  return r;
}

// Exclusive prefix of four sums over the block's threads in thread order, on top of `carry`, which moves on by their
// totals. `scratch` holds 4 * kPlanWarps values.
__device__ __forceinline__ void block_prefix(uint32_t (&v)[4], uint32_t (&carry)[4], uint32_t* scratch) {
  const int warp = threadIdx.x >> 5;
  const uint32_t lane = lane_id();
#pragma unroll
  for (int k = 0; k < 4; ++k) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t below = __shfl_up_sync(0xffffffffu, v[k], o);
      if (lane >= uint32_t(o)) v[k] = add_saturated(v[k], below);
    }
    if (lane == 31) scratch[k * kPlanWarps + warp] = v[k];
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    uint32_t before = carry[k], total = carry[k];
    for (int w = 0; w < kPlanWarps; ++w) {
      const uint32_t s = scratch[k * kPlanWarps + w];
      if (w < warp) before = add_saturated(before, s);
      total = add_saturated(total, s);
    }
    const uint32_t inclusive_before = __shfl_up_sync(0xffffffffu, v[k], 1);
    v[k] = add_saturated(before, lane == 0 ? 0u : inclusive_before);
    carry[k] = total;
  }
  __syncthreads();  // scratch is free again
}

// The last request whose prefix is at or before `k`: of those that share a prefix only the last has anything.
__device__ __forceinline__ int last_at_or_before(const uint32_t* prefix, int batch, int k) {
  int low = 0, high = batch;
  while (high - low > 1) {
    const int mid = (low + high) >> 1;
    if (prefix[mid] <= uint32_t(k)) low = mid; else high = mid;
  }
  return low;
}

// One launch, no communication between blocks: every block scans all request lengths by itself (a few loads per thread)
// and then fills its own part of the slot map, the run list and the table. Bound by latency: launch, one pass over the
// lengths, a binary search per row: 3.8 us for 16 requests, 6.7 us for 1000 with 41 000 new rows and 40 finished ones.
__global__ void __launch_bounds__(kPlanThreads) cache_plan_kernel(PlanParams p, DeviceStatus* status) {
  extern __shared__ uint32_t plan_smem[];
  uint32_t* start = plan_smem;                 // [batch + 1] first row of each request
  uint32_t* first = start + p.batch + 1;       // [batch] first page taken from the ring
  uint32_t* run = first + p.batch;             // [batch] first entry of the run list
  uint32_t* back = run + p.batch;              // [batch] first page given back to the ring
  uint32_t* scratch = back + p.batch;          // [4 * kPlanWarps]
  const int page = 1 << p.page_shift;
  wait_for_kernel_before();
  launch_dependents();

  // totals first: a step that does not fit takes nothing
  uint32_t carry[4] = {0, 0, 0, 0};
  bool wide = false;
  for (int base = 0; base < p.batch; base += kPlanThreads) {
    const int i = base + int(threadIdx.x);
    uint32_t v[4] = {0, 0, 0, 0};
    if (i < p.batch) {
      const Request r = request_at(p, i);
      wide |= r.wide;
      v[0] = uint32_t(r.rows);
      v[1] = r.need;
      v[2] = r.lead;
      v[3] = r.back;
    }
    block_prefix(v, carry, scratch);
    if (i < p.batch) {
      start[i] = v[0];
      first[i] = v[1];
      run[i] = v[2];
      back[i] = v[3];
    }
  }
  const long long taken = p.pool_state[0], given = p.pool_state[1];
  const long long available = max(0ll, min(given - taken, (long long)p.capacity));
  const bool any_wide = __syncthreads_or(wide) != 0;
  const bool refused = any_wide || carry[0] > uint32_t(p.rows) || (long long)carry[1] > available;
  const bool overfull = available + carry[3] > p.capacity;  // pages given back that the ring has no room for
  const uint32_t rows = refused ? 0u : carry[0], runs = refused ? 0u : carry[2];
  if (threadIdx.x == 0) start[p.batch] = rows;
  __syncthreads();

  const int here = blockIdx.x * kPlanThreads + threadIdx.x, stride = gridDim.x * kPlanThreads;
  if (here == 0) {
    p.state_out[0] = taken + (refused ? 0u : carry[1]);
    p.state_out[1] = given + (overfull ? 0u : carry[3]);
    p.state_out[2] = (refused ? 1 : 0) | (overfull ? 2 : 0);
  }
  for (int i = here; i <= p.batch; i += stride) {
    p.row_start[i] = refused ? 0 : int(start[i]);
    if (i < p.batch) {
      const Request r = request_at(p, i);
      p.context_out[i] = p.new_len[i] < 0 ? (overfull ? r.context : 0) : r.context + (refused ? 0 : r.rows);
    }
  }
  for (int i = here; i < p.runs_len; i += stride) {
    if (i >= int(runs)) p.runs[i] = -1;
  }

  // rows: request by binary search, page from the table or from the ring
  const long long taken_at = ((taken % p.capacity) + p.capacity) % p.capacity;
  const long long given_at = ((given % p.capacity) + p.capacity) % p.capacity;
  for (int r = here; r < p.rows; r += stride) {
    if (r >= int(rows)) {
      p.slot_map[r] = -1;
      continue;
    }
    const int low = last_at_or_before(start, p.batch, r);
    const long long most = (long long)p.max_pages << p.page_shift;
    const int context = int(min((long long)max(p.context_len[low], 0), most));
    const int have = (context + page - 1) >> p.page_shift;
    const int pos = context + r - int(start[low]);
    const int at = pos >> p.page_shift;
    int id;
    if (at < have) {
      id = p.page_table[low * p.table_pitch + at];
    } else {
      long long spot = taken_at + first[low] + (at - have);
      if (spot >= p.capacity) spot -= p.capacity;
      id = p.free_pages[spot];
    }
    const bool lead = r == int(start[low]) || (pos & (page - 1)) == 0;
    if (lead) {
      const int entry = int(run[low]) + at - (context >> p.page_shift);
      if (entry < p.runs_len) p.runs[entry] = r;
      if (at >= have) p.page_table[low * p.table_pitch + at] = id;
    }
    const bool good = uint32_t(id) < uint32_t(p.num_pages);
    if (!good) report_failure(status, kErrDeviceIndex, kSitePlanPage, uint32_t(id) & 0x7fffffffu);
    p.slot_map[r] = good ? ((long long)id << p.page_shift) + (pos & (page - 1)) : -1;
  }

  // pages of finished requests: handed out from the next step on
  if (!overfull) {
    for (int k = here; k < int(carry[3]); k += stride) {
      const int low = last_at_or_before(back, p.batch, k);
      long long spot = given_at + k;
      if (spot >= p.capacity) spot -= p.capacity;
      p.free_pages[spot] = p.page_table[low * p.table_pitch + (k - int(back[low]))];
    }
  }
}

size_t plan_smem_bytes(int64_t batch) { return size_t(4 * batch + 1 + 4 * kPlanWarps) * 4; }

// ---- append ----------------------------------------------------------------------------------------------------------

constexpr int kLeastExponent = -100;  // of a page's scale: a page of zeros, and of values that e4m3 * 2^-100 cannot tell from it

struct AppendSide {
  const uint16_t* x;   // [rows, heads, d] bf16 or f16
  long long x_row, x_head;
  uint8_t* pages;      // [num_pages, page_size, heads, d]
  long long page_pitch, token_pitch, head_pitch;
  float* scale;        // [num_pages, heads]
};

struct AppendParams {
  AppendSide side[2];      // K, V
  const int64_t* slot_map; // [rows]
  const int32_t* runs;     // [runs_len]
  int rows, runs_len, heads, page_shift, num_pages;
};

// The least power of two 2^k, k >= kLeastExponent, with a <= 448 * 2^k, read off a's exponent: 448 = 1.75 * 2^8.
__device__ __forceinline__ float scale_of(float a) {
  const uint32_t bits = __float_as_uint(a);
  int k = int(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  k = max(k, kLeastExponent);
  return __uint_as_float(uint32_t(k + 127) << 23);
}

__device__ __forceinline__ uint32_t codes_of(float2 v) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(v.y), "f"(v.x));
  return r;
}

__device__ __forceinline__ uint32_t rescale_two(uint32_t codes, float ratio) {
  const uint32_t h = halves_of(codes);
  const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&h));
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(v.y * ratio), "f"(v.x * ratio));
  return r;
}

// A thread group of `Threads` owns one (run, kv head, K or V): no two groups share a page's scale, so the new scale, the
// page's old codes and its new ones are settled without atomics, and the result does not depend on any order.
//   1. the group reads its rows once (16 bytes a thread and pass; up to kHeld passes stay in registers) and takes the
//      largest finite magnitude: bit patterns of magnitudes are ordered as they are, two 16-bit ones at a time, and only a
//      run that holds an infinity or a NaN is gone through value by value;
//   2. scale = max(old, least power of two that fits); a run that begins a page ignores what the page held;
//   3. where the scale grew, the codes already in the page are brought to it (a power-of-two ratio: only what falls below
//      e4m3's normal range is rounded again);
//   4. the rows go out as codes, 8 bytes a thread. Multiplying by the reciprocal of a power of two is the division itself;
//      a page that some other program filled may have any scale, and is divided by.
// The rows are under way before the slots that they go to are known. Bound by HBM for prompts (2 bytes in, 1 out per value):
// 16384 rows of 8 heads of 128, K and V, in pages of 64: 101 MB in 21.6 us = 4.7 TB/s; by launch and load latency for single
// tokens (64 of them: 2.4 us).
constexpr int kHeld = 8;

template <int D, bool BF16, int Threads>
__global__ void __launch_bounds__(128) cache_append_kernel(AppendParams p, DeviceStatus* status) {
  constexpr int kLanes = D / 8;                // threads per row
  constexpr int kRows = Threads / kLanes;      // rows per pass
  constexpr int kGroups = 128 / Threads;       // (run, head, side) items per block
  constexpr uint32_t kInfinity = BF16 ? 0x7f80u : 0x7c00u;
  __shared__ uint32_t peaks[4];
  const int tid = threadIdx.x % Threads;
  const uint32_t item = blockIdx.x * kGroups + threadIdx.x / Threads, per_run = 2u * uint32_t(p.heads);
  const int u = int(item / per_run), which = int(item - uint32_t(u) * per_run);
  wait_for_kernel_before();
  launch_dependents();
  if (u >= p.runs_len) return;
  const int first = p.runs[u], next = u + 1 < p.runs_len ? p.runs[u + 1] : -1;
  if (uint32_t(first) >= uint32_t(p.rows)) return;
  const int page_size = 1 << p.page_shift;
  int most = min(page_size, p.rows - first);
  if (next > first) most = min(most, next - first);
  const AppendSide& side = p.side[which >= p.heads ? 1 : 0];
  const int head = which >= p.heads ? which - p.heads : which;
  const int lane = tid % kLanes, row0 = tid / kLanes;
  const uint16_t* x = side.x + first * side.x_row + head * side.x_head + lane * 8;
  uint4 held[kHeld];
#pragma unroll
  for (int i = 0; i < kHeld; ++i) {
    const int row = row0 + i * kRows;
    held[i] = row < most ? *reinterpret_cast<const uint4*>(x + row * side.x_row) : make_uint4(0, 0, 0, 0);
  }

  // where the rows go: slots that follow one another within the page
  const long long slot = p.slot_map[first];
  const long long page_id = slot >> p.page_shift;
  if (slot < 0 || page_id >= p.num_pages) {
    if (slot >= 0) report_failure(status, kErrDeviceIndex, kSiteAppendSlot, uint32_t(first));
    return;
  }
  const int offset = int(slot) & (page_size - 1);
  most = min(most, page_size - offset);
  int count = 0;
  for (int base = 0; base < most; base += 32) {
    const int i = base + int(lane_id());
    const uint32_t follows = __ballot_sync(0xffffffffu, i < most && p.slot_map[first + i] == slot + i);
    count = base + (follows == 0xffffffffu ? 32 : __ffs(int(~follows)) - 1);
    if (follows != 0xffffffffu) break;
  }
  float* scale_at = side.scale + page_id * p.heads + head;
  const float old = offset > 0 ? *scale_at : 0.f;

  // the largest magnitude
  auto all_rows = [&](auto take) {
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
      if (row0 + i * kRows < count) take(held[i], row0 + i * kRows);
    }
    for (int row = row0 + kHeld * kRows; row < count; row += kRows) take(*reinterpret_cast<const uint4*>(x + row * side.x_row), row);
  };
  auto group_max = [&](uint32_t v) {  // of both halves, over the group
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = __vmaxu2(v, __shfl_xor_sync(0xffffffffu, v, o));
    if constexpr (Threads > 32) {
      __syncthreads();
      if (lane_id() == 0) peaks[threadIdx.x >> 5] = v;
      __syncthreads();
      v = __vmaxu2(__vmaxu2(peaks[0], peaks[1]), __vmaxu2(peaks[2], peaks[3]));
    }
    return max(v & 0xffffu, v >> 16);
  };
  uint32_t bits = 0;
  all_rows([&](const uint4& w, int) {
    constexpr uint32_t kSize = 0x7fff7fffu;
    bits = __vmaxu2(__vmaxu2(bits, __vmaxu2(w.x & kSize, w.y & kSize)), __vmaxu2(w.z & kSize, w.w & kSize));
  });
  bits = group_max(bits);
  if (bits >= kInfinity) {
    bits = 0;
    all_rows([&](const uint4& w, int) {
      const uint32_t words[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint32_t size = (words[e >> 1] >> (16 * (e & 1))) & 0x7fffu;
        if (size < kInfinity) bits = max(bits, size);
      }
    });
    bits = group_max(bits);
  }
  const float now = fmaxf(old, scale_of(unpack<BF16>(bits).x));

  uint8_t* page = side.pages + page_id * side.page_pitch + head * side.head_pitch;
  if (now != old && offset > 0) {
    const float ratio = old / now;
    for (int i = tid; i < offset * (D / 16); i += Threads) {
      uint4* spot = reinterpret_cast<uint4*>(page + (i / (D / 16)) * side.token_pitch + (i % (D / 16)) * 16);
      uint4 w = *spot;
      w.x = rescale_two(w.x, ratio) | rescale_two(w.x >> 16, ratio) << 16;
      w.y = rescale_two(w.y, ratio) | rescale_two(w.y >> 16, ratio) << 16;
      w.z = rescale_two(w.z, ratio) | rescale_two(w.z >> 16, ratio) << 16;
      w.w = rescale_two(w.w, ratio) | rescale_two(w.w >> 16, ratio) << 16;
      *spot = w;
    }
  }
  uint8_t* out = page + offset * side.token_pitch + lane * 8;
  if ((__float_as_uint(now) & 0x7fffffu) == 0) {
    const float by = 1.0f / now;
    auto two = [&](uint32_t w) {
      const float2 v = unpack<BF16>(w);
      return codes_of(make_float2(v.x * by, v.y * by));
    };
    all_rows([&](const uint4& w, int row) {
      *reinterpret_cast<uint2*>(out + row * side.token_pitch) = make_uint2(two(w.x) | two(w.y) << 16, two(w.z) | two(w.w) << 16);
    });
  } else {
    all_rows([&](const uint4& w, int row) {
      const uint32_t words[4] = {w.x, w.y, w.z, w.w};
      uint32_t codes[4];
#pragma unroll 1
      for (int e = 0; e < 4; ++e) {
        const float2 v = unpack<BF16>(words[e]);
        codes[e] = codes_of(make_float2(v.x / now, v.y / now));
      }
      *reinterpret_cast<uint2*>(out + row * side.token_pitch) = make_uint2(codes[0] | codes[1] << 16, codes[2] | codes[3] << 16);
    });
  }
  // every thread has read the old scale before it is replaced
  if constexpr (Threads > 32) __syncthreads(); else __syncwarp();
  if (tid == 0 && now != old) *scale_at = now;
}

template <int D, bool BF16, int Threads>
int launch_append(const AppendParams& p, DeviceStatus* status, cudaStream_t stream) {
  const long long items = (long long)p.runs_len * 2 * p.heads;
  const long long blocks = (items + 128 / Threads - 1) / (128 / Threads);
  return launch_dependent(cache_append_kernel<D, BF16, Threads>, dim3(unsigned(blocks)), 128, 0, stream, p, status);
}

struct Span {
  const void* at;
  int64_t bytes;
};

bool overlap(const Span& a, const Span& b) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a.at), y = reinterpret_cast<uintptr_t>(b.at);
  return a.bytes > 0 && b.bytes > 0 && (x < y ? y - x < uint64_t(a.bytes) : x - y < uint64_t(b.bytes));
}

// Whether `a` meets one of `count` rows of `bytes` bytes, `pitch` bytes apart: the row that begins at or before it, or the
// next one.
bool overlaps_table(const Span& a, const void* table, int64_t count, int64_t bytes, int64_t pitch) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a.at), y = reinterpret_cast<uintptr_t>(table);
  const int64_t row = x < y ? 0 : int64_t((x - y) / uint64_t(pitch));
  for (int64_t i = row; i <= row + 1 && i < count; ++i) {
    if (overlap(a, {static_cast<const char*>(table) + i * pitch, bytes})) return true;
  }
  return false;
}

}  // namespace
}  // namespace krnb

extern "C" int64_t krn_b200_cache_runs(int64_t rows, int64_t batch, int64_t page_size) {
  if (rows <= 0 || batch <= 0 || page_size <= 0) return 0;
  // a request of n rows touches at most (n + page_size - 2) / page_size + 1 pages, and at most n
  const int64_t bound = rows / page_size + 2 * batch;
  return rows < bound ? rows : bound;
}

extern "C" int krn_b200_cache_plan(const int32_t* context_len, const int32_t* new_len, int32_t* page_table,
                                   int32_t* free_pages, const int64_t* pool_state, int32_t* context_out, int32_t* row_start,
                                   int64_t* slot_map, int32_t* runs, int64_t* state_out, int64_t batch, int64_t max_pages,
                                   int64_t table_pitch, int64_t capacity, int64_t page_size, int64_t num_pages, int64_t rows,
                                   int64_t runs_len, void* stream_handle) {
  using namespace krnb;
  if (int rc = check_page_size(page_size)) return rc;
  if (batch < 0 || max_pages <= 0 || capacity <= 0 || num_pages <= 0 || rows < 0 || table_pitch < max_pages) {
    return fail(KRN_B200_ERR_INVALID_ARGUMENT, "bad extents (batch %lld, %lld table entries at pitch %lld, ring of %lld, %lld "
                "pages, %lld rows)", (long long)batch, (long long)max_pages, (long long)table_pitch, (long long)capacity,
                (long long)num_pages, (long long)rows);
  }
  if (batch > kMaxBatch) {
    return fail(KRN_B200_ERR_UNSUPPORTED, "a plan for %lld requests is not available: their prefix sums sit in shared memory, "
                "at most %d fit. Instead: plan the batch in parts", (long long)batch, kMaxBatch);
  }
  if (rows >= int64_t(kSaturated) || capacity >= int64_t(kSaturated) || num_pages >= INT32_MAX ||
      max_pages * page_size >= int64_t(kSaturated)) {
    return fail(KRN_B200_ERR_UNSUPPORTED, "extents too large for this kernel's 32-bit sums");
  }
  if (runs_len < krn_b200_cache_runs(rows, batch, page_size) || runs_len > INT32_MAX) {
    return fail(KRN_B200_ERR_INVALID_ARGUMENT, "a run list of %lld entries is too short: %lld needed", (long long)runs_len,
                (long long)krn_b200_cache_runs(rows, batch, page_size));
  }
  if (batch == 0) return fail(KRN_B200_ERR_INVALID_ARGUMENT, "a plan needs at least one request");
  if (context_len == nullptr || new_len == nullptr || page_table == nullptr || free_pages == nullptr || pool_state == nullptr ||
      context_out == nullptr || row_start == nullptr || state_out == nullptr || (rows > 0 && slot_map == nullptr) ||
      (runs_len > 0 && runs == nullptr)) {
    return fail(KRN_B200_ERR_INVALID_ARGUMENT, "null tensor address");
  }
  // what is written comes first: it shares no memory with anything before or behind it in the list
  const Span spans[] = {{context_out, batch * 4}, {row_start, (batch + 1) * 4}, {slot_map, rows * 8}, {runs, runs_len * 4},
                        {state_out, 24}, {free_pages, capacity * 4}, {context_len, batch * 4}, {new_len, batch * 4},
                        {pool_state, 24}};
  constexpr int kWritten = 6, kSpans = int(sizeof(spans) / sizeof(spans[0]));
  bool shared = false;
  for (int i = 0; i < kSpans; ++i) {
    for (int j = i + 1; j < kSpans && i < kWritten; ++j) shared |= overlap(spans[i], spans[j]);
    shared |= overlaps_table(spans[i], page_table, batch, max_pages * 4, table_pitch * 4);
  }
  if (shared) {
    return fail(KRN_B200_ERR_INVALID_ARGUMENT, "the plan's outputs must not share memory with its inputs or with one another: "
                "blocks read the lengths while others write");
  }
  DeviceContext* ctx = current_context();
  if (ctx == nullptr) return KRN_B200_ERR_CUDA;
  if (int rc = require_sm100(ctx)) return rc;
  PlanParams p = {context_len, new_len, page_table, free_pages, pool_state, context_out, row_start, slot_map, runs, state_out,
                  table_pitch, int(batch), int(max_pages), shift_of(page_size), int(rows), int(runs_len), int(num_pages),
                  int(capacity)};
  const size_t smem = plan_smem_bytes(batch);
  static OncePerDevice ready;
  if (int rc = ready(ctx->device, [] {
        KRNB_CUDA(cudaFuncSetAttribute(cache_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(plan_smem_bytes(kMaxBatch))));
        return KRN_B200_OK;
      })) {
    return rc;
  }
  // a thread per row, and blocks enough for the pages of a few finished requests
  const int64_t wanted = (rows + batch * 8 + kPlanThreads - 1) / kPlanThreads;
  const int blocks = int(wanted < 1 ? 1 : wanted > ctx->sm_count ? ctx->sm_count : wanted);
  return launch_dependent(cache_plan_kernel, dim3(unsigned(blocks)), kPlanThreads, smem, static_cast<cudaStream_t>(stream_handle), p,
                          ctx->status_dev);
}

extern "C" int krn_b200_cache_append(int type, const void* k, const void* v, const int64_t* slot_map, const int32_t* runs,
                                     void* k_pages, void* v_pages, float* k_scale, float* v_scale, int64_t rows,
                                     int64_t runs_len, int64_t heads, int64_t d, int64_t page_size, int64_t num_pages,
                                     const int64_t* strides, void* stream_handle) {
  using namespace krnb;
  if (type != KRN_B200_BF16 && type != KRN_B200_F16) {
    return fail(KRN_B200_ERR_UNSUPPORTED, "cache append of element type %d is not available on sm_100a: keys and values come in "
                "16 bits. Instead: pass bf16 or f16 tensors", type);
  }
  if (d != 64 && d != 128) {
    return fail(KRN_B200_ERR_UNSUPPORTED, "head dimension %lld is not available on sm_100a. Instead: use d = 64 or d = 128",
                (long long)d);
  }
  if (int rc = check_page_size(page_size)) return rc;
  if (rows < 0 || runs_len < 0 || heads <= 0 || num_pages <= 0) {
    return fail(KRN_B200_ERR_INVALID_ARGUMENT, "bad extents (%lld rows, %lld runs, %lld heads, %lld pages)", (long long)rows,
                (long long)runs_len, (long long)heads, (long long)num_pages);
  }
  if (rows == 0 || runs_len == 0) return KRN_B200_OK;
  if (rows > INT32_MAX / 2 || num_pages >= INT32_MAX || heads > 65535 || runs_len * 2 * heads > INT32_MAX) {
    return fail(KRN_B200_ERR_UNSUPPORTED, "extents too large for this kernel's 32-bit indices");
  }
  if (k == nullptr || v == nullptr || slot_map == nullptr || runs == nullptr || k_pages == nullptr || v_pages == nullptr ||
      k_scale == nullptr || v_scale == nullptr || strides == nullptr) {
    return fail(KRN_B200_ERR_INVALID_ARGUMENT, "null tensor address");
  }
  const int64_t *k_strides = strides, *v_strides = strides + 2, *k_page_strides = strides + 4, *v_page_strides = strides + 7;
  if (!aligned16(k) || !aligned16(v) || !aligned16(k_pages) || !aligned16(v_pages) || k_strides[0] % 8 || k_strides[1] % 8 ||
      v_strides[0] % 8 || v_strides[1] % 8) {
    return fail(KRN_B200_ERR_INVALID_ARGUMENT, "rows are read 16 bytes at a time: addresses and strides must be multiples of 16 bytes");
  }
  for (int i = 0; i < 3; ++i) {
    if (k_page_strides[i] % 16 || v_page_strides[i] % 16 || k_page_strides[i] <= 0 || v_page_strides[i] <= 0) {
      return fail(KRN_B200_ERR_INVALID_ARGUMENT, "the strides of a page pool must be positive multiples of 16 bytes");
    }
  }
  DeviceContext* ctx = current_context();
  if (ctx == nullptr) return KRN_B200_ERR_CUDA;
  if (int rc = require_sm100(ctx)) return rc;
  AppendParams p;
  p.side[0] = {static_cast<const uint16_t*>(k), k_strides[0], k_strides[1], static_cast<uint8_t*>(k_pages), k_page_strides[0],
               k_page_strides[1], k_page_strides[2], k_scale};
  p.side[1] = {static_cast<const uint16_t*>(v), v_strides[0], v_strides[1], static_cast<uint8_t*>(v_pages), v_page_strides[0],
               v_page_strides[1], v_page_strides[2], v_scale};
  p.slot_map = slot_map;
  p.runs = runs;
  p.rows = int(rows);
  p.runs_len = int(runs_len);
  p.heads = int(heads);
  p.page_shift = shift_of(page_size);
  p.num_pages = int(num_pages);
  cudaStream_t stream = static_cast<cudaStream_t>(stream_handle);
  const bool bf16 = type == KRN_B200_BF16;
  // A warp per (run, head, side) or a block? The run list is padded, and a block costs as much for an empty entry as for a
  // full one; a warp is slow at runs that its registers (16 rows of 128) do not hold. Where all blocks are resident at once
  // a block pays from 6 rows an entry: 20 requests of 16 / 24 / 64 rows, 8 heads of 128, pages of 64: warp 2.6 / 3.5 / 7.0 us,
  // block 2.6 / 2.7 / 3.0. Where they are not, from 16 rows an entry in pages that hold more than 32: 200 requests of
  // 16 / 40 / 64 rows: warp 5.3 / 16.3 / 22.3, block 12.0 / 18.1 / 22.1; 8 of 2048 in pages of 16 / 32 / 64: warp
  // 19.9 / 25.1 / 34.8, block 40.5 / 25.3 / 21.6.
  const bool resident = runs_len * 2 * heads <= 8 * int64_t(ctx->sm_count);
  const bool block = resident ? page_size > 16 && rows > 6 * runs_len : page_size > 32 && rows > 16 * runs_len;
  if (!block) {
    if (d == 128) return bf16 ? launch_append<128, true, 32>(p, ctx->status_dev, stream) : launch_append<128, false, 32>(p, ctx->status_dev, stream);
    return bf16 ? launch_append<64, true, 32>(p, ctx->status_dev, stream) : launch_append<64, false, 32>(p, ctx->status_dev, stream);
  }
  if (d == 128) return bf16 ? launch_append<128, true, 128>(p, ctx->status_dev, stream) : launch_append<128, false, 128>(p, ctx->status_dev, stream);
  return bf16 ? launch_append<64, true, 128>(p, ctx->status_dev, stream) : launch_append<64, false, 128>(p, ctx->status_dev, stream);
}
