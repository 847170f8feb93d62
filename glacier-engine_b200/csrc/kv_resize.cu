// Block tables and slot maps on the device, from request lengths: the page
// bookkeeping of PagedKVCache (src/paged_kv_cache.zig:44-48 request page tables,
// :1074 appendRowTxn's page of a position) for all lanes of a batch in one launch.
#include <algorithm>

#include "kv_q4.cuh"

namespace glacier {

namespace {

constexpr int kMaxLanes = 1024;     // one per thread
constexpr int kRowsPerCta = 2048;   // rows that a CTA of the rows kernel takes before another is started

struct ResizeParams {
  int32_t* lens;
  const int32_t* targets;
  int32_t* tables;       // [lanes, max_pages]
  int32_t* free_pages;   // stack of capacity entries
  int32_t* free_count;
  int32_t* status;
  int32_t* row_offsets;  // [lanes + 1] or null
  int32_t* positions;    // [rows] each, or null
  int32_t* row_lanes;
  int64_t* slots;
  long long rows;
  int lanes, max_pages, capacity, row_stride;
};

// Inclusive sums over the block's first `warps` warps of N values per thread, and their totals.  Each
// warp scans its own, then every warp scans the warps' sums for itself: one barrier.  `sh` is used once.
template <int N, typename T>
__device__ __forceinline__ void block_scan(T (&v)[N], T (&total)[N], T (*sh)[32], int warps) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1)
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const T t = __shfl_up_sync(0xffffffffu, v[i], o);
      if (lane >= o) v[i] += t;
    }
  if (lane == 31)
#pragma unroll
    for (int i = 0; i < N; ++i) sh[i][warp] = v[i];
  asm volatile("bar.sync 1, %0;" ::"r"(32 * warps) : "memory");
#pragma unroll
  for (int i = 0; i < N; ++i) {
    T w = lane < warps ? sh[i][lane] : 0;
    const T own = __shfl_sync(0xffffffffu, w, warp);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const T t = __shfl_up_sync(0xffffffffu, w, o);
      if (lane >= o) w += t;
    }
    v[i] += __shfl_sync(0xffffffffu, w, warp) - own;
    total[i] = __shfl_sync(0xffffffffu, w, 31);
  }
}

// Lane `b` of the sorted prefix sums `first` (n of them) that holds item i: the last with first <= i.
__device__ __forceinline__ int holder(const int* first, int n, int i) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (first[mid] <= i) lo = mid; else hi = mid - 1;
  }
  return lo;
}

__device__ __forceinline__ int pages_of(int positions) { return (positions + kQ4Page - 1) / kQ4Page; }

// Every CTA works the whole batch out for itself (a thread per lane, two scans over the warps that
// have lanes): that takes less time than passing results on.  The stack's order is arithmetic: pages
// that shrinking lanes give back lie above the old top so that the next pops return them in lane and page
// order (growing again undoes the shrink), and growing lanes pop in lane order.  A page that is given back
// and taken in one call is therefore found in the table it comes from, and nothing waits for another
// thread's writes.  Once the pages or rows run out, that lane and every later one that
// needs any is refused and left as it was.  No atomics: the result depends on the inputs alone.
//
// MOVE writes rows and pages: nothing in it reads what it writes (rows read the pages that a lane
// held before, pages given back go above the old top).  STATE sets lengths, count and statuses,
// which everything reads.  Few rows: one CTA does both.  Many: a grid of MOVE CTAs, then a STATE CTA
// behind it.
//
// The time is latency: the floor of 64 lanes' bytes is a nanosecond.  A decode step's call takes 2.8 us (64
// lanes, most with no page to move), half of it the launch and the first loads; code that runs once is
// fetched for it, so the form for few rows takes a row and a page per thread (four of each, laid out
// straight, took 5.6).  128 prompts of 1 to 4096 positions (267,000 rows, 16,800 pages): 17.9 us to grow
// and to give back.
template <bool MOVE, bool STATE>
__global__ void __launch_bounds__(kMaxLanes, 1) kv_resize_kernel(const ResizeParams p) {
  __shared__ long long sh_want[3][32];
  __shared__ int sh_got[2][32];
  __shared__ int s_old[kMaxLanes], s_first[kMaxLanes], s_give[kMaxLanes], s_new[kMaxLanes];
  __shared__ int s_given, s_taken;  // pages given back and taken by all lanes
  __shared__ int s_off[kMaxLanes + 1];  // packed: each lane's first row; padded: its number of rows, one further on
  griddep_launch();
  griddep_wait();
  const int tid = threadIdx.x, scanners = (p.lanes + 31) / 32;  // warps that have lanes
  const bool lane_on = tid < p.lanes;
  const int count = min(max(*p.free_count, 0), p.capacity);
  bool valid = false, ok = false;
  int target = 0;
  if (tid < 32 * scanners) {
    const int old_len = lane_on ? p.lens[tid] : 0;
    target = lane_on ? p.targets[tid] : 0;
    const int limit = p.max_pages * kQ4Page;
    valid = lane_on && old_len >= 0 && old_len <= limit && target >= 0 && target <= limit &&
            (p.row_stride == 0 || target - old_len <= p.row_stride);
    const int have = valid ? pages_of(old_len) : 0, want = valid ? pages_of(target) : 0;
    const int give = max(have - want, 0), need = max(want - have, 0), grow = valid ? max(target - old_len, 0) : 0;

    long long want_sum[3] = {give, need, grow}, want_all[3];
    block_scan(want_sum, want_all, sh_want, scanners);
    const int give_sum = (int)want_sum[0], need_sum = (int)want_sum[1];
    const bool rows_fit = p.row_stride != 0 || want_sum[2] <= (p.slots ? p.rows : (long long)INT32_MAX);
    ok = valid && (need == 0 || need_sum <= min(count + want_all[0], (long long)p.capacity)) && (grow == 0 || rows_fit);
    int got[2] = {ok ? grow : 0, ok ? need : 0}, got_all[2];
    block_scan(got, got_all, sh_got, scanners);
    s_old[tid] = old_len;
    s_new[tid] = ok ? target : -1;
    s_first[tid] = need_sum - need;
    s_give[tid] = give_sum - give;
    s_off[tid + 1] = p.row_stride ? (ok ? grow : 0) : got[0];
    if (tid == 0) {
      s_off[0] = 0;
      s_given = (int)want_all[0];
      s_taken = got_all[1];
    }
  }
  __syncthreads();
  const int given = s_given, taken = s_taken, avail = (int)min((long long)count + given, (long long)p.capacity);
  const unsigned top = (unsigned)count + given;  // of the stack with all of them: up to 2^32
  // Entry `at` of the stack after the shrinking lanes gave their pages back.
  auto stack = [&](int at) -> const int32_t* {
    if (at < count) return p.free_pages + at;
    const int j = (int)(top - 1 - at), b = holder(s_give, p.lanes, j);
    return p.tables + (size_t)b * p.max_pages + pages_of(s_new[b]) + j - s_give[b];
  };
  // Page k of lane b, of those it held (h) or takes.
  auto page_at = [&](int b, int k) {
    const int h = pages_of(s_old[b]);
    return k < h ? p.tables + (size_t)b * p.max_pages + k : stack(avail - 1 - (s_first[b] + k - h));
  };

  if constexpr (MOVE) {
    const int n = p.slots ? (int)p.rows : 0, live_end = s_off[p.lanes];
    const long long me = (long long)blockIdx.x * blockDim.x + tid, all = (long long)gridDim.x * blockDim.x;
    auto lane_of = [&](int r) { return p.row_stride ? r / p.row_stride : holder(s_off, p.lanes, r); };
    auto one_row = [&](int r, int b) {
      const int i = r - (p.row_stride ? b * p.row_stride : s_off[b]);
      const bool live = p.row_stride ? i < s_off[b + 1] : r < live_end;
      const int pos = live ? s_old[b] + i : -1;
      p.positions[r] = pos;
      p.row_lanes[r] = live ? b : -1;
      p.slots[r] = live ? (long long)*page_at(b, pos / kQ4Page) * kQ4Page + pos % kQ4Page : -1;
    };
    if constexpr (STATE) {
#pragma unroll 1
      for (long long r = me; r < n; r += all) one_row((int)r, lane_of((int)r));
    } else {
      // Four rows per thread: at most two pages, when they are one lane's.
      const bool vec = (((uintptr_t)p.positions | (uintptr_t)p.row_lanes | (uintptr_t)p.slots) & 15) == 0;
#pragma unroll 1
      for (long long r4 = 4 * me; r4 < n; r4 += 4 * all) {
        const int r = (int)r4, b = lane_of(r), i = r - (p.row_stride ? b * p.row_stride : s_off[b]);
        const int left = (p.row_stride ? s_off[b + 1] : s_off[b + 1] - s_off[b]) - i;  // the lane's rows from here
        const bool none = p.row_stride ? left <= 0 && i + 4 <= p.row_stride : r >= live_end;
        if (vec && r4 + 4 <= n && (left >= 4 || none)) {
          int4 pos = make_int4(-1, -1, -1, -1), who = pos;
          longlong2 s0 = make_longlong2(-1, -1), s1 = s0;
          if (!none) {
            const int at = s_old[b] + i, k = at / kQ4Page;
            const int32_t *first = page_at(b, k), *last = (at + 3) / kQ4Page == k ? first : page_at(b, k + 1);
            const long long x = (long long)*first * kQ4Page, y = (long long)*last * kQ4Page;
            const int in = at % kQ4Page;
            pos = make_int4(at, at + 1, at + 2, at + 3);
            who = make_int4(b, b, b, b);
            s0.x = x + in;
            s0.y = (in + 1 < kQ4Page ? x : y) + (in + 1) % kQ4Page;
            s1.x = (in + 2 < kQ4Page ? x : y) + (in + 2) % kQ4Page;
            s1.y = (in + 3 < kQ4Page ? x : y) + (in + 3) % kQ4Page;
          }
          *reinterpret_cast<int4*>(p.positions + r) = pos;
          *reinterpret_cast<int4*>(p.row_lanes + r) = who;
          *reinterpret_cast<longlong2*>(p.slots + r) = s0;
          *reinterpret_cast<longlong2*>(p.slots + r + 2) = s1;
        } else {
#pragma unroll 1
          for (int c = 0; c < 4 && r4 + c < n; ++c) one_row(r + c, lane_of(r + c));
        }
      }
    }
    // Pages given back and taken.
    const int moves = given + taken;
    if (moves <= all) {
      // Laid end to end, one per thread; the block's last threads begin, beside the first ones' rows.
      const int i = (int)(me - tid) + (int)blockDim.x - 1 - tid;
      if (i < given) {
        const int b = holder(s_give, p.lanes, i);
        const unsigned at = top - 1 - i;
        if (at < (unsigned)p.capacity)  // more pages than the stack holds are dropped
          p.free_pages[at] = p.tables[(size_t)b * p.max_pages + pages_of(s_new[b]) + i - s_give[b]];
      } else if (i < moves) {
        const int j = i - given, b = holder(s_first, p.lanes, j);
        p.tables[(size_t)b * p.max_pages + pages_of(s_old[b]) + j - s_first[b]] = *stack(avail - 1 - j);
      }
    } else {
      // A lane's pages to a group of threads (as many as a lane has pages on average, a warp at most), or
      // to several when there are more groups than lanes: four per thread, loads before stores.
      const int log = min(5, 31 - __clz(max(1, moves / p.lanes))), size = 1 << log;
      const int groups = (int)(all >> log), per = max(1, groups / p.lanes), group = (int)(me >> log);
#pragma unroll 1
      for (int b = group / per; b < p.lanes; b += groups / per) {
        const int old_pages = pages_of(s_old[b]), diff = s_new[b] < 0 ? 0 : pages_of(s_new[b]) - old_pages;
        int32_t* table = p.tables + (size_t)b * p.max_pages + min(old_pages, old_pages + diff);
#pragma unroll 1
        for (int x0 = 4 * size * (group % per) + (tid & (size - 1)); x0 < abs(diff); x0 += 4 * size * per) {
          int page[4];
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const int x = x0 + size * c;
            if (x < abs(diff)) page[c] = diff < 0 ? table[x] : *stack(avail - 1 - (s_first[b] + x));
          }
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const int x = x0 + size * c;
            const unsigned at = top - 1 - (s_give[b] + x);
            if (x < abs(diff) && diff > 0) table[x] = page[c];
            if (x < -diff && at < (unsigned)p.capacity) p.free_pages[at] = page[c];
          }
        }
      }
    }
  }
  if constexpr (STATE) {
    if (ok) p.lens[tid] = target;
    if (lane_on) p.status[tid] = ok ? GLACIER_CUDA_OK : valid ? GLACIER_CUDA_ENOMEM : GLACIER_CUDA_EINVAL;
    if (tid == 0) *p.free_count = avail - taken;
    if (p.row_offsets)
      for (int i = tid; i <= p.lanes; i += blockDim.x) p.row_offsets[i] = p.row_stride ? i * p.row_stride : s_off[i];
  }
}

}  // namespace

int kv_resize(int32_t* lens, const int32_t* targets, size_t lanes, int32_t* block_tables, size_t max_pages,
              int32_t* free_pages, size_t capacity, int32_t* free_count, int32_t* status, size_t row_stride,
              size_t rows, int32_t* positions, int32_t* row_lanes, int64_t* slots, int32_t* row_offsets,
              cudaStream_t stream) {
  GLC_REQUIRE(lens && targets && block_tables && free_pages && free_count && status, "kv_resize: null argument");
  GLC_REQUIRE(lens != targets, "kv_resize: lens and targets are the same array");
  GLC_REQUIRE(lanes > 0 && lanes <= (size_t)kMaxLanes, "kv_resize: %zu lanes (1 to %d)", lanes, kMaxLanes);
  GLC_REQUIRE(max_pages > 0 && max_pages <= ((size_t)1 << 26) && lanes * max_pages < ((size_t)1 << 31) && capacity > 0 &&
                  capacity < ((size_t)1 << 31),
              "kv_resize: %zu pages per lane, %zu in all", max_pages, capacity);
  const int given = (positions ? 1 : 0) + (row_lanes ? 1 : 0) + (slots ? 1 : 0);
  GLC_REQUIRE(given == 0 || given == 3, "kv_resize: positions, row_lanes and slots go together");
  GLC_REQUIRE(rows < ((size_t)1 << 31) && row_stride < ((size_t)1 << 31), "kv_resize: %zu rows", rows);
  GLC_REQUIRE(row_stride == 0 || given == 0 || rows == lanes * row_stride,
              "kv_resize: %zu rows for %zu lanes of %zu", rows, lanes, row_stride);
  GLC_REQUIRE(row_stride == 0 || lanes * row_stride < ((size_t)1 << 31), "kv_resize: too many rows");
  GLC_REQUIRE(given == 0 || rows > 0, "kv_resize: no rows");
  ResizeParams p;
  p.lens = lens;
  p.targets = targets;
  p.tables = block_tables;
  p.free_pages = free_pages;
  p.free_count = free_count;
  p.status = status;
  p.row_offsets = row_offsets;
  p.positions = positions;
  p.row_lanes = row_lanes;
  p.slots = slots;
  p.rows = (long long)rows;
  p.lanes = (int)lanes;
  p.max_pages = (int)max_pages;
  p.capacity = (int)capacity;
  p.row_stride = (int)row_stride;
  const unsigned lane_threads = (unsigned)ceil_div(lanes, (size_t)32) * 32;
  if (!given)  // pages only, and how many is known on the device alone: threads for all that there can be
    return launch_pdl(kv_resize_kernel<true, true>, dim3(1),
                      dim3(std::max(lane_threads, lanes * max_pages > 1024 ? 1024u : 256u)), 0, stream, 1, p);
  // Two rows per thread in one CTA: from there on a second launch pays (64 lanes grown from nothing: 5.4
  // us in one CTA against 5.3 in two launches at 2048 rows, 6.0 and 5.5 at 4096, 9.4 and 5.7 at 8192, 56
  // and 6.0 at 65536; at 64 rows one CTA takes 2.7).
  if (rows <= 2 * kMaxLanes) {
    const unsigned threads = std::max({128u, lane_threads, std::min(1024u, (unsigned)ceil_div(rows, (size_t)32) * 32)});
    return launch_pdl(kv_resize_kernel<true, true>, dim3(1), dim3(threads), 0, stream, 1, p);
  }
  const unsigned ctas = (unsigned)std::min<size_t>((size_t)sm_count(), ceil_div(rows, (size_t)kRowsPerCta));
  const dim3 threads(std::max(512u, lane_threads));
  const int rc = launch_pdl(kv_resize_kernel<true, false>, dim3(ctas), threads, 0, stream, 1, p);
  if (rc) return rc;
  return launch_pdl(kv_resize_kernel<false, true>, dim3(1), dim3(std::max(128u, lane_threads)), 0, stream, 1, p);
}

}  // namespace glacier
