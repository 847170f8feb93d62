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

// Inclusive sums over the block's threads of N values each, and their totals.  Each warp scans its
// own, then every warp scans the warps' sums for itself: one barrier.  `sh` is used once.
template <int N, typename T>
__device__ __forceinline__ void block_scan(T (&v)[N], T (&total)[N], T (*sh)[32]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
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
  __syncthreads();
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

// Every CTA works the whole batch out for itself (a thread per lane, two block scans): that
// takes less time than passing results on.  The stack's order is arithmetic: pages that shrinking
// lanes give back lie above the old top so that the next pops return them in lane and page order
// (growing again undoes the shrink), and growing lanes pop in lane order.  A page that is
// given back and taken in one call is therefore found in the table it comes from, and nothing waits
// for another thread's writes.  Once the pages or rows run out, that lane and every later one that
// needs any is refused and left as it was.  No atomics: the result depends on the inputs alone.
//
// MOVE writes rows and pages: nothing in it reads what it writes (rows read the pages that a lane
// held before, pages given back go above the old top).  STATE sets lengths, count and statuses,
// which everything reads.  Few rows: one CTA does both.  Many: a grid of MOVE CTAs, then a STATE CTA
// behind it.
template <bool MOVE, bool STATE>
__global__ void __launch_bounds__(kMaxLanes, 1) kv_resize_kernel(const ResizeParams p) {
  __shared__ long long sh_want[3][32];
  __shared__ int sh_got[2][32];
  __shared__ int s_old[kMaxLanes], s_first[kMaxLanes], s_give[kMaxLanes], s_new[kMaxLanes];
  __shared__ int s_off[kMaxLanes + 1];  // packed: each lane's first row; padded: its number of rows, one further on
  griddep_launch();
  griddep_wait();
  const int tid = threadIdx.x;
  const bool lane_on = tid < p.lanes;
  const int old_len = lane_on ? p.lens[tid] : 0, target = lane_on ? p.targets[tid] : 0;
  const int count = min(max(*p.free_count, 0), p.capacity);
  const int limit = p.max_pages * kQ4Page;
  const bool valid = lane_on && old_len >= 0 && old_len <= limit && target >= 0 && target <= limit &&
                     (p.row_stride == 0 || target - old_len <= p.row_stride);
  const int have = valid ? (old_len + kQ4Page - 1) / kQ4Page : 0, want = valid ? (target + kQ4Page - 1) / kQ4Page : 0;
  const int give = max(have - want, 0), need = max(want - have, 0), grow = valid ? max(target - old_len, 0) : 0;

  long long want_sum[3] = {give, need, grow}, want_all[3];
  block_scan(want_sum, want_all, sh_want);
  const int give_sum = (int)want_sum[0], need_sum = (int)want_sum[1];
  const int given = (int)want_all[0], avail = (int)min((long long)count + given, (long long)p.capacity);
  const bool rows_fit = p.row_stride != 0 || want_sum[2] <= (p.slots ? p.rows : (long long)INT32_MAX);
  const bool ok = valid && (need == 0 || need_sum <= avail) && (grow == 0 || rows_fit);
  int got[2] = {ok ? grow : 0, ok ? need : 0}, got_all[2];
  block_scan(got, got_all, sh_got);
  s_old[tid] = old_len;
  s_new[tid] = ok ? target : -1;
  s_first[tid] = need_sum - need;
  s_give[tid] = give_sum - give;
  s_off[tid + 1] = p.row_stride ? (ok ? grow : 0) : got[0];
  if (tid == 0) s_off[0] = 0;
  __syncthreads();
  // Entry `at` of the stack after the shrinking lanes gave their pages back.
  auto stack = [&](int at) {
    if (at < count) return p.free_pages[at];
    const int j = count + given - 1 - at, b = holder(s_give, p.lanes, j);
    return p.tables[(size_t)b * p.max_pages + (s_new[b] + kQ4Page - 1) / kQ4Page + j - s_give[b]];
  };
  auto fresh_page = [&](int b, int k, int h) { return stack(avail - 1 - (s_first[b] + k - h)); };

  if constexpr (MOVE) {
    // Four rows per thread: one search, then the lanes in order.
    const bool vec = (((uintptr_t)p.positions | (uintptr_t)p.row_lanes | (uintptr_t)p.slots) & 15) == 0;
    const int n = p.slots ? (int)p.rows : 0, live_end = s_off[p.lanes];
    for (long long r0 = 4 * ((long long)blockIdx.x * blockDim.x + tid); r0 < n; r0 += 4ll * gridDim.x * blockDim.x) {
      int pos[4], who[4];
      long long slot[4];
      int b = p.row_stride ? (int)r0 / p.row_stride : holder(s_off, p.lanes, (int)r0);
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int r = (int)r0 + c;
        int i;
        bool live;
        if (p.row_stride) {
          if (r >= (b + 1) * p.row_stride) ++b;
          i = r - b * p.row_stride;
          live = b < p.lanes && i < s_off[b + 1];
        } else {
          live = r < live_end;
          while (live && r >= s_off[b + 1]) ++b;
          i = r - s_off[b];
        }
        pos[c] = who[c] = -1;
        slot[c] = -1;
        if (live) {
          pos[c] = s_old[b] + i;
          who[c] = b;
          const int k = pos[c] / kQ4Page, h = (s_old[b] + kQ4Page - 1) / kQ4Page;
          const int page = k < h ? p.tables[(size_t)b * p.max_pages + k] : fresh_page(b, k, h);
          slot[c] = (long long)page * kQ4Page + (pos[c] & (kQ4Page - 1));
        }
      }
      if (vec && r0 + 4 <= n) {
        *reinterpret_cast<int4*>(p.positions + r0) = make_int4(pos[0], pos[1], pos[2], pos[3]);
        *reinterpret_cast<int4*>(p.row_lanes + r0) = make_int4(who[0], who[1], who[2], who[3]);
        *reinterpret_cast<longlong2*>(p.slots + r0) = make_longlong2(slot[0], slot[1]);
        *reinterpret_cast<longlong2*>(p.slots + r0 + 2) = make_longlong2(slot[2], slot[3]);
      } else {
        for (int c = 0; c < 4 && r0 + c < n; ++c) {
          p.positions[r0 + c] = pos[c];
          p.row_lanes[r0 + c] = who[c];
          p.slots[r0 + c] = slot[c];
        }
      }
    }
  }
  if constexpr (MOVE) {
    // Pages given back and taken, laid end to end: four per thread and search, loads before stores.
    // The block's last threads begin, beside the first ones' rows.
    const int moves = given + got_all[1];
    for (long long i0 = 4 * ((long long)blockIdx.x * blockDim.x + blockDim.x - 1 - tid); i0 < moves; i0 += 4ll * gridDim.x * blockDim.x) {
      int32_t *dst[4], page[4];
      int b = 0;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int i = (int)i0 + c;
        dst[c] = nullptr;
        if (i >= moves) continue;
        const bool back = i < given;
        const int* first = back ? s_give : s_first;
        const int j = back ? i : i - given;
        if (c == 0 || j == 0) b = holder(first, p.lanes, j);
        while (b + 1 < p.lanes && first[b + 1] <= j) ++b;
        const int h = (s_old[b] + kQ4Page - 1) / kQ4Page, w = (s_new[b] + kQ4Page - 1) / kQ4Page;
        int32_t* table = p.tables + (size_t)b * p.max_pages;
        if (back) {
          const int at = count + given - 1 - j;
          if (at < p.capacity) dst[c] = p.free_pages + at;  // more pages than the stack holds are dropped
          page[c] = table[w + j - s_give[b]];
        } else {
          dst[c] = table + h + j - s_first[b];
          page[c] = stack(avail - 1 - j);
        }
      }
#pragma unroll
      for (int c = 0; c < 4; ++c)
        if (dst[c]) *dst[c] = page[c];
    }
  }
  if constexpr (STATE) {
    if (ok) p.lens[tid] = target;
    if (lane_on) p.status[tid] = ok ? GLACIER_CUDA_OK : valid ? GLACIER_CUDA_ENOMEM : GLACIER_CUDA_EINVAL;
    if (tid == 0) *p.free_count = avail - got_all[1];
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
  // One CTA's threads at four rows each: from there on a second launch pays (64 lanes grown from
  // nothing and released again: 8.4 us in one CTA against 10.0 in two launches at 2048 rows, 10.0 and 9.9
  // at 4096, 12.8 and 10.0 at 8192, 48 and 12.5 at 65536).
  if (rows <= 4 * kMaxLanes) {
    const unsigned threads = std::max({128u, lane_threads, std::min(1024u, (unsigned)ceil_div(rows, (size_t)128) * 32)});
    return launch_pdl(kv_resize_kernel<true, true>, dim3(1), dim3(threads), 0, stream, 1, p);
  }
  const unsigned ctas = (unsigned)std::min<size_t>((size_t)sm_count(), ceil_div(rows, (size_t)kRowsPerCta));
  const int rc = launch_pdl(kv_resize_kernel<true, false>, dim3(ctas), dim3(std::max(512u, lane_threads)), 0, stream, 1, p);
  if (rc) return rc;
  return launch_pdl(kv_resize_kernel<false, true>, dim3(1), dim3(std::max(128u, lane_threads)), 0, stream, 1, p);
}

}  // namespace glacier
