// Block tables and slot maps on the device, from request lengths: the page
// bookkeeping of PagedKVCache (src/paged_kv_cache.zig:44-48 request page tables,
// :1074 appendRowTxn's page of a position) for all lanes of a batch in one launch.
#include "kv_q4.cuh"

namespace glacier {

namespace {

constexpr int kResizeThreads = 1024;  // one lane per thread
constexpr int kResizeCtas = 8;        // CTAs of the cluster that serves many rows

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

// Inclusive sum over the block's threads (one value each), in `sh` of 32 words.
__device__ __forceinline__ long long block_scan(long long v, long long* sh) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long t = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += t;
  }
  __syncthreads();
  if (lane == 31) sh[warp] = v;
  __syncthreads();
  if (warp == 0) {
    long long w = sh[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long t = __shfl_up_sync(0xffffffffu, w, o);
      if (lane >= o) w += t;
    }
    sh[lane] = w;
  }
  __syncthreads();
  return warp ? v + sh[warp - 1] : v;
}

// Every CTA of the cluster scans all lanes (at most 1024, one per thread) for itself:
// that is cheaper than passing the sums around.  Then the cluster shares the work:
//   1. pages that shrinking lanes give back go on the stack so that the next pops
//      return them in lane and page order (growing again undoes the shrink);
//   2. cluster barrier: the stack is whole, and nobody reads the old lengths or the
//      old count any more;
//   3. growing lanes take pages off the top in lane order; rows get positions and
//      slots, the page of a new position read from the stack itself, so no CTA waits
//      for another's table writes; rank 0 stores lengths, count, statuses, offsets.
// Lanes are served in order; once the pages or rows run out, that lane and every later
// one that needs any is refused and left as it was.  No atomics: the result depends
// on the inputs alone.
__global__ void __launch_bounds__(kResizeThreads, 1) kv_resize_kernel(const ResizeParams p) {
  __shared__ long long sh[32];
  __shared__ int s_old[kResizeThreads], s_first[kResizeThreads];
  __shared__ int s_off[kResizeThreads + 1];
  griddep_launch();
  griddep_wait();
  const int tid = threadIdx.x;
  const int cr = (int)cluster_ctarank(), cn = (int)cluster_nctarank();
  const bool lane_on = tid < p.lanes;
  const int old_len = lane_on ? p.lens[tid] : 0, target = lane_on ? p.targets[tid] : 0;
  const int count = min(max(*p.free_count, 0), p.capacity);
  const long long limit = (long long)p.max_pages * kQ4Page;
  const bool valid = lane_on && old_len >= 0 && old_len <= limit && target >= 0 && target <= limit &&
                     (p.row_stride == 0 || target - old_len <= p.row_stride);
  const int have = (int)(((long long)old_len + kQ4Page - 1) / kQ4Page);
  const int want = (int)(((long long)target + kQ4Page - 1) / kQ4Page);
  const long long give = valid && want < have ? have - want : 0;
  const long long need = valid && want > have ? want - have : 0;
  const long long grow = valid && target > old_len ? target - old_len : 0;

  const long long give_incl = block_scan(give, sh);
  const long long given = sh[31];
  const long long need_incl = block_scan(need, sh);
  const long long rows_incl = block_scan(grow, sh);
  // The stack holds `capacity` entries: pages beyond it cannot come back (a table that
  // lists more pages than the pool has), and are dropped.
  const long long avail = min(count + given, (long long)p.capacity);
  const bool rows_fit = p.row_stride != 0 || rows_incl <= (p.slots ? p.rows : (long long)INT32_MAX);
  const bool ok = valid && (need == 0 || need_incl <= avail) && (grow == 0 || rows_fit);
  const long long got = ok ? grow : 0;
  const long long got_incl = block_scan(got, sh);
  block_scan(ok ? need : 0, sh);
  const long long taken = sh[31];
  s_old[tid] = old_len;
  s_first[tid] = (int)(need_incl - need);
  if (tid == 0) s_off[0] = 0;
  // Row bookkeeping: packed lanes follow one another; padded ones keep their count.
  s_off[tid + 1] = p.row_stride ? (int)got : (int)got_incl;
  __syncthreads();

  // 1. pages given back, in lane and page order from the new top downwards
  __shared__ int s_give[kResizeThreads], s_ok[kResizeThreads];
  s_give[tid] = (int)(give_incl - give);
  s_ok[tid] = ok ? target : (valid ? -2 : -1);
  __syncthreads();
  if (given > 0) {
    const int warp = tid >> 5, lane = tid & 31;
    for (int b = cr * (kResizeThreads / 32) + warp; b < p.lanes; b += cn * (kResizeThreads / 32)) {
      const int t = s_ok[b];
      if (t < 0) continue;
      const int h = (s_old[b] + kQ4Page - 1) / kQ4Page, w = (t + kQ4Page - 1) / kQ4Page;
      for (int j = w + lane; j < h; j += 32) {
        const long long at = count + given - 1 - (s_give[b] + j - w);
        if (at < p.capacity) p.free_pages[at] = p.tables[(size_t)b * p.max_pages + j];
      }
    }
  }
  // 2.
  if (cn > 1) cluster_sync_all(); else __syncthreads();
  // 3.
  if (cr == 0) {
    if (ok) p.lens[tid] = target;
    if (lane_on) p.status[tid] = ok ? GLACIER_CUDA_OK : valid ? GLACIER_CUDA_ENOMEM : GLACIER_CUDA_EINVAL;
    if (tid == 0) *p.free_count = (int32_t)(avail - taken);
    if (p.row_offsets)
      for (int i = tid; i <= p.lanes; i += kResizeThreads)
        p.row_offsets[i] = p.row_stride ? i * p.row_stride : s_off[i];
  }
  auto fresh_page = [&](int b, int k, int h) {  // k-th page of lane b, k >= h pages held
    return p.free_pages[avail - 1 - (s_first[b] + k - h)];
  };
  {
    const int warp = tid >> 5, lane = tid & 31;
    for (int b = cr * (kResizeThreads / 32) + warp; b < p.lanes; b += cn * (kResizeThreads / 32)) {
      const int t = s_ok[b];
      if (t < 0) continue;
      const int h = (s_old[b] + kQ4Page - 1) / kQ4Page, w = (t + kQ4Page - 1) / kQ4Page;
      for (int j = h + lane; j < w; j += 32) p.tables[(size_t)b * p.max_pages + j] = fresh_page(b, j, h);
    }
  }
  if (!p.slots) return;
  for (long long r = (long long)cr * kResizeThreads + tid; r < p.rows; r += (long long)cn * kResizeThreads) {
    int b, i;
    bool live;
    if (p.row_stride) {
      b = (int)(r / p.row_stride);
      i = (int)(r - (long long)b * p.row_stride);
      live = b < p.lanes && i < s_off[b + 1];
    } else {
      live = r < s_off[p.lanes];
      int lo = 0, hi = p.lanes - 1;
      while (lo < hi) {  // the lane whose rows hold r: last b with offset <= r
        const int mid = (lo + hi + 1) >> 1;
        if (s_off[mid] <= r) lo = mid; else hi = mid - 1;
      }
      b = lo;
      i = (int)(r - s_off[b]);
    }
    int pos = -1;
    int64_t slot = -1;
    if (live) {
      pos = s_old[b] + i;
      const int k = pos / kQ4Page, h = (s_old[b] + kQ4Page - 1) / kQ4Page;
      const int page = k < h ? p.tables[(size_t)b * p.max_pages + k] : fresh_page(b, k, h);
      slot = (int64_t)page * kQ4Page + (pos & (kQ4Page - 1));
    }
    p.positions[r] = pos;
    p.row_lanes[r] = live ? b : -1;
    p.slots[r] = slot;
  }
}

}  // namespace

int kv_resize(int32_t* lens, const int32_t* targets, size_t lanes, int32_t* block_tables, size_t max_pages,
              int32_t* free_pages, size_t capacity, int32_t* free_count, int32_t* status, size_t row_stride,
              size_t rows, int32_t* positions, int32_t* row_lanes, int64_t* slots, int32_t* row_offsets,
              cudaStream_t stream) {
  GLC_REQUIRE(lens && targets && block_tables && free_pages && free_count && status, "kv_resize: null argument");
  GLC_REQUIRE(lens != targets, "kv_resize: lens and targets are the same array");
  GLC_REQUIRE(lanes > 0 && lanes <= (size_t)kResizeThreads, "kv_resize: %zu lanes (1 to %d)", lanes, kResizeThreads);
  GLC_REQUIRE(max_pages > 0 && max_pages <= ((size_t)1 << 26) && capacity > 0 && capacity < ((size_t)1 << 31),
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
  const int ctas = rows > 4096 ? kResizeCtas : 1;
  return launch_pdl(kv_resize_kernel, dim3((unsigned)ctas), dim3(kResizeThreads), 0, stream, ctas, p);
}

}  // namespace glacier
