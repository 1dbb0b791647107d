// The paged cache's book-keeping on the device: block tables and slot maps from
// the requests' lengths, and pages given back.  paged.cuh has the layout.
//
// The free pages are a stack, free[0, n).  With the requests' new pages counted
// through in order of request and page (an exclusive prefix sum over requests),
// the i-th takes free[n - 1 - i].  Giving back puts the i-th of them at free[n + F
// - 1 - i], F their number, so that what a step took and gave back leaves the
// stack as it was.
#include <algorithm>
#include <mutex>
#include <vector>

#include "paged.cuh"

namespace fpb {
namespace {

constexpr int kPageMaxThreads = 1024, kPageMaxBatch = 16384;

struct PageArgs {
  int32_t *table, *lengths, *free, *free_count;
  const int32_t *change;  // new tokens, or new lengths
  long long pitch;        // elements between the table's rows
  int batch, max_pages, pages, page_size;
  int rows, width, vec;  // width: rows a request where they are padded, 0 where they are packed
  int32_t *slots, *positions, *requests, *starts;
  int *error;
};

__device__ __forceinline__ void page_error(const PageArgs &a, int code) {
  if (a.error) atomicCAS(a.error, 0, code);
}

__device__ __forceinline__ int pages_of(int tokens, int page_size) {
  return tokens / page_size + (tokens % page_size != 0);
}

// Sum of the values before this thread's, and of all of them in *total; the
// whole block calls this.
__device__ __forceinline__ long long before(long long v, long long *total, long long *sums) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  long long x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();  // the sums of the call before are read
  if (lane == 31) sums[warp] = x;
  __syncthreads();
  long long s = lane < warps ? sums[lane] : 0;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long y = __shfl_up_sync(0xffffffffu, s, o);
    if (lane >= o) s += y;
  }
  *total = __shfl_sync(0xffffffffu, s, 31);
  const long long mine = __shfl_sync(0xffffffffu, s, warp == 0 ? 0 : warp - 1);
  return x - v + (warp == 0 ? 0 : mine);
}

// The last i in [0, n) with at[i] <= x (at[0] <= x).
__device__ __forceinline__ int last_at(const int *at, int n, int x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (at[mid] <= x)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

// What a launch does of a step: all of it (a block, or a cluster), the rows and pages
// (many blocks), or the state that those have read (one block, behind them).
enum PagePart { kPageAll, kPageRows, kPageState };

// Behind code that lanes may leave apart: the barrier counts whole warps.
__device__ __forceinline__ void cluster_meet() {
  __syncwarp();
  cluster_sync();
}

// Each block scans all requests for itself, then the blocks share the rows and the
// new pages.  A request is served whole (its rows fit, its table and the pool have
// the pages) or not at all.  Bound by latency: two loads, two scans and the pages'
// loads in a row (with page_truncate behind it, 64 requests of a token each 9.7 us,
// 144000 rows of 96 requests, 1.7 MB, 14.5).
template <PagePart PART>
__global__ void __launch_bounds__(kPageMaxThreads) page_extend_kernel(const __grid_constant__ PageArgs a) {
  pdl_enter();
  extern __shared__ int page_sm[];
  int *row0 = page_sm, *off = row0 + a.batch + 1, *len = off + a.batch + 1;  // len -1: not served
  __shared__ long long sums[32];
  __shared__ int used_s;
  const int tid = threadIdx.x, width = blockDim.x;
  if (tid == 0) used_s = 0;
  int free_n = *a.free_count;
  if (free_n < 0 || free_n > a.pages) {
    if (tid == 0) page_error(a, kErrLength);
    free_n = 0;
  }
  const long long most = (long long)a.max_pages * a.page_size;
  long long rows_before = 0, pages_before = 0;
  for (int b0 = 0; b0 < a.batch; b0 += width) {
    const int b = b0 + tid;
    const bool in = b < a.batch;
    const int n = in ? a.lengths[b] : 0, c = in ? a.change[b] : 0;
    const bool bad = n < 0 || c < 0 || n > most;
    if (bad) page_error(a, kErrLength);
    const long long count = max(c, 0);
    long long total, first;
    if (a.width) {
      first = (long long)b * a.width;
      total = 0;
    } else {
      first = rows_before + before(count, &total, sums);
    }
    bool served = in && !bad && n + count <= most && (a.width ? count <= a.width : first + count <= a.rows);
    const long long need = served ? pages_of(n + (int)count, a.page_size) - pages_of(n, a.page_size) : 0;
    long long taken;
    const long long at = pages_before + before(need, &taken, sums);
    served = served && (need == 0 || at + need <= free_n);
    if (served && need > 0) atomicMax(&used_s, (int)(at + need));
    if (in) {
      row0[b] = (int)min(first, (long long)a.rows);
      off[b] = (int)min(at, (long long)free_n);
      len[b] = served ? n : -1;
    }
    rows_before += total;
    pages_before += taken;
  }
  // (a request that is not served for want of pages keeps its place in the sum:
  // those after it that need any are not served either, so the pages used are the
  // stack's first ones)
  if (tid == 0) {
    row0[a.batch] = a.width ? a.rows : (int)min(rows_before, (long long)a.rows);
    off[a.batch] = (int)min(pages_before, (long long)free_n);
  }
  __syncthreads();
  const int used = used_s;
  auto state = [&]() {
    for (int b = tid; b < a.batch; b += width)
      if (len[b] >= 0) a.lengths[b] = len[b] + a.change[b];
    if (a.starts)
      for (int b = tid; b <= a.batch; b += width) a.starts[b] = row0[b];
    if (tid == 0 && used > 0) *a.free_count = free_n - used;
  };
  if (PART == kPageState) return state();
  // (whole numbers without a sign: a step past the last row may pass 2^31)
  const uint32_t threads = gridDim.x * width, me = blockIdx.x * width + tid;
  for (uint32_t i = me; i < (uint32_t)used; i += threads) {
    const int b = last_at(off, a.batch, (int)i);
    const int page = a.free[free_n - 1 - (int)i];
    if (page < 0 || page >= a.pages) page_error(a, kErrPage);
    a.table[b * a.pitch + pages_of(len[b], a.page_size) + (int)i - off[b]] = page;
  }
  // four rows a thread
  for (uint32_t u0 = me * 4; u0 < (uint32_t)a.rows; u0 += threads * 4) {
    const int r0 = (int)u0;
    int slot[4], pos[4], req[4];
    int b = a.width ? r0 / a.width : last_at(row0, a.batch, r0);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int r = r0 + k;
      slot[k] = pos[k] = req[k] = -1;
      if (r >= a.rows) break;
      while (b + 1 < a.batch && row0[b + 1] <= r) ++b;
      const int i = r - row0[b], n = len[b];
      if (n < 0 || i >= (a.width ? a.change[b] : row0[b + 1] - row0[b])) continue;
      const int t = n + i, p = t / a.page_size, held = pages_of(n, a.page_size);
      const int page = p < held ? a.table[b * a.pitch + p] : a.free[free_n - 1 - (off[b] + p - held)];
      pos[k] = t;
      req[k] = b;
      if (page < 0 || page >= a.pages)
        page_error(a, kErrPage);
      else
        slot[k] = page * a.page_size + t - p * a.page_size;
    }
    if (a.vec && r0 + 4 <= a.rows) {
      *reinterpret_cast<int4 *>(a.slots + r0) = make_int4(slot[0], slot[1], slot[2], slot[3]);
      *reinterpret_cast<int4 *>(a.positions + r0) = make_int4(pos[0], pos[1], pos[2], pos[3]);
      if (a.requests) *reinterpret_cast<int4 *>(a.requests + r0) = make_int4(req[0], req[1], req[2], req[3]);
    } else {
      for (int k = 0; k < 4 && r0 + k < a.rows; ++k) {
        a.slots[r0 + k] = slot[k];
        a.positions[r0 + k] = pos[k];
        if (a.requests) a.requests[r0 + k] = req[k];
      }
    }
  }
  if (PART == kPageAll) {
    if (gridDim.x > 1) cluster_meet();  // every block has read the state
    if (blockIdx.x == 0) state();
  }
}

// Likewise.
template <PagePart PART>
__global__ void __launch_bounds__(kPageMaxThreads) page_truncate_kernel(const __grid_constant__ PageArgs a) {
  pdl_enter();
  extern __shared__ int page_sm[];
  int *off = page_sm, *kept = off + a.batch + 1;  // kept: pages that the request keeps
  __shared__ long long sums[32];
  const int tid = threadIdx.x, width = blockDim.x;
  const int free_n = *a.free_count;
  const long long most = (long long)a.max_pages * a.page_size;
  long long back = 0;
  for (int b0 = 0; b0 < a.batch; b0 += width) {
    const int b = b0 + tid;
    const bool in = b < a.batch;
    const int n = in ? a.lengths[b] : 0, to = in ? a.change[b] : -1;
    const bool bad = n < 0 || n > most, cut = !bad && to >= 0 && to < n;
    if (bad) page_error(a, kErrLength);
    const int keeps = cut ? pages_of(to, a.page_size) : 0;
    const long long given = cut ? pages_of(n, a.page_size) - keeps : 0;
    long long total;
    const long long at = back + before(given, &total, sums);
    if (in) {
      off[b] = (int)min(at, (long long)a.pages);
      kept[b] = cut ? keeps : -1;
    }
    back += total;
  }
  if (tid == 0) off[a.batch] = (int)min(back, (long long)a.pages);
  __syncthreads();
  if (free_n < 0 || back > a.pages - free_n) {  // more than the pool can have: nothing is taken back
    if (tid == 0) page_error(a, kErrLength);
    return;
  }
  auto state = [&]() {
    for (int b = tid; b < a.batch; b += width)
      if (kept[b] >= 0) a.lengths[b] = a.change[b];
    if (tid == 0 && back > 0) *a.free_count = free_n + (int)back;
  };
  if (PART == kPageState) return state();
  for (uint32_t u = blockIdx.x * width + tid; u < (uint32_t)back; u += gridDim.x * width) {
    const int i = (int)u, b = last_at(off, a.batch, i);
    int32_t *entry = a.table + b * a.pitch + kept[b] + i - off[b];
    const int page = *entry;
    if (page < 0 || page >= a.pages) page_error(a, kErrPage);
    a.free[free_n + (int)back - 1 - i] = page;
    *entry = -1;
  }
  if (PART == kPageAll) {
    if (gridDim.x > 1) cluster_meet();
    if (blockIdx.x == 0) state();
  }
}

int check_tables(const char *name, const PageArgs &a, size_t table_pitch, size_t batch, size_t max_pages,
                 size_t pages, size_t page_size) {
  if (!a.table || !a.lengths || !a.change || !a.free || !a.free_count)
    return fail(FPB_ERR_INVALID_ARGUMENT, "%s: null pointer", name);
  if (batch == 0 || batch > (size_t)kPageMaxBatch || max_pages == 0 || pages == 0 || page_size == 0 ||
      pages > 0x7fffffffu / page_size || max_pages > 0x7fffffffu / page_size || table_pitch < max_pages ||
      table_pitch >> 38)
    return fail(FPB_ERR_SHAPE, "%s: batch %zu (at most %d), tables of %zu pages (pitch %zu), pool of %zu x %zu rows "
                "(both fewer than 2^31 rows)", name, batch, kPageMaxBatch, max_pages, table_pitch, pages, page_size);
  return FPB_OK;
}

// One block where a step has few rows or pages; else many for those, and one behind
// them for the state (extend and truncate, one block and many: 4096 rows 9.5 and 11.5
// us, 8192 12.4 and 11.4, 144000 120 and 14).  Where it is not known how much of `work`
// there is, as for the pages that a step gives back of all that the requests may hold, a
// cluster takes it up to `cluster` (a truncation of 64 requests of 564 pages, by a cluster
// and by many blocks: one page each 5.4 and 6.1 us, all of them 9.5 and 8.7; of 1024 pages
// 5.4 and 6.1, 12.3 and 8.2: a step gives few back, and the host has a launch less, 2 us;
// rows, which are known, go better by many: 65536 15.7 and 11.7).
int launch_pages(void (*const (&kernel)[3])(PageArgs), const char *name, const PageArgs &a, size_t work,
                 size_t cluster, size_t smem, cudaStream_t s) {
  {
    static std::mutex mu;
    static std::vector<int> done;
    int dev = 0;
    FPB_CUDA_TRY(cudaGetDevice(&dev));
    std::lock_guard<std::mutex> lock(mu);
    if (std::find(done.begin(), done.end(), dev) == done.end()) {
      for (auto k : {page_extend_kernel<kPageAll>, page_extend_kernel<kPageRows>, page_extend_kernel<kPageState>,
                     page_truncate_kernel<kPageAll>, page_truncate_kernel<kPageRows>, page_truncate_kernel<kPageState>})
        FPB_CUDA_TRY(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                          (int)(3 * (kPageMaxBatch + 1) * sizeof(int))));
      done.push_back(dev);
    }
  }
  auto launch = [&](PagePart part, unsigned blocks, unsigned threads) {
    cudaError_t e = part == kPageAll && blocks > 1 ? launch_pdl_cluster(kernel[part], blocks, threads, smem, s, blocks, a)
                                                   : launch_pdl(kernel[part], blocks, threads, smem, s, a);
    if (e != cudaSuccess) return cuda_fail(e, name);
    FPB_LAUNCH_CHECK(name);
    return (int)FPB_OK;
  };
  // (a wide block's barriers take longer, a narrow one goes through its work more often)
  const unsigned scan = a.batch <= 256 ? 256 : kPageMaxThreads;
  if (work <= 6144) return launch(kPageAll, 1, work <= 1024 ? scan : kPageMaxThreads);
  if (work <= cluster) return launch(kPageAll, 8, kPageMaxThreads);
  const size_t blocks = std::min<size_t>((work + 4 * scan - 1) / (4 * scan), 2 * sm_count());
  if (int st = launch(kPageRows, (unsigned)blocks, scan)) return st;
  return launch(kPageState, 1, scan);
}

PageArgs page_args(int32_t *table, size_t table_pitch, size_t batch, size_t max_pages, int32_t *lengths,
                   const int32_t *change, int32_t *free_pages, int32_t *free_count, size_t pages, size_t page_size) {
  PageArgs a{};
  a.table = table;
  a.pitch = (long long)table_pitch;
  a.batch = (int)batch;
  a.max_pages = (int)max_pages;
  a.lengths = lengths;
  a.change = change;
  a.free = free_pages;
  a.free_count = free_count;
  a.pages = (int)pages;
  a.page_size = (int)page_size;
  return a;
}

}  // namespace
}  // namespace fpb

using namespace fpb;

extern "C" int fpb_page_extend(int32_t *table, size_t table_pitch, size_t batch, size_t max_pages, int32_t *lengths,
                               const int32_t *counts, int32_t *free_pages, int32_t *free_count, size_t pages,
                               size_t page_size, size_t rows, int padded, int32_t *slots, int32_t *positions,
                               int32_t *requests, int32_t *starts, void *stream) {
  PageArgs a = page_args(table, table_pitch, batch, max_pages, lengths, counts, free_pages, free_count, pages,
                         page_size);
  if (int st = check_tables("fpb_page_extend", a, table_pitch, batch, max_pages, pages, page_size)) return st;
  if (!slots || !positions) return fail(FPB_ERR_INVALID_ARGUMENT, "fpb_page_extend: null pointer");
  if (rows == 0 || rows > FPB_PAGE_MAX_ROWS || (padded && rows % batch))
    return fail(FPB_ERR_SHAPE, "fpb_page_extend: %zu rows (padded: a multiple of the batch, %zu)", rows, batch);
  if (counts < lengths + batch && lengths < counts + batch)  // (a block reads counts behind another's lengths)
    return fail(FPB_ERR_INVALID_ARGUMENT, "fpb_page_extend: counts overlap the lengths");
  a.rows = (int)rows;
  a.width = padded ? (int)(rows / batch) : 0;
  a.slots = slots;
  a.positions = positions;
  a.requests = requests;
  a.starts = starts;
  a.vec = aligned_to(slots, 16) && aligned_to(positions, 16) && aligned_to(requests, 16);
  a.error = device_error_ptr();
  return launch_pages({page_extend_kernel<kPageAll>, page_extend_kernel<kPageRows>, page_extend_kernel<kPageState>},
                      "page_extend_kernel", a, rows, 0, 3 * (batch + 1) * sizeof(int), as_stream(stream));
}

extern "C" int fpb_page_truncate(int32_t *table, size_t table_pitch, size_t batch, size_t max_pages, int32_t *lengths,
                                 const int32_t *new_lengths, int32_t *free_pages, int32_t *free_count, size_t pages,
                                 size_t page_size, void *stream) {
  PageArgs a = page_args(table, table_pitch, batch, max_pages, lengths, new_lengths, free_pages, free_count, pages,
                         page_size);
  if (int st = check_tables("fpb_page_truncate", a, table_pitch, batch, max_pages, pages, page_size)) return st;
  // (read again where lengths are written; the lengths themselves change nothing)
  if (new_lengths != lengths && new_lengths < lengths + batch && lengths < new_lengths + batch)
    return fail(FPB_ERR_INVALID_ARGUMENT, "fpb_page_truncate: new_lengths overlap the lengths");
  a.error = device_error_ptr();
  return launch_pages({page_truncate_kernel<kPageAll>, page_truncate_kernel<kPageRows>, page_truncate_kernel<kPageState>},
                      "page_truncate_kernel", a, std::min(batch * max_pages, pages), 65536,
                      2 * (batch + 1) * sizeof(int),
                      as_stream(stream));
}
