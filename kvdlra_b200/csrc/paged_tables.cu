// Page tables, slot map and positions of one step, from the requests' lengths
// (sm_100a).
//
// Request b holds c_b tokens in ceil(c_b / S) pages and gets t_b more.  With
// n_b = ceil((c_b + t_b) / S) - ceil(c_b / S) new pages and P_b = sum_{a<b} n_a,
// its j-th new page is free[count - 1 - (P_b + j)] (the free list is a stack);
// row i of the step belongs to the request with cu_b <= i < cu_{b+1}, cu the
// exclusive prefix sum of t, at position p = c_b + i - cu_b and slot
// table[b][p / S] * S + p % S.  Rows behind the last request get slot -1, and so do,
// with a status bit, rows of a page whose id in the table names none.
//
// A few integers per request and row: latency bounds it, the writes of slots and
// positions where there are a million rows.  A small step is one launch of one
// CTA.  A larger one is two: one CTA scans the requests, then a grid takes the
// rows and the table's new entries; a row's page is looked up in the table or on
// the stack, whichever holds it, so the grid's CTAs need nothing of one another.
#include <algorithm>
#include <climits>

#include "paged.cuh"

namespace kvd {

constexpr int kTabThreads = 1024;
constexpr int kTabMaxBatch = 12288;  // two prefix sums of them in shared memory
constexpr int kPagedNoRoom = 4;      // status bit

struct TableArgs {
  int batch, max_pages, lg_page, num_free, capacity;
  const int* cached;
  const int* added;
  int* table;
  long table_stride;
  const int* free_pages;
  const int* free_count;
  int* lens;        // may be `cached`
  int* free_left;   // may be `free_count`
  int* cu;
  int* slots;
  int* positions;
  int* status;
  int* pages_before;  // [batch + 1], two launches
};

// largest b with pre[b] <= x (pre ascending, pre[0] = 0, x < pre[n])
KVD_DEVICE int find_owner(const int* pre, int n, int x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (pre[mid] <= x) lo = mid; else hi = mid;
  }
  return lo;
}

// The table's new entries and the rows, by `threads` threads, `me` one of them.
// cu and pp (new pages of the requests before) in any memory, cached(b) the tokens
// held, top the free count before the step.
template <typename F>
KVD_DEVICE void table_rows(const TableArgs& a, const int* cu, const int* pp, F cached, int top, int rows, int pages, long me, long threads) {
  const int mask = (1 << a.lg_page) - 1;
  for (long e = me; e < pages; e += threads) {
    const int b = find_owner(pp, a.batch, (int)e);
    const int have = (cached(b) + mask) >> a.lg_page;
    a.table[(long)b * a.table_stride + have + (e - pp[b])] = a.free_pages[top - 1 - e];
  }
  const bool wide = ((reinterpret_cast<uintptr_t>(a.slots) | reinterpret_cast<uintptr_t>(a.positions)) & 15) == 0;
  for (long r0 = 4 * me; r0 < a.capacity; r0 += 4 * threads) {  // four neighbours a thread
    int s[4], q[4];
    int b = r0 < rows ? find_owner(cu, a.batch, (int)r0) : 0;
    int next = r0 < rows ? cu[b + 1] : 0, c_of = -1, c = 0, begin = 0, page_no = -1, id = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = (int)r0 + i;
      s[i] = -1;
      q[i] = 0;
      if (r < rows) {
        while (next <= r) next = cu[++b + 1];
        if (b != c_of) { c_of = b; c = cached(b); begin = cu[b]; page_no = -1; }
        q[i] = c + r - begin;
        const int pn = q[i] >> a.lg_page;
        if (pn != page_no) {
          page_no = pn;
          const int have = (c + mask) >> a.lg_page;
          id = pn < have ? a.table[(long)b * a.table_stride + pn] : a.free_pages[top - 1 - (pp[b] + pn - have)];
          if (id < 0 || id > INT_MAX >> a.lg_page) {  // names no page: its tokens go nowhere
            id = -1;
            if (a.status) atomicOr(a.status + kStatusBounds, kPagedBadPage);
          }
        }
        s[i] = id < 0 ? -1 : (id << a.lg_page) + (q[i] & mask);
      }
    }
    if (wide && r0 + 4 <= a.capacity) {
      *reinterpret_cast<int4*>(a.slots + r0) = make_int4(s[0], s[1], s[2], s[3]);
      *reinterpret_cast<int4*>(a.positions + r0) = make_int4(q[0], q[1], q[2], q[3]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (r0 + i < a.capacity) { a.slots[r0 + i] = s[i]; a.positions[r0 + i] = q[i]; }
    }
  }
}

// The scan, by one CTA; with ALL the rest of the step too.
template <bool ALL>
__global__ void __launch_bounds__(kTabThreads) paged_tables_kernel(const __grid_constant__ TableArgs a) {
  extern __shared__ int tsm[];
  int* cu = tsm;                    // [batch + 1]
  int* pp = tsm + a.batch + 1;      // [batch + 1] new pages of the requests before
  __shared__ long wsum[2][32];
  __shared__ int bad_sm;
  if constexpr (!ALL) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid == 0) bad_sm = 0;
  const int mask = (1 << a.lg_page) - 1;
  const int per = (a.batch + kTabThreads - 1) / kTabThreads;
  const int b0 = min(a.batch, tid * per), b1 = min(a.batch, b0 + per);
  const int free_count = *a.free_count;
  long st = 0, sp = 0;
  bool bad = false;
  for (int b = b0; b < b1; ++b) {
    const int c = a.cached[b], t = a.added[b];
    const long total = (long)c + t;
    if (c < 0 || t < 0 || total > ((long)a.max_pages << a.lg_page)) { bad = true; continue; }
    st += t;
    sp += ((total + mask) >> a.lg_page) - (((long)c + mask) >> a.lg_page);
  }
  long it = st, ip = sp;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long yt = __shfl_up_sync(0xffffffffu, it, o), yp = __shfl_up_sync(0xffffffffu, ip, o);
    if (lane >= o) { it += yt; ip += yp; }
  }
  if (lane == 31) { wsum[0][warp] = it; wsum[1][warp] = ip; }
  __syncthreads();
  long bt = 0, bp = 0, rows = 0, pages = 0;
#pragma unroll 8
  for (int w = 0; w < kTabThreads / 32; ++w) {
    if (w < warp) { bt += wsum[0][w]; bp += wsum[1][w]; }
    rows += wsum[0][w]; pages += wsum[1][w];
  }
  // everything fits, or nothing is done
  if (bad || rows > a.capacity || pages > free_count || free_count > a.num_free) bad_sm = 1;
  __syncthreads();
  const bool ok = bad_sm == 0;
  if (!ok) rows = pages = 0;
  {
    int t = (int)(bt + it - st), p = (int)(bp + ip - sp);
    for (int b = b0; b < b1; ++b) {
      const int c = a.cached[b], n = a.added[b];
      cu[b] = ok ? t : 0;
      pp[b] = ok ? p : 0;
      if (ok) {
        t += n;
        p += ((c + n + mask) >> a.lg_page) - ((c + mask) >> a.lg_page);
      }
    }
    if (tid == 0) { cu[a.batch] = (int)rows; pp[a.batch] = (int)pages; }
  }
  __syncthreads();
  if constexpr (ALL) {
    table_rows(a, cu, pp, [&](int b) { return a.cached[b]; }, free_count, (int)rows, (int)pages, tid, kTabThreads);
    __syncthreads();  // nobody reads the lengths any more
  }
  for (int b = tid; b <= a.batch; b += kTabThreads) {
    a.cu[b] = cu[b];
    if constexpr (!ALL) a.pages_before[b] = pp[b];
    if (b < a.batch) a.lens[b] = a.cached[b] + (ok ? a.added[b] : 0);
  }
  if (tid == 0) {
    *a.free_left = free_count - (int)pages;
    if (!ok && a.status) atomicOr(a.status + kStatusBounds, kPagedNoRoom);
  }
}

// The rest of a large step, after the scan.  What the scan read may be
// overwritten by now: the lengths and the count before the step are those after
// it less what the step added.
__global__ void __launch_bounds__(256) paged_rows_map_kernel(const __grid_constant__ TableArgs a) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int rows = a.cu[a.batch], pages = a.pages_before[a.batch];
  table_rows(a, a.cu, a.pages_before, [&](int b) { return a.lens[b] - a.added[b]; }, *a.free_left + pages, rows, pages,
             (long)blockIdx.x * 256 + threadIdx.x, (long)gridDim.x * 256);
}

// Requests b with done[b] give their ceil(len / S) pages back, in request
// order, on top of the free list, and are empty from then on.  One CTA.
__global__ void __launch_bounds__(kTabThreads)
    paged_release_kernel(int batch, int max_pages, int lg_page, int num_free, const unsigned char* done, int* lens,
                         const int* table, long table_stride, int* free_pages, int* free_count, int* status) {
  extern __shared__ int tsm[];
  int* pp = tsm;  // [batch + 1]
  __shared__ long wsum[32];
  __shared__ int bad_sm;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, mask = (1 << lg_page) - 1;
  const int per = (batch + kTabThreads - 1) / kTabThreads;
  const int b0 = min(batch, tid * per), b1 = min(batch, b0 + per);
  if (tid == 0) bad_sm = 0;
  auto pages_of = [&](int b) -> int {
    if (!done[b]) return 0;
    const int n = lens[b];
    return n < 0 || n > (max_pages << lg_page) ? -1 : (n + mask) >> lg_page;
  };
  long mine = 0;
  bool bad = false;
  for (int b = b0; b < b1; ++b) {
    const int n = pages_of(b);
    if (n < 0) bad = true; else mine += n;
  }
  long incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long y = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += y;
  }
  if (lane == 31) wsum[warp] = incl;
  const int count = *free_count;
  __syncthreads();
  long before = 0, total = 0;
  for (int w = 0; w < kTabThreads / 32; ++w) {
    if (w < warp) before += wsum[w];
    total += wsum[w];
  }
  if (bad || count < 0 || count + total > num_free) bad_sm = 1;
  __syncthreads();
  if (bad_sm) {  // more pages than there are: nothing is done
    if (tid == 0 && status) atomicOr(status + kStatusBounds, kPagedNoRoom);
    return;
  }
  int p = (int)(before + incl - mine);
  for (int b = b0; b < b1; ++b) {
    pp[b] = p;
    p += pages_of(b);
  }
  if (tid == 0) pp[batch] = (int)total;
  __syncthreads();
  for (int e = tid; e < (int)total; e += kTabThreads) {
    const int b = find_owner(pp, batch, e);
    free_pages[count + e] = table[(long)b * table_stride + (e - pp[b])];
  }
  __syncthreads();
  for (int b = b0; b < b1; ++b)
    if (done[b]) lens[b] = 0;
  if (tid == 0) *free_count = count + (int)total;
}

}  // namespace kvd

namespace kvd_host {
using namespace kvd;

static int lg_of(int page) { return page == 16 ? 4 : page == 32 ? 5 : page == 64 ? 6 : page == 128 ? 7 : -1; }

static int table_checks(const char* what, int batch, int max_pages, int64_t stride, int page_size, int num_free) {
  if (lg_of(page_size) < 0) { set_error("%s: page_size %d is none of 16, 32, 64, 128", what, page_size); return KVD_ERR_ARG; }
  if (batch < 1 || batch > kTabMaxBatch) { set_error("%s: batch %d is not in [1, %d]", what, batch, kTabMaxBatch); return KVD_ERR_ARG; }
  if (max_pages < 1 || stride < max_pages || (int64_t)max_pages * page_size > INT32_MAX / 2 || num_free < 0) {
    set_error("%s: table of %d pages a request (stride %lld), %d free pages", what, max_pages, (long long)stride, num_free);
    return KVD_ERR_ARG;
  }
  return KVD_OK;
}

}  // namespace kvd_host

using namespace kvd_host;

extern "C" size_t kvd_page_tables_workspace_bytes(int32_t batch, int32_t capacity) {
  return (long)capacity + batch <= 8192 || batch < 0 ? 0 : (size_t)(batch + 1) * sizeof(int);
}

extern "C" int kvd_page_tables(int32_t batch, int32_t max_pages, int32_t page_size, const int32_t* cached_lens,
                               const int32_t* new_lens, int32_t* table, int64_t table_stride,
                               const int32_t* free_pages, int32_t num_free, const int32_t* free_count, int32_t capacity,
                               int32_t* lens, int32_t* free_left, int32_t* cu_new, int32_t* slots, int32_t* positions,
                               int32_t* status, void* workspace, size_t ws_bytes, kvd_stream_t stream) try {
  if (int rc = table_checks("page tables", batch, max_pages, table_stride, page_size, num_free)) return rc;
  if (capacity < 0 || capacity > INT32_MAX - 8192 * 4) { set_error("page tables: capacity %d", capacity); return KVD_ERR_ARG; }
  if (!cached_lens || !new_lens || !table || (!free_pages && num_free) || !free_count || !lens || !free_left || !cu_new ||
      (capacity && (!slots || !positions))) {
    set_error("page tables: null pointer");
    return KVD_ERR_ARG;
  }
  kvd::TableArgs a{batch, max_pages, lg_of(page_size), num_free, capacity, cached_lens, new_lens, table, (long)table_stride,
                   free_pages, free_count, lens, free_left, cu_new, slots, positions, status, (int*)workspace};
  const size_t smem = 2 * (size_t)(batch + 1) * sizeof(int);
  const cudaStream_t s = (cudaStream_t)stream;
  // One CTA takes 5.4 us for 8 rows (calls in a row, without the host), 5.7 for 4096,
  // 7.4 for 8192 and 10.5 for 16384; the second
  // launch, which spreads them over the SMs, makes it 7.3, 7.7 and 7.8.
  const bool one = (long)capacity + batch <= 8192;
  const void* scan = one ? (const void*)kvd::paged_tables_kernel<true> : (const void*)kvd::paged_tables_kernel<false>;
  // always: the default limit counts the kernel's static memory too
  if (int rc = ensure_smem(scan, smem, "paged_tables_kernel")) return rc;
  if (one) {
    KTimerScope kts_("paged_tables_kernel", s);
    kvd::paged_tables_kernel<true><<<1, kvd::kTabThreads, smem, s>>>(a);
    return check_launch("paged_tables_kernel");
  }
  if (!workspace || ws_bytes < kvd_page_tables_workspace_bytes(batch, capacity)) {
    set_error("page tables: workspace of %zu bytes is needed", kvd_page_tables_workspace_bytes(batch, capacity));
    return KVD_ERR_WORKSPACE;
  }
  {
    KTimerScope kts_("paged_tables_kernel", s);
    kvd::paged_tables_kernel<false><<<1, kvd::kTabThreads, smem, s>>>(a);
  }
  if (int rc = check_launch("paged_tables_kernel")) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)std::max(1L, std::min(4L * paged_sm_count(), ((long)capacity + 1023) / 1024)));
  cfg.blockDim = dim3(256);
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  KTimerScope kts_("paged_rows_map_kernel", s);
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kvd::paged_rows_map_kernel, a);
  if (e != cudaSuccess) { set_error("paged_rows_map_kernel: %s", cudaGetErrorString(e)); return KVD_ERR_CUDA; }
  return KVD_OK;
} catch (...) {
  set_error("page tables: host error");
  return KVD_ERR_CUDA;
}

extern "C" int kvd_page_release(int32_t batch, int32_t max_pages, int32_t page_size, const uint8_t* done, int32_t* lens,
                                const int32_t* table, int64_t table_stride, int32_t* free_pages, int32_t num_free,
                                int32_t* free_count, int32_t* status, kvd_stream_t stream) try {
  if (int rc = table_checks("page release", batch, max_pages, table_stride, page_size, num_free)) return rc;
  if (!done || !lens || !table || !free_pages || !free_count) { set_error("page release: null pointer"); return KVD_ERR_ARG; }
  const size_t smem = (size_t)(batch + 1) * sizeof(int);
  if (int rc = ensure_smem((const void*)kvd::paged_release_kernel, smem, "paged_release_kernel")) return rc;
  KTimerScope kts_("paged_release_kernel", (cudaStream_t)stream);
  kvd::paged_release_kernel<<<1, kvd::kTabThreads, smem, (cudaStream_t)stream>>>(
      batch, max_pages, lg_of(page_size), num_free, done, lens, table, (long)table_stride, free_pages, free_count, status);
  return check_launch("paged_release_kernel");
} catch (...) {
  set_error("page release: host error");
  return KVD_ERR_CUDA;
}
