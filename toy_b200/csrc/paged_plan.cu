// Page accounting of a paged KV cache on the GPU: the pages a step's new
// tokens need, the block-table entries, the slot map, and the return of
// finished requests' pages.
//
// With P tokens to a page, request b of length l_b that appends a_b tokens
// needs n_b = ceil((l_b + a_b) / P) - ceil(l_b / P) pages. Exclusive prefix
// sums over the requests, T_b of a and N_b of n, number the new tokens and the
// new pages: page i of the step is free_pages[count - 1 - i], entry
// ceil(l_b / P) + (i - N_b) of the request b with N_b <= i < N_{b+1}; token t
// is position l_b + (t - T_b) of the request b with T_b <= t < T_{b+1}. So
// once the sums are known, tokens and pages are two flat index spaces that any
// thread can fill without hearing from another.
//
// The work is small (16 bytes written per token) and bound by latency: one
// launch, in which every CTA computes the whole prefix sums for itself in
// shared memory (n_req <= 16384; each length is read once) and fills its slice of
// tokens and pages, instead of a scan, a barrier over the grid and a fill.
// Lengths and the stack's count may be updated in place: a single CTA writes
// them after its own reads; a larger grid leaves that to a second, tiny
// kernel. Measured on one B200: 5.0 us for 16 requests, 8.4 us for 524288 slots
// of 1024 requests (8.4 MB written). The return of pages is filled the same
// way: 3.5 us for 16 requests, 6.9 us for 33000 pages of 1024.
#include <algorithm>

#include "paged.cuh"
#include "pdl.cuh"
#include "runtime.cuh"

namespace tb2 {
namespace {

constexpr int kMaxReq = 16384;
constexpr int kThreads = 1024;
constexpr int kRun = 4;   // consecutive tokens of a thread

// The totals of a scan: tokens and pages of every request, and whether any
// input was bad (codes as the C API documents them).
struct Totals {
  long long tokens, pages;
  int bad;
};

__device__ __forceinline__ int div_up(int a, int b) { return (int)(((long long)a + b - 1) / b); }

// Exclusive prefix sums of two values per request into st[0 .. n] and
// sp[0 .. n]: the caller has put the values themselves there and synchronised.
// Sums are 64 bits wide and stored cut to 32; totals that do not fit are
// reported by the caller's own limits before the stored values are used. `bad`
// is this thread's; the result's is the CTA's largest.
__device__ Totals scan_requests(int n, int* st, int* sp, int bad) {
  __shared__ long long wt[32], wp[32];
  __shared__ int wb[32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, nw = blockDim.x >> 5;
  const int per = (n + (int)blockDim.x - 1) / (int)blockDim.x;
  const int b0 = min(n, tid * per), b1 = min(n, b0 + per);
  long long ts = 0, ps = 0;
  for (int b = b0; b < b1; ++b) {
    ts += st[b];
    ps += sp[b];
  }
  long long ti = ts, pi = ps;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long a = __shfl_up_sync(0xffffffffu, ti, o), c = __shfl_up_sync(0xffffffffu, pi, o);
    if (lane >= o) {
      ti += a;
      pi += c;
    }
  }
  bad = __reduce_max_sync(0xffffffffu, bad);
  if (lane == 31) {
    wt[warp] = ti;
    wp[warp] = pi;
    wb[warp] = bad;
  }
  __syncthreads();
  // the warps' totals, scanned by every warp for itself
  long long at = lane < nw ? wt[lane] : 0, ap = lane < nw ? wp[lane] : 0;
  bad = __reduce_max_sync(0xffffffffu, lane < nw ? wb[lane] : 0);
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long a = __shfl_up_sync(0xffffffffu, at, o), c = __shfl_up_sync(0xffffffffu, ap, o);
    if (lane >= o) {
      at += a;
      ap += c;
    }
  }
  const long long tt = __shfl_sync(0xffffffffu, at, 31), tp = __shfl_sync(0xffffffffu, ap, 31);
  long long bt = __shfl_sync(0xffffffffu, at, max(0, warp - 1)), bp = __shfl_sync(0xffffffffu, ap, max(0, warp - 1));
  if (warp == 0) bt = bp = 0;
  bt += ti - ts;
  bp += pi - ps;
  for (int b = b0; b < b1; ++b) {
    const int tok = st[b], pg = sp[b];
    st[b] = (int)bt;
    sp[b] = (int)bp;
    bt += tok;
    bp += pg;
  }
  if (tid == 0) {
    st[n] = (int)tt;
    sp[n] = (int)tp;
  }
  __syncthreads();
  return {tt, tp, bad};
}

// The request b with cu[b] <= i < cu[b + 1].
__device__ __forceinline__ int find_request(const int* cu, int n, int i) {
  int lo = 0, hi = n;   // cu[lo] <= i < cu[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (cu[mid] <= i) lo = mid;
    else hi = mid;
  }
  return lo;
}

// Four values from element i on, one 16-byte store where the address allows it.
__device__ __forceinline__ void store4(int* p, int i, int n, const int (&v)[kRun]) {
  if (i + kRun <= n && (reinterpret_cast<uintptr_t>(p + i) & 15) == 0) {
    *reinterpret_cast<int4*>(p + i) = make_int4(v[0], v[1], v[2], v[3]);
  } else {
#pragma unroll
    for (int k = 0; k < kRun; ++k)
      if (i + k < n) p[i + k] = v[k];
  }
}
__device__ __forceinline__ void store4(long long* p, int i, int n, const long long (&v)[kRun]) {
  if (i + kRun <= n && (reinterpret_cast<uintptr_t>(p + i) & 15) == 0) {
    *reinterpret_cast<longlong2*>(p + i) = make_longlong2(v[0], v[1]);
    *reinterpret_cast<longlong2*>(p + i + 2) = make_longlong2(v[2], v[3]);
  } else {
#pragma unroll
    for (int k = 0; k < kRun; ++k)
      if (i + k < n) p[i + k] = v[k];
  }
}

__global__ void __launch_bounds__(kThreads) paged_plan_kernel(const tb2_paged_plan_args a, int in_place, int* err) {
  extern __shared__ int sm[];
  const int P = a.page_size, n = a.n_req;
  int* cu_tok = sm;
  int* cu_pg = sm + n + 1;
  int* held = cu_pg + n + 1;   // the lengths
  griddep_wait_release();
  const int count = a.state[0];
  int bad = 0;
  for (int b = threadIdx.x; b < n; b += blockDim.x) {
    const int len = a.lens[b], add = a.add[b];
    const long long end = (long long)len + add;
    int tok = 0, pg = 0;
    if (len < 0 || add < 0) {
      bad = 4;
    } else if (end > (long long)a.table_width * P) {
      bad = max(bad, 2);
    } else {
      tok = add;
      pg = div_up((int)end, P) - div_up(len, P);
    }
    cu_tok[b] = tok;
    cu_pg[b] = pg;
    held[b] = len;
  }
  __syncthreads();
  const Totals tot = scan_requests(n, cu_tok, cu_pg, bad);
  int status = tot.bad;
  if (count < 0 || count > a.n_free) status = 4;
  else if (!status && tot.tokens > a.n_tokens) status = 3;
  else if (!status && tot.pages > count) status = 1;
  const int tokens = status ? 0 : (int)tot.tokens, pages = status ? 0 : (int)tot.pages;
  const int step = gridDim.x * blockDim.x, first = blockIdx.x * blockDim.x + threadIdx.x;
  for (int i = first; i < pages; i += step) {
    const int page = a.free_pages[count - 1 - i], b = find_request(cu_pg, n, i);
    a.table[b * a.table_stride + div_up(held[b], P) + (i - cu_pg[b])] = page;
  }
  for (long long t0 = (long long)first * kRun; t0 < a.n_tokens; t0 += (long long)step * kRun) {
    long long slot[kRun];
    int pos[kRun], req[kRun];
    int b = t0 < tokens ? find_request(cu_tok, n, (int)t0) : -1, blk = -1, page = 0;
#pragma unroll
    for (int k = 0; k < kRun; ++k) {
      slot[k] = req[k] = -1;
      pos[k] = 0;
      const int t = (int)t0 + k;
      if (t >= tokens) continue;
      while (t >= cu_tok[b + 1]) {   // the next request with a token
        ++b;
        blk = -1;
      }
      req[k] = b;
      pos[k] = held[b] + (t - cu_tok[b]);
      const int at = pos[k] / P;
      if (at != blk) {
        blk = at;
        const int old = div_up(held[b], P);
        page = at < old ? a.table[b * a.table_stride + at] : a.free_pages[count - 1 - (cu_pg[b] + at - old)];
      }
      if (page >= 0 && page < a.n_pages) slot[k] = (long long)page * P + (pos[k] - at * P);
      else *err = kErrPagedPage;
    }
    store4(a.slots, (int)t0, a.n_tokens, slot);
    store4(a.positions, (int)t0, a.n_tokens, pos);
    store4(a.requests, (int)t0, a.n_tokens, req);
  }
  if (blockIdx.x == 0)
    for (int b = threadIdx.x; b <= n; b += blockDim.x) a.cu_tokens[b] = status ? 0 : cu_tok[b];
  // lengths and count: by this kernel unless another CTA may still have to read what they overwrite
  const bool alone = gridDim.x == 1;
  if (alone) __syncthreads();
  if (blockIdx.x == 0 && (alone || !in_place)) {
    for (int b = threadIdx.x; b < n; b += blockDim.x)
      a.lens_out[b] = status ? held[b] : held[b] + (cu_tok[b + 1] - cu_tok[b]);
    if (threadIdx.x == 0) a.state_out[0] = count - pages;
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    a.state_out[1] = status;
    a.state_out[2] = tokens;
    a.state_out[3] = pages;
  }
}

// After a plan in place on more than one CTA: the lengths and the stack's count.
__global__ void paged_plan_commit_kernel(const tb2_paged_plan_args a) {
  griddep_wait_release();
  const int b = blockIdx.x * blockDim.x + threadIdx.x;
  if (b < a.n_req) a.lens_out[b] = a.lens[b] + (a.state_out[1] ? 0 : a.add[b]);
  if (b == 0) a.state_out[0] = a.state[0] - a.state_out[3];
}

// Takes the entries below 0 out of x[0 .. n), in place and in order, by one
// CTA; returns how many are left.
__device__ int drop_negative(int* x, int n) {
  __shared__ int wc[32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, nw = blockDim.x >> 5;
  int kept = 0;
  for (int i0 = 0; i0 < n; i0 += blockDim.x) {
    const int i = i0 + tid, v = i < n ? x[i] : -1;
    const unsigned on = __ballot_sync(0xffffffffu, v >= 0);
    if (lane == 0) wc[warp] = __popc(on);
    __syncthreads();   // (and every entry of the round is read)
    int at = kept, round = 0;
    for (int w = 0; w < nw; ++w) {
      if (w < warp) at += wc[w];
      round += wc[w];
    }
    if (v >= 0) x[at + __popc(on & ((1u << lane) - 1))] = v;
    kept += round;
    __syncthreads();   // the counts are read
  }
  return kept;
}

// Pages go on the stack in the order of their numbers; an entry that is no page
// goes there as -1 and is taken out again (rarely: it is an error), by this
// kernel's only CTA or, counted in state_out[2], by the commit kernel.
__global__ void __launch_bounds__(kThreads) paged_release_kernel(const tb2_paged_release_args a, int* err) {
  extern __shared__ int sm[];
  __shared__ int none;   // entries that are no page, of a single CTA
  const int P = a.page_size, n = a.n_req;
  int* gone = sm;   // requests that are done, counted like tokens
  int* cu_pg = sm + n + 1;
  griddep_wait_release();
  if (threadIdx.x == 0) none = 0;
  const int count = a.state[0];
  int bad = 0;
  for (int b = threadIdx.x; b < n; b += blockDim.x) {
    const int len = a.lens[b];
    const bool fits = len >= 0 && len <= (long long)a.table_width * P, done = a.done[b] != 0;
    if (!fits) bad = 4;
    gone[b] = fits && done;
    cu_pg[b] = fits && done ? div_up(len, P) : 0;
  }
  __syncthreads();
  const Totals tot = scan_requests(n, gone, cu_pg, bad);
  int status = tot.bad;
  if (count < 0 || count > a.n_free) status = 4;
  else if (!status && tot.pages > a.n_free - count) status = 1;
  int pages = status ? 0 : (int)tot.pages;
  const int step = gridDim.x * blockDim.x;
  const bool alone = gridDim.x == 1;
  for (int i = blockIdx.x * blockDim.x + threadIdx.x; i < pages; i += step) {
    const int b = find_request(cu_pg, n, i);
    int* e = a.table + b * a.table_stride + (i - cu_pg[b]);
    int page = *e;
    if (page < 0 || page >= a.n_pages) {
      *err = kErrPagedPage;
      atomicAdd(alone ? &none : a.state_out + 2, 1);
      page = -1;
    }
    a.free_pages[count + i] = page;
    *e = -1;
  }
  if (alone) {
    __syncthreads();
    if (none) pages = drop_negative(a.free_pages + count, pages);
    // (a length is read and written by one thread after the first barrier)
    for (int b = threadIdx.x; b < n; b += blockDim.x) a.lens_out[b] = !status && gone[b + 1] > gone[b] ? 0 : a.lens[b];
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    if (alone) {
      a.state_out[0] = count + pages;
      a.state_out[2] = 0;
    }
    a.state_out[1] = status;
    a.state_out[3] = pages;
  }
}

// Before a release on more than one CTA: its count of entries that are no page.
__global__ void paged_release_begin_kernel(const tb2_paged_release_args a) {
  griddep_wait_release();
  if (threadIdx.x == 0) a.state_out[2] = 0;
}

// And after it: the lengths, the stack's count, and the stack without such entries.
__global__ void __launch_bounds__(256) paged_release_commit_kernel(const tb2_paged_release_args a) {
  griddep_wait_release();
  const int b = blockIdx.x * blockDim.x + threadIdx.x;
  if (b < a.n_req) a.lens_out[b] = !a.state_out[1] && a.done[b] ? 0 : a.lens[b];
  if (blockIdx.x) return;
  const int count = a.state[0];
  int pages = a.state_out[3];
  if (a.state_out[2]) pages = drop_negative(a.free_pages + count, pages);
  __syncthreads();   // the state is read
  if (threadIdx.x) return;
  a.state_out[0] = count + pages;
  a.state_out[2] = 0;
  a.state_out[3] = pages;
}

int smem_setup(int) {
  const int bytes = 3 * (kMaxReq + 1) * (int)sizeof(int);
  cudaFuncAttributes at;   // (asking for them loads a kernel)
  if (cudaFuncGetAttributes(&at, paged_plan_commit_kernel) != cudaSuccess ||
      cudaFuncGetAttributes(&at, paged_release_begin_kernel) != cudaSuccess ||
      cudaFuncGetAttributes(&at, paged_release_commit_kernel) != cudaSuccess ||
      cudaFuncSetAttribute(paged_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess)
    return -3;
  return cudaFuncSetAttribute(paged_release_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) == cudaSuccess
             ? 0
             : -3;
}

// CTAs for `items` threads' worth of work: a full CTA before another one pays
// for its own prefix sums; one CTA of fewer threads (cheaper barriers) where
// requests and work are few.
int grid_for(long long items) { return (int)std::max<long long>(1, std::min<long long>(148, items / kThreads)); }
int threads_for(int n_req, long long items) { return n_req <= 256 && items <= 512 ? 256 : kThreads; }

// n ints that are updated: in place (1), elsewhere (0), or in part over themselves (-1).
int placed(const int* x, const int* y, long long n) { return x == y ? 1 : x < y + n && y < x + n ? -1 : 0; }

}  // namespace

int paged_plan_prepare() {
  static DeviceOnce setup;
  return setup.ensure(smem_setup);
}

int paged_plan_launch(const tb2_paged_plan_args& a, int* err, cudaStream_t st) {
  if (paged_plan_prepare()) return -3;
  const size_t smem = 3 * (size_t)(a.n_req + 1) * sizeof(int);
  const long long items = ((long long)a.n_tokens + kRun - 1) / kRun;
  const int grid = grid_for(items);
  const int in_place = placed(a.lens, a.lens_out, a.n_req) || placed(a.state, a.state_out, 4);
  if (launch_pdl(paged_plan_kernel, dim3(grid), dim3(threads_for(a.n_req, items)), smem, st, a, in_place, err)) return -3;
  if (grid == 1 || !in_place) return 0;
  return launch_pdl(paged_plan_commit_kernel, dim3((a.n_req + 255) / 256), dim3(256), 0, st, a);
}

int paged_release_launch(const tb2_paged_release_args& a, int* err, cudaStream_t st) {
  if (paged_plan_prepare()) return -3;
  const size_t smem = 2 * (size_t)(a.n_req + 1) * sizeof(int);
  const long long items = (long long)a.n_req * a.table_width;   // (at most: the lengths are on the device)
  const int grid = grid_for(items / 4), threads = threads_for(a.n_req, items);
  if (grid > 1 && launch_pdl(paged_release_begin_kernel, dim3(1), dim3(32), 0, st, a)) return -3;
  if (launch_pdl(paged_release_kernel, dim3(grid), dim3(threads), smem, st, a, err)) return -3;
  return grid == 1 ? 0 : launch_pdl(paged_release_commit_kernel, dim3((a.n_req + 255) / 256), dim3(256), 0, st, a);
}

}  // namespace tb2

extern "C" {

int tb2_paged_plan(const tb2_paged_plan_args* a, void* stream) {
  if (!a || a->n_req < 1 || a->n_req > tb2::kMaxReq || a->table_width < 1 || a->table_stride < a->table_width ||
      a->page_size < 1 || a->page_size > (1 << 20) || a->n_pages < 1 || a->n_free < 0 || a->n_tokens < 0 ||
      a->n_tokens > 0x7fffff00)
    return -1;
  if (!a->lens || !a->add || !a->table || !a->state || !a->lens_out || !a->state_out || !a->cu_tokens ||
      (a->n_free && !a->free_pages) || (a->n_tokens && (!a->slots || !a->positions || !a->requests)))
    return -1;
  if (!tb2::all_aligned(4, {a->lens, a->add, a->table, a->free_pages, a->state, a->lens_out, a->state_out, a->cu_tokens,
                            a->positions, a->requests}) ||
      !tb2::aligned(a->slots, 8))
    return -1;
  if (tb2::placed(a->lens, a->lens_out, a->n_req) < 0 || tb2::placed(a->state, a->state_out, 4) < 0) return -1;
  if ((long long)a->table_width * a->page_size > 0x7fffff00LL) return -1;   // positions are 32 bits wide
  int* err = tb2::device_error_word();
  if (!err) return -3;
  return tb2::paged_plan_launch(*a, err, static_cast<cudaStream_t>(stream));
}

int tb2_paged_release(const tb2_paged_release_args* a, void* stream) {
  if (!a || a->n_req < 1 || a->n_req > tb2::kMaxReq || a->table_width < 1 || a->table_stride < a->table_width ||
      a->page_size < 1 || a->page_size > (1 << 20) || a->n_pages < 1 || a->n_free < 0)
    return -1;
  if (!a->lens || !a->done || !a->table || !a->state || !a->lens_out || !a->state_out ||
      (a->n_free && !a->free_pages))
    return -1;
  if (!tb2::all_aligned(4, {a->lens, a->done, a->table, a->free_pages, a->state, a->lens_out, a->state_out})) return -1;
  if (tb2::placed(a->lens, a->lens_out, a->n_req) < 0 || tb2::placed(a->state, a->state_out, 4) < 0) return -1;
  if ((long long)a->table_width * a->page_size > 0x7fffff00LL) return -1;
  int* err = tb2::device_error_word();
  if (!err) return -3;
  return tb2::paged_release_launch(*a, err, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
