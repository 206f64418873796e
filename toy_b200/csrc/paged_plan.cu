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
// shared memory (n_req <= 16384; two loads per request) and fills its slice of
// tokens and pages, instead of a scan, a barrier over the grid and a fill.
// Lengths and the stack's count may be updated in place: a single CTA writes
// them after its own reads; a larger grid leaves that to a second, tiny
// kernel.
#include <algorithm>

#include "paged.cuh"
#include "pdl.cuh"
#include "runtime.cuh"

namespace tb2 {
namespace {

constexpr int kMaxReq = 16384;
constexpr int kThreads = 1024;

// The totals of a scan: tokens and pages of every request, and whether any
// input was bad (codes as the C API documents them).
struct Totals {
  long long tokens, pages;
  int bad;
};

__device__ __forceinline__ int div_up(int a, int b) { return (int)(((long long)a + b - 1) / b); }

// Exclusive prefix sums of two values per request into st[0 .. n] and
// sp[0 .. n]; item(b, tok, pg) returns a status and the two values. Sums are
// 64 bits wide and stored cut to 32; totals that do not fit are reported by
// the caller's own limits before the stored values are used.
template <class F>
__device__ Totals scan_requests(int n, int* st, int* sp, F&& item) {
  __shared__ long long wt[32], wp[32];
  __shared__ int sbad;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, nw = blockDim.x >> 5;
  if (tid == 0) sbad = 0;
  __syncthreads();
  const int per = (n + (int)blockDim.x - 1) / (int)blockDim.x;
  const int b0 = min(n, tid * per), b1 = min(n, b0 + per);
  long long ts = 0, ps = 0;
  int bad = 0;
  for (int b = b0; b < b1; ++b) {
    int tok = 0, pg = 0;
    bad = max(bad, item(b, tok, pg));
    ts += tok;
    ps += pg;
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
  if (lane == 31) {
    wt[warp] = ti;
    wp[warp] = pi;
  }
  if (bad) atomicMax(&sbad, bad);
  __syncthreads();
  long long bt = 0, bp = 0, tt = 0, tp = 0;
  for (int w = 0; w < nw; ++w) {
    if (w < warp) {
      bt += wt[w];
      bp += wp[w];
    }
    tt += wt[w];
    tp += wp[w];
  }
  bt += ti - ts;
  bp += pi - ps;
  for (int b = b0; b < b1; ++b) {
    int tok = 0, pg = 0;
    item(b, tok, pg);
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
  return {tt, tp, sbad};
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

__global__ void __launch_bounds__(kThreads) paged_plan_kernel(const tb2_paged_plan_args a, int* err) {
  extern __shared__ int sm[];
  int* cu_tok = sm;
  int* cu_pg = sm + a.n_req + 1;
  griddep_wait_release();
  const int P = a.page_size, n = a.n_req;
  const int count = a.state[0];
  const Totals tot = scan_requests(n, cu_tok, cu_pg, [&](int b, int& tok, int& pg) {
    const int len = a.lens[b], add = a.add[b];
    if (len < 0 || add < 0) return 4;
    const long long end = (long long)len + add;
    if ((end + P - 1) / P > a.table_width) return 2;
    tok = add;
    pg = div_up((int)end, P) - div_up(len, P);
    return 0;
  });
  int status = tot.bad;
  if (count < 0 || count > a.n_free) status = 4;
  else if (!status && tot.tokens > a.n_tokens) status = 3;
  else if (!status && tot.pages > count) status = 1;
  const int tokens = status ? 0 : (int)tot.tokens, pages = status ? 0 : (int)tot.pages;
  const int step = gridDim.x * blockDim.x, first = blockIdx.x * blockDim.x + threadIdx.x;
  for (int i = first; i < pages; i += step) {
    const int b = find_request(cu_pg, n, i);
    a.table[b * a.table_stride + div_up(a.lens[b], P) + (i - cu_pg[b])] = a.free_pages[count - 1 - i];
  }
  for (int t = first; t < a.n_tokens; t += step) {
    long long slot = -1;
    int pos = 0, req = -1;
    if (t < tokens) {
      req = find_request(cu_tok, n, t);
      const int len = a.lens[req], held = div_up(len, P);
      pos = len + (t - cu_tok[req]);
      const int blk = pos / P;
      const int page =
          blk < held ? a.table[req * a.table_stride + blk] : a.free_pages[count - 1 - (cu_pg[req] + blk - held)];
      if (page >= 0 && page < a.n_pages) slot = (long long)page * P + (pos - blk * P);
      else *err = kErrPagedPage;
    }
    a.slots[t] = slot;
    a.positions[t] = pos;
    a.requests[t] = req;
  }
  if (blockIdx.x == 0)
    for (int b = threadIdx.x; b <= n; b += blockDim.x) a.cu_tokens[b] = status ? 0 : cu_tok[b];
  const bool alone = gridDim.x == 1;
  if (alone) __syncthreads();   // every read of lens and state is done
  if (alone)
    for (int b = threadIdx.x; b < n; b += blockDim.x) a.lens_out[b] = a.lens[b] + (status ? 0 : a.add[b]);
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    a.state_out[1] = status;
    a.state_out[2] = tokens;
    a.state_out[3] = pages;
    if (alone) a.state_out[0] = count - pages;
  }
}

// After a plan on more than one CTA: the lengths and the stack's count.
__global__ void paged_plan_commit_kernel(const tb2_paged_plan_args a) {
  griddep_wait_release();
  const int b = blockIdx.x * blockDim.x + threadIdx.x;
  if (b < a.n_req) a.lens_out[b] = a.lens[b] + (a.state_out[1] ? 0 : a.add[b]);
  if (b == 0) a.state_out[0] = a.state[0] - a.state_out[3];
}

__global__ void __launch_bounds__(kThreads) paged_release_kernel(const tb2_paged_release_args a, int* err) {
  extern __shared__ int sm[];
  int* cu_pg = sm;
  int* unused = sm + a.n_req + 1;
  griddep_wait_release();
  const int P = a.page_size, n = a.n_req;
  const int count = a.state[0];
  const Totals tot = scan_requests(n, unused, cu_pg, [&](int b, int& tok, int& pg) {
    const int len = a.lens[b];
    if (len < 0 || ((long long)len + P - 1) / P > a.table_width) return 4;
    pg = a.done[b] ? div_up(len, P) : 0;
    tok = 0;
    return 0;
  });
  int status = tot.bad;
  if (count < 0 || count > a.n_free) status = 4;
  else if (!status && tot.pages > a.n_free - count) status = 1;
  const int pages = status ? 0 : (int)tot.pages;
  const int step = gridDim.x * blockDim.x;
  for (int i = blockIdx.x * blockDim.x + threadIdx.x; i < pages; i += step) {
    const int b = find_request(cu_pg, n, i);
    int* e = a.table + b * a.table_stride + (i - cu_pg[b]);
    const int page = *e;
    if (page < 0 || page >= a.n_pages) *err = kErrPagedPage;
    a.free_pages[count + i] = page;
    *e = -1;
  }
  const bool alone = gridDim.x == 1;
  if (alone) {
    __syncthreads();
    for (int b = threadIdx.x; b < n; b += blockDim.x) a.lens_out[b] = !status && a.done[b] ? 0 : a.lens[b];
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    a.state_out[1] = status;
    a.state_out[2] = 0;
    a.state_out[3] = pages;
    if (alone) a.state_out[0] = count + pages;
  }
}

__global__ void paged_release_commit_kernel(const tb2_paged_release_args a) {
  griddep_wait_release();
  const int b = blockIdx.x * blockDim.x + threadIdx.x;
  if (b < a.n_req) a.lens_out[b] = !a.state_out[1] && a.done[b] ? 0 : a.lens[b];
  if (b == 0) a.state_out[0] = a.state[0] + a.state_out[3];
}

int smem_setup(int) {
  const int bytes = 2 * (kMaxReq + 1) * (int)sizeof(int);
  if (cudaFuncSetAttribute(paged_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess)
    return -3;
  return cudaFuncSetAttribute(paged_release_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) == cudaSuccess
             ? 0
             : -3;
}

// CTAs for `items` tokens and pages: four a thread before another CTA pays
// for its own prefix sums.
int grid_for(long long items) {
  return (int)std::max<long long>(1, std::min<long long>(148, items / (4 * kThreads)));
}

}  // namespace

int paged_plan_launch(const tb2_paged_plan_args& a, int* err, cudaStream_t st) {
  static DeviceOnce setup;
  if (setup.ensure(smem_setup)) return -3;
  const size_t smem = 2 * (size_t)(a.n_req + 1) * sizeof(int);
  const int grid = grid_for(a.n_tokens);
  if (launch_pdl(paged_plan_kernel, dim3(grid), dim3(kThreads), smem, st, a, err)) return -3;
  if (grid == 1) return 0;
  return launch_pdl(paged_plan_commit_kernel, dim3((a.n_req + 255) / 256), dim3(256), 0, st, a);
}

int paged_release_launch(const tb2_paged_release_args& a, int* err, cudaStream_t st) {
  static DeviceOnce setup;
  if (setup.ensure(smem_setup)) return -3;
  const size_t smem = 2 * (size_t)(a.n_req + 1) * sizeof(int);
  const int grid = grid_for((long long)a.n_req * a.table_width);
  if (launch_pdl(paged_release_kernel, dim3(grid), dim3(kThreads), smem, st, a, err)) return -3;
  if (grid == 1) return 0;
  return launch_pdl(paged_release_commit_kernel, dim3((a.n_req + 255) / 256), dim3(256), 0, st, a);
}

}  // namespace tb2

extern "C" {

int tb2_paged_plan(const tb2_paged_plan_args* a, void* stream) {
  if (!a || a->n_req < 1 || a->n_req > tb2::kMaxReq || a->table_width < 1 || a->table_stride < a->table_width ||
      a->page_size < 1 || a->page_size > (1 << 20) || a->n_pages < 1 || a->n_free < 0 || a->n_tokens < 0)
    return -1;
  if (!a->lens || !a->add || !a->table || !a->state || !a->lens_out || !a->state_out || !a->cu_tokens ||
      (a->n_free && !a->free_pages) || (a->n_tokens && (!a->slots || !a->positions || !a->requests)))
    return -1;
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
  if ((long long)a->table_width * a->page_size > 0x7fffff00LL) return -1;
  int* err = tb2::device_error_word();
  if (!err) return -3;
  return tb2::paged_release_launch(*a, err, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
