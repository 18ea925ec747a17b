// plan.hip -- a serving step's rows, cache pages and slots from the requests'
// lengths (btf_hip_launch_page_plan; gfx950).
//
// Two phases, integers only:
//  * plan_requests: one workgroup over all requests, 1024 at a time. Two
//    prefix sums over the requests (rows, then the pages that the sound ones
//    need) decide who is served; then the new table entries, numbered 0 .. sum
//    of the needs, are spread over the threads, each finding its request by
//    bisection of the sums in LDS. Reads come before the writes of the same
//    request's values and of the free count, so held_out and n_free_out may be
//    the inputs.
//  * plan_rows: one wave per request (and per 1024 of its rows). A tree has at
//    most 64 nodes, one per lane: depth and ancestor bits come from six rounds
//    of pointer doubling over the lanes (after round r a lane has collected its
//    2^r nearest ancestors), whatever the tree's shape.
#include <string>

#include "../../include/btf/hip_abi.h"
#include "common.h"

namespace btfhip {
namespace {

constexpr int kPlanThreads = 1024;
constexpr int kRowsPerWave = 1024;

__device__ void plan_requests(const btf_page_plan& a) {
  __shared__ uint64_t part[kPlanThreads / 64];
  __shared__ long long got[kPlanThreads];  // pages handed out up to and including each request of the chunk
  __shared__ int first[kPlanThreads];      // its pages before the step
  const long long free0 = max(*a.n_free, 0);
  long long rows = 0, pages = 0, taken = 0;
  for (int s0 = 0; s0 < a.S; s0 += kPlanThreads) {
    const int s = s0 + (int)threadIdx.x;
    const bool live = s < a.S;
    const long long c = live ? a.ctx[s] : 0, nn = live ? a.n_new[s] : 0, h = live ? a.held[s] : 0;
    const long long n = max(nn, 0ll);
    uint64_t all;
    const long long end = rows + (long long)block_scan<kPlanThreads>(n, part, &all);
    if (live) a.row0[s] = (int)min(end - n, (long long)a.T);
    rows += all;
    const long long total = (c + nn + a.page - 1) / a.page;
    const bool sound = live && c >= 0 && nn >= 0 && h >= 0 && h <= a.ldt && c <= h * a.page && end <= a.T &&
                       total <= a.ldt && c + nn <= 0x7fffffffll;
    const long long want = sound ? max(total - h, 0ll) : 0;
    const long long upto = pages + (long long)block_scan<kPlanThreads>(want, part, &all);
    pages += all;
    const bool served = sound && (want == 0 || upto <= free0);
    // the served needs are the first ones: their sums are those of all needs
    const long long need = served ? want : 0;
    uint64_t chunk_u;
    got[threadIdx.x] = (long long)block_scan<kPlanThreads>(need, part, &chunk_u);
    const long long chunk = (long long)chunk_u;
    first[threadIdx.x] = (int)h;
    if (live) {
      a.kv_len[s] = served ? (int)(c + nn) : 0;
      a.held_out[s] = (int)(h + need);
    }
    __syncthreads();
    for (long long k = threadIdx.x; k < chunk; k += kPlanThreads) {
      int lo = 0, hi = kPlanThreads - 1;  // the first request with got > k
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (got[mid] > k) hi = mid;
        else lo = mid + 1;
      }
      const long long j = k - (lo ? got[lo - 1] : 0);
      a.table[(size_t)(s0 + lo) * a.ldt + first[lo] + j] = a.free_list[free0 - 1 - taken - k];
    }
    taken += chunk;
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    a.row0[a.S] = (int)min(rows, (long long)a.T);
    *a.n_free_out = (int)(free0 - taken);
  }
}

// Rows [i0, i0 + kRowsPerWave) of request s, by one wave.
__device__ void plan_rows(const btf_page_plan& a, int s, int i0) {
  const int lane = threadIdx.x & 63;
  const int r0 = a.row0[s], n = a.row0[s + 1] - r0;
  if (i0 >= n) return;
  const int kv = a.kv_len[s];
  const bool served = kv > 0;
  const int ctx = kv - n;
  const bool tree = a.parent && n <= BTF_TREE_NODES;
  int depth = 0;
  unsigned long long bits = 0;
  if (tree) {
    int up = lane < n ? a.parent[r0 + lane] : -1;
    if (up < 0 || up >= lane) up = -1;
    bits = 1ull << lane;
    depth = up >= 0;
#pragma unroll
    for (int r = 0; r < 6; ++r) {
      const int at = up >= 0 ? up : lane;
      const unsigned long long b = __shfl(bits, at, 64);
      const int d = __shfl(depth, at, 64), u = __shfl(up, at, 64);
      if (up >= 0) {
        bits |= b;
        depth += d;
        up = u;
      }
    }
  }
  const int end = min(n, i0 + kRowsPerWave);
  for (int i = i0 + lane; i < end; i += 64) {
    int pos = 0, slot = -1;
    if (served) {
      const int at = ctx + i;
      pos = ctx + (tree ? depth : i);
      const int pg = a.table[(size_t)s * a.ldt + at / a.page];
      if (pg >= 0 && pg < a.pages) slot = pg * a.page + at % a.page;
    }
    a.pos[r0 + i] = pos;
    a.slot[r0 + i] = slot;
    if (a.parent) a.tree[r0 + i] = served && tree ? bits : 0;
  }
}

__global__ void __launch_bounds__(kPlanThreads) plan_requests_kernel(btf_page_plan a) { plan_requests(a); }

__global__ void __launch_bounds__(64) plan_rows_kernel(btf_page_plan a) {
  plan_rows(a, blockIdx.x, blockIdx.y * kRowsPerWave);
}

}  // namespace

int page_plan(const btf_page_plan& a, hipStream_t st) {
  hipLaunchKernelGGL(plan_requests_kernel, dim3(1), dim3(kPlanThreads), 0, st, a);
  const int rc = launch_status("plan_requests_kernel");
  if (rc != BTF_OK || a.T == 0) return rc;
  hipLaunchKernelGGL(plan_rows_kernel, dim3(a.S, (a.T + kRowsPerWave - 1) / kRowsPerWave), dim3(64), 0, st, a);
  return launch_status("plan_rows_kernel");
}

}  // namespace btfhip
