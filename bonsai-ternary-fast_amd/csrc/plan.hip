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
//  * the rows: a tree has at most 64 nodes, one per lane of a wave: depth and
//    ancestor bits come from six rounds of pointer doubling over the lanes (after
//    round r a lane has collected its 2^r nearest ancestors), whatever the tree's
//    shape.
// Small plans do both in the one workgroup, with the requests' places still in
// LDS and the new pages straight from the free list (plan_small_kernel); larger
// ones in a second launch, a wave for each request and each 1024 of its rows.
// Bound by latency: a launch and its chain of reads and scans (8 requests of one token
// 5.5 us, 256 trees of up to 48 nodes 5.0 + 2.9; one launch for all sizes would leave the
// rows of large plans to one CU).
#include <string>

#include "../../include/btf/hip_abi.h"
#include "common.h"

namespace btfhip {
namespace {

constexpr int kPlanThreads = 1024;
constexpr int kRowsPerWave = 1024;

// What a chunk's requests were found to be, in LDS.
struct Chunk {
  uint64_t part[kPlanThreads / 64];
  long long got[kPlanThreads];  // pages handed out up to and including each request of the chunk
  int first[kPlanThreads];      // its pages before the step
  int row0[kPlanThreads + 1];   // its first row
  int ctx[kPlanThreads];        // its tokens in the cache; -1: refused
};

__device__ __forceinline__ void plan_requests(const btf_page_plan& a, Chunk& c, long long free0) {
  long long rows = 0, pages = 0, taken = 0;
  for (int s0 = 0; s0 < a.S; s0 += kPlanThreads) {
    const int s = s0 + (int)threadIdx.x;
    const bool live = s < a.S;
    const long long ctx = live ? a.ctx[s] : 0, nn = live ? a.n_new[s] : 0, h = live ? a.held[s] : 0;
    const long long n = max(nn, 0ll);
    uint64_t all;
    const long long end = rows + (long long)block_scan<kPlanThreads>(n, c.part, &all);
    const int row0 = (int)min(end - n, (long long)a.T);
    c.row0[threadIdx.x] = row0;
    if (live) a.row0[s] = row0;
    rows += (long long)all;
    const long long total = (ctx + nn + a.page - 1) / a.page;
    const bool sound = live && ctx >= 0 && nn >= 0 && h >= 0 && h <= a.ldt && ctx <= h * a.page && end <= a.T &&
                       total <= a.ldt && ctx + nn <= 0x7fffffffll;
    const long long want = sound ? max(total - h, 0ll) : 0;
    const long long upto = pages + (long long)block_scan<kPlanThreads>(want, c.part, &all);
    // (the served needs are the first ones: their sums are those of all needs)
    const bool served = sound && (want == 0 || upto <= free0);
    const long long need = served ? want : 0;
    c.got[threadIdx.x] = upto - pages;
    pages += (long long)all;
    c.first[threadIdx.x] = (int)h;
    c.ctx[threadIdx.x] = served ? (int)ctx : -1;
    if (live) {
      a.kv_len[s] = served ? (int)(ctx + nn) : 0;
      a.held_out[s] = (int)(h + need);
    }
    __syncthreads();
    // entries k of the chunk's needs, as far as the free list reaches
    const long long chunk = min(max(free0 - (pages - (long long)all), 0ll), (long long)all);
    for (long long k = threadIdx.x; k < chunk; k += kPlanThreads) {
      int lo = 0, hi = kPlanThreads - 1;  // the first request with got > k
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (c.got[mid] > k) hi = mid;
        else lo = mid + 1;
      }
      if (c.ctx[lo] < 0) continue;  // (refused: its pages did not reach)
      const long long j = k - (lo ? c.got[lo - 1] : 0);
      a.table[(size_t)(s0 + lo) * a.ldt + c.first[lo] + j] = a.free_list[free0 - 1 - taken - k];
    }
    uint64_t handed;
    (void)block_scan<kPlanThreads>(need, c.part, &handed);
    taken += (long long)handed;
  }
  if (threadIdx.x == 0) {
    a.row0[a.S] = (int)min(rows, (long long)a.T);
    *a.n_free_out = (int)(free0 - taken);
  }
  c.row0[min(a.S, kPlanThreads)] = (int)min(rows, (long long)a.T);  // (one chunk: the end of its rows)
  __syncthreads();
}

// Depth and bits (ancestors and itself) of node `lane` of a tree of n nodes, by one wave.
__device__ __forceinline__ void tree_node(const int* parent, int n, int lane, int& depth, unsigned long long& bits) {
  int up = lane < n ? parent[lane] : -1;
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
  if (tree) tree_node(a.parent + r0, n, lane, depth, bits);
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

__global__ void __launch_bounds__(kPlanThreads) plan_requests_kernel(btf_page_plan a) {
  __shared__ Chunk c;
  const long long free0 = max(*a.n_free, 0);
  plan_requests(a, c, free0);
}

__global__ void __launch_bounds__(64) plan_rows_kernel(btf_page_plan a) {
  plan_rows(a, blockIdx.x, blockIdx.y * kRowsPerWave);
}

// Both phases of at most 1024 requests.
__global__ void __launch_bounds__(kPlanThreads) plan_small_kernel(btf_page_plan a) {
  __shared__ Chunk c;
  const long long free0 = max(*a.n_free, 0);
  plan_requests(a, c, free0);
  auto slot_of = [&](int s, int at) {
    const int p = at / a.page, h = c.first[s];
    const int pg = p < h ? a.table[(size_t)s * a.ldt + p] : a.free_list[free0 - 1 - (s ? c.got[s - 1] : 0) - (p - h)];
    return pg >= 0 && pg < a.pages ? pg * a.page + at % a.page : -1;
  };
  if (!a.parent) {  // a row a thread, its request by bisection of the rows' starts
    const int end = c.row0[a.S];
    for (int t = threadIdx.x; t < end; t += kPlanThreads) {
      int lo = 0, hi = a.S - 1;  // the last request with row0 <= t
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (c.row0[mid] <= t) lo = mid;
        else hi = mid - 1;
      }
      const int ctx = c.ctx[lo], at = ctx + t - c.row0[lo];
      a.pos[t] = ctx < 0 ? 0 : at;
      a.slot[t] = ctx < 0 ? -1 : slot_of(lo, at);
    }
    return;
  }
  const int lane = threadIdx.x & 63;
  for (int s = threadIdx.x >> 6; s < a.S; s += kPlanThreads / 64) {  // a request a wave
    const int r0 = c.row0[s], n = c.row0[s + 1] - r0, ctx = c.ctx[s];
    const bool tree = n <= BTF_TREE_NODES;
    int depth = 0;
    unsigned long long bits = 0;
    if (tree) tree_node(a.parent + r0, n, lane, depth, bits);
    for (int i = lane; i < n; i += 64) {
      a.pos[r0 + i] = ctx < 0 ? 0 : ctx + (tree ? depth : i);
      a.slot[r0 + i] = ctx < 0 ? -1 : slot_of(s, ctx + i);
      a.tree[r0 + i] = ctx >= 0 && tree ? bits : 0;
    }
  }
}

}  // namespace

int page_plan(const btf_page_plan& a, hipStream_t st) {
  // One launch where the workgroup has few rows a thread, or few trees a wave (a call's time in one launch and in two, us:
  // one request of 4005 rows 8.5 and 11.3, 64 of 4965 in all 10.2 and 11.3, of 7954 12.8 and 10.9; 16 trees of up to 64
  // nodes 8.2 and 10.8, 48 9.9 and 11.2, 64 11.1 and 11.0, 128 16.3 and 11.2).
  if (a.T > 0 && (a.parent ? a.S <= 64 && a.T <= 4096 : a.S <= kPlanThreads && a.T <= 4096)) {
    hipLaunchKernelGGL(plan_small_kernel, dim3(1), dim3(kPlanThreads), 0, st, a);
    return launch_status("plan_small_kernel");
  }
  hipLaunchKernelGGL(plan_requests_kernel, dim3(1), dim3(kPlanThreads), 0, st, a);
  const int rc = launch_status("plan_requests_kernel");
  if (rc != BTF_OK || a.T == 0) return rc;
  hipLaunchKernelGGL(plan_rows_kernel, dim3(a.S, (a.T + kRowsPerWave - 1) / kRowsPerWave), dim3(64), 0, st, a);
  return launch_status("plan_rows_kernel");
}

}  // namespace btfhip
