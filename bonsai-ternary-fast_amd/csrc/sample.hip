// sample.hip -- one token per row of logits with temperature, top-k, top-p and
// min-p from a given uniform number (btf_hip_launch_sample; gfx950).
//
// The kept set is a prefix of the order (falling logit, rising index), so it is
// a threshold key and the number of the logits equal to it that stay. Keys are
// the logits' bits in an order-preserving form (as the greedy pick's), found
// eight bits at a time from histograms of counts and weights in LDS. Weights are
// whole numbers (units of 2^-43, in 64 bits), so sums do not depend on their
// order and no threshold can be crossed by a rounding.
//
// One workgroup per row.
#include <cmath>
#include <string>

#include "../../include/btf/hip_abi.h"
#include "common.h"
#include "slice.h"

namespace btfhip {
namespace {

typedef unsigned long long u64;
constexpr int kThreads = 1024;
constexpr double kOne = 8796093022208.0;  // 2^43

__device__ __forceinline__ uint32_t key_of(float x) { return (uint32_t)(argmax_key(x, 0) >> 32); }
__device__ __forceinline__ float of_key(uint32_t k) { return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k); }

// Weight of a logit in units of 2^-43.
__device__ __forceinline__ u64 weight(float x, float top, double inv_t) {
  if (x == top) return (u64)kOne;
  const double d = ((double)x - (double)top) * inv_t;
  return d > -31.0 ? (u64)rint(exp(d) * kOne) : 0;  // (2^-44 is exp(-30.5); a NaN gives 0)
}

struct Shared {
  u64 sum[256];
  uint32_t cnt[256];
  u64 scan[kThreads / 64];
  u64 key;
  uint32_t prefix, n;
  u64 s;
  int flag;
};

// Inclusive prefix sum over the workgroup; *total: the whole sum.
__device__ u64 block_scan(u64 v, u64* part, u64* total) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const u64 u = __shfl_up(v, o, 64);
    if (lane >= o) v += u;
  }
  __syncthreads();
  if (lane == 63) part[w] = v;
  __syncthreads();
  u64 before = 0, all = 0;
  for (int i = 0; i < kThreads / 64; ++i) {
    const u64 p = part[i];
    if (i < w) before += p;
    all += p;
  }
  *total = all;
  return v + before;
}

// The key at which the count (by_count) or the weight of the logits from the
// largest down reaches `want`, with what lies above it, over keys > floor.
// False if nothing reaches it.
__device__ bool find_key(const float* x, int V, float top, double inv_t, bool by_count, double want, uint32_t floor,
                         Shared& sh, uint32_t* key, u64* above) {
  uint32_t prefix = 0;
  u64 got = 0;
  for (int shift = 24; shift >= 0; shift -= 8) {
    __syncthreads();
    if (threadIdx.x < 256) sh.sum[threadIdx.x] = 0, sh.cnt[threadIdx.x] = 0;
    if (threadIdx.x == 0) sh.flag = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < V; i += kThreads) {
      const uint32_t k = key_of(x[i]);
      if (k <= floor || (shift < 24 && (k >> (shift + 8)) != prefix)) continue;
      if (by_count) atomicAdd(&sh.cnt[k >> shift & 255], 1u);
      else atomicAdd(&sh.sum[k >> shift & 255], weight(x[i], top, inv_t));
    }
    __syncthreads();
    if (threadIdx.x == 0) {
      u64 s = got;
      for (int b = 255; b >= 0; --b) {
        const u64 v = by_count ? sh.cnt[b] : sh.sum[b];
        if (v && (double)(s + v) >= want) {
          sh.prefix = prefix << 8 | b;
          sh.s = s;
          sh.flag = 1;
          break;
        }
        s += v;
      }
      if (!sh.flag) sh.s = s;
    }
    __syncthreads();
    got = sh.s;
    if (!sh.flag) break;
    prefix = sh.prefix;
  }
  *above = got;
  *key = prefix;
  const bool found = sh.flag != 0;
  __syncthreads();
  return found;
}

__global__ void __launch_bounds__(kThreads) sample_row_kernel(btf_sampling a) {
  __shared__ Shared sh;
  const int m = blockIdx.x;
  const float* x = a.logits + (size_t)m * a.ldl;
  if (threadIdx.x == 0) sh.key = 0;
  __syncthreads();
  u64 best = 0;
  for (int i = threadIdx.x; i < a.V; i += kThreads) best = key_max(best, argmax_key(x[i], i));
  best = wave_max_key(best);
  if ((threadIdx.x & 63) == 0) atomicMax(&sh.key, best);
  __syncthreads();
  best = sh.key;
  const float temp = a.temperature ? a.temperature[m] : 1.f;
  if (!(temp > 0.f) || best == 0) {
    if (threadIdx.x == 0) {
      a.token[m] = argmax_key_index(best);
      if (a.logprob) a.logprob[m] = 0.f;
    }
    return;
  }
  const float top = of_key((uint32_t)(best >> 32));
  const double inv_t = 1.0 / (double)temp;
  // top-k
  uint32_t key = 0;       // kept: keys > key, and the first `ties` logits at it
  uint32_t ties = 0;
  const int k = a.top_k ? a.top_k[m] : 0;
  u64 n_above = 0;
  if (k > 0 && k < a.V && find_key(x, a.V, top, inv_t, true, k, 0, sh, &key, &n_above)) ties = (uint32_t)(k - n_above);
  // top-p, within the top-k
  const float p = a.top_p ? a.top_p[m] : 1.f;
  if (p < 1.f) {
    u64 mine = 0, total;
    for (int i = threadIdx.x; i < a.V; i += kThreads)
      if (key_of(x[i]) > key) mine += weight(x[i], top, inv_t);
    block_scan(mine, sh.scan, &total);
    const u64 wt = key ? weight(of_key(key), top, inv_t) : 0;
    const double want = (double)p * (double)(total + ties * wt);
    uint32_t pk;
    u64 above;
    if (find_key(x, a.V, top, inv_t, false, want, key, sh, &pk, &above)) {
      const u64 w = weight(of_key(pk), top, inv_t);
      const double more = ceil((want - (double)above) / (double)w);
      key = pk;
      ties = more < 1.0 ? 1u : (uint32_t)more;
    } else if (ties) {
      const double more = wt ? ceil((want - (double)total) / (double)wt) : 1.0;
      ties = (uint32_t)fmin((double)ties, fmax(more, 1.0));
    }
  }
  const float mp = a.min_p ? a.min_p[m] : 0.f;
  const double floor_w = mp > 0.f ? (double)fminf(mp, 1.f) * kOne : 0.0;
  // the kept weights in index order: a contiguous piece per thread
  const int per = (a.V + kThreads - 1) / kThreads;
  const int i0 = min(a.V, (int)threadIdx.x * per), i1 = min(a.V, i0 + per);
  u64 eq = 0, total;
  for (int i = i0; i < i1; ++i) eq += key_of(x[i]) == key;
  const u64 eq0 = block_scan(eq, sh.scan, &total) - eq;
  auto kept = [&](int i, u64* rank) -> u64 {
    const uint32_t kk = key_of(x[i]);
    if (kk < key || kk == 0) return 0;
    if (kk == key && (*rank)++ >= ties) return 0;
    const u64 w = weight(x[i], top, inv_t);
    return (double)w >= floor_w ? w : 0;
  };
  u64 mine = 0, rank = eq0;
  for (int i = i0; i < i1; ++i) mine += kept(i, &rank);
  const u64 end = block_scan(mine, sh.scan, &total);
  const double u = a.u[m];
  u64 at = u > 0.0 ? (u64)fmin(u * (double)total, 9.0e18) : 0;
  if (at >= total) at = total - 1;
  if (end > at && end - mine <= at) {
    u64 s = end - mine;
    rank = eq0;
    for (int i = i0; i < i1; ++i) {
      const u64 w = kept(i, &rank);
      s += w;
      if (s > at) {
        a.token[m] = i;
        if (a.logprob) a.logprob[m] = (float)log((double)w / (double)total);
        break;
      }
    }
  }
}

}  // namespace

int64_t sample_ws_bytes(int M, int V) { return 0; }

int sample(const btf_sampling& a, hipStream_t st, const DevState& ds) {
  hipLaunchKernelGGL(sample_row_kernel, dim3(a.M), dim3(kThreads), 0, st, a);
  return launch_status("sample_row_kernel");
}

}  // namespace btfhip
