// sample.hip -- one token per row of logits with temperature, top-k, top-p and
// min-p from a given uniform number (btf_hip_launch_sample; gfx950).
//
// The kept set is a prefix of the order (falling logit, rising index): a
// threshold in the 64-bit key (logit's bits in an order-preserving form, the
// complement of the index), the greedy pick's key. Weights are whole numbers
// (units of 2^-43, in 64 bits), so no sum depends on its order.
//
// Four launches over the row, cut into parts of 4096 to 16384 logits:
//  * top: the parts' largest key and smallest logit;
//  * hist (rows with top-k or top-p): counts and weights by 1024 bins of the
//    distance to the maximum, in LDS, then added to the row's;
//  * border: from the bins, those in which a border can lie. top-k's is the bin
//    in which the count passes k; top-p's lies between the bins in which the sum
//    passes p times the least and the most that the top-k may weigh. Below them
//    everything stays: its weights are summed part by part. What lies in them is
//    written out, logit and index, as candidates;
//  * pick: one workgroup per row sorts the candidates (a bin of a row of 248320
//    normal logits holds 1500 of them at most), finds the borders exactly, adds
//    what stays to its parts, and walks the one part in which the sum passes u.
// A row whose border bins hold more than kCand logits (many equal ones) is done by
// that workgroup alone, eight key bits at a time.
#include <cmath>
#include <string>

#include "../../include/btf/hip_abi.h"
#include "common.h"
#include "slice.h"

namespace btfhip {
namespace {

typedef unsigned long long u64;
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
constexpr int kPartThreads = 256;
constexpr int kPickThreads = 1024;
constexpr int kBins = 1024;
constexpr int kCand = 4096;
constexpr int kMinPart = 4096, kMaxPart = 16384;  // logits of a part
constexpr double kOne = 8796093022208.0;          // 2^43: the weight of the largest
constexpr double kFar = 31.0;                     // exp(-31) is below half a unit

__device__ __forceinline__ uint32_t key_of(float x) { return (uint32_t)(argmax_key(x, 0) >> 32); }
__device__ __forceinline__ float of_key(uint32_t k) { return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k); }

// exp(-d) in units of 2^-43, for 0 <= d < kFar: with n the nearest whole number to
// -d / ln 2 and r = -d - n ln 2 (ln 2 in two parts), the series of exp(r) up to r^12
// (|r| <= 0.347: 2e-16 off), scaled by its exponent; rounded to a whole number by
// adding 2^52.
__device__ __forceinline__ u64 weight_at(double d) {
  const double n = rint(d * -1.4426950408889634);
  const double r = fma(n, -2.3190468138462996e-17, fma(n, -0.6931471805599453, -d));
  double p = 1.0 / 479001600;
  p = fma(p, r, 1.0 / 39916800);
  p = fma(p, r, 1.0 / 3628800);
  p = fma(p, r, 1.0 / 362880);
  p = fma(p, r, 1.0 / 40320);
  p = fma(p, r, 1.0 / 5040);
  p = fma(p, r, 1.0 / 720);
  p = fma(p, r, 1.0 / 120);
  p = fma(p, r, 1.0 / 24);
  p = fma(p, r, 1.0 / 6);
  p = fma(p, r, 0.5);
  p = fma(p, r, 1.0);
  p = fma(p, r, 1.0);
  const double v = ldexp(p, (int)n + 43) + 4503599627370496.0;
  return (u64)(__double_as_longlong(v) & 0xfffffffffffffll);
}

// Distance of a logit to the row's largest in units of the temperature; kFar or more (or NaN): no weight.
__device__ __forceinline__ double distance(float x, float top, double inv_t) {
  return x == top ? 0.0 : ((double)top - (double)x) * inv_t;
}
__device__ __forceinline__ u64 weight(float x, float top, double inv_t) {
  const double d = distance(x, top, inv_t);
  return d < kFar ? weight_at(d) : 0;
}

// ---- what the launches share: scratch, the row's settings ----
struct Scratch {
  u64 sum[kBins];
  uint32_t cnt[kBins];
  uint32_t cand[kCand][2];  // logit's bits, index
  u64 pmax[256];            // (2^20 / kMinPart parts at most)
  u64 psum[256];
  float pmin[256];
  uint32_t ncand;
  uint32_t pad;
};

struct Row {
  bool greedy;
  float top;
  double inv_t, scale, floor_w;  // scale: bins for a unit of distance
  int k;                         // 0: no top-k
  float p;                       // 1: no top-p
};

struct Parts {
  int n, size;  // size a multiple of 4
};
__host__ __device__ inline Parts parts_of(int M, int V) {
  // about 1024 workgroups over the rows
  int want = (1024 + M - 1) / M;
  int size = (V + want - 1) / want;
  size = size < kMinPart ? kMinPart : size > kMaxPart ? kMaxPart : (size + 3) / 4 * 4;
  return {(V + size - 1) / size, size};
}

// Settings of row m; `best` its largest key. By every thread of the workgroup, which waits here.
__device__ Row settings(const btf_sampling& a, const Scratch& s, int m, int parts, u64* best) {
  u64 b = 0;
  float lo = INFINITY;
  const int lane = threadIdx.x & 63;
  for (int i = lane; i < parts; i += 64) b = key_max(b, s.pmax[i]), lo = fminf(lo, s.pmin[i]);
  b = wave_max_key(b);
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) lo = fminf(lo, __shfl_xor(lo, o, 64));
  Row r;
  const float t = a.temperature ? a.temperature[m] : 1.f;
  r.greedy = !(t > 0.f) || b == 0;
  r.top = of_key((uint32_t)(b >> 32));
  r.inv_t = 1.0 / (double)t;
  const double range = ((double)r.top - (double)lo) * r.inv_t;  // (NaN and infinities: the widest)
  r.scale = (double)kBins / (range > 0.0 && range < 32.0 ? range * 1.000001 : 32.0);
  const int k = a.top_k ? a.top_k[m] : 0;
  r.k = k > 0 && k < a.V ? k : 0;
  const float p = a.top_p ? a.top_p[m] : 1.f;
  r.p = p < 1.f ? p : 1.f;
  const float mp = a.min_p ? a.min_p[m] : 0.f;
  r.floor_w = mp > 0.f ? (double)fminf(mp, 1.f) * kOne : 0.0;
  *best = b;
  return r;
}

__device__ __forceinline__ int bin_of(double d, const Row& r) {
  const int b = (int)(d * r.scale);
  return b < kBins ? b : kBins - 1;
}

// fn(logit, index) over a part, four at a time.
template <class F>
__device__ __forceinline__ void over_part(const float* x, int i0, int i1, F fn) {
  for (int i = i0 + 4 * (int)threadIdx.x; i < i1; i += 4 * kPartThreads) {
    if (i + 4 <= i1) {
      const f32x4u v = *reinterpret_cast<const f32x4u*>(x + i);
#pragma unroll
      for (int j = 0; j < 4; ++j) fn(v[j], i + j);
    } else {
      for (int j = i; j < i1; ++j) fn(x[j], j);
    }
  }
}

// Inclusive prefix sum over the N threads of the workgroup; *total: the whole sum.
template <int N>
__device__ u64 block_scan(u64 v, u64* part, u64* total) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  constexpr int nw = N / 64;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const u64 u = __shfl_up(v, o, 64);
    if (lane >= o) v += u;
  }
  __syncthreads();
  if (lane == 63) part[w] = v;
  __syncthreads();
  u64 sums = lane < nw ? part[lane] : 0;
#pragma unroll
  for (int o = 1; o < nw; o <<= 1) {
    const u64 u = __shfl_up(sums, o, 64);
    if (lane >= o) sums += u;
  }
  const u64 before = w ? __shfl(sums, w - 1, 64) : 0;
  *total = __shfl(sums, nw - 1, 64);
  return v + before;
}

// ---- launches 1 to 3 ----
__global__ void __launch_bounds__(kPartThreads) sample_top_kernel(btf_sampling a, int size) {
  __shared__ u64 wk[kPartThreads / 64];
  __shared__ float wm[kPartThreads / 64];
  const int m = blockIdx.y, i0 = blockIdx.x * size, i1 = min(a.V, i0 + size);
  Scratch& s = static_cast<Scratch*>(a.ws)[m];
  for (int i = blockIdx.x * kPartThreads + threadIdx.x; i < kBins; i += gridDim.x * kPartThreads) s.sum[i] = 0, s.cnt[i] = 0;
  if (blockIdx.x == 0 && threadIdx.x == 0) s.ncand = 0;
  u64 best = 0;
  float lo = INFINITY;
  over_part(a.logits + (size_t)m * a.ldl, i0, i1, [&](float x, int i) {
    best = key_max(best, argmax_key(x, i));
    if (x > -INFINITY) lo = fminf(lo, x);
  });
  best = wave_max_key(best);
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) lo = fminf(lo, __shfl_xor(lo, o, 64));
  if ((threadIdx.x & 63) == 0) wk[threadIdx.x >> 6] = best, wm[threadIdx.x >> 6] = lo;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kPartThreads / 64; ++w) best = key_max(best, wk[w]), lo = fminf(lo, wm[w]);
    s.pmax[blockIdx.x] = best;
    s.pmin[blockIdx.x] = lo;
  }
}

__global__ void __launch_bounds__(kPartThreads) sample_hist_kernel(btf_sampling a, int size) {
  __shared__ u64 sum[kBins];
  __shared__ uint32_t cnt[kBins];
  const int m = blockIdx.y, i0 = blockIdx.x * size, i1 = min(a.V, i0 + size);
  Scratch& s = static_cast<Scratch*>(a.ws)[m];
  u64 best;
  const Row r = settings(a, s, m, gridDim.x, &best);
  if (r.greedy || (r.k == 0 && r.p == 1.f)) return;
  for (int i = threadIdx.x; i < kBins; i += kPartThreads) sum[i] = 0, cnt[i] = 0;
  __syncthreads();
  over_part(a.logits + (size_t)m * a.ldl, i0, i1, [&](float x, int) {
    const double d = distance(x, r.top, r.inv_t);
    if (!(d < kFar)) return;
    const u64 w = weight_at(d);
    if (w == 0) return;
    const int b = bin_of(d, r);
    atomicAdd(&sum[b], w);
    atomicAdd(&cnt[b], 1u);
  });
  __syncthreads();
  for (int i = threadIdx.x; i < kBins; i += kPartThreads)
    if (cnt[i]) {
      atomicAdd(&s.sum[i], sum[i]);
      atomicAdd(&s.cnt[i], cnt[i]);
    }
}

// Where the borders lie, by bins: [0, lo) stays whole; candidates are in [lo, hi] and kb.
struct Borders {
  int lo, hi, kb;         // kBins: none
  uint32_t k_left;        // top-k: how many of bin kb stay
  u64 below_lo, below_kb; // weights of the bins before lo, before kb
};

template <int N>
__device__ Borders borders(const Scratch& s, const Row& r, u64* part, u64* sh) {
  Borders b = {kBins, -1, kBins, 0, 0, 0};
  if (r.k == 0 && r.p == 1.f) return b;
  constexpr int PER = kBins / N > 0 ? kBins / N : 1;
  const int b0 = threadIdx.x * PER;
  u64 c[PER], w[PER], cs = 0, ws = 0, total;
#pragma unroll
  for (int i = 0; i < PER; ++i) cs += c[i] = s.cnt[b0 + i], ws += w[i] = s.sum[b0 + i];
  u64 c0 = block_scan<N>(cs, part, &total) - cs;
  if (threadIdx.x < 8) sh[threadIdx.x] = threadIdx.x < 3 ? kBins : 0;
  u64 all;
  const u64 w0 = block_scan<N>(ws, part, &all) - ws;  // (waits: sh is set)
  if (r.k && total > (u64)r.k) {  // at most k with a weight: top-k takes nothing away
    u64 at = c0, wat = w0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      if (at < (u64)r.k && at + c[i] >= (u64)r.k) sh[0] = b0 + i, sh[3] = r.k - at, sh[4] = wat, sh[5] = wat + w[i];
      at += c[i], wat += w[i];
    }
  }
  __syncthreads();
  b.kb = (int)sh[0];
  b.k_left = (uint32_t)sh[3];
  b.below_kb = b.kb < kBins ? sh[4] : all;
  const u64 upto_kb = b.kb < kBins ? sh[5] : all;
  if (r.p < 1.f) {
    const double least = (double)r.p * (double)b.below_kb, most = (double)r.p * (double)upto_kb;
    u64 at = w0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const bool first = b0 + i == 0;
      const double before = (double)at, after = (double)(at + w[i]);
      if ((first || before < least) && after >= least) sh[1] = b0 + i, sh[6] = at;
      if ((first || before < most) && after >= most) sh[2] = b0 + i;
      at += w[i];
    }
    __syncthreads();
    b.lo = (int)sh[1], b.hi = (int)sh[2], b.below_lo = sh[6];
  } else {
    b.lo = b.hi = b.kb;
    b.below_lo = b.below_kb;
  }
  if (b.hi >= kBins) b.hi = -1;
  return b;
}

__global__ void __launch_bounds__(kPartThreads) sample_border_kernel(btf_sampling a, int size) {
  __shared__ u64 part[kPartThreads / 64], sh[8];
  const int m = blockIdx.y, i0 = blockIdx.x * size, i1 = min(a.V, i0 + size);
  Scratch& s = static_cast<Scratch*>(a.ws)[m];
  u64 best;
  const Row r = settings(a, s, m, gridDim.x, &best);
  if (r.greedy) return;
  const Borders b = borders<kPartThreads>(s, r, part, sh);
  u64 mine = 0;
  over_part(a.logits + (size_t)m * a.ldl, i0, i1, [&](float x, int i) {
    const double d = distance(x, r.top, r.inv_t);
    if (!(d < kFar)) return;
    const int bin = bin_of(d, r);
    if (bin < b.lo) {
      const u64 w = weight_at(d);
      if ((double)w >= r.floor_w) mine += w;
    } else if (bin <= b.hi || bin == b.kb) {
      const uint32_t n = atomicAdd(&s.ncand, 1u);
      if (n < kCand) s.cand[n][0] = __float_as_uint(x), s.cand[n][1] = (uint32_t)i;
    }
  });
  u64 total;
  block_scan<kPartThreads>(mine, part, &total);
  if (threadIdx.x == 0) s.psum[blockIdx.x] = total;
}

// ---- launch 4 ----
struct Pick {
  union {
    struct {
      u64 key[kCand];  // candidates, sorted
      u64 sum[256];    // weights that stay, by parts
    } c;
    struct {
      u64 sum[256];
      uint32_t cnt[256];
      uint32_t prefix, flag;
      u64 s;
    } f;
  };
  u64 part[kPickThreads / 64];
  u64 sh[8];
  u64 kth;
};

// The smallest key at which the count (by_count) or the weight of the logits from
// the largest down reaches `want`, over keys > floor, and what lies above it. False
// if nothing reaches it.
__device__ bool find_key(const float* x, int V, const Row& r, bool by_count, double want, uint32_t floor, Pick& sh,
                         uint32_t* key, u64* above) {
  uint32_t prefix = 0;
  u64 got = 0;
  for (int shift = 24; shift >= 0; shift -= 8) {
    __syncthreads();
    if (threadIdx.x < 256) sh.f.sum[threadIdx.x] = 0, sh.f.cnt[threadIdx.x] = 0;
    if (threadIdx.x == 0) sh.f.flag = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < V; i += kPickThreads) {
      const uint32_t k = key_of(x[i]);
      if (k <= floor || (shift < 24 && (k >> (shift + 8)) != prefix)) continue;
      if (by_count) atomicAdd(&sh.f.cnt[k >> shift & 255], 1u);
      else atomicAdd(&sh.f.sum[k >> shift & 255], weight(x[i], r.top, r.inv_t));
    }
    __syncthreads();
    if (threadIdx.x == 0) {
      u64 s = got;
      for (int b = 255; b >= 0; --b) {
        const u64 v = by_count ? sh.f.cnt[b] : sh.f.sum[b];
        if (v && (double)(s + v) >= want) {
          sh.f.prefix = prefix << 8 | b;
          sh.f.flag = 1;
          break;
        }
        s += v;
      }
      sh.f.s = s;
    }
    __syncthreads();
    got = sh.f.s;
    if (!sh.f.flag) break;
    prefix = sh.f.prefix;
  }
  *above = got;
  *key = prefix;
  const bool found = sh.f.flag != 0;
  __syncthreads();
  return found;
}

// The index at which the sum of the kept weights in [i0, i1) passes `at`, by the whole workgroup; the kept are those
// with keys > key and the first `ties` at it.
__device__ void walk(const btf_sampling& a, const float* x, int m, int i0, int i1, const Row& r, uint32_t key, u64 ties,
                     u64 at, bool relative, Pick& sh, u64 total) {
  const int per = (i1 - i0 + kPickThreads - 1) / kPickThreads;
  const int j0 = min(i1, i0 + (int)threadIdx.x * per), j1 = min(i1, j0 + per);
  u64 eq = 0, n;
  for (int i = j0; i < j1; ++i) eq += key_of(x[i]) == key;
  const u64 eq0 = block_scan<kPickThreads>(eq, sh.part, &n) - eq;
  auto kept = [&](int i, u64& rank) -> u64 {
    const uint32_t kk = key_of(x[i]);
    if (kk < key || kk == 0) return 0;
    if (kk == key && rank++ >= ties) return 0;
    const u64 w = weight(x[i], r.top, r.inv_t);
    return (double)w >= r.floor_w ? w : 0;
  };
  u64 mine = 0, rank = eq0;
  for (int i = j0; i < j1; ++i) mine += kept(i, rank);
  const u64 end = block_scan<kPickThreads>(mine, sh.part, &n);
  if (!relative) {  // the whole row: its sum is the total
    total = n;
    const double u = a.u[m];
    at = u > 0.0 ? (u64)fmin(u * (double)total, 9.0e18) : 0;
    if (at >= total) at = total - 1;
  }
  if (end > at && end - mine <= at) {
    u64 s = end - mine;
    rank = eq0;
    for (int i = j0; i < j1; ++i) {
      const u64 w = kept(i, rank);
      s += w;
      if (s > at) {
        a.token[m] = i;
        if (a.logprob) a.logprob[m] = (float)log((double)w / (double)total);
        break;
      }
    }
  }
}

// A row by one workgroup alone: thresholds eight key bits at a time.
__device__ void pick_alone(const btf_sampling& a, const float* x, int m, const Row& r, Pick& sh) {
  uint32_t key = 0, ties = 0;  // kept: keys > key, and the first `ties` logits at it
  u64 n_above = 0;
  if (r.k && find_key(x, a.V, r, true, r.k, 0, sh, &key, &n_above)) ties = (uint32_t)(r.k - n_above);
  if (r.p < 1.f) {
    u64 mine = 0, total;
    for (int i = threadIdx.x; i < a.V; i += kPickThreads)
      if (key_of(x[i]) > key) mine += weight(x[i], r.top, r.inv_t);
    block_scan<kPickThreads>(mine, sh.part, &total);
    const u64 wt = key ? weight(of_key(key), r.top, r.inv_t) : 0;
    const double want = (double)r.p * (double)(total + ties * wt);
    uint32_t pk;
    u64 above;
    if (find_key(x, a.V, r, false, want, key, sh, &pk, &above)) {
      const double more = ceil((want - (double)above) / (double)weight(of_key(pk), r.top, r.inv_t));
      key = pk;
      ties = more < 1.0 ? 1u : (uint32_t)more;
    } else if (ties) {
      const double more = wt ? ceil((want - (double)total) / (double)wt) : 1.0;
      ties = (uint32_t)fmin((double)ties, fmax(more, 1.0));
    }
  }
  walk(a, x, m, 0, a.V, r, key, ties, 0, false, sh, 0);
}

__global__ void __launch_bounds__(kPickThreads) sample_pick_kernel(btf_sampling a, int parts, int size) {
  __shared__ Pick sh;
  const int m = blockIdx.x, tid = threadIdx.x;
  const float* x = a.logits + (size_t)m * a.ldl;
  const Scratch& s = static_cast<const Scratch*>(a.ws)[m];
  u64 best;
  const Row r = settings(a, s, m, parts, &best);
  if (r.greedy) {
    if (tid == 0) {
      a.token[m] = argmax_key_index(best);
      if (a.logprob) a.logprob[m] = 0.f;
    }
    return;
  }
  const uint32_t n = s.ncand;
  if (n > kCand) {
    pick_alone(a, x, m, r, sh);
    return;
  }
  const Borders b = borders<kPickThreads>(s, r, sh.part, sh.sh);
  // candidates in order, by a bitonic sort of the next power of two of them
  int size2 = 1;
  while (size2 < (int)n) size2 *= 2;
  for (int i = tid; i < size2; i += kPickThreads)
    sh.c.key[i] = i < (int)n ? argmax_key(__uint_as_float(s.cand[i][0]), (int)s.cand[i][1]) : 0;
  if (tid < parts) sh.c.sum[tid] = s.psum[tid];
  if (tid == 0) sh.kth = 0;
  __syncthreads();
  for (int k = 2; k <= size2; k *= 2)
    for (int j = k / 2; j > 0; j /= 2) {
      for (int i = tid; i < size2 / 2; i += kPickThreads) {
        const int lo = 2 * i - (i & (j - 1)), hi = lo + j;  // falling order in the end
        const u64 x0 = sh.c.key[lo], x1 = sh.c.key[hi];
        if ((x0 < x1) == ((lo & k) == 0)) sh.c.key[lo] = x1, sh.c.key[hi] = x0;
      }
      __syncthreads();
    }
  // prefix sums of their weights, four consecutive ones a thread
  constexpr int PER = kCand / kPickThreads;
  u64 w[PER], ws = 0, w_all;
  int bin[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int at = tid * PER + i;
    w[i] = 0, bin[i] = kBins;
    if (at < (int)n) {
      const double d = distance(of_key((uint32_t)(sh.c.key[at] >> 32)), r.top, r.inv_t);
      w[i] = weight_at(d), bin[i] = bin_of(d, r);
    }
    ws += w[i];
  }
  const u64 w0 = block_scan<kPickThreads>(ws, sh.part, &w_all) - ws;
  // top-k: of bin kb the first k_left; its place in the list and the weights before it
  uint32_t n_before = 0, n_stay = n;
  u64 w_top = b.below_kb;  // weights of the top-k
  if (b.kb < kBins) {
    u64 c = 0, n_b, in = 0, w_in;
#pragma unroll
    for (int i = 0; i < PER; ++i) c += bin[i] < b.kb;
    block_scan<kPickThreads>(c, sh.part, &n_b);
    n_before = (uint32_t)n_b;
    n_stay = n_before + b.k_left;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const uint32_t at = tid * PER + i;
      if (at >= n_before && at < n_stay) in += w[i];
    }
    block_scan<kPickThreads>(in, sh.part, &w_in);
    w_top += w_in;
  }
  if (r.p < 1.f) {
    const double want = (double)r.p * (double)w_top;
    u64 c = 0, stay, at = b.below_lo + w0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      // the list is without gaps up to bin hi, behind which nothing stays
      const bool first = b.below_lo == 0 && tid == 0 && i == 0;
      c += bin[i] <= b.hi && (first || (double)at < want);
      at += w[i];
    }
    block_scan<kPickThreads>(c, sh.part, &stay);
    n_stay = min(n_stay, (uint32_t)stay);
  }
  // what stays of them, added to its parts
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const uint32_t at = tid * PER + i;
    if (at >= n_stay) break;
    const int idx = argmax_key_index(sh.c.key[at]);
    if ((double)w[i] >= r.floor_w) atomicAdd(&sh.c.sum[idx / size], w[i]);
    if (at == n_stay - 1) sh.kth = sh.c.key[at];
  }
  __syncthreads();
  // the part in which the sum passes u times the total
  const u64 ps = tid < parts ? sh.c.sum[tid] : 0;
  u64 total;
  const u64 end = block_scan<kPickThreads>(ps, sh.part, &total);
  const double u = a.u[m];
  u64 at = u > 0.0 ? (u64)fmin(u * (double)total, 9.0e18) : 0;
  if (at >= total) at = total - 1;
  if (end > at && end - ps <= at) sh.sh[0] = tid, sh.sh[1] = at - (end - ps);
  __syncthreads();
  const int part = (int)sh.sh[0];
  at = sh.sh[1];
  const u64 kth = sh.kth;  // the last that stays; 0: all of the bins before lo, and nothing else
  // walk the part: 16 logits a thread at most
  const int i0 = part * size, i1 = min(a.V, i0 + size);
  const int per = (i1 - i0 + kPickThreads - 1) / kPickThreads;
  const int j0 = min(i1, i0 + tid * per), j1 = min(i1, j0 + per);
  auto kept = [&](int i) -> u64 {
    const float v = x[i];
    const double d = distance(v, r.top, r.inv_t);
    if (!(d < kFar)) return 0;
    if (bin_of(d, r) >= b.lo && !(kth && argmax_key(v, i) >= kth)) return 0;
    const u64 wt = weight_at(d);
    return (double)wt >= r.floor_w ? wt : 0;
  };
  u64 mine = 0, all;
  for (int i = j0; i < j1; ++i) mine += kept(i);
  const u64 upto = block_scan<kPickThreads>(mine, sh.part, &all);
  if (upto > at && upto - mine <= at) {
    u64 sum = upto - mine;
    for (int i = j0; i < j1; ++i) {
      const u64 wt = kept(i);
      sum += wt;
      if (sum > at) {
        a.token[m] = i;
        if (a.logprob) a.logprob[m] = (float)log((double)wt / (double)total);
        break;
      }
    }
  }
}

}  // namespace

int64_t sample_ws_bytes(int M, int V) { return (int64_t)M * (int64_t)sizeof(Scratch); }

int sample(const btf_sampling& a, hipStream_t st, const DevState& ds) {
  const Parts p = parts_of(a.M, a.V);
  for (int m0 = 0; m0 < a.M; m0 += 65535) {  // (rows are the grid's second dimension)
    btf_sampling b = a;
    const int M = a.M - m0 < 65535 ? a.M - m0 : 65535;
    b.logits += (size_t)m0 * a.ldl;
    if (a.temperature) b.temperature += m0;
    if (a.top_k) b.top_k += m0;
    if (a.top_p) b.top_p += m0;
    if (a.min_p) b.min_p += m0;
    b.u += m0;
    b.token += m0;
    if (a.logprob) b.logprob += m0;
    b.ws = static_cast<Scratch*>(a.ws) + m0;
    const dim3 grid(p.n, M), blk(kPartThreads);
    hipLaunchKernelGGL(sample_top_kernel, grid, blk, 0, st, b, p.size);
    int rc = launch_status("sample_top_kernel");
    if (rc != BTF_OK) return rc;
    if (a.top_k || a.top_p) {
      hipLaunchKernelGGL(sample_hist_kernel, grid, blk, 0, st, b, p.size);
      if ((rc = launch_status("sample_hist_kernel")) != BTF_OK) return rc;
    }
    hipLaunchKernelGGL(sample_border_kernel, grid, blk, 0, st, b, p.size);
    if ((rc = launch_status("sample_border_kernel")) != BTF_OK) return rc;
    hipLaunchKernelGGL(sample_pick_kernel, dim3(M), dim3(kPickThreads), 0, st, b, p.n, p.size);
    if ((rc = launch_status("sample_pick_kernel")) != BTF_OK) return rc;
  }
  return BTF_OK;
}

}  // namespace btfhip
