// sample.hip -- one token per row of logits with temperature, top-k, top-p and
// min-p from a given uniform number (btf_hip_launch_sample; gfx950).
//
// The kept set is a prefix of the order (falling logit, rising index): a
// threshold in the 64-bit key (logit's bits in an order-preserving form, the
// complement of the index), the greedy pick's key. Weights are whole numbers
// (units of 2^-43, in 64 bits), so no sum depends on its order.
//
// Four launches over the row, cut into parts of 2048 to 16384 logits:
//  * top: the parts' largest key and smallest logit, and the largest key of every 128
//    logits, by which the next launches skip what lies below all that they look for;
//  * hist (rows with top-k or top-p): weights (top-p) and counts (top-k) by 1024 bins
//    of the distance to the maximum, in LDS, then added to the row's. With top-k only
//    the bins down to the one in which the k-th largest of the maxima lies: k logits
//    are at least as large. The row's last workgroup finds from the bins those in which
//    a border can lie: top-k's is the bin in which the count passes k; top-p's lies
//    between the bins in which the sum passes p times the least and the most that the
//    top-k may weigh;
//  * border: below those bins everything stays: its weights are summed for every 256
//    logits. What lies in them is written out, logit and index, as candidates;
//  * pick: one workgroup per row puts the candidates in order (a bin of a row of 248320
//    normal logits spread over less than 32 temperatures holds 1500 at most), finds the borders exactly, adds
//    what stays to its 256 logits, and walks those in which the sum passes u.
// A row whose border bins hold more than kCand logits (many equal ones, or a
// flat row beside one logit far below, which makes the bins 1/32 of the temperature wide)
// is done by that workgroup alone, eight key bits at a time: right, and slow (248320
// normal logits at temperature 2, one of -10^4, top-p 0.7: 1.0 ms instead of 30 us).
//
// What bounds it: one row waits, for four launches and the chain of reads in each (248320
// logits: 19 to 25 us a call; on the GPU top 3.6, hist 8.4, border 4.3, pick 6.3). Many rows read the logits three
// times, 10 us a pass for 48 rows of 248320 at the copy rate, and where there is no top-k work
// out every logit's weight in each of two (36 vector instructions): 59 us (top 12.3, hist 20.9,
// border 14.5, pick 9.2).
#include <cmath>
#include <string>

#include "../../include/btf/hip_abi.h"
#include "common.h"
#include "slice.h"

namespace btfhip {
namespace {

typedef uint64_t u64;
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
constexpr int kPartThreads = 256;
constexpr int kPickThreads = 512;
constexpr int kBins = 1024;
constexpr int kCand = 4096;
constexpr int kFine = 512;                        // pieces of a border bin
constexpr int kMinPart = 2048, kMaxPart = 16384;  // logits of a part
constexpr int kRound = 4 * kPartThreads;          // logits of a part's round, four a thread
constexpr int kSum = 256, kTop = 128;             // logits of a partial sum (a wave's of a round), of a maximum (half of it)
constexpr int kMaxV = 1 << 20;
constexpr double kOne = 8796093022208.0;          // 2^43: the weight of the largest
constexpr double kFar = 31.0;                     // exp(-31) is below half a unit
constexpr double kMost = 1.8e19;                  // above 2^20 weights of one, and fits 64 bits

__device__ __forceinline__ uint32_t key_of(float x) { return (uint32_t)(argmax_key(x, 0) >> 32); }
__device__ __forceinline__ float of_key(uint32_t k) { return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k); }

// exp(-d) in units of 2^-43 as a whole number plus 2^52 (its low 52 bits), for d >= 0 (no units from 30.6 on, and for
// NaN): with n the nearest whole number to -d / ln 2 and r = -d - n ln 2 (ln 2 in two parts), the polynomial of degree 9
// that agrees with exp at the Chebyshev points of |r| <= ln 2 / 2 (2e-14 off, a third of the unit's half) times 2^43,
// scaled by 2^n in its exponent. Whole numbers come from adding 2^52 and 1.5 2^52: products and sums run at full rate,
// conversions and the rounding instruction do not.
constexpr double kWhole = 4503599627370496.0;
__device__ __forceinline__ double weight_bits(double d) {
  d = fmin(d, 64.0);
  const double t = fma(d, -1.4426950408889634, 1.5 * kWhole);
  const double n = t - 1.5 * kWhole;
  const double r = fma(n, -2.3190468138462996e-17, fma(n, -0.6931471805599453, -d));
  double p = kOne * 2.7632640690513381e-06;
  p = fma(p, r, kOne * 2.4884459768350122e-05);
  p = fma(p, r, kOne * 0.00019841190647512536);
  p = fma(p, r, kOne * 0.0013888801749621653);
  p = fma(p, r, kOne * 0.0083333333673116239);
  p = fma(p, r, kOne * 0.041666667040552129);
  p = fma(p, r, kOne * 0.16666666666615648);
  p = fma(p, r, kOne * 0.49999999999438588);
  p = fma(p, r, kOne * 1.0000000000000013);
  p = fma(p, r, kOne * 1.0000000000000135);
  const u64 b = (u64)__double_as_longlong(p) + ((u64)(uint32_t)__double_as_longlong(t) << 52);
  return __longlong_as_double((long long)b) + kWhole;
}
__device__ __forceinline__ u64 low52(double v) { return (u64)__double_as_longlong(v) & 0xfffffffffffffull; }
__device__ __forceinline__ u64 whole(double v) { return low52(v + kWhole); }  // of a whole number below 2^52
__device__ __forceinline__ u64 weight_at(double d) { return low52(weight_bits(d)); }

// Distance of a logit to the row's largest in units of the temperature; kFar or more (or NaN): no weight.
__device__ __forceinline__ double distance(float x, float top, double inv_t) {
  return x == top ? 0.0 : ((double)top - (double)x) * inv_t;
}
// The same for the data passes, without its comparison: where the largest is infinite, `finite` makes the logits equal to
// it 0 and the others NaN, and the largest 0.
__device__ __forceinline__ f32x4u finite(f32x4u x, float top) {
  if (fabsf(top) == INFINITY)
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = x[j] == top ? 0.f : NAN;
  return x;
}
__device__ __forceinline__ u64 weight(float x, float top, double inv_t) {
  const double d = distance(x, top, inv_t);
  return d < kFar ? weight_at(d) : 0;
}

// ---- what the launches share: scratch, the row's settings ----
struct Row {
  bool greedy;
  float top;
  double inv_t, scale;           // scale: bins for a unit of distance
  u64 floor_w;                   // the least weight that min-p keeps
  int k;                         // 0: no top-k
  float p;                       // 1: no top-p
};

// The same in every lane, which the compiler does not know of what it loads.
__device__ __forceinline__ uint32_t same(uint32_t v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ u64 same(u64 v) { return (u64)same((uint32_t)(v >> 32)) << 32 | same((uint32_t)v); }
__device__ __forceinline__ double same(double v) { return __longlong_as_double((long long)same((u64)__double_as_longlong(v))); }
__device__ __forceinline__ Row same(const Row& r) {
  return {(bool)same((uint32_t)r.greedy), __uint_as_float(same(__float_as_uint(r.top))), same(r.inv_t), same(r.scale),
          same(r.floor_w), (int)same((uint32_t)r.k), __uint_as_float(same(__float_as_uint(r.p)))};
}

// Where the borders lie, by bins: [0, lo) stays whole; candidates are in [lo, hi] and kb.
struct Borders {
  int lo, hi, kb;         // kBins: none
  uint32_t k_left;        // top-k: how many of bin kb stay
  u64 below_lo, below_kb; // weights of the bins before lo, before kb
};
__device__ __forceinline__ Borders same(const Borders& b) {
  return {(int)same((uint32_t)b.lo), (int)same((uint32_t)b.hi), (int)same((uint32_t)b.kb), same(b.k_left), same(b.below_lo),
          same(b.below_kb)};
}

struct Scratch {
  u64 sum[kBins];
  uint32_t cnt[kBins];
  uint32_t cand[kCand][2];  // logit's bits, index
  u64 pmax[kMaxV / kMinPart];
  float pmin[kMaxV / kMinPart];
  uint32_t ncand;
  uint32_t done;            // workgroups of the row that have added their bins
  Row row;
  u64 best;                 // the row's largest key
  Borders borders;
  // then u64 psum[V / kSum], uint32_t tops[V / kTop] (rounded up)
  __device__ u64* psum() { return reinterpret_cast<u64*>(this + 1); }
  __device__ uint32_t* tops(int V) { return reinterpret_cast<uint32_t*>(psum() + (V + kSum - 1) / kSum); }
};
__host__ __device__ inline int64_t scratch_bytes(int V) {
  return (int64_t)sizeof(Scratch) + 8 * (int64_t)((V + kSum - 1) / kSum) + 8 * (int64_t)((V + 2 * kTop - 1) / (2 * kTop));
}
__device__ __forceinline__ Scratch& scratch_of(const btf_sampling& a, int m) {
  return *reinterpret_cast<Scratch*>(static_cast<char*>(a.ws) + (size_t)m * scratch_bytes(a.V));
}

struct Parts {
  int n, size;  // size a multiple of kRound
};
__host__ __device__ inline Parts parts_of(int M, int V) {
  // about 2048 workgroups over the rows: eight to a CU, as many as there is room for (48 rows of 248320 in 64.9 us with
  // 1024, 59.1 with 2048, 59.7 with 2560; 130 of 50257 in 50.1, 45.6 and 46.5)
  int want = (2048 + M - 1) / M;
  int size = (V + want - 1) / want;
  size = size < kMinPart ? kMinPart : size > kMaxPart ? kMaxPart : (size + kRound - 1) / kRound * kRound;
  return {(V + size - 1) / size, size};
}

// Smallest of the wave, in every lane.
__device__ __forceinline__ float wave_min(float v) {
  auto at = [&](int x) { return __int_as_float(x); };
  v = fminf(v, at(dpp_i<0xB1>(__float_as_int(v))));
  v = fminf(v, at(dpp_i<0x4E>(__float_as_int(v))));
  v = fminf(v, at(dpp_i<0x141>(__float_as_int(v))));
  v = fminf(v, at(dpp_i<0x140>(__float_as_int(v))));
  auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fminf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fminf(__uint_as_float(a[0]), __uint_as_float(a[1]));
}

// Settings of row m; `best` its largest key. By every thread of the workgroup, which waits here.
__device__ Row settings(const btf_sampling& a, const Scratch& s, int m, int parts, u64* best) {
  u64 b = 0;
  float lo = INFINITY;
  const int lane = threadIdx.x & 63;
  for (int i = lane; i < parts; i += 64) b = key_max(b, s.pmax[i]), lo = fminf(lo, s.pmin[i]);
  b = wave_max_key(b);
  lo = wave_min(lo);
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
  r.floor_w = mp > 0.f ? (u64)ceil((double)fminf(mp, 1.f) * kOne) : 1;
  *best = b;
  return r;
}

__device__ __forceinline__ int bin_of(double d, const Row& r) {
  const int b = (int)(d * r.scale);
  return b < kBins ? b : kBins - 1;
}

// A logit below which every bin is deeper than `bin`: what a row's bulk is skipped by, without the 64-bit distance.
// (Less by more than the roundings of the distance and its bin.)
__device__ __forceinline__ float cut_below(int bin, const Row& r) {
  const double c = (double)r.top - (double)(bin + 1) / r.scale / r.inv_t * (1.0 + 1e-9);
  return __double2float_rd(c - fabs(c) * 1e-12);  // (NaN, nothing skipped, where the maximum is infinite)
}

// Rounds of part [i0, i1) in which the wave's 256 logits hold one that is not below `cut`, by the maxima of 128: bit 2 r
// for round r. By whole waves.
constexpr uint32_t kAllRounds = 0x55555555u;
static_assert(kMaxPart / kRound <= 16, "two bits a round");
__device__ __forceinline__ uint32_t rounds_from(const uint32_t* top, int i0, int i1, float cut) {
  const int lane = threadIdx.x & 63, i = i0 + (lane >> 1) * kRound + (threadIdx.x >> 6) * kSum + (lane & 1) * kTop;
  bool live = false;
  if (i < i1) {
    const uint32_t k = top[i / kTop];
    live = k != 0 && !(of_key(k) < cut);
  }
  const uint32_t b = (uint32_t)__ballot(live);
  return (b | b >> 1) & kAllRounds;
}

// fn(the thread's four logits, their indices, how many there are; NaN behind them) for the rounds of a part that `rounds`
// names, by whole waves.
template <class F>
__device__ __forceinline__ void over_part(const float* x, int i0, int i1, uint32_t rounds, F fn) {
  constexpr int AHEAD = 2;  // rounds whose loads are on their way together
  rounds &= (uint32_t)((1ull << 2 * ((i1 - i0 + kRound - 1) / kRound)) - 1);
  while (rounds) {
    f32x4u v[AHEAD];
    int n[AHEAD], at[AHEAD];
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      v[k] = f32x4u{NAN, NAN, NAN, NAN};
      n[k] = 0, at[k] = i1;
      if (!rounds) continue;
      const int i = at[k] = i0 + (__builtin_ctz(rounds) >> 1) * kRound + 4 * (int)threadIdx.x;
      rounds &= rounds - 1;
      n[k] = min(4, i1 - i);
      if (n[k] == 4) v[k] = *reinterpret_cast<const f32x4u*>(x + i);
      else
        for (int j = 0; j < 3; ++j)
          if (j < n[k]) v[k][j] = x[i + j];
    }
#pragma unroll
    for (int k = 0; k < AHEAD; ++k)
      if (__any(n[k] > 0)) fn(v[k], at[k], n[k]);
  }
}

// Sum over the wave, in every lane. (Halves by DPP within 16 lanes, then the row swaps.)
__device__ __forceinline__ double wave_sum_f64(double v) {
  auto half = [&](int h) { return h ? (int)((u64)__double_as_longlong(v) >> 32) : (int)__double_as_longlong(v); };
  auto join = [](uint32_t lo, uint32_t hi) { return __longlong_as_double((long long)((u64)hi << 32 | lo)); };
  v += join(dpp_i<0xB1>(half(0)), dpp_i<0xB1>(half(1)));
  v += join(dpp_i<0x4E>(half(0)), dpp_i<0x4E>(half(1)));
  v += join(dpp_i<0x141>(half(0)), dpp_i<0x141>(half(1)));
  v += join(dpp_i<0x140>(half(0)), dpp_i<0x140>(half(1)));
  {
    const auto a = __builtin_amdgcn_permlane16_swap(half(0), half(0), false, false);
    const auto b = __builtin_amdgcn_permlane16_swap(half(1), half(1), false, false);
    v = join(a[0], b[0]) + join(a[1], b[1]);
  }
  const auto a = __builtin_amdgcn_permlane32_swap(half(0), half(0), false, false);
  const auto b = __builtin_amdgcn_permlane32_swap(half(1), half(1), false, false);
  return join(a[0], b[0]) + join(a[1], b[1]);
}
// Largest of each half of the wave, in its lanes.
__device__ __forceinline__ uint32_t half_max(uint32_t v) {
  v = max(v, (uint32_t)dpp_i<0xB1>((int)v));
  v = max(v, (uint32_t)dpp_i<0x4E>((int)v));
  v = max(v, (uint32_t)dpp_i<0x141>((int)v));
  v = max(v, (uint32_t)dpp_i<0x140>((int)v));
  const auto a = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  return max(a[0], a[1]);
}

// ---- launches 1 to 3 ----
__global__ void __launch_bounds__(kPartThreads) sample_top_kernel(btf_sampling a, int size) {
  __shared__ u64 wk[kPartThreads / 64];
  __shared__ float wm[kPartThreads / 64];
  const int m = blockIdx.y, i0 = blockIdx.x * size, i1 = min(a.V, i0 + size);
  Scratch& s = scratch_of(a, m);
  for (int i = blockIdx.x * kPartThreads + threadIdx.x; i < kBins; i += gridDim.x * kPartThreads) s.sum[i] = 0, s.cnt[i] = 0;
  if (blockIdx.x == 0 && threadIdx.x == 0) s.ncand = 0, s.done = 0;
  const bool tops = a.top_k || a.top_p;  // what the next launches skip by
  uint32_t* top = s.tops(a.V);
  const float* x0 = a.logits + (size_t)m * a.ldl;
  // Four logits at a time: their largest as a key, their smallest, and where the thread's largest key came first; its
  // index is found at the end.
  uint32_t most = 0;
  int at = 0;
  float lo = INFINITY;
  over_part(x0, i0, i1, kAllRounds, [&](f32x4u x, int i, int n) {
    uint32_t k = key_of(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])));
    float least = fminf(fminf(x[0], x[1]), fminf(x[2], x[3]));
    if (__any(least == -INFINITY)) {
      least = INFINITY;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (x[j] > -INFINITY) least = fminf(least, x[j]);
    }
    lo = fminf(lo, least);
    if (k > most) most = k, at = i;
    if (tops) {
      k = half_max(k);
      if ((threadIdx.x & 31) == 0 && n > 0) top[i / kTop] = k;
    }
  });
  u64 best = 0;
  if (most) {
    const float v = of_key(most);
    int j = 0;
    while (j < 3 && !(x0[at + j] == v)) ++j;  // (one of the four is it)
    best = (u64)most << 32 | (uint32_t)~(uint32_t)(at + j);
  }
  best = wave_max_key(best);
  lo = wave_min(lo);
  if ((threadIdx.x & 63) == 0) wk[threadIdx.x >> 6] = best, wm[threadIdx.x >> 6] = lo;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kPartThreads / 64; ++w) best = key_max(best, wk[w]), lo = fminf(lo, wm[w]);
    s.pmax[blockIdx.x] = best;
    s.pmin[blockIdx.x] = lo;
  }
}

// The borders of a row whose bins are complete, by the whole workgroup. (The bins come from other workgroups of this
// launch: they are read past the caches that those may not share.)
template <int N>
__device__ Borders borders(Scratch& s, const Row& r, u64* part, u64* sh) {
  Borders b = {kBins, -1, kBins, 0, 0, 0};
  if (r.k == 0 && r.p == 1.f) return b;
  constexpr int PER = kBins / N > 0 ? kBins / N : 1;
  const int b0 = threadIdx.x * PER;
  u64 c[PER], w[PER], cs = 0, ws = 0, total;
#pragma unroll
  for (int i = 0; i < PER; ++i) cs += c[i] = __hip_atomic_load(&s.cnt[b0 + i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT),
                                    ws += w[i] = __hip_atomic_load(&s.sum[b0 + i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  u64 c0 = block_scan<N>(cs, part, &total) - cs;
  if (threadIdx.x < 8) sh[threadIdx.x] = threadIdx.x < 3 ? kBins : 0;
  u64 all;
  const u64 w0 = block_scan<N>(ws, part, &all) - ws;  // (waits: sh is set)
  // (Without top-k there are no counts, without top-p no weights; with top-k both stop at a bin that it does reach. Less
  // than k in all: fewer than k have a weight, and top-k takes nothing away.)
  if (r.k && total >= (u64)r.k) {
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

__global__ void __launch_bounds__(kPartThreads) sample_hist_kernel(btf_sampling a, int size) {
  __shared__ u64 sum[kBins];
  __shared__ uint32_t cnt[kBins];
  __shared__ u64 part[kPartThreads / 64];
  __shared__ u64 sh[8];
  __shared__ int deepest;
  __shared__ bool last;
  const int m = blockIdx.y, i0 = blockIdx.x * size, i1 = min(a.V, i0 + size);
  Scratch& s = scratch_of(a, m);
  // (the first maxima are on their way while the settings are worked out)
  const uint32_t* top = s.tops(a.V);
  const int nt = (a.V + kTop - 1) / kTop;
  uint32_t t[8] = {};
  auto fetch = [&](int i) {
#pragma unroll
    for (int j = 0; j < 8; ++j) t[j] = i + j * kPartThreads < nt ? top[i + j * kPartThreads] : 0;
  };
  if (a.top_k && a.top_k[m] > 0) fetch(threadIdx.x);
  u64 best;
  const Row r = same(settings(a, s, m, gridDim.x, &best));
  if (r.greedy || (r.k == 0 && r.p == 1.f)) {
    if (blockIdx.x == 0 && threadIdx.x == 0) s.row = r, s.best = best, s.borders = Borders{kBins, -1, kBins, 0, 0, 0};
    return;
  }
  for (int i = threadIdx.x; i < kBins; i += kPartThreads) sum[i] = 0, cnt[i] = 0;
  if (threadIdx.x == 0) deepest = kBins - 1;
  __syncthreads();
  const bool weigh = r.p < 1.f;
  int deep = kBins - 1;
  if (r.k) {  // the deepest bin that top-k reaches, by the maxima of 128
    if (r.k < nt) {
      // (the maxima of 1024 logits, in eight places, where there are twice as many of them as top-k keeps, or more: an
      // eighth of the work of those of 128, and hardly deeper)
      const bool by8 = 2 * r.k <= nt / 8;
      auto count = [&](uint32_t k) {
        const double d = distance(of_key(k), r.top, r.inv_t);
        if (k && d < kFar) atomicAdd(&cnt[bin_of(d, r)], 1u);
      };
      for (int i = threadIdx.x; i < nt; i += 8 * kPartThreads) {
        if (i >= 8 * kPartThreads) fetch(i);
        if (by8) {
          count(max(max(max(t[0], t[1]), max(t[2], t[3])), max(max(t[4], t[5]), max(t[6], t[7]))));
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) count(t[j]);
        }
      }
      __syncthreads();
      constexpr int PER = kBins / kPartThreads;
      u64 c[PER], mine = 0, total;
#pragma unroll
      for (int i = 0; i < PER; ++i) mine += c[i] = cnt[threadIdx.x * PER + i];
      u64 at = block_scan<kPartThreads>(mine, part, &total) - mine;
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        if (at < (u64)r.k && at + c[i] >= (u64)r.k) deepest = threadIdx.x * PER + i;
        at += c[i];
        cnt[threadIdx.x * PER + i] = 0;
      }
      __syncthreads();
      deep = deepest;
    }
  }
  const float cut = cut_below(deep, r);
  const double top0 = fabsf(r.top) == INFINITY ? 0.0 : (double)r.top;
  const uint32_t rounds = deep < kBins - 1 ? rounds_from(top, i0, i1, cut) : kAllRounds;
  over_part(a.logits + (size_t)m * a.ldl, i0, i1, rounds, [&](f32x4u x, int, int) {
    if (!__any(!(x[0] < cut) | !(x[1] < cut) | !(x[2] < cut) | !(x[3] < cut))) return;
    x = finite(x, r.top);
    u64 w[4];
    int bin[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {  // (without branches, so that the four go through the arithmetic together)
      const double d = fmin((top0 - (double)x[j]) * r.inv_t, 64.0);
      w[j] = weight_at(d);
      bin[j] = bin_of(d, r);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (!((w[j] != 0) & (bin[j] <= deep))) continue;
      if (weigh) atomicAdd(reinterpret_cast<unsigned long long*>(&sum[bin[j]]), (unsigned long long)w[j]);
      if (r.k) atomicAdd(&cnt[bin[j]], 1u);
    }
  });
  __syncthreads();
  for (int i = threadIdx.x; i < kBins; i += kPartThreads) {
    if (sum[i]) atomicAdd(reinterpret_cast<unsigned long long*>(&s.sum[i]), (unsigned long long)sum[i]);
    if (cnt[i]) atomicAdd(&s.cnt[i], cnt[i]);
  }
  // The row's last workgroup finds the borders for the launches that follow. What it reads of the others is the bins
  // alone, and those only ever change by atomics, which are done in memory when the wait below ends: no cache has to be
  // written back (with a fence in every workgroup this launch took 70 us instead of 20 on 48 rows of 248320).
  asm volatile("s_waitcnt vmcnt(0)" : : : "memory");
  __syncthreads();
  if (threadIdx.x == 0) last = __hip_atomic_fetch_add(&s.done, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == gridDim.x - 1;
  __syncthreads();
  if (!last) return;
  const Borders b = borders<kPartThreads>(s, r, part, sh);
  if (threadIdx.x == 0) s.row = r, s.best = best, s.borders = b;
}

__global__ void __launch_bounds__(kPartThreads) sample_border_kernel(btf_sampling a, int size) {
  constexpr int kHere = 1024;  // candidates of a part collected in LDS
  __shared__ uint32_t cand[kHere][2];
  __shared__ uint32_t n_cand, at;
  const int m = blockIdx.y, i0 = blockIdx.x * size, i1 = min(a.V, i0 + size);
  Scratch& s = scratch_of(a, m);
  u64 best;
  Row r;
  Borders b = {kBins, -1, kBins, 0, 0, 0};
  if (a.top_k || a.top_p) {
    r = same(s.row), b = same(s.borders);
  } else {  // no launch before this one has found them
    r = same(settings(a, s, m, gridDim.x, &best));
    if (blockIdx.x == 0 && threadIdx.x == 0) s.row = r, s.best = best, s.borders = b;
  }
  if (r.greedy) return;
  if (threadIdx.x == 0) n_cand = 0;
  __syncthreads();
  u64* psum = s.psum();
  const float cut = cut_below(b.lo < kBins ? max(b.hi, b.kb < kBins ? b.kb : 0) : kBins - 1, r);
  // In units of bins: what is below lo stays, candidates are below end
  const double top0 = fabsf(r.top) == INFINITY ? 0.0 : (double)r.top, floor_w = (double)r.floor_w;
  const int deep = max(b.hi, b.kb < kBins ? b.kb : -1);
  const double lo = b.lo < kBins ? (double)b.lo : INFINITY, end = fmin(deep < kBins - 1 ? (double)(deep + 1) : INFINITY, kFar * r.scale);
  uint32_t rounds = kAllRounds;
  if (b.lo < kBins) {
    rounds = rounds_from(s.tops(a.V), i0, i1, cut);
    const int lane = threadIdx.x & 63, i = i0 + lane * kRound + (threadIdx.x >> 6) * kSum;  // a lane for each round
    if (lane < kMaxPart / kRound && i < i1 && !(rounds >> 2 * lane & 1)) psum[i / kSum] = 0;
  }
  over_part(a.logits + (size_t)m * a.ldl, i0, i1, rounds, [&](f32x4u x, int i, int n) {
    double mine = 0.0;  // (whole numbers; 256 of them stay below 2^52)
    if (__any(!(x[0] < cut) | !(x[1] < cut) | !(x[2] < cut) | !(x[3] < cut))) {
      const f32x4u y = finite(x, r.top);
      double d[4];
      bool stays[4], any = false, cands = false;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        d[j] = fmin((top0 - (double)y[j]) * r.inv_t, 64.0);
        const double at = d[j] * r.scale;
        stays[j] = at < lo;
        any |= stays[j];
        cands |= !stays[j] & (at < end);
      }
      if (__any(any))
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const double w = weight_bits(d[j]) - kWhole;
          mine += (stays[j] & (w >= floor_w)) ? w : 0.0;
        }
      if (cands)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int bin = bin_of(d[j], r);
          if (stays[j] | !(d[j] * r.scale < end) | !((bin <= b.hi) | (bin == b.kb))) continue;
          const uint32_t k = atomicAdd(&n_cand, 1u);
          if (k < kHere) {
            cand[k][0] = __float_as_uint(x[j]), cand[k][1] = (uint32_t)(i + j);
          } else {  // (more than a part's share)
            const uint32_t g = atomicAdd(&s.ncand, 1u);
            if (g < kCand) s.cand[g][0] = __float_as_uint(x[j]), s.cand[g][1] = (uint32_t)(i + j);
          }
        }
    }
    if (__any(mine != 0.0)) mine = wave_sum_f64(mine);
    if ((threadIdx.x & 63) == 0 && n > 0) psum[i / kSum] = whole(mine);
  });
  __syncthreads();
  const uint32_t here = min(n_cand, (uint32_t)kHere);
  if (here == 0) return;
  if (threadIdx.x == 0) at = atomicAdd(&s.ncand, here);
  __syncthreads();
  for (uint32_t k = threadIdx.x; k < here; k += kPartThreads)
    if (at + k < kCand) s.cand[at + k][0] = cand[k][0], s.cand[at + k][1] = cand[k][1];
}

// ---- launch 4 ----
struct Pick {
  union {
    struct {
      u64 key[kCand];           // candidates, sorted
      u64 sum[kMaxV / kSum];    // weights that stay, of every kSum logits
      u64 fine[kFine];          // counts or weights of a border bin's pieces
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
  uint32_t n, before;
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
      else atomicAdd(reinterpret_cast<unsigned long long*>(&sh.f.sum[k >> shift & 255]),
                     (unsigned long long)weight(x[i], r.top, r.inv_t));
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

// Draws from a row whose kept logits are those with keys > key and the first `ties` at it, a piece of it a thread.
__device__ void walk(const btf_sampling& a, const float* x, int m, const Row& r, uint32_t key, u64 ties, Pick& sh) {
  const int per = (a.V + kPickThreads - 1) / kPickThreads;
  const int j0 = min(a.V, (int)threadIdx.x * per), j1 = min(a.V, j0 + per);
  u64 eq = 0, n, total;
  for (int i = j0; i < j1; ++i) eq += key_of(x[i]) == key;
  const u64 eq0 = block_scan<kPickThreads>(eq, sh.part, &n) - eq;
  auto kept = [&](int i, u64& rank) -> u64 {
    const uint32_t kk = key_of(x[i]);
    if (kk < key || kk == 0) return 0;
    if (kk == key && rank++ >= ties) return 0;
    const u64 w = weight(x[i], r.top, r.inv_t);
    return w >= r.floor_w ? w : 0;
  };
  u64 mine = 0, rank = eq0;
  for (int i = j0; i < j1; ++i) mine += kept(i, rank);
  const u64 end = block_scan<kPickThreads>(mine, sh.part, &total);
  const double u = a.u[m];
  u64 at = u > 0.0 ? (u64)fmin(u * (double)total, kMost) : 0;
  if (at >= total) at = total - 1;
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
  walk(a, x, m, r, key, ties, sh);
}

// The borders in the sorted candidates, PER consecutive ones a thread: what stays of them is added to its parts.
template <int PER>
__device__ __forceinline__ void pick_borders(Pick& sh, const Row& r, const Borders& b, uint32_t n) {
  const uint32_t at0 = threadIdx.x * PER;
  u64 w[PER], ws = 0, all, key[PER];
  int bin[PER];
  uint32_t before = 0;  // bins before top-k's border
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    w[i] = 0, bin[i] = kBins, key[i] = 0;
    if (at0 + i < n) {
      key[i] = sh.c.key[at0 + i];
      const double d = distance(of_key((uint32_t)(key[i] >> 32)), r.top, r.inv_t);
      w[i] = weight_at(d), bin[i] = bin_of(d, r);
    }
    ws += w[i];
    before += bin[i] < b.kb && at0 + i < n;
  }
  const bool by_k = b.kb < kBins;
  if (by_k && before) atomicAdd(&sh.before, before);
  const u64 w0 = block_scan<kPickThreads>(ws, sh.part, &all) - ws;  // (waits: sh.before is complete)
  // top-k: of bin kb the first k_left, and the weights of the top-k
  uint32_t n_stay = n;
  u64 w_top = b.below_kb;
  if (by_k) {
    const uint32_t n_before = sh.before;
    n_stay = n_before + b.k_left;
    u64 at = w0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      if (at0 + i == n_before) sh.sh[2] = at;
      at += w[i];
      if (at0 + i + 1 == n_stay) sh.sh[3] = at;
    }
    __syncthreads();  // (n_before < n_stay <= n: both are set)
    w_top += sh.sh[3] - sh.sh[2];
  }
  if (r.p < 1.f) {
    const double want = (double)r.p * (double)w_top;
    u64 at = b.below_lo + w0;
    uint32_t stay = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      // the list is without gaps up to bin hi, behind which nothing stays
      const bool first = b.below_lo == 0 && at0 + i == 0;
      stay += at0 + i < n && bin[i] <= b.hi && (first || (double)at < want);
      at += w[i];
    }
    u64 sum;
    block_scan<kPickThreads>(stay, sh.part, &sum);
    n_stay = min(n_stay, (uint32_t)sum);
  }
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    if (at0 + i >= n_stay) break;
    const int idx = argmax_key_index(key[i]);
    if (w[i] >= r.floor_w) atomicAdd(reinterpret_cast<unsigned long long*>(&sh.c.sum[idx / kSum]), (unsigned long long)w[i]);
    if (at0 + i == n_stay - 1) sh.kth = key[i];
  }
  __syncthreads();
}

__global__ void __launch_bounds__(kPickThreads) sample_pick_kernel(btf_sampling a) {
  __shared__ Pick sh;
  const int m = blockIdx.x, tid = threadIdx.x;
  const float* x = a.logits + (size_t)m * a.ldl;
  Scratch& s = scratch_of(a, m);
  const Row r = s.row;
  if (r.greedy) {
    if (tid == 0) {
      a.token[m] = argmax_key_index(s.best);
      if (a.logprob) a.logprob[m] = 0.f;
    }
    return;
  }
  uint32_t n = s.ncand;
  if (n > kCand) {
    pick_alone(a, x, m, r, sh);
    return;
  }
  Borders b = s.borders;
  const int nsum = (a.V + kSum - 1) / kSum;
  const u64* psum = s.psum();
  for (int i = tid; i < nsum; i += kPickThreads) sh.c.sum[i] = psum[i];
  if (tid == 0) sh.kth = 0, sh.n = 0, sh.before = 0;
  constexpr int PER = kCand / kPickThreads;
  const bool by_k = b.kb < kBins;
  if (n > 64 && b.lo == b.hi && (by_k ? b.lo == b.kb && r.p == 1.f : true)) {
    // One border in one bin: the bin again in kFine pieces. What lies in the pieces before the border's stays, only what
    // lies in that is sorted.
    for (int i = tid; i < kFine; i += kPickThreads) sh.c.fine[i] = 0;
    __syncthreads();
    u64 key[PER], w[PER];
    int f[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      f[i] = -1;
      const uint32_t at = tid + i * kPickThreads;
      if (at >= n) continue;
      const float v = __uint_as_float(s.cand[at][0]);
      key[i] = argmax_key(v, (int)s.cand[at][1]);
      const double d = distance(of_key((uint32_t)(key[i] >> 32)), r.top, r.inv_t);
      w[i] = weight_at(d);
      f[i] = max(0, min(kFine - 1, (int)((d * r.scale - (double)b.lo) * kFine)));
      atomicAdd(reinterpret_cast<unsigned long long*>(&sh.c.fine[f[i]]), by_k ? 1ull : (unsigned long long)w[i]);
    }
    __syncthreads();
    constexpr int FPER = kFine / kPickThreads;
    u64 c[FPER], mine = 0, total;
#pragma unroll
    for (int i = 0; i < FPER; ++i) mine += c[i] = sh.c.fine[tid * FPER + i];
    u64 at = block_scan<kPickThreads>(mine, sh.part, &total) - mine;
    const double want = by_k ? (double)b.k_left : (double)r.p * (double)b.below_kb;
    const u64 from = by_k ? 0 : b.below_lo;  // (below_kb: all of the row)
#pragma unroll
    for (int i = 0; i < FPER; ++i) {
      const double before = (double)(from + at), after = (double)(from + at + c[i]);
      const bool first = from + at == 0 && c[i] > 0;
      if ((first || before < want) && after >= want && c[i] > 0) sh.sh[0] = tid * FPER + i, sh.sh[1] = at;
      at += c[i];
    }
    __syncthreads();
    const int piece = (int)sh.sh[0];
    if (by_k) b.k_left -= (uint32_t)sh.sh[1];
    else b.below_lo += sh.sh[1];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      if (f[i] < 0) continue;
      if (f[i] < piece && w[i] >= r.floor_w)
        atomicAdd(reinterpret_cast<unsigned long long*>(&sh.c.sum[argmax_key_index(key[i]) / kSum]), (unsigned long long)w[i]);
      if (f[i] == piece) sh.c.key[atomicAdd(&sh.n, 1u)] = key[i];
    }
    __syncthreads();
    n = sh.n;
  } else {
    for (int i = tid; i < (int)n; i += kPickThreads) sh.c.key[i] = argmax_key(__uint_as_float(s.cand[i][0]), (int)s.cand[i][1]);
  }
  // candidates in order
  int size2 = 32;
  while (size2 < (int)n) size2 *= 2;
  const bool few = size2 <= kPickThreads;
  uint32_t* rank = reinterpret_cast<uint32_t*>(sh.c.fine);
  for (int i = n + tid; i < size2; i += kPickThreads) sh.c.key[i] = 0;
  if (tid < kPickThreads) rank[tid] = 0;
  __syncthreads();
  if (few) {
    // by their ranks: how many keys are larger, counted by kPickThreads / size2 threads for each (75 candidates: 0.5 us;
    // the passes of a sort wait for each other, 5 us)
    const int c = tid & (size2 - 1), share = size2 * size2 / kPickThreads, j0 = tid / size2 * share;
    const u64 key = sh.c.key[c];
    uint32_t larger = 0;
#pragma unroll 4
    for (int j = j0; j < j0 + share; ++j) larger += sh.c.key[j] > key;
    if (c < (int)n && larger) atomicAdd(&rank[c], larger);
    __syncthreads();
    if (tid < (int)n) sh.c.key[rank[tid]] = key;  // (tid < n: c is tid; every key has been read)
  } else {
    // by a bitonic sort. (a wave's pairs of a pass with j <= 64 lie in 128 keys that no other wave touches in such a pass:
    // its LDS accesses are in order, so only passes over longer distances need the workgroup to wait)
    bool far = false;
    for (int k = 2; k <= size2; k *= 2)
      for (int j = k / 2; j > 0; j /= 2) {
        if (far || j > 64) __syncthreads();
        far = j > 64;
        for (int i = tid; i < size2 / 2; i += kPickThreads) {
          const int lo = 2 * i - (i & (j - 1)), hi = lo + j;  // falling order in the end
          const u64 x0 = sh.c.key[lo], x1 = sh.c.key[hi];
          if ((x0 < x1) == ((lo & k) == 0)) sh.c.key[lo] = x1, sh.c.key[hi] = x0;
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
      }
  }
  __syncthreads();
  if (n == 0) {  // no border: nothing but the parts
  } else if (few) pick_borders<1>(sh, r, b, n);
  else pick_borders<kCand / kPickThreads>(sh, r, b, n);
  // the kSum logits in which the sum passes u times the total
  constexpr int SPER = kMaxV / kSum / kPickThreads;
  const int per = (nsum + kPickThreads - 1) / kPickThreads;  // at most SPER
  u64 ps = 0, total;
#pragma unroll
  for (int i = 0; i < SPER; ++i)
    if (i < per && tid * per + i < nsum) ps += sh.c.sum[tid * per + i];
  u64 end = block_scan<kPickThreads>(ps, sh.part, &total);
  const double u = a.u[m];
  u64 at = u > 0.0 ? (u64)fmin(u * (double)total, kMost) : 0;
  if (at >= total) at = total - 1;
  if (end > at && end - ps <= at) {
    u64 before = end - ps;
    for (int i = tid * per; i < nsum; ++i) {
      if (before + sh.c.sum[i] > at) {
        sh.sh[0] = i, sh.sh[1] = at - before;
        break;
      }
      before += sh.c.sum[i];
    }
  }
  __syncthreads();
  if (tid >= 64) return;
  // one wave walks them, four a lane
  const int i0 = (int)min(sh.sh[0], (u64)nsum - 1) * kSum + 4 * tid;
  at = sh.sh[1];
  const u64 kth = sh.kth;  // the last that stays; 0: all of the bins before lo, and nothing else
  u64 wt[4], mine = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    wt[j] = 0;
    if (i0 + j >= a.V) continue;
    const float v = x[i0 + j];
    const double d = distance(v, r.top, r.inv_t);
    if (!(d < kFar)) continue;
    if (bin_of(d, r) >= b.lo && !(kth && argmax_key(v, i0 + j) >= kth)) continue;
    const u64 y = weight_at(d);
    if (y >= r.floor_w) wt[j] = y, mine += y;
  }
  u64 upto = mine;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const u64 y = __shfl_up(upto, o, 64);
    if (tid >= o) upto += y;
  }
  if (upto > at && upto - mine <= at) {
    u64 sum = upto - mine;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      sum += wt[j];
      if (sum > at && sum - wt[j] <= at) {
        a.token[m] = i0 + j;
        if (a.logprob) a.logprob[m] = (float)log((double)wt[j] / (double)total);
      }
    }
  }
}

}  // namespace

int64_t sample_ws_bytes(int M, int V) { return (int64_t)M * scratch_bytes(V); }

int sample(const btf_sampling& a, hipStream_t st) {
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
    b.ws = static_cast<char*>(a.ws) + (size_t)m0 * scratch_bytes(a.V);
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
    hipLaunchKernelGGL(sample_pick_kernel, dim3(M), dim3(kPickThreads), 0, st, b);
    if ((rc = launch_status("sample_pick_kernel")) != BTF_OK) return rc;
  }
  return BTF_OK;
}

}  // namespace btfhip
