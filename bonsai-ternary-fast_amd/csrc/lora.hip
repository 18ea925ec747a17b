// lora.hip -- low-rank adapters of many requests beside a shared projection
// (btf_hip_launch_lora; gfx950): y += scale B (A x), each request's rows with its
// own A [rank][K] and B [N][rank].
//
// Two launches (one where rows are few and A is small). lora_shrink: h = A x, a tile of rows of one request by a slice of K a
// workgroup; its waves take every fourth 64 columns, join in LDS, and leave the slice's
// sums in the workspace. lora_expand: the slices' sums in order, times scale, then
// B h for a tile of rows and a run of outputs, added to y (or through silu(g) u).
// No sum's order depends on which workgroup comes first.
//
// Products on 16x16x32 bf16 MFMA with exact factors: a 32-bit x is the sum of three
// bf16 numbers (8 bits each, cut off, not rounded, so that no part overflows), h
// likewise, an fp16 weight of two. All products of parts are taken, so only the sums
// round, in 32 bits. (The three parts cost less than a third of 32-bit MFMA would, and
// where few rows have an adapter nothing but its bytes counts.) Infinite x or weights give NaN.
//
// Bound by HBM where rows or adapters are many, by latency where few.
#include <string>

#include "../../include/btf/hip_abi.h"
#include "common.h"

namespace btfhip {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));  // (in memory: rows of y start anywhere)

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kBlockK = 64;       // columns of a wave's step
constexpr int kGroups = 512;      // workgroups that a launch is cut into, at least
constexpr int kChunk = 256;       // outputs of a workgroup, or a multiple
// Workgroups below which the ranks (of few rows) and the outputs are cut further: 8 rows of five requests, ranks of 128, 547 + 2 * 109
// outputs 26.8 us, with the ranks cut 21.2, with both 13.7; 26 rows, gate and up of 684 21.8, 20.7, 15.9; 60 rows of one request,
// ranks of 16 14.4 and 12.5.
constexpr int kSplit = 512;

struct Segs {
  btf_lora_seg s[3];
};

__device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0, 0);
}

// The upper halves of two 32-bit numbers (bf16, cut off), and what they leave.
__device__ __forceinline__ uint32_t cut2(float& x, float& y) {
  const uint32_t a = __float_as_uint(x), b = __float_as_uint(y);
  x -= __uint_as_float(a & 0xffff0000u);
  y -= __uint_as_float(b & 0xffff0000u);
  return __builtin_amdgcn_perm(b, a, 0x07060302u);
}
// Eight numbers as three times eight bf16.
__device__ __forceinline__ void cut3(f32x4 lo, f32x4 hi, u32x4 (&p)[3]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    float x = j < 2 ? lo[2 * j] : hi[2 * j - 4], y = j < 2 ? lo[2 * j + 1] : hi[2 * j - 3];
    p[0][j] = cut2(x, y);
    p[1][j] = cut2(x, y);
    p[2][j] = cut2(x, y);
  }
}
// Eight weights as one or two times eight bf16.
template <bool BF>
__device__ __forceinline__ void weights(u32x4 v, u32x4 (&w)[BF ? 1 : 2]) {
  if constexpr (BF) {
    w[0] = v;
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float x = h2f((uint16_t)v[j]), y = h2f((uint16_t)(v[j] >> 16));
      w[0][j] = cut2(x, y);
      w[1][j] = cut2(x, y);
    }
  }
}

// Inclusive sum over the lanes.
__device__ __forceinline__ int wave_scan(int v) {
  v += dpp_i<0x111>(v);
  v += dpp_i<0x112>(v);
  v += dpp_i<0x114>(v);
  v += dpp_i<0x118>(v);
  const int t0 = __builtin_amdgcn_readlane(v, 15), t1 = __builtin_amdgcn_readlane(v, 31), t2 = __builtin_amdgcn_readlane(v, 47);
  const int row = (threadIdx.x & 63) >> 4;
  return v + (row > 0 ? t0 : 0) + (row > 1 ? t1 : 0) + (row > 2 ? t2 : 0);
}

// Tile `id` of R rows of the requests, found by every wave for itself: its first row and
// rows, its adapter (-1: none) and that one's rank. False: there is no such tile.
struct Tile {
  int row, n, adapter, rank;
};
template <int R>
__device__ bool find(const btf_lora& a, int id, Tile& t) {
  const int lane = threadIdx.x & 63;
  int before = 0;
  for (int s0 = 0; s0 < a.S; s0 += 64) {
    int r0 = 0, n = 0, who = -1;
    if (s0 + lane < a.S) {
      r0 = min(max(a.row0[s0 + lane], 0), a.T);
      n = min(max(a.row0[s0 + lane + 1], 0), a.T) - r0;
      who = a.adapter[s0 + lane];
    }
    const int mine = n > 0 ? (n + R - 1) / R : 0, upto = before + wave_scan(mine);
    const unsigned long long here = __ballot(mine > 0 && id >= upto - mine && id < upto);
    if (here) {
      const int l = __builtin_ctzll(here), k = id - __builtin_amdgcn_readlane(upto - mine, l);
      t.row = __builtin_amdgcn_readlane(r0, l) + k * R;
      t.n = min(__builtin_amdgcn_readlane(n, l) - k * R, R);
      t.adapter = __builtin_amdgcn_readlane(who, l);
      if (t.adapter < 0 || t.adapter >= a.adapters) t.adapter = -1;
      t.rank = t.adapter < 0 ? 0 : a.ranks ? min(max(a.ranks[t.adapter], 0), a.rank) : a.rank;
      return true;
    }
    before = __builtin_amdgcn_readlane(upto, 63);
  }
  return false;
}

// h of row `row`, rank 0, slice k of K.
__device__ __forceinline__ float* h_of(const btf_lora& a, int nseg, int k, int seg, int row) {
  return static_cast<float*>(a.ws) + ((size_t)(k * nseg + seg) * a.T + row) * a.rank;
}

// RT tiles of 16 rows by NT tiles of 16 ranks, those of all segments in a row: x is read and cut once for all of them.
// grid: (tile, slice of K), NT tiles of ranks.
template <bool BF, int RT, int NT>
__global__ void __launch_bounds__(kThreads, 2) lora_shrink_kernel(btf_lora a, Segs segs, int nseg, int slices, int slice) {
  constexpr int R = 16 * RT, LD = 16 * NT + 4;
  __shared__ float sh[kWaves][R][LD];
  Tile t;
  const int k = blockIdx.x % slices, of_seg = (a.rank + 15) / 16;
  if (!find<R>(a, blockIdx.x / slices, t)) return;  // the whole workgroup
  int seg[NT], first[NT];  // of each tile of ranks; first at or behind the adapter's rank: nothing to do
  bool any = false;
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int i = blockIdx.y * NT + n;
    seg[n] = min(i / of_seg, nseg - 1);
    first[n] = i / of_seg < nseg ? 16 * (i % of_seg) : a.rank;
    any |= first[n] < t.rank;
  }
  if (!any) return;  // the whole workgroup
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, c16 = lane & 15, g = lane >> 4;
  const int end = min(a.K, (k + 1) * slice);
  // lane's columns of a step: 16 g .. 16 g + 15; its row of x in each tile, its rank's row of A
  const float* x = a.x + (size_t)(t.row + c16) * a.ldx + 16 * g;
  const uint16_t* m[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n)
    m[n] = static_cast<const uint16_t*>(segs.s[seg[n]].a) + (size_t)t.adapter * segs.s[seg[n]].a_stride + (size_t)(first[n] + c16) * a.K + 16 * g;
  f32x4 acc[RT][NT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt)
#pragma unroll
    for (int n = 0; n < NT; ++n) acc[rt][n] = f32x4{0.f, 0.f, 0.f, 0.f};
  f32x4 xv[RT][4];
  u32x4 av[NT][2];
  auto load = [&](int kb) {
    const bool in = kb + 16 * g < end;  // (K is a multiple of 32: a lane's columns are all there or none)
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        av[n][u] = u32x4{0, 0, 0, 0};
        if (in && first[n] + c16 < t.rank) av[n][u] = *reinterpret_cast<const u32x4*>(m[n] + kb + 8 * u);
      }
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        xv[rt][u] = f32x4{0.f, 0.f, 0.f, 0.f};
        if (in && 16 * rt + c16 < t.n)
          xv[rt][u] = *reinterpret_cast<const f32x4*>(x + (size_t)(16 * rt) * a.ldx + kb + 4 * u);
      }
  };
  // Few rows: the next step's loads are on their way while this one is worked on. Many: a wave's loads are 16 KB
  // anyway, and its registers are the rows'.
  constexpr bool kAhead = RT == 1;
  constexpr int kStep = kBlockK * kWaves;
  int kb = k * slice + kBlockK * w;
  if (kAhead && kb < end) load(kb);
  for (; kb < end; kb += kStep) {
    if (!kAhead) load(kb);
    u32x4 xp[kAhead ? 2 : 1][RT][3], ap[kAhead ? 2 : 1][NT][BF ? 1 : 2];
    auto cut = [&](int u, int at) {
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) cut3(xv[rt][2 * u], xv[rt][2 * u + 1], xp[at][rt]);
#pragma unroll
      for (int n = 0; n < NT; ++n) weights<BF>(av[n][u], ap[at][n]);
    };
    auto multiply = [&](int at) {
#pragma unroll
      for (int p = 0; p < 3; ++p)
#pragma unroll
        for (int q = 0; q < (BF ? 1 : 2); ++q)
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) acc[rt][n] = mfma(ap[at][n][q], xp[at][rt][p], acc[rt][n]);
    };
    if constexpr (kAhead) {
      cut(0, 0);
      cut(1, 1);
      if (kb + kStep < end) load(kb + kStep);
      multiply(0);
      multiply(1);
    } else {
      cut(0, 0);
      multiply(0);
      cut(1, 0);
      multiply(0);
    }
  }
  // the waves' sums (lane: row c16, ranks 4 g .. 4 g + 3)
#pragma unroll
  for (int rt = 0; rt < RT; ++rt)
#pragma unroll
    for (int n = 0; n < NT; ++n) *reinterpret_cast<f32x4*>(&sh[w][16 * rt + c16][16 * n + 4 * g]) = acc[rt][n];
  __syncthreads();
  for (int i = threadIdx.x; i < t.n * 4; i += kThreads) {
    const int r = i / 4, c = 4 * (i % 4);
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      if (first[n] + c >= a.rank) continue;  // (a.rank is a multiple of 8)
      f32x4 v = *reinterpret_cast<const f32x4*>(&sh[0][r][16 * n + c]);
#pragma unroll
      for (int j = 1; j < kWaves; ++j) v += *reinterpret_cast<const f32x4*>(&sh[j][r][16 * n + c]);
      *reinterpret_cast<f32x4*>(h_of(a, nseg, k, seg[n], t.row + r) + first[n] + c) = v;
    }
  }
}

// The slices' sums, in the first one's place: where there are more than kSlices, lora_expand's many workgroups would each
// read them all (441 rows of 16544 columns in 33 slices, gate and up of 1248 outputs: the call 49 us, so 30).
constexpr int kSlices = 8;
__global__ void __launch_bounds__(kThreads) lora_join_kernel(float* h, int64_t n, int slices) {
  const int64_t i = 4 * ((int64_t)blockIdx.x * kThreads + threadIdx.x);
  if (i >= n) return;
  f32x4 v = {0.f, 0.f, 0.f, 0.f};
  for (int k = 0; k < slices; k += 8) {
    f32x4 x[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) x[u] = *reinterpret_cast<const f32x4*>(h + i + min(k + u, slices - 1) * n);
#pragma unroll
    for (int u = 0; u < 8; ++u)
      if (k + u < slices) v += x[u];
  }
  *reinterpret_cast<f32x4*>(h + i) = v;
}

// Row of h's parts in LDS, in bf16: the ranks in steps of 32, and 16 bytes so that rows lie in other banks.
__host__ __device__ constexpr int parts_ld(int rank) { return (rank + 31) / 32 * 32 + 8; }

// RT tiles of 16 rows by `chunk` outputs. GLU: both segments, into out.
template <bool BF, int RT, bool GLU>
__global__ void __launch_bounds__(kThreads, 2) lora_expand_kernel(btf_lora a, Segs segs, int nseg, int slices, int chunk, int chunks) {
  constexpr int R = 16 * RT, NS = GLU ? 2 : 1;
  constexpr int TN = GLU && RT > 2 ? 1 : GLU || RT > 1 ? 2 : 4;  // tiles of 16 outputs of a wave at a time
  extern __shared__ uint16_t sh_h[];         // [segment][part][row][parts_ld]
  Tile t;
  if (!find<R>(a, blockIdx.x / chunks, t) || (!GLU && t.rank == 0)) return;  // the whole workgroup
  int c = blockIdx.x % chunks, seg = 0;
  if (!GLU)
    while (seg < nseg - 1 && c >= (segs.s[seg].N + chunk - 1) / chunk) c -= (segs.s[seg].N + chunk - 1) / chunk, ++seg;
  const int N = segs.s[seg].N, ld = parts_ld(a.rank), steps = (t.rank + 31) / 32;
  const float scale = t.adapter >= 0 && a.scale ? a.scale[t.adapter] : 1.f;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, c16 = lane & 15, g = lane >> 4;
  const int n1 = min(N, (c + 1) * chunk);
  // y of the lane's row in each tile (outputs n0 + 16 i + 4 g .. + 3) and 64 ranks of B from rank 32 k on
  f32x4 y[NS][TN][RT];
  u32x4 bv[2][NS][TN];
  auto load_y = [&](int n0) {
#pragma unroll
    for (int sg = 0; sg < NS; ++sg)
#pragma unroll
      for (int i = 0; i < TN; ++i)
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
          const btf_lora_seg& s = segs.s[GLU ? sg : seg];
          const int n = n0 + 16 * i + 4 * g, r = 16 * rt + c16;
          const float* p = s.y + (size_t)(t.row + r) * s.ldy + n;
          y[sg][i][rt] = f32x4{0.f, 0.f, 0.f, 0.f};
          if (r < t.n) {
            if (n + 3 < n1) {
              y[sg][i][rt] = *reinterpret_cast<const f32x4_any*>(p);
            } else {
#pragma unroll
              for (int j = 0; j < 4; ++j)
                if (n + j < n1) y[sg][i][rt][j] = p[j];
            }
          }
        }
  };
  auto load_b = [&](int n0, int k) {
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int sg = 0; sg < NS; ++sg) {
        const btf_lora_seg& s = segs.s[GLU ? sg : seg];
        const uint16_t* b = static_cast<const uint16_t*>(s.b) + (size_t)max(t.adapter, 0) * s.b_stride + (size_t)(n0 + c16) * a.rank + 8 * g;
#pragma unroll
        for (int i = 0; i < TN; ++i) {
          bv[u][sg][i] = u32x4{0, 0, 0, 0};
          if (32 * (k + u) + 8 * g < t.rank && n0 + 16 * i + c16 < n1)
            bv[u][sg][i] = *reinterpret_cast<const u32x4*>(b + (size_t)(16 * i) * a.rank + 32 * (k + u));
        }
      }
  };
  int n0 = c * chunk + 16 * TN * w;
  load_b(n0, 0);  // (on their way while h is put together)
  load_y(n0);
  // h, scaled, in parts
  for (int i = threadIdx.x; i < NS * R * steps * 8; i += kThreads) {
    const int q = 4 * (i % (steps * 8)), r = i / (steps * 8) % R, sg = i / (steps * 8) / R;
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    if (r < t.n && q < t.rank) {
      const float* h = h_of(a, nseg, 0, GLU ? sg : seg, t.row + r) + q;
      const size_t next = (size_t)nseg * a.T * a.rank;
      for (int k = 0; k < slices; k += 8) {
        f32x4 x[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) x[u] = *reinterpret_cast<const f32x4*>(h + min(k + u, slices - 1) * next);
#pragma unroll
        for (int u = 0; u < 8; ++u)
          if (k + u < slices) v += x[u];
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = q + j < t.rank ? v[j] * scale : 0.f;
    }
    float x[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
    for (int p = 0; p < 3; ++p) {
      const uint32_t lo = cut2(x[0], x[1]), hi = cut2(x[2], x[3]);
      *reinterpret_cast<uint2*>(sh_h + (size_t)((sg * 3 + p) * R + r) * ld + q) = uint2{lo, hi};
    }
  }
  __syncthreads();
  while (n0 < n1) {
    const int next = n0 + 16 * TN * kWaves;
    f32x4 d[NS][TN][RT];
#pragma unroll
    for (int sg = 0; sg < NS; ++sg)
#pragma unroll
      for (int i = 0; i < TN; ++i)
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) d[sg][i][rt] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int k = 0; k < steps; k += 2) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        if (k + u >= steps) break;
        const int left = t.rank - 32 * (k + u) - 8 * g;  // ranks from the lane's first on
#pragma unroll
        for (int sg = 0; sg < NS; ++sg) {
          u32x4 hp[RT][3];
#pragma unroll
          for (int rt = 0; rt < RT; ++rt)
#pragma unroll
            for (int p = 0; p < 3; ++p)
              hp[rt][p] = *reinterpret_cast<const u32x4*>(sh_h + (size_t)((sg * 3 + p) * R + 16 * rt + c16) * ld + 32 * (k + u) + 8 * g);
#pragma unroll
          for (int i = 0; i < TN; ++i) {
            u32x4 v = bv[u][sg][i], bp[BF ? 1 : 2];
#pragma unroll
            for (int j = 0; j < 4; ++j)  // what lies behind the adapter's rank
              v[j] &= left > 2 * j + 1 ? 0xffffffffu : left > 2 * j ? 0xffffu : 0u;
            weights<BF>(v, bp);
#pragma unroll
            for (int p = 0; p < 3; ++p)
#pragma unroll
              for (int q = 0; q < (BF ? 1 : 2); ++q)
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) d[sg][i][rt] = mfma(bp[q], hp[rt][p], d[sg][i][rt]);
          }
        }
      }
      if (k + 2 < steps) load_b(n0, k + 2);
    }
    if (next < n1) load_b(next, 0);
#pragma unroll
    for (int i = 0; i < TN; ++i)
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        f32x4 v = y[0][i][rt] + d[0][i][rt];
        if (GLU) {
          const f32x4 up = y[NS - 1][i][rt] + d[NS - 1][i][rt];
#pragma unroll
          for (int j = 0; j < 4; ++j) v[j] = v[j] / (1.0f + expf(-v[j])) * up[j];
        }
        d[0][i][rt] = v;
      }
    const int at = n0;
    n0 = next;
    if (n0 < n1) load_y(n0);  // (before the stores, whose ends a wait for it would include)
#pragma unroll
    for (int i = 0; i < TN; ++i)
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        const int n = at + 16 * i + 4 * g, r = 16 * rt + c16;
        const f32x4 v = d[0][i][rt];
        float* p = GLU ? a.out + (size_t)(t.row + r) * a.ldo + n : segs.s[seg].y + (size_t)(t.row + r) * segs.s[seg].ldy + n;
        if (r < t.n) {
          if (n + 3 < n1) {
            *reinterpret_cast<f32x4_any*>(p) = v;
          } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (n + j < n1) p[j] = v[j];
          }
        }
      }
  }
}

// ---- few rows: a row or four a request, each adapter's bytes read for next to nothing ----
// Vector arithmetic in 32 bits: for one row matrix instructions spend 15 of 16 rows on
// nothing, and the registers that hold them are then missing for loads in flight.

// Eight weights times eight numbers, added to s.
template <bool BF>
__device__ __forceinline__ float dot8(u32x4 w, const float* x, float s) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float lo = BF ? __uint_as_float(w[j] << 16) : h2f((uint16_t)w[j]);
    const float hi = BF ? __uint_as_float(w[j] & 0xffff0000u) : h2f((uint16_t)(w[j] >> 16));
    s = __builtin_fmaf(lo, x[2 * j], s);
    s = __builtin_fmaf(hi, x[2 * j + 1], s);
  }
  return s;
}
__device__ __forceinline__ float swap16(float v) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float swap32(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// Workgroups that a launch of few rows is cut into, at least (64 requests of one token, three segments, ranks to 64: shrink
// and expand 38.6 us with 512, 33.8 with 1024, 36.0 with 2048).
constexpr int kFewGroups = 1024;
constexpr int kFewK = 512;     // columns of a wave's step, eight a lane
constexpr int kFewRanks = 8;   // ranks of a wave at a time
// One launch in place of two, in which each workgroup multiplies A itself: as long as there is a CU for each and A is small
// (one row, K and N 5120: ranks of 16 11.4 us in two launches, 8.1 so; 32 10.9 and 9.2; 64 11.5 and 12.0; eight rows, K 17408,
// ranks of 32 11.1 and 20.2; gate and up of four rows, ranks of 8, 272 workgroups, 11.3 and 18.0).
constexpr int kOneGroups = 256, kOneValues = 160 * 1024;

// R rows by the adapter's ranks, columns k0 .. end - 1: the workgroup's W waves share the ranks by eights; where there are
// fewer than W of these, several waves share one by steps of K and join in LDS. store(rank, row, sum) by some lane.
template <bool BF, int R, int W, class Store>
__device__ __forceinline__ void shrink_few(const btf_lora& a, const btf_lora_seg& s, const Tile& t, int k0, int end, int part, int parts,
                                           float (&sh)[W][R][kFewRanks], const Store& store) {
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int all = (t.rank + kFewRanks - 1) / kFewRanks;
  int groups = 1;
  while (2 * groups <= W && 2 * groups <= all) groups *= 2;
  const int share = W / groups;
  // Steps (ranks from g0 on, columns from kb on) in turn, the next one's loads under way while one is worked on.
  struct Step {
    int g0, kb;
  };
  const int kb0 = k0 + w % share * kFewK;
  auto next_of = [&](Step p) { return p.kb + share * kFewK < end ? Step{p.g0, p.kb + share * kFewK} : Step{p.g0 + parts * groups, kb0}; };
  auto ranks_of = [&](int g0) { return min(t.rank - (g0 + w / share) * kFewRanks, kFewRanks); };
  u32x4 av[kFewRanks];
  f32x4 xv[R][2];
  auto load = [&](Step p) {
    const int first = (p.g0 + w / share) * kFewRanks, ranks = ranks_of(p.g0);
    const uint16_t* m = static_cast<const uint16_t*>(s.a) + (size_t)t.adapter * s.a_stride + (size_t)first * a.K + p.kb;
    const float* x = a.x + (size_t)t.row * a.ldx + p.kb;
    const bool in = p.kb + 8 * lane < end;
#pragma unroll
    for (int i = 0; i < kFewRanks; ++i) {
      av[i] = u32x4{0, 0, 0, 0};
      if (in && i < ranks) av[i] = reinterpret_cast<const u32x4*>(m + (size_t)i * a.K)[lane];
    }
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        xv[r][u] = f32x4{0.f, 0.f, 0.f, 0.f};
        if (in && r < t.n) xv[r][u] = reinterpret_cast<const f32x4*>(x + (size_t)r * a.ldx)[2 * lane + u];
      }
  };
  Step at{part * groups, kb0};
  if (at.g0 >= all) return;  // the whole workgroup
  load(at);
  float acc[kFewRanks][R] = {};
  while (at.g0 < all) {
    const Step next = next_of(at);
    u32x4 ac[kFewRanks];
    float xs[R][8];
#pragma unroll
    for (int i = 0; i < kFewRanks; ++i) ac[i] = av[i];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int j = 0; j < 8; ++j) xs[r][j] = xv[r][j >> 2][j & 3];
    if (next.g0 < all) load(next);
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int i = 0; i < kFewRanks; ++i) acc[i][r] = dot8<BF>(ac[i], xs[r], acc[i][r]);
    if (next.g0 != at.g0) {  // the lanes' sums: rank i of row r to lane i; then the waves'
      const int first = (at.g0 + w / share) * kFewRanks, ranks = ranks_of(at.g0);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        float mine = 0.f;
#pragma unroll
        for (int i = 0; i < kFewRanks; ++i) {
          const float v = swap32(swap16(row16_sum(acc[i][r])));
          mine = lane == i ? v : mine;
          acc[i][r] = 0.f;
        }
        if (lane < kFewRanks) sh[w][r][lane] = mine;
      }
      if (share > 1) __syncthreads();
      if (w % share == 0 && lane < ranks)
        for (int r = 0; r < t.n; ++r) {
          float v = sh[w][r][lane];
          for (int j = 1; j < share; ++j) v += sh[w + j][r][lane];
          store(first + lane, r, v);
        }
      if (share > 1) __syncthreads();
    }
    at = next;
  }
}

// grid: (tile, slice of K), (segment, one of `parts` shares of the ranks).
template <bool BF, int R>
__global__ void __launch_bounds__(kThreads, 2)
    lora_shrink_few_kernel(btf_lora a, Segs segs, int nseg, int slices, int slice, int parts) {
  __shared__ float sh[kWaves][R][kFewRanks];
  Tile t;
  const int k = blockIdx.x % slices, seg = blockIdx.y / parts;
  if (!find<R>(a, blockIdx.x / slices, t) || t.rank == 0) return;  // the whole workgroup
  shrink_few<BF, R, kWaves>(a, segs.s[seg], t, k * slice, min(a.K, (k + 1) * slice), blockIdx.y % parts, parts, sh,
                            [&](int q, int r, float v) { h_of(a, nseg, k, seg, t.row + r)[q] = v; });
}

// R rows by `chunk` outputs. The lanes of 2^lg hold one row of B, eight ranks each, so that a wave's load is 1 KB in one
// piece; kFewLoads of them are on their way at a time.
// ONE: h by the workgroup itself, in place of the launch before.
constexpr int kFewLoads = 8;
constexpr int kOneWaves = 16;
template <bool BF, int R, bool GLU, bool ONE>
__global__ void __launch_bounds__(ONE ? 64 * kOneWaves : kThreads, ONE ? 1 : 2)
    lora_expand_few_kernel(btf_lora a, Segs segs, int nseg, int slices, int chunk, int chunks) {
  constexpr int NS = GLU ? 2 : 1, U = ONE ? 2 : kFewLoads / NS / (R > 1 ? 2 : 1), W = ONE ? kOneWaves : kWaves;
  __shared__ float sh_h[NS][R][256], sh_part[kThreads];
  Tile t;
  if (!find<R>(a, blockIdx.x / chunks, t) || (!GLU && t.rank == 0)) return;  // the whole workgroup
  int c = blockIdx.x % chunks, seg = 0;
  if (!GLU)
    while (seg < nseg - 1 && c >= (segs.s[seg].N + chunk - 1) / chunk) c -= (segs.s[seg].N + chunk - 1) / chunk, ++seg;
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lg = t.rank <= 8 ? 0 : 32 - __builtin_clz((t.rank + 7) / 8 - 1), per = 64 >> lg;  // outputs of a load
  const int j = lane & ((1 << lg) - 1), n_of = lane >> lg;
  const int n1 = min(segs.s[seg].N, (c + 1) * chunk);
  const bool in = 8 * j < t.rank;
  u32x4 bv[NS][U];
  float y[NS][U][R];
  auto load = [&](int n0) {
#pragma unroll
    for (int sg = 0; sg < NS; ++sg) {
      const btf_lora_seg& s = segs.s[GLU ? sg : seg];
      const uint16_t* b = static_cast<const uint16_t*>(s.b) + (size_t)max(t.adapter, 0) * s.b_stride + 8 * j;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int n = n0 + u * per + n_of;
        bv[sg][u] = u32x4{0, 0, 0, 0};
        if (in && n < n1) bv[sg][u] = *reinterpret_cast<const u32x4*>(b + (size_t)n * a.rank);
#pragma unroll
        for (int r = 0; r < R; ++r) {
          y[sg][u][r] = 0.f;
          if (n < n1 && r < t.n) y[sg][u][r] = s.y[(size_t)(t.row + r) * s.ldy + n];
        }
      }
    }
  };
  int n0 = c * chunk + w * U * per;
  load(n0);  // (on their way while h is put together)
  const float scale = t.adapter >= 0 && a.scale ? a.scale[t.adapter] : 1.f;
  // h, scaled; behind the rank zero.
  if constexpr (ONE) {
    __shared__ float sh[W][R][kFewRanks];
    for (int i = threadIdx.x; i < NS * R * 256; i += 64 * W) (&sh_h[0][0][0])[i] = 0.f;
    __syncthreads();
    if (t.rank > 0)
#pragma unroll 1
      for (int sg = 0; sg < NS; ++sg) {
        const btf_lora_seg& s = segs.s[GLU ? sg : seg];
        shrink_few<BF, R, W>(a, s, t, 0, a.K, 0, 1, sh, [&](int q, int r, float v) { sh_h[sg][r][q] = v * scale; });
      }
  } else {
    // Several threads share a sum over the slices: slice k goes to thread k % share.
    const int lr = 3 + lg, items = NS * R << lr;
    int share = 1;
    while (share * 2 * items <= kThreads && share < slices) share *= 2;
    for (int i = threadIdx.x; i < items * share; i += kThreads) {
      const int part = i / items, e = i % items, q = e & ((1 << lr) - 1), r = (e >> lr) % R, sg = (e >> lr) / R;
      float v = 0.f;
      if (r < t.n && q < t.rank) {
        const float* h = h_of(a, nseg, 0, GLU ? sg : seg, t.row + r) + q;
        const size_t next = (size_t)nseg * a.T * a.rank;
        for (int k = part; k < slices; k += 8 * share) {
          float x[8];
#pragma unroll
          for (int u = 0; u < 8; ++u) x[u] = h[min(k + u * share, slices - 1) * next];
#pragma unroll
          for (int u = 0; u < 8; ++u)
            if (k + u * share < slices) v += x[u];
        }
      }
      if (share > 1) sh_part[i] = v;
      else sh_h[sg][r][q] = v * scale;
    }
    if (share > 1) {
      __syncthreads();
      for (int e = threadIdx.x; e < items; e += kThreads) {
        float v = sh_part[e];
        for (int j = 1; j < share; ++j) v += sh_part[j * items + e];
        sh_h[(e >> lr) / R][(e >> lr) % R][e & ((1 << lr) - 1)] = v * scale;
      }
    }
  }
  __syncthreads();
  while (n0 < n1) {
    float d[NS][U][R];
#pragma unroll
    for (int sg = 0; sg < NS; ++sg)
#pragma unroll
      for (int r = 0; r < R; ++r) {
        float h[8];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const f32x4 v = *reinterpret_cast<const f32x4*>(&sh_h[sg][r][8 * j + 4 * i]);
          h[4 * i] = v[0], h[4 * i + 1] = v[1], h[4 * i + 2] = v[2], h[4 * i + 3] = v[3];
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          u32x4 b = bv[sg][u];
#pragma unroll
          for (int i = 0; i < 4; ++i)  // what lies behind the adapter's rank
            b[i] &= t.rank - 8 * j > 2 * i + 1 ? 0xffffffffu : t.rank - 8 * j > 2 * i ? 0xffffu : 0u;
          float v = dot8<BF>(b, h, 0.f);
          if (lg > 0) v += dpp_f<0xB1>(v);
          if (lg > 1) v += dpp_f<0x4E>(v);
          if (lg > 2) v += dpp_f<0x141>(v);
          if (lg > 3) v += dpp_f<0x140>(v);
          if (lg > 4) v = swap16(v);
          d[sg][u][r] = v + y[sg][u][r];
        }
      }
    const int at = n0;
    n0 += U * per * W;
    if (n0 < n1) load(n0);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int n = at + u * per + n_of;
#pragma unroll
      for (int r = 0; r < R; ++r)
        if (j == 0 && n < n1 && r < t.n) {
          float v = d[0][u][r];
          if (GLU) v = v / (1.0f + expf(-v)) * d[NS - 1][u][r];
          (GLU ? a.out + (size_t)(t.row + r) * a.ldo : segs.s[seg].y + (size_t)(t.row + r) * segs.s[seg].ldy)[n] = v;
        }
    }
  }
}

// Tiles of the requests' rows, at most: a request's last one may be a part of one.
int most_tiles(const btf_lora& a, int R) { return a.T / R + a.S < a.T ? a.T / R + a.S : a.T; }

// Rows of h (a segment's, of one slice) that the workspace has room for: with tiles of at most 64 rows kGroups workgroups
// are at most kGroups * 64 + T rows of each segment, and there are at most as many slices as steps of K.
int64_t ws_rows(int T, int K, int nseg) {
  const int64_t most = (K + kBlockK * kWaves - 1) / (kBlockK * kWaves), all = nseg * T * most, cut = nseg * ((int64_t)T + kGroups * 64);
  return all < cut ? all : cut;
}
// Slices of K for `groups` workgroups or more of which `each` belong to a slice: of `step` columns or a multiple, and as
// many as there is room for.
struct Slices {
  int n, columns;
};
Slices slices_of(const btf_lora& a, int nseg, int groups, int64_t each, int step) {
  const int64_t most = (a.K + step - 1) / step, room = ws_rows(a.T, a.K, nseg) / ((int64_t)nseg * a.T);
  int64_t n = (groups + each - 1) / each;
  n = n < most ? n : most;
  n = n < room ? n : room;
  const int columns = (int)((a.K + n - 1) / n + step - 1) / step * step;
  return {(a.K + columns - 1) / columns, columns};
}

template <bool BF, int RT>
int lora_shrink(const btf_lora& a, const Segs& segs, int nseg, int& slices, hipStream_t st) {
  const int tiles = most_tiles(a, 16 * RT);
  const int all = nseg * ((a.rank + 15) / 16), nt = all <= 2 ? all : 4, groups = (all + nt - 1) / nt;
  const Slices sl = slices_of(a, nseg, kGroups, (int64_t)tiles * groups, kBlockK * kWaves);
  slices = sl.n;
  const int slice = sl.columns;
  const dim3 grid((unsigned)tiles * slices, groups), blk(kThreads);
  if (nt == 1) hipLaunchKernelGGL((lora_shrink_kernel<BF, RT, 1>), grid, blk, 0, st, a, segs, nseg, slices, slice);
  else if (nt == 2) hipLaunchKernelGGL((lora_shrink_kernel<BF, RT, 2>), grid, blk, 0, st, a, segs, nseg, slices, slice);
  else hipLaunchKernelGGL((lora_shrink_kernel<BF, RT, 4>), grid, blk, 0, st, a, segs, nseg, slices, slice);
  int rc = launch_status("lora_shrink_kernel");
  if (rc != BTF_OK) return rc;
  if (slices > kSlices) {
    const int64_t n = (int64_t)nseg * a.T * a.rank;
    hipLaunchKernelGGL(lora_join_kernel, dim3((unsigned)((n / 4 + kThreads - 1) / kThreads)), blk, 0, st, static_cast<float*>(a.ws), n, slices);
    rc = launch_status("lora_join_kernel");
    if (rc != BTF_OK) return rc;
    slices = 1;
  }
  return BTF_OK;
}

template <bool BF, int RT>
int lora_expand(const btf_lora& a, const Segs& segs, int nseg, int slices, hipStream_t st) {
  constexpr int R = 16 * RT;
  const int tiles = most_tiles(a, R);
  const bool glu = a.mode == BTF_GEMV_SWIGLU;
  int outs = 0;
  for (int i = 0; i < (glu ? 1 : nseg); ++i) outs += segs.s[i].N;
  int chunk = kChunk;
  while (chunk < 4 * kChunk && (int64_t)tiles * (outs / (2 * chunk)) >= kGroups) chunk *= 2;
  auto chunks_of = [&](int chunk) {
    int n = 0;
    for (int i = 0; i < (glu ? 1 : nseg); ++i) n += (segs.s[i].N + chunk - 1) / chunk;
    return n;
  };
  while (chunk > 64 && (int64_t)tiles * chunks_of(chunk) < kSplit) chunk /= 2;
  const int chunks = chunks_of(chunk);
  const size_t lds = (size_t)(glu ? 2 : 1) * 3 * R * parts_ld(a.rank) * 2;
  const dim3 eg((unsigned)tiles * chunks), blk(kThreads);
  auto expand = [&](auto kernel) { hipLaunchKernelGGL(kernel, eg, blk, lds, st, a, segs, nseg, slices, chunk, chunks); };
  if (glu) expand(lora_expand_kernel<BF, RT, true>);
  else expand(lora_expand_kernel<BF, RT, false>);
  return launch_status("lora_expand_kernel");
}

template <bool BF, int R>
int lora_few(const btf_lora& a, const Segs& segs, int nseg, hipStream_t st) {
  const int tiles = most_tiles(a, R);
  const bool glu = a.mode == BTF_GEMV_SWIGLU;
  int outs = 0, chunk = kChunk;
  for (int i = 0; i < (glu ? 1 : nseg); ++i) outs += segs.s[i].N;
  while (chunk < 4 * kChunk && (int64_t)tiles * (outs / (2 * chunk)) >= kFewGroups) chunk *= 2;
  auto chunks_of = [&](int chunk) {
    int n = 0;
    for (int i = 0; i < (glu ? 1 : nseg); ++i) n += (segs.s[i].N + chunk - 1) / chunk;
    return n;
  };
  int chunks = chunks_of(chunk);
  if (R == 1 && (int64_t)tiles * chunks <= kOneGroups && (int64_t)a.rank * a.K * (glu ? 2 : 1) <= kOneValues) {
    const dim3 grid((unsigned)tiles * chunks), blk(64 * kOneWaves);
    if (glu) hipLaunchKernelGGL((lora_expand_few_kernel<BF, 1, true, true>), grid, blk, 0, st, a, segs, nseg, 1, chunk, chunks);
    else hipLaunchKernelGGL((lora_expand_few_kernel<BF, 1, false, true>), grid, blk, 0, st, a, segs, nseg, 1, chunk, chunks);
    return launch_status("lora_expand_few_kernel");
  }
  const int together = a.rank > 2 * kFewRanks ? 1 : a.rank > kFewRanks ? 2 : 4;  // waves that share ranks
  const Slices sl = slices_of(a, nseg, kFewGroups, (int64_t)tiles * nseg, kFewK * together);
  const int slices = sl.n, slice = sl.columns;
  int parts = 1;  // as many as give each wave its eights of ranks, where there are few workgroups
  while (parts * 4 * kFewRanks < a.rank && (int64_t)tiles * slices * nseg * parts < kSplit) parts *= 2;
  hipLaunchKernelGGL((lora_shrink_few_kernel<BF, R>), dim3((unsigned)tiles * slices, nseg * parts), dim3(kThreads), 0, st, a, segs, nseg, slices, slice,
                     parts);
  const int rc = launch_status("lora_shrink_few_kernel");
  if (rc != BTF_OK) return rc;
  while (chunk > 64 && (int64_t)tiles * chunks_of(chunk) < kSplit / 2) chunk /= 2;
  chunks = chunks_of(chunk);
  const dim3 grid((unsigned)tiles * chunks);
  if (glu) hipLaunchKernelGGL((lora_expand_few_kernel<BF, R, true, false>), grid, dim3(kThreads), 0, st, a, segs, nseg, slices, chunk, chunks);
  else hipLaunchKernelGGL((lora_expand_few_kernel<BF, R, false, false>), grid, dim3(kThreads), 0, st, a, segs, nseg, slices, chunk, chunks);
  return launch_status("lora_expand_few_kernel");
}

// Which form: by the rows that a request has on average, as the sizes of the requests are device data. Where they are very
// unlike, one form does for rows that the other would do better (K 5120, gate and up of 17408, ranks of 64: 199 single rows and
// a prompt of 512 430 us, as two launches 101 + 66; 63 and 190 177 and 82, 63 and 200, above four rows on average, 107 and 82;
// ranks of 16 57, 44; 64, 45. Q, K and V, ranks of 64: 171 and 85; 75, 47; 56, 48. 31 and 2048, ranks of 16, 52 and 56).
template <bool BF>
int lora_any(const btf_lora& a, const Segs& segs, int nseg, hipStream_t st) {
  if (a.T <= a.S) return lora_few<BF, 1>(a, segs, nseg, st);
  if (a.T <= 4 * (int64_t)a.S) return lora_few<BF, 4>(a, segs, nseg, st);
  // Rows of a tile: 64 where A and B are worth reading less often, from ranks above 32 and 1024 rows on (ranks of 64, K 17408, N
  // 5120, 8000 rows 183 us, in tiles of 16 228; ranks of 128, three segments, 2048 rows 127 and 150; 16 ranks of three segments,
  // 2048 rows 64 and 58; 1000 rows are alike), as far as requests are long and, for B, as the parts of h fit 64 KB of LDS, or half
  // of the rows do (ranks of 128, gate and up of 17408, 5000 rows in tiles of 32 474 us, of 16 556).
  const bool large = (int64_t)a.T > 16 * (int64_t)a.S && a.T >= 1024 && a.rank > 32;
  const int ranks = a.rank * (a.mode == BTF_GEMV_SWIGLU ? 2 : 1), b_rows = !large ? 16 : ranks <= 128 ? 64 : ranks <= 256 ? 32 : 16;
  int slices;
  const int rc = large ? lora_shrink<BF, 4>(a, segs, nseg, slices, st) : lora_shrink<BF, 1>(a, segs, nseg, slices, st);
  if (rc != BTF_OK) return rc;
  return b_rows == 64   ? lora_expand<BF, 4>(a, segs, nseg, slices, st)
         : b_rows == 32 ? lora_expand<BF, 2>(a, segs, nseg, slices, st)
                        : lora_expand<BF, 1>(a, segs, nseg, slices, st);
}

}  // namespace

int64_t lora_ws_bytes(int S, int T, int K, int rank, int nseg) {
  (void)S;
  return ws_rows(T, K, nseg) * rank * 4;
}

// Workgroups of a launch at most (apart from small ones, which are cut further): a tile by 1024 outputs.
int64_t lora_most_groups(int S, int T, int64_t outs, int nseg) {
  const int64_t tiles = T <= 4 * (int64_t)S ? T : (int64_t)T / 16 + S;
  return tiles * (outs / (4 * kChunk) + nseg);
}

int lora(const btf_lora& a, const btf_lora_seg* s, int nseg, hipStream_t st) {
  Segs segs{};
  for (int i = 0; i < nseg; ++i) segs.s[i] = s[i];
  return a.type == BTF_BF16 ? lora_any<true>(a, segs, nseg, st) : lora_any<false>(a, segs, nseg, st);
}

}  // namespace btfhip
