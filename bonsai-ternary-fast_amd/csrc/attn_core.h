// attn_core.h -- the attention kernels that launch_paged_attention (attn.hip) and
// launch_shared_attention (shared.hip) have in common: one item, a tile of rows over a piece of keys, by one workgroup.
// A kernel's argument is a struct that begins with the two argument structs (Args) and finds the item of a workgroup:
//   template <int R, bool SCALAR> bool find(int id, Req& q) const   (false: there is none)
#pragma once
#include "common.h"

namespace btfhip {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));

constexpr int kWaves = 4;
constexpr int kKeys = 32;      // keys of a block
constexpr int kStep = kWaves * kKeys;
// Items that a launch is cut into, for tiles of R rows.
constexpr int target(int R) { return R <= 32 ? 1536 : 1024; }
// Of launches with less work, pieces of up to `least` keys where that leaves one for each of 512 workgroups, the two a CU
// that every instance has room for (attn_tile_kernel with tiles of 64 rows has room for three at heads of 128, five at 64;
// one number serves all): a tile of many rows costs more to begin, leave and join than a few blocks of keys (694 rows of 24
// heads of 256 behind 157 tokens 57 us in pieces of 128 keys, 47 so; trees of up to 57 nodes of three requests over 6000
// keys 63 and 48, of 49 nodes of five requests, heads of 64, 26 and 27; 25 rows of one request over 16000 keys, 8 KV
// heads of 128, 33 and 24). Up to 16 rows the smallest pieces (the smallest calls, 11.5 us, take 13 in pieces of 256 or
// 512 keys).
constexpr int least(int R) { return R <= 16 ? kStep : 512; }
constexpr int kPlaces = 512;
// Keys of a request at most: the loops count some blocks beyond the last key in 32 bits.
constexpr int kMostKeys = 0x7fffffff & ~8191;

template <bool BF>
__device__ __forceinline__ float from16(uint16_t h) {
  if (BF) return __uint_as_float((uint32_t)h << 16);
  return h2f(h);
}

template <bool BF>
__device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
  if (BF) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0, 0);
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
}

// Two values rounded to 16 bits, and what the rounding left. (The empty asm keeps the
// compiler from rounding a second time for the difference.)
template <bool BF>
__device__ __forceinline__ uint32_t round2(float& x, float& y) {
  uint32_t u;
  if (BF) {
    typedef __bf16 b2 __attribute__((ext_vector_type(2)));
    u = __builtin_bit_cast(uint32_t, b2{(__bf16)x, (__bf16)y});
    asm("" : "+v"(u));
    x -= __uint_as_float(u << 16);
    y -= __uint_as_float(u & 0xffff0000u);
    return u;
  }
  typedef _Float16 h2 __attribute__((ext_vector_type(2)));
  u = __builtin_bit_cast(uint32_t, h2{(_Float16)x, (_Float16)y});
  asm("" : "+v"(u));
  const h2 r = __builtin_bit_cast(h2, u);
  x = __builtin_fmaf((float)r[0], -1.f, x);  // (one instruction, with the conversion)
  y = __builtin_fmaf((float)r[1], -1.f, y);
  return u;
}

// 2^x in one instruction (1 ulp; below 2^-126 it gives 0, which is no weight here).
__device__ __forceinline__ float fast_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

// Max / sum over the four lane groups (lanes l, l ^ 16, l ^ 32, l ^ 48).
__device__ __forceinline__ float groups_max(float v) {
  auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
}
__device__ __forceinline__ float groups_sum(float v) {
  auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(a[0]) + __uint_as_float(a[1]);
}

// A request as an item sees it.
struct Req {
  int s, row0, n;         // request, its first row, its rows
  int len, ctx;           // keys; keys before its rows (negative: its first rows see nothing)
  int tiles, pieces;      // row tiles, pieces of its keys
  int local;              // the item's (or row's) number in the request's items
  int slot;               // workspace slot of the request's first item (cut)
  int C;                  // keys of a piece
  int begin;              // the first piece's first key
  bool tree;              // its rows see what their bits say of the new tokens
  bool cut;               // its items leave their sums in the workspace
};

__device__ __forceinline__ float wave_sum_f(float v) { return groups_sum(row16_sum(v)); }
// Inclusive sum over the lanes (within 16-lane rows by shifts, then the rows before).
__device__ __forceinline__ int wave_scan_i(int v) {
  v += dpp_i<0x111>(v);
  v += dpp_i<0x112>(v);
  v += dpp_i<0x114>(v);
  v += dpp_i<0x118>(v);
  const int t0 = __builtin_amdgcn_readlane(v, 15), t1 = __builtin_amdgcn_readlane(v, 31), t2 = __builtin_amdgcn_readlane(v, 47);
  const int row = (threadIdx.x & 63) >> 4;
  return v + (row > 0 ? t0 : 0) + (row > 1 ? t1 : 0) + (row > 2 ? t2 : 0);
}

// A workspace slot: R rows of D values, then R maxima, then R sums.
template <int D, int R>
constexpr size_t kSlot = (size_t)R * (D + 2);
// With SKIP (attn_tile) a slot has 16, 32, .. rows, as the request's tiles need, and Req::slot counts in 16 rows.
__device__ __forceinline__ int slot_rows(int R, int rows) { return min(R, (rows + 15) & ~15); }

// Row r of the item by the plain loop over keys [k0, k1), by one wave: lane's
// D / 64 values, the row's maximum and sum. Any input.
template <int D, bool BF>
__device__ void plain_row(const btf_paged_attention& a, const btf_kv_cache& kv, const Req& q, int kvh, int row, int k0, int k1,
                          float* o, float& m, float& l) {
  constexpr int E = D / 64;
  const int lane = threadIdx.x & 63, G = a.heads / kv.heads, i = row / G, t = q.row0 + i, h = kvh * G + row % G;
  const bool tree = q.tree;
  const unsigned long long bits = tree ? a.tree[t] : 0;
  const uint16_t* x = static_cast<const uint16_t*>(a.q) + (size_t)t * a.ldq + h * D + lane * E;
  float qf[E];
#pragma unroll
  for (int e = 0; e < E; ++e) qf[e] = from16<BF>(x[e]), o[e] = 0.f;
  m = -INFINITY, l = 0.f;
  for (int j = k0; j < k1; ++j) {
    const int nj = j - q.ctx;
    if (nj >= 0 && (tree ? nj >= 64 || !(bits >> nj & 1) : nj > i)) continue;
    const int pg = a.table[(size_t)q.s * a.ldt + j / kv.page];
    if (pg < 0 || pg >= kv.pages) continue;
    const size_t at = (size_t)pg * kv.page_stride + (size_t)kvh * kv.head_stride + (size_t)(j % kv.page) * kv.tok_stride +
                      lane * E;
    float d = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) d += qf[e] * from16<BF>(static_cast<const uint16_t*>(kv.k)[at + e]);
    d = wave_sum_f(d) * (a.scale * 1.4426950408889634f);
    if (d == -INFINITY) continue;
    const float mn = fmaxf(m, d), c = fast_exp2(m - mn), p = fast_exp2(d - mn);
    l = l * c + p;
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = o[e] * c + p * from16<BF>(static_cast<const uint16_t*>(kv.v)[at + e]);
    m = mn;
  }
}

// A block's scores s of the lane's row before their scale (tiles 0 and 1: keys 8 g ..
// 8 g + 7): the running base m (in powers of two, as the scores times c2 > 0 are), the
// lane's share of the sum and the values so far scaled to the new base, and the
// probabilities 2^(score - m) in 16-bit parts. The base follows the scores only when it
// has to, so that the values are rarely scaled. Sums and values go with it: the joins
// need not know where it is.
// bf16: the running maximum, moved when it is more than kLag below. A part has the
// exponents of 32 bits: a probability of any size has all of its bits.
// fp16: a part ends at 2^-25, so the base stays near the block, not near the row's
// maximum: else a key that takes nearly all of the weight leaves every later key a few
// bits or none (one 11 above 690 others, its V 0: 1e-3 of the output was lost). It is a
// whole number (scaling is exact) and moves when the block's largest probability leaves
// [2^-kLow, 2^15]: up to make that 2^11, down to 2^7. A probability is then off by 2^-22
// of itself or 2^-20 of the largest of its block's 32 keys. Blocks more than kFar below
// the highest base are not followed, so sums stay below 2^71 times the number of keys.
// It costs scaling, the more the wider a row's scores are spread (2048 rows over 8191
// keys, heads of 256, queries and keys normal: 499 -> 504 us, with twice the spread 495
// -> 510, with four times 485 -> 521, part of it the power of fewer zeros).
constexpr float kLag = 8.f, kLow = 5.f, kFar = 48.f;
template <bool BF, int PARTS, int N>
__device__ __forceinline__ void softmax_block(const f32x4 (&s)[2], float c2, float& m, float& high, float& l, f32x4 (&o)[N],
                                              u32x4 (&p)[PARTS]) {
  const float mx = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])),
                         fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
  const float mn = groups_max(mx) * c2;
  auto rebase = [&](float to, float c) {
    l *= c;
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] *= c;
    m = to;
  };
  if (BF) {
    if (__any(mn > m + kLag)) {
      const float to = fmaxf(m, mn);
      rebase(to, to == -INFINITY ? 1.f : fast_exp2(m - to));
    }
  } else if (__any(fabsf(mn - m - 0.5f * (15.f - kLow)) > 0.5f * (15.f + kLow))) {
    const bool up = mn > m + 15.f, down = mn < m - kLow && mn > high - kFar;
    if (__any(up | down)) {
      const float to = up ? floorf(mn) - 11.f : down ? floorf(mn) - 7.f : m;
      high = fmaxf(high, to);
      rebase(to, to == m ? 1.f : fast_exp2(m - to));
    }
  }
  const float base = m == -INFINITY ? 0.f : m;
  float x[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    x[j] = fast_exp2(__builtin_fmaf(s[j >> 2][j & 3], c2, -base));
    l += x[j];
  }
#pragma unroll
  for (int n = 0; n < PARTS; ++n)
#pragma unroll
    for (int j = 0; j < 4; ++j) p[n][j] = round2<BF>(x[2 * j], x[2 * j + 1]);
}

// Scores of keys key0 .. key0 + 7 that the row (new token tok, -1: none) does not see become -infinity; there are keys
// up to end. A tree's row sees its bits of the new tokens, another's those up to its own. All by selects: the lanes
// differ in everything here, and a branch for each of 16 scores costs more than the arithmetic. A form with branches has
// also been seen to lose the causal mask in one build (the tests of prompts failed; the cause was not found): keep the
// selects.
__device__ __forceinline__ void mask_block(f32x4 (&s)[2], int key0, int end, int ctx, bool tree, int tok,
                                           unsigned long long bits) {
  const int upto = tree ? ctx - 1 : ctx + tok, nj = key0 - ctx;
  const uint32_t later = (uint32_t)(bits >> (nj & 63)), sooner = (uint32_t)(bits << (-nj & 63));
  const uint32_t own = (tree & (nj > -8) & (nj < 64)) ? (nj >= 0 ? later : sooner) : 0u;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const bool see = (key0 + j < end) & ((key0 + j <= upto) | ((own >> j & 1) != 0));
    s[j >> 2][j & 3] = see ? s[j >> 2][j & 3] : -INFINITY;
  }
}

// The scale of the scores in powers of two, as a positive number: the sign goes to Q, and
// zero, with which a masked score's infinity would be NaN, becomes the smallest number
// there is, 2^-149 (2^128 times that, the largest score, is 2^-21 away from zero: a
// weight's relative error of 3e-7 at most).
__device__ __forceinline__ float scale2(float scale) {
  return fmaxf(fabsf(scale) * 1.4426950408889634f, 1.40129846e-45f);
}
__device__ __forceinline__ u32x4 signed_q(u32x4 q, float scale) {
  const uint32_t f = scale < 0.f ? 0x80008000u : 0u;
  return q ^ u32x4{f, f, f, f};
}

// What an item's waves leave for each other.
template <int D, int RT>
struct StreamLds {
  static constexpr int LD = D + 4;  // row of a wave's values, in floats
  float o[kWaves * 16 * RT * LD];
  float m[kWaves][16 * RT], l[kWaves][16 * RT];
  int odd;
};

template <int D, bool BF, int RT>
__device__ __forceinline__ void attn_stream(const btf_paged_attention& a, const btf_kv_cache& kv, const Req& q, StreamLds<D, RT>& lds) {
  constexpr int R = 16 * RT;             // rows of a tile
  constexpr int KS = D / 32;             // steps over the dims in Q K^T
  constexpr int VD = D < 128 ? D / 16 : 8;  // dims that a lane reads of a key of V
  constexpr int VG = D / (16 * VD);      // ... in so many groups of 16 lanes
  constexpr int PARTS = BF ? 3 : 2;      // 16-bit parts of a probability
  constexpr int LD = StreamLds<D, RT>::LD;
  auto& sh_o = lds.o;
  auto& sh_m = lds.m;
  auto& sh_l = lds.l;
  int& sh_odd = lds.odd;
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c16 = lane & 15, g = lane >> 4;
  const int G = a.heads / kv.heads;
  const int kvh = q.local % kv.heads, rest = q.local / kv.heads;
  const int tile = q.tiles - 1 - rest % q.tiles, piece = rest / q.tiles;
  const int nrows = min(R, q.n * G - tile * R);  // of this tile
  const bool tree = q.tree;
  const float c2 = scale2(a.scale);
  // keys: [k0, k1) is the piece, cut behind the last key that any row of the tile sees; all rows see those before `all`
  const int i0 = tile * R / G, i1 = (tile * R + nrows - 1) / G;
  const int kend = tree ? q.len : max(0, min(q.len, q.ctx + i1 + 1));
  const int k0 = q.begin + piece * q.C, k1 = (int)min((unsigned)kend, (unsigned)k0 + (unsigned)q.C);
  const int all = min(kend, tree ? q.ctx : q.ctx + i0 + 1);

  // Q^T: row c16 of row tile rt, dims 32 ks + 8 g ..
  u32x4 qf[RT][KS];
  int tok[RT];                     // the lane's row: its token
  unsigned long long bits[RT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int row = tile * R + rt * 16 + c16;
    const bool live = rt * 16 + c16 < nrows;
    tok[rt] = live ? row / G : -1;
    bits[rt] = tree && live ? a.tree[q.row0 + row / G] : 0;
    const uint16_t* x = static_cast<const uint16_t*>(a.q) + (size_t)(q.row0 + row / G) * a.ldq + (kvh * G + row % G) * D + 8 * g;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) qf[rt][ks] = live ? signed_q(*reinterpret_cast<const u32x4*>(x + 32 * ks), a.scale) : u32x4{0, 0, 0, 0};
  }
  f32x4 o[RT][VG * VD];
  float m[RT], high[RT], l[RT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    m[rt] = high[rt] = -INFINITY, l[rt] = 0.f;
#pragma unroll
    for (int i = 0; i < VG * VD; ++i) o[rt][i] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  const uint16_t* kp = static_cast<const uint16_t*>(kv.k) + (size_t)kvh * kv.head_stride;
  const uint16_t* vp = static_cast<const uint16_t*>(kv.v) + (size_t)kvh * kv.head_stride;
  const int* tab = a.table + (size_t)q.s * a.ldt;
  const int sh = __builtin_ctz(kv.page), last = (q.len - 1) >> sh;
  // the lane's key of K in a block (tile 0; tile 1: 4 on) and first key of V
  const int kk = 8 * (c16 >> 2) + (c16 & 3), kv0 = 8 * g;
  auto page_of = [&](int key) {  // page id of a key, -1: none
    const int p = key < q.len ? tab[min(key >> sh, last)] : -1;
    return p >= 0 && p < kv.pages ? p : -1;
  };
  u32x4 kf[2][KS];
  auto load_k = [&](int kb, int pg) {
    const uint16_t* x = kp + (size_t)max(pg, 0) * kv.page_stride + (size_t)((kb + kk) & (kv.page - 1)) * kv.tok_stride + 8 * g;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) kf[t][ks] = *reinterpret_cast<const u32x4*>(x + (size_t)(4 * t) * kv.tok_stride + 32 * ks);
  };
  typedef uint32_t vdw __attribute__((ext_vector_type(VD / 2)));
  vdw vf[VG][8];
  auto load_v = [&](int kb, int pg) {
    const uint16_t* x = vp + (size_t)max(pg, 0) * kv.page_stride + (size_t)((kb + kv0) & (kv.page - 1)) * kv.tok_stride + VD * c16;
#pragma unroll
    for (int i = 0; i < VG; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) vf[i][j] = *reinterpret_cast<const vdw*>(x + (size_t)j * kv.tok_stride + 16 * VD * i);
  };

  int kb = k0 + w * kKeys;
  int pk = kb < k1 ? page_of(kb + kk) : -1, pv = kb < k1 ? page_of(kb + kv0) : -1;
  if (kb < k1) {
    load_k(kb, pk);
    load_v(kb, pv);
  }
  for (; kb < k1; kb += kStep) {
    const int nb = kb + kStep;
    const bool more = nb < k1;
    int npk = -1, npv = -1;
    if (more) npk = page_of(nb + kk), npv = page_of(nb + kv0);
    f32x4 s[RT][2];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        s[rt][t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) s[rt][t] = mfma<BF>(kf[t][ks], qf[rt][ks], s[rt][t]);
      }
    // a block that some row does not see all of
    const bool edge = kb + kKeys > all || __any(pk < 0 || pv < 0);
    if (edge) {
      const int end = pv >= 0 ? k1 : 0, key0 = kb + kv0;  // keys that there are
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int i = 0; i < VG; ++i) vf[i][j] = key0 + j < end ? vf[i][j] : vdw(0);
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) mask_block(s[rt], key0, end, q.ctx, tree, tok[rt], bits[rt]);
    }
    if (more) load_k(nb, npk);
    // the running maximum and sum; probabilities in 16-bit parts, keys 8 g .. 8 g + 7
    u32x4 p[RT][PARTS];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) softmax_block<BF, PARTS>(s[rt], c2, m[rt], high[rt], l[rt], o[rt], p[rt]);
    // O^T += V^T P^T: dim VD c16 + e of each lane group's eight keys
#pragma unroll
    for (int i = 0; i < VG; ++i)
#pragma unroll
      for (int e = 0; e < VD; ++e) {
        u32x4 vt;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          vt[j] = __builtin_amdgcn_perm(vf[i][2 * j + 1][e >> 1], vf[i][2 * j][e >> 1], (e & 1) ? 0x07060302u : 0x05040100u);
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
          for (int n = 0; n < PARTS; ++n) o[rt][i * VD + e] = mfma<BF>(vt, p[rt][n], o[rt][i * VD + e]);
      }
    if (more) load_v(nb, npv);
    pk = npk, pv = npv;
  }

  // join the waves
  if (threadIdx.x == 0) sh_odd = 0;
  __syncthreads();
  bool odd = false;
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    l[rt] = groups_sum(l[rt]);
    float chk = l[rt];
    if (g == 0) sh_m[w][rt * 16 + c16] = m[rt], sh_l[w][rt * 16 + c16] = l[rt];
    float* y = sh_o + (size_t)(w * R + rt * 16 + c16) * LD;
#pragma unroll
    for (int i = 0; i < VG; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) {  // row r of the MFMA tiles: dim VD (4 g + r) + e
#pragma unroll
        for (int e = 0; e < VD; e += 4) {
          const f32x4* t = o[rt] + i * VD + e;
          const f32x4 v = {t[0][r], t[1][r], t[2][r], t[3][r]};
          chk += (v[0] - v[0]) + (v[1] - v[1]) + (v[2] - v[2]) + (v[3] - v[3]);
          *reinterpret_cast<f32x4*>(y + 16 * VD * i + VD * (4 * g + r) + e) = v;
        }
      }
    odd |= !(fabsf(chk) < INFINITY);  // (x - x is NaN for an infinity and for NaN)
  }
  if (__any(odd) && lane == 0) sh_odd = 1;
  __syncthreads();

  const bool cut = q.cut;
  float* slot = nullptr;
  if (cut) slot = static_cast<float*>(a.ws) + (size_t)(q.slot + q.local) * kSlot<D, R>;
  if (sh_odd) {
    for (int r = w; r < nrows; r += kWaves) {
      constexpr int E = D / 64;
      float po[E], pm, pl;
      const int row = tile * R + r;
      plain_row<D, BF>(a, kv, q, kvh, row, k0, max(k0, k1), po, pm, pl);
      float* y = cut ? slot + (size_t)r * D : a.out + (size_t)(q.row0 + row / G) * a.ldo + (kvh * G + row % G) * D;
#pragma unroll
      for (int e = 0; e < E; ++e) y[lane * E + e] = cut ? po[e] : pl == 0.f ? 0.f : po[e] / pl;
      if (cut && lane == 0) slot[R * D + r] = pm, slot[R * D + R + r] = pl;
    }
    return;
  }
  constexpr int TPR = D / 4, RPP = 64 * kWaves / TPR;  // threads per row (4 values each), rows at a time
  const int d4 = (threadIdx.x % TPR) * 4;
  for (int r = threadIdx.x / TPR; r < nrows; r += RPP) {
    float top = sh_m[0][r];
#pragma unroll
    for (int i = 1; i < kWaves; ++i) top = fmaxf(top, sh_m[i][r]);
    const float base = top == -INFINITY ? 0.f : top;
    float sum = 0.f;
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < kWaves; ++i) {
      const float c = fast_exp2(sh_m[i][r] - base);
      sum += c * sh_l[i][r];
      v += c * *reinterpret_cast<const f32x4*>(sh_o + (size_t)(i * R + r) * LD + d4);
    }
    const int row = tile * R + r;
    if (cut) {
      *reinterpret_cast<f32x4*>(slot + (size_t)r * D + d4) = v;
      if (d4 == 0) slot[R * D + r] = top, slot[R * D + R + r] = sum;
    } else {
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
      *reinterpret_cast<f32x4*>(a.out + (size_t)(q.row0 + row / G) * a.ldo + (kvh * G + row % G) * D + d4) = v * inv;
    }
  }
}

// ---- many rows: K and V through LDS ----
// A workgroup's 4 waves have 16 or 32 rows each (RT MFMA tiles, which share every operand
// of K and V; one for heads of 256, whose sums take twice the registers) and walk the
// same keys, 32 at a time, from two buffers in LDS: the next block is on its way to
// one while the other is worked on. K's rows lie in the order of the score tiles'
// rows, their 16-byte chunks turned by the row, so that the 16 rows that a lane group
// reads at once lie in different banks. V is read by the transposing LDS read: 16
// lanes read 4 keys of 16 dims and get one dim's 4 keys each; its rows are turned by
// 32 bytes for the same reason.
__device__ __forceinline__ u32x2 read_tr(const void* p) {
  typedef short s4 __attribute__((ext_vector_type(4)));
  typedef __attribute__((address_space(3))) s4 lds_s4;
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)p));
}

// 16 bytes a lane from base + off to LDS, 64 lanes in a row from `to` (the same in all lanes). As asm, which has no
// output and whose end `landed` waits for: the compiler would wait for the builtin's end before the next read of any of
// LDS, the other buffer's too (2048 rows over 6143 keys 602 us).
__device__ __forceinline__ void to_lds(const void* base, uint32_t off, const void* to) {
  const uint32_t lds = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const char*)to;
  asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" : : "v"(off), "s"(base), "{m0}"(__builtin_amdgcn_readfirstlane(lds)) : "memory");
}
__device__ __forceinline__ void to_lds(const void* from, const void* to) {
  const uint32_t lds = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const char*)to;
  asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, off" : : "v"(from), "{m0}"(__builtin_amdgcn_readfirstlane(lds)) : "memory");
}
__device__ __forceinline__ void landed() { asm volatile("s_waitcnt vmcnt(0)" : : : "memory"); }

// The thread's number, of which the compiler does not know that it had it before: what
// follows from it is worked out anew and takes no registers in the loop.
__device__ __forceinline__ int fresh_tid() {
  int t = threadIdx.x;
  asm volatile("" : "+v"(t));
  return t;
}

// The launch's arguments, with which those of every kernel here begin, read again: what only the end needs is not kept
// in scalar registers over the loop.
struct Args {
  btf_paged_attention a;
  btf_kv_cache kv;
};
typedef __attribute__((address_space(4))) const Args* args_p;
__device__ __forceinline__ Args fresh_args() {
  args_p p = (args_p)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  Args g;
  __builtin_memcpy(&g, (const Args*)p, sizeof g);
  return g;
}

template <int D>
struct TileLds {
  u32x4 k[2][kKeys * D / 8], v[2][kKeys * D / 8];
};

// SKIP: waves whose rows there are not load their share and work nothing out.
template <int D, bool BF, int RT, bool SKIP>
__device__ __forceinline__ void attn_tile(const btf_paged_attention& a, const btf_kv_cache& kv, const Req& q, TileLds<D>& lds) {
  constexpr int NW = kWaves, RW = 16 * RT, R = NW * RW;
  constexpr int KS = D / 32;
  constexpr int DT = D / 16;            // dim tiles of the values
  constexpr int DB = 4, KB = 2;         // ... read at a time, and steps of K
  constexpr int PARTS = BF ? 3 : 2;
  constexpr int CH = D / 8;             // 16-byte chunks of a row
  constexpr int NC = kKeys * CH / (64 * NW);  // of a block, for each thread
  auto& sh_k = lds.k;
  auto& sh_v = lds.v;
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) & (NW - 1);
  const int c16 = lane & 15, g = lane >> 4;
  const int G = a.heads / kv.heads;
  const int kvh = q.local % kv.heads, rest = q.local / kv.heads;
  const int tile = q.tiles - 1 - rest % q.tiles, piece = rest / q.tiles;
  const int nrows = min(R, q.n * G - tile * R);
  const bool tree = q.tree;
  const float c2 = scale2(a.scale);
  const int i0 = tile * R / G, i1 = (tile * R + nrows - 1) / G;
  const int kend = tree ? q.len : max(0, min(q.len, q.ctx + i1 + 1));
  const int k0 = q.begin + piece * q.C, k1 = (int)min((unsigned)kend, (unsigned)k0 + (unsigned)q.C);
  const int all = min(kend, tree ? q.ctx : q.ctx + i0 + 1);

  u32x4 qf[RT][KS];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int r = w * RW + rt * 16 + c16, row = tile * R + r;
    const bool live = r < nrows;
    const uint16_t* x = static_cast<const uint16_t*>(a.q) + (size_t)(q.row0 + row / G) * a.ldq + (kvh * G + row % G) * D + 8 * g;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
      qf[rt][ks] = live ? signed_q(*reinterpret_cast<const u32x4*>(x + 32 * ks), a.scale) : u32x4{0, 0, 0, 0};
  }
  f32x4 o[RT][DT];
  float m[RT], high[RT], l[RT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    m[rt] = high[rt] = -INFINITY, l[rt] = 0.f;
#pragma unroll
    for (int i = 0; i < DT; ++i) o[rt][i] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  const uint16_t* kp = static_cast<const uint16_t*>(kv.k) + (size_t)kvh * kv.head_stride;
  const uint16_t* vp = static_cast<const uint16_t*>(kv.v) + (size_t)kvh * kv.head_stride;
  const int* tab = a.table + (size_t)q.s * a.ldt;
  const int sh = __builtin_ctz(kv.page), last = (q.len - 1) >> sh;
  // Pages of a block's two halves. They are looked up two blocks ahead (lanes 0 and 1, by a vector load that comes
  // before the block's own: waiting for those waits for it).
  int p0 = -1, p1 = -1, ahead = -1;
  auto look = [&](int kb) {
    const int key = kb + 16 * (lane & 1);
    ahead = -1;
    if (key < q.len) ahead = tab[min(key >> sh, last)];
  };
  auto take = [&] {
    p0 = __builtin_amdgcn_readlane(ahead, 0), p1 = __builtin_amdgcn_readlane(ahead, 1);
    if (p0 >= kv.pages) p0 = -1;
    if (p1 >= kv.pages) p1 = -1;
  };
  // A block goes from memory to LDS with no register between: a wave's load fills 64 chunks in a row, each lane says
  // where its chunk comes from. A half's start is in scalar registers, the lane's place in it the same for every block.
  auto key_of = [](int row) { return 8 * (row >> 2 & 3) + 4 * (row >> 4) + (row & 3); };  // of a row of K in LDS
  uint32_t off_k[NC], off_v[NC];
#pragma unroll
  for (int n = 0; n < NC; ++n) {
    const int c = threadIdx.x + 64 * NW * n, row = c / CH, ch = c % CH;
    const int turn_k = D == 64 ? row >> 1 & 7 : row & 15, turn_v = 2 * ((4 * (row >> 3) + (row & 3)) & (DT - 1));
    off_k[n] = 2 * ((uint32_t)(key_of(row) & 15) * (uint32_t)kv.tok_stride + 8 * (ch ^ turn_k));
    off_v[n] = 2 * ((uint32_t)(row & 15) * (uint32_t)kv.tok_stride + 8 * (ch ^ turn_v));
  }
  auto load = [&](int kb, int buf) {
    const uint32_t tok = (uint32_t)kv.tok_stride;  // (at most 2^24, and 256 tokens a page)
    const size_t b0 = (size_t)max(p0, 0) * kv.page_stride + (uint32_t)(kb & (kv.page - 1)) * tok;
    const size_t b1 = (size_t)max(p1, 0) * kv.page_stride + (uint32_t)((kb + 16) & (kv.page - 1)) * tok;
#pragma unroll
    for (int n = 0; n < NC; ++n) {
      const int c0 = 64 * (w + NW * n), row = (D == 64 ? c0 + lane : c0) / CH;  // (a wave's rows share a half from 128 dims on)
      const uint16_t *k = kp + (key_of(row) < 16 ? b0 : b1), *v = vp + (row < 16 ? b0 : b1);
      if constexpr (D == 64) {
        to_lds(reinterpret_cast<const char*>(k) + off_k[n], &sh_k[buf][c0]);
        to_lds(reinterpret_cast<const char*>(v) + off_v[n], &sh_v[buf][c0]);
      } else {
        to_lds(k, off_k[n], &sh_k[buf][c0]);
        to_lds(v, off_v[n], &sh_v[buf][c0]);
      }
    }
  };
  auto finish = [&](int kb, int buf) {  // the block has landed; what no row sees of it is cleared by who loaded it
    landed();
    if (p0 < 0 || p1 < 0 || kb + kKeys > k1)
#pragma unroll
      for (int n = 0; n < NC; ++n) {
        const int c = threadIdx.x + 64 * NW * n, j = c / CH, key = key_of(j);
        if ((key < 16 ? p0 : p1) < 0 || kb + key >= k1) sh_k[buf][c] = u32x4{0, 0, 0, 0};
        if ((j < 16 ? p0 : p1) < 0 || kb + j >= k1) sh_v[buf][c] = u32x4{0, 0, 0, 0};
      }
  };
  // the lane's places in a buffer: K chunk g of its row in score tile 0, V's key 8 g + c16 / 4 and dims 4 (c16 % 4) ..
  const uint32_t at_k = c16 * CH * 16 + ((g ^ (D == 64 ? c16 >> 1 & 7 : c16)) << 4);
  const uint32_t at_v = (8 * g + (c16 >> 2)) * CH * 16 + (((4 * g + (c16 >> 2)) & (DT - 1)) << 5) + 8 * (c16 & 3);
  if (k0 < k1) {
    look(k0);
    take();
    look(k0 + kKeys);
    load(k0, 0);
    finish(k0, 0);
  }
  u32x4 p[RT][PARTS];
  // scores, softmax and probabilities of the block at kb, in buffer buf; its pages
  auto scores = [&](int kb, int buf, int h0, int h1) {
    const char* bk = reinterpret_cast<const char*>(sh_k[buf]);
    u32x4 kf[2][2][KB];
    auto read_k = [&](int k) {
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < KB; ++i)
          kf[k / KB & 1][t][i] = *reinterpret_cast<const u32x4*>(bk + (at_k ^ (k + i) << 6) + t * 16 * CH * 16);
    };
    read_k(0);
    f32x4 s[RT][2];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) s[rt][t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < KS; k += KB) {
      if (k + KB < KS) read_k(k + KB);
      __builtin_amdgcn_sched_barrier(0);  // the next reads are on their way before these products
#pragma unroll
      for (int i = 0; i < KB; ++i)
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int rt = 0; rt < RT; ++rt) s[rt][t] = mfma<BF>(kf[k / KB & 1][t][i], qf[rt][k + i], s[rt][t]);
      __builtin_amdgcn_sched_barrier(0);
    }
    if (kb + kKeys > all || h0 < 0 || (h1 < 0 && kb + 16 < k1)) {
      // (what the rows see is looked up here, not kept in registers over the loop)
      const int tid = fresh_tid(), key0 = kb + 8 * (tid >> 4 & 3);
      const int end = ((tid >> 4 & 3) < 2 ? h0 : h1) >= 0 ? k1 : 0;  // keys that there are
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        const int r = (tid >> 6) * RW + rt * 16 + (tid & 15), tok = r < nrows ? (tile * R + r) / G : -1;
        mask_block(s[rt], key0, end, q.ctx, tree, tok, tree && tok >= 0 ? fresh_args().a.tree[q.row0 + tok] : 0);
      }
    }
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) softmax_block<BF, PARTS>(s[rt], c2, m[rt], high[rt], l[rt], o[rt], p[rt]);
  };
  auto values = [&](int buf) {  // O^T += V^T P^T
    const char* bv = reinterpret_cast<const char*>(sh_v[buf]);
    u32x4 vf[2][DB];
    auto read_v = [&](int d0) {
#pragma unroll
      for (int d = 0; d < DB; ++d) {
        const char* x = bv + (at_v ^ (d0 + d) << 5);
        const u32x2 lo = read_tr(x), hi = read_tr(x + 4 * CH * 16);
        vf[d0 / DB & 1][d] = u32x4{lo[0], lo[1], hi[0], hi[1]};
      }
    };
    read_v(0);
    // (these products before another wave's softmax, which then runs in their shadow: trees of 8 requests 186 -> 177 us;
    // with one row tile a wave, heads of 256, it costs: a prompt 481 -> 500)
    if (RT == 2) __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int d0 = 0; d0 < DT; d0 += DB) {
      if (d0 + DB < DT) read_v(d0 + DB);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int n = 0; n < PARTS; ++n)  // (a sum's next product comes after all the others')
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
          for (int rt = 0; rt < RT; ++rt) o[rt][d0 + d] = mfma<BF>(vf[d0 / DB & 1][d], p[rt][n], o[rt][d0 + d]);
    }
    if (RT == 2) __builtin_amdgcn_s_setprio(0);
  };
  int buf = 0;
  for (int kb = k0; kb < k1; kb += kKeys, buf ^= 1) {
    const int h0 = p0, h1 = p1, nb = kb + kKeys;  // (p0 and p1 are this block's until take())
    const bool more = nb < k1;
    __syncthreads();  // this block is in LDS; the other buffer's readers are done
    if (more) {
      take();
      look(nb + kKeys);
      load(nb, buf ^ 1);
    }
    if (!SKIP || w * RW < nrows) {
      scores(kb, buf, h0, h1);
      values(buf);
    }
    if (more) finish(nb, buf ^ 1);
  }

  const bool cut = q.cut;
  float* slot = nullptr;
  bool odd = false;
  const int tid = fresh_tid();
  const Args end = fresh_args();
  const int SR = SKIP ? slot_rows(R, q.n * G) : R;  // rows of the slot
  if (cut) {
    if (SKIP) slot = static_cast<float*>(end.a.ws) + (size_t)q.slot * kSlot<D, 16> + (size_t)q.local * (SR * (D + 2));
    else slot = static_cast<float*>(end.a.ws) + (size_t)(q.slot + q.local) * kSlot<D, R>;
  }
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int r = (tid >> 6) * RW + rt * 16 + (tid & 15), row = tile * R + r, g = tid >> 4 & 3;
    l[rt] = groups_sum(l[rt]);
    float chk = l[rt] - l[rt];
    const float f = cut ? 1.f : l[rt] == 0.f ? 0.f : 1.f / l[rt];
    float* y = cut ? slot + (size_t)r * D : end.a.out + (size_t)(q.row0 + row / G) * end.a.ldo + (kvh * G + row % G) * D;
    const bool live = r < nrows;
#pragma unroll
    for (int i = 0; i < DT; ++i) {
      const f32x4 v = o[rt][i];  // dims 16 i + 4 g ..
      chk += (v[0] - v[0]) + (v[1] - v[1]) + (v[2] - v[2]) + (v[3] - v[3]);
      if (live) *reinterpret_cast<f32x4*>(y + 16 * i + 4 * g) = v * f;
    }
    if (cut && live && g == 0) slot[SR * D + r] = m[rt], slot[SR * D + SR + r] = l[rt];
    odd |= !(chk == 0.f);
  }
  if (!__any(odd)) return;
  __threadfence_block();  // (the rows below are written again by other lanes of this wave)
  const int lane2 = tid & 63, r0 = __builtin_amdgcn_readfirstlane(tid >> 6) * RW;
  for (int r = r0; r < min(nrows, r0 + RW); ++r) {
    constexpr int E = D / 64;
    float po[E], pm, pl;
    const int row = tile * R + r;
    plain_row<D, BF>(end.a, end.kv, q, kvh, row, k0, max(k0, k1), po, pm, pl);
    float* y = cut ? slot + (size_t)r * D : end.a.out + (size_t)(q.row0 + row / G) * end.a.ldo + (kvh * G + row % G) * D;
#pragma unroll
    for (int e = 0; e < E; ++e) y[lane2 * E + e] = cut ? po[e] : pl == 0.f ? 0.f : po[e] / pl;
    if (cut && lane2 == 0) slot[SR * D + r] = pm, slot[SR * D + SR + r] = pl;
  }
}

// The kernels. args.find: the item of a workgroup, false: there is none.
template <int D, bool BF, int RT, class Launch>
__global__ void __launch_bounds__(64 * kWaves) __attribute__((amdgpu_waves_per_eu(D < 256 ? 2 : 1)))
    attn_stream_kernel(Launch args) {
  __shared__ StreamLds<D, RT> sh;
  Req q;
  if (args.template find<16 * RT, false>(blockIdx.x, q)) attn_stream<D, BF, RT>(args.a, args.kv, q, sh);
}
template <int D, bool BF, int RT, class Launch>
__global__ void __launch_bounds__(64 * kWaves) __attribute__((amdgpu_waves_per_eu(2)))
    attn_tile_kernel(Launch args) {
  __shared__ TileLds<D> sh;
  Req q;
  if (args.template find<64 * RT, true>(blockIdx.x, q)) attn_tile<D, BF, RT, false>(args.a, args.kv, q, sh);
}

}  // namespace
}  // namespace btfhip
