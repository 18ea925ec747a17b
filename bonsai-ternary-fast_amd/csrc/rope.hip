// rope.hip -- Q and K head norms, rotary positions and the KV cache write of a
// step's rows (btf_hip_launch_rope_cache; gfx950), and the host's table of
// frequencies.
//
// One head of a row is dim / 4 lanes of a wave (64, 32 or 16), four values a
// lane: the two neighbouring pairs (p, p + 1). In the halves layout a pair is
// (p, p + n_rot / 2), beyond the turned part (n_rot + j, n_rot + j + (dim -
// n_rot) / 2) with the angle 0; in the pairs layout (2p, 2p + 1) throughout. So
// a pair's two values always sit in one lane and no lane needs another's, but
// for the norm's sum of squares (a butterfly over the head's lanes).
//
// Angles: pos * turns in 64 bits and only the fraction of a turn goes on in 32
// (position 10^6 turns 1.6e5 times; in 32 bits the angle would be off by
// 2^-24 of that, 0.06 rad). A lane keeps its cosines and sines for all the heads
// that its wave does.
//
// Bound by HBM for many rows (2048 of 56 heads of 128, 88 MB: 16.8 us, 5.2 TB/s), by the
// launch for one (3.7 us).
#include <algorithm>
#include <cmath>
#include <string>

#include "../../include/btf/hip_abi.h"
#include "common.h"

#pragma clang fp contract(off)

namespace btfhip {
namespace {

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));

template <bool BF>
__device__ __forceinline__ uint16_t to16(float f) {
  uint16_t h;
  if (BF) {
    const __bf16 x = (__bf16)f;
    __builtin_memcpy(&h, &x, 2);
  } else {
    const _Float16 x = (_Float16)f;
    __builtin_memcpy(&h, &x, 2);
  }
  return h;
}

constexpr int kRopeWaves = 4;

// Heads [h0, h1) of the list Q heads, K heads, V heads of one row, by one wave.
// VEC: two neighbouring values of a half (or the lane's four) in one access.
template <int D, bool BF, bool VEC>
__global__ void __launch_bounds__(64 * kRopeWaves) rope_cache_kernel(btf_rope_cache a, btf_kv_cache kv, int per) {
  constexpr int LPH = D / 4, HPW = 64 / LPH;  // lanes per head, heads per wave
  const int lane = threadIdx.x & 63, li = lane % LPH;
  const int t = blockIdx.x;
  if (a.rows && t >= *a.rows) return;
  const int nq = a.q ? a.heads : 0, nk = a.k ? kv.heads : 0;
  const int h0 = (blockIdx.y * kRopeWaves + (threadIdx.x >> 6)) * per * HPW, h1 = min(h0 + per * HPW, nq + 2 * nk);
  if (h0 >= h1) return;
  const int half = a.n_rot / 2, rest = (D - a.n_rot) / 2;
  // the lane's pairs: places of their values, and their turns
  int e0[2], e1[2];
  float cs[2], sn[2];
  bool turn[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int p = 2 * li + i;
    turn[i] = p < half;
    if (a.layout == BTF_ROPE_PAIRS) {
      e0[i] = 2 * p;
      e1[i] = 2 * p + 1;
    } else if (turn[i]) {
      e0[i] = p;
      e1[i] = p + half;
    } else {
      e0[i] = a.n_rot + (p - half);
      e1[i] = e0[i] + rest;
    }
    cs[i] = 1.f;
    sn[i] = 0.f;
    if (turn[i] && h0 < nq + nk) {
      const double x = (double)a.pos[t] * a.turns[p];
      const float f = 2.f * (float)(x - rint(x));
      sincospif(f, &sn[i], &cs[i]);
      cs[i] *= a.mscale;
      sn[i] *= a.mscale;
    }
  }
  const int slot = nk ? a.slot[t] : -1;
  const bool keep = slot >= 0 && slot < kv.pages * kv.page;
  const size_t at = keep ? (size_t)(slot / kv.page) * kv.page_stride + (size_t)(slot % kv.page) * kv.tok_stride : 0;
  for (int h = h0 + lane / LPH; h < h1; h += HPW) {
    const bool isq = h < nq, isv = h >= nq + nk;
    const int hh = isq ? h : isv ? h - nq - nk : h - nq;
    if (!isq && !keep) continue;  // (the lanes of one head go together)
    const float* x = (isq ? a.q + (size_t)t * a.ldq : isv ? a.v + (size_t)t * a.ldv : a.k + (size_t)t * a.ldk) + hh * D;
    const float* norm = isq ? a.q_norm : isv ? nullptr : a.k_norm;
    float u[2], w[2];
    if (VEC && a.layout == BTF_ROPE_PAIRS) {
      typedef float f32x4 __attribute__((ext_vector_type(4)));
      const f32x4 r = *reinterpret_cast<const f32x4*>(x + e0[0]);
      u[0] = r[0], w[0] = r[1], u[1] = r[2], w[1] = r[3];
    } else if (VEC) {
      const f32x2 r = *reinterpret_cast<const f32x2*>(x + e0[0]), q = *reinterpret_cast<const f32x2*>(x + e1[0]);
      u[0] = r[0], u[1] = r[1], w[0] = q[0], w[1] = q[1];
    } else {
      u[0] = x[e0[0]], u[1] = x[e0[1]], w[0] = x[e1[0]], w[1] = x[e1[1]];
    }
    if (norm) {
      float ss = u[0] * u[0] + w[0] * w[0] + u[1] * u[1] + w[1] * w[1];
#pragma unroll
      for (int o = 1; o < LPH; o <<= 1) ss += __shfl_xor(ss, o, LPH);
      const float r = 1.0f / sqrtf(ss / (float)D + a.eps);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        u[i] = u[i] * r * norm[e0[i]];
        w[i] = w[i] * r * norm[e1[i]];
      }
    }
    uint16_t o0[2], o1[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float y0 = u[i], y1 = w[i];
      if (!isv && turn[i]) {
        y0 = u[i] * cs[i] - w[i] * sn[i];
        y1 = u[i] * sn[i] + w[i] * cs[i];
      }
      o0[i] = to16<BF>(y0);
      o1[i] = to16<BF>(y1);
    }
    uint16_t* y = isq ? static_cast<uint16_t*>(a.q_out) + (size_t)t * a.ldqo + hh * D
                      : static_cast<uint16_t*>(isv ? kv.v : kv.k) + at + (size_t)hh * kv.head_stride;
    if (VEC && a.layout == BTF_ROPE_PAIRS) {
      typedef uint16_t u16x4 __attribute__((ext_vector_type(4)));
      *reinterpret_cast<u16x4*>(y + e0[0]) = u16x4{o0[0], o1[0], o0[1], o1[1]};
    } else if (VEC) {
      *reinterpret_cast<u16x2*>(y + e0[0]) = u16x2{o0[0], o0[1]};
      *reinterpret_cast<u16x2*>(y + e1[0]) = u16x2{o1[0], o1[1]};
    } else {
      y[e0[0]] = o0[0], y[e0[1]] = o0[1], y[e1[0]] = o1[0], y[e1[1]] = o1[1];
    }
  }
}

template <int D, bool BF>
void rope_go(const btf_rope_cache& a, const btf_kv_cache& kv, bool vec, hipStream_t st) {
  const int nh = (a.q ? a.heads : 0) + (a.k ? 2 * kv.heads : 0);
  const int slots = (nh + 64 / (D / 4) - 1) / (64 / (D / 4));  // a wave's passes over the heads, all of them
  // Passes of a wave: one, but for rows that leave 8192 waves with more, up to 8: a wave works its angles out once
  // (2048 rows of 56 heads of 128: 25.8 us with one pass, 19.7 with two, 18.0 with seven).
  const int per = (int)std::min<int64_t>(8, std::max<int64_t>(1, (int64_t)a.T * slots / 8192));
  const dim3 grid(a.T, (slots + kRopeWaves * per - 1) / (kRopeWaves * per));
  if (vec) hipLaunchKernelGGL((rope_cache_kernel<D, BF, true>), grid, dim3(64 * kRopeWaves), 0, st, a, kv, per);
  else hipLaunchKernelGGL((rope_cache_kernel<D, BF, false>), grid, dim3(64 * kRopeWaves), 0, st, a, kv, per);
}

}  // namespace

int rope_cache(const btf_rope_cache& a, const btf_kv_cache& kv, bool vec, hipStream_t st) {
  const bool bf = kv.type == BTF_BF16;
  if (kv.dim == 64) bf ? rope_go<64, true>(a, kv, vec, st) : rope_go<64, false>(a, kv, vec, st);
  else if (kv.dim == 128) bf ? rope_go<128, true>(a, kv, vec, st) : rope_go<128, false>(a, kv, vec, st);
  else bf ? rope_go<256, true>(a, kv, vec, st) : rope_go<256, false>(a, kv, vec, st);
  return launch_status("rope_cache_kernel");
}

// The frequencies of the pairs in turns per position (host).
int rope_table(int n_rot, double base, const btf_rope_scale* sc, double* turns, float* mscale) {
  const double kTwoPi = 6.283185307179586476925286766559;
  const int kind = sc ? sc->kind : BTF_ROPE_NONE;
  const double f = kind == BTF_ROPE_NONE ? 1.0 : sc->factor;
  if (kind == BTF_ROPE_NTK) base *= std::pow(f, (double)n_rot / (n_rot - 2));
  double low = 0, high = 0;
  if (kind == BTF_ROPE_YARN) {
    // the pair that turns beta times over the trained context
    auto pair = [&](double beta) { return n_rot * std::log(sc->trained / (beta * kTwoPi)) / (2.0 * std::log(base)); };
    low = std::fmax(std::floor(pair(sc->beta_fast)), 0.0);
    high = std::fmin(std::ceil(pair(sc->beta_slow)), n_rot - 1.0);
    if (high <= low) high = low + 1e-3;
  }
  for (int i = 0; i < n_rot / 2; ++i) {
    double w = std::pow(base, -2.0 * i / n_rot);
    if (kind == BTF_ROPE_LINEAR) w /= f;
    if (kind == BTF_ROPE_YARN) {
      const double r = std::fmin(std::fmax((i - low) / (high - low), 0.0), 1.0);
      w = w * (1.0 - r) + w / f * r;
    }
    turns[i] = w / kTwoPi;
  }
  *mscale = kind == BTF_ROPE_YARN ? (float)(0.1 * std::log(f) + 1.0) : 1.0f;
  return BTF_OK;
}

}  // namespace btfhip
