// attn.hip -- attention of a step's rows over the paged KV cache
// (btf_hip_launch_paged_attention; gfx950).
//
// One wave per row and head: the keys one after the other with the running
// maximum and sum of the softmax, the head's values spread over the lanes.
#include <string>

#include "../../include/btf/hip_abi.h"
#include "common.h"

namespace btfhip {
namespace {

template <bool BF>
__device__ __forceinline__ float from16(uint16_t h) {
  if (BF) return __uint_as_float((uint32_t)h << 16);
  return h2f(h);
}

template <int D, bool BF>
__global__ void __launch_bounds__(64) attn_row_kernel(btf_paged_attention a, btf_kv_cache kv) {
  constexpr int E = D / 64;
  const int lane = threadIdx.x, t = blockIdx.x, h = blockIdx.y;
  if (t >= a.row0[a.S]) return;
  int lo = 0, hi = a.S - 1;  // the last request with row0 <= t that has rows
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (a.row0[mid] <= t) lo = mid;
    else hi = mid - 1;
  }
  const int s = lo, i = t - a.row0[s], n = a.row0[s + 1] - a.row0[s];
  const int kvh = h / (a.heads / kv.heads);
  const long long cap = (long long)a.ldt * kv.page;
  const int len = (int)min((long long)a.kv_len[s], cap), ctx = a.kv_len[s] - n;
  const bool tree = a.tree && n <= BTF_TREE_NODES;
  const unsigned long long bits = tree ? a.tree[t] : 0;
  const uint16_t* q = static_cast<const uint16_t*>(a.q) + (size_t)t * a.ldq + h * D + lane * E;
  float qf[E], o[E] = {};
#pragma unroll
  for (int e = 0; e < E; ++e) qf[e] = from16<BF>(q[e]);
  float m = -INFINITY, l = 0.f;
  for (int j = 0; j < len; ++j) {
    const int nj = j - ctx;
    if (nj >= 0 && (tree ? !(bits >> nj & 1) : nj > i)) continue;
    const int pg = a.table[(size_t)s * a.ldt + j / kv.page];
    if (pg < 0 || pg >= kv.pages) continue;
    const size_t at = (size_t)pg * kv.page_stride + (size_t)kvh * kv.head_stride + (size_t)(j % kv.page) * kv.tok_stride +
                      lane * E;
    float x = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) x += qf[e] * from16<BF>(static_cast<const uint16_t*>(kv.k)[at + e]);
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) x += __shfl_xor(x, d, 64);
    x *= a.scale;
    if (x == -INFINITY) continue;
    const float mn = fmaxf(m, x), c = __expf(m - mn), p = __expf(x - mn);
    l = l * c + p;
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = o[e] * c + p * from16<BF>(static_cast<const uint16_t*>(kv.v)[at + e]);
    m = mn;
  }
  float* y = a.out + (size_t)t * a.ldo + h * D + lane * E;
#pragma unroll
  for (int e = 0; e < E; ++e) y[e] = l == 0.f ? 0.f : o[e] / l;
}

template <int D, bool BF>
void attn_go(const btf_paged_attention& a, const btf_kv_cache& kv, hipStream_t st) {
  hipLaunchKernelGGL((attn_row_kernel<D, BF>), dim3(a.T, a.heads), dim3(64), 0, st, a, kv);
}

}  // namespace

int64_t paged_attention_ws_bytes(int S, int T, int heads, const btf_kv_cache& kv) { return 0; }

int paged_attention(const btf_paged_attention& a, const btf_kv_cache& kv, hipStream_t st, const DevState& ds) {
  const bool bf = kv.type == BTF_BF16;
  if (kv.dim == 64) bf ? attn_go<64, true>(a, kv, st) : attn_go<64, false>(a, kv, st);
  else if (kv.dim == 128) bf ? attn_go<128, true>(a, kv, st) : attn_go<128, false>(a, kv, st);
  else bf ? attn_go<256, true>(a, kv, st) : attn_go<256, false>(a, kv, st);
  return launch_status("attn_row_kernel");
}

}  // namespace btfhip
