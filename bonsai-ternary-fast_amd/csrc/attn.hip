// attn.hip -- attention of a step's rows over the paged KV cache
// (btf_hip_launch_paged_attention; gfx950).
//
// Work. A request's rows are its new tokens times the G = heads / kv->heads
// query heads of one KV head, in tiles of R; its keys are cut into pieces of C.
// An item, the work of one workgroup, is one (request, KV head, row tile,
// piece). C follows from all requests' lengths (read on the device), so that
// about target(R) items of like size come out whatever the lengths: one long
// request among short ones is cut, the short ones are not. An item of a request
// that is not cut writes out; the others leave (maximum, sum, values) in the
// workspace and attn_join_kernel puts the pieces of a row together.
//
// Inside an item each of 4 waves takes every fourth block of 32 keys, with its
// own running maximum m and sum l of the softmax, and the waves join in LDS at
// the end. Scores come transposed, S^T = K Q^T, from 16x16x32 MFMA: a lane then
// has one row (column of the result) and, of two key tiles, eight keys. Which
// eight is free, as any order of the keys will do if V has the same: tile t row
// m is key 8 (m / 4) + 4 t + m % 4, so lane group g (lanes 16 g ..) holds keys
// 8 g .. 8 g + 7, which is also what the second product wants from it, O^T = V^T
// P^T: no probability changes its lane. V^T's operand, eight keys of one dim, is
// put together from eight 16-byte loads (eight dims of one key) by one byte
// permute per register: lane c of a group reads dims 8 c .. 8 c + 7 and serves
// MFMA e with dim 8 c + e. K and V go from HBM to registers, with no LDS between.
//
// Probabilities are 32-bit; as MFMA takes 16-bit factors they are carried in
// parts, p = hi + lo (+ lo2 for bf16), each the rounding of what the parts
// before leave: 22 and 24 bits (fp16: as far as its small end allows, see softmax_block).
// One part would put 2^-11 or 2^-8 on fp32 output.
//
// What a row does not see takes no part, whatever it holds: masked scores become
// -infinity, V of keys behind the end is cleared. Where V or a score is not
// finite all the same (0 * infinity in a product), the item's result shows it,
// and the item (attn_tile_kernel: the wave's rows of it) is done again one row at a time
// by the plain loop: right, and slow (one NaN in V that all rows see: one token over
// 4097 keys 15 -> 150 us, 2048 rows over 8191 0.5 -> 130 ms).
//
// Which kernel: by the rows that a request has on average for a KV head (tile_rows).
// Up to 16 or 32 (one new token, few heads more), attn_stream_kernel as above: bound
// by HBM once the cache is long (one token each of 32 requests, 2.7 GB of cache: 465
// us, 5.8 TB/s), by the chain of reads when it is short (one token over 4097: 14 us,
// find 1.1, pages and first block 3.4, products 1.8, the waves' join 1.5, the pieces'
// join 3.7). More rows, attn_tile_kernel below: bound by the issue of matrix and vector
// instructions (trees of up to 64 nodes of 8 requests 175 us, matrix units 46 % busy and
// vector 43 %; 2048 rows of heads of 256 over 8191 keys 490-508 us: 4.5e11 operations
// with both parts of P, 0.91 PFLOP/s, 45 % and 30 %). The join of the pieces takes 5 to
// 28 us of these: without pieces 512 tiles of unlike length end one after another.
#include <string>

#include "../../include/btf/hip_abi.h"
#include "attn_core.h"

namespace btfhip {
namespace {

// The request of item `id` (BY_ROW: of row `id`), found by every wave for itself:
// the lanes take 64 requests at a time. False: there is no such item.
// SCALAR: most of the answer in scalar registers (the stream kernel has none to spare).
template <int R, bool BY_ROW, bool SCALAR>
__device__ bool find(const btf_paged_attention& a, const btf_kv_cache& kv, int id, Req& q) {
  const int lane = threadIdx.x & 63, G = a.heads / kv.heads;
  const long long cap = min((long long)a.ldt * kv.page, (long long)kMostKeys);
  auto read = [&](int s, int& r0, int& n, int& len, int& full) {
    r0 = n = len = full = 0;
    if (s < a.S) {
      r0 = max(a.row0[s], 0);
      n = min(a.row0[s + 1], a.T) - r0;
      full = a.kv_len[s];
      len = (int)max(0ll, min((long long)full, cap));
    }
  };
  float work = 0.f;  // (a whole number below 2^24 times its size: the split need not be exact)
  int r0, n, len, full;
  for (int s0 = 0; s0 < a.S; s0 += 64) {
    read(s0 + lane, r0, n, len, full);
    if (n > 0) work += (float)((n * G + R - 1) / R) * (float)len;
  }
  work = wave_sum_f(work) * (float)kv.heads;
  work /= (float)kStep;  // (in the smallest pieces)
  const int C = kStep * __builtin_amdgcn_readfirstlane(
                            max((int)(work / (float)target(R) + 1.f), min(least(R) / kStep, (int)(work / (float)kPlaces + 1.f))));
  int items = 0, slots = 0;  // before the chunk
  for (int s0 = 0; s0 < a.S; s0 += 64) {
    if (a.S > 64) read(s0 + lane, r0, n, len, full);  // (up to 64 requests are still there)
    const int tiles = n > 0 ? (n * G + R - 1) / R : 0, pieces = max(1, (int)((unsigned)(len + C - 1) / (unsigned)C));
    const int mine = kv.heads * tiles * pieces, cut = pieces > 1 ? mine : 0;
    const int upto = wave_scan_i(mine), cuts = wave_scan_i(cut);
    const bool here = BY_ROW ? n > 0 && id >= r0 && id < r0 + n : mine > 0 && id >= items + upto - mine && id < items + upto;
    const unsigned long long who = __ballot(here);
    if (who) {
      const int l = __builtin_ctzll(who);
      auto of = [&](int v) { return SCALAR ? __builtin_amdgcn_readlane(v, l) : __shfl(v, l, 64); };
      q.s = s0 + l;
      q.row0 = __shfl(r0, l, 64);
      q.n = of(n);
      q.len = of(len);
      q.ctx = of(full) - q.n;
      q.tiles = of(tiles);
      q.pieces = of(pieces);
      q.local = id - (BY_ROW ? q.row0 : items + of(upto - mine));
      q.slot = slots + __shfl(cuts - cut, l, 64);
      q.C = C;
      q.begin = 0;
      q.tree = a.tree && q.n <= BTF_TREE_NODES;
      q.cut = q.pieces > 1;
      return true;
    }
    items += __builtin_amdgcn_readlane(upto, 63);
    slots += __builtin_amdgcn_readlane(cuts, 63);
  }
  return false;
}

// The launch's arguments as the kernels take them.
struct Alone : Args {
  template <int R, bool SCALAR>
  __device__ __forceinline__ bool find(int id, Req& q) const {
    return btfhip::find<R, false, SCALAR>(a, kv, id, q);
  }
};

// The pieces of one row of one head put together. Few rows: by the four waves of a
// workgroup, each its share of the pieces (so that many loads are in flight), joined
// in LDS. Many rows (ONE): by one wave.
constexpr int kJoinWaves = 4;
template <int D, int R, bool ONE>
__global__ void __launch_bounds__(64 * kJoinWaves) attn_join_kernel(btf_paged_attention a, btf_kv_cache kv) {
  constexpr int E = D / 64;  // values of a lane
  constexpr int BY = ONE ? 1 : kJoinWaves;  // waves of a row
  typedef float vE __attribute__((ext_vector_type(E)));
  Req q;
  if (!find<R, true, true>(a, kv, blockIdx.x, q) || q.pieces == 1) return;  // the whole workgroup
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int G = a.heads / kv.heads, h = ONE ? blockIdx.y * kJoinWaves + w : blockIdx.y, kvh = h / G;
  if (h >= a.heads) return;
  const int row = q.local * G + h % G, tile = row / R, r = row % R;
  const float* slot = static_cast<const float*>(a.ws) + (size_t)(q.slot + (q.tiles - 1 - tile) * kv.heads + kvh) * kSlot<D, R>;
  const size_t step = (size_t)q.tiles * kv.heads * kSlot<D, R>;
  // the first pieces' maxima, sums and values are all on their way before the first is needed
  constexpr int AT = ONE ? 4 : 8;
  float top = -INFINITY, sum = 0.f, l0 = 0.f;
  if (lane < q.pieces) top = slot[lane * step + R * D + r], l0 = slot[lane * step + R * D + R + r];
  vE x[AT];
  auto read = [&](int i0, int i, int n) {
#pragma unroll
    for (int u = 0; u < AT; ++u)
      x[u] = *reinterpret_cast<const vE*>(slot + (i0 + min(i + u * BY, n - 1)) * step + (size_t)r * D + lane * E);
  };
  const int first = ONE ? 0 : w;
  read(0, first, min(64, q.pieces));
  const float m0 = top;
  for (int i = 64 + lane; i < q.pieces; i += 64) top = fmaxf(top, slot[i * step + R * D + r]);
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
  const float base = top == -INFINITY ? 0.f : top;
  vE v = vE(0.f);
  for (int i0 = 0; i0 < q.pieces; i0 += 64) {
    float c = 0.f;
    if (i0 + lane < q.pieces) {
      const float* y = slot + (i0 + lane) * step + R * D + r;
      c = fast_exp2((i0 ? y[0] : m0) - base);
      sum += c * (i0 ? y[R] : l0);
    }
    const int n = min(64, q.pieces - i0);
    for (int i = first; i < n; i += AT * BY) {
      if (i0 + i != first) read(i0, i, n);
#pragma unroll
      for (int u = 0; u < AT; ++u) {
        const int j = min(i + u * BY, n - 1);
        const float f = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(c), j));
        if (i + u * BY < n) v += f * x[u];
      }
    }
  }
  sum = wave_sum_f(sum);
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  float* y = a.out + (size_t)(q.row0 + q.local) * a.ldo + h * D;
  if (ONE) {
    *reinterpret_cast<vE*>(y + lane * E) = v * inv;
    return;
  }
  __shared__ float sh[kJoinWaves][D];
  *reinterpret_cast<vE*>(&sh[w][lane * E]) = v;
  __syncthreads();
  for (int d = threadIdx.x; d < D; d += 64 * kJoinWaves) {
    float x = sh[0][d];
#pragma unroll
    for (int i = 1; i < kJoinWaves; ++i) x += sh[i][d];
    y[d] = x * inv;
  }
}

// Rows of an item's tile, by the rows that a request has on average for a KV head. (32 rows of heads of 256 do not
// fit a wave's registers with K and V there too, nor do two tiles of 16 a wave in attn_tile_kernel.) 128 rows read K and V
// half as often as 64, which leave room for three workgroups a CU instead of two and half the work in an item: heads of
// 64 gain by 64 rows throughout (2000 rows over 6000 keys, 16 heads, 131 us in tiles of 128, 119 in tiles of 64), heads
// of 128 up to two such tiles (120 rows over 4000 keys 31 and 25, over 16000 143 and 149; 200 over 6000 45 and 52, 2560
// over 16500 276 and 350). Up to 32 rows attn_stream_kernel: 30 rows of 32 requests over up to 32768 keys 489, in tiles of
// 64 rows 545. Rows are those of the launch: one prompt piece beside many single tokens puts
// these into its tiles, too (512 rows behind 2048 tokens and 31 single tokens over 7000 to 16000 keys, 20 / 4 heads of 256:
// 323 us, 71 + 282 apart; 2048 rows, 40 / 8 heads of 128: 619, 267 + 289 apart).
int tile_rows(int S, int T, int heads, const btf_kv_cache& kv) {
  const int64_t rows = (int64_t)T * (heads / kv.heads);
  if (rows <= 16 * (int64_t)S) return 16;
  if (kv.dim == 256) return 64;
  if (rows <= 32 * (int64_t)S) return 32;
  return kv.dim == 64 || rows <= 128 * (int64_t)S ? 64 : 128;
}

// (request, KV head, row tile) of a launch, at most: a request's last tile may be a part of one.
int64_t most_tiles(int S, int T, int heads, const btf_kv_cache& kv) {
  return ((int64_t)T * (heads / kv.heads) / tile_rows(S, T, heads, kv) + S) * kv.heads;
}

template <int D, bool BF>
int attn_go(const btf_paged_attention& a, const btf_kv_cache& kv, hipStream_t st) {
  const int R = tile_rows(a.S, a.T, a.heads, kv);
  // items: one for each tile and target(R) more, or all the pieces that the table has room for
  const int64_t room = ((int64_t)a.ldt * kv.page + kStep - 1) / kStep, most = most_tiles(a.S, a.T, a.heads, kv);
  const dim3 grid((unsigned)(most * room < most + target(R) ? most * room : most + target(R))), blk(64 * kWaves);
  // One wave a row of the join from 2048 rows of heads on: 20 of them, one token over 4097 keys, 17.6 us by one wave each
  // and 14.4 by four; 640 466.9 and 465.1; 13 thousand, trees of 8 requests, 180 and 197; 41 thousand 484 and 560.
  const bool one = (int64_t)a.T * a.heads >= 2048;
  const dim3 join(a.T, one ? (a.heads + kJoinWaves - 1) / kJoinWaves : a.heads);
  int rc = BTF_OK;
  auto joined = [&](auto few, auto many) {
    rc = launch_status("attn kernel");
    if (rc != BTF_OK) return;
    if (one) hipLaunchKernelGGL(many, join, dim3(64 * kJoinWaves), 0, st, a, kv);
    else hipLaunchKernelGGL(few, join, dim3(64 * kJoinWaves), 0, st, a, kv);
    rc = launch_status("attn_join_kernel");
  };
  if (R == 16) {
    hipLaunchKernelGGL((attn_stream_kernel<D, BF, 1, Alone>), grid, blk, 0, st, Alone{{a, kv}});
    joined(attn_join_kernel<D, 16, false>, attn_join_kernel<D, 16, true>);
  } else if (R == 64) {
    hipLaunchKernelGGL((attn_tile_kernel<D, BF, 1, Alone>), grid, blk, 0, st, Alone{{a, kv}});
    joined(attn_join_kernel<D, 64, false>, attn_join_kernel<D, 64, true>);
  } else if constexpr (D < 256) {
    if (R == 32) {
      hipLaunchKernelGGL((attn_stream_kernel<D, BF, 2, Alone>), grid, blk, 0, st, Alone{{a, kv}});
      joined(attn_join_kernel<D, 32, false>, attn_join_kernel<D, 32, true>);
    } else if constexpr (D == 128) {
      hipLaunchKernelGGL((attn_tile_kernel<D, BF, 2, Alone>), grid, blk, 0, st, Alone{{a, kv}});
      joined(attn_join_kernel<D, 128, false>, attn_join_kernel<D, 128, true>);
    }
  }
  return rc;
}

}  // namespace

int64_t paged_attention_most_items(int S, int T, int heads, const btf_kv_cache& kv) {
  return most_tiles(S, T, heads, kv) + target(tile_rows(S, T, heads, kv));
}

// Cut requests have at most 2 target(R) items: a piece of them holds at least C / 2 keys on average, and C is at least
// all the work over target(R).
int64_t paged_attention_ws_bytes(int S, int T, int heads, const btf_kv_cache& kv) {
  const int R = tile_rows(S, T, heads, kv);
  return (int64_t)2 * target(R) * R * (kv.dim + 2) * 4;
}

int paged_attention(const btf_paged_attention& a, const btf_kv_cache& kv, hipStream_t st) {
  const bool bf = kv.type == BTF_BF16;
  if (kv.dim == 64) return bf ? attn_go<64, true>(a, kv, st) : attn_go<64, false>(a, kv, st);
  if (kv.dim == 128) return bf ? attn_go<128, true>(a, kv, st) : attn_go<128, false>(a, kv, st);
  return bf ? attn_go<256, true>(a, kv, st) : attn_go<256, false>(a, kv, st);
}

}  // namespace btfhip
