// shared.hip -- attention of requests of which some share a prefix
// (btf_hip_launch_shared_attention; gfx950).
//
// A row's softmax over prefix and own keys is put together from sums over pieces
// of the keys, (maximum, sum, values) each, so the pieces of the prefix can be done
// for the rows of all requests that see them at once. Two roles: a group's rows are
// one request of many rows over the prefix, all of which they see; each request's
// rows go over its own keys, from where the prefix ends. Both are items of
// attn_core.h, of one launch: a group's items are bound by matrix instructions, a
// request's by HBM, and run beside each other. shared_join_kernel puts a row's pieces
// of both together.
//
// shared_plan_kernel, one workgroup, finds who takes part (a member needs the whole
// prefix before its new rows), cuts both roles into items and writes down which item
// is whose: with hundreds of requests a workgroup that looked for itself, as
// launch_paged_attention's do, would read all lengths several times. Up to 128 requests
// each workgroup does that, and there is no plan. The prefix counts in steps of 32
// keys, a block of the kernels; what is left of it is done with each member's own
// keys, which its row of table has, too.
#include <string>

#include "../../include/btf/hip_abi.h"
#include "attn_core.h"

namespace btfhip {
namespace {

// What the plan found of a group (first in the list) or a request.
struct alignas(16) Found {  // (as the workspace, which need not begin at a line)
  int s, row0, n, len, ctx, tiles, pieces, begin;  // as Req
  int item0, slot0, C;
  int flags;                                       // kTree, kCut
  int group;                                       // of a request that takes part, else -1
  int b, e, whole;                                 // requests of a group; tokens of its prefix
};
constexpr int kTree = 1, kCut = 2;
static_assert(sizeof(Found) == 64, "as wide as a line");

// The parts of the workspace.
struct Ws {
  int* items;     // [1]
  Found* found;   // [groups + S]
  int* map;       // [most] the group or request of an item, as found has them
  int* request;   // [T] of a row, -1: none
  float* slots;   // the groups', then the requests'
  int most;       // items at most
  int units;      // room for slots, in 16 rows
};

struct Plan : Args {
  Ws ws;
  int groups;
  const int *group0, *lead, *shared;
  int R[2];       // rows of a tile of a group, of a request
  int G, cap;     // rows of a token and KV head; tokens that a row of table holds
  int own;        // items that the requests' keys are cut into: kOwnItems, or kFewItems
  int alone;      // no launch before: find_few of so many requests a lane, and the first workgroup writes down `found` for the join
};

constexpr int kPlanThreads = 1024;

// A group's items are long and bound by matrix instructions, a
// request's short and bound by HBM; the groups' come first. 512 workgroups run at a time, two a CU: the groups get their
// share of these by the roles' work (a request's keys count twice, for what an item costs beside its keys), at least half,
// the requests' items fill the rest and follow (64 requests behind 16384 keys with 250 to 1000 of their own, heads of 256:
// the call 85 us, with 512 items of the groups 95, 192 104; a group alone 56 us in 512 items, 69 in 256).
// 256 own items where that leaves no more than run at a time (48 behind 2500 keys with 900 of their own, heads of 256, 42.4
// us in 384, 37.2 so; the trees of 24 behind three prefixes, more items in any case, 110 and 134), and of attn_stream with heads
// of 256, of which a CU runs one workgroup (2 requests of 8200 keys 27.1 and 20.4).
constexpr int kRunning = 512, kOwnItems = 384, kFewItems = 256;
// (Sums of the work in 32 bits are off by 2^-17 at most, for which the last factor stands: there are never more items.)
// Tiles above 16 rows, whose waves take all keys of an item, in pieces of 64 keys where that leaves no more items either and
// makes up to 32 of a request (4 requests behind 1000 keys 16.2 us in pieces of 128, 14.3 in 64, 14.9 in 32; 6 of two groups
// behind 6500 keys, whose rows would have 100 pieces to join, 13.8, 16.5, 16.2).
constexpr int kHalf = kStep / 2, kMostHalves = 32;
__device__ __forceinline__ int piece_keys(float groups, float requests, int role, int R, int own) {
  const float share = (float)kRunning * (groups / (groups + 2.f * requests + 1.f));
  const float items = role ? (float)own : fmaxf(floorf(share), (float)(kRunning / 2));
  const float keys = (role ? requests : groups) * 1.0001f / items;
  return R > 16 && keys <= (float)kHalf ? kHalf : kStep * (int)fminf(keys / (float)kStep + 1.f, 1.6e7f);  // (below 2^31)
}
__device__ __forceinline__ void into_pieces(Found& f, int C) {
  const int keys = max(f.len - f.begin, 0);
  f.C = C < kStep && keys > kMostHalves * kHalf ? kStep : C;
  f.pieces = max(1, (int)((unsigned)(keys + f.C - 1) / (unsigned)f.C));
}

__device__ __forceinline__ int tiles_of(const Plan& p, int n, int R) {  // (R is a power of two)
  return n > 0 ? (int)((unsigned)(n * p.G + R - 1) >> __builtin_ctz(R)) : 0;
}

// A group of requests b .. e - 1 whose rows are r0 .. r1 - 1.
__device__ __forceinline__ Found group_of(const Plan& p, int b, int e, int r0, int r1, int lead, int whole) {
  Found f{};
  f.b = b, f.e = e;
  f.row0 = r0;
  f.n = max(r1 - r0, 0);
  const bool there = lead >= 0 && lead < p.a.S && f.n > 0 && e - b > 1;
  f.s = there ? lead : 0;
  f.whole = whole;
  f.len = f.ctx = there ? min(max(whole, 0), p.cap) & ~31 : 0;
  f.tiles = f.len > 0 ? tiles_of(p, f.n, p.R[0]) : 0;
  f.flags = kCut;
  f.group = -1;
  return f;
}
// Request s alone.
__device__ __forceinline__ Found request_of(const Plan& p, int s, int r0, int r1, int full) {
  Found f{};
  f.s = s;
  f.row0 = min(max(r0, 0), p.a.T);
  f.n = max(min(max(r1, 0), p.a.T) - f.row0, 0);
  f.len = max(0, min(full, p.cap));
  f.ctx = max(full, -1) - f.n;
  f.tiles = tiles_of(p, f.n, p.R[1]);
  f.flags = p.a.tree && f.n <= BTF_TREE_NODES ? kTree : 0;
  f.group = -1;
  return f;
}
__device__ __forceinline__ bool takes_part(const Found& f, const Found& g) {
  return f.n > 0 && g.len > 0 && f.s >= g.b && f.s < g.e && f.ctx >= g.whole && f.row0 >= g.row0 && f.row0 + f.n <= g.row0 + g.n;
}
__device__ __forceinline__ uint64_t work_of(const Found& f) { return (uint64_t)f.tiles * (uint64_t)max(f.len - f.begin, 0); }
// 16 rows of a slot of f's, and what f's items take from slot0 on if they leave their sums. Row starts that do not ascend
// can ask for more than there is (of those that do, no launch does): such a request or group is left out.
__device__ __forceinline__ int units_of(const Plan& p, const Found& f, int role) {
  return slot_rows(p.R[role], f.n * p.G) >> 4;
}
__device__ __forceinline__ void fit(const Plan& p, Found& f, int units) {
  if (f.slot0 < 0 || f.slot0 > p.ws.units - units) f.n = f.tiles = f.pieces = 0, f.flags &= ~kCut;
}
// The last of n ascending numbers that is at most v (0 if none is).
__device__ __forceinline__ int last_at_most(const int* x, int n, int v) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (x[mid] <= v) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// block_scan of two numbers a thread.
__device__ __forceinline__ void scan2(uint64_t (&v)[2], uint64_t (&part)[2][kPlanThreads / 64], uint64_t (&all)[2]) {
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
#pragma unroll
  for (int i = 0; i < 2; ++i) v[i] = wave_scan_u64(v[i]);
  __syncthreads();  // (part may still be read from the scan before)
  if (lane == 63)
#pragma unroll
    for (int i = 0; i < 2; ++i) part[i][w] = v[i];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint64_t sums = wave_scan_u64(lane < kPlanThreads / 64 ? part[i][lane] : 0);
    auto of = [&](int l) {
      return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(sums >> 32), l) << 32 |
             (uint32_t)__builtin_amdgcn_readlane((int)sums, l);
    };
    all[i] = of(kPlanThreads / 64 - 1);
    v[i] += w ? of(w - 1) : 0;
  }
}

// Up to 1024 requests, one a thread, with the groups and row starts in LDS: one trip to memory for all that is read.
__global__ void __launch_bounds__(kPlanThreads) shared_plan_small_kernel(Plan p) {
  __shared__ uint64_t part[2][kPlanThreads / 64];
  __shared__ int sh_row0[kPlanThreads + 1], sh_group0[kPlanThreads], sh_upto[2][kPlanThreads];
  __shared__ Found sh_group[kPlanThreads];
  const btf_paged_attention& a = p.a;
  const int tid = threadIdx.x;
  const bool group = tid < p.groups, request = tid < a.S;
  const int r0 = request ? a.row0[tid] : 0, r1 = request ? a.row0[tid + 1] : 0, full = request ? a.kv_len[tid] : 0;
  const int b = group ? p.group0[tid] : 0, e = group ? p.group0[tid + 1] : 0, lead = group ? p.lead[tid] : 0, whole = group ? p.shared[tid] : 0;
  if (request) sh_row0[tid] = r0;
  if (tid == a.S - 1) sh_row0[a.S] = r1;
  if (group) sh_group0[tid] = b;
  __syncthreads();
  Found f[2];
  if (group) {
    const int gb = min(max(b, 0), a.S), ge = min(max(e, gb), a.S);
    auto row_of = [&](int s) { return min(max(sh_row0[s], 0), a.T); };
    f[0] = group_of(p, gb, ge, row_of(gb), row_of(ge), lead, whole);
    sh_group[tid] = f[0];
  }
  __syncthreads();
  uint64_t v[2] = {group ? work_of(f[0]) : 0, 0}, all[2];
  if (request) {
    f[1] = request_of(p, tid, r0, r1, full);
    if (p.groups > 0) {
      const int g = last_at_most(sh_group0, p.groups, tid);
      if (takes_part(f[1], sh_group[g])) f[1].group = g, f[1].begin = sh_group[g].len;
    }
    v[1] = work_of(f[1]);
  }
  scan2(v, part, all);
  int own[2] = {0, 0}, cut[2] = {0, 0};
#pragma unroll
  for (int role = 0; role < 2; ++role)
    if (role ? request : group) {
      into_pieces(f[role], piece_keys((float)(all[0] * p.kv.heads), (float)(all[1] * p.kv.heads), role, p.R[role], p.own));
      own[role] = p.kv.heads * f[role].tiles * f[role].pieces;
      if (f[role].group >= 0 || f[role].pieces > 1) f[role].flags |= kCut;
      cut[role] = f[role].flags & kCut ? own[role] * units_of(p, f[role], role) : 0;
    }
#pragma unroll
  for (int role = 0; role < 2; ++role) v[role] = (uint64_t)(uint32_t)own[role] | (uint64_t)(uint32_t)cut[role] << 32;
  scan2(v, part, all);
  // (row starts that do not ascend can ask for more items than there are)
  const int first[2] = {0, (int)min((uint32_t)all[0], (uint32_t)p.ws.most)}, behind = (int)(all[0] >> 32);
#pragma unroll
  for (int role = 0; role < 2; ++role) {
    sh_upto[role][tid] = (int)v[role];
    if (role ? request : group) {
      f[role].item0 = first[role] + (int)v[role] - own[role];
      f[role].slot0 = (role ? behind : 0) + (int)(v[role] >> 32) - cut[role];
      fit(p, f[role], cut[role]);
      p.ws.found[role ? p.groups + tid : tid] = f[role];
    }
  }
  if (tid == 0) *p.ws.items = first[1] + (int)min((uint32_t)all[1], (uint32_t)(p.ws.most - first[1]));
  __syncthreads();
#pragma unroll
  for (int role = 0; role < 2; ++role)
    for (int k = tid; k < (int)min((uint32_t)all[role], (uint32_t)(p.ws.most - first[role])); k += kPlanThreads) {
      int lo = 0, hi = (role ? a.S : p.groups) - 1;  // the first one with upto > k
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (sh_upto[role][mid] > k) hi = mid;
        else lo = mid + 1;
      }
      p.ws.map[first[role] + k] = role ? p.groups + lo : lo;
    }
  for (int t = tid; t < a.T; t += kPlanThreads) {
    const int s = last_at_most(sh_row0, a.S, t);
    p.ws.request[t] = t >= sh_row0[s] && t < sh_row0[s + 1] ? s : -1;
  }
}

// Any number of requests and groups.
__global__ void __launch_bounds__(kPlanThreads) shared_plan_kernel(Plan p) {
  __shared__ uint64_t part[kPlanThreads / 64];
  __shared__ int sh_upto[kPlanThreads], sh_row0[kPlanThreads], sh_n[kPlanThreads];
  const btf_paged_attention& a = p.a;
  const btf_kv_cache& kv = p.kv;
  const int tid = threadIdx.x;
  auto row_of = [&](int s) { return min(max(a.row0[s], 0), a.T); };
  uint64_t work[2] = {0, 0};
  for (int g = tid; g < p.groups; g += kPlanThreads) {
    const int b = min(max(p.group0[g], 0), a.S), e = min(max(p.group0[g + 1], b), a.S);
    const Found f = group_of(p, b, e, row_of(b), row_of(e), p.lead[g], p.shared[g]);
    work[0] += work_of(f);
    p.ws.found[g] = f;
  }
  for (int t = tid; t < a.T; t += kPlanThreads) p.ws.request[t] = -1;
  __threadfence_block();
  __syncthreads();
  Found* const mine = p.ws.found + p.groups;
  for (int s = tid; s < a.S; s += kPlanThreads) {
    Found f = request_of(p, s, a.row0[s], a.row0[s + 1], a.kv_len[s]);
    if (p.groups > 0) {
      const int g = last_at_most(p.group0, p.groups, s);
      if (takes_part(f, p.ws.found[g])) f.group = g, f.begin = p.ws.found[g].len;
    }
    work[1] += work_of(f);
    mine[s] = f;
  }
  uint64_t all[2];
  (void)block_scan<kPlanThreads>(work[0], part, &all[0]);
  (void)block_scan<kPlanThreads>(work[1], part, &all[1]);
  long long items = 0, slots = 0;  // before the chunk
#pragma unroll
  for (int role = 0; role < 2; ++role) {
    const int count = role ? a.S : p.groups;
    Found* const list = role ? mine : p.ws.found;
    const int C = piece_keys((float)(all[0] * kv.heads), (float)(all[1] * kv.heads), role, p.R[role], p.own);
    for (int i0 = 0; i0 < count; i0 += kPlanThreads) {
      const int i = i0 + tid;
      int own = 0, cut = 0, row0 = 0, n = 0;
      if (i < count) {
        Found& f = list[i];
        into_pieces(f, C);
        own = kv.heads * f.tiles * f.pieces;
        cut = role == 0 || f.group >= 0 || f.pieces > 1 ? own * units_of(p, f, role) : 0;
        row0 = f.row0, n = f.n;
      }
      uint64_t chunk, cuts;
      const int upto = (int)block_scan<kPlanThreads>((uint64_t)own, part, &chunk);
      const int slot = (int)block_scan<kPlanThreads>((uint64_t)cut, part, &cuts);
      sh_upto[tid] = upto;
      sh_row0[tid] = row0, sh_n[tid] = n;
      if (i < count) {
        Found& f = list[i];
        f.item0 = (int)items + upto - own;
        f.slot0 = (int)slots + slot - cut;
        if (cut) f.flags |= kCut;
        fit(p, f, cut);
      }
      __syncthreads();
      for (int k = tid; k < (int)chunk; k += kPlanThreads) {
        int lo = 0, hi = kPlanThreads - 1;  // the first one with upto > k
        while (lo < hi) {
          const int mid = (lo + hi) >> 1;
          if (sh_upto[mid] > k) hi = mid;
          else lo = mid + 1;
        }
        if (items + k < p.ws.most) p.ws.map[items + k] = (role ? p.groups : 0) + i0 + lo;
      }
      if (role)
        for (int w = tid >> 6; w < min(kPlanThreads, count - i0); w += kPlanThreads / 64)
          for (int r = tid & 63; r < sh_n[w]; r += 64) p.ws.request[sh_row0[w] + r] = i0 + w;
      items += (long long)chunk;
      slots += (long long)cuts;
      __syncthreads();
    }
  }
  if (tid == 0) *p.ws.items = (int)min(items, (long long)p.ws.most);
}

typedef __attribute__((address_space(4))) const Found* found_p;
typedef __attribute__((address_space(4))) const int* ints_p;

// The workgroup's tile, piece and head of the requests' or groups' item `local`.
__device__ __forceinline__ int order_of(const Req& q, int heads, int local) {
  if (q.tiles <= 1) return local;
  // The tiles that read the same keys eight workgroups apart, so that they share an XCD's L2 (workgroups go to the eight
  // XCDs in turn): pairs (piece, KV head) by eights, each with all its tiles.
  const int pairs = q.pieces * heads, at = local / (8 * q.tiles), rest = local - at * 8 * q.tiles;
  const int wide = min(8, pairs - 8 * at), tile = rest / wide, pair = 8 * at + rest - tile * wide;
  return (pair / heads * q.tiles + tile) * heads + pair % heads;
}

// Item `id`, in scalar registers. False: there is none.
__device__ __forceinline__ bool find_item(const Plan& p, int id, Req& q, bool& group) {
  if (id >= *(ints_p)p.ws.items) return false;
  const int v = ((ints_p)p.ws.map)[id];
  const found_p f = (found_p)p.ws.found + v;
  group = v < p.groups;
  q.s = f->s, q.row0 = f->row0, q.n = f->n, q.len = f->len, q.ctx = f->ctx;
  q.tiles = f->tiles, q.pieces = f->pieces, q.begin = f->begin, q.C = f->C;
  q.slot = f->slot0;
  q.tree = f->flags & kTree;
  q.cut = f->flags & kCut;
  const int local = id - f->item0;
  if ((unsigned)local >= (unsigned)(q.tiles * q.pieces * p.kv.heads)) return false;  // (left out by `fit`)
  q.local = order_of(q, p.kv.heads, local);
  return true;
}

// The same for up to 64 groups and 128 requests, one or two (N) a lane, by the workgroup itself: one trip to memory for all that it reads, in place of
// the plan's launch and two more trips behind it (4 requests behind 1000 keys 21.2 us,
// so 16.2; 64 behind 16384 85.6 and 81.9; 78 behind 6400 55.6 and 50.4).
constexpr int kFew = 64;
template <int N>
__device__ __forceinline__ bool find_few(const Plan& p, int id, Req& q, bool& group) {
  const btf_paged_attention& a = p.a;
  const int lane = threadIdx.x & 63, heads = p.kv.heads;
  const bool is_group = lane < p.groups;
  int r0[N], r1[N], full[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int s = lane * N + i;
    const bool there = s < a.S;
    r0[i] = there ? a.row0[s] : 0, r1[i] = there ? a.row0[s + 1] : 0, full[i] = there ? a.kv_len[s] : 0;
  }
  const int b = is_group ? p.group0[lane] : 0, e = is_group ? p.group0[lane + 1] : 0;
  const int lead = is_group ? p.lead[lane] : 0, whole = is_group ? p.shared[lane] : 0;
  const int last = __builtin_amdgcn_readlane(r1[(a.S - 1) % N], (a.S - 1) / N);
  auto row_of = [&](int s) {
    int row = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int v = __shfl(r0[i], s / N & 63, 64);  // (by all lanes)
      if (s % N == i) row = v;
    }
    return min(max(s < a.S ? row : last, 0), a.T);
  };
  const int gb = min(max(b, 0), a.S), ge = min(max(e, gb), a.S), g0 = row_of(gb), g1 = row_of(ge);
  Found f = group_of(p, gb, ge, g0, g1, lead, whole), r[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int s = lane * N + i;
    r[i] = request_of(p, s, r0[i], r1[i], full[i]);
    if (p.groups > 0) {
      int lo = 0, hi = p.groups - 1;  // last_at_most
      while (__any(lo < hi)) {
        const int mid = (lo + hi + 1) >> 1, v = __shfl(b, mid, 64);
        if (lo < hi) {
          if (v <= s) lo = mid;
          else hi = mid - 1;
        }
      }
      Found g{};
      g.b = __shfl(gb, lo, 64), g.e = __shfl(ge, lo, 64), g.row0 = __shfl(f.row0, lo, 64), g.n = __shfl(f.n, lo, 64);
      g.len = __shfl(f.len, lo, 64), g.whole = __shfl(whole, lo, 64);
      if (takes_part(r[i], g)) r[i].group = lo, r[i].begin = g.len;
    }
  }
  auto work_of_lane = [](const Found& f) { return (float)f.tiles * (float)max(f.len - f.begin, 0); };
  float mine = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) mine += lane * N + i < a.S ? work_of_lane(r[i]) : 0.f;
  const float work0 = wave_sum_f(is_group ? work_of_lane(f) : 0.f) * heads, work1 = wave_sum_f(mine) * heads;
  into_pieces(f, piece_keys(work0, work1, 0, p.R[0], p.own));
  const int own0 = is_group ? heads * f.tiles * f.pieces : 0, cut0 = own0 * units_of(p, f, 0);
  const int upto0 = wave_scan_i(own0), cuts0 = wave_scan_i(cut0);
  f.slot0 = cuts0 - cut0;
  fit(p, f, cut0);
  int C = piece_keys(work0, work1, 1, p.R[1], kFewItems);
  if (p.own != kFewItems) {
    float few = (float)own0;
#pragma unroll
    for (int i = 0; i < N; ++i)
      few += lane * N + i < a.S ? (float)(heads * r[i].tiles) * ceilf((float)max(r[i].len - r[i].begin, 1) * __builtin_amdgcn_rcpf((float)C)) : 0.f;
    if (wave_sum_f(few) > (float)kRunning) C = piece_keys(work0, work1, 1, p.R[1], p.own);
  }
  int own[N], cut[N], all = 0, cuts = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    into_pieces(r[i], C);
    own[i] = lane * N + i < a.S ? heads * r[i].tiles * r[i].pieces : 0;
    if (r[i].group >= 0 || r[i].pieces > 1) r[i].flags |= kCut;
    cut[i] = r[i].flags & kCut ? own[i] * units_of(p, r[i], 1) : 0;
    all += own[i], cuts += cut[i];
  }
  const int upto1 = wave_scan_i(all);
  int slot = __builtin_amdgcn_readlane(cuts0, 63) + wave_scan_i(cuts) - cuts;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    r[i].slot0 = slot;
    slot += cut[i];
    fit(p, r[i], cut[i]);
  }
  if (id == 0 && threadIdx.x < 64) {
    if (is_group) p.ws.found[lane] = f;
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (lane * N + i < a.S) p.ws.found[p.groups + lane * N + i] = r[i];
  }
  const int groups = __builtin_amdgcn_readlane(upto0, 63);
  group = id < groups;
  const int at = group ? id : id - groups;
  const uint64_t behind = __ballot((group ? upto0 : upto1) > at);
  if (!behind) return false;
  const int l = __builtin_ctzll(behind);
  auto of = [&](int x) { return __builtin_amdgcn_readlane(x, l); };
  int local = at - of(group ? upto0 - own0 : upto1 - all);
  Found x = f;
  if (!group) {
    x = r[0];
#pragma unroll
    for (int i = 1; i < N; ++i)
      if (local >= of(own[i - 1])) local -= of(own[i - 1]), x = r[i];
  }
  q.s = of(x.s), q.row0 = of(x.row0), q.n = of(x.n), q.len = of(x.len), q.ctx = of(x.ctx);
  q.tiles = of(x.tiles), q.pieces = of(x.pieces), q.begin = of(x.begin), q.C = of(x.C), q.slot = of(x.slot0);
  const int flags = of(x.flags);
  q.tree = flags & kTree;
  q.cut = flags & kCut;
  if ((unsigned)local >= (unsigned)(q.tiles * q.pieces * heads)) return false;
  q.local = order_of(q, heads, local);
  return true;
}

// A tile of R rows: attn_stream up to 16, attn_tile with one or two tiles of 16 a wave.
template <int D, int R>
struct LdsOf {
  typedef TileLds<D> type;
};
template <int D>
struct LdsOf<D, 16> {
  typedef StreamLds<D, 1> type;
};
template <int D, bool BF, int R, bool TWO>
__device__ __forceinline__ void item(const Plan& p, Req& q, void* lds) {
  const Args own = TWO ? fresh_args() : Args{p.a, p.kv};  // (two kinds of tiles: nothing kept from before the branch)
  if constexpr (R == 16) {
    auto vector = [](int& v) { asm("" : "+v"(v)); };  // (attn_stream has no scalar registers to spare)
    vector(q.s), vector(q.row0), vector(q.n), vector(q.len), vector(q.ctx), vector(q.tiles), vector(q.pieces);
    vector(q.begin), vector(q.C), vector(q.local), vector(q.slot);
    attn_stream<D, BF, 1>(own.a, own.kv, q, *static_cast<StreamLds<D, 1>*>(lds));
  } else {
    attn_tile<D, BF, R / 64, true>(own.a, own.kv, q, *static_cast<TileLds<D>*>(lds));
  }
}
template <int D, bool BF, int R0, int R1>
__global__ void __launch_bounds__(64 * kWaves) __attribute__((amdgpu_waves_per_eu(D == 256 && R1 == 16 ? 1 : 2))) shared_kernel(Plan p) {
  constexpr size_t a = sizeof(typename LdsOf<D, R0>::type), b = sizeof(typename LdsOf<D, R1>::type);
  __shared__ __attribute__((aligned(16))) char lds[a > b ? a : b];
  Req q;
  bool group;
  const int id = blockIdx.x;
  const bool found = p.alone == 1 ? find_few<1>(p, id, q, group) : p.alone ? find_few<2>(p, id, q, group) : find_item(p, id, q, group);
  if (!found) return;  // the whole workgroup
  if (R0 == R1 || group) item<D, BF, R0, R0 != R1>(p, q, lds);
  else item<D, BF, R1, R0 != R1>(p, q, lds);
}

// The pieces of one row of one head, the group's and its own, put together: as attn_join_kernel.
constexpr int kJoinWaves = 4;
template <int D, bool ONE>
__global__ void __launch_bounds__(64 * kJoinWaves) shared_join_kernel(Plan p) {
  constexpr int E = D / 64;                 // values of a lane
  constexpr int BY = ONE ? 1 : kJoinWaves;  // waves of a row
  constexpr int AT = ONE ? 4 : 8;
  typedef float vE __attribute__((ext_vector_type(E)));
  const btf_paged_attention& a = p.a;
  int s;
  if (p.alone) {
    s = -1;
    for (int s0 = 0; s0 < a.S; s0 += 64) {
      const int l = min(s0 + (int)(threadIdx.x & 63), a.S - 1), t = blockIdx.x;
      const uint64_t m = __ballot(a.row0[l] <= t && t < a.row0[l + 1]);
      if (m) s = min(s0 + 63 - (int)__builtin_clzll(m), a.S - 1);
    }
  } else {
    s = ((ints_p)p.ws.request)[blockIdx.x];
  }
  if (s < 0) return;  // the whole workgroup
  const found_p f = (found_p)p.ws.found + p.groups + s;
  if (!(f->flags & kCut)) return;
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int G = a.heads / p.kv.heads, h = ONE ? blockIdx.y * kJoinWaves + w : blockIdx.y, kvh = h / G;
  if (h >= a.heads) return;
  // a role's first piece of the row, and from one to the next
  auto first_of = [&](const found_p f, int role, size_t& step, int& r, int& rows) {
    const int R = p.R[role], row = (blockIdx.x - f->row0) * G + h % G, tile = row / R;
    rows = slot_rows(R, f->n * G);
    const size_t slot = (size_t)rows * (D + 2);
    r = row % R;
    step = (size_t)f->tiles * p.kv.heads * slot;
    return p.ws.slots + (size_t)f->slot0 * (16 * (D + 2)) + ((size_t)(f->tiles - 1 - tile) * p.kv.heads + kvh) * slot;
  };
  int n0 = 0, r0 = 0, r1, R0 = 0, R1;
  size_t step0 = 0, step1;
  const float* base0 = nullptr;
  if (f->group >= 0) {
    const found_p g = (found_p)p.ws.found + f->group;
    n0 = g->pieces;
    base0 = first_of(g, 0, step0, r0, R0);
  }
  const float* base1 = first_of(f, 1, step1, r1, R1);
  const int n = n0 + f->pieces;
  auto values = [&](int i) { return i < n0 ? base0 + i * step0 + r0 * D : base1 + (i - n0) * step1 + r1 * D; };
  auto top_of = [&](int i) { return i < n0 ? base0[i * step0 + R0 * D + r0] : base1[(i - n0) * step1 + R1 * D + r1]; };
  auto sum_of = [&](int i) { return i < n0 ? base0[i * step0 + R0 * D + R0 + r0] : base1[(i - n0) * step1 + R1 * D + R1 + r1]; };
  float top = -INFINITY, sum = 0.f, l0 = 0.f;
  if (lane < n) top = top_of(lane), l0 = sum_of(lane);
  vE x[AT];
  auto read = [&](int i0, int i, int m) {
#pragma unroll
    for (int u = 0; u < AT; ++u) x[u] = *reinterpret_cast<const vE*>(values(i0 + min(i + u * BY, m - 1)) + lane * E);
  };
  const int first = ONE ? 0 : w;
  read(0, first, min(64, n));
  const float m0 = top;
  for (int i = 64 + lane; i < n; i += 64) top = fmaxf(top, top_of(i));
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
  const float base = top == -INFINITY ? 0.f : top;
  vE v = vE(0.f);
  for (int i0 = 0; i0 < n; i0 += 64) {
    float c = 0.f;
    if (i0 + lane < n) {
      c = fast_exp2((i0 ? top_of(i0 + lane) : m0) - base);
      sum += c * (i0 ? sum_of(i0 + lane) : l0);
    }
    const int m = min(64, n - i0);
    for (int i = first; i < m; i += AT * BY) {
      if (i0 + i != first) read(i0, i, m);
#pragma unroll
      for (int u = 0; u < AT; ++u) {
        const int j = min(i + u * BY, m - 1);
        const float f = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(c), j));
        if (i + u * BY < m) v += f * x[u];
      }
    }
  }
  sum = wave_sum_f(sum);
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  float* y = a.out + (size_t)blockIdx.x * a.ldo + h * D;
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

// Rows of a tile of `count` groups or requests that have T rows in all.
int tile_rows(int count, int T, int heads, const btf_kv_cache& kv) {
  const int64_t rows = (int64_t)T * (heads / kv.heads);
  if (rows <= 16 * (int64_t)count) return 16;
  return kv.dim != 128 || rows <= 128 * (int64_t)count ? 64 : 128;
}

// Items of the groups (role 0) or requests at most: each tile's last piece may be a part of one.
int64_t most_items(int role, int count, int T, int heads, const btf_kv_cache& kv, int R) {
  return ((int64_t)T * (heads / kv.heads) / R + count) * kv.heads + (role ? kOwnItems : kRunning);
}

// Slots of a launch of up to S requests and groups, in 16 rows: a tile's slot has the rows of the request or group, up to the
// next multiple of 16 (of more than one tile, up to twice its rows), and each piece beyond a tile's first is one of the items
// that the work is cut into.
int64_t slot_units(int S, int T, int heads, const btf_kv_cache& kv) {
  return (int64_t)T * heads / 4 + 2 * (int64_t)S * kv.heads + (kRunning + kOwnItems) * (kv.dim == 128 ? 8 : 4);
}

int64_t up(int64_t n) { return (n + 255) & ~(int64_t)255; }

// Bytes before the slots, for up to S requests and groups.
int64_t plan_bytes(int S, int T, int heads, const btf_kv_cache& kv) {
  return up(64 + 2 * (int64_t)S * sizeof(Found) + 4 * (most_items(0, S, T, heads, kv, 16) + most_items(1, S, T, heads, kv, 16)) + 4 * (int64_t)T);
}

template <int D, bool BF>
int shared_go(const Plan& p, hipStream_t st) {
  int rc = BTF_OK;
  if (!p.alone) {
    if (p.a.S <= kPlanThreads) hipLaunchKernelGGL(shared_plan_small_kernel, dim3(1), dim3(kPlanThreads), 0, st, p);
    else hipLaunchKernelGGL(shared_plan_kernel, dim3(1), dim3(kPlanThreads), 0, st, p);
    rc = launch_status("shared_plan_kernel");
    if (rc != BTF_OK) return rc;
  }
  auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3((unsigned)p.ws.most), dim3(64 * kWaves), 0, st, p); };
  const int R0 = p.R[0], R1 = p.R[1];
  if (R0 == 16) {
    go(shared_kernel<D, BF, 16, 16>);
  } else if (R1 == 16) {
    if constexpr (D == 128) {
      if (R0 == 64) go(shared_kernel<D, BF, 64, 16>);
      else go(shared_kernel<D, BF, 128, 16>);
    }
  } else if (R0 == 64) {
    go(shared_kernel<D, BF, 64, 64>);
  } else if constexpr (D == 128) {
    if (R1 == 64) go(shared_kernel<D, BF, 128, 64>);
    else go(shared_kernel<D, BF, 128, 128>);
  }
  rc = launch_status("shared_kernel");
  if (rc != BTF_OK) return rc;
  const bool one = (int64_t)p.a.T * p.a.heads >= 2048;
  const dim3 join(p.a.T, one ? (p.a.heads + kJoinWaves - 1) / kJoinWaves : p.a.heads), blk(64 * kJoinWaves);
  if (one) hipLaunchKernelGGL((shared_join_kernel<D, true>), join, blk, 0, st, p);
  else hipLaunchKernelGGL((shared_join_kernel<D, false>), join, blk, 0, st, p);
  return launch_status("shared_join_kernel");
}

}  // namespace

int64_t shared_attention_most_items(int S, int T, int heads, const btf_kv_cache& kv) {
  return most_items(0, S, T, heads, kv, 16) + most_items(1, S, T, heads, kv, 16);
}

int64_t shared_attention_ws_bytes(int S, int T, int heads, const btf_kv_cache& kv) {
  return plan_bytes(S, T, heads, kv) + up(4 * slot_units(S, T, heads, kv) * 16 * (kv.dim + 2));
}

int shared_attention(const btf_shared_attention& a, const btf_kv_cache& kv, hipStream_t st) {
  Plan p{};
  p.kv = kv;
  p.groups = a.groups;
  p.group0 = a.group0, p.lead = a.lead, p.shared = a.shared;
  p.R[1] = tile_rows(a.S, a.T, a.heads, kv);
  p.R[0] = a.groups > 0 ? tile_rows(a.groups, a.T, a.heads, kv) : p.R[1];
  // (heads of 64 and 256 have one kind of tile in a launch: attn_stream with 256 leaves room for one workgroup a CU only)
  if (kv.dim != 128 && p.R[0] == 64) p.R[1] = 64;
  char* at = static_cast<char*>(a.ws);
  p.ws.items = reinterpret_cast<int*>(at);
  p.ws.found = reinterpret_cast<Found*>(at + 64);
  p.ws.map = reinterpret_cast<int*>(p.ws.found + a.groups + a.S);
  p.ws.most = (int)(most_items(1, a.S, a.T, a.heads, kv, p.R[1]) + (a.groups ? most_items(0, a.groups, a.T, a.heads, kv, p.R[0]) : 0));
  p.ws.request = p.ws.map + p.ws.most;
  p.ws.slots = reinterpret_cast<float*>(at + plan_bytes(a.S, a.T, a.heads, kv));
  p.ws.units = (int)slot_units(a.S, a.T, a.heads, kv);
  p.a = btf_paged_attention{a.S,   a.T,    a.heads, a.q,   a.ldq, a.table,    a.ldt,
                            a.row0, a.kv_len, a.tree, a.scale, a.out, a.ldo, p.ws.slots};
  p.G = a.heads / kv.heads;
  p.own = kv.dim == 256 && p.R[0] == 16 ? kFewItems : kOwnItems;
  p.cap = (int64_t)a.ldt * kv.page < kMostKeys ? a.ldt * kv.page : kMostKeys;
  p.alone = a.groups > kFew ? 0 : a.S <= kFew ? 1 : a.S <= 2 * kFew ? 2 : 0;
  const bool bf = kv.type == BTF_BF16;
  if (kv.dim == 64) return bf ? shared_go<64, true>(p, st) : shared_go<64, false>(p, st);
  if (kv.dim == 128) return bf ? shared_go<128, true>(p, st) : shared_go<128, false>(p, st);
  return bf ? shared_go<256, true>(p, st) : shared_go<256, false>(p, st);
}

}  // namespace btfhip
