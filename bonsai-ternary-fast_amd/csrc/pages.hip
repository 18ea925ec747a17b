// pages.hip -- cache pages that several requests hold, and tokens that change
// their places (btf_hip_launch_page_fork, _page_copy, _page_free, _cache_move;
// gfx950).
//
// fork and free are integers: which row holds which page, and how many rows hold a
// page beyond one (shared). Counts change by 32-bit atomic additions, whose order
// does not show in the sums. Pages go back in an order that does not depend on the
// threads' either: after all counts have been lowered, those of the pages to give
// back are below zero; each place (row, page of the row) that gives one up puts the
// smallest mark, INT_MIN + its number, there, and the one whose mark stays owns the
// page. Its number among the owners is a prefix sum.
//
// copy and move are bytes. A wave's lanes take runs of 128 bytes (a cache line) or
// more of a token's values (a move with few workgroups less); up to eight 16-byte loads a thread are on their way
// before the first store.
#include <climits>
#include <string>

#include "../../include/btf/hip_abi.h"
#include "common.h"

namespace btfhip {
namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// ---- fork ----
constexpr int kForkThreads = 1024;
// Entries of table (forks times ldt) up to which the deciding workgroup copies the ids itself.
constexpr int kForkSmall = 8192;

// Entry j of row dst becomes row src's, if it is one of its whole pages.
constexpr int kForkEach = 4;  // entries of a thread at a time
struct Entry {
  int src, dst, j;  // j below zero: none
};
__device__ __forceinline__ void fork_entries(const btf_page_fork& a, const Entry (&e)[kForkEach]) {
  int p[kForkEach];
#pragma unroll
  for (int i = 0; i < kForkEach; ++i)
    if (e[i].j >= 0) p[i] = a.table[(size_t)e[i].src * a.ldt + e[i].j];
#pragma unroll
  for (int i = 0; i < kForkEach; ++i)
    if (e[i].j >= 0) {
      a.table[(size_t)e[i].dst * a.ldt + e[i].j] = p[i];
      if (p[i] >= 0 && p[i] < a.pages) __hip_atomic_fetch_add(a.shared + p[i], 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
}

template <bool ROWS>
__global__ void __launch_bounds__(kForkThreads) page_fork_kernel(btf_page_fork a) {
  __shared__ uint64_t part[kForkThreads / 64];
  __shared__ int sh_dst[kForkThreads], sh_src[kForkThreads], sh_whole[kForkThreads];
  const int f = threadIdx.x;
  const bool live = f < a.F;
  const int s = live ? a.src[f] : -1, d = live ? a.dst[f] : -1, n = live ? a.tokens[f] : -1;
  const long long free0 = max(*a.n_free, 0);
  bool sound = s >= 0 && s < a.S && d >= 0 && d < a.S && s != d && n >= 0;
  if (sound) {
    const int hs = a.held[s];
    sound = hs <= a.ldt && n <= (long long)hs * a.page && a.held[d] == 0;
  }
  sh_dst[f] = sound ? d : -1;
  sh_src[f] = s;
  __syncthreads();  // (all of held, and *n_free, has been read)
  bool taken = false;
  for (int i = 0; i < (sound ? f : 0); ++i) taken |= sh_dst[i] == d;
  sound = sound && !taken;
  const int whole = sound ? n / a.page : 0;
  const bool part_page = sound && n % a.page != 0;
  uint64_t all;
  const long long upto = (long long)block_scan<kForkThreads>(part_page, part, &all);
  const bool ok = sound && (!part_page || upto <= free0);
  sh_whole[f] = ok ? whole : 0;
  if (live) {
    int from = -1, to = -1;
    if (ok && part_page) {
      from = a.table[(size_t)s * a.ldt + whole];
      to = a.free_list[free0 - upto];
      a.table[(size_t)d * a.ldt + whole] = to;
    }
    if (ok) a.held[d] = whole + part_page;
    a.got[f] = ok ? n : -1;
    a.copy_from[f] = from;
    a.copy_to[f] = to;
    a.copy_tokens[f] = ok && part_page ? n % a.page : 0;
  }
  if (f == 0) *a.n_free = (int)(free0 - min((long long)all, free0));  // (each takes one: the first ones are served)
  if (!ROWS) return;
  __syncthreads();
  for (int k0 = f; k0 < a.F * a.ldt; k0 += kForkEach * kForkThreads) {
    Entry e[kForkEach];
#pragma unroll
    for (int i = 0; i < kForkEach; ++i) {
      const int k = k0 + i * kForkThreads, g = k < a.F * a.ldt ? k / a.ldt : 0, j = k - g * a.ldt;
      e[i] = Entry{sh_src[g], sh_dst[g], k < a.F * a.ldt && j < sh_whole[g] ? j : -1};
    }
    fork_entries(a, e);
  }
}

__global__ void __launch_bounds__(256) page_fork_rows_kernel(btf_page_fork a) {
  const int f = blockIdx.x, n = a.got[f];
  if (n < a.page) return;
  const int whole = min(n / a.page, a.ldt), src = a.src[f], dst = a.dst[f];
  for (int j0 = blockIdx.y * 256 * kForkEach + threadIdx.x; j0 < whole; j0 += gridDim.y * 256 * kForkEach) {
    Entry e[kForkEach];
#pragma unroll
    for (int i = 0; i < kForkEach; ++i) e[i] = Entry{src, dst, j0 + 256 * i < whole ? j0 + 256 * i : -1};
    fork_entries(a, e);
  }
}

// ---- free ----
constexpr int kFreeThreads = 1024;
constexpr int kFreeEach = 4;                          // places of a thread
constexpr int kFreeChunk = kFreeThreads * kFreeEach;  // ... of a workgroup
constexpr int kFreeMost = 8;                          // ... of a thread at most, where one workgroup does it all

// Whether places e0, e0 + 1, ... (place s * ldt + j is page j of row s) give up their pages, and the pages' ids, -1: none
// that the cache has. (Loads without branches, so that all are on their way at once.)
template <int EACH>
struct Places {
  unsigned in = 0;
  int page[EACH];
};
template <int EACH>
__device__ __forceinline__ Places<EACH> places_of(const btf_page_free& a, const int* held, int e0) {
  const int end = a.S * a.ldt;
  int keep[EACH], have[EACH], j[EACH];
  Places<EACH> p;
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    const int e = min(e0 + i, end - 1), s = e / a.ldt;
    j[i] = e - s * a.ldt;
    keep[i] = a.keep[s];
    have[i] = held[s];
    p.page[i] = a.table[e];
  }
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    const int first = (int)(((long long)max(keep[i], 0) + a.page - 1) / a.page);
    const bool in = e0 + i < end && j[i] >= first && j[i] < have[i];
    p.in |= (unsigned)in << i;
    if (!in || p.page[i] >= a.pages || p.page[i] < 0) p.page[i] = -1;
  }
  return p;
}
// Lowers the page's count; what it was.
__device__ __forceinline__ int lower(const btf_page_free& a, int page) {
  return page < 0 ? -1 : __hip_atomic_fetch_add(a.shared + page, -1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ int count_of(const btf_page_free& a, int page) {
  return __hip_atomic_load(a.shared + page, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void mark(const btf_page_free& a, int page, int count, int e) {
  // (a count below zero is more than -2^29, a mark less than INT_MIN + 2^29)
  if (page >= 0 && count < 0)
    __hip_atomic_fetch_min(a.shared + page, INT_MIN + e, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
// The places' counts (page 0's for a place without a page).
template <int EACH>
__device__ __forceinline__ void counts_of(const btf_page_free& a, const Places<EACH>& p, int (&count)[EACH]) {
#pragma unroll
  for (int i = 0; i < EACH; ++i) count[i] = a.shared ? count_of(a, max(p.page[i], 0)) : 0;
}
template <int EACH>
__device__ __forceinline__ unsigned owned(const btf_page_free& a, const Places<EACH>& p, int e0) {
  int count[EACH];
  counts_of(a, p, count);
  unsigned own = 0;
#pragma unroll
  for (int i = 0; i < EACH; ++i) own |= (unsigned)(p.page[i] >= 0 && (!a.shared || count[i] == INT_MIN + e0 + i)) << i;
  return own;
}
// The places' pages go to the list, which has n0 entries, `behind` of the call's after them.
template <int EACH>
__device__ __forceinline__ void give_back(const btf_page_free& a, const Places<EACH>& p, unsigned own, int e0,
                                          long long n0, long long behind) {
#pragma unroll
  for (int i = EACH - 1; i >= 0; --i) {
    if (own >> i & 1) {
      if (n0 + behind < a.pages) a.free_list[n0 + behind] = p.page[i];
      ++behind;
      if (a.shared) a.shared[p.page[i]] = 0;
    }
    if (p.in >> i & 1) a.table[e0 + i] = -1;
  }
}
__device__ __forceinline__ int stays(const btf_page_free& a, int held, int s) {
  return (int)min((long long)held, ((long long)max(a.keep[s], 0) + a.page - 1) / a.page);
}

// All memory accesses of the workgroup's threads so far are done (atomics on counts among them, which act in L2, as the
// loads of counts do: nothing has to be written back or thrown away for these).
__device__ __forceinline__ void all_done() {
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
}

// All of it by one workgroup.
template <int EACH>
__global__ void __launch_bounds__(kFreeThreads) page_free_small_kernel(btf_page_free a) {
  __shared__ uint64_t part[kFreeThreads / 64];
  __shared__ int sh_several;
  const int e0 = threadIdx.x * EACH;
  const long long n0 = min((long long)max(*a.n_free, 0), (long long)a.pages);
  const Places<EACH> p = places_of<EACH>(a, a.held, e0);
  unsigned own = 0;
  if (!a.shared) {
    own = owned(a, p, e0);
  } else {
    // Who lowers a count from 0 gives the page back, unless other places gave up the same page: these found it above 0 (or
    // below) and find it below 0 now. Only then the marks decide.
    int was[EACH], count[EACH];
#pragma unroll
    for (int i = 0; i < EACH; ++i) was[i] = lower(a, p.page[i]);
    bool several = false;
    if (threadIdx.x == 0) sh_several = 0;
    all_done();
#pragma unroll
    for (int i = 0; i < EACH; ++i) count[i] = p.page[i] >= 0 && was[i] != 0 ? count_of(a, p.page[i]) : 0;
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      several |= count[i] < 0;
      own |= (unsigned)(p.page[i] >= 0 && was[i] == 0) << i;
    }
    if (several) sh_several = 1;
    __syncthreads();
    if (sh_several) {
      counts_of(a, p, count);
      all_done();
#pragma unroll
      for (int i = 0; i < EACH; ++i) mark(a, p.page[i], count[i], e0 + i);
      all_done();
      own = owned(a, p, e0);
    }
  }
  uint64_t all;
  const uint64_t upto = block_scan<kFreeThreads>(__popc(own), part, &all);  // (and all have read what is written below)
  give_back(a, p, own, e0, n0, (long long)(all - upto));
  for (int s = threadIdx.x; s < a.S; s += kFreeThreads) a.held[s] = stays(a, a.held[s], s);
  if (threadIdx.x == 0) *a.n_free = (int)min(n0 + (long long)all, (long long)a.pages);
}

// The same in four launches, a workgroup for each kFreeChunk places. ws: owners of each
// chunk, then held and *n_free as they were (the last launch writes them while other
// workgroups read).
__global__ void __launch_bounds__(kFreeThreads) page_free_lower_kernel(btf_page_free a) {
  const int e0 = blockIdx.x * kFreeChunk + threadIdx.x * kFreeEach;
  const Places<kFreeEach> p = places_of<kFreeEach>(a, a.held, e0);
#pragma unroll
  for (int i = 0; i < kFreeEach; ++i) lower(a, p.page[i]);
}
__global__ void __launch_bounds__(kFreeThreads) page_free_mark_kernel(btf_page_free a) {
  const int e0 = blockIdx.x * kFreeChunk + threadIdx.x * kFreeEach;
  const Places<kFreeEach> p = places_of<kFreeEach>(a, a.held, e0);
  int count[kFreeEach];
  counts_of(a, p, count);
#pragma unroll
  for (int i = 0; i < kFreeEach; ++i) mark(a, p.page[i], count[i], e0 + i);
}
__global__ void __launch_bounds__(kFreeThreads) page_free_count_kernel(btf_page_free a) {
  __shared__ uint64_t part[kFreeThreads / 64];
  int* owners = static_cast<int*>(a.ws);
  const int e0 = blockIdx.x * kFreeChunk + threadIdx.x * kFreeEach;
  const Places<kFreeEach> p = places_of<kFreeEach>(a, a.held, e0);
  uint64_t all;
  const uint64_t n = __popc(owned(a, p, e0));
#pragma unroll
  for (int i = 0; i < kFreeEach; ++i) {
    if (e0 + i < a.S * a.ldt && (e0 + i) % a.ldt == 0) owners[gridDim.x + (e0 + i) / a.ldt] = a.held[(e0 + i) / a.ldt];
  }
  (void)block_scan<kFreeThreads>(n, part, &all);
  if (threadIdx.x == 0) owners[blockIdx.x] = (int)all;
  if (blockIdx.x == 0 && threadIdx.x == 0) owners[gridDim.x + a.S] = *a.n_free;
}
__global__ void __launch_bounds__(kFreeThreads) page_free_kernel(btf_page_free a) {
  __shared__ uint64_t part[kFreeThreads / 64];
  const int* owners = static_cast<const int*>(a.ws);
  const int* held = owners + gridDim.x;
  const int e0 = blockIdx.x * kFreeChunk + threadIdx.x * kFreeEach;
  const long long n0 = min((long long)max(held[a.S], 0), (long long)a.pages);
  const Places<kFreeEach> p = places_of<kFreeEach>(a, held, e0);
  const unsigned own = owned(a, p, e0);
  uint64_t later = 0, behind, all;  // owners of the chunks behind this one
  for (int c = blockIdx.x + 1 + threadIdx.x; c < (int)gridDim.x; c += kFreeThreads) later += owners[c];
  (void)block_scan<kFreeThreads>(later, part, &behind);
  const uint64_t upto = block_scan<kFreeThreads>(__popc(own), part, &all);
  give_back(a, p, own, e0, n0, (long long)(behind + all - upto));
#pragma unroll
  for (int i = 0; i < kFreeEach; ++i)
    if (e0 + i < a.S * a.ldt && (e0 + i) % a.ldt == 0) a.held[(e0 + i) / a.ldt] = stays(a, held[(e0 + i) / a.ldt], (e0 + i) / a.ldt);
  if (blockIdx.x == 0 && threadIdx.x == 0) *a.n_free = (int)min(n0 + (long long)(behind + all), (long long)a.pages);
}

// ---- copy ----
constexpr int kCopyThreads = 256;
constexpr int kInFlight = 8;  // 16-byte loads of a thread before its first store

// One (entry, K or V, head) of a layer: up to a page's tokens.
__global__ void __launch_bounds__(kCopyThreads) page_copy_kernel(btf_page_copy a, btf_kv_cache kv) {
  const int h = blockIdx.x % kv.heads, rest = blockIdx.x / kv.heads, i = rest >> 1;
  const int from = a.from[i], to = a.to[i], n = min(a.tokens ? a.tokens[i] : kv.page, kv.page);
  if (from < 0 || from >= kv.pages || to < 0 || to >= kv.pages || from == to || n <= 0) return;
  uint16_t* base = static_cast<uint16_t*>(rest & 1 ? kv.v : kv.k) + (size_t)blockIdx.y * a.layer_stride + (size_t)h * kv.head_stride;
  const uint16_t* x = base + (size_t)from * kv.page_stride;
  uint16_t* y = base + (size_t)to * kv.page_stride;
  const int sh = __builtin_ctz(kv.dim) - 3, mask = (1 << sh) - 1, end = n << sh;  // 16-byte chunks
  auto at = [&](int c) { return (size_t)(c >> sh) * kv.tok_stride + 8 * (c & mask); };
  for (int c0 = threadIdx.x; c0 < end; c0 += kCopyThreads * kInFlight) {
    u32x4 v[kInFlight];
#pragma unroll
    for (int u = 0; u < kInFlight; ++u)
      if (c0 + u * kCopyThreads < end) v[u] = *reinterpret_cast<const u32x4*>(x + at(c0 + u * kCopyThreads));
#pragma unroll
    for (int u = 0; u < kInFlight; ++u)
      if (c0 + u * kCopyThreads < end) *reinterpret_cast<u32x4*>(y + at(c0 + u * kCopyThreads)) = v[u];
  }
}

// ---- move ----
// The kept tokens of request s: in a tree's bits, or list entries from `lo` on.
struct Kept {
  unsigned long long bits;
  int lo, n;
};
template <bool TREE>
__device__ __forceinline__ Kept kept_of(const btf_cache_move& a, int s) {
  Kept k{0, 0, 0};
  if (TREE) {
    const int leaf = a.leaf[s];
    if (leaf >= 0 && leaf < a.T) k.bits = a.tree[leaf];
    k.n = __popcll(k.bits);
  } else {
    k.lo = min(max(a.source0[s], 0), a.T);
    k.n = max(min(max(a.source0[s + 1], 0), a.T) - k.lo, 0);
  }
  return k;
}

// In place a token's new place may be another's old one, but never that of a later
// token of the list (places ascend, none goes up). A workgroup has one run (32 to 128 bytes) of
// the values of one (request, K or V, head, layer) for all tokens: it reads a batch,
// waits until all of its threads have theirs, writes it, and goes on. So no two
// workgroups touch the same bytes, and nothing is overwritten before it was read.
// L lanes have a token, 16 bytes each.
template <int N, bool TREE, int L>
__global__ void __launch_bounds__(N) cache_move_kernel(btf_cache_move a, btf_kv_cache kv) {
  const int runs = kv.dim / (8 * L);
  int id = blockIdx.x;
  const int run = id % runs;
  id /= runs;
  const int h = id % kv.heads;
  id /= kv.heads;
  const int s = id >> 1;
  const int first = a.first[s];
  const Kept kept = kept_of<TREE>(a, s);
  const unsigned long long bits = kept.bits;
  const int lo = kept.lo, n = kept.n;
  if (blockIdx.y == 0 && run == 0 && h == 0 && !(id & 1) && threadIdx.x == 0 && a.kv_len) a.kv_len[s] = first + n;
  uint16_t* base = static_cast<uint16_t*>(id & 1 ? kv.v : kv.k) + (size_t)blockIdx.y * a.layer_stride +
                   (size_t)h * kv.head_stride + 8 * (L * run + (threadIdx.x & (L - 1)));
  const int* tab = a.table + (size_t)s * a.ldt;
  const int* tab_to = a.to_table ? a.to_table + (size_t)s * a.ldt_to : tab;
  const int ld_to = a.to_table ? a.ldt_to : a.ldt;
  const int sh = __builtin_ctz(kv.page);
  // where a place's values are, counted from base; -1: not in the table or the cache
  auto where = [&](const int* t, int ld, long long place) -> long long {
    if (place < 0 || place >= (long long)ld << sh) return -1;
    const int p = t[place >> sh];
    return p < 0 || p >= kv.pages ? -1 : p * (long long)kv.page_stride + (place & (kv.page - 1)) * (long long)kv.tok_stride;
  };
  constexpr int kAtOnce = N / L;  // tokens
  // Two batches in flight: while one's values arrive, the places and page ids of the next are looked up; its values are
  // under way before this one's are stored.
  constexpr int kMine = 2;  // tokens of a thread (with more than 64 registers only one workgroup of 1024 threads fits a CU)
  u32x4 v[2][kMine];
  long long from[2][kMine], to[2][kMine];
  auto look = [&](int i0, int b) {
#pragma unroll
    for (int u = 0; u < kMine; ++u) {
      const int i = i0 + u * kAtOnce + threadIdx.x / L;
      from[b][u] = to[b][u] = -1;
      if (i < n) {
        long long place;
        if (TREE) {  // the i-th set bit
          unsigned long long w = bits;
          int k = i, pos = 0;
#pragma unroll
          for (int half = 32; half; half >>= 1) {
            const int c = __popcll(w & ((1ull << half) - 1));
            if (k >= c) k -= c, pos += half, w >>= half;
          }
          place = (long long)first + pos;
        } else {
          place = a.source[lo + i];
        }
        const long long dst = (long long)first + i;
        if (a.to_table || place != dst) {
          from[b][u] = where(tab, a.ldt, place);
          to[b][u] = where(tab_to, ld_to, dst);
        }
      }
    }
  };
  auto load = [&](int b) {
#pragma unroll
    for (int u = 0; u < kMine; ++u) {
      if (from[b][u] < 0) to[b][u] = -1;
      if (to[b][u] >= 0) v[b][u] = *reinterpret_cast<const u32x4*>(base + from[b][u]);
    }
  };
  constexpr int kBatch = kAtOnce * kMine;
  if (n <= 0) return;
  look(0, 0);
  load(0);
  for (int i0 = 0; i0 < n; i0 += 2 * kBatch)
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const int at = i0 + b * kBatch;
      if (at >= n) break;
      const bool more = at + kBatch < n;
      if (more) look(at + kBatch, b ^ 1);
      // every thread's values have arrived before any thread stores
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();
      if (more) load(b ^ 1);
#pragma unroll
      for (int u = 0; u < kMine; ++u)
        if (to[b][u] >= 0) *reinterpret_cast<u32x4*>(base + to[b][u]) = v[b][u];
    }
}

// kv_len alone.
template <bool TREE>
__global__ void __launch_bounds__(256) cache_move_len_kernel(btf_cache_move a) {
  const int s = blockIdx.x * 256 + threadIdx.x;
  if (s < a.S) a.kv_len[s] = a.first[s] + kept_of<TREE>(a, s).n;
}

int free_chunks(int S, int ldt) { return (int)(((int64_t)S * ldt + kFreeChunk - 1) / kFreeChunk); }

}  // namespace

int page_fork(const btf_page_fork& a, hipStream_t st) {
  if ((int64_t)a.F * a.ldt <= kForkSmall) {
    hipLaunchKernelGGL(page_fork_kernel<true>, dim3(1), dim3(kForkThreads), 0, st, a);
    return launch_status("page_fork_kernel");
  }
  hipLaunchKernelGGL(page_fork_kernel<false>, dim3(1), dim3(kForkThreads), 0, st, a);
  const int rc = launch_status("page_fork_kernel");
  if (rc != BTF_OK) return rc;
  const int y = (a.ldt + 256 * kForkEach - 1) / (256 * kForkEach);
  hipLaunchKernelGGL(page_fork_rows_kernel, dim3(a.F, y < 64 ? y : 64), dim3(256), 0, st, a);
  return launch_status("page_fork_rows_kernel");
}

int64_t page_free_ws_bytes(int S, int ldt) {
  const int n = free_chunks(S, ldt);
  return n * kFreeEach <= kFreeMost ? 0 : ((int64_t)n + S + 1) * 4;
}

int page_free(const btf_page_free& a, hipStream_t st) {
  const int n = free_chunks(a.S, a.ldt);
  if (n * kFreeEach <= kFreeMost) {
    if ((int64_t)a.S * a.ldt <= kFreeThreads) hipLaunchKernelGGL(page_free_small_kernel<1>, dim3(1), dim3(kFreeThreads), 0, st, a);
    else if (n <= 1) hipLaunchKernelGGL(page_free_small_kernel<kFreeEach>, dim3(1), dim3(kFreeThreads), 0, st, a);
    else hipLaunchKernelGGL(page_free_small_kernel<kFreeMost>, dim3(1), dim3(kFreeThreads), 0, st, a);
    return launch_status("page_free_small_kernel");
  }
  if (a.shared) {
    hipLaunchKernelGGL(page_free_lower_kernel, dim3(n), dim3(kFreeThreads), 0, st, a);
    int rc = launch_status("page_free_lower_kernel");
    if (rc != BTF_OK) return rc;
    hipLaunchKernelGGL(page_free_mark_kernel, dim3(n), dim3(kFreeThreads), 0, st, a);
    rc = launch_status("page_free_mark_kernel");
    if (rc != BTF_OK) return rc;
  }
  hipLaunchKernelGGL(page_free_count_kernel, dim3(n), dim3(kFreeThreads), 0, st, a);
  int rc = launch_status("page_free_count_kernel");
  if (rc != BTF_OK) return rc;
  hipLaunchKernelGGL(page_free_kernel, dim3(n), dim3(kFreeThreads), 0, st, a);
  return launch_status("page_free_kernel");
}

int page_copy(const btf_page_copy& a, const btf_kv_cache& kv, hipStream_t st) {
  hipLaunchKernelGGL(page_copy_kernel, dim3(2 * a.n * kv.heads, a.layers), dim3(kCopyThreads), 0, st, a, kv);
  return launch_status("page_copy_kernel");
}

int cache_move(const btf_cache_move& args, const btf_kv_cache& kv, hipStream_t st) {
  btf_cache_move a = args;
  const bool behind = a.kv_len == a.first;  // (the lengths are written when all workgroups have read what they were)
  if (behind) a.kv_len = nullptr;
  const int groups = 2 * a.S * kv.heads * (kv.dim / 64);
  // A tree's path in batches of 16 tokens. A list in batches of 256 with as many threads as there are: 8 requests of up to
  // 16384 tokens, half of which stay, 2 layers, 187 us (3.9 TB/s read and written) with 1024 threads, 247 with 512, 278 with 256.
  // Where that leaves CUs idle, shorter runs of more tokens at once: one request of 9000 tokens, heads of 256, runs of 128, 64, 32, 16
  // bytes: 1 KV head (8 workgroups of 128 bytes) 30, 22, 19, 16 us, 4 heads (32) 42, 27, 24, 36, 8 (64) 41, 28, 30, 55, 16 (128)
  // 46, 35, 57, 94; 160 workgroups 53 and 62 in runs of 64.
  auto go = [&](auto kernel, int parts) { hipLaunchKernelGGL(kernel, dim3(parts * groups, a.layers), dim3(1024), 0, st, a, kv); };
  const int64_t all = (int64_t)groups * a.layers;
  if (a.tree) hipLaunchKernelGGL((cache_move_kernel<64, true, 8>), dim3(groups, a.layers), dim3(64), 0, st, a, kv);
  else if (all <= 48) go(cache_move_kernel<1024, false, 2>, 4);
  else if (all <= 128) go(cache_move_kernel<1024, false, 4>, 2);
  else go(cache_move_kernel<1024, false, 8>, 1);
  const int rc = launch_status("cache_move_kernel");
  if (rc != BTF_OK || !behind) return rc;
  const dim3 grid((a.S + 255) / 256), blk(256);
  if (a.tree) hipLaunchKernelGGL(cache_move_len_kernel<true>, grid, blk, 0, st, args);
  else hipLaunchKernelGGL(cache_move_len_kernel<false>, grid, blk, 0, st, args);
  return launch_status("cache_move_len_kernel");
}

}  // namespace btfhip
