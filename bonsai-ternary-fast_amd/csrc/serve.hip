// serve.hip -- the extern "C" boundary of a serving step's operators
// (include/btf/hip_abi.h): host-side argument checks, as in abi.hip before any
// HIP call.
#include <cmath>
#include <string>

#include "../../include/btf/hip_abi.h"
#include "common.h"

using namespace btfhip;

namespace {

bool aligned(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

// A grid has at most 2^32 - 1 threads along x and 65535 workgroups along y.
constexpr int kMaxGroups = (1 << 24) - 1;  // of 256 threads
constexpr int kMaxY = 65535;

int bad(const char* who, const char* what) { return fail(BTF_ERR_ARGS, std::string(who) + ": " + what); }

int check_kv(const btf_kv_cache* kv, const char* who, bool need_data) {
  if (!kv) return bad(who, "null cache");
  if (kv->type != BTF_F16 && kv->type != BTF_BF16) return bad(who, "unknown cache type");
  if (kv->page < 16 || kv->page > 256 || (kv->page & (kv->page - 1)))
    return bad(who, "a page holds 16, 32, 64, 128 or 256 tokens");
  if (kv->dim != 64 && kv->dim != 128 && kv->dim != 256) return bad(who, "head dim must be 64, 128 or 256");
  if (kv->heads < 1) return bad(who, "no KV heads");
  if (!need_data) return BTF_OK;
  if (!kv->k || !kv->v) return bad(who, "null cache pointer");
  if (!aligned(kv->k, 16) || !aligned(kv->v, 16)) return bad(who, "k and v must be 16-byte aligned");
  if (kv->pages < 1 || kv->pages > (int64_t)0x7fffffff / kv->page) return bad(who, "pages * page must be in [1, 2^31)");
  if (kv->page_stride < 0 || kv->head_stride < 0 || kv->tok_stride < kv->dim || kv->page_stride % 8 ||
      kv->head_stride % 8 || kv->tok_stride % 8)
    return bad(who, "cache strides must be multiples of 8 values, a token's at least the head dim");
  if (kv->tok_stride > 1 << 24) return bad(who, "a token's stride must be at most 2^24 values");
  return BTF_OK;
}

// What the attentions ask of the arguments that they have in common.
template <class A>
int check_attention(const A* a, const btf_kv_cache* kv, const char* who) {
  const int rc = check_kv(kv, who, true);
  if (rc != BTF_OK) return rc;
  if (a->heads < 1 || a->heads % kv->heads) return bad(who, "heads must be a multiple of the KV heads");
  if (!a->q || !a->table || !a->row0 || !a->kv_len || !a->out) return bad(who, "null pointer");
  if (!aligned(a->q, 16) || a->ldq % 8 || (int64_t)a->ldq < (int64_t)a->heads * kv->dim)
    return bad(who, "q must be 16-byte aligned with ldq % 8 == 0 and ldq >= heads * dim");
  if (!aligned(a->out, 16) || a->ldo % 4 || (int64_t)a->ldo < (int64_t)a->heads * kv->dim)
    return bad(who, "out must be 16-byte aligned with ldo % 4 == 0 and ldo >= heads * dim");
  if (a->heads > 65535 || (int64_t)a->T * a->heads > 0x7fffffff)
    return bad(who, "heads above 65535, or rows times heads above 2^31");
  if (a->ldt < 1) return bad(who, "ldt must be at least 1");
  if (!aligned(a->tree, 8)) return bad(who, "tree must be 8-byte aligned");
  if (!(a->scale == a->scale)) return bad(who, "scale is not a number");
  if (!a->ws || !aligned(a->ws, 16)) return bad(who, "ws must be 16-byte aligned scratch");
  return BTF_OK;
}

// A cache that is written, in several layers.
int check_layers(const btf_kv_cache* kv, int layers, int64_t stride, const char* who) {
  const int rc = check_kv(kv, who, true);
  if (rc != BTF_OK) return rc;
  if (layers < 1 || layers > kMaxY) return bad(who, "layers must be in [1, 65535]");
  if ((kv->heads > 1 && kv->head_stride < kv->dim) || (kv->pages > 1 && kv->page_stride < kv->dim) ||
      (layers > 1 && stride < kv->dim))
    return bad(who, "heads, pages or layers of the cache overlap");
  if (layers > 1 && stride % 8) return bad(who, "layer_stride must be a multiple of 8 values");
  return BTF_OK;
}

}  // namespace

extern "C" {

int btf_hip_launch_page_plan(const btf_page_plan* a, btf_stream_t stream) {
  if (!a) return bad("page_plan", "null arguments");
  if (a->S <= 0) return BTF_OK;
  if (a->T < 0) return bad("page_plan", "negative rows");
  if (a->page < 1 || (a->page & (a->page - 1))) return bad("page_plan", "page must be a power of two");
  if (a->ldt < 1) return bad("page_plan", "ldt must be at least 1");
  if (a->pages < 1 || a->pages > (int64_t)0x7fffffff / a->page) return bad("page_plan", "pages * page must be in [1, 2^31)");
  if (!a->ctx || !a->n_new || !a->held || !a->free_list || !a->n_free || !a->table || !a->held_out || !a->n_free_out ||
      !a->row0 || !a->kv_len || (a->T && (!a->pos || !a->slot)))
    return bad("page_plan", "null pointer");
  if ((a->parent == nullptr) != (a->tree == nullptr)) return bad("page_plan", "parent and tree go together");
  if (!aligned(a->tree, 8)) return bad("page_plan", "tree must be 8-byte aligned");
  if (a->S >= 1 << 26 || a->T > kMaxY * 1024) return bad("page_plan", "more requests or rows than a launch takes");
  if (!current_state()) return BTF_ERR_NOT_INIT;
  return page_plan(*a, static_cast<hipStream_t>(stream));
}

int btf_hip_rope_table(int n_rot, double base, const btf_rope_scale* sc, double* turns, float* mscale) {
  if (!turns || !mscale) return bad("rope_table", "null output");
  if (n_rot < 2 || n_rot % 2) return bad("rope_table", "n_rot must be even and positive");
  if (!(base > 1.0) || std::isinf(base)) return bad("rope_table", "base must be above 1 and finite");
  if (sc && sc->kind != BTF_ROPE_NONE) {
    if (sc->kind != BTF_ROPE_LINEAR && sc->kind != BTF_ROPE_NTK && sc->kind != BTF_ROPE_YARN)
      return bad("rope_table", "unknown scaling");
    if (!(sc->factor >= 1.0) || std::isinf(sc->factor)) return bad("rope_table", "factor must be at least 1 and finite");
    if (sc->kind == BTF_ROPE_NTK && n_rot < 4) return bad("rope_table", "ntk needs n_rot > 2");
    if (sc->kind == BTF_ROPE_NTK && std::isinf(base * std::pow(sc->factor, (double)n_rot / (n_rot - 2))))
      return bad("rope_table", "ntk makes the base infinite");
    if (sc->kind == BTF_ROPE_YARN && !(sc->trained > 0.0 && std::isfinite(sc->trained) && sc->beta_slow > 0.0 &&
                                       sc->beta_fast > sc->beta_slow && std::isfinite(sc->beta_fast)))
      return bad("rope_table", "yarn needs finite trained > 0 and beta_fast > beta_slow > 0");
  }
  return rope_table(n_rot, base, sc, turns, mscale);
}

int btf_hip_launch_rope_cache(const btf_rope_cache* a, const btf_kv_cache* kv, btf_stream_t stream) {
  if (!a) return bad("rope_cache", "null arguments");
  if (a->T <= 0) return BTF_OK;
  const bool q = a->q != nullptr, k = a->k != nullptr;
  if (!q && !k) return bad("rope_cache", "neither q nor k");
  if (k != (a->v != nullptr)) return bad("rope_cache", "k and v go together");
  const int rc = check_kv(kv, "rope_cache", k);
  if (rc != BTF_OK) return rc;
  const int D = kv->dim;
  if (q && (a->heads < 1 || !a->q_out)) return bad("rope_cache", "q needs heads and q_out");
  if (q && ((int64_t)a->ldq < (int64_t)a->heads * D || (int64_t)a->ldqo < (int64_t)a->heads * D))
    return bad("rope_cache", "ldq or ldqo below the heads' values");
  if (k && ((int64_t)a->ldk < (int64_t)kv->heads * D || (int64_t)a->ldv < (int64_t)kv->heads * D))
    return bad("rope_cache", "ldk or ldv below the heads' values");
  if (k && !a->slot) return bad("rope_cache", "k needs slots");
  if (k && ((kv->heads > 1 && kv->head_stride < D) || (kv->pages > 1 && kv->page_stride < D)))
    return bad("rope_cache", "heads or pages of the cache overlap");
  if (a->n_rot < 0 || a->n_rot > D || a->n_rot % 2) return bad("rope_cache", "n_rot must be even, in [0, dim]");
  if (a->layout != BTF_ROPE_HALF && a->layout != BTF_ROPE_PAIRS) return bad("rope_cache", "unknown layout");
  if (a->n_rot && (!a->turns || !a->pos)) return bad("rope_cache", "null turns or pos");
  if (!aligned(a->turns, 8) || !aligned(a->q, 4) || !aligned(a->k, 4) || !aligned(a->v, 4) || !aligned(a->q_out, 2))
    return bad("rope_cache", "pointers must have their types' alignment");
  if (a->T > kMaxGroups || (q ? a->heads : 0) + (k ? (int64_t)2 * kv->heads : 0) > kMaxY)
    return bad("rope_cache", "more rows or heads than a launch takes");
  if (!current_state()) return BTF_ERR_NOT_INIT;
  // Vector accesses where every head's pairs start at a multiple of their size
  const bool pairs = a->layout == BTF_ROPE_PAIRS;
  const int u = pairs ? 4 : 2;  // values in an access
  bool vec = pairs || a->n_rot % 4 == 0;
  if (q) vec = vec && aligned(a->q, 4 * u) && a->ldq % u == 0 && aligned(a->q_out, 2 * u) && a->ldqo % u == 0;
  if (k) vec = vec && aligned(a->k, 4 * u) && a->ldk % u == 0 && aligned(a->v, 4 * u) && a->ldv % u == 0;
  return rope_cache(*a, *kv, vec, static_cast<hipStream_t>(stream));
}

int64_t btf_hip_paged_attention_ws_bytes(int S, int T, int heads, const btf_kv_cache* kv) {
  if (S <= 0 || T <= 0 || check_kv(kv, "paged_attention_ws_bytes", false) != BTF_OK || heads < 1 || heads % kv->heads)
    return 0;
  return paged_attention_ws_bytes(S, T, heads, *kv);
}

int btf_hip_launch_paged_attention(const btf_paged_attention* a, const btf_kv_cache* kv, btf_stream_t stream) {
  if (!a) return bad("paged_attention", "null arguments");
  if (a->S <= 0 || a->T <= 0) return BTF_OK;
  const int rc = check_attention(a, kv, "paged_attention");
  if (rc != BTF_OK) return rc;
  if (a->T > kMaxGroups || paged_attention_most_items(a->S, a->T, a->heads, *kv) > kMaxGroups)
    return bad("paged_attention", "more rows or requests than a launch takes");
  if (!current_state()) return BTF_ERR_NOT_INIT;
  return paged_attention(*a, *kv, static_cast<hipStream_t>(stream));
}

int64_t btf_hip_sample_ws_bytes(int M, int V) { return M > 0 && V > 0 ? sample_ws_bytes(M, V) : 0; }

int btf_hip_launch_sample(const btf_sampling* a, btf_stream_t stream) {
  if (!a) return bad("sample", "null arguments");
  if (a->M <= 0) return BTF_OK;
  if (a->V <= 0) return bad("sample", "empty vocabulary");
  if (a->V > 1 << 20) return bad("sample", "more than 2^20 logits");
  if (a->M > 1 && a->ldl < a->V) return bad("sample", "ldl < V");
  if (!a->logits || !a->u || !a->token) return bad("sample", "null pointer");
  if (sample_ws_bytes(a->M, a->V) > 0 && (!a->ws || !aligned(a->ws, 8))) return bad("sample", "ws must be 8-byte aligned scratch");
  if (!current_state()) return BTF_ERR_NOT_INIT;
  return sample(*a, static_cast<hipStream_t>(stream));
}

int btf_hip_launch_page_fork(const btf_page_fork* a, btf_stream_t stream) {
  if (!a) return bad("page_fork", "null arguments");
  if (a->F <= 0) return BTF_OK;
  if (a->F > 1024) return bad("page_fork", "more than 1024 forks");
  if (a->S < 1) return bad("page_fork", "no rows of table");
  if (a->page < 1 || (a->page & (a->page - 1))) return bad("page_fork", "page must be a power of two");
  if (a->ldt < 1) return bad("page_fork", "ldt must be at least 1");
  if (a->pages < 1 || a->pages > (int64_t)0x7fffffff / a->page) return bad("page_fork", "pages * page must be in [1, 2^31)");
  if (!a->src || !a->dst || !a->tokens || !a->free_list || !a->n_free || !a->table || !a->held || !a->shared || !a->got ||
      !a->copy_from || !a->copy_to || !a->copy_tokens)
    return bad("page_fork", "null pointer");
  if (!current_state()) return BTF_ERR_NOT_INIT;
  return page_fork(*a, static_cast<hipStream_t>(stream));
}

int btf_hip_launch_page_copy(const btf_page_copy* a, const btf_kv_cache* kv, btf_stream_t stream) {
  if (!a) return bad("page_copy", "null arguments");
  if (a->n <= 0) return BTF_OK;
  const int rc = check_layers(kv, a->layers, a->layer_stride, "page_copy");
  if (rc != BTF_OK) return rc;
  if (!a->from || !a->to) return bad("page_copy", "null pointer");
  if ((int64_t)2 * a->n * kv->heads > kMaxGroups) return bad("page_copy", "more entries times heads than a launch takes");
  if (!current_state()) return BTF_ERR_NOT_INIT;
  return page_copy(*a, *kv, static_cast<hipStream_t>(stream));
}

int64_t btf_hip_page_free_ws_bytes(int S, int ldt) {
  return S > 0 && ldt > 0 && (int64_t)S * ldt < 1 << 29 ? page_free_ws_bytes(S, ldt) : 0;
}

int btf_hip_launch_page_free(const btf_page_free* a, btf_stream_t stream) {
  if (!a) return bad("page_free", "null arguments");
  if (a->S <= 0) return BTF_OK;
  if (a->page < 1 || (a->page & (a->page - 1))) return bad("page_free", "page must be a power of two");
  if (a->ldt < 1) return bad("page_free", "ldt must be at least 1");
  if ((int64_t)a->S * a->ldt >= 1 << 29) return bad("page_free", "S * ldt must be below 2^29");
  if (a->pages < 1 || a->pages > (int64_t)0x7fffffff / a->page) return bad("page_free", "pages * page must be in [1, 2^31)");
  if (!a->keep || !a->table || !a->held || !a->free_list || !a->n_free) return bad("page_free", "null pointer");
  if (page_free_ws_bytes(a->S, a->ldt) > 0 && (!a->ws || !aligned(a->ws, 4)))
    return bad("page_free", "ws must be 4-byte aligned scratch");
  if (!current_state()) return BTF_ERR_NOT_INIT;
  return page_free(*a, static_cast<hipStream_t>(stream));
}

int btf_hip_launch_cache_move(const btf_cache_move* a, const btf_kv_cache* kv, btf_stream_t stream) {
  if (!a) return bad("cache_move", "null arguments");
  if (a->S <= 0) return BTF_OK;
  const int rc = check_layers(kv, a->layers, a->layer_stride, "cache_move");
  if (rc != BTF_OK) return rc;
  if (a->T < 0 || a->T > 1 << 30) return bad("cache_move", "T must be in [0, 2^30]");
  if (!a->table || !a->first) return bad("cache_move", "null pointer");
  if ((a->tree != nullptr) == (a->source != nullptr)) return bad("cache_move", "either tree or source");
  if (a->tree ? !a->leaf : !a->source0) return bad("cache_move", "tree needs leaf, source needs source0");
  if (!aligned(a->tree, 8)) return bad("cache_move", "tree must be 8-byte aligned");
  if (a->ldt < 1 || (a->to_table && a->ldt_to < 1)) return bad("cache_move", "ldt must be at least 1");
  if ((int64_t)2 * a->S * kv->heads * (kv->dim / 64) > kMaxGroups / 4)
    return bad("cache_move", "more requests times heads than a launch takes");
  if (!current_state()) return BTF_ERR_NOT_INIT;
  return cache_move(*a, *kv, static_cast<hipStream_t>(stream));
}

int64_t btf_hip_shared_attention_ws_bytes(int S, int T, int heads, const btf_kv_cache* kv) {
  if (S <= 0 || T <= 0 || check_kv(kv, "shared_attention_ws_bytes", false) != BTF_OK || heads < 1 || heads % kv->heads)
    return 0;
  return shared_attention_ws_bytes(S, T, heads, *kv);
}

int btf_hip_launch_shared_attention(const btf_shared_attention* a, const btf_kv_cache* kv, btf_stream_t stream) {
  if (!a) return bad("shared_attention", "null arguments");
  if (a->S <= 0 || a->T <= 0) return BTF_OK;
  const int rc = check_attention(a, kv, "shared_attention");
  if (rc != BTF_OK) return rc;
  if (a->groups < 0 || a->groups > a->S) return bad("shared_attention", "groups must be in [0, S]");
  if (a->groups && (!a->group0 || !a->lead || !a->shared)) return bad("shared_attention", "null pointer of the groups");
  if (a->T > kMaxGroups || shared_attention_most_items(a->S, a->T, a->heads, *kv) > kMaxGroups)
    return bad("shared_attention", "more rows or requests than a launch takes");
  if (!current_state()) return BTF_ERR_NOT_INIT;
  return shared_attention(*a, *kv, static_cast<hipStream_t>(stream));
}

int64_t btf_hip_lora_ws_bytes(int S, int T, int K, int rank, int nseg) {
  if (S <= 0 || T <= 0 || K <= 0 || rank <= 0 || rank > 256 || nseg < 1 || nseg > 3) return 0;
  return lora_ws_bytes(S, T, K, rank, nseg);
}

int btf_hip_launch_lora(const btf_lora* a, const btf_lora_seg* segs, int nseg, btf_stream_t stream) {
  if (!a) return bad("lora", "null arguments");
  if (a->S <= 0 || a->T <= 0) return BTF_OK;
  if (nseg < 1 || nseg > 3 || !segs) return bad("lora", "1..3 segments");
  if (a->mode != BTF_GEMV_ADD && a->mode != BTF_GEMV_SWIGLU) return bad("lora", "mode must be add or swiglu");
  const bool glu = a->mode == BTF_GEMV_SWIGLU;
  if (glu && (nseg != 2 || segs[0].N != segs[1].N)) return bad("lora", "swiglu takes two segments of the same N");
  if (a->K < 32 || a->K % 32 || a->K > 1 << 24) return bad("lora", "K must be a multiple of 32 in [32, 2^24]");
  if (a->rank < 8 || a->rank % 8 || a->rank > 256) return bad("lora", "rank must be a multiple of 8 up to 256");
  if (a->adapters < 0) return bad("lora", "negative number of adapters");
  if (a->type != BTF_F16 && a->type != BTF_BF16) return bad("lora", "unknown type");
  if (!a->row0 || !a->adapter || !a->x) return bad("lora", "null pointer");
  if (!aligned(a->x, 16) || a->ldx % 4 || a->ldx < a->K) return bad("lora", "x must be 16-byte aligned with ldx % 4 == 0 and ldx >= K");
  if (glu && (!a->out || !aligned(a->out, 4) || a->ldo < segs[0].N)) return bad("lora", "swiglu needs out with ldo >= N");
  int64_t outs = 0;
  for (int i = 0; i < nseg; ++i) {
    const btf_lora_seg& g = segs[i];
    if (g.N < 1) return bad("lora", "a segment needs outputs");
    if (!g.y || !aligned(g.y, 4) || g.ldy < g.N) return bad("lora", "y must be given with ldy >= N");
    if (a->adapters && (!g.a || !g.b)) return bad("lora", "null adapters");
    if (!aligned(g.a, 16) || !aligned(g.b, 16)) return bad("lora", "a and b must be 16-byte aligned");
    if (g.a_stride < 0 || g.b_stride < 0 || g.a_stride % 8 || g.b_stride % 8)
      return bad("lora", "adapter strides must be multiples of 8 values");
    outs += g.N;
  }
  if (a->S > kMaxGroups / 4 || a->T > kMaxGroups / 4 || outs > 1 << 24 || lora_most_groups(a->S, a->T, glu ? segs[0].N : outs, nseg) > kMaxGroups)
    return bad("lora", "more requests, rows or outputs than a launch takes");
  if (!a->ws || !aligned(a->ws, 16)) return bad("lora", "ws must be 16-byte aligned scratch");
  if (!current_state()) return BTF_ERR_NOT_INIT;
  return lora(*a, segs, nseg, static_cast<hipStream_t>(stream));
}

}  // extern "C"
