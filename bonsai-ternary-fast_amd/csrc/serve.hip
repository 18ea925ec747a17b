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
  const int rc = check_kv(kv, "paged_attention", true);
  if (rc != BTF_OK) return rc;
  if (a->heads < 1 || a->heads % kv->heads) return bad("paged_attention", "heads must be a multiple of the KV heads");
  if (!a->q || !a->table || !a->row0 || !a->kv_len || !a->out) return bad("paged_attention", "null pointer");
  if (!aligned(a->q, 16) || a->ldq % 8 || (int64_t)a->ldq < (int64_t)a->heads * kv->dim)
    return bad("paged_attention", "q must be 16-byte aligned with ldq % 8 == 0 and ldq >= heads * dim");
  if (!aligned(a->out, 16) || a->ldo % 4 || (int64_t)a->ldo < (int64_t)a->heads * kv->dim)
    return bad("paged_attention", "out must be 16-byte aligned with ldo % 4 == 0 and ldo >= heads * dim");
  if (a->heads > 65535 || (int64_t)a->T * a->heads > 0x7fffffff)
    return bad("paged_attention", "heads above 65535, or rows times heads above 2^31");
  if (a->T > kMaxGroups || paged_attention_most_items(a->S, a->T, a->heads, *kv) > kMaxGroups)
    return bad("paged_attention", "more rows or requests than a launch takes");
  if (a->ldt < 1) return bad("paged_attention", "ldt must be at least 1");
  if (!aligned(a->tree, 8)) return bad("paged_attention", "tree must be 8-byte aligned");
  if (!(a->scale == a->scale)) return bad("paged_attention", "scale is not a number");
  if (paged_attention_ws_bytes(a->S, a->T, a->heads, *kv) > 0 && (!a->ws || !aligned(a->ws, 16)))
    return bad("paged_attention", "ws must be 16-byte aligned scratch");
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

}  // extern "C"
