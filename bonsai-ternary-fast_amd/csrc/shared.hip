#include "common.h"
namespace btfhip {
int64_t shared_attention_most_items(int, int, int, const btf_kv_cache&) { return 0; }
int64_t shared_attention_ws_bytes(int, int, int, const btf_kv_cache&) { return 16; }
int shared_attention(const btf_shared_attention&, const btf_kv_cache&, hipStream_t) { return fail(BTF_ERR_LAUNCH, "shared_attention: not built"); }
}
