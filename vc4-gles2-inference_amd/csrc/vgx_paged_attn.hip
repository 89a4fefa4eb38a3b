// Attention of a ragged batch's new tokens over a paged cache.
#include "vgx_paged_attn.h"

hipError_t vgx_paged_attn_init() { return attn_init<false>(); }

extern "C" {

size_t vgx_paged_attn_ws(vgx_ctx* ctx, const vgx_paged* cache, const vgx_ragged* batch, int window) {
    return attn_ws<false>("vgx_paged_attn_ws", ctx, cache, batch, window);
}

int vgx_paged_attn(vgx_ctx* ctx, const vgx_paged* cache, const vgx_ragged* batch, const vgx_paged_query* r) {
    return attn_call<false>("vgx_paged_attn", ctx, cache, batch, r, nullptr);
}

}  // extern "C"
