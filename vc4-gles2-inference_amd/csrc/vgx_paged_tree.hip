// Attention of drafted trees over a paged cache: the same kernels with a mask
// for each row.
#include "vgx_paged_attn.h"

hipError_t vgx_paged_tree_init() { return attn_init<true>(); }

extern "C" {

size_t vgx_paged_attn_tree_ws(vgx_ctx* ctx, const vgx_paged* cache, const vgx_ragged* batch, int window) {
    return attn_ws<true>("vgx_paged_attn_tree_ws", ctx, cache, batch, window);
}

int vgx_paged_attn_tree(vgx_ctx* ctx, const vgx_paged* cache, const vgx_ragged* batch, const vgx_paged_query* r,
                        const vgx_tree* tree) {
    return attn_call<true>("vgx_paged_attn_tree", ctx, cache, batch, r, tree);
}

}  // extern "C"
