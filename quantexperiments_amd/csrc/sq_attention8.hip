// sq_tree_attention8: argument checks and launch.  Calls are cut into workgroups as over a 16-bit cache (attn_plan).
#include "sq_attention8.h"

namespace sq {

// the cache as one of 16-bit elements, for what does not read it
static sq_cache as_cache(const sq_cache8& c, int dtype) {
    return {c.k, c.v, c.k_page, c.k_slot, c.k_head, c.v_page, c.v_slot, c.v_head, c.pages, c.page, c.heads, c.dim, dtype};
}

static int check_attention8(const char* who, const sq_attention* a, const sq_cache8* cache, int dtype, sq_cache& c) {
    if (!a || !cache) return fail(SQ_EINVAL, "%s: null argument", who);
    if (int rc = check_cache8(who, cache)) return rc;
    c = as_cache(*cache, dtype);
    return check_attention(who, a, &c);
}

}  // namespace sq

using namespace sq;

extern "C" {

size_t sq_tree_attention8_workspace_bytes(const sq_attention* a, const sq_cache8* cache, int dtype) {
    sq_cache c;
    if (check_attention8("sq_tree_attention8_workspace_bytes", a, cache, dtype, c) || attn_nothing(*a)) return 0;
    return attn_workspace(*a, attn_plan(*a, c, true));
}

int sq_tree_attention8(const sq_attention* a, const sq_cache8* cache, int dtype, void* workspace, size_t ws_bytes, void* stream) {
    const char* who = "sq_tree_attention8";
    sq_cache c;
    if (int rc = check_attention8(who, a, cache, dtype, c)) return rc;
    if (attn_nothing(*a)) return SQ_OK;
    const AttnPlan p = attn_plan(*a, c, true);
    Attn8Shared k;
    if (int rc = attn_prepare(who, *a, c, p, workspace, ws_bytes, k)) return rc;
    k.k_page = cache->k_page; k.k_slot = cache->k_slot; k.k_head = cache->k_head; k.v_page = cache->v_page; k.v_slot = cache->v_slot; k.v_head = cache->v_head;
    k.near = 1;
    k.ks = cache->k_scale; k.vs = cache->v_scale;
    k.ks_page = cache->ks_page; k.ks_block = cache->ks_block; k.ks_head = cache->ks_head;
    k.vs_page = cache->vs_page; k.vs_block = cache->vs_block; k.vs_head = cache->vs_head;
    k.size = cache->page / cache->blocks;
    k.block = p.nw ? __builtin_ctz((unsigned)(p.mt * 16 * p.nw)) : 0;
    k.parts = p.workgroups ? (int32_t*)(k.pml + (size_t)a->tokens * a->q_heads * p.slots) : nullptr;
    // Rows of heads that share lines of 128 bytes are fetched into each die's cache that reads one: 64 sequences of 4000 slots, 8 key heads of 64, 84 us, with a line's heads on
    // one die 62.  Of others, dealt out one behind the other, 32 sequences of 8192 x 8 of 128 108 us, so 115.
    k.inner = (cache->dim % 128 ? cache->heads : 1) * p.row_blocks;
    // What is read once, and more than a few MB, is read past the dies' caches and those in front of HBM (between two calls on a layer's cache lie the other layers' and the weights): 32
    // sequences of 4000 slots x 4 key heads of 128, one set of several 32.6 us, so 28.6; the same set again and again 29.1 and 26.6; one of 131,072 35.8 and 31.5; 32 of 2,240 to 8,192 x 8
    // 74 and 62.  Less is bound by its chain of loads: 8 of 2000 9.3 us where it is still in those caches, so 10.0 (where not, 14.0 and 12.9).  (By the tables' width: lengths are on the device.)
    k.passing = 2 * (int64_t)a->seqs * a->max_pages * cache->page * cache->heads * cache->dim > (int64_t)16 << 20;
    return dtype == SQ_F16 ? attn8_launch_f16(k, p, (hipStream_t)stream) : attn8_launch_bf16(k, p, (hipStream_t)stream);
}

}  // extern "C"
