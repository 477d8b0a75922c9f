// sq_tree_attention: argument checks, and how a call is cut into workgroups.
#include "sq_attention.h"

namespace sq {

// Up to 32 rows (16 of wide heads): one workgroup for all of them, its waves splitting the keys; more: four or eight waves with 32 rows each (16).
// Sequences are cut until the chip has a workgroup per compute unit, few rows not into less than a step per wave nor into two such parts, many rows not into
// less than four steps, or two in up to eight parts.  (The joining launch takes 2 to 3 us, a step of a wave 1: one token behind 300 slots whole 8.0, in two parts 8.9 us;
// behind 500 whole 10.5, in four 9.1; behind 4000 in 15 parts of two steps a wave 12.3, in 31 of one 10.0.  40 tokens behind 1000 in 8 parts 22.5, in 16 28.9; behind
// 256 in two parts 18.7, in four 18.2.)  Sequences of several lengths are cut for two rounds of workgroups where a wave then still has eight steps: 32 of 2,240 to 8,192 slots x 8 key
// heads 131 us, 154 in one round, 64 of up to 4000 x 4 heads 69 and 77; with fewer steps it costs more than it evens out: 64 of up to 500 14.1 us in one round, 19.5 in
// two, 16 of 2000 x 8 heads 26.6 and 30.4.
// A last block of rows that fills at most half of its waves takes 0.6 of the time, and gets as many fewer parts: 8 trees of 32 tokens of 5 heads of 256 per
// key head (160 rows in blocks of 128) 42.3 us evenly, 39.3 so; with 0.75 42.1.
// (All times of captured calls, one behind the other; calls back to back take up to 4 % less.)
// A sequence's length is its table's width here: lengths are on the device.  Under a table of 131,072 slots one token behind 500 takes 10.2 us instead of 8.8, 48 26.7 instead of 21.4,
// 64 sequences of 500 27.9 instead of 18.6, 64 of 2000 59.8 instead of 53.1.
static AttnPlan attn_plan(const sq_attention& a, const sq_cache& c) {
    AttnPlan p;
    p.dp = c.dim <= 64 ? 64 : c.dim <= 128 ? 128 : 256;
    const int64_t rows = (int64_t)a.most_new * (a.q_heads / c.heads), steps = ((int64_t)a.max_pages * c.page + ATTN_STEP - 1) / ATTN_STEP;
    const int waves = attn_waves(p.dp);
    int64_t per, most;
    if (rows <= (p.dp == 256 ? 16 : 32)) {
        p.nw = 0;
        p.mt = rows <= 16 ? 1 : 2;
        per = p.mt * 16;
        most = steps / waves;
        if (most <= 2) most = 1;
    } else {
        p.mt = attn_tiles(p.dp);
        p.nw = rows <= 4 * 16 * p.mt ? 4 : 8;
        per = p.mt * 16 * p.nw;
        most = steps / 4 > 8 ? steps / 4 : steps / 2 < 8 ? steps / 2 : 8;
    }
    p.row_blocks = (int)((rows + per - 1) / per);
    const int64_t base = (int64_t)a.seqs * c.heads * p.row_blocks, cus = device_cus();
    int64_t want = cus / base;
    if (a.seqs > 1 && !p.nw && 2 * cus / base > 1 && steps / (2 * cus / base) >= 8 * waves) want = 2 * cus / base;
    p.splits = (int)(want < most ? want : most);
    if (p.splits < 1) p.splits = 1;
    if (p.splits > ATTN_SPLITS_MAX) p.splits = ATTN_SPLITS_MAX;
    p.last_splits = p.splits;
    p.last_row = (int)((p.row_blocks - 1) * per);
    const int64_t waves_last = (rows - p.last_row + p.mt * 16 - 1) / (p.mt * 16);
    if (p.nw == 8 && p.row_blocks > 1 && waves_last <= 4) {
        const int64_t room = cus / ((int64_t)a.seqs * c.heads);
        for (int s = (int)(room < most ? room : most); s > 1; --s) {
            const int last = (s * 60 + 99) / 100;            // (two or more)
            if ((p.row_blocks - 1) * (int64_t)s + last > room) continue;
            if (s <= ATTN_SPLITS_MAX) p.splits = s, p.last_splits = last;
            break;
        }
    }
    return p;
}

static int check_attention(const char* who, const sq_attention* a, const sq_cache* c) {
    if (!a || !c) return fail(SQ_EINVAL, "%s: null argument", who);
    if (c->dtype != SQ_F16 && c->dtype != SQ_BF16) return fail(SQ_EINVAL, "%s: dtype %d (fp16 or bf16)", who, c->dtype);
    if (c->dim < 8 || c->dim > 256 || c->dim % 8) return fail(SQ_EUNSUPPORTED, "%s: heads of %d elements (a multiple of 8 up to 256)", who, c->dim);
    if (c->heads < 1 || a->q_heads < 1 || a->q_heads % c->heads) return fail(SQ_EINVAL, "%s: %d query heads for %d key heads", who, a->q_heads, c->heads);
    if (a->tokens < 0 || a->seqs < 0 || a->most_new < 0 || a->q_heads > (1 << 16) || a->max_pages < 0 || c->pages < 0 || c->page < 1 || a->mask_words < 0 ||
        a->ld_table < a->max_pages)
        return fail(SQ_EINVAL, "%s: %d tokens, %d sequences, at most %d new, tables of %d (ld %lld), %d pages of %d", who, a->tokens, a->seqs, a->most_new, a->max_pages,
                    (long long)a->ld_table, c->pages, c->page);
    if ((int64_t)a->seqs * a->most_new > INT32_MAX / a->q_heads)          // (no more rows than 32 bits count: a plan of more would wrap)
        return fail(SQ_EUNSUPPORTED, "%s: %d sequences of up to %d new tokens and %d heads at once", who, a->seqs, a->most_new, a->q_heads);
    if (!(a->scale > 0.f) || a->scale > 2.3e38f) return fail(SQ_EINVAL, "%s: scale %g", who, (double)a->scale);          // (times log2 e a number)
    if (!a->starts && (int64_t)a->seqs * a->most_new != a->tokens)
        return fail(SQ_EINVAL, "%s: %d tokens are not %d for each of %d sequences", who, a->tokens, a->most_new, a->seqs);
    return SQ_OK;
}

static bool attn_nothing(const sq_attention& a) { return a.tokens == 0 || a.seqs == 0 || a.most_new == 0; }

}  // namespace sq

using namespace sq;

extern "C" {

size_t sq_tree_attention_workspace_bytes(const sq_attention* a, const sq_cache* cache) {
    if (check_attention("sq_tree_attention_workspace_bytes", a, cache) || attn_nothing(*a)) return 0;
    const AttnPlan p = attn_plan(*a, *cache);
    if (p.splits == 1) return 0;
    return (size_t)a->tokens * a->q_heads * p.splits * (p.dp * 4 + 8);
}

int sq_tree_attention(const sq_attention* a, const sq_cache* cache, void* workspace, size_t ws_bytes, void* stream) {
    const char* who = "sq_tree_attention";
    if (int rc = check_attention(who, a, cache)) return rc;
    if (attn_nothing(*a)) return SQ_OK;
    if (!a->max_pages || !cache->pages) return fail(SQ_EINVAL, "%s: new tokens without a page", who);
    if (!a->q || !a->out || !a->table || !a->lens || !cache->k || !cache->v) return fail(SQ_EINVAL, "%s: null argument", who);
    const int64_t strides = a->q_token | a->q_head | a->out_token | a->out_head | cache->k_page | cache->k_slot | cache->k_head | cache->v_page | cache->v_slot | cache->v_head;
    if (strides % 8 || (((uintptr_t)a->q | (uintptr_t)a->out | (uintptr_t)cache->k | (uintptr_t)cache->v) & 15))
        return fail(SQ_EUNSUPPORTED, "%s: q, out, keys and values need 16-byte aligned heads", who);
    const int64_t ot = a->out_token < 0 ? -a->out_token : a->out_token, oh = a->out_head < 0 ? -a->out_head : a->out_head;
    if (!rows_apart(a->tokens, a->q_heads, ot, oh, cache->dim)) return fail(SQ_EINVAL, "%s: rows of the output overlap (strides %lld, %lld)", who, (long long)ot, (long long)oh);
    const AttnPlan p = attn_plan(*a, *cache);
    if ((int64_t)a->seqs * cache->heads * p.row_blocks * p.splits > (1 << 23) || (p.splits > 1 && (int64_t)a->seqs * a->most_new * a->q_heads > (1 << 23)))
        return fail(SQ_EUNSUPPORTED, "%s: %d sequences of up to %d new tokens and %d heads at once", who, a->seqs, a->most_new, a->q_heads);
    const size_t need = p.splits == 1 ? 0 : (size_t)a->tokens * a->q_heads * p.splits * (p.dp * 4 + 8);
    if (ws_bytes < need || (need && (!workspace || ((uintptr_t)workspace & 255))))
        return fail(SQ_EWORKSPACE, "%s: workspace of %zu bytes (256-byte aligned) needed, %zu given", who, need, ws_bytes);
    AttnArgs k;
    k.q = (const char*)a->q; k.out = (char*)a->out; k.lse = a->lse; k.kc = (const char*)cache->k; k.vc = (const char*)cache->v;
    k.table = a->table; k.lens = a->lens; k.starts = a->starts; k.mask = a->mask;
    k.po = (float*)workspace;
    k.pml = (float2v*)((float*)workspace + (need ? (size_t)a->tokens * a->q_heads * p.splits * p.dp : 0));
    k.q_t = a->q_token * 2; k.q_h = a->q_head * 2; k.o_t = a->out_token * 2; k.o_h = a->out_head * 2;
    k.k_page = cache->k_page * 2; k.k_slot = cache->k_slot * 2; k.k_head = cache->k_head * 2;
    k.v_page = cache->v_page * 2; k.v_slot = cache->v_slot * 2; k.v_head = cache->v_head * 2;
    k.ld_table = a->ld_table; k.ld_mask = a->ld_mask;
    k.tokens = a->tokens; k.seqs = a->seqs; k.most_new = a->most_new; k.q_heads = a->q_heads; k.kv_heads = cache->heads; k.group = a->q_heads / cache->heads;
    k.dim = cache->dim; k.pages = cache->pages; k.page = cache->page; k.max_pages = a->max_pages; k.mask_words = a->mask_words;
    k.row_blocks = p.row_blocks; k.splits = p.splits; k.last_splits = p.last_splits; k.last_row = p.last_row;
    auto near = [&](int64_t b) { return b >= 0 && b < (1 << 24) && b * (cache->page + 32) < INT32_MAX; };
    k.near = near(k.k_slot) && near(k.v_slot);
    k.scale2 = a->scale * 1.4426950408889634f;
    return cache->dtype == SQ_F16 ? attn_launch_f16(k, p, (hipStream_t)stream) : attn_launch_bf16(k, p, (hipStream_t)stream);
}

}  // extern "C"
