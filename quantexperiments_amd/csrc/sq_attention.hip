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
// Over a cache held in 8 bits a compute unit holds two of the few-row workgroups (four of heads up to 64 in blocks of 16 rows), and sequences are also cut into parts of 20 steps a wave, which ends
// them closer together: 64 sequences of 8192 slots x 8 key heads in three parts 205 us, whole 218; of 2,240 to 8,192 131 and 152; 32 of those 72 and 91; 32 of 4000 x 2 key heads of 64 in
// eight 12.9, in four 14.3.
// One of up to four steps a wave is not cut (a step takes 0.6 us then: one token behind 500 slots 8.7 us call by call, in four parts 10.1; captured 8.5 and 8.1; of heads of 256 12.1 and 9.9,
// which are).
// There the few-row kernel also takes more rows, in blocks of 32 or 16, one workgroup each, that read the same keys on one die: it has no barriers, starts and ends in 5 us where the many-row kernel
// takes 10, and reads ahead twice as far.  Up to 128 rows always, but for the shortest tables (28 + 4 heads of 128: 8 new tokens behind 64 x 2000 slots 70.5 us in the other, 40.2 in this; 5 behind 128 x 100
// 17.3 and 20.5).  More while the many-row kernel leaves half of the compute units idle (a batch of 4 x 250 new tokens 31.1 and 20.8, of 4 x 500 31.5 and 42.0) and a unit has at
// most 96 products of a 16-row block with a step, 256 of sequences that are short: 48 behind 4000 27.9 and 20.2, 200 behind 4000 40 and 46; 500 behind 1000 36.4 and 27.2, 1000 behind 1000
// 56.1 and 58.4.  Heads of 256, blocks of 16 and one workgroup a compute unit: 48 per unit and a unit per block (16 new tokens of 5 heads behind 8 x 500 26.1 and 16.6, behind 16 x 500 27.1 and 30.1), up
// to 32 rows where there are 32 steps (4 behind 32 x 4000 94 and 61; 8 behind 64 x 200 19.6 and 30.8).  Blocks of 16 while all of them run at once and products are few: a step then takes
// 0.6 us, of 32 1.2 (8 behind 500 9.9 and 12.3, behind 4000 11.9 and 14.0; behind 32,000 25.9 and 22.5).
// A sequence's length is its table's width here: lengths are on the device.  Under a table of 131,072 slots, over a 16-bit cache, one token behind 500 takes 10.0 us instead of 8.9, 48 25.0 instead
// of 20.3, 64 sequences of 500 27.1 instead of 18.3, 32 of 4000 57.7 instead of 53.2; over one held in 8 bits, where a batch is then cut into 51 parts and drafts go to tiles, 9.7 instead of 8.3, 21.2 and
// 10.2, 85.8 and 11.1, 64.9 and 28.3; 64 of 2000 102 and 25.5, 8 new tokens behind 8 x 4000 57 and 21.7, 64 of 500 with heads of 64 50 and 9.3.
AttnPlan attn_plan(const sq_attention& a, const sq_cache& c, bool held8) {
    AttnPlan p;
    p.dp = c.dim <= 64 ? 64 : c.dim <= 128 ? 128 : 256;
    const int64_t rows = (int64_t)a.most_new * (a.q_heads / c.heads), steps = ((int64_t)a.max_pages * c.page + ATTN_STEP - 1) / ATTN_STEP;
    const int waves = held8 ? ATTN8_WAVES : attn_waves(p.dp);
    int64_t per, most;
    const int64_t cus = device_cus(), units = (int64_t)a.seqs * c.heads * ((rows + 15) / 16), load = units * steps;
    bool few = rows <= (p.dp == 256 ? 16 : 32);
    if (held8 && !few) {
        const int64_t tiles = (int64_t)a.seqs * c.heads * (rows <= 128 ? 1 : (rows + 255) / 256);
        if (p.dp == 256) few = (units <= cus && load <= 48 * cus) || (rows <= 32 && steps >= 32);
        else few = (rows <= 128 && steps >= 8) || (tiles * (steps < 4 ? 4 : 2) <= cus && (load <= 96 * cus || (steps <= 96 && load <= 256 * cus)));
    }
    if (few) {
        p.nw = 0;
        p.mt = rows <= 16 || p.dp == 256 || (held8 && units <= 2 * cus && load <= 32 * cus) ? 1 : 2;
        per = p.mt * 16;
        most = steps / waves;
        if (most <= (held8 && p.dp < 256 ? 4 : 2)) most = 1;
    } else {
        p.mt = attn_tiles(p.dp);
        p.nw = rows <= 4 * 16 * p.mt ? 4 : 8;
        per = p.mt * 16 * p.nw;
        most = steps / 4 > 8 ? steps / 4 : steps / 2 < 8 ? steps / 2 : 8;
    }
    p.row_blocks = (int)((rows + per - 1) / per);
    const int64_t base = (int64_t)a.seqs * c.heads * p.row_blocks;
    int64_t want = cus / base;
    if (held8 && !p.nw) {
        if (p.dp == 64) want = 2 * cus / base;
        if (want < steps / (20 * waves)) want = steps / (20 * waves);
    } else if (a.seqs > 1 && !p.nw && 2 * cus / base > 1 && steps / (2 * cus / base) >= 8 * waves) want = 2 * cus / base;
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
    p.slots = p.splits;
    // Over a cache held in 8 bits the blocks of rows of all sequences share a key head's workgroups by their work (attn8_share), where these are half as many again; an eighth more are enough for one
    // sequence's, of which the last sees most: 1900 tokens behind 2100 131 us, so 129.  (16 x 100 behind 1000, 48 blocks on 64 workgroups, 49.8 and 58.6.)
    const int64_t items = a.seqs * (int64_t)p.row_blocks, room = cus / c.heads;
    p.workgroups = 0;
    if (held8 && p.nw && items > 1 && items <= 64 && (a.seqs == 1 ? 8 * items <= 7 * room : 3 * items <= 2 * room) && steps < (1 << 17)) {
        p.workgroups = (int)room;
        const int64_t slots = 2 * p.workgroups / items;      // (two or more; the join of more than eight takes longer)
        p.slots = (int)(slots > 8 && slots <= 16 ? 8 : slots < ATTN_SPLITS_MAX ? slots : ATTN_SPLITS_MAX);
    }
    return p;
}

int check_attention(const char* who, const sq_attention* a, const sq_cache* c) {
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

bool attn_nothing(const sq_attention& a) { return a.tokens == 0 || a.seqs == 0 || a.most_new == 0; }

size_t attn_workspace(const sq_attention& a, const AttnPlan& p) {
    return p.slots == 1 ? 0 : (size_t)a.tokens * a.q_heads * p.slots * (p.dp * 4 + 8) + (p.workgroups ? (size_t)p.row_blocks * a.seqs * 4 : 0);
}

// Everything of a call that the kernels are told but the strides of its cache
int attn_prepare(const char* who, const sq_attention& a, const sq_cache& c, const AttnPlan& p, void* workspace, size_t ws_bytes, AttnArgs& k) {
    if (!a.max_pages || !c.pages) return fail(SQ_EINVAL, "%s: new tokens without a page", who);
    if (!a.q || !a.out || !a.table || !a.lens || !c.k || !c.v) return fail(SQ_EINVAL, "%s: null argument", who);
    const int64_t strides = a.q_token | a.q_head | a.out_token | a.out_head | c.k_page | c.k_slot | c.k_head | c.v_page | c.v_slot | c.v_head;
    if (strides % 8 || (((uintptr_t)a.q | (uintptr_t)a.out | (uintptr_t)c.k | (uintptr_t)c.v) & 15))
        return fail(SQ_EUNSUPPORTED, "%s: q, out, keys and values need 16-byte aligned heads", who);
    const int64_t ot = a.out_token < 0 ? -a.out_token : a.out_token, oh = a.out_head < 0 ? -a.out_head : a.out_head;
    if (!rows_apart(a.tokens, a.q_heads, ot, oh, c.dim)) return fail(SQ_EINVAL, "%s: rows of the output overlap (strides %lld, %lld)", who, (long long)ot, (long long)oh);
    if ((int64_t)a.seqs * c.heads * p.row_blocks * p.splits > (1 << 23) || (p.slots > 1 && (int64_t)a.seqs * a.most_new * a.q_heads > (1 << 23)))
        return fail(SQ_EUNSUPPORTED, "%s: %d sequences of up to %d new tokens and %d heads at once", who, a.seqs, a.most_new, a.q_heads);
    const size_t need = attn_workspace(a, p);
    if (ws_bytes < need || (need && (!workspace || ((uintptr_t)workspace & 255))))
        return fail(SQ_EWORKSPACE, "%s: workspace of %zu bytes (256-byte aligned) needed, %zu given", who, need, ws_bytes);
    k.q = (const char*)a.q; k.out = (char*)a.out; k.lse = a.lse; k.kc = (const char*)c.k; k.vc = (const char*)c.v;
    k.table = a.table; k.lens = a.lens; k.starts = a.starts; k.mask = a.mask;
    k.po = (float*)workspace;
    k.pml = (float2v*)((float*)workspace + (need ? (size_t)a.tokens * a.q_heads * p.slots * p.dp : 0));
    k.q_t = a.q_token * 2; k.q_h = a.q_head * 2; k.o_t = a.out_token * 2; k.o_h = a.out_head * 2;
    k.ld_table = a.ld_table; k.ld_mask = a.ld_mask;
    k.tokens = a.tokens; k.seqs = a.seqs; k.most_new = a.most_new; k.q_heads = a.q_heads; k.kv_heads = c.heads; k.group = a.q_heads / c.heads;
    k.dim = c.dim; k.pages = c.pages; k.page = c.page; k.max_pages = a.max_pages; k.mask_words = a.mask_words;
    k.row_blocks = p.row_blocks; k.splits = p.slots; k.last_splits = p.last_splits; k.last_row = p.last_row;
    k.scale2 = a.scale * 1.4426950408889634f;
    return SQ_OK;
}

}  // namespace sq

using namespace sq;

extern "C" {

size_t sq_tree_attention_workspace_bytes(const sq_attention* a, const sq_cache* cache) {
    if (check_attention("sq_tree_attention_workspace_bytes", a, cache) || attn_nothing(*a)) return 0;
    return attn_workspace(*a, attn_plan(*a, *cache));
}

int sq_tree_attention(const sq_attention* a, const sq_cache* cache, void* workspace, size_t ws_bytes, void* stream) {
    const char* who = "sq_tree_attention";
    if (int rc = check_attention(who, a, cache)) return rc;
    if (attn_nothing(*a)) return SQ_OK;
    const AttnPlan p = attn_plan(*a, *cache);
    AttnArgs k;
    if (int rc = attn_prepare(who, *a, *cache, p, workspace, ws_bytes, k)) return rc;
    k.k_page = cache->k_page * 2; k.k_slot = cache->k_slot * 2; k.k_head = cache->k_head * 2;
    k.v_page = cache->v_page * 2; k.v_slot = cache->v_slot * 2; k.v_head = cache->v_head * 2;
    auto near = [&](int64_t b) { return b >= 0 && b < (1 << 24) && b * (cache->page + 32) < INT32_MAX; };
    k.near = near(k.k_slot) && near(k.v_slot);
    return cache->dtype == SQ_F16 ? attn_launch_f16(k, p, (hipStream_t)stream) : attn_launch_bf16(k, p, (hipStream_t)stream);
}

}  // extern "C"
