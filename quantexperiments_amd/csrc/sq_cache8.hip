// A paged cache of keys and values held in 8 bits: new tokens put into it, and the accepted path of a draft moved behind its cached tokens.
//
// A block of tokens of one head has one scale 2^e, and an element x the code rne_e4m3(x * 2^-e): three bits of mantissa whatever e is, down to 2^-6 of the scale, so a
// scale that is a power of two loses nothing beside the exact a / 448 but, at worst, the last of the bits below that.  It buys that attention multiplies by the scale while it
// unpacks codes, exactly, and that a block whose scale grows with later tokens is scaled to it without another rounding (below 2^-6: with one).
#include "sq_common.h"

namespace sq {

struct Cache8 {
    char *k, *v;
    uint8_t *ks, *vs;
    int64_t k_page, k_slot, k_head, v_page, v_slot, v_head, ks_page, ks_block, ks_head, vs_page, vs_block, vs_head;      // bytes
    int pages, page, blocks, size, heads, dim;                     // size: tokens of a block
};
struct Put8Args {
    Cache8 c;
    const char *k, *v;
    int64_t k_t, k_h, v_t, v_h;                                     // bytes
    const int32_t *table, *lens, *starts;
    int64_t ld_table;
    int tokens, seqs, most_new, max_pages, runs;                    // runs: blocks that a sequence's new tokens may lie in
};
struct Keep8Args {
    Cache8 c;
    int64_t k_layer, v_layer, ks_layer, vs_layer;
    const int32_t *table, *lens, *path, *counts;
    int64_t ld_table, ld_path;
    int layers, max_pages, most;
};

// One head's codes and scales, of keys or of values
struct Plane8 { char* at; uint8_t* scale; int64_t page, slot, s_page, s_block; };
__device__ __forceinline__ Plane8 plane_of(const Cache8& c, bool v, int head) {
    if (v) return {c.v + head * c.v_head, c.vs + head * c.vs_head, c.v_page, c.v_slot, c.vs_page, c.vs_block};
    return {c.k + head * c.k_head, c.ks + head * c.ks_head, c.k_page, c.k_slot, c.ks_page, c.ks_block};
}

__device__ __forceinline__ float two_to(int e) { return __builtin_bit_cast(float, (uint32_t)min(max(e + 127, 1), 254) << 23); }

__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
    const auto h = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    v = max((uint32_t)h[0], (uint32_t)h[1]);
    const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = max((uint32_t)r[0], (uint32_t)r[1]);
    v = max(v, row_rotated_bits<8>(v));
    v = max(v, row_rotated_bits<4>(v));
    v = max(v, row_rotated_bits<2>(v));
    return max(v, row_rotated_bits<1>(v));
}

// 16 codes times 2^-down
__device__ __forceinline__ u32x4 scaled_codes(u32x4 x, int down) {
    const float by = two_to(-down);
    u32x4 y;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2v lo = __builtin_amdgcn_cvt_pk_f32_fp8(x[i], false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(x[i], true);
        y[i] = __builtin_amdgcn_cvt_pk_fp8_f32(lo[0] * by, lo[1] * by, 0, false);
        y[i] = __builtin_amdgcn_cvt_pk_fp8_f32(hi[0] * by, hi[1] * by, y[i], true);
    }
    return y;
}

// Scales slots of a page down, a piece of 16 elements per lane
__device__ __forceinline__ void scale_slots(const Plane8& p, int page, int slot, int n, int per, int down, int lane) {
    for (int x = lane; x < n * per; x += 64) {
        u32x4* at = reinterpret_cast<u32x4*>(p.at + page * p.page + (slot + x / per) * p.slot + x % per * 16);
        *at = scaled_codes(*at, down);
    }
}

template <int DT> struct Put8Type;
template <> struct Put8Type<SQ_F16> { static constexpr float MOST = 0x1.Ep15f; static __device__ __forceinline__ float get(uint32_t b) { return h2f((uint16_t)b); } };
template <> struct Put8Type<SQ_BF16> { static constexpr float MOST = 0x1.Ep127f; static __device__ __forceinline__ float get(uint32_t b) { return bf2f((uint16_t)b); } };

// One wave per block that gets new tokens, head, and keys or values: the largest magnitude over its tokens, then the codes.  Up to 8 pieces of
// 16 elements a lane stay in registers between the two (64 tokens of 128), larger blocks are read again.
constexpr int PUT8_KEEP = 8;
template <int DT>
__global__ __launch_bounds__(256) void put8_kernel(Put8Args a) {
    typedef Put8Type<DT> T;
    const int lane = threadIdx.x & 63;
    const uint32_t unit = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const bool v = unit & 1;
    const uint32_t run_of = (unit >> 1) / (uint32_t)a.c.heads;
    const int head = (int)((unit >> 1) - run_of * a.c.heads), b = (int)(run_of / (uint32_t)a.runs), run = (int)(run_of - (uint32_t)b * a.runs);
    if (b >= a.seqs) return;
    int first, end;
    if (a.starts) {
        first = min(max(a.starts[b], 0), a.tokens);
        end = min(max(a.starts[b + 1], first), a.tokens);
    } else {
        first = (int)min((int64_t)b * a.most_new, (int64_t)a.tokens);
        end = (int)min((int64_t)first + a.most_new, (int64_t)a.tokens);
    }
    const int64_t len = max(a.lens[b], 0), last = len + min(end - first, a.most_new);
    const int64_t block = len / a.c.size + run, from = max(len, block * a.c.size), to = min(last, (block + 1) * a.c.size);
    if (from >= to) return;
    const int64_t pg = from / a.c.page;
    if (pg >= a.max_pages) return;
    const int32_t id = a.table[b * a.ld_table + pg];
    if ((uint32_t)id >= (uint32_t)a.c.pages) return;
    const Plane8 p = plane_of(a.c, v, head);
    const int off = (int)(from - pg * a.c.page), in_block = off % a.c.size, n = (int)(to - from), per = a.c.dim / 16, pieces = n * per;
    const int64_t t_b = v ? a.v_t : a.k_t;
    const char* in = (v ? a.v + head * a.v_h : a.k + head * a.k_h) + (first + (from - len)) * t_b;
    uint8_t* scale = p.scale + id * p.s_page + off / a.c.size * p.s_block;
    const int was = in_block ? *scale : 0;

    u32x4 x[PUT8_KEEP][2];
    auto load = [&](int j0) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < PUT8_KEEP; ++j)
            if ((j0 + j) * 64 < pieces) {
                const int i = min((j0 + j) * 64 + lane, pieces - 1), t = i / per;
                const u32x4* at = reinterpret_cast<const u32x4*>(in + t * t_b + (i - t * per) * 32);
                x[j][0] = at[0];
                x[j][1] = at[1];
            }
    };
    auto value = [&](int j, int i) __attribute__((always_inline)) { return T::get(x[j][i >> 3][(i & 7) >> 1] >> (16 * (i & 1)) & 0xFFFF); };
    float top = 0.f;
    for (int j0 = 0; j0 * 64 < pieces; j0 += PUT8_KEEP) {
        load(j0);
#pragma unroll
        for (int j = 0; j < PUT8_KEEP; ++j)
            if ((j0 + j) * 64 < pieces)
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const float m = fabsf(value(j, i));
                    top = m < INFINITY ? fmaxf(top, m) : top;
                }
    }
    // (magnitudes order as their bits)
    const uint32_t bits = wave_max(__builtin_bit_cast(uint32_t, fminf(top, T::MOST)));
    int e = (int)(bits >> 23) - 127 - 8 + ((bits & 0x7FFFFF) > 0x600000);
    e = max(max(e, -100), was - 127);
    if (in_block && e > was - 127) scale_slots(p, id, off - in_block, in_block, per, e + 127 - was, lane);
    if (lane == 0) *scale = (uint8_t)(e + 127);
    const float by = two_to(-e);
    for (int j0 = 0; j0 * 64 < pieces; j0 += PUT8_KEEP) {
        if (pieces > PUT8_KEEP * 64) load(j0);
#pragma unroll
        for (int j = 0; j < PUT8_KEEP; ++j)
            if ((j0 + j) * 64 + lane < pieces) {
                const int i = (j0 + j) * 64 + lane, t = i / per;
                u32x4 y;
#pragma unroll
                for (int d = 0; d < 4; ++d) {
                    float f[4];
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const float one = value(j, 4 * d + q);
                        f[q] = fabsf(one) < INFINITY ? fminf(fmaxf(one, -T::MOST), T::MOST) * by : NAN;
                    }
                    y[d] = __builtin_amdgcn_cvt_pk_fp8_f32(f[0], f[1], 0, false);
                    y[d] = __builtin_amdgcn_cvt_pk_fp8_f32(f[2], f[3], y[d], true);
                }
                *reinterpret_cast<u32x4*>(p.at + id * p.page + (off + t) * p.slot + (i - t * per) * 16) = y;
            }
    }
}

// One wave per sequence, layer, head, and keys or values, a block that rows move to at a time.  The path ascends, so row i comes from a slot at or behind lens + i:
// no row is read after its slot was written, and what goes to a block comes from it or from blocks behind it, whose scales have not changed yet.
constexpr int KEEP8_FLY = 4;
__global__ __launch_bounds__(256) void keep8_kernel(Keep8Args a) {
    const int lane = threadIdx.x & 63, b = blockIdx.y;
    const uint32_t unit = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    if (unit >= 2 * (uint32_t)a.layers * a.c.heads) return;
    const uint32_t lk = unit / (uint32_t)a.c.heads, layer = lk >> 1;
    const bool v = lk & 1;
    const int head = (int)(unit - lk * a.c.heads);
    Plane8 p = plane_of(a.c, v, head);
    p.at += (int64_t)layer * (v ? a.v_layer : a.k_layer);
    p.scale += (int64_t)layer * (v ? a.vs_layer : a.ks_layer);
    const int count = min(a.counts[b], a.most), size = a.c.size, page = a.c.page, per = a.c.dim / 16, rows = 64 / per;
    const int64_t len = max(a.lens[b], 0), cap = (int64_t)a.max_pages * page;
    const int32_t *path = a.path + b * a.ld_path, *table = a.table + b * a.ld_table;
    // a lane's path entry: where it comes from and goes to, and the scale there
    struct Entry { int src, src_off, dst, dst_off, scale, ok; };
    auto look = [&](int w) __attribute__((always_inline)) {
        Entry r = {0, 0, 0, 0, 0, 0};
        const int i = w * 64 + lane, x = i < count ? path[i] : -1, before = i < count && i ? path[i - 1] : -1;
        const int64_t s = len + x, d = len + i;
        if (x > max(before, -1) && s < cap && d < cap) {
            const int sp = (int)(s / page), dp = (int)(d / page), src = table[sp], dst = table[dp];
            if ((uint32_t)src < (uint32_t)a.c.pages && (uint32_t)dst < (uint32_t)a.c.pages) {
                const int src_off = (int)(s - (int64_t)sp * page);
                r = {src, src_off, dst, (int)(d - (int64_t)dp * page), p.scale[src * p.s_page + src_off / size * p.s_block], 1};
            }
        }
        return r;
    };
    Entry r = {};
    int window = -1;
    auto at_window = [&](int w) __attribute__((always_inline)) { if (w != window) { r = look(w); window = w; } };
    int m = 0;
    for (int w = 0; w * 64 < count; ++w) {
        at_window(w);
        const uint64_t all = __ballot(r.ok);
        m = all == ~0ull ? (w + 1) * 64 : w * 64 + __builtin_ctzll(~all);
        if (all != ~0ull) break;
    }
    if (m == 0) return;
    for (int64_t block = len / size; block * size < len + m; ++block) {
        const int lo = (int)max((int64_t)0, block * size - len), hi = (int)min((int64_t)m, (block + 1) * size - len), w0 = lo / 64, w1 = (hi - 1) / 64;
        at_window(w0);
        const int to = __builtin_amdgcn_readlane(r.dst, lo & 63), to_off = __builtin_amdgcn_readlane(r.dst_off, lo & 63), in_block = to_off % size;
        uint8_t* to_scale = p.scale + to * p.s_page + to_off / size * p.s_block;
        const int was = in_block ? *to_scale : 0;
        uint32_t e = was;
        for (int w = w0; w <= w1; ++w) {
            at_window(w);
            const int i = w * 64 + lane;
            e = max(e, wave_max(i >= lo && i < hi ? (uint32_t)r.scale : 0u));
        }
        if (in_block && (int)e > was) scale_slots(p, to, to_off - in_block, in_block, per, (int)e - was, lane);
        for (int w = w0; w <= w1; ++w) {
            at_window(w);
            const int end = min(hi, (w + 1) * 64);
            for (int i0 = max(lo, w * 64); i0 < end; i0 += rows * KEEP8_FLY) {
                u32x4 x[KEEP8_FLY];
                int down[KEEP8_FLY];
                char* at[KEEP8_FLY];
                const int row = lane / per, piece = lane - row * per;
#pragma unroll
                for (int j = 0; j < KEEP8_FLY; ++j) {
                    const int i = i0 + j * rows + row, l = min(i, end - 1) & 63;
                    const int from = __shfl(r.src, l), from_off = __shfl(r.src_off, l), goes = __shfl(r.dst, l), goes_off = __shfl(r.dst_off, l);
                    down[j] = (int)e - __shfl(r.scale, l);
                    at[j] = i < end && row < rows ? p.at + goes * p.page + goes_off * p.slot + piece * 16 : nullptr;
                    if (at[j]) x[j] = *reinterpret_cast<const u32x4*>(p.at + from * p.page + from_off * p.slot + piece * 16);
                }
#pragma unroll
                for (int j = 0; j < KEEP8_FLY; ++j)
                    if (at[j]) *reinterpret_cast<u32x4*>(at[j]) = down[j] ? scaled_codes(x[j], down[j]) : x[j];
            }
        }
        if (lane == 0) *to_scale = (uint8_t)e;
    }
}

int check_cache8(const char* who, const sq_cache8* c) {
    if (c->dim < 16 || c->dim > 256 || c->dim % 16) return fail(SQ_EUNSUPPORTED, "%s: heads of %d elements (a multiple of 16 up to 256)", who, c->dim);
    if (c->heads < 0 || c->heads > (1 << 16) || c->pages < 0 || c->page < 1 || (int64_t)c->pages * c->page > INT32_MAX || c->blocks < 1 || c->page % c->blocks)
        return fail(SQ_EINVAL, "%s: %d pages of %d slots in %d blocks, %d heads", who, c->pages, c->page, c->blocks, c->heads);
    if (c->page / c->blocks % 16) return fail(SQ_EUNSUPPORTED, "%s: blocks of %d tokens (a multiple of 16)", who, c->page / c->blocks);
    const int64_t strides = c->k_page | c->k_slot | c->k_head | c->v_page | c->v_slot | c->v_head;
    if (strides % 16 || (((uintptr_t)c->k | (uintptr_t)c->v) & 15)) return fail(SQ_EUNSUPPORTED, "%s: keys and values need 16-byte aligned heads", who);
    if (c->k_slot < 0 || c->v_slot < 0 || c->k_slot >= (1 << 27) || c->v_slot >= (1 << 27))
        return fail(SQ_EUNSUPPORTED, "%s: slots %lld and %lld bytes apart (ascending, less than 2^27)", who, (long long)c->k_slot, (long long)c->v_slot);
    if (c->pages && c->heads && (!c->k || !c->v || !c->k_scale || !c->v_scale)) return fail(SQ_EINVAL, "%s: null cache", who);
    return SQ_OK;
}

static Cache8 cache8_of(const sq_cache8& c) {
    return {(char*)c.k, (char*)c.v, c.k_scale, c.v_scale, c.k_page, c.k_slot, c.k_head, c.v_page, c.v_slot, c.v_head, c.ks_page, c.ks_block, c.ks_head,
            c.vs_page, c.vs_block, c.vs_head, c.pages, c.page, c.blocks, c.page / c.blocks, c.heads, c.dim};
}

}  // namespace sq

using namespace sq;

extern "C" {

int sq_put_tokens8(const sq_heads* k, const sq_heads* v, int32_t tokens, int dtype, const sq_cache8* cache, const int32_t* table, int64_t ld_table, int32_t max_pages,
                   const int32_t* lens, const int32_t* starts, int32_t seqs, int32_t most_new, void* stream) {
    const char* who = "sq_put_tokens8";
    if (!k || !v || !cache) return fail(SQ_EINVAL, "%s: null argument", who);
    if (dtype != SQ_F16 && dtype != SQ_BF16) return fail(SQ_EINVAL, "%s: dtype %d (fp16 or bf16)", who, dtype);
    if (int rc = check_cache8(who, cache)) return rc;
    if (k->heads != cache->heads || v->heads != cache->heads) return fail(SQ_EINVAL, "%s: %d key and %d value heads for %d of the cache", who, k->heads, v->heads, cache->heads);
    if (tokens < 0 || seqs < 0 || most_new < 0 || max_pages < 0 || ld_table < max_pages)
        return fail(SQ_EINVAL, "%s: %d tokens, %d sequences, at most %d new, tables of %d (ld %lld)", who, tokens, seqs, most_new, max_pages, (long long)ld_table);
    if (!starts && (int64_t)seqs * most_new != tokens) return fail(SQ_EINVAL, "%s: %d tokens are not %d for each of %d sequences", who, tokens, most_new, seqs);
    if (!tokens || !seqs || !most_new || !cache->heads) return SQ_OK;
    if (!max_pages || !cache->pages) return fail(SQ_EINVAL, "%s: new tokens without a page", who);
    if (!k->in || !v->in || !table || !lens) return fail(SQ_EINVAL, "%s: null argument", who);
    if ((k->in_token | k->in_head | v->in_token | v->in_head) % 8 || (((uintptr_t)k->in | (uintptr_t)v->in) & 15))
        return fail(SQ_EUNSUPPORTED, "%s: k and v need 16-byte aligned heads", who);
    Put8Args a = {};
    a.c = cache8_of(*cache);
    a.k = (const char*)k->in; a.v = (const char*)v->in;
    a.k_t = k->in_token * 2; a.k_h = k->in_head * 2; a.v_t = v->in_token * 2; a.v_h = v->in_head * 2;
    a.table = table; a.ld_table = ld_table; a.max_pages = max_pages; a.lens = lens; a.starts = starts;
    a.tokens = tokens; a.seqs = seqs; a.most_new = most_new;
    a.runs = (int)(((int64_t)most_new + 2 * a.c.size - 2) / a.c.size);          // the first token may be its block's last
    const int64_t units = 2 * (int64_t)seqs * a.runs * a.c.heads, groups = (units + 3) / 4;
    if (groups > (1 << 23)) return fail(SQ_EUNSUPPORTED, "%s: %d sequences of up to %d new tokens and %d heads at once", who, seqs, most_new, cache->heads);
    if (dtype == SQ_F16) hipLaunchKernelGGL(put8_kernel<SQ_F16>, dim3((unsigned)groups), dim3(256), 0, (hipStream_t)stream, a);
    else hipLaunchKernelGGL(put8_kernel<SQ_BF16>, dim3((unsigned)groups), dim3(256), 0, (hipStream_t)stream, a);
    return check_launch(who);
}

int sq_keep_drafted8(const sq_cache8* cache, int32_t layers, int64_t k_layer, int64_t v_layer, int64_t ks_layer, int64_t vs_layer, const int32_t* table, int64_t ld_table,
                     int32_t max_pages, const int32_t* lens, const int32_t* path, int64_t ld_path, int32_t most, const int32_t* counts, int32_t seqs, void* stream) {
    const char* who = "sq_keep_drafted8";
    if (!cache) return fail(SQ_EINVAL, "%s: null cache", who);
    if (int rc = check_cache8(who, cache)) return rc;
    if (layers < 0 || layers > (1 << 20) || seqs < 0 || seqs > 65535 || most < 0 || max_pages < 0 || ld_table < max_pages || ld_path < most)
        return fail(SQ_EINVAL, "%s: %d layers, %d sequences, paths of %d (ld %lld), tables of %d (ld %lld)", who, layers, seqs, most, (long long)ld_path, max_pages,
                    (long long)ld_table);
    if (!layers || !seqs || !most || !max_pages || !cache->pages || !cache->heads) return SQ_OK;
    if (!table || !lens || !path || !counts) return fail(SQ_EINVAL, "%s: null argument", who);
    if ((k_layer | v_layer) % 16) return fail(SQ_EUNSUPPORTED, "%s: keys and values need 16-byte aligned heads", who);
    Keep8Args a = {};
    a.c = cache8_of(*cache);
    a.k_layer = k_layer; a.v_layer = v_layer; a.ks_layer = ks_layer; a.vs_layer = vs_layer;
    a.table = table; a.ld_table = ld_table; a.max_pages = max_pages; a.lens = lens; a.path = path; a.ld_path = ld_path; a.counts = counts;
    a.layers = layers; a.most = most;
    const int64_t groups = (2 * (int64_t)layers * a.c.heads + 3) / 4;
    if (groups > (1 << 23)) return fail(SQ_EUNSUPPORTED, "%s: %d layers of %d heads", who, layers, cache->heads);
    hipLaunchKernelGGL(keep8_kernel, dim3((unsigned)groups, (unsigned)seqs), dim3(256), 0, (hipStream_t)stream, a);
    return check_launch(who);
}

}  // extern "C"
