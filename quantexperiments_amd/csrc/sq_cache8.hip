// A paged cache of keys and values held in 8 bits: new tokens put into it, and the accepted path of a draft moved behind its cached tokens.
//
// A block of tokens of one head has one scale 2^e, and an element x the code rne_e4m3(x * 2^-e): three bits of mantissa whatever e is, down to 2^-6 of the scale, so a
// scale that is a power of two loses nothing beside the exact a / 448 but, at worst, the last of the bits below that.  It buys that attention multiplies by the scale while it
// unpacks codes, exactly, and that a block whose scale grows with later tokens is scaled to it without another rounding (below 2^-6: with one).
#include <type_traits>
#include "sq_common.h"

namespace sq {

struct Cache8 {
    char *k, *v;
    uint8_t *ks, *vs;
    int64_t k_page, k_slot, k_head, v_page, v_slot, v_head, ks_page, ks_block, ks_head, vs_page, vs_block, vs_head;      // bytes
    int pages, page, blocks, size, heads, dim, per;                // size: tokens of a block; per: 16-byte pieces of a head
    uint32_t over_per;                                              // 2^32 / per, rounded up
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

// over a wave, or over each 16 lanes of it
template <bool WAVE>
__device__ __forceinline__ uint32_t lanes_max(uint32_t v) {
    if constexpr (WAVE) {
        const auto h = __builtin_amdgcn_permlane32_swap(v, v, false, false);
        v = max((uint32_t)h[0], (uint32_t)h[1]);
        const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
        v = max((uint32_t)r[0], (uint32_t)r[1]);
    }
    v = max(v, row_rotated_bits<8>(v));
    v = max(v, row_rotated_bits<4>(v));
    v = max(v, row_rotated_bits<2>(v));
    return max(v, row_rotated_bits<1>(v));
}

// over a wave, of 16-bit halves
__device__ __forceinline__ uint32_t wave_max2(uint32_t x) {
    typedef unsigned short pair __attribute__((ext_vector_type(2)));
    auto most = [](uint32_t a, uint32_t b) { return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(pair, a), __builtin_bit_cast(pair, b))); };
    const auto h = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    x = most((uint32_t)h[0], (uint32_t)h[1]);
    const auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    x = most((uint32_t)r[0], (uint32_t)r[1]);
    x = most(x, row_rotated_bits<8>(x));
    x = most(x, row_rotated_bits<4>(x));
    x = most(x, row_rotated_bits<2>(x));
    return most(x, row_rotated_bits<1>(x));
}

// i / per, for i below 2^28
__device__ __forceinline__ int row_of(const Cache8& c, int i) { return c.per == 1 ? i : (int)__umulhi((uint32_t)i, c.over_per); }

// 16 codes times 2^-down.  (By way of fp16, which has every one of these numbers down to 2^-24, where the nearest code is zero.)
__device__ __forceinline__ u32x4 scaled_codes(u32x4 x, int down) {
    typedef short short2v __attribute__((ext_vector_type(2)));
    const float by = two_to(-down);
    u32x4 y;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const half2v lo = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x[i], by, false), hi = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x[i], by, true);
        y[i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(__builtin_amdgcn_cvt_scalef32_pk_fp8_f16(short2v{0, 0}, lo, 1.f, false), hi, 1.f, true));
    }
    return y;
}

// Scales n slots from `first` on down, U pieces of 16 elements per lane of G in flight
template <int G, int U>
__device__ __forceinline__ void scale_slots(const Cache8& c, char* first, int64_t slot, int n, int down, int lane) {
    const int pieces = n * c.per;
    for (int x = lane; x < pieces; x += G * U) {
        u32x4 y[U];
        auto at = [&](int u) __attribute__((always_inline)) {
            const int i = min(x + u * G, pieces - 1), row = row_of(c, i);
            return reinterpret_cast<u32x4*>(first + row * slot + (i - row * c.per) * 16);
        };
#pragma unroll
        for (int u = 0; u < U; ++u) y[u] = *at(u);
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (x + u * G < pieces) *at(u) = scaled_codes(y[u], down);
    }
}

constexpr int PUT8_PIECES = 8;
// MOST: the largest magnitude that is held, 1.875 * 2^15 and 1.875 * 2^127
template <int DT> struct Put8Type;
template <> struct Put8Type<SQ_F16> {
    static constexpr uint32_t MOST = 0x7B80;
    typedef half2v two;
    static __device__ __forceinline__ float get(uint32_t b) { return h2f((uint16_t)b); }
    template <bool HI, typename V> static __device__ __forceinline__ V codes(V old, uint32_t x, float scale) { return __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(old, __builtin_bit_cast(two, x), scale, HI); }
};
template <> struct Put8Type<SQ_BF16> {
    static constexpr uint32_t MOST = 0x7F70;
    typedef __bf16 two __attribute__((ext_vector_type(2)));
    static __device__ __forceinline__ float get(uint32_t b) { return bf2f((uint16_t)b); }
    template <bool HI, typename V> static __device__ __forceinline__ V codes(V old, uint32_t x, float scale) { return __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(old, __builtin_bit_cast(two, x), scale, HI); }
};

// One wave per block that gets new tokens, head, and keys or values: the largest magnitude over its tokens, then the codes.  Magnitudes order as their bits, so the largest is
// looked for two elements at a time, and v_cvt_scalef32_pk_fp8 makes two codes of the elements as they are (one by one, as where some element is beyond what is
// held, 8000 tokens of 8 heads of 128 take 3 us more).  Up to 8 pieces of 16 elements a lane stay in registers between the two: 64 tokens of 128 a wave.  LANES: four waves share
// a block of more than that (8000 tokens of 4 heads of 256 in blocks of 64: read twice by one wave 6 us more); of more than four hold, the elements are read again.  One of
// up to 16 pieces, a decode batch's single token, has 16 lanes: 1024 sequences x 8 heads of 128 4.7 us, with a
// wave each 12.8; 64 x 4 heads 3.4 and 3.8.
// Bound by HBM: 8000 tokens of 8 heads of 128, 49 MB, 11.0 us (4.5 TB/s; 7.1 where they still are in the caches in front of it); a token of each of 64 sequences 3.4, a launch and one chain of loads.
constexpr int64_t PUT8_CACHED = 4 << 20;         // bytes of codes up to which heads that share lines of 128 bytes are put together in the caches; others are written past them (2000 tokens of
                                                 // 8 heads of 128 7.0 us, so 5.5; heads of 16 4.1, so 4.4)
template <int DT, int LANES, bool PASSING>
__global__ __launch_bounds__(256) void put8_kernel(Put8Args a) {
    typedef Put8Type<DT> T;
    constexpr int G = LANES, WAVES = LANES > 64 ? LANES / 64 : 1, PUT8_KEEP = LANES < 64 ? 1 : PUT8_PIECES;
    const int lane = threadIdx.x % G, mine = threadIdx.x / G;
    const uint32_t unit = blockIdx.x * (256 / G) + (G == 64 ? __builtin_amdgcn_readfirstlane(mine) : mine);
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
    const uint32_t size = a.c.size, page = a.c.page, cached = max(a.lens[b], 0);          // (64-bit divisions would be most of a small call's instructions)
    const int64_t len = cached, last = len + min(end - first, a.most_new);
    const int64_t block = (int64_t)(cached / size) + run, from = max(len, block * size), to = min(last, (block + 1) * size);
    if (from >= to) return;
    const int n = (int)(to - from), per = a.c.per, pieces = n * per;
    const int64_t t_b = v ? a.v_t : a.k_t;
    const char* in = (v ? a.v + head * a.v_h : a.k + head * a.k_h) + (first + (from - len)) * t_b;
    u32x4 x[PUT8_KEEP][2];
    auto load = [&](int j0) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < PUT8_KEEP; ++j)
            if ((j0 + j) * G < pieces) {
                const int i = min((j0 + j) * G + lane, pieces - 1), t = row_of(a.c, i);
                const u32x4* at = reinterpret_cast<const u32x4*>(in + t * t_b + (i - t * per) * 32);
                x[j][0] = at[0];
                x[j][1] = at[1];
            }
    };
    load(0);                                                 // (beside the page and the scale, not behind them)
    const uint32_t pg = (uint32_t)from / page;
    if (pg >= (uint32_t)a.max_pages) return;
    const int32_t id = a.table[b * a.ld_table + pg];
    if ((uint32_t)id >= (uint32_t)a.c.pages) return;
    const Plane8 p = plane_of(a.c, v, head);
    const int off = (int)((uint32_t)from - pg * page), in_block = (int)((uint32_t)off % size);
    uint8_t* scale = p.scale + id * p.s_page + (int)((uint32_t)off / size) * p.s_block;
    const int was = in_block ? *scale : 0;
    // One wave has all of its pieces; four go over them again
    const bool again = WAVES > 1 && pieces > PUT8_KEEP * G;
    const int rounds = WAVES > 1 ? (pieces + PUT8_KEEP * G - 1) / (PUT8_KEEP * G) : 1;
    typedef unsigned short pair __attribute__((ext_vector_type(2)));
    pair both = {0, 0};
    for (int q = 0; q < rounds; ++q) {
        const int j0 = q * PUT8_KEEP;
        if (q) load(j0);
#pragma unroll
        for (int j = 0; j < PUT8_KEEP; ++j)
            if ((j0 + j) * G < pieces)
#pragma unroll
                for (int i = 0; i < 8; ++i) both = __builtin_elementwise_max(both, __builtin_bit_cast(pair, x[j][i >> 2][i & 3] & 0x7FFF7FFFu));
    }
    __shared__ uint32_t tops[2][WAVES];
    auto most_of = [&](uint32_t v, int which) __attribute__((always_inline)) {
        v = lanes_max<(LANES >= 64)>(v);
        if constexpr (WAVES > 1) {
            if (lane % 64 == 0) tops[which][lane / 64] = v;
            __syncthreads();                                 // (which all waves pass behind having read the block's scale)
#pragma unroll
            for (int w = 0; w < WAVES; ++w) v = max(v, tops[which][w]);
        }
        return v;
    };
    uint32_t top = most_of(max((uint32_t)both[0], (uint32_t)both[1]), 0);
    const bool plain = top <= T::MOST;
    if (!plain) {                                            // the largest that is finite, or MOST
        top = 0;
        for (int q = 0; q < rounds; ++q) {
            const int j0 = q * PUT8_KEEP;
            if (again) load(j0);
#pragma unroll
            for (int j = 0; j < PUT8_KEEP; ++j)
                if ((j0 + j) * G < pieces)
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const uint32_t m = x[j][i >> 3][(i & 7) >> 1] >> (16 * (i & 1)) & 0x7FFF;
                        if (fabsf(T::get(m)) < INFINITY) top = max(top, m);
                    }
        }
        top = most_of(min(top, T::MOST), 1);
    }
    const uint32_t bits = __builtin_bit_cast(uint32_t, T::get(top));
    int e = (int)(bits >> 23) - 127 - 8 + ((bits & 0x7FFFFF) > 0x600000);
    e = max(max(e, -100), was - 127);
    if (in_block && e > was - 127) scale_slots<G, G == 16 ? 4 : G == 64 ? 2 : 1>(a.c, p.at + id * p.page + (off - in_block) * p.slot, p.slot, in_block, e + 127 - was, lane);
    if (lane == 0) *scale = (uint8_t)(e + 127);
    const float by = two_to(-e), unit_of = two_to(e), most = T::get(T::MOST);
    for (int q = 0; q < rounds; ++q) {
        const int j0 = q * PUT8_KEEP;
        if (again) load(j0);
#pragma unroll
        for (int j = 0; j < PUT8_KEEP; ++j)
            if ((j0 + j) * G + lane < pieces) {
                const int i = (j0 + j) * G + lane, t = row_of(a.c, i);
                u32x4 y;
#pragma unroll
                for (int d = 0; d < 4; ++d) {
                    const uint32_t lo = x[j][d >> 1][2 * (d & 1)], hi = x[j][d >> 1][2 * (d & 1) + 1];
                    if (plain) {
                        typedef short short2v __attribute__((ext_vector_type(2)));
                        y[d] = __builtin_bit_cast(uint32_t, T::template codes<true>(T::template codes<false>(short2v{0, 0}, lo, unit_of), hi, unit_of));
                        continue;
                    }
                    float f[4];
#pragma unroll
                    for (int z = 0; z < 4; ++z) {
                        const float one = T::get((z & 2 ? hi : lo) >> (16 * (z & 1)) & 0xFFFF);
                        f[z] = fabsf(one) < INFINITY ? fminf(fmaxf(one, -most), most) * by : NAN;
                    }
                    y[d] = __builtin_amdgcn_cvt_pk_fp8_f32(f[0], f[1], 0, false);
                    y[d] = __builtin_amdgcn_cvt_pk_fp8_f32(f[2], f[3], y[d], true);
                }
                u32x4* to = reinterpret_cast<u32x4*>(p.at + id * p.page + (off + t) * p.slot + (i - t * per) * 16);
                if constexpr (PASSING) __builtin_nontemporal_store(y, to); else *to = y;
            }
    }
}

// One wave per sequence and U units (heads of a layer's keys or values), a block that rows move to at a time.  The path ascends, so row i comes from a slot at or
// behind lens + i: no row is read after its slot was written, and what goes to a block comes from it or from blocks behind it, whose scales have not changed yet.
// The path and the pages are looked up once for the units; then the scales and the first rows of all of them are in flight together, whatever blocks they go to, and further rows are
// fetched as they come.  Bound by that chain of loads (lengths, path, pages, rows) and by what is worked out along it: 64 sequences, 28 layers of 4 heads, 8 rows of 128, 10.9 us for 21 MB
// read and 20 written (what blocks that grow cost is in that), with a wave per unit 17.5; 256 sequences 30 and 52; one sequence 4.2.
template <int U>
__global__ __launch_bounds__(256) void keep8_kernel(Keep8Args a) {
    const int lane = threadIdx.x & 63, b = blockIdx.y;
    const bool v = blockIdx.z;
    const uint32_t units = (uint32_t)a.layers * a.c.heads, first = (blockIdx.x * 4 + __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6))) * U;
    if (first >= units) return;
    const Plane8 p = plane_of(a.c, v, 0);
    char* at[U];
    uint8_t* scale_at[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {                            // (units behind the last one: the last one again, not written)
        const uint32_t unit = min(first + u, units - 1), layer = unit / (uint32_t)a.c.heads;
        const int64_t head = unit - layer * a.c.heads;
        at[u] = p.at + layer * (v ? a.v_layer : a.k_layer) + head * (v ? a.c.v_head : a.c.k_head);
        scale_at[u] = p.scale + layer * (v ? a.vs_layer : a.ks_layer) + head * (v ? a.c.vs_head : a.c.ks_head);
    }
    const int count = min(a.counts[b], a.most), per = a.c.per, rows = 64 / per, entries = 64 / rows * rows;         // rows of a wave's load, path entries looked up at once
    const int64_t len = max(a.lens[b], 0), cap = (int64_t)a.max_pages * a.c.page;
    const uint32_t size = a.c.size, page = a.c.page;
    const int32_t *path = a.path + b * a.ld_path, *table = a.table + b * a.ld_table;
    // a lane's path entry: where it comes from and goes to (bytes of a unit), its target's block, and the units' scales where it comes from
    struct Entry { int64_t src, dst, block; int ok; };
    Entry r;
    uint32_t scale[U];
    int window = -1;
    auto at_window = [&](int w) __attribute__((always_inline)) {
        if (w == window) return;
        window = w;
        r = {0, 0, 0, 0};
        const int i = w * entries + lane, x = lane < entries && i < count ? path[i] : -1, before = x >= 0 && i ? path[i - 1] : -1;
        const int64_t s = len + x, d = len + i;
        int64_t from = 0;
        if (x > max(before, -1) && s < cap && d < cap) {
            const uint32_t sp = (uint32_t)s / page, dp = (uint32_t)d / page, so = (uint32_t)s - sp * page, to = (uint32_t)d - dp * page;
            const int src = table[sp], dst = table[dp];
            if ((uint32_t)src < (uint32_t)a.c.pages && (uint32_t)dst < (uint32_t)a.c.pages) {
                r = {src * p.page + so * p.slot, dst * p.page + to * p.slot, dst * p.s_page + to / size * p.s_block, 1};
                from = src * p.s_page + so / size * p.s_block;
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) scale[u] = scale_at[u][from];
    };
    auto of_lane = [](int64_t x, int l) __attribute__((always_inline)) {
        return (int64_t)(uint32_t)__builtin_amdgcn_readlane((int)x, l) | (int64_t)__builtin_amdgcn_readlane((int)(x >> 32), l) << 32;
    };
    // a load's rows: from rows * chunk on
    const int row = min(row_of(a.c, lane), rows - 1), piece = lane - row * per;
    const bool whole = piece < per;                          // (a last lane may have no row)
    u32x4 x[U];
    int chunk = -1;
    auto fetch = [&](int c) __attribute__((always_inline)) {
        if (c == chunk) return;
        chunk = c;
        const int64_t src = __shfl(r.src, (c * rows + row) % entries) + min(piece, per - 1) * 16;
#pragma unroll
        for (int u = 0; u < U; ++u) x[u] = *reinterpret_cast<const u32x4*>(at[u] + src);
    };
    at_window(0);
    fetch(0);
    uint32_t was[U];                                         // the scales of the block that the first row goes to
    const int64_t block0 = of_lane(r.block, 0);
#pragma unroll
    for (int u = 0; u < U; ++u) was[u] = scale_at[u][block0];
    int m = 0;
    for (int w = 0; w * entries < count; ++w) {
        at_window(w);
        const uint64_t all = __ballot(r.ok) | (entries < 64 ? ~0ull << entries : 0);
        m = w * entries + (all == ~0ull ? entries : __builtin_ctzll(~all));
        if (all != ~0ull) break;
    }
    const int in_first = (int)(len % size);                  // cached tokens in that block
    for (int lo = 0, hi; lo < m; lo = hi) {
        const int held = lo ? 0 : in_first, w0 = lo / entries;
        hi = min(m, lo + (int)size - held);
        const int w1 = (hi - 1) / entries;
        at_window(w0);
        const int64_t to = of_lane(r.dst, lo - w0 * entries), block = of_lane(r.block, lo - w0 * entries);
        uint32_t e[U];
#pragma unroll
        for (int u = 0; u < U; ++u) e[u] = 0;
        for (int w = w0; w <= w1; ++w) {
            at_window(w);
            const int i = w * entries + lane;
            const bool mine = lane < entries && i >= lo && i < hi;
#pragma unroll
            for (int u = 0; u < U; u += 2) {                 // (two units' at a time)
                const uint32_t two = mine ? scale[u] | (u + 1 < U ? scale[min(u + 1, U - 1)] << 16 : 0u) : 0u, most = wave_max2(two);
                e[u] = max(e[u], most & 0xFFFF);
                if (u + 1 < U) e[min(u + 1, U - 1)] = max(e[min(u + 1, U - 1)], most >> 16);
            }
        }
        if (held) {                                          // scaled to it, the units' pieces in flight together
            int down[U];
            bool any = false;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                down[u] = first + u < units ? (int)e[u] - (int)was[u] : 0;
                e[u] = max(e[u], was[u]);
                any |= down[u] > 0;
            }
            if (any)
                for (int i = lane; i < held * per; i += 64) {
                    u32x4 y[U];
                    const int slot = row_of(a.c, i);
                    const int64_t where = to + (slot - held) * p.slot + (i - slot * per) * 16;
#pragma unroll
                    for (int u = 0; u < U; ++u)
                        if (down[u] > 0) y[u] = *reinterpret_cast<const u32x4*>(at[u] + where);
#pragma unroll
                    for (int u = 0; u < U; ++u)
                        if (down[u] > 0) *reinterpret_cast<u32x4*>(at[u] + where) = scaled_codes(y[u], down[u]);
                }
        }
        for (int c = lo / rows; c * rows < hi; ++c) {
            at_window(c * rows / entries);
            fetch(c);
            const int i = c * rows + row, l = i % entries;
            const int64_t dst = __shfl(r.dst, l) + piece * 16;
            const bool mine = whole && i >= lo && i < hi;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int down = (int)e[u] - __shfl((int)scale[u], l);
                if (mine && first + u < units) *reinterpret_cast<u32x4*>(at[u] + dst) = down ? scaled_codes(x[u], down) : x[u];
            }
        }
        if (lane == 0)
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (first + u < units) scale_at[u][block] = (uint8_t)e[u];
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
            c.vs_page, c.vs_block, c.vs_head, c.pages, c.page, c.blocks, c.page / c.blocks, c.heads, c.dim, c.dim / 16, (uint32_t)(((1ull << 32) + c.dim / 16 - 1) / (c.dim / 16))};
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
    const int64_t pieces = (int64_t)(a.c.size < most_new ? a.c.size : most_new) * a.c.per;
    const int lanes = pieces > PUT8_PIECES * 64 ? 256 : pieces > 16 ? 64 : 16;
    const int64_t units = 2 * (int64_t)seqs * a.runs * a.c.heads, groups = (units + 256 / lanes - 1) / (256 / lanes);
    if (groups > (1 << 23)) return fail(SQ_EUNSUPPORTED, "%s: %d sequences of up to %d new tokens and %d heads at once", who, seqs, most_new, cache->heads);
    auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3((unsigned)groups), dim3(256), 0, (hipStream_t)stream, a); };
    auto of = [&](auto dt) {
        constexpr int DT = decltype(dt)::value;
        if (a.c.dim % 128 == 0 || (int64_t)tokens * a.c.heads * a.c.dim * 2 > PUT8_CACHED) go(lanes == 256 ? put8_kernel<DT, 256, true> : lanes == 64 ? put8_kernel<DT, 64, true> : put8_kernel<DT, 16, true>);
        else go(lanes == 256 ? put8_kernel<DT, 256, false> : lanes == 64 ? put8_kernel<DT, 64, false> : put8_kernel<DT, 16, false>);
    };
    if (dtype == SQ_F16) of(std::integral_constant<int, SQ_F16>()); else of(std::integral_constant<int, SQ_BF16>());
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
    // (few units: a wave each, more of them at once)
    const int64_t units = (int64_t)layers * a.c.heads;
    const int each = 2 * units * seqs > 16 * device_cus() ? 4 : 1;
    const int64_t groups = (units + 4 * each - 1) / (4 * each);
    if (groups > (1 << 23)) return fail(SQ_EUNSUPPORTED, "%s: %d layers of %d heads", who, layers, cache->heads);
    const dim3 grid((unsigned)groups, (unsigned)seqs, 2);
    if (each == 4) hipLaunchKernelGGL(keep8_kernel<4>, grid, dim3(256), 0, (hipStream_t)stream, a);
    else hipLaunchKernelGGL(keep8_kernel<1>, grid, dim3(256), 0, (hipStream_t)stream, a);
    return check_launch(who);
}

}  // extern "C"
