// What happens to the heads of a q|k|v product before attention: RMS norm of each query and key head, rotation by the token's
// position, keys and values put in their slots of a paged cache; and the slots of an accepted draft moved behind the cache.
//
// Rotation of pair i of a token at position p, with frequency f_i (64 bit, radians per position):
//     a' = s (a cos(p f_i) - b sin(p f_i)),   b' = s (b cos(p f_i) + a sin(p f_i))
// The angle is worked out in 64 bits and reduced to an eighth of a turn there, so that far positions are as exact as near ones and
// no table of cosines has to be kept or read (a table row would be a fifth of what a token of 28 + 4 heads reads, and one position
// more than the table has an error); sine and cosine of what is left are their Taylor sums in 32 bits.
#include <type_traits>
#include "sq_common.h"

namespace sq {

constexpr int HEADS_MAX_THREADS = 512;

struct HeadsPart {
    const void* in;
    void* out;                          // NULL: not written
    const void* w;                      // norm weights, NULL: no norm
    void* cache;                        // NULL: not written there
    int64_t in_t, in_h, out_t, out_h, c_page, c_slot, c_head;
    int heads, turn;
};

struct HeadsArgs {
    HeadsPart p[3];
    const double* freqs;
    const void* positions;
    const void* slots;
    float scale, eps, w_offset, sign, inv_dim;
    int tokens, dim, pairs, interleaved, w_dtype, wide_positions, wide_slots, pages, page, lanes_log2, heads;
};

__device__ __forceinline__ int64_t load_index(const void* p, int wide, int64_t i) {
    return wide ? reinterpret_cast<const int64_t*>(p)[i] : (int64_t)reinterpret_cast<const int32_t*>(p)[i];
}

// scale * (cos, sign * sin) of position p times f.  q quarter turns are taken off in 64 bits; |r| <= pi / 4 is left, for which the sums to
// r^10 and r^9 are off by less than 4e-10 and 2e-9 relative to one, half a step of 32 bits being 6e-8.
__device__ __forceinline__ float2v angle_of(int64_t p, double f, float scale, float sign) {
    const double turns4 = (double)p * f * 0.63661977236758134308;          // 2 / pi
    const double q = __builtin_rint(turns4);
    const float r = (float)((turns4 - q) * 1.57079632679489661923), z = r * r;
    float s = __builtin_fmaf(z, 2.7557319e-6f, -1.9841270e-4f);
    s = __builtin_fmaf(z, s, 8.3333333e-3f);
    s = __builtin_fmaf(z, s, -1.6666667e-1f);
    s = __builtin_fmaf(z * r, s, r);
    float c = __builtin_fmaf(z, -2.7557319e-7f, 2.4801587e-5f);
    c = __builtin_fmaf(z, c, -1.3888889e-3f);
    c = __builtin_fmaf(z, c, 4.1666667e-2f);
    c = __builtin_fmaf(z, c, -0.5f);
    c = __builtin_fmaf(z, c, 1.f);
    const int k = (int)(q - 4.0 * __builtin_floor(q * 0.25));              // 0 .. 3
    const float cc = k & 1 ? s : c, ss = k & 1 ? c : s;
    return float2v{scale * (k == 1 || k == 2 ? -cc : cc), scale * sign * (k & 2 ? -ss : ss)};
}

// (chosen by selects: indexed by a lane's part the arguments would be fetched from memory)
__device__ __forceinline__ HeadsPart part_of(const HeadsArgs& a, int& h) {
    HeadsPart r = a.p[0];
    const int h1 = h - a.p[0].heads, h2 = h1 - a.p[1].heads;
    auto pick = [](HeadsPart& to, const HeadsPart& from, bool yes) {
        to.in = yes ? from.in : to.in; to.out = yes ? from.out : to.out; to.w = yes ? from.w : to.w; to.cache = yes ? from.cache : to.cache;
        to.in_t = yes ? from.in_t : to.in_t; to.in_h = yes ? from.in_h : to.in_h; to.out_t = yes ? from.out_t : to.out_t; to.out_h = yes ? from.out_h : to.out_h;
        to.c_page = yes ? from.c_page : to.c_page; to.c_slot = yes ? from.c_slot : to.c_slot; to.c_head = yes ? from.c_head : to.c_head;
        to.turn = yes ? from.turn : to.turn;
    };
    pick(r, a.p[1], h1 >= 0);
    pick(r, a.p[2], h1 >= 0 && h2 >= 0);
    h = h1 < 0 ? h : h2 < 0 ? h1 : h2;
    return r;
}

template <int DT> struct Chunk { u32x4 v; };                               // 8 elements
template <> struct Chunk<SQ_F32> { float4v v[2]; };

template <int DT> __device__ __forceinline__ void load8(Chunk<DT>& c, const void* p, int64_t i) {
    if constexpr (DT == SQ_F32) {
        c.v[0] = reinterpret_cast<const float4v*>(reinterpret_cast<const float*>(p) + i)[0];
        c.v[1] = reinterpret_cast<const float4v*>(reinterpret_cast<const float*>(p) + i)[1];
    } else {
        c.v = *reinterpret_cast<const u32x4*>(reinterpret_cast<const uint16_t*>(p) + i);
    }
}
template <int DT> __device__ __forceinline__ void store8(const Chunk<DT>& c, void* p, int64_t i) {
    if constexpr (DT == SQ_F32) {
        reinterpret_cast<float4v*>(reinterpret_cast<float*>(p) + i)[0] = c.v[0];
        reinterpret_cast<float4v*>(reinterpret_cast<float*>(p) + i)[1] = c.v[1];
    } else {
        *reinterpret_cast<u32x4*>(reinterpret_cast<uint16_t*>(p) + i) = c.v;
    }
}
template <int DT> __device__ __forceinline__ void widen(const Chunk<DT>& c, float* v) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        if constexpr (DT == SQ_F32) v[e] = c.v[e >> 2][e & 3];
        else if constexpr (DT == SQ_F16) v[e] = h2f((uint16_t)(c.v[e >> 1] >> (16 * (e & 1))));
        else v[e] = bf2f((uint16_t)(c.v[e >> 1] >> (16 * (e & 1))));
    }
}
template <int DT> __device__ __forceinline__ void narrow(Chunk<DT>& c, const float* v) {
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
        if constexpr (DT == SQ_F32) c.v[e >> 2][e & 3] = v[e], c.v[e >> 2][(e & 3) + 1] = v[e + 1];
        else if constexpr (DT == SQ_F16) c.v[e >> 1] = f2h_x2(v[e], v[e + 1]);
        else c.v[e >> 1] = f2bf_x2(v[e], v[e + 1]);
    }
}
// Sum over groups of 2^log2n neighbouring lanes, the same in all of them
__device__ __forceinline__ float lanes_sum(float v, int log2n) {        // (of lanes that all are active)
    auto other = [](float x, auto ctrl) {
        const int b = __builtin_bit_cast(int, x);
        return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(b, b, decltype(ctrl)::value, 0xF, 0xF, false));
    };
    if (log2n > 0) v += other(v, std::integral_constant<int, 0xB1>());          // lane ^ 1
    if (log2n > 1) v += other(v, std::integral_constant<int, 0x4E>());          // lane ^ 2
    if (log2n > 2) v += other(v, std::integral_constant<int, 0x141>());         // the half row backwards: its other quad
    if (log2n > 3) v += other(v, std::integral_constant<int, 0x140>());         // the row backwards: its other half
    if (log2n > 4) {
        const uint32_t a = __builtin_bit_cast(uint32_t, v);
        const auto h = __builtin_amdgcn_permlane16_swap(a, a, false, false);
        v = __builtin_bit_cast(float, (uint32_t)h[0]) + __builtin_bit_cast(float, (uint32_t)h[1]);
    }
    return v;
}

// One workgroup per token (and part of its heads, blockIdx.y).  A thread takes 16 elements of a head, whichever the layout: the 8 pairs
// whose angles are 8c .. 8c + 7, or 16 neighbours behind the rotated part, so that a head is dim / 16 lanes (rounded up to a power
// of two for the sum of its squares) with two 16-byte loads each, in flight while the token's angles are worked out, once for all heads.
// WT: the type of the norm weights, or none; they are fetched with the elements (behind the sum of squares they cost 2048 tokens of 28 + 4 + 4 heads of
// 128 another 4 us), and layout and type are chosen at compile time (chosen here they take a fifth of the waves' registers and more than that was worth).
// Bound by HBM from about 1000 tokens on (norm, rotation and cache slots of 8192 tokens of 28 + 4 + 4 heads of 128 37 us, 151 MB, 4.1 TB/s; rotation of 32 heads of 2048
// tokens 7.3 us, 4.6 TB/s), by its chain of loads, angles, sum and stores below (8 tokens 3.9 us).
constexpr int NO_NORM = -1;
template <int DT, int WT, bool INTERLEAVED>
__global__ __launch_bounds__(HEADS_MAX_THREADS) void heads_kernel(HeadsArgs a) {
    extern __shared__ __attribute__((aligned(16))) float2v angles[];
    constexpr bool NORM = WT != NO_NORM;
    constexpr int WD = NORM ? WT : DT;
    const int tid = threadIdx.x, lanes = 1 << a.lanes_log2, items = a.heads << a.lanes_log2, c = tid & (lanes - 1);
    const bool live = c < a.dim / 16, turned = c < a.pairs / 8;
    const int e0 = turned && !INTERLEAVED ? 8 * c : 16 * c, e1 = turned && !INTERLEAVED ? a.pairs + 8 * c : 16 * c + 8;
    for (int n = blockIdx.x; n < a.tokens; n += gridDim.x) {
        const int64_t pos = a.pairs ? load_index(a.positions, a.wide_positions, n) : 0;
        int64_t slot = -1;
        if (a.slots) slot = load_index(a.slots, a.wide_slots, n);
        const double f = tid < a.pairs ? a.freqs[tid] : 0.0;
        bool first = true;
        for (int item = blockIdx.y * blockDim.x + tid; first || item < items; item += gridDim.y * blockDim.x) {
            int h = item >> a.lanes_log2;
            const HeadsPart p = part_of(a, h);
            const bool mine = live && item < items, normed = NORM && mine && p.w;
            Chunk<DT> x0, x1;
            Chunk<WD> w0, w1;
            if (mine) {
                load8(x0, p.in, n * p.in_t + h * p.in_h + e0);
                load8(x1, p.in, n * p.in_t + h * p.in_h + e1);
            }
            if (NORM && normed) {
                load8(w0, p.w, e0);
                load8(w1, p.w, e1);
            }
            if (first) {
                if (tid < a.pairs) angles[tid] = angle_of(pos, f, a.scale, a.sign);
                for (int i = tid + blockDim.x; i < a.pairs; i += blockDim.x) angles[i] = angle_of(pos, a.freqs[i], a.scale, a.sign);
                __syncthreads();
                first = false;
            }
            float v[16], rstd = 0.f;
            if (mine) {
                widen(x0, v);
                widen(x1, v + 8);
            }
            if (NORM) {                                   // (by all lanes: those behind a narrow head's elements add zeros)
                float ss = 0.f;
                if (mine)
#pragma unroll
                    for (int e = 0; e < 16; ++e) ss = __builtin_fmaf(v[e], v[e], ss);
                rstd = rsqrtf(lanes_sum(ss, a.lanes_log2) * a.inv_dim + a.eps);
            }
            if (!mine) continue;
            if (NORM && normed) {
                float w[16];
                widen(w0, w);
                widen(w1, w + 8);
#pragma unroll
                for (int e = 0; e < 16; ++e) v[e] = v[e] * rstd * (w[e] + a.w_offset);
            }
            if (p.turn && turned) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float2v t = angles[8 * c + i];
                    float &x = v[INTERLEAVED ? 2 * i : i], &y = v[INTERLEAVED ? 2 * i + 1 : i + 8];
                    const float xx = __builtin_fmaf(x, t[0], -y * t[1]), yy = __builtin_fmaf(y, t[0], x * t[1]);
                    x = xx;
                    y = yy;
                }
            }
            if ((NORM && normed) || (p.turn && turned)) {    // (else the bits as they are: NaN payloads, signs)
                narrow(x0, v);
                narrow(x1, v + 8);
            }
            if (p.out) {
                store8(x0, p.out, n * p.out_t + h * p.out_h + e0);
                store8(x1, p.out, n * p.out_t + h * p.out_h + e1);
            }
            if (p.cache && slot >= 0 && slot < (int64_t)a.pages * a.page) {
                const uint32_t pg = (uint32_t)slot / (uint32_t)a.page, off = (uint32_t)slot - pg * (uint32_t)a.page;
                const int64_t at = (int64_t)pg * p.c_page + (int64_t)off * p.c_slot + h * p.c_head;
                store8(x0, p.cache, at + e0);
                store8(x1, p.cache, at + e1);
            }
        }
        if (n + (int64_t)gridDim.x < a.tokens) __syncthreads();             // the angles have been read
    }
}

template <int DT> __device__ __forceinline__ float load_one(const void* p, int64_t i) {
    if constexpr (DT == SQ_F32) return reinterpret_cast<const float*>(p)[i];
    else return load16(p, DT, i);
}
__device__ __forceinline__ float load_any(const void* p, int dtype, int64_t i) {
    return dtype == SQ_F32 ? reinterpret_cast<const float*>(p)[i] : load16(p, dtype, i);
}
template <int DT> __device__ __forceinline__ void store_one(void* p, int64_t i, float v) {
    reinterpret_cast<typename store_as<DT>::type*>(p)[i] = store_as<DT>::cvt(v);
}

// Any width, part, stride and alignment: a wave per head, a lane per pair.  (Where 16-byte pieces fit, heads_kernel takes as long for up to 64 tokens of 32 heads
// of 128 and is two to five times as fast for more: 2048 tokens 11.1 against 40.5 us with norms, 7.7 against 32.1 without.  Bound by the angles, in 64 bits for each head again, and by
// single elements, read twice where there is a norm.)
template <int DT>
__global__ __launch_bounds__(256) void heads_any_kernel(HeadsArgs a) {
    const int lane = threadIdx.x & 63;
    const int64_t total = (int64_t)a.tokens * a.heads;
    for (int64_t i = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); i < total; i += (int64_t)gridDim.x * 4) {
        const int n = (int)(i / a.heads);
        int h = (int)(i % a.heads);
        const HeadsPart p = part_of(a, h);
        const int64_t from = n * p.in_t + h * p.in_h, to = n * p.out_t + h * p.out_h;
        int64_t at = -1;
        if (p.cache) {
            const int64_t slot = load_index(a.slots, a.wide_slots, n);
            if (slot >= 0 && slot < (int64_t)a.pages * a.page) {
                const uint32_t pg = (uint32_t)slot / (uint32_t)a.page, off = (uint32_t)slot - pg * (uint32_t)a.page;
                at = (int64_t)pg * p.c_page + (int64_t)off * p.c_slot + h * p.c_head;
            }
        }
        float rstd = 1.f;
        if (p.w) {
            float ss = 0.f;
            for (int e = lane; e < a.dim; e += 64) { const float v = load_one<DT>(p.in, from + e); ss = __builtin_fmaf(v, v, ss); }
            rstd = rsqrtf(wave_sum(ss) * a.inv_dim + a.eps);
        }
        auto normed = [&](int e) {
            const float v = load_one<DT>(p.in, from + e);
            return p.w ? v * rstd * (load_any(p.w, a.w_dtype, e) + a.w_offset) : v;
        };
        auto put = [&](int e, float v) {
            if (p.out) store_one<DT>(p.out, to + e, v);
            if (at >= 0) store_one<DT>(p.cache, at + e, v);
        };
        const int pairs = p.turn ? a.pairs : 0;
        if (pairs) {
            const int64_t pos = load_index(a.positions, a.wide_positions, n);
            for (int k = lane; k < pairs; k += 64) {
                const float2v t = angle_of(pos, a.freqs[k], a.scale, a.sign);
                const int ea = a.interleaved ? 2 * k : k, eb = a.interleaved ? 2 * k + 1 : k + pairs;
                const float x = normed(ea), y = normed(eb);
                put(ea, __builtin_fmaf(x, t[0], -y * t[1]));
                put(eb, __builtin_fmaf(y, t[0], x * t[1]));
            }
        }
        for (int e = 2 * pairs + lane; e < a.dim; e += 64) put(e, normed(e));
    }
}

static bool wide_ok(const HeadsArgs& a, int dtype) {
    const int unit = dtype == SQ_F32 ? 4 : 8;                               // elements of 16 bytes
    if (a.dim % 16 || a.dim > 512 || a.pairs % 8) return false;
    if ((a.p[0].w || a.p[1].w) && a.w_dtype != dtype && a.w_dtype != SQ_F32) return false;
    uintptr_t at = 0;
    int64_t strides = 0;
    for (const HeadsPart& p : a.p) {
        if (!p.heads) continue;
        at |= (uintptr_t)p.in | (uintptr_t)p.out | (uintptr_t)p.w | (uintptr_t)p.cache;
        strides |= p.in_t | p.in_h | p.out_t | p.out_h | p.c_page | p.c_slot | p.c_head;
    }
    return (at & 15) == 0 && strides % unit == 0;
}

int launch_heads(const HeadsArgs& args, int dtype, const char* who, hipStream_t s) {
    HeadsArgs a = args;
    a.heads = a.p[0].heads + a.p[1].heads + a.p[2].heads;
    if (a.tokens == 0 || a.heads == 0) return SQ_OK;
    a.inv_dim = 1.f / (float)a.dim;
    if (wide_ok(a, dtype)) {
        a.lanes_log2 = 0;
        while ((16 << a.lanes_log2) < a.dim) ++a.lanes_log2;
        const int items = a.heads << a.lanes_log2;
        // Many tokens: two waves each, the heads in turn, so that fewer waves hold their places while one or two work the angles out (28 + 4 + 4 heads of 128 normed,
        // 2048 tokens 15.1 us with a thread per item, 12.8 so, with one wave 13.7; 8192: 45.7, 34.0, 32.6; 1024: 8.2, 8.3, 9.9; over the same memory each time)
        const int most = a.tokens > 4 * device_cus() ? 128 : HEADS_MAX_THREADS, rounds = (items + most - 1) / most;
        const int threads = ((items + rounds - 1) / rounds + 63) / 64 * 64;
        // few tokens: their heads over several workgroups (each works the angles out again); enough of them: one workgroup takes a token whole
        const int parts = a.tokens >= 2 * device_cus() ? 1 : rounds;
        const dim3 grid((unsigned)(a.tokens < (1 << 20) ? a.tokens : 1 << 20), (unsigned)(parts < 65535 ? parts : 65535));
        const size_t lds = (size_t)(a.pairs ? a.pairs : 1) * sizeof(float2v);
        const int wt = !(a.p[0].w || a.p[1].w) ? NO_NORM : a.w_dtype;
        auto go = [&](auto dt, auto w) {
            constexpr int DT = decltype(dt)::value, WT = decltype(w)::value;
            if (a.interleaved) hipLaunchKernelGGL((heads_kernel<DT, WT, true>), grid, dim3(threads), lds, s, a);
            else hipLaunchKernelGGL((heads_kernel<DT, WT, false>), grid, dim3(threads), lds, s, a);
        };
        auto of = [&](auto dt) {
            if (wt == NO_NORM) go(dt, std::integral_constant<int, NO_NORM>());
            else if (wt == SQ_F32) go(dt, std::integral_constant<int, SQ_F32>());
            else go(dt, dt);
        };
        if (dtype == SQ_F32) of(std::integral_constant<int, SQ_F32>());
        else if (dtype == SQ_F16) of(std::integral_constant<int, SQ_F16>());
        else of(std::integral_constant<int, SQ_BF16>());
        return check_launch(who);
    }
    const int64_t blocks = ((int64_t)a.tokens * a.heads + 3) / 4;
    const dim3 grid((unsigned)(blocks < (1 << 20) ? blocks : 1 << 20));
    if (dtype == SQ_F32) hipLaunchKernelGGL(heads_any_kernel<SQ_F32>, grid, dim3(256), 0, s, a);
    else if (dtype == SQ_F16) hipLaunchKernelGGL(heads_any_kernel<SQ_F16>, grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL(heads_any_kernel<SQ_BF16>, grid, dim3(256), 0, s, a);
    return check_launch(who);
}

// Whether heads of dim elements, t apart from token to token and h from head to head, share no element: heads lie within tokens or tokens within heads,
// as far as there are several
bool rows_apart(int tokens, int heads, int64_t t, int64_t h, int dim) {
    if (heads <= 1) return tokens <= 1 || t >= dim;
    if (tokens <= 1) return h >= dim;
    return (h >= dim && t >= (heads - 1) * h + dim) || (t >= dim && h >= (tokens - 1) * t + dim);
}

static int check_heads(const char* who, const sq_heads* p, int tokens, int dim, bool needs_out) {
    if (p->heads < 0 || p->heads > (1 << 20)) return fail(SQ_EINVAL, "%s: %d heads", who, p->heads);
    if (tokens && p->heads && (!p->in || (needs_out && !p->out))) return fail(SQ_EINVAL, "%s: null in / out", who);
    if (p->out && tokens && p->heads) {
        const int64_t t = p->out_token < 0 ? -p->out_token : p->out_token, h = p->out_head < 0 ? -p->out_head : p->out_head;
        const bool ok = rows_apart(tokens, p->heads, t, h, dim);
        if (!ok) return fail(SQ_EINVAL, "%s: rows of the output overlap (strides %lld, %lld)", who, (long long)p->out_token, (long long)p->out_head);
        if (p->out == p->in && ((tokens > 1 && p->out_token != p->in_token) || (p->heads > 1 && p->out_head != p->in_head)))
            return fail(SQ_EINVAL, "%s: in place with other strides", who);
    }
    return SQ_OK;
}

static int check_rotation(const char* who, const sq_rotation* r, int tokens, int dim, HeadsArgs& a) {
    if (r->pairs < 0 || 2 * (int64_t)r->pairs > dim) return fail(SQ_EINVAL, "%s: %d pairs of %d elements", who, r->pairs, dim);
    if (r->pairs && tokens && (!r->freqs || !r->positions)) return fail(SQ_EINVAL, "%s: null freqs / positions", who);
    a.freqs = r->freqs; a.positions = r->positions; a.wide_positions = r->positions_64 != 0; a.pairs = r->pairs;
    a.interleaved = r->interleaved != 0; a.scale = r->scale; a.sign = r->inverse ? -1.f : 1.f;
    return SQ_OK;
}

static void put_part(HeadsPart& p, const sq_heads* h, int turn) {
    p.in = h->in; p.out = h->out; p.w = h->w; p.in_t = h->in_token; p.in_h = h->in_head; p.out_t = h->out_token; p.out_h = h->out_head;
    p.heads = h->heads; p.turn = turn;
}

// ------------------------------------------------------------------------------------------ the accepted path of a draft

struct KeepArgs {
    char *k, *v;
    int64_t k_layer, k_page, k_slot, k_head, v_layer, v_page, v_slot, v_head;     // bytes
    const int32_t *table, *lens, *path, *counts;
    int64_t ld_table, ld_path;
    int layers, pages, page, max_pages, heads, pieces, most;                      // pieces of a head's row
};

constexpr int KEEP_STEP = 64;           // path entries looked up at a time, one per lane
constexpr int KEEP_FLY = 8;             // rows in flight per thread

// A thread moves one piece (16 bytes, or one element) of a head's rows, of one layer's keys or values: a sequence's kept rows in turn.  The path
// ascends and starts at 0 or behind, so row i comes from slot path[i] >= i and no row is read after it was written; entries from the
// first one on that does not ascend, or that leaves the table or names a page outside the cache, are ignored.
// Bound by HBM: 64 sequences' paths through 28 layers, 58.7 MB read and written, 11.4 us; one sequence's by its launch and two dependent loads, 3.7 us.
template <typename T>
__global__ __launch_bounds__(256) void keep_kernel(KeepArgs a) {
    __shared__ int64_t from_page[KEEP_STEP], to_page[KEEP_STEP];
    __shared__ int from_off[KEEP_STEP], to_off[KEEP_STEP], valid;
    const int b = blockIdx.y, tid = threadIdx.x;
    const int64_t unit = (int64_t)blockIdx.x * 256 + tid, per_layer = (int64_t)a.heads * a.pieces, units = 2 * a.layers * per_layer;
    const int count = min(a.counts[b], a.most);
    const int64_t len = max(a.lens[b], 0), cap = (int64_t)a.max_pages * a.page;
    const int64_t lk = unit / per_layer, rest = unit - lk * per_layer;
    const bool is_v = lk & 1;
    const int64_t layer = lk >> 1, head = rest / a.pieces, piece = rest - head * a.pieces;
    char* base = (is_v ? a.v + layer * a.v_layer + head * a.v_head : a.k + layer * a.k_layer + head * a.k_head) + piece * (int64_t)sizeof(T);
    const int64_t page_b = is_v ? a.v_page : a.k_page, slot_b = is_v ? a.v_slot : a.k_slot;
    for (int i0 = 0; i0 < count; i0 += KEEP_STEP) {
        if (i0) __syncthreads();
        if (tid < KEEP_STEP) {
            const int i = i0 + tid;
            bool ok = i < count;
            if (ok) {
                const int32_t* path = a.path + (int64_t)b * a.ld_path;
                const int p = path[i];
                const int64_t src = len + p, dst = len + i;
                ok = p >= 0 && (i == 0 || p > path[i - 1]) && src < cap && dst < cap;          // (behind an entry that does not ascend, dst may lie behind src)
                if (ok) {
                    const int sp = (int)(src / a.page), dp = (int)(dst / a.page);
                    const int32_t sid = a.table[(int64_t)b * a.ld_table + sp], did = a.table[(int64_t)b * a.ld_table + dp];
                    ok = (uint32_t)sid < (uint32_t)a.pages && (uint32_t)did < (uint32_t)a.pages;
                    from_page[tid] = sid; to_page[tid] = did;
                    from_off[tid] = (int)(src - (int64_t)sp * a.page); to_off[tid] = (int)(dst - (int64_t)dp * a.page);
                }
            }
            const uint64_t all = __ballot(ok);
            if (tid == 0) valid = all == ~0ull ? KEEP_STEP : __builtin_ctzll(~all);
        }
        __syncthreads();
        const int m = valid;
        if (unit < units)
            for (int i = 0; i < m; i += KEEP_FLY) {
                T v[KEEP_FLY];
#pragma unroll
                for (int j = 0; j < KEEP_FLY; ++j)
                    if (i + j < m) v[j] = *reinterpret_cast<const T*>(base + from_page[i + j] * page_b + from_off[i + j] * slot_b);
#pragma unroll
                for (int j = 0; j < KEEP_FLY; ++j)
                    if (i + j < m) *reinterpret_cast<T*>(base + to_page[i + j] * page_b + to_off[i + j] * slot_b) = v[j];
            }
        if (m < KEEP_STEP) return;
    }
}

}  // namespace sq

using namespace sq;

extern "C" {

int sq_rotary(const sq_heads* x, int32_t tokens, int32_t dim, int dtype, const sq_rotation* rot, void* stream) {
    const char* who = "sq_rotary";
    if (!x || !rot) return fail(SQ_EINVAL, "%s: null argument", who);
    if (dtype < SQ_F32 || dtype > SQ_BF16) return fail(SQ_EINVAL, "%s: dtype %d", who, dtype);
    if (tokens < 0 || tokens > (1 << 30) || dim < 1 || dim > 65536) return fail(SQ_EINVAL, "%s: %d tokens of heads of %d", who, tokens, dim);
    HeadsArgs a = {};
    if (int rc = check_heads(who, x, tokens, dim, true)) return rc;
    if (int rc = check_rotation(who, rot, tokens, dim, a)) return rc;
    put_part(a.p[0], x, 1);
    a.p[0].w = nullptr;
    a.tokens = tokens; a.dim = dim;
    return launch_heads(a, dtype, who, (hipStream_t)stream);
}

int sq_qk_norm_rotary(const sq_heads* q, const sq_heads* k, const sq_heads* v, int32_t tokens, int32_t dim, int dtype, const sq_rotation* rot, int w_dtype,
                      float eps, float w_offset, const sq_cache* cache, const void* slots, int slots_64, void* stream) {
    const char* who = "sq_qk_norm_rotary";
    if (!q || !k || !rot) return fail(SQ_EINVAL, "%s: null argument", who);
    if (dtype < SQ_F32 || dtype > SQ_BF16 || w_dtype < SQ_F32 || w_dtype > SQ_BF16) return fail(SQ_EINVAL, "%s: dtype %d, w_dtype %d", who, dtype, w_dtype);
    if (tokens < 0 || tokens > (1 << 30) || dim < 1 || dim > 65536) return fail(SQ_EINVAL, "%s: %d tokens of heads of %d", who, tokens, dim);
    if ((v != nullptr) != (cache != nullptr)) return fail(SQ_EINVAL, "%s: values go to a cache, and a cache takes both", who);
    HeadsArgs a = {};
    if (int rc = check_heads(who, q, tokens, dim, true)) return rc;
    if (int rc = check_heads(who, k, tokens, dim, !cache)) return rc;
    if (int rc = check_rotation(who, rot, tokens, dim, a)) return rc;
    put_part(a.p[0], q, 1);
    put_part(a.p[1], k, 1);
    if (cache) {
        if (int rc = check_heads(who, v, tokens, dim, false)) return rc;
        if (v->heads != k->heads || cache->heads != k->heads || cache->dim != dim || cache->dtype != dtype)
            return fail(SQ_EINVAL, "%s: cache of %d heads of %d, type %d, for %d key and %d value heads of %d, type %d", who, cache->heads, cache->dim,
                        cache->dtype, k->heads, v->heads, dim, dtype);
        if (cache->pages < 0 || cache->page < 1 || (int64_t)cache->pages * cache->page > INT32_MAX)
            return fail(SQ_EINVAL, "%s: %d pages of %d slots", who, cache->pages, cache->page);
        if (tokens && k->heads && (!slots || !cache->k || !cache->v)) return fail(SQ_EINVAL, "%s: null slots / cache", who);
        put_part(a.p[2], v, 0);
        a.p[2].w = nullptr;
        a.p[1].cache = cache->k; a.p[1].c_page = cache->k_page; a.p[1].c_slot = cache->k_slot; a.p[1].c_head = cache->k_head;
        a.p[2].cache = cache->v; a.p[2].c_page = cache->v_page; a.p[2].c_slot = cache->v_slot; a.p[2].c_head = cache->v_head;
        a.slots = slots; a.wide_slots = slots_64 != 0; a.pages = cache->pages; a.page = cache->page;
    }
    a.tokens = tokens; a.dim = dim; a.w_dtype = w_dtype; a.eps = eps; a.w_offset = w_offset;
    return launch_heads(a, dtype, who, (hipStream_t)stream);
}

int sq_keep_drafted(const sq_cache* cache, int32_t layers, int64_t k_layer, int64_t v_layer, const int32_t* table, int64_t ld_table, int32_t max_pages,
                    const int32_t* lens, const int32_t* path, int64_t ld_path, int32_t most, const int32_t* counts, int32_t seqs, void* stream) {
    const char* who = "sq_keep_drafted";
    if (!cache) return fail(SQ_EINVAL, "%s: null cache", who);
    if (cache->dtype < SQ_F32 || cache->dtype > SQ_BF16) return fail(SQ_EINVAL, "%s: dtype %d", who, cache->dtype);
    if (layers < 0 || seqs < 0 || seqs > 65535 || most < 0 || cache->pages < 0 || cache->page < 1 || cache->heads < 0 || cache->dim < 1 || cache->heads > (1 << 20) ||
        cache->dim > 65536 || layers > (1 << 20) || max_pages < 0 || ld_table < max_pages || ld_path < most)
        return fail(SQ_EINVAL, "%s: %d layers, %d sequences, paths of %d (ld %lld), tables of %d (ld %lld), %d pages of %d, %d heads of %d", who, layers, seqs, most,
                    (long long)ld_path, max_pages, (long long)ld_table, cache->pages, cache->page, cache->heads, cache->dim);
    if (!layers || !seqs || !most || !max_pages || !cache->pages || !cache->heads) return SQ_OK;
    if (!cache->k || !cache->v || !table || !lens || !path || !counts) return fail(SQ_EINVAL, "%s: null argument", who);
    const int size = cache->dtype == SQ_F32 ? 4 : 2;
    KeepArgs a;
    a.k = (char*)cache->k; a.v = (char*)cache->v;
    a.k_layer = k_layer * size; a.k_page = cache->k_page * size; a.k_slot = cache->k_slot * size; a.k_head = cache->k_head * size;
    a.v_layer = v_layer * size; a.v_page = cache->v_page * size; a.v_slot = cache->v_slot * size; a.v_head = cache->v_head * size;
    a.table = table; a.lens = lens; a.path = path; a.counts = counts; a.ld_table = ld_table; a.ld_path = ld_path;
    a.layers = layers; a.pages = cache->pages; a.page = cache->page; a.max_pages = max_pages; a.heads = cache->heads; a.most = most;
    const int64_t strides = a.k_layer | a.k_page | a.k_slot | a.k_head | a.v_layer | a.v_page | a.v_slot | a.v_head | (int64_t)cache->dim * size;
    const int piece = strides % 16 == 0 && (((uintptr_t)a.k | (uintptr_t)a.v) & 15) == 0 ? 16 : size;
    a.pieces = cache->dim * size / piece;
    const int64_t units = 2 * (int64_t)layers * a.heads * a.pieces, blocks = (units + 255) / 256;
    if (blocks > (1 << 23)) return fail(SQ_EUNSUPPORTED, "%s: %lld pieces per slot", who, (long long)units);
    const dim3 grid((unsigned)blocks, (unsigned)seqs);
    if (piece == 16) hipLaunchKernelGGL(keep_kernel<u32x4>, grid, dim3(256), 0, (hipStream_t)stream, a);
    else if (piece == 4) hipLaunchKernelGGL(keep_kernel<uint32_t>, grid, dim3(256), 0, (hipStream_t)stream, a);
    else hipLaunchKernelGGL(keep_kernel<uint16_t>, grid, dim3(256), 0, (hipStream_t)stream, a);
    return check_launch(who);
}

}  // extern "C"
