// Attention of few rows over a cache held in 8 bits (sq_tree_attention8), built once per 16-bit type of the rows; that of many rows is
// attn_tile_kernel of sq_attention.h, and so is all that does not read the cache.
//
// A key's codes are half the bytes of 16-bit elements, and what holds the kernel up is reading them.  They reach LDS as they are, become the
// matrix instructions' 16-bit operands in registers, scale included, and from there on all is as over a 16-bit cache: the products are of the very numbers that are held.
// First operand, keys: lane l reads 16 elements of key l % 16 at once, two operands of 8 (the rows' elements are in the same order).
// First operand, values: ds_read_b64_tr_b8 lets 16 lanes read 8 keys x 16 elements and gives lane i the 8 keys of element i; the keys are the
// scores' (4 * (l / 16) .. + 3 and 16 + 4 * (l / 16) .. + 3), so each half of them has one scale.
#pragma once
#include "sq_attention.h"

namespace sq {

// Layout of a step's keys (or values) in LDS: rows of DP bytes, their 16-byte pieces placed by XOR with the key's number so that 16 keys' pieces (first product), and the
// 16 keys that two groups of lanes read at once (transposing reads), lie in different banks
template <int DP> struct Attn8Tile {
    static constexpr int PIECES = DP / 16;                  // of a key
    static constexpr int ROWS = 64 / PIECES;                // keys per copy
    static constexpr int COPIES = ATTN_STEP / ROWS;
    static constexpr int PITCH = DP, BYTES = ATTN_STEP * PITCH;
    static __device__ __forceinline__ constexpr int k_xor(int key) { return PIECES == 4 ? (key >> 2) & 3 : PIECES == 8 ? (key >> 1) & 7 : key & 15; }
    static __device__ __forceinline__ constexpr int v_xor(int key) {
        const int half = (key >> 4) & 1;
        return PIECES == 4 ? ((key >> 2) & 1) | half << 1 : PIECES == 8 ? ((key >> 1) & 3) | half << 2 : (key & 7) | half << 3;
    }
};

// Copies 16 keys (or values), of half x of a step, to `to`; from: the first one's byte of the head.  PASSING: past the caches (see attn_copy16)
__device__ __forceinline__ void attn8_copy16_passing(uint32_t to, const char* at, uint32_t offset) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2 nt" ::"s"(to), "v"(offset), "s"(at) : "memory");
}
template <int DP, bool FULL, bool VALUES, bool PASSING>
__device__ __forceinline__ void attn8_copy(const Attn8Args& a, int x, int lane, const char* from, const char* to) {
    typedef Attn8Tile<DP> T;
    const int row = lane / T::PIECES, pos = lane % T::PIECES, pieces = a.dim >> 4, slot = (int)(VALUES ? a.v_slot : a.k_slot);
    const uint32_t lds = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(lds_ptr)to);
#pragma unroll
    for (int j = 0; j < 16 / T::ROWS; ++j) {
        const int key = 16 * x + j * T::ROWS + row, c = pos ^ (VALUES ? T::v_xor(key) : T::k_xor(key));
        if (FULL || c < pieces) {
            if constexpr (PASSING) attn8_copy16_passing(lds + j * 1024, from, (uint32_t)((j * T::ROWS + row) * slot + c * 16));
            else attn_copy16(lds + j * 1024, from, (uint32_t)((j * T::ROWS + row) * slot + c * 16));
        }
    }
}

// scores of a step: codes of its keys at k, scales of its halves
template <int DT, int DP, int MT>
__device__ __forceinline__ void attn8_scores(const AttnRows<DP, MT>& r, const char* k, const float (&by)[2], int lane, float4v (&st)[MT][2]) {
    typedef Attn8Tile<DP> T;
    const int g = lane >> 4, i16 = lane & 15;
#pragma unroll
    for (int t = 0; t < MT; ++t) st[t][0] = st[t][1] = float4v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int c = 0; c < DP / 64; ++c)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const u32x4 w = *reinterpret_cast<const u32x4*>(k + (h * 16 + i16) * T::PITCH + (((c * 4 + g) ^ T::k_xor(h * 16 + i16)) * 16));
            const u32x4 f0 = attn8_unpack<DT>(w[0], w[1], by[h], by[h]), f1 = attn8_unpack<DT>(w[2], w[3], by[h], by[h]);
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                st[t][h] = AttnType<DT>::mfma(f0, r.q[t][2 * c], st[t][h]);
                st[t][h] = AttnType<DT>::mfma(f1, r.q[t][2 * c + 1], st[t][h]);
            }
        }
}

// sums of a step: codes of its values at v.  Where MASKED, values that are not finite (codes of NaN; in fp16 what a scale carries beyond its range) do not go
// through the product, see attn_sums.
template <int DT, int DP, int MT, bool MASKED>
__device__ __forceinline__ void attn8_sums(AttnRows<DP, MT>& r, const char* v, const float (&by)[2], int lane, const u32x4 (&p)[MT], const uint32_t (&sees)[MT]) {
    typedef Attn8Tile<DP> T;
    typedef AttnType<DT> E;
    typedef int int2v __attribute__((ext_vector_type(2)));
    typedef __attribute__((address_space(3))) int2v* tr_ptr;
    const int g = lane >> 4, i16 = lane & 15, key = ((i16 & 8) << 1) + 4 * g + ((i16 >> 1) & 3);
#pragma unroll
    for (int d = 0; d < DP / 16; ++d) {
        const u32x2 w = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr8_b64_v2i32((tr_ptr)(lds_ptr)(v + key * T::PITCH + ((d ^ T::v_xor(key)) * 16) + (i16 & 1) * 8)));
        u32x4 f = attn8_unpack<DT>(w[0], w[1], by[0], by[1]);
        if constexpr (MASKED) {
            uint32_t odd = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) odd |= (f[i] & 0x7FFF7FFFu) + (0x8000u - E::INF) * 0x10001u;
            if (__any((odd & 0x80008000u) != 0)) {
                u32x4 up, down;                              // ones where a value is not below +inf, not above -inf
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    uint32_t clean = 0, u = 0, n = 0;
#pragma unroll
                    for (int y = 0; y < 2; ++y) {
                        const uint32_t bits = (f[i] >> (16 * y)) & 0xFFFF;
                        const bool nan = (bits & 0x7FFF) > E::INF, inf = (bits & 0x7FFF) == E::INF;
                        if (!nan && !inf) clean |= bits << (16 * y);
                        if (nan || (inf && !(bits & 0x8000))) u |= E::ONE << (16 * y);
                        if (nan || (inf && (bits & 0x8000))) n |= E::ONE << (16 * y);
                    }
                    f[i] = clean; up[i] = u; down[i] = n;
                }
#pragma unroll
                for (int t = 0; t < MT; ++t) {
                    u32x4 vis;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const uint32_t two = sees[t] >> ((i >> 1) * 16 + g * 4 + (i & 1) * 2);
                        vis[i] = (two & 1 ? E::ONE : 0u) | (two & 2 ? E::ONE << 16 : 0u);
                    }
                    const float4v zero = float4v{0.f, 0.f, 0.f, 0.f};
                    const float4v cu = E::mfma(up, vis, zero), cd = E::mfma(down, vis, zero);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        if (cu[i] > 0.f) r.o[t][d][i] += INFINITY;
                        if (cd[i] > 0.f) r.o[t][d][i] -= INFINITY;
                    }
                }
            }
        }
#pragma unroll
        for (int t = 0; t < MT; ++t) r.o[t][d] = E::mfma(f, p[t], r.o[t][d]);
    }
}

// Workgroups of ATTN8_WAVES that a compute unit holds, and steps of codes that each wave has in LDS (two or four), 128 KB of a unit in all.  A step is a chain (wait, read, unpack,
// multiply, exponentials, read, unpack, multiply) of which a second wave of the SIMD fills the gaps: with all data in the caches, 32 sequences of 8192 x 8 key heads of 128 take 80 us
// with one wave a SIMD, 55 with two; heads of 256 have no registers for it.
constexpr int attn8_groups(int dp, int mt) { return dp == 256 ? 1 : dp == 64 && mt == 1 ? 4 : 2; }
constexpr int attn8_ring(int dp, int mt) { return 131072 / attn8_groups(dp, mt) / (ATTN8_WAVES * 2 * ATTN_STEP * dp); }
// and the scales of the groups they are of: of 64 groups of keys and 64 of values, twice
constexpr int ATTN8_SCALES = 1024;
// Copies a byte per lane to LDS, lane l's to `to` + 4 l, as 32 bits (see attn_copy16)
__device__ __forceinline__ void attn8_copy_scale(uint32_t to, const uint8_t* at) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_ubyte %1, off" ::"s"(to), "v"(at) : "memory");
}
template <int DP, int MT, int NW> constexpr int attn8_lds() {
    constexpr int ring = NW * (attn8_ring(DP, MT) * 2 * Attn8Tile<DP>::BYTES + ATTN8_SCALES), join = NW * MT * 16 * ((DP + 4) * 4 + 8) + 64;
    return ring > join ? ring : join;
}

// Few rows, as attn_kernel: the waves of a workgroup share the rows and split its keys, no barrier until their sums are joined.
template <int DT, int DP, int MT, int NW, bool FULL, bool PASSING>
__global__ __launch_bounds__(NW * 64) __attribute__((amdgpu_waves_per_eu(NW * attn8_groups(DP, MT) / 4, NW * attn8_groups(DP, MT) / 4))) void attn8_kernel(Attn8Args a) {
    typedef Attn8Tile<DP> T;
    extern __shared__ __attribute__((aligned(1024))) char smem[];
    constexpr int C = T::COPIES, ROWS = MT * 16, RING = attn8_ring(DP, MT);          // (C: of a step's keys, or values)
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    int id = blockIdx.x, in = 0;
    if (a.inner > 1) {                                       // as far as eights of parts go
        const int parts = gridDim.x / a.inner, eights = parts & ~7, over = id - eights * a.inner;
        in = over < 0 ? id / 8 % a.inner : over % a.inner;
        id = over < 0 ? id / 8 / a.inner * 8 + id % 8 : eights + over / a.inner;
    }
    // (the last rows, which see most keys without a mask, begin first: a prompt of 700 tokens 24.1 us, so 20.8)
    const int row0 = (a.row_blocks - 1 - in % a.row_blocks) * ROWS, split = id % a.splits;
    id /= a.splits;
    int head = in / a.row_blocks;
    if (a.inner == a.row_blocks) { head = id % a.kv_heads; id /= a.kv_heads; }
    const int b = id;
    const AttnSeq s = attn_seq(a, b);
    const int rows = s.n * a.group;
    if (row0 >= rows) return;
    const int last = min(row0 + ROWS, rows) - 1;
    const int seen = a.mask ? s.total : min(s.total, s.len + last / a.group + 1);            // keys that some row sees
    const int whole = a.mask ? min(s.len, s.total) : min(s.total, s.len + row0 / a.group + 1);        // and that all do
    const int steps = (seen + ATTN_STEP - 1) / ATTN_STEP;
    const int per = max((steps + a.splits - 1) / a.splits, NW), begin = min(split * per, steps), end = min(begin + per, steps);
    const int each = (end - begin + NW - 1) / NW, w0 = min(begin + wave * each, end), w1 = min(w0 + each, end);

    AttnRows<DP, MT> r;
    attn_rows_begin<DP, MT, true>(a, s, head, row0, lane, r);
    const char *kb = a.kc + head * a.k_head, *vb = a.vc + head * a.v_head;
    char* ring = smem + wave * (RING * 2 * T::BYTES);
    Attn8Groups groups;
    char* scales = smem + NW * (RING * 2 * T::BYTES) + wave * ATTN8_SCALES;
    auto slot = [&](int i) __attribute__((always_inline)) { return ring + (i % RING) * (2 * T::BYTES); };
    auto get_k = [&](int i) __attribute__((always_inline)) {
        const int n = i - w0;
        if (n % 32 == 0) {                                   // the groups of the next 32 steps, their scales ahead of the keys
            groups.find(a, b, head, i * ATTN_STEP, 16, min(s.total, w1 * ATTN_STEP), lane);
            const uint32_t to = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(lds_ptr)(scales + n / 32 % 2 * 512));
            attn8_copy_scale(to, groups.ks);
            attn8_copy_scale(to + 256, groups.vs);
        }
#pragma unroll
        for (int x = 0; x < 2; ++x) attn8_copy<DP, FULL, false, PASSING>(a, x, lane, kb + groups.lane64(groups.k, 2 * (n % 32) + x), slot(i) + x * 16 * T::PITCH);
    };
    auto get_v = [&](int i) __attribute__((always_inline)) {         // (behind get_k of the same step)
#pragma unroll
        for (int x = 0; x < 2; ++x) attn8_copy<DP, FULL, true, PASSING>(a, x, lane, vb + groups.lane64(groups.v, 2 * ((i - w0) % 32) + x), slot(i) + T::BYTES + x * 16 * T::PITCH);
    };
    if constexpr (!FULL) {
        attn_clear(ring, RING * 2 * T::BYTES, lane, 64);
        attn_reads_done();
    }
#pragma unroll
    for (int i = 0; i < RING; ++i)
        if (w0 + i < w1) { get_k(w0 + i); get_v(w0 + i); }
    attn_rows_ready(r);
    auto step = [&](int i, auto masked) __attribute__((always_inline)) {
        constexpr bool MASKED = decltype(masked)::value;
        float4v st[MT][2];
        u32x4 p[MT];
        uint32_t sees[MT] = {};
        const int behind = min(w1 - 1 - i, RING - 1);        // steps that follow on their way
        // (steps that follow are on their way: their keys and values, and of this one its values)
        auto arrived = [&](auto extra) __attribute__((always_inline)) {
            constexpr int X = decltype(extra)::value;
            if (RING > 2 && behind == 3) attn_wait<(6 + X) * C>();
            else if (RING > 2 && behind == 2) attn_wait<(4 + X) * C>();
            else if (behind == 1) attn_wait<(2 + X) * C>();
            else attn_wait<X * C>();
        };
        arrived(std::integral_constant<int, 1>());
        const u32x2* sc = reinterpret_cast<const u32x2*>(scales + (i - w0) / 32 % 2 * 512 + (i - w0) % 32 * 8);
        const u32x2 ksc = sc[0], vsc = sc[32];
        const float kby[2] = {attn8_scale(ksc[0]), attn8_scale(ksc[1])}, vby[2] = {attn8_scale(vsc[0]), attn8_scale(vsc[1])};
        attn8_scores<DT, DP, MT>(r, slot(i), kby, lane, st);
        __builtin_amdgcn_sched_barrier(0);
        attn_reads_done();
        const bool more = i + RING < w1;
        if (more) get_k(i + RING);
        if constexpr (MASKED)
#pragma unroll
            for (int t = 0; t < MT; ++t) sees[t] = attn_sees(a, s, i, r.tok[t]);
        attn_weights<DT, DP, MT, MASKED>(a, r, st, sees, lane, p);
        if (more) arrived(std::integral_constant<int, 1>()); else arrived(std::integral_constant<int, 0>());
        attn8_sums<DT, DP, MT, MASKED>(r, slot(i) + T::BYTES, vby, lane, p, sees);
        __builtin_amdgcn_sched_barrier(0);
        attn_reads_done();
        if (more) get_v(i + RING);
    };
    const int clear = min(max(whole / ATTN_STEP, w0), w1);
    for (int i = w0; i < clear; ++i) step(i, std::false_type());
    for (int i = clear; i < w1; ++i) step(i, std::true_type());
    // the waves' sums meet in LDS
    __syncthreads();
    constexpr int PITCH = DP + 4;
    float* sums = reinterpret_cast<float*>(smem);
    float2v* ml = reinterpret_cast<float2v*>(smem + NW * ROWS * PITCH * 4);
    int* flags = reinterpret_cast<int*>(ml + NW * ROWS);
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        const int row = t * 16 + (lane & 15);
        const float l = groups_fold(r.l[t], [](float x, float y) { return x + y; });
        if (lane < 16) ml[wave * ROWS + row] = float2v{r.m[t], l};
#pragma unroll
        for (int d = 0; d < DP / 16; ++d)
            *reinterpret_cast<float4v*>(sums + (size_t)(wave * ROWS + row) * PITCH + d * 16 + (lane >> 4) * 4) = r.o[t][d];
    }
    const bool bad = __any(groups.bad) || s.over;
    if (lane == 0) flags[wave] = bad;
    __syncthreads();
    bool any = false;
#pragma unroll
    for (int w = 0; w < NW; ++w) any |= flags[w] != 0;
    attn_write<DT, DP>(a, s, head, row0, ROWS, split, sums, ml, NW, ROWS, any, tid, NW * 64);
}

// ------------------------------------------------------------------------------------------ host

template <int DT, int DP, int MT, bool FULL, bool PASSING>
int attn8_launch_few(const Attn8Args& a, unsigned grid, hipStream_t s) {
    constexpr int NW = ATTN8_WAVES, LDS = attn8_lds<DP, MT, NW>();
    static bool raised[64];
    attn_raise((const void*)attn8_kernel<DT, DP, MT, NW, FULL, PASSING>, LDS, raised);
    hipLaunchKernelGGL((attn8_kernel<DT, DP, MT, NW, FULL, PASSING>), dim3(grid), dim3(NW * 64), LDS, s, a);
    return check_launch("sq_tree_attention8");
}
template <int DT, int DP, int NW, bool FULL, typename ARGS>
int attn8_launch_many(const ARGS& a, unsigned grid, hipStream_t s) {
    constexpr int LDS = attn8_tile_lds<DP, NW>();
    static bool raised[64];
    attn_raise((const void*)attn_tile_kernel<DT, DP, NW, FULL, ARGS>, LDS, raised);
    hipLaunchKernelGGL((attn_tile_kernel<DT, DP, NW, FULL, ARGS>), dim3(grid), dim3(NW * 64), LDS, s, a);
    return check_launch("sq_tree_attention8");
}
template <int DT, int DP, bool FULL>
int attn8_launch_dim(const Attn8Shared& a, const AttnPlan& p, hipStream_t s) {
    const unsigned grid = (unsigned)(p.workgroups ? (int64_t)a.kv_heads * p.workgroups : (int64_t)a.seqs * a.kv_heads * ((p.row_blocks - 1) * p.splits + p.last_splits));
    int rc;
    if (p.nw) {
        auto many = [&](const auto& args) {
            typedef std::decay_t<decltype(args)> ARGS;
            return p.nw == 4 ? attn8_launch_many<DT, DP, 4, FULL, ARGS>(args, grid, s) : attn8_launch_many<DT, DP, 8, FULL, ARGS>(args, grid, s);
        };
        rc = a.parts ? many(a) : many((const Attn8Args&)a);
    }
    else {
        auto few = [&](auto passing) {
            constexpr bool P = decltype(passing)::value;
            return p.mt == 1 ? attn8_launch_few<DT, DP, 1, FULL, P>(a, grid, s) : attn8_launch_few<DT, DP, DP == 256 ? 1 : 2, FULL, P>(a, grid, s);
        };
        constexpr bool lines = FULL && DP >= 128;            // (heads that are lines of their own: nobody else reads them)
        rc = lines && a.passing ? few(std::integral_constant<bool, lines>()) : few(std::false_type());
    }
    if (rc || p.slots == 1) return rc;
    return a.parts ? attn_launch_join<DT, DP, Attn8Shared>(a, s) : attn_launch_join<DT, DP, AttnArgs>(a, s);
}
template <int DT>
int attn8_launch(const Attn8Shared& a, const AttnPlan& p, hipStream_t s) {
    auto go = [&](auto dp) {
        constexpr int DP = decltype(dp)::value;
        return a.dim == DP ? attn8_launch_dim<DT, DP, true>(a, p, s) : attn8_launch_dim<DT, DP, false>(a, p, s);
    };
    return p.dp == 64 ? go(std::integral_constant<int, 64>()) : p.dp == 128 ? go(std::integral_constant<int, 128>()) : go(std::integral_constant<int, 256>());
}
int attn8_launch_f16(const Attn8Shared& a, const AttnPlan& p, hipStream_t s);
int attn8_launch_bf16(const Attn8Shared& a, const AttnPlan& p, hipStream_t s);

}  // namespace sq
