// Attention of new tokens over a paged cache (sq_tree_attention): the kernels, built once per 16-bit type.
//
//   s_j = scale q . k_j over the keys j a token sees,  m = max s_j,  out = sum exp(s_j - m) v_j / sum exp(s_j - m)
//
// in one pass over the keys with the running maximum and sum.  The query heads that share a key head, of all new tokens of a
// sequence, are the rows of one matrix (row = token * group + head in group), so a key is read once for all of them.
//
// A step is 32 keys.  v_mfma_f32_16x16x32 takes the keys as its A operand (lane l: key l % 16, elements 8 * (l / 16) ..) and the rows
// as its B operand (lane l: row l % 16), so lane l holds, of row l % 16, the scores of keys 4 * (l / 16) .. + 3 and 16 + 4 * (l / 16) .. + 3: eight keys
// which, taken in that order, are the eight consecutive k of the second product's B operand.  Its A operand, values with the
// keys in the same order, is two transposing LDS reads (ds_read_b64_tr_b16: 16 lanes read 4 keys x 16 elements, lane i gets the 4 keys of element i).
// So weights go from one product to the other in registers, and the running maximum of a row, which its lanes share, scales the sums of that row without a shuffle.
//
// The matrix instructions take both operands in one type, so the weights are rounded to that of the values, once (in 32 bits, as a high and a low part, the second product
// would be two): by up to half a step, 2^-8 of a weight in bf16, 2^-11 in fp16.  fp16 holds them so down to 2^-14 only, in steps of 2^-24 below, and a key that has nearly all of
// the weight, as the first ones of a sequence often do, leaves the others there.  So in fp16 weights are 2^7 times what they are, at most 2^15: full precision down to 2^-21 of a
// row's largest weight, below that off by up to 2^-32 of it.  (2000 keys 17 below one whose value is zero: off by 4 % without the factor, by 2^-17 with it.  A larger one leaves
// less room for a maximum to rise, and sums are scaled more often: 2^11 and 2^4 of room, trees of 48 tokens 46.3 -> 49.5 us, 1900 tokens 134 -> 140.)
//
// Keys and values reach LDS with global_load_lds, whole rows at a time (16 bytes per lane, a key's elements by neighbouring lanes), their
// 16-byte pieces placed by XOR with the key's number so that 16 keys' pieces (first product) and 8 keys' pairs of pieces (transposing reads) lie in
// different banks; the XOR is in the source address, the copy itself is linear.
#pragma once
#include <type_traits>
#include <utility>
#include "sq_common.h"

namespace sq {

struct AttnArgs {
    const char* q;
    char* out;
    float* lse;
    const char *kc, *vc;
    const int32_t *table, *lens, *starts;
    const int64_t* mask;
    float* po;                   // splits > 1: sums [token, head, split, DP] and (maximum, total) [token, head, split]
    float2v* pml;
    int64_t q_t, q_h, o_t, o_h, k_page, k_slot, k_head, v_page, v_slot, v_head;      // bytes
    int64_t ld_table, ld_mask;
    int tokens, seqs, most_new, q_heads, kv_heads, group, dim, pages, page, max_pages, mask_words, row_blocks, splits, last_splits, last_row;
    // (splits: of the row blocks before the last one, whose first row is last_row and which has last_splits)
    int near;                    // the slots of a page lie within 2^31 bytes, in order
    float scale2;                // scale * log2(e): weights are powers of two
};

constexpr int ATTN_STEP = 32;                // keys of a step
constexpr int ATTN_KEYS_MAX = INT32_MAX - 4096;
constexpr int ATTN_SPLITS_MAX = 128;         // parts of a sequence
constexpr float ATTN_SLACK = 8.f;            // so far (log2) a row's scores may rise before what is taken off its exponents, and so its sums, follow
constexpr float ATTN_NOTHING = -3e38f;       // maximum of no scores: weights of -inf are zero against it, and it is nothing beside any other

// A sequence's rows and keys.  What its arguments say beyond the buffers is cut off here: no index below leaves them.
struct AttnSeq { int first, n, len, total; bool over; };
__device__ __forceinline__ AttnSeq attn_seq(const AttnArgs& a, int b) {
    AttnSeq s;
    int end;
    if (a.starts) {
        s.first = min(max(a.starts[b], 0), a.tokens);
        end = min(max(a.starts[b + 1], s.first), a.tokens);
    } else {
        s.first = (int)min((int64_t)b * a.most_new, (int64_t)a.tokens);
        end = (int)min((int64_t)s.first + a.most_new, (int64_t)a.tokens);
    }
    s.n = min(end - s.first, a.most_new);
    const int64_t cap = min((int64_t)a.max_pages * a.page, (int64_t)ATTN_KEYS_MAX), want = (int64_t)max(a.lens[b], 0) + s.n;
    s.over = want > cap;
    s.total = (int)min(want, cap);
    s.len = max(s.total - s.n, 0);                           // (of a sequence that does not fit, which is NaN, what keeps len + n a number of 32 bits)
    return s;
}

template <int DT> struct AttnType;
template <> struct AttnType<SQ_F16> {
    typedef _Float16 v8 __attribute__((ext_vector_type(8)));
    static constexpr uint32_t INF = 0x7C00, ONE = 0x3C00;
    static constexpr float SHIFT = 7.f;      // log2 of the factor on weights.  (Not 8: with ATTN_SLACK they would reach 2^16, which is none; and where 32 bits go in steps of 16, x - 7 is x)
    static __device__ __forceinline__ float4v mfma(u32x4 x, u32x4 y, float4v c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8, x), __builtin_bit_cast(v8, y), c, 0, 0, 0);
    }
    // (no f2h_x2: its empty asm would keep these in order)
    static __device__ __forceinline__ uint32_t pack(float lo, float hi) { return __builtin_bit_cast(uint32_t, __builtin_convertvector((float2v){lo, hi}, half2v)); }
    static __device__ __forceinline__ uint16_t one(float v) { return f2h(v); }
};
template <> struct AttnType<SQ_BF16> {
    typedef __bf16 v8 __attribute__((ext_vector_type(8)));
    static constexpr uint32_t INF = 0x7F80, ONE = 0x3F80;
    static constexpr float SHIFT = 0.f;
    static __device__ __forceinline__ float4v mfma(u32x4 x, u32x4 y, float4v c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8, x), __builtin_bit_cast(v8, y), c, 0, 0, 0);
    }
    static __device__ __forceinline__ uint32_t pack(float lo, float hi) { return f2bf_x2(lo, hi); }
    static __device__ __forceinline__ uint16_t one(float v) { return f2bf(v); }
};

// The product that exponents of large scores are made from (attn_weights), in fp16 rounded by itself whatever is done with it
template <int DT> __device__ __forceinline__ float attn_rounded(float s, float scale2) {
    float x = s * scale2;
    if constexpr (DT == SQ_F16) asm("" : "+v"(x));
    return x;
}
// Whether the score `top` is more than SHIFT + ATTN_SLACK above m, which is taken off the exponents.  In fp16 by the rounded product: from 2^24 on it can lie further
// above m than the exact one does, and a weight of 2^16 would be an infinity.
template <int DT> __device__ __forceinline__ bool attn_above(float top, float scale2, float m) {
    if constexpr (DT == SQ_F16) return attn_rounded<DT>(top, scale2) - m > AttnType<DT>::SHIFT + ATTN_SLACK;
    return __builtin_fmaf(top, scale2, -(AttnType<DT>::SHIFT + ATTN_SLACK)) > m;
}
// log of the sum of exponentials, from what was taken off and the total
template <int DT> __device__ __forceinline__ float attn_lse(float m, float l) {
    constexpr float S = AttnType<DT>::SHIFT;
    if (l == 0.f) return -INFINITY;
    const float bits = fabsf(m) <= 0x1p20f ? (m + S) + __builtin_amdgcn_logf(l * __builtin_exp2f(-S)) : m + __builtin_amdgcn_logf(l);
    return bits * 0.6931471805599453f;
}

typedef __attribute__((address_space(3))) char* lds_ptr;

// Copies 16 bytes per lane to LDS, lane l's to `to` + 16 l, and waits for all but the newest N memory operations.  Written out, because the
// compiler waits for every copy in flight before a transposing read; they write no register, and what reads LDS stays behind the waits (memory clobber).
// (m0 is reserved: the compiler keeps nothing in it, takes no clobber of that name, and its own code for these kernels does not use it.)
// What the compiler loads into registers itself it waits for as if these were not there, that is for more than it has to.
__device__ __forceinline__ void attn_copy16(uint32_t to, const char* at, uint32_t offset) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(to), "v"(offset), "s"(at) : "memory");
}
__device__ __forceinline__ void attn_copy16(uint32_t to, const char* at) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(to), "v"(at) : "memory");
}
__device__ __forceinline__ void attn_reads_done() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }      // before copies to where was read (or written)
template <int N> __device__ __forceinline__ void attn_wait() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }

// value of every lane 16, 32 and 48 lanes away combined: the four groups of lanes that hold one row
template <typename F> __device__ __forceinline__ float groups_fold(float v, F f) {
    const uint32_t a = __builtin_bit_cast(uint32_t, v);
    const auto h = __builtin_amdgcn_permlane32_swap(a, a, false, false);
    v = f(__builtin_bit_cast(float, (uint32_t)h[0]), __builtin_bit_cast(float, (uint32_t)h[1]));
    const uint32_t b = __builtin_bit_cast(uint32_t, v);
    const auto r = __builtin_amdgcn_permlane16_swap(b, b, false, false);
    return f(__builtin_bit_cast(float, (uint32_t)r[0]), __builtin_bit_cast(float, (uint32_t)r[1]));
}

// Layout of a step's keys (or values) in LDS for heads of DP elements, and its copy
template <int DP> struct AttnTile {
    static constexpr int PIECES = DP / 8;                   // 16-byte pieces of a key
    static constexpr int ROWS = 64 / PIECES;                // keys per copy
    static constexpr int COPIES = ATTN_STEP / ROWS;
    static constexpr int PITCH = DP * 2, BYTES = ATTN_STEP * PITCH;
    static __device__ __forceinline__ constexpr int k_xor(int key) { return PIECES == 8 ? (key >> 1) & 7 : key & 15; }
    static __device__ __forceinline__ constexpr int v_xor(int key) { return PIECES == 8 ? 2 * ((key >> 1) & 3) : 2 * (key & 7); }
};

// Heads narrower than DP: what lies in LDS behind their pieces, which no copy writes, is zero, as the rows' elements there are (a piece of the key again would make
// NaN of an infinity in it).  Such heads have kernels of their own (FULL: none of a key's pieces is missing): lanes told apart in each copy cost 500 slots 2 of
// 11 us, a branch between two kinds of copies 1.  By `threads` of them, before the first copies; the caller waits.
__device__ __forceinline__ void attn_clear(char* to, int bytes, int tid, int threads) {
    for (int i = tid * 16; i < bytes; i += threads * 16) *reinterpret_cast<u32x4*>(to + i) = u32x4{0u, 0u, 0u, 0u};
}

// The pages of a wave's keys: 64 table entries at a time in a register, and the place of each of up to 32 keys
struct AttnPages {
    int window = -1;             // first page of the entries, -1: none
    int entries;
    int id, off;                 // lane l: of key l % N of the keys looked up last
    bool bad = false;
};

template <int N>
__device__ __forceinline__ void attn_lookup(const AttnArgs& a, const AttnSeq& s, int b, int first, int lane, AttnPages& p) {
    const int key = min(first + (lane & (N - 1)), s.total - 1);
    const int pg = (int)((uint32_t)key / (uint32_t)a.page);
    p.off = key - pg * a.page;
    const int lo = __builtin_amdgcn_readfirstlane(pg), hi = __builtin_amdgcn_readlane(pg, N - 1);
    if (p.window < 0 || lo < p.window || hi >= p.window + 64) {
        p.window = lo;
        p.entries = lo + lane < a.max_pages ? a.table[(int64_t)b * a.ld_table + lo + lane] : 0;
    }
    int id = __builtin_amdgcn_ds_bpermute((pg - p.window) * 4, p.entries);
    if ((uint32_t)id >= (uint32_t)a.pages) id = 0, p.bad = true;
    p.id = id;
}

// Copies the N keys (or values) looked up, from `first` on, of one head to `to`: `base` is the head's first byte of the pool.  at: the first one's
// place in its step
template <int DP, bool FULL, bool VALUES, int N>
__device__ __forceinline__ void attn_copy(const AttnArgs& a, const AttnSeq& s, int first, int place, int lane, const AttnPages& p, const char* base, const char* to) {
    typedef AttnTile<DP> T;
    static_assert(N % T::ROWS == 0, "whole copies");
    const int64_t page_b = VALUES ? a.v_page : a.k_page, slot_b = VALUES ? a.v_slot : a.k_slot;
    const int row = lane / T::PIECES, pos = lane % T::PIECES, pieces = a.dim >> 3;
    const uint32_t lds = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(lds_ptr)to);
    auto piece = [&](int j) { const int key = place + j * T::ROWS + row; return pos ^ (VALUES ? T::v_xor(key) : T::k_xor(key)); };
    if (a.near && a.page % T::ROWS == 0 && first + N <= s.total) {          // the keys of a copy lie in one page
#pragma unroll
        for (int j = 0; j < N / T::ROWS; ++j) {
            const int id = __builtin_amdgcn_readlane(p.id, j * T::ROWS), off = __builtin_amdgcn_readlane(p.off, j * T::ROWS), c = piece(j);
            if (FULL || c < pieces) attn_copy16(lds + j * 1024, base + id * page_b + off * slot_b, (uint32_t)(row * (int)slot_b + c * 16));
        }
    } else {
#pragma unroll
        for (int j = 0; j < N / T::ROWS; ++j) {
            const int id = __shfl(p.id, j * T::ROWS + row), off = __shfl(p.off, j * T::ROWS + row), c = piece(j);
            if (FULL || c < pieces) attn_copy16(lds + j * 1024, base + id * page_b + off * slot_b + c * 16);
        }
    }
}

// The same where groups of keys that follow each other lie in one page and the slots of a page near each other: the place of the next group is walked to,
// and everything but a lane's own offset is worked out once for the wave (with the above a step of 32 keys took 1.8 us of a wave's time, most
// of it on addresses).
struct AttnPlace { int64_t k, v; };          // a group's first key and value, bytes from the head's first
struct AttnWalk {
    int pg, off;
    __device__ __forceinline__ void begin(const AttnArgs& a, int key) { pg = (int)((uint32_t)key / (uint32_t)a.page); off = key - pg * a.page; }
    __device__ __forceinline__ void go(const AttnArgs& a, int pages, int slots) {      // pages * page + slots keys on, slots < page
        pg += pages;
        off += slots;
        if (off >= a.page) { off -= a.page; ++pg; }
    }
    __device__ __forceinline__ AttnPlace find(const AttnArgs& a, int b, int lane, AttnPages& p) const {
        if (p.window < 0 || pg < p.window || pg >= p.window + 64) {
            p.window = pg;
            p.entries = pg + lane < a.max_pages ? a.table[(int64_t)b * a.ld_table + pg + lane] : 0;
        }
        int id = __builtin_amdgcn_readlane(p.entries, pg - p.window);
        if ((uint32_t)id >= (uint32_t)a.pages) id = 0, p.bad = true;
        return {id * a.k_page + (uint32_t)(off * (int)a.k_slot), id * a.v_page + (uint32_t)(off * (int)a.v_slot)};
    }
};

// Copies N keys (values) of one group; where: the first one's place in its step
template <int DP, bool FULL, bool VALUES, int N>
__device__ __forceinline__ void attn_copy_group(const AttnArgs& a, int where, int lane, const char* from, const char* to) {
    typedef AttnTile<DP> T;
    static_assert(N % T::ROWS == 0, "whole copies");
    const int row = lane / T::PIECES, pos = lane % T::PIECES, pieces = a.dim >> 3, slot_b = (int)(VALUES ? a.v_slot : a.k_slot);
    const uint32_t lds = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(lds_ptr)to);
#pragma unroll
    for (int j = 0; j < N / T::ROWS; ++j) {
        const int key = where + j * T::ROWS + row, c = pos ^ (VALUES ? T::v_xor(key) : T::k_xor(key));
        if (FULL || c < pieces) attn_copy16(lds + j * 1024, from, (uint32_t)((j * T::ROWS + row) * slot_b + c * 16));
    }
}

// ------------------------------------------------------------------------------------------ a cache held in 8 bits (sq_tree_attention8)

// Keys and values as e4m3 codes with a power of two for each block of tokens and head.  Strides of the cache are its bytes.
struct Attn8Args : AttnArgs {
    const uint8_t *ks, *vs;
    int64_t ks_page, ks_block, ks_head, vs_page, vs_block, vs_head;
    int size;                    // tokens of a block, a multiple of 16
    int inner;                   // few rows: workgroups that read the same lines (blocks of rows; heads that share lines), dealt to one die one behind the other
    int passing;                 // few rows: keys and values are read past the caches
};
// many rows: the blocks of rows of all sequences share the workgroups of a key head by how many keys they see
struct Attn8Shared : Attn8Args {
    int32_t* parts;              // of each block of rows and sequence: into how many its keys are cut; `splits` is the most
    int block;                   // rows of a block are 2^block
};

// 8 codes times a power of two as a matrix instruction's operand: v_cvt_scalef32_pk takes two at a time and the scale with them, exactly
template <int DT> __device__ __forceinline__ u32x4 attn8_unpack(uint32_t x, uint32_t y, float sx, float sy) {
    if constexpr (DT == SQ_F16)
        return u32x4{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x, sx, false)), __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x, sx, true)),
                     __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(y, sy, false)), __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(y, sy, true))};
    else
        return u32x4{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, sx, false)), __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, sx, true)),
                     __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(y, sy, false)), __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(y, sy, true))};
}
__device__ __forceinline__ float attn8_scale(uint32_t byte) { return __builtin_bit_cast(float, byte << 23); }

// Where 64 groups of keys lie that a wave copies one after the other (lane l: the l-th, `step` keys after the one before), and their scales.  A group's keys are in
// one block, so in one page.  Groups from key `limit` on: the first page, whose slots and scales may be read as well.
struct Attn8Groups {
    int64_t k, v;                // bytes from the head's first
    const uint8_t *ks, *vs;
    bool bad = false;

    __device__ __forceinline__ void find(const Attn8Args& a, int b, int head, int key, int step, int limit, int lane) {
        const int64_t at = key + (int64_t)lane * step;
        int id = 0, off = 0;
        if (at < limit) {
            const int pg = (int)((uint32_t)at / (uint32_t)a.page);
            off = (int)at - pg * a.page;
            id = a.table[(int64_t)b * a.ld_table + pg];
            if ((uint32_t)id >= (uint32_t)a.pages) bad = true, id = 0, off = 0;
        }
        const int block = off / a.size;
        k = id * a.k_page + off * a.k_slot;
        v = id * a.v_page + off * a.v_slot;
        ks = a.ks + id * a.ks_page + block * a.ks_block + head * a.ks_head;
        vs = a.vs + id * a.vs_page + block * a.vs_block + head * a.vs_head;
    }
    static __device__ __forceinline__ int64_t lane64(int64_t x, int l) {
        return (int64_t)(uint32_t)__builtin_amdgcn_readlane((int)x, l) | (int64_t)__builtin_amdgcn_readlane((int)(x >> 32), l) << 32;
    }
};

// What a wave keeps of its MT * 16 rows
template <int DP, int MT> struct AttnRows {
    u32x4 q[MT][DP / 32];
    float4v o[MT][DP / 16];      // lane l: row l % 16, elements 16 * i + 4 * (l / 16) .. + 3
    float m[MT], l[MT];          // what is taken off the row's exponents (some maximum times scale2, less SHIFT), this lane's part of the total
    int tok[MT];                 // new token of the row
    bool far;                    // some maximum is none yet, or beyond 2^20 (the same for the wave)

    __device__ __forceinline__ AttnRows<DP, 1> tile(int t) const {
        AttnRows<DP, 1> x;
        for (int c = 0; c < DP / 32; ++c) x.q[0][c] = q[t][c];
        for (int d = 0; d < DP / 16; ++d) x.o[0][d] = o[t][d];
        x.m[0] = m[t]; x.l[0] = l[t]; x.tok[0] = tok[t]; x.far = true;
        return x;
    }
    __device__ __forceinline__ void put(int t, const AttnRows<DP, 1>& x) {
        for (int d = 0; d < DP / 16; ++d) o[t][d] = x.o[0][d];
        m[t] = x.m[0]; l[t] = x.l[0];
    }
};

// (PAIRS: an operand of keys is 8 of the 16 elements that a lane reads of a key at once, the next one the others)
template <int DP, int MT, bool PAIRS = false>
__device__ __forceinline__ void attn_rows_begin(const AttnArgs& a, const AttnSeq& s, int head, int row0, int lane, AttnRows<DP, MT>& r) {
    const int rows = s.n * a.group;
    r.far = true;
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        const int row = min(row0 + t * 16 + (lane & 15), rows - 1), tok = row / a.group;
        const char* q = a.q + (int64_t)(s.first + tok) * a.q_t + (int64_t)(head * a.group + row - tok * a.group) * a.q_h;
        r.tok[t] = tok;
        r.m[t] = ATTN_NOTHING;
        r.l[t] = 0.f;
#pragma unroll
        for (int c = 0; c < DP / 32; ++c) {
            const int e = PAIRS ? (c >> 1) * 64 + (lane >> 4) * 16 + (c & 1) * 8 : c * 32 + (lane >> 4) * 8;
            r.q[t][c] = e < a.dim ? *reinterpret_cast<const u32x4*>(q + e * 2) : u32x4{0u, 0u, 0u, 0u};
        }
#pragma unroll
        for (int i = 0; i < DP / 16; ++i) r.o[t][i] = float4v{0.f, 0.f, 0.f, 0.f};
    }
}

// The rows' loads waited for, behind the first copies: with the table's entries, which those wait for anyway.  (Not at all, the loop over the keys would wait for them, and so
// for all that is in flight, in every step.)
template <int DP, int MT> __device__ __forceinline__ void attn_rows_ready(AttnRows<DP, MT>& r) {
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int c = 0; c < DP / 32; ++c) asm volatile("" : "+v"(r.q[t][c]));
}

// Which of a step's 32 keys a row sees
__device__ __forceinline__ uint32_t attn_sees(const AttnArgs& a, const AttnSeq& s, int step, int tok) {
    const int base = step * ATTN_STEP;
    auto below = [&](int n) { return n >= 32 ? ~0u : n <= 0 ? 0u : (1u << n) - 1u; };         // keys base .. base + n - 1
    const uint32_t there = below(s.total - base);
    if (!a.mask) return there & below(s.len - base + tok + 1);
    const int j = base - s.len;                              // new token of the step's first key
    if (j <= -32) return there;
    const int64_t* words = a.mask + (int64_t)(s.first + tok) * a.ld_mask;
    auto word = [&](int i) { return i < a.mask_words ? (uint64_t)words[i] : 0ull; };
    if (j < 0) return there & ((uint32_t)(word(0) << -j) | below(-j));
    const int i = j >> 6, sh = j & 63;
    uint64_t w = word(i) >> sh;
    if (sh > 32) w |= word(i + 1) << (64 - sh);
    return there & (uint32_t)w;
}

// scores of a step: keys at k
template <int DT, int DP, int MT>
__device__ __forceinline__ void attn_scores(const AttnRows<DP, MT>& r, const char* k, int lane, float4v (&st)[MT][2]) {
    typedef AttnTile<DP> T;
    const int g = lane >> 4, i16 = lane & 15;
#pragma unroll
    for (int t = 0; t < MT; ++t) st[t][0] = st[t][1] = float4v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int c = 0; c < DP / 32; ++c)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const u32x4 f = *reinterpret_cast<const u32x4*>(k + (h * 16 + i16) * T::PITCH + (((c * 4 + g) ^ T::k_xor(h * 16 + i16)) * 16));
#pragma unroll
            for (int t = 0; t < MT; ++t) st[t][h] = AttnType<DT>::mfma(f, r.q[t][c], st[t][h]);
        }
}

// softmax weights of a step from its scores; the rows' maxima, totals and sums brought up to date.  sees: where MASKED.
// What is taken off the exponents need not be the maximum itself: it is raised when a weight would be more than 2^ATTN_SLACK times the one it stands for, so that most steps
// neither fold their maxima over lanes nor scale the sums; weights stay below 2^(SHIFT + ATTN_SLACK), inside fp16 too.
template <int DT, int DP, int MT, bool MASKED>
__device__ __forceinline__ void attn_weights(const AttnArgs& a, AttnRows<DP, MT>& r, float4v (&st)[MT][2], const uint32_t (&sees)[MT], int lane, u32x4 (&p)[MT]) {
    const int g = lane >> 4;
    float mx[MT];
    bool up = false;
    if constexpr (MASKED)
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int i = 0; i < 4; ++i) st[t][h][i] = (sees[t] >> (h * 16 + g * 4 + i)) & 1 ? st[t][h][i] : -INFINITY;
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        mx[t] = fmaxf(fmaxf(fmaxf(st[t][0][0], st[t][0][1]), fmaxf(st[t][0][2], st[t][0][3])), fmaxf(fmaxf(st[t][1][0], st[t][1][1]), fmaxf(st[t][1][2], st[t][1][3])));
        up |= attn_above<DT>(mx[t], a.scale2, r.m[t]);
    }
    if (__any(up)) {
        bool far = false;
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            // (row by row, so that no row's bits depend on what the wave's other rows see)
            const float top = groups_fold(mx[t], [](float x, float y) { return fmaxf(x, y); });
            const float m = attn_above<DT>(top, a.scale2, r.m[t]) ? attn_rounded<DT>(top, a.scale2) - AttnType<DT>::SHIFT : r.m[t], by = __builtin_amdgcn_exp2f(r.m[t] - m);
            r.m[t] = m;
            r.l[t] *= by;
            far |= !(fabsf(m) <= 0x1p20f);
#pragma unroll
            for (int i = 0; i < DP / 16; ++i) r.o[t][i] *= by;
        }
        r.far = __any(far);
    }
    // The exponent in one operation, exact but for its rounding, where the rounding of what is taken off is of no account (a factor of 2^(1/16) of all
    // weights at most); of larger maxima it could reach past the largest float, so there a rounded product less the maximum, zero at it.
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        float m = r.m[t], by = a.scale2;
        if (r.far && !(fabsf(m) <= 0x1p20f)) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                float x = st[t][i >> 2][i & 3] * a.scale2;
                asm("" : "+v"(x));                           // (not one operation again)
                st[t][i >> 2][i & 3] = x - m;
            }
            m = 0.f; by = 1.f;
        }
        float e[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) e[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(st[t][i >> 2][i & 3], by, -m));
        r.l[t] += ((e[0] + e[1]) + (e[2] + e[3])) + ((e[4] + e[5]) + (e[6] + e[7]));
#pragma unroll
        for (int i = 0; i < 4; ++i) p[t][i] = AttnType<DT>::pack(e[2 * i], e[2 * i + 1]);
    }
}

// sums of a step: values at v.  Where MASKED, values that are not finite do not go through the product, whose zero weights would make NaN of
// them in rows that do not see their keys: such elements are set to zero, the rows' keys that hold them are counted by products of zeros and ones,
// and rows that see one get what it makes of their sum (an infinity, or NaN).
template <int DT, int DP, int MT, bool MASKED>
__device__ __forceinline__ void attn_sums(AttnRows<DP, MT>& r, const char* v, int lane, const u32x4 (&p)[MT], const uint32_t (&sees)[MT]) {
    typedef AttnTile<DP> T;
    typedef AttnType<DT> E;
    typedef short short4v __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) short4v* tr_ptr;
    const int g = lane >> 4, i16 = lane & 15, key = 4 * g + (i16 >> 2);
    auto read = [&](int d) {
        u32x4 f;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const char* at = v + (h * 16 + key) * T::PITCH + (((d * 2 + ((i16 & 3) >> 1)) ^ T::v_xor(h * 16 + key)) * 16) + (i16 & 1) * 8;
            const u32x2 w = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((tr_ptr)(lds_ptr)at));
            f[2 * h] = w[0];
            f[2 * h + 1] = w[1];
        }
        return f;
    };
    if constexpr (!MASKED) {
#pragma unroll
        for (int d = 0; d < DP / 16; ++d) {
            const u32x4 f = read(d);
#pragma unroll
            for (int t = 0; t < MT; ++t) r.o[t][d] = E::mfma(f, p[t], r.o[t][d]);
        }
        return;
    }
    // (looked for in all values of a few operands at once, two per instruction: an exponent of all ones carries into the sign's place.  One by one they
    // took a step of 16 rows a microsecond.)
    constexpr int CHUNK = 4;
#pragma unroll
    for (int d0 = 0; d0 < DP / 16; d0 += CHUNK) {
        u32x4 f[CHUNK];
        uint32_t odd = 0;
#pragma unroll
        for (int x = 0; x < CHUNK; ++x) {
            f[x] = read(d0 + x);
#pragma unroll
            for (int i = 0; i < 4; ++i) odd |= (f[x][i] & 0x7FFF7FFFu) + (0x8000u - E::INF) * 0x10001u;
        }
        if (__any((odd & 0x80008000u) != 0)) {
#pragma unroll
            for (int x = 0; x < CHUNK; ++x) {
                u32x4 up, down;                              // ones where a value is not below +inf, not above -inf
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    uint32_t clean = 0, u = 0, n = 0;
#pragma unroll
                    for (int y = 0; y < 2; ++y) {
                        const uint32_t bits = (f[x][i] >> (16 * y)) & 0xFFFF;
                        const bool nan = (bits & 0x7FFF) > E::INF, inf = (bits & 0x7FFF) == E::INF;
                        if (!nan && !inf) clean |= bits << (16 * y);
                        if (nan || (inf && !(bits & 0x8000))) u |= E::ONE << (16 * y);
                        if (nan || (inf && (bits & 0x8000))) n |= E::ONE << (16 * y);
                    }
                    f[x][i] = clean; up[i] = u; down[i] = n;
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
                        if (cu[i] > 0.f) r.o[t][d0 + x][i] += INFINITY;
                        if (cd[i] > 0.f) r.o[t][d0 + x][i] -= INFINITY;
                    }
                }
            }
        }
#pragma unroll
        for (int x = 0; x < CHUNK; ++x)
#pragma unroll
            for (int t = 0; t < MT; ++t) r.o[t][d0 + x] = E::mfma(f[x], p[t], r.o[t][d0 + x]);
    }
}

// Joined and written: `parts` waves' sums of the same rows (each as parts x ROWS x PITCH floats in LDS), maxima and totals
template <int DT, int DP>
__device__ __forceinline__ void attn_write(const AttnArgs& a, const AttnSeq& s, int head, int row0, int rows_here, int split, const float* sums, const float2v* ml, int parts,
                                           int ml_pitch, bool bad, int tid, int threads) {
    constexpr int PITCH = DP + 4;
    const int rows = min(s.n * a.group - row0, rows_here);
    for (int i = tid; i < rows * (DP / 8); i += threads) {
        const int row = i / (DP / 8), e = i % (DP / 8) * 8, all = row0 + row, tok = all / a.group, hq = head * a.group + all - tok * a.group;
        float m = ATTN_NOTHING, l = 0.f;
        for (int w = 0; w < parts; ++w) m = fmaxf(m, ml[w * ml_pitch + row][0]);
        float v[8];
#pragma unroll
        for (int x = 0; x < 8; ++x) v[x] = 0.f;
        for (int w = 0; w < parts; ++w) {
            const float2v one = ml[w * ml_pitch + row];
            const float by = __builtin_amdgcn_exp2f(one[0] - m);
            l += one[1] * by;
            if (by == 0.f) continue;
            const float4v* from = reinterpret_cast<const float4v*>(sums + (size_t)(w * rows_here + row) * PITCH + e);
            const float4v x0 = from[0], x1 = from[1];
#pragma unroll
            for (int x = 0; x < 4; ++x) { v[x] = __builtin_fmaf(x0[x], by, v[x]); v[4 + x] = __builtin_fmaf(x1[x], by, v[4 + x]); }
        }
        if (bad) l = NAN;
        const int64_t tok_all = s.first + tok;
        if (a.splits > 1) {
            const int64_t at = (tok_all * a.q_heads + hq) * a.splits + split;
            float4v* to = reinterpret_cast<float4v*>(a.po + at * DP + e);
            to[0] = float4v{v[0], v[1], v[2], v[3]};
            to[1] = float4v{v[4], v[5], v[6], v[7]};
            if (e == 0) a.pml[at] = float2v{m, l};
            continue;
        }
        const float inv = l == 0.f ? 0.f : 1.f / l;
        if (e < a.dim) {
            u32x4 o;
#pragma unroll
            for (int x = 0; x < 4; ++x) o[x] = (uint32_t)AttnType<DT>::one(v[2 * x] * inv) | ((uint32_t)AttnType<DT>::one(v[2 * x + 1] * inv) << 16);
            *reinterpret_cast<u32x4*>(a.out + tok_all * a.o_t + (int64_t)hq * a.o_h + e * 2) = o;
        }
        if (e == 0 && a.lse) a.lse[tok_all * a.q_heads + hq] = attn_lse<DT>(m, l);
    }
}

template <int DP, int MT, int NW> constexpr int attn_lds() {
    constexpr int ring = NW * 4 * AttnTile<DP>::BYTES, join = NW * MT * 16 * ((DP + 4) * 4 + 8) + 64;
    return ring > join ? ring : join;
}

// Few rows (MT * 16 at a time): the waves of a workgroup share the rows and split its keys, each with two steps of keys and values of its
// own in LDS, no barrier until the end, where their sums are joined.  Sequences are cut into `splits` workgroups too.  Bound by HBM on long caches (32 sequences of
// 2,240 to 8,192 slots, 8 key heads of 128, 5 query heads each: 123 us, 5.6 TB/s; 64 of 8192 364 us, 5.9 TB/s), by its chain of loads on short ones (500 slots 7 us).
template <int DT, int DP, int MT, int NW, bool FULL>
__global__ __launch_bounds__(NW * 64) __attribute__((amdgpu_waves_per_eu(1, 1))) void attn_kernel(AttnArgs a) {
    typedef AttnTile<DP> T;
    extern __shared__ __attribute__((aligned(1024))) char smem[];
    constexpr int C = T::COPIES, ROWS = MT * 16;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    int id = blockIdx.x;
    const int split = id % a.splits; id /= a.splits;
    const int head = id % a.kv_heads; id /= a.kv_heads;
    const int row0 = id % a.row_blocks * ROWS, b = id / a.row_blocks;
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
    attn_rows_begin<DP, MT>(a, s, head, row0, lane, r);
    AttnPages pages;
    const char *kb = a.kc + head * a.k_head, *vb = a.vc + head * a.v_head;
    char* ring = smem + wave * (4 * T::BYTES);
    auto slot_k = [&](int i) { return ring + (i & 1) * T::BYTES; };
    auto slot_v = [&](int i) { return ring + (2 + (i & 1)) * T::BYTES; };
    // (pages of whole groups of 16: a step is two groups, each in one page)
    const bool easy = a.near && a.page % 16 == 0;
    AttnWalk walk;
    walk.begin(a, w0 * ATTN_STEP);
    AttnPlace at[2];
    auto get_k = [&](int i) __attribute__((always_inline)) {
        if (easy && (i + 1) * ATTN_STEP <= s.total) {
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                at[x] = walk.find(a, b, lane, pages);
                attn_copy_group<DP, FULL, false, 16>(a, 16 * x, lane, kb + at[x].k, slot_k(i) + x * 16 * T::PITCH);
                walk.go(a, 16 / a.page, 16 % a.page);
            }
            return;
        }
        attn_lookup<ATTN_STEP>(a, s, b, i * ATTN_STEP, lane, pages);
        attn_copy<DP, FULL, false, ATTN_STEP>(a, s, i * ATTN_STEP, 0, lane, pages, kb, slot_k(i));
    };
    auto get_v = [&](int i) __attribute__((always_inline)) {
        if (easy && (i + 1) * ATTN_STEP <= s.total) {
#pragma unroll
            for (int x = 0; x < 2; ++x) attn_copy_group<DP, FULL, true, 16>(a, 16 * x, lane, vb + at[x].v, slot_v(i) + x * 16 * T::PITCH);
            return;
        }
        attn_copy<DP, FULL, true, ATTN_STEP>(a, s, i * ATTN_STEP, 0, lane, pages, vb, slot_v(i)); };
    if constexpr (!FULL) {
        attn_clear(ring, 4 * T::BYTES, lane, 64);
        attn_reads_done();
    }
    if (w0 < w1) { get_k(w0); get_v(w0); }
    if (w0 + 1 < w1) { get_k(w0 + 1); get_v(w0 + 1); }
    attn_rows_ready(r);
    auto step = [&](int i, auto masked) __attribute__((always_inline)) {
        constexpr bool MASKED = decltype(masked)::value;
        float4v st[MT][2];
        u32x4 p[MT];
        uint32_t sees[MT] = {};
        if (i + 1 < w1) attn_wait<3 * C>(); else attn_wait<C>();
        attn_scores<DT, DP, MT>(r, slot_k(i), lane, st);
        __builtin_amdgcn_sched_barrier(0);
        attn_reads_done();
        if (i + 2 < w1) get_k(i + 2);
        if constexpr (MASKED)
#pragma unroll
            for (int t = 0; t < MT; ++t) sees[t] = attn_sees(a, s, i, r.tok[t]);
        attn_weights<DT, DP, MT, MASKED>(a, r, st, sees, lane, p);
        if (i + 2 < w1) attn_wait<3 * C>(); else if (i + 1 < w1) attn_wait<2 * C>(); else attn_wait<0>();
        attn_sums<DT, DP, MT, MASKED>(r, slot_v(i), lane, p, sees);
        __builtin_amdgcn_sched_barrier(0);
        attn_reads_done();
        if (i + 2 < w1) get_v(i + 2);
    };
    // (two loops: one with a choice in it would keep two versions of the sums in registers)
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
    const bool bad = __any(pages.bad) || s.over;
    if (lane == 0) flags[wave] = bad;
    __syncthreads();
    bool any = false;
#pragma unroll
    for (int w = 0; w < NW; ++w) any |= flags[w] != 0;
    attn_write<DT, DP>(a, s, head, row0, ROWS, split, sums, ml, NW, ROWS, any, tid, NW * 64);
}

// ------------------------------------------------------------------------------------------ many rows

// Waves of a workgroup (8, or 4 for fewer rows), tiles of 16 rows of a wave, steps of 32 keys in a stage, stages in LDS
constexpr int attn_tiles(int dp) { return dp == 256 ? 1 : 2; }
constexpr int attn_stage_steps(int dp, int nw) { return dp == 256 || nw == 4 ? 1 : 2; }
constexpr int ATTN_STAGES = 4;
template <int DP, int NW> constexpr int attn_stage_bytes() { return attn_stage_steps(DP, NW) * 2 * AttnTile<DP>::BYTES; }
template <int DP, int NW> constexpr int attn_tile_lds() { return ATTN_STAGES * attn_stage_bytes<DP, NW>() + 64; }
// Over a cache held in 8 bits: stages of 16 bits in LDS, stages of codes on their way to them (each wave's own part, half as many bytes)
constexpr int ATTN8_STAGES = 3, ATTN8_RAW = 3;
template <int DP, int NW> constexpr int attn8_copies() { return (attn_stage_steps(DP, NW) * ATTN_STEP / NW * DP + 1023) / 1024; }      // of a wave's keys of a stage
template <int DP, int NW> constexpr int attn8_tile_lds() { return ATTN8_STAGES * attn_stage_bytes<DP, NW>() + ATTN8_RAW * NW * 2048 * attn8_copies<DP, NW>() + 64; }

// The blocks of rows of all sequences share the workgroups of a key head by their work, not evenly: with the least T such that all of them, cut into parts of T, are no more parts than
// there are workgroups.  Work is the stages that a block's rows see, of a block that fills half of its waves or less 0.6 of them.  Workgroup `which` becomes part `split` of `splits` of one.
// (Lengths are on the device; up to 64 blocks, one a lane.)
// 8 trees of 48 tokens behind 1408 to 4096 slots, 28 + 4 heads of 128: 52.2 us in as many parts each, 45.3 so, of 20 + 4 heads of 256 67.1 and 57.8 (61 with END zero); 4 x 200 behind 1000 to
// 4000 84.4 and 73.5; 1500 tokens behind 2100 120 and 109, 1000 of 20 + 4 heads of 256 147 and 132; 8 trees of one length 51.9 and 53.2.
template <typename F> __device__ __forceinline__ uint32_t attn8_fold(uint32_t v, F f) {          // over the wave
    const auto h = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    v = f((uint32_t)h[0], (uint32_t)h[1]);
    const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = f((uint32_t)r[0], (uint32_t)r[1]);
    v = f(v, row_rotated_bits<8>(v));
    v = f(v, row_rotated_bits<4>(v));
    v = f(v, row_rotated_bits<2>(v));
    return (uint32_t)__builtin_amdgcn_readfirstlane((int)f(v, row_rotated_bits<1>(v)));
}
template <int N> __device__ __forceinline__ int attn8_from_left(int v) { return __builtin_amdgcn_update_dpp(0, v, 0x110 + N, 0xF, 0xF, false); }      // of the lane N before, in a row of 16
// x / d rounded up, for x up to 2^21 (a 32-bit float tells it from the integers beside it), in a fifth of the instructions of a division
__device__ __forceinline__ int attn8_parts(int x, int d, float by) {
    const int q = (int)((float)x * by);
    return q + (q * d < x);
}
template <int KEYS, int ROWS, int END>
__device__ __forceinline__ bool attn8_share(const Attn8Shared& a, int which, int all, int head, int lane, int& b, int& row0, int& split, int& splits, AttnSeq& seq) {
    auto sum = [](int v) __attribute__((always_inline)) { return (int)attn8_fold((uint32_t)v, [](uint32_t x, uint32_t y) { return x + y; }); };
    const int items = a.seqs * a.row_blocks, item = min(lane, items - 1), of = item / a.row_blocks, first = (a.row_blocks - 1 - (item - of * a.row_blocks)) * ROWS;
    const AttnSeq s = attn_seq(a, of);
    // (about how much: what a part has of it is worked out from the sequence itself)
    const int rows = s.n * a.group, here = min(rows - first, ROWS);
    const int seen = a.mask ? s.total : min(s.total, s.len + (int)((float)(first + here - 1) * __builtin_amdgcn_rcpf((float)a.group)) + 1);
    const int work = lane < items && here > 0 ? (max(seen + KEYS - 1, 0) / KEYS + END) * (2 * here <= ROWS ? 3 : 5) : 0;          // (never below zero: parts would be)
    const int most = (int)attn8_fold((uint32_t)work, [](uint32_t x, uint32_t y) { return max(x, y); });
    const float total = (float)sum(work);
    // (T = total / (all - items) is enough, since each block's last part may be short; fewer than two stages are not worth a part)
    int t = max(max((int)(total * __builtin_amdgcn_rcpf((float)all)), attn8_parts(most, a.splits, __builtin_amdgcn_rcpf((float)a.splits))), 10);
    int enough = max(t, min(most, (int)(total * __builtin_amdgcn_rcpf((float)(all - items))) + 2));
    while (t < enough) {
        const int half = (t + enough) / 2;
        if (sum(attn8_parts(work, half, __builtin_amdgcn_rcpf((float)half))) <= all) enough = half; else t = half + 1;
    }
    const int parts = attn8_parts(work, t, __builtin_amdgcn_rcpf((float)t));
    int upto = parts;
    upto += attn8_from_left<1>(upto);
    upto += attn8_from_left<2>(upto);
    upto += attn8_from_left<4>(upto);
    upto += attn8_from_left<8>(upto);
    const int r0 = __builtin_amdgcn_readlane(upto, 15), r1 = __builtin_amdgcn_readlane(upto, 31), r2 = __builtin_amdgcn_readlane(upto, 47);
    upto += lane < 16 ? 0 : lane < 32 ? r0 : lane < 48 ? r0 + r1 : r0 + r1 + r2;
    if (which == 0 && head == 0 && threadIdx.x < (unsigned)items) a.parts[first / ROWS * a.seqs + of] = parts;
    const uint64_t mine = __ballot(which >= upto - parts && which < upto);
    if (!mine) return false;
    const int l = __builtin_ctzll(mine);
    b = __builtin_amdgcn_readlane(of, l);
    row0 = __builtin_amdgcn_readlane(first, l);
    splits = __builtin_amdgcn_readlane(parts, l);
    split = which - __builtin_amdgcn_readlane(upto - parts, l);
    seq = {__builtin_amdgcn_readlane(s.first, l), __builtin_amdgcn_readlane(s.n, l), __builtin_amdgcn_readlane(s.len, l), __builtin_amdgcn_readlane(s.total, l),
           __builtin_amdgcn_readlane((int)s.over, l) != 0};
    return true;
}

// In which order a region's instructions are issued: N times one matrix instruction, D LDS reads, V vector instructions, X exponentials
template <int N, int V, int X, int D> __device__ __forceinline__ void attn_order() {
#pragma unroll
    for (int i = 0; i < N; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        if constexpr (D > 0) __builtin_amdgcn_sched_group_barrier(0x100, D, 0);
        if constexpr (V > 0) __builtin_amdgcn_sched_group_barrier(0x002, V, 0);
        if constexpr (X > 0) __builtin_amdgcn_sched_group_barrier(0x400, X, 0);
    }
}
// Largest of eight scores (fmaxf would make each quiet first: twice the instructions)
__device__ __forceinline__ float attn_most(float4v x, float4v y) {
    float m;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(m) : "v"(x[0]), "v"(x[1]), "v"(x[2]));
    asm("v_max3_f32 %0, %0, %1, %2" : "+v"(m) : "v"(x[3]), "v"(y[0]));
    asm("v_max3_f32 %0, %0, %1, %2" : "+v"(m) : "v"(y[1]), "v"(y[2]));
    return fmaxf(m, y[3]);
}
// Many rows: each wave has MT tiles of 16 rows of its own and all waves share the keys, a stage at a time.  One barrier per stage: behind it every wave's
// part of the stage has arrived, and all waves are done with the stage two before it, whose place takes the copies of the one that comes two later.
//
// A slot is one tile of one step: the products of its scores, the exponentials of the tile before it and the sums of the tile before that one, none of
// which waits for another.  Keys and values of a step stay in registers for its tiles, and each register is filled again, for the next
// step, right behind its last use.  Two waves per SIMD: with one of 48 rows (a third less to read from LDS) the compiler keeps the sums in the accumulation
// registers and moves them around the branch that scales them, 1300 cycles a slot instead of 500.  Bound by what a SIMD's two waves issue: matrix and other vector
// instructions hardly overlap (1900 tokens of 28 heads of 128 behind 2100, 4 key heads: 121 us, 686 TFLOP/s, matrix cores busy 44 % of the time).
// The stages at a sequence's end that some row does not see whole go step by step, behind the pipeline, and all of them (those that every row sees without masks) for
// heads wider than 128 elements, whose keys and values would take the registers of four tiles.  There a wave has one tile, so a key's pieces are read from LDS once per 16 rows: 256 KB a
// stage for eight waves, 2048 cycles at 128 bytes each, beside 1024 of matrix instructions (1000 tokens of 20 heads of 256 behind 2100: 133 us, 97 stages of some 3000 cycles).
// Over a cache held in 8 bits (Attn8Args) each wave copies its part of a stage as codes to a place of its own, and unpacks it into the stage, scaled,
// before the barrier that lets all waves read it; all that follows is the same.
template <int DT, int DP, int NW, bool FULL, typename ARGS = AttnArgs>
__global__ __launch_bounds__(NW * 64, 2) void attn_tile_kernel(ARGS a) {
    typedef AttnTile<DP> T;
    typedef AttnType<DT> E;
    typedef short short4v __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) short4v* tr_ptr;
    extern __shared__ __attribute__((aligned(1024))) char smem[];
    constexpr bool C8 = !std::is_same_v<ARGS, AttnArgs>, SHARED = std::is_same_v<ARGS, Attn8Shared>;
    constexpr int MT = attn_tiles(DP), SK = attn_stage_steps(DP, NW), KEYS = SK * ATTN_STEP, NB = C8 ? ATTN8_STAGES : ATTN_STAGES, STAGE = attn_stage_bytes<DP, NW>(), ROWS = NW * MT * 16;
    constexpr int MINE = KEYS / NW, C = MINE / T::ROWS, KC = DP / 32, VD = DP / 16;
    constexpr int END = SHARED && MT < 2 ? 2 : 0;                // (stages that a sequence's end, which goes step by step, costs beside its own)
    constexpr bool PIPELINE = MT >= 2;                       // (a tile's maximum is raised while the sums of the tile before it are outstanding)
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 4, i16 = lane & 15;
    // the workgroups of one key head are dealt to as few dies as there are: neighbours are other heads'; last rows, which have most keys, first
    int id = blockIdx.x, head, b, row0, split, splits;
    AttnSeq s;
    if constexpr (SHARED) {
        head = id % a.kv_heads;
        if (!attn8_share<KEYS, ROWS, END>(a, id / a.kv_heads, gridDim.x / a.kv_heads, head, lane, b, row0, split, splits, s)) return;
    } else {
        const int groups = a.seqs * a.kv_heads;
        b = id % groups / a.kv_heads;
        head = id % groups % a.kv_heads;
        id /= groups;
        const bool end_block = id < a.last_splits;
        splits = end_block ? a.last_splits : a.splits;
        if (!end_block) id -= a.last_splits;
        split = id % splits;
        row0 = (a.row_blocks - (end_block ? 1 : 2) - id / splits) * ROWS;
        s = attn_seq(a, b);
    }
    const int rows = s.n * a.group;
    if (row0 >= rows) return;
    const int last = min(row0 + ROWS, rows) - 1;
    const int seen = a.mask ? s.total : min(s.total, s.len + last / a.group + 1);
    const int stages = (seen + KEYS - 1) / KEYS, per = (stages + END + splits - 1) / splits, begin = min(split * per, stages), end = min(begin + per, stages);

    AttnRows<DP, MT> r;
    const int mine = row0 + wave * MT * 16;
    attn_rows_begin<DP, MT>(a, s, head, mine, lane, r);
    const int from = min(mine, rows - 1) / a.group, to = min(mine + MT * 16, rows) - 1;
    const int whole = a.mask ? min(s.len, s.total) : min(s.total, s.len + from + 1);                  // keys that all of the wave's rows see
    const int some = mine >= rows ? 0 : a.mask ? s.total : min(s.total, s.len + to / a.group + 1);    // and that any does
    const int clear = !PIPELINE || mine >= rows ? begin : min(max(whole / KEYS, begin), end);
    AttnPages pages;
    const char *kb = a.kc + head * a.k_head, *vb = a.vc + head * a.v_head;
    const bool easy = a.near && a.page % MINE == 0;
    AttnWalk walk;
    walk.begin(a, begin * KEYS + wave * MINE);
    Attn8Groups held;                                        // of stages `window` on, and their scales
    int window = 1 << 30;
    uint32_t scales = 0;
    uint64_t coming = 0;                                     // scales of the stages on their way, 16 bits each, the newest on top
    constexpr int C8N = attn8_copies<DP, NW>(), RAW = 2048 * C8N, P8 = DP / 16, ROWS8 = 64 / P8;          // (16-byte pieces of a key's codes, keys per copy)
    char* raw = smem + NB * STAGE + 64 + wave * (ATTN8_RAW * RAW);
    // where a lane's codes go in a stage: their first 8 elements of keys, of values in the upper half (the other 8: 16 bytes on or back).  Held in one register each, because
    // there are none to spare for what they are worked out from, which took more instructions than the unpacking.
    uint32_t goes[C8N];
    if constexpr (C8)
#pragma unroll
        for (int j = 0; j < C8N; ++j) {
            const int row = wave * MINE + j * ROWS8 + lane / P8, key = row % ATTN_STEP, two = 2 * (lane % P8);
            goes[j] = (row * T::PITCH + (two ^ T::k_xor(key)) * 16) | (SK * T::BYTES + row * T::PITCH + (two ^ T::v_xor(key)) * 16) << 16;
            asm volatile("" : "+v"(goes[j]));
        }
    auto place = [&](int i) __attribute__((always_inline)) { return smem + (i - begin) % NB * STAGE; };      // keys of SK steps, values of SK steps
    auto get = [&](int i) __attribute__((always_inline)) {           // this wave copies keys wave * MINE .. of a stage
        if constexpr (C8) {
            const int piece = lane % P8;
            if (i < window || i >= window + 64) {
                held.find(a, b, head, i * KEYS + wave * MINE, KEYS, min(s.total, end * KEYS), lane);
                scales = *held.ks | (uint32_t)*held.vs << 8;
                window = i;
            }
            const uint32_t to = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(lds_ptr)(raw + (i - begin) % ATTN8_RAW * RAW));
            const int64_t k_at = held.lane64(held.k, i - window), v_at = held.lane64(held.v, i - window);
#pragma unroll
            for (int j = 0; j < C8N; ++j) {
                const int row = j * ROWS8 + lane / P8;
                if (row < MINE && (FULL || piece < a.dim >> 4)) {
                    attn_copy16(to + j * 1024, kb + k_at, (uint32_t)(row * (int)a.k_slot + piece * 16));
                    attn_copy16(to + RAW / 2 + j * 1024, vb + v_at, (uint32_t)(row * (int)a.v_slot + piece * 16));
                }
            }
            coming = coming >> 16 | (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)scales, i - window) << (16 * (ATTN8_RAW - 1));
            return;
        }
        char* at = place(i) + wave * MINE * T::PITCH;
        const int first = i * KEYS + wave * MINE, in_step = wave * MINE % ATTN_STEP;
        if (easy && first + MINE <= s.total) {
            const AttnPlace from = walk.find(a, b, lane, pages);
            attn_copy_group<DP, FULL, false, MINE>(a, in_step, lane, kb + from.k, at);
            attn_copy_group<DP, FULL, true, MINE>(a, in_step, lane, vb + from.v, at + SK * T::BYTES);
            walk.go(a, KEYS / a.page, KEYS % a.page);
            return;
        }
        attn_lookup<MINE>(a, s, b, first, lane, pages);
        attn_copy<DP, FULL, false, MINE>(a, s, first, in_step, lane, pages, kb, at);
        attn_copy<DP, FULL, true, MINE>(a, s, first, in_step, lane, pages, vb, at + SK * T::BYTES);
    };
    // C8: this wave's part of stage i unpacked.  Once for each stage, in order, behind the barrier of the stage before it: the stage's place is that of the one three before it, which
    // no wave reads from then on.
    auto unpack = [&](int i) __attribute__((always_inline)) {
        if constexpr (C8) {
            const int ahead = ATTN8_RAW - min(end - i, ATTN8_RAW);      // (its place in `coming`)
            if (i + ATTN8_RAW <= end) attn_wait<2 * C8N * (ATTN8_RAW - 1)>(); else attn_wait<0>();
            const uint32_t sc = (uint32_t)(coming >> (16 * ahead));
#pragma unroll
            for (int j = 0; j < C8N; ++j)
                if (j * ROWS8 + lane / P8 < MINE && (FULL || lane % P8 < a.dim >> 4)) {
                    const char* from = raw + (i - begin) % ATTN8_RAW * RAW + j * 1024 + lane * 16;
                    char* stage = place(i);
                    const u32x4 both[2] = {*reinterpret_cast<const u32x4*>(from), *reinterpret_cast<const u32x4*>(from + RAW / 2)};
#pragma unroll
                    for (int v = 0; v < 2; ++v) {
                        const u32x4 w = both[v];
                        const float by = attn8_scale(v ? sc >> 8 & 0xFF : sc & 0xFF);
                        const uint32_t to = v ? goes[j] >> 16 : goes[j] & 0xFFFF;
                        *reinterpret_cast<u32x4*>(stage + to) = attn8_unpack<DT>(w[0], w[1], by, by);
                        *reinterpret_cast<u32x4*>(stage + (to ^ 16)) = attn8_unpack<DT>(w[2], w[3], by, by);
                    }
                }
            // (its codes are read, all but the writes behind them done: the stage that comes three later takes their place)
            asm volatile("s_waitcnt lgkmcnt(%0)" ::"n"(4 * C8N) : "memory");
            if (i + ATTN8_RAW < end) get(i + ATTN8_RAW);
        }
    };
    auto arrive = [&](int i) __attribute__((always_inline)) {        // stage i is there
        if constexpr (C8) {
            attn_reads_done();
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
            return;
        }
        if (i + NB - 2 <= end) attn_wait<2 * C * (NB - 3)>(); else attn_wait<0>();
        attn_reads_done();
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        if (i + NB - 2 < end) get(i + NB - 2);
    };
    if constexpr (!FULL) {
        attn_clear(smem, NB * STAGE, tid, NW * 64);
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < (C8 ? ATTN8_RAW : NB - 2); ++i)
        if (begin + i < end) get(begin + i);
    attn_rows_ready(r);
    if constexpr (C8) if (begin < end) unpack(begin);

    if constexpr (PIPELINE) if (begin < clear) {
        // Where this lane reads in a step: of key l % 16 (the step's other half 16 keys behind) its first piece, of 4 keys their first elements (likewise).
        // A step begins at a multiple of a key's bytes, so the others are an XOR away from the step's own address: no registers for each.
        const uint32_t kat = i16 * T::PITCH + (g ^ T::k_xor(i16)) * 16;
        const uint32_t vat = (4 * g + (i16 >> 2)) * T::PITCH + (((i16 & 3) >> 1) ^ T::v_xor(4 * g + (i16 >> 2))) * 16 + (i16 & 1) * 8;
        typedef const __attribute__((address_space(3))) u32x4* k_ptr;
        auto lds = [](const char* at) __attribute__((always_inline)) { return (uint32_t)(uintptr_t)(lds_ptr)at; };
        auto read_k = [&](uint32_t step, int c, int h) __attribute__((always_inline)) { return *(k_ptr)(uintptr_t)(((step + kat) ^ (c * 64)) + h * 16 * T::PITCH); };
        auto read_v = [&](uint32_t step, int d) __attribute__((always_inline)) {
            const uint32_t at = (step + vat) ^ (d * 32);
            const u32x2 x = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((tr_ptr)(uintptr_t)at));
            const u32x2 y = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((tr_ptr)(uintptr_t)(at + 16 * T::PITCH)));
            return u32x4{x[0], x[1], y[0], y[1]};
        };
        u32x4 kf[KC][2], vf[VD], p = {0u, 0u, 0u, 0u};
        float4v now[2], was[2], old[2];                      // scores of a slot's tile, of the tile before and the one two before
        float e[8], by1 = a.scale2, less1 = 0.f, by2 = a.scale2, less2 = 0.f;         // exponents of the latter two: by * score - less
#pragma unroll
        for (int h = 0; h < 2; ++h) was[h] = old[h] = float4v{-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int i = 0; i < 8; ++i) e[i] = 0.f;
#pragma unroll
        for (int d = 0; d < VD; ++d) vf[d] = u32x4{0u, 0u, 0u, 0u};
        uint64_t far = ~0ull;                                // lanes with a maximum that is none yet, or beyond 2^20
        constexpr int HALF = 6;                              // exponentials of a tile beside the sums, the others beside the scores
        auto scores = [&](int t, auto last, uint32_t next) __attribute__((always_inline)) {    // last use of these keys: the next ones read behind it
            now[0] = now[1] = float4v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int c = 0; c < KC; ++c)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    now[h] = E::mfma(kf[c][h], r.q[t][c], now[h]);
                    if constexpr (decltype(last)::value) kf[c][h] = read_k(next, c, h);
                }
        };
        auto finish = [&](int t) __attribute__((always_inline)) {       // of the tile two before: the rest of its exponentials, its total and its weights
#pragma unroll
            for (int i = HALF; i < 8; ++i) e[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(old[i >> 2][i & 3], by2, -less2));
            r.l[t] += ((e[0] + e[1]) + (e[2] + e[3])) + ((e[4] + e[5]) + (e[6] + e[7]));
#pragma unroll
            for (int i = 0; i < 4; ++i) p[i] = E::pack(e[2 * i], e[2 * i + 1]);
        };
        auto raise = [&](int t, float mx) __attribute__((always_inline)) {      // of the tile before: its maximum against what is taken off
            by1 = a.scale2;
            less1 = r.m[t];
            // (one operation less than attn_above in fp16.  Rows beyond 2^20, where that is not enough, always come here; for others the second condition says nothing more)
            auto above = [&](float x) __attribute__((always_inline)) { return __builtin_fmaf(x, a.scale2, -(E::SHIFT + ATTN_SLACK)) > r.m[t]; };
            if ((__ballot(above(mx)) | far) != 0) {
                const float top = groups_fold(mx, [](float x, float y) { return fmaxf(x, y); }), x = attn_rounded<DT>(top, a.scale2);
                const bool up = above(top) || (DT == SQ_F16 && x - r.m[t] >= 16.f);
                const float m = up ? x - E::SHIFT : r.m[t], f = __builtin_amdgcn_exp2f(r.m[t] - m);
                r.m[t] = less1 = m;
                r.l[t] *= f;
#pragma unroll
                for (int d = 0; d < VD; ++d) r.o[t][d] *= f;
                far = 0;
#pragma unroll
                for (int i = 0; i < MT; ++i) far |= __ballot(!(fabsf(r.m[i]) <= 0x1p20f));
                if (!(fabsf(m) <= 0x1p20f)) {                // (see attn_weights)
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        float x = was[i >> 2][i & 3] * a.scale2;
                        asm("" : "+v"(x));
                        was[i >> 2][i & 3] = x - m;
                    }
                    by1 = 1.f;
                    less1 = 0.f;
                }
            }
        };
        auto sums = [&](int t, auto last, uint32_t next) __attribute__((always_inline)) {      // likewise
#pragma unroll
            for (int d = 0; d < VD; ++d) {
                r.o[t][d] = E::mfma(vf[d], p, r.o[t][d]);
                if constexpr (decltype(last)::value) vf[d] = read_v(next, d);
            }
        };
        auto half = [&]() __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < HALF; ++i) e[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(was[i >> 2][i & 3], by1, -less1));
        };
        auto most = [&]() __attribute__((always_inline)) { return attn_most(was[0], was[1]); };
        auto slot_end = [&]() __attribute__((always_inline)) {
#pragma unroll
            for (int h = 0; h < 2; ++h) { old[h] = was[h]; was[h] = now[h]; }
            by2 = by1;
            less2 = less1;
        };
        arrive(begin);
#pragma unroll
        for (int c = 0; c < KC; ++c)
#pragma unroll
            for (int h = 0; h < 2; ++h) kf[c][h] = read_k(lds(place(begin)), c, h);
        for (int i = begin; i < clear; ++i) {
            const uint32_t cur = lds(place(i)), nxt = lds(place(i + 1));
            auto slot = [&](auto number) __attribute__((always_inline)) {
                constexpr int n = decltype(number)::value, h = n / MT, t = n % MT, t1 = (t + MT - 1) % MT, t2 = (t + MT - 2) % MT;
                // (a SIMD's two waves at different times: 1900 tokens behind 2100 142 -> 136 us)
                if constexpr (C8) if (n == wave / 4 % 2 * (SK * MT / 2) && i + 1 < end) unpack(i + 1);
                if (n == SK * MT - 1 && i + 1 < clear) arrive(i + 1);
                __builtin_amdgcn_sched_barrier(0);
                // (behind the last stage of the pipeline: whatever lies in the next one's place, for nothing)
                __builtin_amdgcn_s_setprio(1);           // (a SIMD's other wave is then more often in another region: 1900 new tokens behind 2100 127 -> 121 us, 8 trees of 48 49.4 -> 47.6)
                scores(t, std::integral_constant<bool, t == MT - 1>(), h + 1 < SK ? cur + (h + 1) * T::BYTES : nxt);
                finish(t2);
                asm volatile("" : "+v"(p), "+v"(r.l[t2]));      // (here, not behind the branch)
                const float mx = most();
                attn_order<2 * KC, KC == 4 ? 2 : 4, 0, t == MT - 1>();
                __builtin_amdgcn_sched_barrier(0);
                __builtin_amdgcn_s_setprio(0);
                raise(t1, mx);
                __builtin_amdgcn_sched_barrier(0);
                sums(t2, std::integral_constant<bool, t2 == MT - 1>(), cur + (SK + h) * T::BYTES);
                half();
                attn_order<VD, VD == 8 ? 1 : 2, VD == 8 ? 1 : 2, 2 * (t2 == MT - 1)>();
                __builtin_amdgcn_sched_barrier(0);
                slot_end();
            };
            [&]<int... N>(std::integer_sequence<int, N...>) __attribute__((always_inline)) { (slot(std::integral_constant<int, N>()), ...); }(std::make_integer_sequence<int, SK * MT>());
        }
        // the two tiles that are still on their way
        finish(MT - 2);
        raise(MT - 1, most());
        sums(MT - 2, std::false_type(), 0);
        half();
        slot_end();
        finish(MT - 1);
        sums(MT - 1, std::false_type(), 0);
    }
    auto plain = [&](int i, auto masked) __attribute__((always_inline)) {
        constexpr bool MASKED = decltype(masked)::value;
        arrive(i);
        if constexpr (C8) if (i + 1 < end) unpack(i + 1);
#pragma unroll 1
        for (int h = 0; h < SK; ++h) {
            const int step = SK * i + h;
            if (step * ATTN_STEP >= some) break;
            const char* at = place(i) + h * T::BYTES;
#pragma unroll
            for (int t = 0; t < MT; ++t) {                   // (a tile at a time: there are no registers for more)
                AttnRows<DP, 1> one = r.tile(t);
                float4v st[1][2];
                u32x4 p[1];
                uint32_t sees[1] = {};
                if constexpr (MASKED) sees[0] = attn_sees(a, s, step, r.tok[t]);
                attn_scores<DT, DP, 1>(one, at, lane, st);
                attn_weights<DT, DP, 1, MASKED>(a, one, st, sees, lane, p);
                attn_sums<DT, DP, 1, MASKED>(one, at + SK * T::BYTES, lane, p, sees);
                r.put(t, one);
            }
        }
    };
    int next = clear;
    if constexpr (!PIPELINE)
        for (const int all = mine >= rows ? begin : min(max(whole / KEYS, begin), end); next < all; ++next) plain(next, std::false_type());
    for (; next < end; ++next) plain(next, std::true_type());
    int* flags = reinterpret_cast<int*>(smem + NB * STAGE);
    const bool wrong = __any(C8 ? held.bad : pages.bad) || s.over;          // (of all lanes: each looks up a key of its own)
    if (lane == 0) flags[wave] = wrong;
    __syncthreads();
    bool bad = false;
#pragma unroll
    for (int w = 0; w < NW; ++w) bad |= flags[w] != 0;
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        const int row = mine + t * 16 + i16, tok = row / a.group, hq = head * a.group + row - tok * a.group, e = g * 4;
        float l = groups_fold(r.l[t], [](float x, float y) { return x + y; });
        if (bad) l = NAN;
        if (row >= rows) continue;
        const int64_t tok_all = s.first + tok;
        if (splits > 1) {
            const int64_t to_row = (tok_all * a.q_heads + hq) * a.splits + split;
#pragma unroll
            for (int d = 0; d < VD; ++d) *reinterpret_cast<float4v*>(a.po + to_row * DP + d * 16 + e) = r.o[t][d];
            if (lane < 16) a.pml[to_row] = float2v{r.m[t], l};
            continue;
        }
        const float inv = l == 0.f ? 0.f : 1.f / l;
        char* out = a.out + tok_all * a.o_t + (int64_t)hq * a.o_h + e * 2;
#pragma unroll
        for (int d = 0; d < VD; ++d)
            if (d * 16 + e < a.dim) {
                u32x2 o;
                o[0] = (uint32_t)E::one(r.o[t][d][0] * inv) | ((uint32_t)E::one(r.o[t][d][1] * inv) << 16);
                o[1] = (uint32_t)E::one(r.o[t][d][2] * inv) | ((uint32_t)E::one(r.o[t][d][3] * inv) << 16);
                *reinterpret_cast<u32x2*>(out + d * 32) = o;
            }
        if (lane < 16 && a.lse) a.lse[tok_all * a.q_heads + hq] = attn_lse<DT>(r.m[t], l);
    }
}

// The splits of a row joined: DP / 4 lanes per row and G parts of its splits, as many rows as that leaves room for.  (One row per workgroup took 15 us for
// 10,752 rows of 4 splits, 22 MB, where this takes 6.)
template <int DT, int DP, int G, typename ARGS = AttnArgs>
__global__ __launch_bounds__(256) void attn_join_kernel(ARGS a) {
    constexpr int Q = DP / 4, R = 256 / (Q * G);
    static_assert(R >= 1, "a workgroup holds a row");
    __shared__ __attribute__((aligned(16))) float4v part[R][G][Q];
    const int tid = threadIdx.x, q = tid % Q, g = tid / Q % G, rr = tid / (Q * G);
    const uint32_t per = (uint32_t)a.most_new * a.q_heads, i = blockIdx.x * R + rr, b = i / per, r = i - b * per, tok = r / a.q_heads, hq = r - tok * a.q_heads;
    const AttnSeq s = attn_seq(a, min((int)b, a.seqs - 1));
    int splits = (int)tok * a.group + (int)hq % a.group < a.last_row ? a.splits : a.last_splits;
    bool live = (int)b < a.seqs && (int)tok < s.n;
    if constexpr (std::is_same_v<ARGS, Attn8Shared>) {
        splits = live ? a.parts[(((int)tok * a.group + (int)hq % a.group) >> a.block) * a.seqs + (int)b] : 1;
        live &= splits > 1;                                  // (a block that is not cut is written as it is)
    }
    const int64_t row = (int64_t)(s.first + tok) * a.q_heads + hq, at = row * a.splits;
    float m = ATTN_NOTHING, l = 0.f;
    float4v v = float4v{0.f, 0.f, 0.f, 0.f};
    const float4v* po = reinterpret_cast<const float4v*>(a.po + at * DP) + q;
    if constexpr (G == 1) {
        // (all of a row's parts in flight at once: one by one eight parts of 2240 rows took 10 us)
        auto join = [&](auto most) __attribute__((always_inline)) {
            constexpr int N = decltype(most)::value;
            float2v ml[N];
            float4v y[N];
#pragma unroll
            for (int x = 0; x < N; ++x) ml[x] = a.pml[at + min(x, splits - 1)];
#pragma unroll
            for (int x = 0; x < N; ++x) y[x] = po[(size_t)min(x, splits - 1) * Q];
#pragma unroll
            for (int x = 0; x < N; ++x) m = fmaxf(m, ml[x][0]);
#pragma unroll
            for (int x = 0; x < N; ++x) {
                const float by = x < splits ? __builtin_amdgcn_exp2f(ml[x][0] - m) : 0.f;
                if (x < splits) l += ml[x][1] * by;
                v += by != 0.f ? y[x] * by : float4v{0.f, 0.f, 0.f, 0.f};
            }
        };
        if (live) {
            if (a.splits <= 2) join(std::integral_constant<int, 2>());
            else if (a.splits <= 4) join(std::integral_constant<int, 4>());
            else join(std::integral_constant<int, 8>());
        }
    } else {
        // (one row: its maxima and totals fetched at once, a part per lane, by every wave; the first parts' sums beside them)
        __shared__ float weight[ATTN_SPLITS_MAX];
        const int lane = tid & 63;
        if (live) {
            float4v y[4];
            auto fetch = [&](int x) __attribute__((always_inline)) {
#pragma unroll
                for (int k = 0; k < 4; ++k) y[k] = po[(size_t)min(x + k * G, splits - 1) * Q];
            };
            float2v one[ATTN_SPLITS_MAX / 64];
#pragma unroll
            for (int k = 0; k < ATTN_SPLITS_MAX / 64; ++k) one[k] = a.pml[at + min(lane + 64 * k, splits - 1)];
            fetch(g);
#pragma unroll
            for (int k = 0; k < ATTN_SPLITS_MAX / 64; ++k) m = fmaxf(m, one[k][0]);
#pragma unroll
            for (int x = 1; x < 64; x <<= 1) m = fmaxf(m, __shfl_xor(m, x));
#pragma unroll
            for (int k = 0; k < ATTN_SPLITS_MAX / 64; ++k) {
                const float by = lane + 64 * k < splits ? __builtin_amdgcn_exp2f(one[k][0] - m) : 0.f;
                if (lane + 64 * k < splits) l += one[k][1] * by;
                if (tid < 64) weight[lane + 64 * k] = by;
            }
#pragma unroll
            for (int x = 1; x < 64; x <<= 1) l += __shfl_xor(l, x);
            __syncthreads();
            for (int x = g; x < splits; x += 4 * G) {
                if (x != g) fetch(x);
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const float by = x + k * G < splits ? weight[min(x + k * G, splits - 1)] : 0.f;
                    v += by != 0.f ? y[k] * by : float4v{0.f, 0.f, 0.f, 0.f};
                }
            }
        }
    }
    if constexpr (G > 1) {
        part[rr][g][q] = v;
        __syncthreads();
#pragma unroll
        for (int x = 1; x < G; ++x) v += part[rr][(g + x) % G][q];
    }
    if (!live || g) return;
    const float inv = l == 0.f ? 0.f : 1.f / l;
    if (q * 4 < a.dim) {
        u32x2 o;
        o[0] = (uint32_t)AttnType<DT>::one(v[0] * inv) | ((uint32_t)AttnType<DT>::one(v[1] * inv) << 16);
        o[1] = (uint32_t)AttnType<DT>::one(v[2] * inv) | ((uint32_t)AttnType<DT>::one(v[3] * inv) << 16);
        *reinterpret_cast<u32x2*>(a.out + (int64_t)(s.first + tok) * a.o_t + (int64_t)hq * a.o_h + q * 8) = o;
    }
    if (q == 0 && a.lse) a.lse[row] = attn_lse<DT>(m, l);
}

// ------------------------------------------------------------------------------------------ host

// nw: waves of the many-row kernel; 0: the few-row one, mt tiles of rows.  slots: the most parts of a row's keys; workgroups: of a key head, where they are shared by work, or 0
struct AttnPlan { int dp, mt, nw, row_blocks, splits, last_splits, last_row, slots, workgroups; };
constexpr int attn_waves(int dp) { return dp == 256 ? 2 : 4; }
constexpr int ATTN8_WAVES = 4;

inline void attn_raise(const void* kernel, int lds, bool (&raised)[64]) {
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) dev = 0;
    if (!raised[dev]) (void)hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
    raised[dev] = true;
}
template <int DT, int DP, int MT, bool FULL>
int attn_launch_few(const AttnArgs& a, unsigned grid, hipStream_t s) {
    constexpr int NW = attn_waves(DP), LDS = attn_lds<DP, MT, NW>();
    static bool raised[64];
    attn_raise((const void*)attn_kernel<DT, DP, MT, NW, FULL>, LDS, raised);
    hipLaunchKernelGGL((attn_kernel<DT, DP, MT, NW, FULL>), dim3(grid), dim3(NW * 64), LDS, s, a);
    return check_launch("sq_tree_attention");
}
template <int DT, int DP, int NW, bool FULL>
int attn_launch_many(const AttnArgs& a, unsigned grid, hipStream_t s) {
    constexpr int LDS = attn_tile_lds<DP, NW>();
    static bool raised[64];
    attn_raise((const void*)attn_tile_kernel<DT, DP, NW, FULL>, LDS, raised);
    hipLaunchKernelGGL((attn_tile_kernel<DT, DP, NW, FULL>), dim3(grid), dim3(NW * 64), LDS, s, a);
    return check_launch("sq_tree_attention");
}

template <int DT, int DP, typename ARGS = AttnArgs>
int attn_launch_join(const ARGS& a, hipStream_t s) {
    const int64_t all = (int64_t)a.seqs * a.most_new * a.q_heads;
    constexpr int MOST = 1024 / DP;                          // parts of a row that fill a workgroup
    if (a.splits > 8) hipLaunchKernelGGL((attn_join_kernel<DT, DP, MOST, ARGS>), dim3((unsigned)all), dim3(256), 0, s, a);
    else hipLaunchKernelGGL((attn_join_kernel<DT, DP, 1, ARGS>), dim3((unsigned)((all + MOST - 1) / MOST)), dim3(256), 0, s, a);
    return check_launch("sq_tree_attention: join");
}

template <int DT, int DP, bool FULL>
int attn_launch_dim(const AttnArgs& a, const AttnPlan& p, hipStream_t s) {
    const unsigned grid = (unsigned)((int64_t)a.seqs * a.kv_heads * ((p.row_blocks - 1) * p.splits + p.last_splits));
    int rc;
    if (p.nw) rc = p.nw == 4 ? attn_launch_many<DT, DP, 4, FULL>(a, grid, s) : attn_launch_many<DT, DP, 8, FULL>(a, grid, s);
    else rc = p.mt == 1 ? attn_launch_few<DT, DP, 1, FULL>(a, grid, s) : attn_launch_few<DT, DP, DP == 256 ? 1 : 2, FULL>(a, grid, s);
    return rc || p.splits == 1 ? rc : attn_launch_join<DT, DP>(a, s);
}

template <int DT>
int attn_launch(const AttnArgs& a, const AttnPlan& p, hipStream_t s) {
    auto go = [&](auto dp) {
        constexpr int DP = decltype(dp)::value;
        return a.dim == DP ? attn_launch_dim<DT, DP, true>(a, p, s) : attn_launch_dim<DT, DP, false>(a, p, s);
    };
    return p.dp == 64 ? go(std::integral_constant<int, 64>()) : p.dp == 128 ? go(std::integral_constant<int, 128>()) : go(std::integral_constant<int, 256>());
}
// sq_attention.hip: what a call must be like, how it is cut, and everything of it that the kernels are told but the cache's own arrays
int check_attention(const char* who, const sq_attention* a, const sq_cache* c);
bool attn_nothing(const sq_attention& a);
AttnPlan attn_plan(const sq_attention& a, const sq_cache& c, bool held8 = false);
size_t attn_workspace(const sq_attention& a, const AttnPlan& p);
int attn_prepare(const char* who, const sq_attention& a, const sq_cache& c, const AttnPlan& p, void* workspace, size_t ws_bytes, AttnArgs& k);
bool rows_apart(int tokens, int heads, int64_t t, int64_t h, int dim);      // sq_heads.hip
int attn_launch_f16(const AttnArgs& a, const AttnPlan& p, hipStream_t s);
int attn_launch_bf16(const AttnArgs& a, const AttnPlan& p, hipStream_t s);

}  // namespace sq
