// The pages of a paged cache: sequences forked (whole pages shared, the last one's slots in use copied) and pages that no sequence uses freed
// (those in use moved to the front of the pool).  A cache of any type, with or without scales, is up to four planes: arrays of
// [layers, pages, rows of a page, heads] of some bytes each, moved in pieces of 16 bytes where strides and addresses allow.
#include "sq_common.h"

namespace sq {

constexpr int PLANES_MAX = 4;
constexpr int PAGES_MAX = 1 << 20;             // pages that compact_pages keeps a bit each for in LDS
constexpr int CHUNK = 1024;                    // pieces that a workgroup of 256 threads has in flight

struct PagePlane {
    char* at;
    int64_t layer, page, row, head;            // bytes
    int rows, row_pieces, pieces, size;        // pieces of a row (of all heads) and of a head, and their bytes
};
struct PageArgs {
    PagePlane p[PLANES_MAX];
    int first[PLANES_MAX + 1];                 // chunk that a plane begins with; the last: how many there are
    const int32_t *table, *lens, *parent, *fresh;
    int32_t *out_table, *out_lens, *used, *ws; // ws: pages that move, [16 ..] to where, [16 + pages ..] which
    int64_t ld_table, ld_out;
    int layers, pages, page, max_pages, seqs;
};

// Pieces of one plane's page `from` to page `to`: its first `rows` rows in all layers, CHUNK of them.  PASSING: past the caches, for what will not be read soon
template <typename T, bool PASSING>
__device__ __forceinline__ void move_pieces(const PagePlane& p, int layers, int rows, int from, int to, uint32_t first) {
    const uint32_t per_layer = (uint32_t)rows * p.row_pieces, all = per_layer * layers;
    const bool split = p.pieces != p.row_pieces;
    T v[CHUNK / 256];
    int64_t at[CHUNK / 256];
#pragma unroll
    for (int j = 0; j < CHUNK / 256; ++j) {
        const uint32_t u = min(first + j * 256 + threadIdx.x, all - 1), layer = u / per_layer, r = u - layer * per_layer, row = r / p.row_pieces;
        uint32_t x = r - row * p.row_pieces;
        at[j] = layer * p.layer + row * p.row;
        if (split) {
            const uint32_t head = x / p.pieces;
            x -= head * p.pieces;
            at[j] += head * p.head;
        }
        at[j] += (int64_t)x * sizeof(T);
        const T* src = reinterpret_cast<const T*>(p.at + from * p.page + at[j]);
        v[j] = PASSING ? __builtin_nontemporal_load(src) : *src;
    }
#pragma unroll
    for (int j = 0; j < CHUNK / 256; ++j)
        if (first + j * 256 + threadIdx.x < all) {
            T* dst = reinterpret_cast<T*>(p.at + to * p.page + at[j]);
            if constexpr (PASSING) __builtin_nontemporal_store(v[j], dst); else *dst = v[j];
        }
}
// chunk of a page, over all planes; slots: of the page, how many there are to move
template <bool PASSING>
__device__ __forceinline__ void move_chunk(const PageArgs& a, int chunk, int from, int to, int slots) {
    int which = 0;
#pragma unroll
    for (int i = 1; i < PLANES_MAX; ++i) which += chunk >= a.first[i];
    const PagePlane& p = a.p[which];
    const int first = a.first[which];
    const int rows = (int)(((int64_t)slots * p.rows + a.page - 1) / a.page);
    const uint32_t at = (uint32_t)(chunk - first) * CHUNK;
    if (at >= (uint32_t)rows * p.row_pieces * a.layers) return;
    if (p.size == 16) move_pieces<u32x4, PASSING>(p, a.layers, rows, from, to, at);
    else if (p.size == 4) move_pieces<uint32_t, PASSING>(p, a.layers, rows, from, to, at);
    else if (p.size == 2) move_pieces<uint16_t, PASSING>(p, a.layers, rows, from, to, at);
    else move_pieces<uint8_t, PASSING>(p, a.layers, rows, from, to, at);
}

// Row i of the new batch goes on where sequence parent[i] of the old one is.  Tables and lengths are read from the old batch and written to
// another one, so rows need not wait for each other, whoever continues whom.
__global__ __launch_bounds__(256) void fork_kernel(PageArgs a) {
    const int i = blockIdx.y, p = a.parent[i], f = a.fresh[i];
    const bool ok = (uint32_t)p < (uint32_t)a.seqs;
    const int len = ok ? a.lens[p] : 0, whole = max(len, 0) / a.page, rest = max(len, 0) - whole * a.page;
    const int32_t* row = a.table + (ok ? p : 0) * a.ld_table;
    if (blockIdx.x == 0) {
        int32_t* out = a.out_table + i * a.ld_out;
        for (int j = threadIdx.x; j < a.max_pages; j += 256) {
            const int32_t id = row[j];
            out[j] = !ok ? -1 : f < 0 || j < whole ? id : j == whole ? f : -1;
        }
        if (threadIdx.x == 0) a.out_lens[i] = len;
    }
    if (!ok || (uint32_t)f >= (uint32_t)a.pages || !rest || whole >= a.max_pages) return;
    const int32_t from = row[whole];
    if ((uint32_t)from >= (uint32_t)a.pages || from == f) return;
    move_chunk<false>(a, blockIdx.x, from, f, rest);
}

// Which pages move where: one workgroup, a bit per page in LDS.  With n pages in use, the ones from n on move to the free ones before n, in
// order; no page is both, so they move in any order, and a call made again on the same tables does the same again.  A page's place among those in use is the sum of the bits
// before it: of whole groups of 256 pages added up beforehand, and of its own.  Bound by its chain (lengths, entries, sums, lists, entries again): 24 sequences
// of 32 entries, 1024 pages 4.5 us, behind 460 MB of other traffic 8.3.
constexpr int COMPACT_GROUP = 8;                   // words of 32 pages
__global__ __launch_bounds__(1024) void compact_plan_kernel(PageArgs a) {
    extern __shared__ uint32_t used[];             // bits, then sums before groups
    __shared__ int part[16];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, groups = (a.pages + 32 * COMPACT_GROUP - 1) / (32 * COMPACT_GROUP), words = groups * COMPACT_GROUP;
    int* before = reinterpret_cast<int*>(used + words);
    int32_t *holes = a.ws + 16, *movers = holes + a.pages;
    for (int i = tid; i < words; i += 1024) used[i] = 0;
    __syncthreads();
    constexpr int FLY = 8;
    auto entries = [&](int b) { return (int)min(((int64_t)max(a.lens[b], 0) + a.page - 1) / a.page, (int64_t)a.max_pages); };
    // the wave's sequences, 64 * FLY entries at a time
    auto walk = [&](auto f) __attribute__((always_inline)) {
        for (int b = wave; b < a.seqs; b += 16) {
            const int n = entries(b);
            const int32_t* row = a.table + b * a.ld_table;
            for (int j0 = 0; j0 < a.max_pages; j0 += 64 * FLY) {
                int32_t id[FLY];                   // (fetched beside the length, not behind it)
#pragma unroll
                for (int x = 0; x < FLY; ++x)
                    if (j0 + x * 64 < a.max_pages) id[x] = row[min(j0 + x * 64 + lane, a.max_pages - 1)];
#pragma unroll
                for (int x = 0; x < FLY; ++x)
                    if (j0 + x * 64 < a.max_pages) f(b, j0 + x * 64 + lane, j0 + x * 64 + lane < n ? id[x] : -1);
            }
        }
    };
    walk([&](int, int, int32_t id) { if ((uint32_t)id < (uint32_t)a.pages) atomicOr(&used[id >> 5], 1u << (id & 31)); });
    __syncthreads();
    // sums of groups, and before each of them
    int n = 0;                                     // in use so far, of all at last
    for (int g0 = 0; g0 < groups; g0 += 1024) {
        int mine = 0, upto;
        if (g0 + tid < groups)
#pragma unroll
            for (int w = 0; w < COMPACT_GROUP; ++w) mine += __popc(used[(g0 + tid) * COMPACT_GROUP + w]);
        upto = mine;
#pragma unroll
        for (int x = 1; x < 64; x <<= 1) {
            const int v = __shfl_up(upto, x);
            if (lane >= x) upto += v;
        }
        if (lane == 63) part[wave] = upto;
        __syncthreads();
        int all = 0;
#pragma unroll
        for (int w = 0; w < 16; ++w) {
            if (w < wave) upto += part[w];
            all += part[w];
        }
        if (g0 + tid < groups) before[g0 + tid] = n + upto - mine;
        n += all;
        __syncthreads();
    }
    auto rank = [&](int id) __attribute__((always_inline)) {         // pages in use before page id
        const int g = id / (32 * COMPACT_GROUP), w = id >> 5;
        int v = before[g] + __popc(used[w] & ((1u << (id & 31)) - 1));
#pragma unroll
        for (int x = 0; x < COMPACT_GROUP - 1; ++x)
            if (g * COMPACT_GROUP + x < w) v += __popc(used[g * COMPACT_GROUP + x]);
        return v;
    };
    const int kept = n < a.pages ? rank(n) : n;    // pages in use before page n
    for (int id = tid; id < a.pages; id += 1024) {
        const bool on = used[id >> 5] >> (id & 31) & 1;
        if (on == (id < n)) continue;
        const int v = rank(id);
        if (on) movers[v - kept] = id;
        else holes[id - v] = id;
    }
    if (tid == 0) {
        a.ws[0] = n - kept;
        a.used[0] = n;
    }
    __syncthreads();
    walk([&](int b, int j, int32_t id) {
        if (j >= a.max_pages) return;
        if (id >= n && id < a.pages) id = holes[rank(id) - kept];
        a.out_table[b * a.ld_out + j] = id;
    });
}

// Bound by HBM: 232 MB read and written (half of a pool of 1024 pages of 28 layers of 4 heads of 128 in bf16) 92 to 98 us with the plan, not past the caches 108.
__global__ __launch_bounds__(256) void compact_move_kernel(PageArgs a) {
    const int chunks = a.first[PLANES_MAX];
    const int64_t all = (int64_t)min(a.ws[0], a.pages / 2) * chunks;
    const int32_t *holes = a.ws + 16, *movers = holes + a.pages;
    for (int64_t c = blockIdx.x; c < all; c += gridDim.x) {
        const int i = (int)(c / chunks);
        move_chunk<true>(a, (int)(c - (int64_t)i * chunks), movers[i], holes[i], a.page);
    }
}

// The planes as the kernels take them
static int take_planes(const char* who, const sq_plane* planes, int n, int layers, int pages, int page, PageArgs& a) {
    if (n < 0 || n > PLANES_MAX || (n && !planes)) return fail(SQ_EINVAL, "%s: %d planes (up to %d)", who, n, PLANES_MAX);
    if (layers < 0 || pages < 0 || page < 1 || (int64_t)pages * page > INT32_MAX) return fail(SQ_EINVAL, "%s: %d layers, %d pages of %d slots", who, layers, pages, page);
    int chunks = 0, used = 0;
    for (int i = 0; i < n; ++i) {
        const sq_plane& s = planes[i];
        if (s.rows < 1 || s.rows > page || page % s.rows || s.heads < 0 || s.bytes < 0) return fail(SQ_EINVAL, "%s: a plane of %d rows per page of %d slots, %d heads of %d bytes", who, s.rows, page, s.heads, s.bytes);
        if (!s.heads || !s.bytes || !layers || !pages) continue;
        if (!s.at) return fail(SQ_EINVAL, "%s: null plane", who);
        PagePlane& p = a.p[used];
        const bool whole = s.heads == 1 || s.head == s.bytes;                 // the heads of a row follow each other
        const int64_t head_bytes = whole ? (int64_t)s.heads * s.bytes : s.bytes;
        uint64_t all = (uint64_t)(uintptr_t)s.at | (uint64_t)head_bytes | (uint64_t)(s.rows > 1 ? s.row : 0) | (uint64_t)(layers > 1 ? s.layer : 0) | (uint64_t)(pages > 1 ? s.page : 0);
        if (!whole) all |= (uint64_t)s.head;
        p.size = all % 16 == 0 ? 16 : all % 4 == 0 ? 4 : all % 2 == 0 ? 2 : 1;
        const int64_t pieces = head_bytes / p.size, row_pieces = whole ? pieces : pieces * s.heads;
        if (row_pieces * s.rows > (INT32_MAX - CHUNK) / layers) return fail(SQ_EUNSUPPORTED, "%s: %lld pieces in a page of %d layers", who, (long long)(row_pieces * s.rows), layers);
        p.at = (char*)s.at; p.layer = s.layer; p.page = s.page; p.row = s.row; p.head = s.head;
        p.rows = s.rows; p.row_pieces = (int)row_pieces; p.pieces = (int)pieces;
        a.first[used++] = chunks;
        chunks += (int)((row_pieces * s.rows * layers + CHUNK - 1) / CHUNK);
    }
    for (int i = used; i <= PLANES_MAX; ++i) a.first[i] = chunks;
    a.layers = layers; a.pages = pages; a.page = page;
    return SQ_OK;
}

static int take_table(const char* who, const int32_t* table, int64_t ld, int max_pages, const int32_t* lens, int seqs, int32_t* out, int64_t ld_out, PageArgs& a) {
    if (seqs < 0 || max_pages < 0 || ld < max_pages || ld_out < max_pages) return fail(SQ_EINVAL, "%s: %d sequences, tables of %d (ld %lld, %lld)", who, seqs, max_pages, (long long)ld, (long long)ld_out);
    if (seqs && (!lens || (max_pages && (!table || !out)))) return fail(SQ_EINVAL, "%s: null argument", who);
    a.table = table; a.ld_table = ld; a.max_pages = max_pages; a.lens = lens; a.seqs = seqs; a.out_table = out; a.ld_out = ld_out;
    return SQ_OK;
}

}  // namespace sq

using namespace sq;

extern "C" {

int sq_fork_pages(const sq_plane* planes, int32_t n_planes, int32_t layers, int32_t pages, int32_t page, const int32_t* table, int64_t ld_table, int32_t max_pages,
                  const int32_t* lens, int32_t seqs, const int32_t* parent, const int32_t* fresh, int32_t rows, int32_t* out_table, int64_t ld_out, int32_t* out_lens,
                  void* stream) {
    const char* who = "sq_fork_pages";
    PageArgs a = {};
    if (int rc = take_planes(who, planes, n_planes, layers, pages, page, a)) return rc;
    if (rows < 0 || rows > 65535) return fail(SQ_EINVAL, "%s: %d rows", who, rows);
    if (!rows) return SQ_OK;
    if (int rc = take_table(who, table, ld_table, max_pages, lens, seqs, out_table, ld_out, a)) return rc;
    if (!seqs) return fail(SQ_EINVAL, "%s: %d rows of no sequence", who, rows);
    if (!parent || !fresh || !out_lens) return fail(SQ_EINVAL, "%s: null argument", who);
    if (out_table == table && max_pages) return fail(SQ_EINVAL, "%s: the new table is the old one", who);
    if (out_lens == lens) return fail(SQ_EINVAL, "%s: the new lengths are the old ones", who);
    a.parent = parent; a.fresh = fresh; a.out_lens = out_lens;
    const int chunks = a.first[PLANES_MAX];
    hipLaunchKernelGGL(fork_kernel, dim3((unsigned)(chunks ? chunks : 1), (unsigned)rows), dim3(256), 0, (hipStream_t)stream, a);
    return check_launch(who);
}

size_t sq_compact_pages_workspace_bytes(int32_t pages) { return pages < 0 || pages > PAGES_MAX ? 0 : (16 + 2 * (size_t)pages) * 4; }

int sq_compact_pages(const sq_plane* planes, int32_t n_planes, int32_t layers, int32_t pages, int32_t page, const int32_t* table, int64_t ld_table, int32_t max_pages,
                     const int32_t* lens, int32_t seqs, int32_t* out_table, int64_t ld_out, int32_t* used, void* workspace, size_t ws_bytes, void* stream) {
    const char* who = "sq_compact_pages";
    PageArgs a = {};
    if (int rc = take_planes(who, planes, n_planes, layers, pages, page, a)) return rc;
    if (int rc = take_table(who, table, ld_table, max_pages, lens, seqs, out_table, ld_out, a)) return rc;
    if (!used) return fail(SQ_EINVAL, "%s: null argument", who);
    if (pages > PAGES_MAX) return fail(SQ_EUNSUPPORTED, "%s: %d pages (up to %d)", who, pages, PAGES_MAX);
    if (out_table == table && max_pages && seqs) return fail(SQ_EINVAL, "%s: the new table is the old one", who);
    const size_t need = sq_compact_pages_workspace_bytes(pages);
    if (ws_bytes < need || !workspace || ((uintptr_t)workspace & 255)) return fail(SQ_EWORKSPACE, "%s: workspace of %zu bytes (256-byte aligned) needed, %zu given", who, need, ws_bytes);
    a.used = used; a.ws = (int32_t*)workspace;
    const auto lds_of = [](int pages) { return (unsigned)((pages + 32 * COMPACT_GROUP - 1) / (32 * COMPACT_GROUP) * (4 * COMPACT_GROUP + 4)); };
    const unsigned lds = lds_of(pages);
    static bool raised[64];
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) dev = 0;
    if (lds > 48 * 1024 && !raised[dev]) raised[dev] = hipFuncSetAttribute((const void*)compact_plan_kernel, hipFuncAttributeMaxDynamicSharedMemorySize, lds_of(PAGES_MAX)) == hipSuccess;
    hipLaunchKernelGGL(compact_plan_kernel, dim3(1), dim3(1024), lds, (hipStream_t)stream, a);
    if (int rc = check_launch(who)) return rc;
    const int64_t most = (int64_t)seqs * max_pages < pages / 2 ? (int64_t)seqs * max_pages : pages / 2, all = most * a.first[PLANES_MAX];
    if (!all) return SQ_OK;
    const int64_t room = 32 * (int64_t)device_cus();
    hipLaunchKernelGGL(compact_move_kernel, dim3((unsigned)(all < room ? all : room)), dim3(256), 0, (hipStream_t)stream, a);
    return check_launch(who);
}

}  // extern "C"
