// Pages of a KV cache: reserving, freeing, forking and copying them, and moving kept rows together.  The reference's cache
// calls take a page table as it is given (flash_api.cpp:356) and have no operations on it.
//
// The state of a pool is one reference count a page, on the device; a page is free when its count is 0.  Pages are handed out
// lowest first, to rows and entries in order, and counts only change by integer additions, so every result is determined and
// nothing has to be read on the host: all of it can be captured into a graph with the step it belongs to.
//
// The tables and counts are small (a 512 x 2048 table is 4 MB): those kernels are bound by launches and latency, and are laid
// out to need few of both.  Copying rows is bound by HBM: 2 bytes moved a byte copied, 16-byte accesses with eight in flight a
// thread.
#include <algorithm>
#include <memory>
#include <new>
#include "fa_utils.cuh"
#include "fa_internal.h"

namespace fa {

namespace {

constexpr int kChunk = 4096;                 // pages whose free ones are listed together
constexpr int kMaxPages = 1 << 24;
constexpr int kMaxForks = 1 << 20;           // every row looks at all rows in front of it: 4096 rows 69 us, 65536 rows 1.2 ms, 2^24 a minute
constexpr int kMaxViews = 56;                // caches (or stacks of them) of one launch: they travel as kernel parameters
constexpr int kSmallThreads = 1024;         // of the one block that does a small call
constexpr int kPiece = 32768;                // bytes of a page that a CTA copies at a time

__device__ __forceinline__ int pages_of(long long rows, int page_size, int width) {
    const long long n = (max(rows, 0ll) + page_size - 1) / page_size;
    return (int)min(n, (long long)width);
}
__device__ __forceinline__ bool in_pool(int page, int num_pages) { return (unsigned)page < (unsigned)num_pages; }
// a count that is 0 already stays 0: a page named once too often is not taken from its next owner
__device__ __forceinline__ void drop_ref(int* refs, int page) {
    if (atomicSub(refs + page, 1) <= 0) atomicAdd(refs + page, 1);
}

struct PoolArgs {
    int32_t* refs;
    int num_pages, page_size;
    int32_t* table;
    int64_t table_stride;
    int b, width;
    const int32_t* seqlens;
    int extra;
    // workspace
    int32_t* need;               // (rows): entries to fill; fork: 1 = the row gets a copy of its partly filled page
    int32_t* first;              // (rows): reserve: first entry to fill; fork: its partly filled page, -1 = none
    int32_t* fill;               // (rows): fork: its length
    int32_t* free_count;         // (chunks)
    int32_t* free_list;          // (pages): the free pages of chunk c from entry c * kChunk on, ascending
    int32_t* missing;
    // fork
    const int32_t* parents;
    int n, keep_parents;
    int32_t* new_table;          // (n, width)
    int32_t* new_seqlens;        // (n)
};

// ---- free pages, chunk by chunk: THREADS threads, kChunk / THREADS consecutive pages each ---------------------------------
template <int THREADS>
__device__ void list_free(const PoolArgs& a, int chunk) {
    constexpr int EACH = kChunk / THREADS, WARPS = THREADS / 32;
    __shared__ int s_warp[WARPS];
    __syncthreads();                                         // may be called again for the next chunk
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int p0 = chunk * kChunk + tid * EACH;
    uint32_t zero = 0;
#pragma unroll
    for (int i = 0; i < EACH; ++i) zero |= (uint32_t)(p0 + i < a.num_pages && a.refs[min(p0 + i, a.num_pages - 1)] == 0) << i;
    const int mine = __popc(zero);
    int upto = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, upto, d);
        if (lane >= d) upto += v;
    }
    if (lane == 31) s_warp[warp] = upto;
    __syncthreads();
    int before = 0, total = 0;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
        before += w < warp ? s_warp[w] : 0;
        total += s_warp[w];
    }
    int32_t* out = a.free_list + (int64_t)chunk * kChunk + before + upto - mine;
    while (zero) {
        const int i = __ffs(zero) - 1;
        zero &= zero - 1;
        *out++ = p0 + i;
    }
    if (tid == 0) a.free_count[chunk] = total;
}

// sum of v[0 .. n), by all 256 threads
__device__ int block_sum(const int32_t* v, int n) {
    __shared__ int s_sum[8];
    int x = 0;
    for (int i = threadIdx.x; i < n; i += 256) x += v[i];
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) s_sum[threadIdx.x >> 5] = x;
    __syncthreads();
    x = 0;
#pragma unroll
    for (int w = 0; w < 8; ++w) x += s_sum[w];
    return x;
}
// page number `slot` of all free ones in ascending order, -1 if there are not so many; a whole warp asks for the same or
// for slots of its own
__device__ int free_page(const PoolArgs& a, int chunks, long long slot) {
    for (int c = 0; c < chunks; ++c) {
        const int k = a.free_count[c];
        if (slot < k) return a.free_list[(int64_t)c * kChunk + slot];
        slot -= k;
    }
    return -1;
}

// ---- reserve ----------------------------------------------------------------------------------------------------------
// what a row needs; a warp a row
__device__ void reserve_count(const PoolArgs& a, int row, int lane) {
    const int n = pages_of((long long)a.seqlens[row] + a.extra, a.page_size, a.width);
    const int32_t* t = a.table + row * a.table_stride;
    int need = 0, first = n;
#pragma unroll 4
    for (int j = lane; j < n; j += 32)
        if (t[j] < 0) { ++need; first = min(first, j); }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) {
        need += __shfl_xor_sync(0xffffffffu, need, d);
        first = min(first, __shfl_xor_sync(0xffffffffu, first, d));
    }
    if (lane == 0) { a.need[row] = need; a.first[row] = first; }
}
// takes the free pages from number `slot` on
__device__ void reserve_take(const PoolArgs& a, int row, int lane, int chunks, long long slot) {
    const int need = a.need[row];
    if (need == 0) return;
    const int n = pages_of((long long)a.seqlens[row] + a.extra, a.page_size, a.width);
    int32_t* t = a.table + row * a.table_stride;
    int lacking = 0, done = 0;
    for (int j0 = a.first[row]; done < need && j0 < n; j0 += 32) {
        const int j = j0 + lane;
        const bool want = j < n && t[j] < 0;
        const uint32_t vote = __ballot_sync(0xffffffffu, want);
        if (want) {
            const int page = free_page(a, chunks, slot + __popc(vote & ((1u << lane) - 1)));
            if (page >= 0) { t[j] = page; a.refs[page] = 1; } else ++lacking;
        }
        slot += __popc(vote);
        done += __popc(vote);
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) lacking += __shfl_xor_sync(0xffffffffu, lacking, d);
    if (lane == 0 && lacking) atomicAdd(a.missing, lacking);
}
// Launch 1: the first row_blocks blocks count, the others list free pages.
__global__ void __launch_bounds__(256) reserve_count_kernel(const __grid_constant__ PoolArgs a, int row_blocks) {
    if ((int)blockIdx.x >= row_blocks) { list_free<256>(a, blockIdx.x - row_blocks); return; }
    if (blockIdx.x == 0 && threadIdx.x == 0) *a.missing = 0;
    const int row = blockIdx.x * 8 + (threadIdx.x >> 5);
    if (row < a.b) reserve_count(a, row, threadIdx.x & 31);
}
// Launch 2: every row takes the pages behind those of the rows in front of it.
__global__ void __launch_bounds__(256) reserve_take_kernel(const __grid_constant__ PoolArgs a, int chunks) {
    const int row0 = blockIdx.x * 8, row = row0 + (threadIdx.x >> 5);
    long long slot = block_sum(a.need, row0);
    if (row >= a.b) return;
    for (int r = row0; r < row; ++r) slot += a.need[r];
    reserve_take(a, row, threadIdx.x & 31, chunks, slot);
}
// Few rows and pages: one block does both, which saves a launch.
__global__ void __launch_bounds__(kSmallThreads) reserve_small_kernel(const __grid_constant__ PoolArgs a, int chunks) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) *a.missing = 0;
    for (int row = warp; row < a.b; row += kSmallThreads / 32) reserve_count(a, row, lane);
    for (int c = 0; c < chunks; ++c) list_free<kSmallThreads>(a, c);
    __syncthreads();
    long long slot = 0;
    for (int row = 0, r = warp; r < a.b; r += kSmallThreads / 32) {
        for (; row < r; ++row) slot += a.need[row];
        reserve_take(a, r, lane, chunks, slot);
    }
}

// ---- free -------------------------------------------------------------------------------------------------------------
__global__ void __launch_bounds__(256) free_kernel(const __grid_constant__ PoolArgs a) {
    const int per = (a.width + 255) / 256;                   // blocks of a row
    const int row = blockIdx.x / per, j = blockIdx.x % per * 256 + threadIdx.x;
    const int keep = a.seqlens ? pages_of((long long)a.seqlens[row] + a.extra, a.page_size, a.width) : 0;
    if (j < keep || j >= a.width) return;
    int32_t* t = a.table + row * a.table_stride + j;
    const int page = *t;
    if (page < 0) return;
    if (in_pool(page, a.num_pages)) drop_ref(a.refs, page);
    *t = -1;
}

// ---- fork -------------------------------------------------------------------------------------------------------------
// A warp a row: children share their parent's pages; with the parents replaced, the old rows (n ..) let go of theirs.
__device__ void fork_share(const PoolArgs& a, int row, int lane) {
    if (row < a.n) {
        const int parent = a.parents[row];
        const bool valid = parent >= 0 && parent < a.b;
        const int len = valid ? (int)max(0ll, min((long long)a.seqlens[parent], (long long)a.width * a.page_size)) : 0;
        const int n = pages_of(len, a.page_size, a.width);
        const int32_t* from = a.table + (valid ? parent : 0) * a.table_stride;
        int32_t* to = a.new_table + (int64_t)row * a.width;
        int last = -1;
        for (int j = lane; j < a.width; j += 32) {
            const int page = j < n ? from[j] : -1;
            const bool have = page >= 0 && in_pool(page, a.num_pages);
            to[j] = have ? page : -1;
            if (have) atomicAdd(a.refs + page, 1);
            if (j == n - 1 && have && len % a.page_size) last = page;
        }
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) last = max(last, __shfl_xor_sync(0xffffffffu, last, d));
        if (lane == 0) { a.first[row] = last; a.fill[row] = len; a.new_seqlens[row] = len; }
    } else if (!a.keep_parents && row - a.n < a.b) {
        const int32_t* t = a.table + (row - a.n) * a.table_stride;
        for (int j = lane; j < a.width; j += 32)
            if (t[j] >= 0 && in_pool(t[j], a.num_pages)) drop_ref(a.refs, t[j]);
    }
}
// Which rows need a page of their own.  Of the c rows that hold the same partly filled page, with e holders
// elsewhere (count = c + e), row number i of them takes a copy when i < c + e - 1: all but the last, or all where e > 0.
__device__ void fork_count(const PoolArgs& a, int row, int lane) {
    const int page = a.first[row];
    int before = 0;
    if (page >= 0) {
#pragma unroll 4
        for (int r = lane; r < row; r += 32) before += a.first[r] == page;
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) before += __shfl_xor_sync(0xffffffffu, before, d);
    }
    if (lane == 0) a.need[row] = page >= 0 && a.refs[page] - before > 1;
}
__global__ void __launch_bounds__(256) fork_share_kernel(const __grid_constant__ PoolArgs a) {
    if (blockIdx.x == 0 && threadIdx.x == 0) *a.missing = 0;
    fork_share(a, blockIdx.x * 8 + (threadIdx.x >> 5), threadIdx.x & 31);
}
__global__ void __launch_bounds__(256) fork_count_kernel(const __grid_constant__ PoolArgs a, int row_blocks) {
    if ((int)blockIdx.x >= row_blocks) { list_free<256>(a, blockIdx.x - row_blocks); return; }
    const int row = blockIdx.x * 8 + (threadIdx.x >> 5);
    if (row < a.n) fork_count(a, row, threadIdx.x & 31);
}
// Few rows and pages: one block does both.
__global__ void __launch_bounds__(kSmallThreads) fork_small_kernel(const __grid_constant__ PoolArgs a, int chunks) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) *a.missing = 0;
    for (int row = warp; row < a.n + (a.keep_parents ? 0 : a.b); row += kSmallThreads / 32) fork_share(a, row, lane);
    __syncthreads();
    for (int row = warp; row < a.n; row += kSmallThreads / 32) fork_count(a, row, lane);
    for (int c = 0; c < chunks; ++c) list_free<kSmallThreads>(a, c);
}

// ---- copies -----------------------------------------------------------------------------------------------------------
struct View {                    // one cache or a stack of them; strides in bytes
    char* ptr;
    int64_t cache, page, row, head;
    int caches, heads, seg, vec; // a row of a cache: `heads` segments of `seg` bytes, moved `vec` bytes at a time
};
struct CopyArgs {
    PoolArgs pool;               // fork: where the copies go is worked out here
    View views[kMaxViews];
    int num_views, num_pages, page_size, chunks;
    const int32_t* src;          // copy_pages: the lists; null: fork
    const int32_t* dst;
    int first_launch;            // fork: this launch also writes tables and counts
    int per_row;                 // CTAs of a row
};

template <typename V>
__device__ __forceinline__ void copy_piece(const View& v, const char* src, char* dst, int64_t from, int64_t to, int row_bytes) {
    const bool flat = v.row == row_bytes && v.head == v.seg;
    auto at = [&](int64_t o) -> int64_t {
        if (flat) return o;
        const int64_t r = o / row_bytes, rest = o % row_bytes;
        return r * v.row + rest / v.seg * v.head + rest % v.seg;
    };
    constexpr int N = 4;
    for (int64_t o = from + (int64_t)threadIdx.x * sizeof(V); o < to; o += (int64_t)N * 256 * sizeof(V)) {
        V x[N];
        int64_t where[N];
#pragma unroll
        for (int k = 0; k < N; ++k) {
            const int64_t ok = o + (int64_t)k * 256 * sizeof(V);
            where[k] = ok < to ? at(ok) : -1;
            if (where[k] >= 0) x[k] = *reinterpret_cast<const V*>(src + where[k]);
        }
#pragma unroll
        for (int k = 0; k < N; ++k)
            if (where[k] >= 0) *reinterpret_cast<V*>(dst + where[k]) = x[k];
    }
}

__global__ void __launch_bounds__(256, 4) copy_kernel(const __grid_constant__ CopyArgs a) {
    const int row = blockIdx.x / a.per_row, part = blockIdx.x % a.per_row;
    int src, dst, rows = a.page_size;
    if (a.src) {
        src = a.src[row];
        dst = a.dst[row];
        if (!in_pool(src, a.num_pages) || !in_pool(dst, a.num_pages) || src == dst) return;
    } else {
        const PoolArgs& p = a.pool;
        const int need = p.need[row], len = p.fill[row];
        src = p.first[row];
        if (!need) return;
        dst = free_page(p, a.chunks, block_sum(p.need, row));
        rows = len % a.page_size;
        if (a.first_launch && part == 0 && threadIdx.x == 0) {
            p.new_table[(int64_t)row * p.width + len / a.page_size] = dst;
            atomicSub(p.refs + src, 1);
            if (dst >= 0) p.refs[dst] = 1;
            else {                                           // no page left: the row ends with its last full page
                p.new_seqlens[row] = len - rows;
                atomicAdd(p.missing, 1);
            }
        }
        if (dst < 0) return;
    }
    int unit = part;
    for (int w = 0; w < a.num_views; ++w) {
        const View& v = a.views[w];
        const int row_bytes = v.heads * v.seg;
        const int64_t bytes = (int64_t)rows * row_bytes;
        const int pieces = (int)((bytes + kPiece - 1) / kPiece);
        // units of this view: (cache, piece); this CTA takes every per_row-th of all views' units
        const int64_t units = (int64_t)v.caches * pieces;
        int64_t u = unit;
        for (; u < units; u += a.per_row) {
            const int64_t c = u / pieces, from = u % pieces * kPiece, to = min(from + kPiece, bytes);
            const char* s = v.ptr + c * v.cache + src * v.page;
            char* d = v.ptr + c * v.cache + dst * v.page;
            if (v.vec == 16) copy_piece<uint4>(v, s, d, from, to, row_bytes);
            else if (v.vec == 4) copy_piece<uint32_t>(v, s, d, from, to, row_bytes);
            else copy_piece<unsigned char>(v, s, d, from, to, row_bytes);
        }
        unit = (int)(u - units);                             // where the next view's units go on
    }
}

// ---- kept rows move together ------------------------------------------------------------------------------------------
struct CompactArgs {
    View views[kMaxViews];
    int num_views;
    int num_entries, page_size, width;   // pages (or dense cache entries), rows of one, entries of a table row (dense: 1)
    const int32_t* table;                // null: dense
    int64_t table_stride;
    const int32_t* batch_idx;            // dense: cache entry of a sequence, or null
    const int32_t* seqlens;
    const int32_t* kept;                 // (b, n): row seqlens + kept[i] becomes row seqlens + i
    int64_t kept_stride;
    const int32_t* counts;               // (b), or null: up to the first entry that is not larger than the one before
    int b, n, first_launch;
    int warps_seq;                       // warps of one sequence: all views' caches x column pieces
    int32_t* new_seqlens;
};

// A warp moves one column piece (32 x vec bytes of a row) of one cache of one sequence, rows in order and U at a time.  Kept
// rows only move forward: what a batch writes lies in front of everything that a later batch reads, so batches need no wait
// on one another.
template <typename V>
__device__ __forceinline__ void compact_piece(const CompactArgs& a, const View& v, char* base, int b, int col, bool mine, bool report) {
    constexpr int U = 8;
    const int lane = threadIdx.x & 31;
    const long long cap = (long long)a.page_size * a.width;
    const int L = (int)max(0ll, min((long long)a.seqlens[b], cap));
    const int32_t* kept = a.kept + b * a.kept_stride;
    const int32_t* table = a.table ? a.table + b * a.table_stride : nullptr;
    const int entry = table ? 0 : a.batch_idx ? a.batch_idx[b] : b;
    const int most = a.counts ? max(0, min(a.counts[b], a.n)) : a.n;
    const int64_t inner = (int64_t)(col / v.seg) * v.head + col % v.seg;
    auto place = [&](int row) -> int64_t {                   // byte offset of a cache row, -1: not in the cache
        const int e = table ? table[row / a.page_size] : entry;
        if (!in_pool(e, a.num_entries)) return -1;
        return e * v.page + (int64_t)(row % a.page_size) * v.row;
    };
    int i0 = 0, before = -1;                                 // the last kept entry of the batch in front
    for (; i0 < most; i0 += U) {
        int k = -1;
        bool good = false;
        int64_t from = -1, to = -1;
        if (lane < U && i0 + lane < most) k = kept[i0 + lane];
        int prev = __shfl_up_sync(0xffffffffu, k, 1);
        if (lane == 0) prev = before;
        if (lane < U && i0 + lane < most) good = k > prev && (long long)L + k < cap;
        const int run = __ffs(~__ballot_sync(0xffffffffu, good)) - 1;    // leading entries that are in order
        if (lane < run && k != i0 + lane) {
            from = place(L + k);
            to = place(L + i0 + lane);
        }
        V x[U];
        int64_t dst[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t f = __shfl_sync(0xffffffffu, from, u);
            dst[u] = __shfl_sync(0xffffffffu, to, u);
            if (f < 0) dst[u] = -1;
            if (dst[u] >= 0 && mine) x[u] = *reinterpret_cast<const V*>(base + f + inner);
        }
        __syncwarp();
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (dst[u] >= 0 && mine) *reinterpret_cast<V*>(base + dst[u] + inner) = x[u];
        before = __shfl_sync(0xffffffffu, k, U - 1);
        if (run < U) { i0 += run; break; }
    }
    if (report && lane == 0) a.new_seqlens[b] = L + min(i0, most);
}

__global__ void __launch_bounds__(128) compact_kernel(const __grid_constant__ CompactArgs a) {
    const int64_t warp = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
    const int b = (int)(warp / a.warps_seq), lane = threadIdx.x & 31;
    if (b >= a.b) return;
    int at = (int)(warp % a.warps_seq);
    for (int w = 0; w < a.num_views; ++w) {
        const View& v = a.views[w];
        const int row_bytes = v.heads * v.seg, pieces = (row_bytes + 32 * v.vec - 1) / (32 * v.vec);
        if (at >= v.caches * pieces) { at -= v.caches * pieces; continue; }
        char* base = v.ptr + (int64_t)(at / pieces) * v.cache;
        const int col = at % pieces * 32 * v.vec + lane * v.vec;
        const bool mine = col < row_bytes, report = a.first_launch && warp % a.warps_seq == 0;
        if (v.vec == 16) compact_piece<uint4>(a, v, base, b, mine ? col : 0, mine, report);
        else if (v.vec == 4) compact_piece<uint32_t>(a, v, base, b, mine ? col : 0, mine, report);
        else compact_piece<unsigned char>(a, v, base, b, mine ? col : 0, mine, report);
        return;
    }
}

// ---- host -------------------------------------------------------------------------------------------------------------
inline size_t align256(size_t x) { return (x + 255) & ~(size_t)255; }
int chunks_of(const fa_pages_params& p) { return (p.num_pages + kChunk - 1) / kChunk; }

// One block instead of two launches of several: up to 64 rows, 1024 table entries a warp and two lists of pages.
bool small_pool(const fa_pages_params& p, int rows) { return rows <= 64 && (int64_t)(rows + 31) / 32 * p.width <= 1024 && chunks_of(p) <= 2; }

size_t workspace(const fa_pages_params& p, int rows, PoolArgs* a) {
    const size_t need = 0, first = align256((size_t)rows * 4), fill = 2 * first, count = 3 * first, list = count + align256((size_t)chunks_of(p) * 4);
    if (a) {
        char* ws = reinterpret_cast<char*>(p.workspace);
        a->need = reinterpret_cast<int32_t*>(ws + need);
        a->first = reinterpret_cast<int32_t*>(ws + first);
        a->fill = reinterpret_cast<int32_t*>(ws + fill);
        a->free_count = reinterpret_cast<int32_t*>(ws + count);
        a->free_list = reinterpret_cast<int32_t*>(ws + list);
    }
    return list + (size_t)chunks_of(p) * kChunk * 4;
}

int check_table(const fa_pages_params& p, bool pool) {
    if (p.b < 0 || p.width < 0 || p.page_size <= 0) return fail(FA_ERR_BAD_SHAPE, "negative size, or page_size not positive");
    if ((long long)p.width * p.page_size > 0x7fffffff) return fail(FA_ERR_BAD_SHAPE, "a sequence holds at most 2^31 - 1 rows");
    if (p.b > 0 && p.width > 0 && !p.table) return fail(FA_ERR_NULL, "page_table is null");
    if (p.b > (1 << 24) || p.n < 0 || p.n > (1 << 24)) return fail(FA_ERR_BAD_SHAPE, "at most 2^24 sequences");
    if (pool) {
        if (p.num_pages <= 0 || p.num_pages > kMaxPages) return fail(FA_ERR_BAD_SHAPE, "a pool has 1 to 2^24 pages");
        if (!p.refs) return fail(FA_ERR_NULL, "page_refs is null");
    }
    return FA_OK;
}

int check_workspace(const fa_pages_params& p, int rows) {
    const size_t need = workspace(p, rows, nullptr);
    if (!p.workspace || p.workspace_bytes < need) return fail(FA_ERR_WORKSPACE, "workspace of %zu bytes required, %zu given", need, p.workspace_bytes);
    if (reinterpret_cast<uintptr_t>(p.workspace) & 15) return fail(FA_ERR_MISALIGNED, "the workspace must be 16-byte aligned");
    return FA_OK;
}

PoolArgs pool_args(const fa_pages_params& p) {
    PoolArgs a = {};
    a.refs = p.refs; a.num_pages = p.num_pages; a.page_size = p.page_size;
    a.table = p.table; a.table_stride = p.table_stride; a.b = p.b; a.width = p.width;
    a.seqlens = p.seqlens; a.extra = p.extra; a.missing = p.missing;
    a.parents = p.rows; a.n = p.n; a.keep_parents = p.keep_parents;
    a.new_table = p.new_table; a.new_seqlens = p.new_seqlens;
    return a;
}

int check_views(const fa_pages_params& p) {
    if (p.num_caches < 0 || (p.num_caches > 0 && !p.caches)) return fail(FA_ERR_NULL, "caches is null");
    for (int i = 0; i < p.num_caches; ++i) {
        const fa_cache_view& v = p.caches[i];
        if (!v.ptr) return fail(FA_ERR_NULL, "cache %d is null", i);
        if (v.caches < 0 || v.heads <= 0 || v.segment_bytes <= 0 || (long long)v.heads * v.segment_bytes > (1 << 28))
            return fail(FA_ERR_BAD_SHAPE, "cache %d has a bad shape", i);
    }
    return FA_OK;
}

// Rows that move in place may not be moved twice: no cache may begin where another does.
int check_apart(const fa_pages_params& p) {
    int64_t n = 0;
    for (int i = 0; i < p.num_caches; ++i) n += p.caches[i].caches;
    if (n < 2 || (p.num_caches == 1 && p.caches[0].stride_cache != 0)) return FA_OK;
    constexpr int kFew = 256;
    uint64_t few[kFew];
    std::unique_ptr<uint64_t[]> many(n > kFew ? new (std::nothrow) uint64_t[n] : nullptr);
    uint64_t* at = n > kFew ? many.get() : few;
    if (!at) return fail(FA_ERR_UNSUPPORTED, "no host memory for %lld caches", (long long)n);
    int64_t k = 0;
    for (int i = 0; i < p.num_caches; ++i)
        for (int c = 0; c < p.caches[i].caches; ++c) at[k++] = (uint64_t)(uintptr_t)p.caches[i].ptr + (uint64_t)c * (uint64_t)p.caches[i].stride_cache;
    std::sort(at, at + n);
    if (std::adjacent_find(at, at + n) != at + n) return fail(FA_ERR_UNSUPPORTED, "a cache may be given once only");
    return FA_OK;
}

View view_of(const fa_cache_view& c) {
    View v = {reinterpret_cast<char*>(c.ptr), c.stride_cache, c.stride_page, c.stride_row, c.stride_head, c.caches, c.heads, c.segment_bytes, 1};
    if (v.heads == 1) v.head = v.seg;
    if (v.head == v.seg) { v.seg *= v.heads; v.heads = 1; v.head = v.seg; }
    const uint64_t all = (uint64_t)(uintptr_t)c.ptr | (uint64_t)(v.caches > 1 ? v.cache : 0) | (uint64_t)v.page | (uint64_t)v.row | (uint64_t)v.head | (uint64_t)v.seg;
    v.vec = all % 16 == 0 ? 16 : all % 4 == 0 ? 4 : 1;
    return v;
}

// fork and copy_pages: p.n rows over all caches, kMaxViews views a launch
int launch_copies(const fa_pages_params& p, const PoolArgs& pool, bool lists, cudaStream_t st) {
    CopyArgs a;
    a.pool = pool;
    a.num_pages = p.num_pages; a.page_size = p.page_size; a.chunks = chunks_of(p);
    a.src = lists ? p.rows : nullptr;
    a.dst = lists ? p.rows2 : nullptr;
    for (int v0 = 0; v0 < (p.num_caches ? p.num_caches : 1); v0 += kMaxViews) {
        a.num_views = p.num_caches - v0 < kMaxViews ? p.num_caches - v0 : kMaxViews;
        a.first_launch = v0 == 0;
        int64_t units = 0;
        for (int i = 0; i < a.num_views; ++i) {
            a.views[i] = view_of(p.caches[v0 + i]);
            units += (int64_t)a.views[i].caches * (((int64_t)p.page_size * a.views[i].heads * a.views[i].seg + kPiece - 1) / kPiece);
        }
        // CTAs of a row: one a unit, but no more than what four to an SM make, so that each works out its page once
        int64_t per = (4ll * sm_count() + p.n - 1) / p.n;
        if (per > units) per = units;
        a.per_row = (int)(per < 1 ? 1 : per);
        copy_kernel<<<(unsigned)(a.per_row * p.n), 256, 0, st>>>(a);
        mark_kernel(st);
        if (int e = cuda_ok(cudaGetLastError(), "page copy launch")) return e;
    }
    return FA_OK;
}

int run_reserve(const fa_pages_params& p) {
    if (int e = check_table(p, true)) return e;
    if (p.b > 0 && !p.seqlens) return fail(FA_ERR_NULL, "cache_seqlens is null");
    if (!p.missing) return fail(FA_ERR_NULL, "missing is null");
    if ((int64_t)p.b * p.width > 0x7fffffff) return fail(FA_ERR_BAD_SHAPE, "the page table is too large");   // needs are summed in 32 bits
    if (int e = check_workspace(p, p.b)) return e;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(p.stream);
    PoolArgs a = pool_args(p);
    workspace(p, p.b, &a);
    const int rows = (p.b + 7) / 8 > 0 ? (p.b + 7) / 8 : 1, chunks = chunks_of(p);
    mark_kernel(st);
    if (small_pool(p, p.b)) {
        reserve_small_kernel<<<1, kSmallThreads, 0, st>>>(a, chunks);
        mark_kernel(st);
        return cuda_ok(cudaGetLastError(), "reserve launch");
    }
    reserve_count_kernel<<<rows + chunks, 256, 0, st>>>(a, rows);
    mark_kernel(st);
    if (int e = cuda_ok(cudaGetLastError(), "reserve launch")) return e;
    reserve_take_kernel<<<rows, 256, 0, st>>>(a, chunks);
    mark_kernel(st);
    return cuda_ok(cudaGetLastError(), "reserve launch");
}

int run_free(const fa_pages_params& p) {
    if (int e = check_table(p, true)) return e;
    if (p.b == 0 || p.width == 0) return FA_OK;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(p.stream);
    const int64_t blocks = (int64_t)p.b * ((p.width + 255) / 256);
    if (blocks >= (1ll << 31)) return fail(FA_ERR_BAD_SHAPE, "the page table is too large");
    mark_kernel(st);
    free_kernel<<<(unsigned)blocks, 256, 0, st>>>(pool_args(p));
    mark_kernel(st);
    return cuda_ok(cudaGetLastError(), "free launch");
}

int run_fork(const fa_pages_params& p) {
    if (int e = check_table(p, true)) return e;
    if (int e = check_views(p)) return e;
    if (p.b > 0 && !p.seqlens) return fail(FA_ERR_NULL, "cache_seqlens is null");
    if (!p.missing) return fail(FA_ERR_NULL, "missing is null");
    if (p.n > kMaxForks) return fail(FA_ERR_BAD_SHAPE, "at most 2^20 rows continue in one call");
    if (p.n > 0 && (!p.rows || !p.new_seqlens || (p.width > 0 && !p.new_table))) return fail(FA_ERR_NULL, "parents or an output is null");
    if (p.width > 0 && p.new_table == p.table && p.table) return fail(FA_ERR_UNSUPPORTED, "the new page table must be another tensor than the old one");
    if (int e = check_workspace(p, p.n)) return e;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(p.stream);
    PoolArgs a = pool_args(p);
    workspace(p, p.n, &a);
    const int share = p.n + (p.keep_parents ? 0 : p.b);
    mark_kernel(st);
    if (small_pool(p, share)) {
        fork_small_kernel<<<1, kSmallThreads, 0, st>>>(a, chunks_of(p));
        mark_kernel(st);
        if (int e = cuda_ok(cudaGetLastError(), "fork launch")) return e;
        return p.n ? launch_copies(p, a, false, st) : FA_OK;
    }
    fork_share_kernel<<<(share + 7) / 8 > 0 ? (share + 7) / 8 : 1, 256, 0, st>>>(a);
    mark_kernel(st);
    if (int e = cuda_ok(cudaGetLastError(), "fork launch")) return e;
    if (p.n == 0) return FA_OK;
    const int rows = (p.n + 7) / 8, chunks = chunks_of(p);
    fork_count_kernel<<<rows + chunks, 256, 0, st>>>(a, rows);
    mark_kernel(st);
    if (int e = cuda_ok(cudaGetLastError(), "fork launch")) return e;
    return launch_copies(p, a, false, st);
}

int run_copy(const fa_pages_params& p) {
    if (p.num_pages <= 0 || p.page_size <= 0 || p.n < 0) return fail(FA_ERR_BAD_SHAPE, "negative or zero size");
    if (int e = check_views(p)) return e;
    if (p.n == 0 || p.num_caches == 0) return FA_OK;
    if (!p.rows || !p.rows2) return fail(FA_ERR_NULL, "src or dst is null");
    if (p.n > (1 << 24)) return fail(FA_ERR_BAD_SHAPE, "at most 2^24 pages a call");
    cudaStream_t st = reinterpret_cast<cudaStream_t>(p.stream);
    mark_kernel(st);
    return launch_copies(p, PoolArgs{}, true, st);
}

int run_compact(const fa_pages_params& p) {
    fa_pages_params q = p;
    if (!p.table) q.width = 1;
    if (q.b < 0 || q.n < 0 || q.width <= 0 || q.page_size <= 0 || q.num_pages <= 0 || q.b > (1 << 24)) return fail(FA_ERR_BAD_SHAPE, "negative or zero size");
    if ((long long)q.width * q.page_size > 0x7fffffff) return fail(FA_ERR_BAD_SHAPE, "a sequence holds at most 2^31 - 1 rows");
    if (q.table && q.cache_batch_idx) return fail(FA_ERR_UNSUPPORTED, "cache_batch_idx is not used with a paged cache");
    if (int e = check_views(q)) return e;
    if (q.num_caches == 0) return fail(FA_ERR_BAD_SHAPE, "no caches");
    if (q.b == 0) return FA_OK;
    if (int e = check_apart(q)) return e;
    if (!q.seqlens || !q.new_seqlens || (q.n > 0 && !q.rows)) return fail(FA_ERR_NULL, "cache_seqlens, kept or the output is null");
    if (q.new_seqlens == q.seqlens) return fail(FA_ERR_UNSUPPORTED, "the new lengths must be another tensor than the old ones");
    cudaStream_t st = reinterpret_cast<cudaStream_t>(q.stream);
    CompactArgs a;
    a.num_entries = q.num_pages; a.page_size = q.page_size; a.width = q.width;
    a.table = q.table; a.table_stride = q.table_stride; a.batch_idx = q.cache_batch_idx;
    a.seqlens = q.seqlens; a.kept = q.rows; a.kept_stride = q.rows_stride; a.counts = q.rows2;
    a.b = q.b; a.n = q.n; a.new_seqlens = q.new_seqlens;
    mark_kernel(st);
    for (int v0 = 0; v0 < q.num_caches; v0 += kMaxViews) {
        a.num_views = q.num_caches - v0 < kMaxViews ? q.num_caches - v0 : kMaxViews;
        a.first_launch = v0 == 0;
        int64_t warps = 0;
        for (int i = 0; i < a.num_views; ++i) {
            const View v = a.views[i] = view_of(q.caches[v0 + i]);
            warps += (int64_t)v.caches * ((v.heads * v.seg + 32 * v.vec - 1) / (32 * v.vec));
        }
        const int64_t blocks = (warps * q.b + 3) / 4;
        if (warps <= 0 || blocks >= (1ll << 31)) return fail(FA_ERR_BAD_SHAPE, "too many caches and sequences, or none");
        a.warps_seq = (int)warps;
        compact_kernel<<<(unsigned)blocks, 128, 0, st>>>(a);
        mark_kernel(st);
        if (int e = cuda_ok(cudaGetLastError(), "compact launch")) return e;
    }
    return FA_OK;
}

}  // namespace
}  // namespace fa

using namespace fa;

extern "C" {

int fa_pages_reserve(const fa_pages_params* p) { return p ? run_reserve(*p) : fail(FA_ERR_NULL, "params is null"); }
int fa_pages_free(const fa_pages_params* p) { return p ? run_free(*p) : fail(FA_ERR_NULL, "params is null"); }
int fa_pages_fork(const fa_pages_params* p) { return p ? run_fork(*p) : fail(FA_ERR_NULL, "params is null"); }
int fa_pages_copy(const fa_pages_params* p) { return p ? run_copy(*p) : fail(FA_ERR_NULL, "params is null"); }
int fa_cache_compact(const fa_pages_params* p) { return p ? run_compact(*p) : fail(FA_ERR_NULL, "params is null"); }
size_t fa_pages_workspace_bytes(int32_t rows, int32_t num_pages) {
    if (rows < 0 || num_pages <= 0) return 0;
    fa_pages_params p = {};
    p.num_pages = num_pages;
    return workspace(p, rows, nullptr);
}

}  // extern "C"
