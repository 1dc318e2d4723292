// The pages of a cache's sequences and the tables of a step, built from the
// requests' lengths (ncm_pages_share_dev, ncm_pages_extend_dev,
// ncm_pages_release_dev).
//
// Request r holds pages 0 .. ceil(tokens / P) - 1 of its table, so what a step
// takes and what a release gives back are differences of such counts, and the
// place of every page on the free stack is a prefix sum over the requests: no
// order of arrival decides anything. A release undoes the extension that it
// follows, down to the stack's order.
//
// A few bytes a row and a page: bound by the launches and the chain of loads in
// each. 48 requests: extend 6.6 us, release 2.8 + 3.0 + 3.2; 200 prompts of about
// 500 tokens behind 2000 shared ones: share 7.1, extend 5.0 + 4.8, release 9.1 +
// 3.3 + 4.9.
//
// Up to 1024 requests and 2048 rows are extended by one workgroup in one launch
// (1024 requests of one row: 6.6 us, 8.8 in two; 16 of 128: 5.9, 6.9), more by one
// that scans the requests and others that fill rows and pages (1024 of 4: 8.9 us,
// 9.9 in one; 16 of 256: 6.9, 7.5).
#include "step.h"

namespace ncm {
namespace {

constexpr int kOneRequests = 1024, kOneRows = 2048;

struct PoolView {
    int32_t* free;
    int32_t* count;
    int32_t* refs;
    unsigned long long* marks;
    int32_t pages;
};

struct PageArgs {
    PoolView pool;  // free NULL: none
    int32_t* table;
    int64_t stride;
    int32_t requests, width, log2;
};

__device__ __forceinline__ int tokens_of(int v) { return min(max(v, 0), (int)kMaxTokens); }
// Pages that t tokens take, at most the table's.
__device__ __forceinline__ int pages_of(int64_t t, const PageArgs& a) {
    return (int)min((t + (1 << a.log2) - 1) >> a.log2, (int64_t)a.width);
}
__device__ __forceinline__ int held_count(const PoolView& p) { return min(max(*p.count, 0), p.pages); }
// The page that rank takes from a stack of `base`, or -1.
__device__ __forceinline__ int taken(const PoolView& p, int base, int rank) {
    if (rank >= base) return -1;
    const int id = p.free[base - 1 - rank];
    return (uint32_t)id < (uint32_t)p.pages ? id : -1;
}

struct ExtendArgs {
    PageArgs p;
    const int32_t* added;
    const int32_t* starts;
    const uint64_t* tree_mask;
    int64_t mask_words;
    int32_t rows;
    int32_t* offsets;    // [requests + 1]
    int32_t* positions;  // [rows]
    int64_t* slots;      // [rows]
    int32_t* missing;    // [1]
    int32_t* space;      // [requests + 2]: pages taken before each request, in all; the stack's height
};

// Exclusive prefix sums of v over 1024 threads; total: of all.
__device__ __forceinline__ int64_t scan(int64_t v, int64_t (&waves)[16], int64_t& total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int64_t s = v;
    for (int x = 1; x < 64; x <<= 1) {
        const int64_t o = __shfl_up(s, x);
        if (lane >= x) s += o;
    }
    __syncthreads();
    if (lane == 63) waves[wave] = s;
    __syncthreads();
    int64_t before = 0;
    total = 0;
    for (int w = 0; w < 16; ++w) {
        before += w < wave ? waves[w] : 0;
        total += waves[w];
    }
    return before + s - v;
}

// The last r with at[r] <= x: x below at[requests].
__device__ __forceinline__ int find(const int32_t* at, int requests, int x) {
    int lo = 0, hi = requests;
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        (at[mid] <= x ? lo : hi) = mid;
    }
    return lo;
}

// Whether the row is a request's first and begins inside a page with more than one
// holder: what it would write there others read.
__device__ __forceinline__ bool fill_row(const ExtendArgs& a, const int32_t* offsets,
                                         const int32_t* ahead, int base, int row) {
    int position = 0;
    int64_t slot = -1;
    bool refused = false;
    if (row < offsets[a.p.requests]) {
        const int r = find(offsets, a.p.requests, row), i = row - offsets[r];
        const int n = offsets[r + 1] - offsets[r], start = tokens_of(a.starts[r]);
        const int64_t t = (int64_t)start + i;
        position = (int)min(t, (int64_t)0x7FFFFFFF);
        if (a.tree_mask) {
            int bits = 0;
            for (int w = 0; w < a.mask_words && 64 * w < n; ++w) {
                uint64_t m = a.tree_mask[row * a.mask_words + w];
                if (n - 64 * w < 64) m &= (uint64_t(1) << (n - 64 * w)) - 1;
                bits += __popcll(m);
            }
            position = start + max(bits - 1, 0);
        }
        const int64_t page = t >> a.p.log2;
        if (page < a.p.width) {
            const int first = pages_of(start, a.p);
            const bool fresh = a.p.pool.free && page >= first;
            const int id = fresh ? taken(a.p.pool, base, ahead[r] + (int)page - first)
                                 : a.p.table[r * a.p.stride + page];
            const bool there = id >= 0 && (!a.p.pool.free || id < a.p.pool.pages);
            const bool others = there && a.p.pool.free && !fresh && a.p.pool.refs[id] > 1;
            if (there && !others) slot = ((int64_t)id << a.p.log2) + (t & ((1 << a.p.log2) - 1));
            refused = others && i == 0;
        }
    }
    a.positions[row] = position;
    a.slots[row] = slot;
    return refused;
}

__device__ __forceinline__ void fill_page(const ExtendArgs& a, const int32_t* ahead, int base,
                                          int rank) {
    const int r = find(ahead, a.p.requests, rank);
    const int id = taken(a.p.pool, base, rank);
    a.p.table[r * a.p.stride + pages_of(tokens_of(a.starts[r]), a.p) + rank - ahead[r]] = id;
    if (id >= 0) a.p.pool.refs[id] = 1;
}

// Offsets and the pages ahead of each request, by one workgroup of 1024; ONE:
// the rows and the pages too.
template <bool ONE>
__global__ __launch_bounds__(1024) void extend_scan_kernel(ExtendArgs a) {
    __shared__ int64_t waves[16];
    __shared__ int32_t near_offsets[ONE ? kOneRequests + 1 : 1], near_ahead[ONE ? kOneRequests + 1 : 1];
    __shared__ int refused;
    const int requests = a.p.requests, per = (requests + 1023) / 1024;
    const int r0 = min((int)threadIdx.x * per, requests), r1 = min(r0 + per, requests);
    int32_t* ahead = ONE ? near_ahead : a.space;
    const int base = a.p.pool.free ? held_count(a.p.pool) : 0;
    int64_t mine = 0, all;
    for (int r = r0; r < r1; ++r) mine += max(a.added[r], 0);
    int64_t at = scan(mine, waves, all);
    auto clipped = [&](int64_t x) { return (int)min(x, (int64_t)a.rows); };
    // New pages of the thread's requests, their rows cut at `rows`.
    auto fresh = [&](int r, int64_t o) {
        const int n = clipped(o + max(a.added[r], 0)) - clipped(o);
        const int start = tokens_of(a.starts[r]);
        return pages_of((int64_t)start + n, a.p) - pages_of(start, a.p);
    };
    mine = 0;
    int64_t o = at;
    for (int r = r0; r < r1; ++r) {
        a.offsets[r] = clipped(o);
        if (ONE) near_offsets[r] = clipped(o);
        if (a.p.pool.free) mine += fresh(r, o);
        o += max(a.added[r], 0);
    }
    int64_t taken_in_all;
    int64_t rank = scan(mine, waves, taken_in_all);
    o = at;
    for (int r = r0; r < r1; ++r) {
        ahead[r] = (int)rank;
        if (a.p.pool.free) rank += fresh(r, o);
        o += max(a.added[r], 0);
    }
    if (threadIdx.x == 0) {
        a.offsets[requests] = clipped(all);
        if (ONE) near_offsets[requests] = clipped(all);
        ahead[requests] = (int)taken_in_all;
        if (!ONE) a.space[requests + 1] = base;
        if (ONE) refused = 0;
        *a.missing = (int)max(taken_in_all - base, (int64_t)0);
    }
    __syncthreads();
    // Every thread has read the height.
    if (threadIdx.x == 0 && a.p.pool.free) *a.p.pool.count = (int)max(base - taken_in_all, (int64_t)0);
    if constexpr (ONE) {
        for (int row = threadIdx.x; row < a.rows; row += 1024)
            if (fill_row(a, near_offsets, near_ahead, base, row)) atomicAdd(&refused, 1);
        for (int e = threadIdx.x; e < (int)taken_in_all; e += 1024) fill_page(a, near_ahead, base, e);
        __syncthreads();
        if (threadIdx.x == 0 && refused)
            *a.missing = (int)max(taken_in_all - base, (int64_t)0) + refused;
    }
}

__global__ __launch_bounds__(256) void extend_fill_kernel(ExtendArgs a, int row_blocks) {
    const int base = a.space[a.p.requests + 1];
    const int i = (int)(blockIdx.x * 256 + threadIdx.x);
    if ((int)blockIdx.x < row_blocks) {
        if (i < a.rows && fill_row(a, a.offsets, a.space, base, i)) atomicAdd(a.missing, 1);
    } else if (i - row_blocks * 256 < a.space[a.p.requests]) {
        fill_page(a, a.space, base, i - row_blocks * 256);
    }
}

__global__ __launch_bounds__(256) void share_kernel(PageArgs a, const int32_t* sources,
                                                    const int32_t* tokens) {
    for (int r = blockIdx.x; r < a.requests; r += gridDim.x) {
        const int from = sources[r];
        if (from == r || (uint32_t)from >= (uint32_t)a.requests) continue;
        const int n = min(tokens_of(tokens[r]) >> a.log2, a.width);
        for (int i = threadIdx.x; i < n; i += 256) {
            const int id = a.table[from * a.stride + i];
            const bool there = (uint32_t)id < (uint32_t)a.pool.pages;
            a.table[r * a.stride + i] = there ? id : -1;
            if (there) atomicAdd(&a.pool.refs[id], 1);
        }
    }
}

// A release in three launches. Its entries are (request, page of its table); a
// page goes back to the stack once, for the first of its entries, where the
// release takes its last holder away. While one runs, refs is kGone less than 0
// for such a page and marks holds its first entry.
constexpr int kGone = 0x40000000;
constexpr unsigned long long kNoMark = ~0ull >> 1;

struct ReleaseArgs {
    PageArgs p;
    const int32_t* lens;
    const int32_t* keep;
    int32_t* space;  // [requests + 2]: pages that go back, of each request; the stack's height
};

struct Part {
    int first, n;  // entries of a request's table
};
__device__ __forceinline__ Part part_of(const ReleaseArgs& a, int r) {
    const int len = tokens_of(a.lens[r]), keep = min(tokens_of(a.keep[r]), len);
    const int first = pages_of(keep, a.p);
    return {first, pages_of(len, a.p) - first};
}
__device__ __forceinline__ unsigned long long entry_of(int r, int i) {
    return ((unsigned long long)r << 32) | (unsigned)i;
}
__device__ __forceinline__ int entry_id(const ReleaseArgs& a, int r, int i) {
    const int id = a.p.table[r * a.p.stride + i];
    return (uint32_t)id < (uint32_t)a.p.pool.pages ? id : -1;
}

__global__ __launch_bounds__(256) void release_mark_kernel(ReleaseArgs a) {
    if (blockIdx.x == 0 && threadIdx.x == 0) a.space[a.p.requests + 1] = held_count(a.p.pool);
    for (int r = blockIdx.x; r < a.p.requests; r += gridDim.x) {
        const Part d = part_of(a, r);
        for (int i = threadIdx.x; i < d.n; i += 256) {
            const int id = entry_id(a, r, d.first + i);
            if (id < 0) continue;
            atomicMin(&a.p.pool.marks[id], entry_of(r, i));
            // Only as many entries as the page has holders see more than 0.
            const int had = atomicSub(&a.p.pool.refs[id], 1);
            if (had <= 0) atomicAdd(&a.p.pool.refs[id], 1);
            else if (had == 1) atomicSub(&a.p.pool.refs[id], kGone);
        }
    }
}

// Whether entry i of request r is the one that puts its page back.
__device__ __forceinline__ bool goes_back(const ReleaseArgs& a, int id, int r, int i) {
    return id >= 0 && a.p.pool.marks[id] == entry_of(r, i) && a.p.pool.refs[id] <= -kGone / 2;
}

__global__ __launch_bounds__(256) void release_count_kernel(ReleaseArgs a) {
    __shared__ int waves[4];
    for (int r = blockIdx.x; r < a.p.requests; r += gridDim.x) {
        const Part d = part_of(a, r);
        int n = 0;
        for (int i = threadIdx.x; i < d.n; i += 256)
            n += goes_back(a, entry_id(a, r, d.first + i), r, i);
        for (int x = 32; x; x >>= 1) n += __shfl_xor(n, x);
        __syncthreads();
        if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = n;
        __syncthreads();
        if (threadIdx.x == 0) a.space[r] = waves[0] + waves[1] + waves[2] + waves[3];
    }
}

// Each workgroup a run of requests, behind the pages of all requests after it:
// the first entry's page ends on the stack's top.
__global__ __launch_bounds__(256) void release_push_kernel(ReleaseArgs a) {
    __shared__ int sums[2][4], there[4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, requests = a.p.requests;
    const int r0 = (int)((int64_t)requests * blockIdx.x / gridDim.x);
    const int r1 = (int)((int64_t)requests * (blockIdx.x + 1) / gridDim.x);
    int all = 0, before = 0;
    for (int r = threadIdx.x; r < requests; r += 256) {
        const int n = a.space[r];
        all += n;
        before += r < r0 ? n : 0;
    }
    for (int x = 32; x; x >>= 1) all += __shfl_xor(all, x), before += __shfl_xor(before, x);
    if (lane == 0) sums[0][wave] = all, sums[1][wave] = before;
    __syncthreads();
    all = sums[0][0] + sums[0][1] + sums[0][2] + sums[0][3];
    before = sums[1][0] + sums[1][1] + sums[1][2] + sums[1][3];
    const int base = a.space[requests + 1];
    const int top = min(base + all, a.p.pool.pages) - 1;
    if (blockIdx.x == 0 && threadIdx.x == 0) *a.p.pool.count = top + 1;
    for (int r = r0; r < r1; ++r) {
        const Part d = part_of(a, r);
        for (int i0 = 0; i0 < d.n; i0 += 256) {
            const int i = i0 + threadIdx.x;
            const int id = i < d.n ? entry_id(a, r, d.first + i) : -1;
            const bool mine = id >= 0 && a.p.pool.marks[id] == entry_of(r, i);
            const bool back = mine && a.p.pool.refs[id] <= -kGone / 2;
            const uint64_t lanes = __ballot(back);
            __syncthreads();
            if (lane == 0) there[wave] = __popcll(lanes);
            __syncthreads();
            int rank = before + __popcll(lanes & ((uint64_t(1) << lane) - 1));
            for (int w = 0; w < wave; ++w) rank += there[w];
            if (back) {
                if (top - rank >= 0) a.p.pool.free[top - rank] = id;
                a.p.pool.refs[id] = 0;
            }
            if (mine) a.p.pool.marks[id] = kNoMark;
            if (i < d.n) a.p.table[r * a.p.stride + d.first + i] = -1;
            before += there[0] + there[1] + there[2] + there[3];
        }
    }
}

int check_pages(const ncm_page_pool_t* pool, bool needed, int32_t* table, int64_t requests,
                int64_t width, int64_t stride, int page_size, PageArgs* a) {
    if (requests < 0 || requests > kMaxRequests || width < 0 || width > 0x7FFFFFFF ||
        stride < width || stride > (int64_t(1) << 40))
        return NCM_E_SHAPE;
    int log2 = 4;
    while (log2 < 10 && (1 << log2) != page_size) ++log2;
    if ((1 << log2) != page_size || width << log2 > kMaxTokens) return NCM_E_SHAPE;
    if (needed && !pool) return NCM_E_NULL;
    if (pool) {
        if (pool->pages < 1 || pool->pages > kMaxTokens) return NCM_E_SHAPE;
        if (!pool->free || !pool->count || !pool->refs || !pool->marks) return NCM_E_NULL;
        if ((uintptr_t)pool->marks % 8) return NCM_E_ARG;
        a->pool = {pool->free, pool->count, pool->refs, (unsigned long long*)pool->marks,
                   (int32_t)pool->pages};
    }
    if (requests > 0 && width > 0 && !table) return NCM_E_NULL;
    a->table = table, a->stride = stride;
    a->requests = (int32_t)requests, a->width = (int32_t)width, a->log2 = log2;
    return NCM_OK;
}

}  // namespace
}  // namespace ncm

extern "C" int ncm_pages_share_dev(ncm_ctx_t* ctx, const ncm_page_pool_t* pool, int32_t* page_table,
                                   const int32_t* sources, const int32_t* tokens, int64_t requests,
                                   int64_t table_width, int64_t table_stride, int page_size) {
    using namespace ncm;
    if (!ctx) return NCM_E_NULL;
    PageArgs a = {};
    int rc = check_pages(pool, true, page_table, requests, table_width, table_stride, page_size, &a);
    if (rc) return rc;
    if (requests == 0 || table_width == 0) return NCM_OK;
    if (!sources || !tokens) return NCM_E_NULL;
    const DeviceScope scope(ncm_ctx_device(ctx));
    rc = step_hip(scope.error(), "pages_share device");
    if (rc) return rc;
    share_kernel<<<(uint32_t)std::min<int64_t>(requests, 1024), 256, 0, ncm_ctx_stream(ctx)>>>(
        a, sources, tokens);
    return step_hip(hipGetLastError(), "pages_share launch");
}

extern "C" int ncm_pages_extend_dev(ncm_ctx_t* ctx, const ncm_page_pool_t* pool,
                                    const int32_t* added, const int32_t* starts,
                                    int32_t* page_table, int64_t requests, int64_t table_width,
                                    int64_t table_stride, int page_size, int64_t rows,
                                    const uint64_t* tree_mask, int64_t mask_words, int32_t* offsets,
                                    int32_t* positions, int64_t* slots, int32_t* missing,
                                    int32_t* workspace) {
    using namespace ncm;
    if (!ctx) return NCM_E_NULL;
    ExtendArgs a = {};
    int rc = check_pages(pool, false, page_table, requests, table_width, table_stride, page_size,
                         &a.p);
    if (rc) return rc;
    if (rows < 0 || rows > kMaxRows || mask_words < 0 || mask_words > kMaxRows / 2)
        return NCM_E_SHAPE;
    if (!offsets || !missing || (rows > 0 && (!positions || !slots)) ||
        (requests > 0 && (!added || !starts)) || !workspace)
        return NCM_E_NULL;
    if ((uintptr_t)slots % 8 || (uintptr_t)tree_mask % 8) return NCM_E_ARG;
    a.added = added, a.starts = starts, a.tree_mask = tree_mask, a.mask_words = mask_words;
    a.rows = (int32_t)rows, a.offsets = offsets, a.positions = positions, a.slots = slots;
    a.missing = missing, a.space = workspace;
    const DeviceScope scope(ncm_ctx_device(ctx));
    rc = step_hip(scope.error(), "pages_extend device");
    if (rc) return rc;
    const hipStream_t st = ncm_ctx_stream(ctx);
    if (requests <= kOneRequests && rows <= kOneRows) {
        extend_scan_kernel<true><<<1, 1024, 0, st>>>(a);
        return step_hip(hipGetLastError(), "pages_extend launch");
    }
    extend_scan_kernel<false><<<1, 1024, 0, st>>>(a);
    rc = step_hip(hipGetLastError(), "pages_extend launch");
    if (rc) return rc;
    // A request's pages: those its rows fill and one that they begin.
    const int64_t most = pool ? (rows >> a.p.log2) + requests : 0;
    const int64_t row_blocks = (rows + 255) / 256, page_blocks = (most + 255) / 256;
    if (row_blocks + page_blocks > 0)
        extend_fill_kernel<<<(uint32_t)(row_blocks + page_blocks), 256, 0, st>>>(a, (int)row_blocks);
    return step_hip(hipGetLastError(), "pages_extend launch");
}

extern "C" int ncm_pages_release_dev(ncm_ctx_t* ctx, const ncm_page_pool_t* pool,
                                     int32_t* page_table, const int32_t* lens, const int32_t* keep,
                                     int64_t requests, int64_t table_width, int64_t table_stride,
                                     int page_size, int32_t* workspace) {
    using namespace ncm;
    if (!ctx) return NCM_E_NULL;
    ReleaseArgs a = {};
    int rc = check_pages(pool, true, page_table, requests, table_width, table_stride, page_size,
                         &a.p);
    if (rc) return rc;
    if (requests == 0 || table_width == 0) return NCM_OK;
    if (!lens || !keep || !workspace) return NCM_E_NULL;
    a.lens = lens, a.keep = keep, a.space = workspace;
    const DeviceScope scope(ncm_ctx_device(ctx));
    rc = step_hip(scope.error(), "pages_release device");
    if (rc) return rc;
    const hipStream_t st = ncm_ctx_stream(ctx);
    const uint32_t blocks = (uint32_t)std::min<int64_t>(requests, 1024);
    release_mark_kernel<<<blocks, 256, 0, st>>>(a);
    release_count_kernel<<<blocks, 256, 0, st>>>(a);
    release_push_kernel<<<blocks, 256, 0, st>>>(a);
    return step_hip(hipGetLastError(), "pages_release launch");
}
