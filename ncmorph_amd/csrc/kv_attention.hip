// Attention of a step's rows over the paged cache (ncm_kv_attention_dev).
//
// The products and the softmax are in kv_attention.h.
//
// Work: a request's (K/V head, block of 16 R pairs) is a unit of ceil(tokens /
// 128) tiles; all units' tiles in a row are cut into equal runs, one per
// workgroup, whatever the requests' lengths, its four wavefronts taking 32
// tokens of each tile. A unit inside one run is written out, the parts of one
// that is cut go to the workspace, and kv_attention_join_kernel adds them in
// order.
//
// 64 requests of 1044 to 8192 tokens, one row each, 32 heads over 8 of 128, fp8:
// 101 us (4.9 TB/s; a copy runs at 5.1), its join 4.7. 8 trees of 13 to 25 rows
// over 523 to 4000 tokens, int8: 34 us, join 5.3. Chunks of 256 rows over 8000
// tokens and of 186 over 2160, bf16: 129 us (318 TFLOP/s of unmasked products),
// join 7.0. Those two are bound by latency, in runs of a few tiles for the trees:
// per 32 tokens and 32 pairs a wavefront issues 305 (bf16) or 606 (int8) vector
// instructions, all included, and 48 MFMAs, which keep the vector pipes busy for
// 30% of the time and the matrix cores for 17 or 9%; wavefronts, 1.4 or 1.1 a
// SIMD, wait for loads, LDS or barriers for 36 or 39% of theirs. (head_dim 128,
// bf16, 32 pairs: all 256 registers and 10 spilled, none touched in the loop over
// tiles that every pair sees whole.)
#include "kv_attention.h"

namespace ncm {
namespace {

template <int R>
__device__ __forceinline__ Need need_of(const AttnArgs& a, int r) {
    Need d;
    d.q = request_of(a.batch, r);
    const int64_t cap = a.batch.capacity;
    d.end = (int)min((int64_t)d.q.before + d.q.n, cap);
    d.before = (int)min((int64_t)d.q.before, cap);
    d.base = d.floor = 0;
    const int64_t low = a.window > 0 ? max((int64_t)d.q.before - a.window + 1, (int64_t)0) : 0;
    d.tile0 = (int)(min(low, cap) / kTile);
    d.tiles = max((d.end + kTile - 1) / kTile - d.tile0, 1);
    d.blocks = (int)(((int64_t)d.q.n * a.group + 16 * R - 1) / (16 * R));
    return d;
}

// Two workgroups a CU. (Three, in 168 registers: 122 us against 105 then for 64
// requests of up to 8192 tokens, fp8: the runs are shorter, and a run begins
// with a chain of loads. Both of a tile's loads a round ahead, in a second
// tile's registers: 105, and 163 against 142 then for chunks of 256 rows.)
template <int HD, int CODES, int R>
__global__ __launch_bounds__(256, 2) void kv_attention_kernel(AttnArgs a) {
    __shared__ Lds<HD, R> lds;
    __shared__ int64_t wave_tiles[4], found_at;
    __shared__ int64_t wave_units[4], found_units;
    __shared__ int found;
    const int tid = threadIdx.x, lane = tid & 63, heads = a.cache.kv_heads;

    // Tiles and units ahead of each thread's share of the requests.
    const int per = (a.batch.requests + 255) / 256, r0 = tid * per;
    const int r1 = min(r0 + per, a.batch.requests);
    int64_t tiles = 0, units = 0;
    for (int r = r0; r < r1; ++r) {
        const Need d = need_of<R>(a, r);
        units += (int64_t)d.blocks * heads;
        tiles += (int64_t)d.blocks * heads * d.tiles;
    }
    int64_t t_sum = tiles, u_sum = units;
    for (int x = 1; x < 64; x <<= 1) {
        const int64_t t = __shfl_up(t_sum, x), u = __shfl_up(u_sum, x);
        if (lane >= x) t_sum += t, u_sum += u;
    }
    if (lane == 63) wave_tiles[tid >> 6] = t_sum, wave_units[tid >> 6] = u_sum;
    __syncthreads();
    int64_t all = 0, t_at = t_sum - tiles, all_units = 0, u_at = u_sum - units;
    for (int w = 0; w < 4; ++w) {
        if (w < (tid >> 6)) t_at += wave_tiles[w], u_at += wave_units[w];
        all += wave_tiles[w], all_units += wave_units[w];
    }
    all = uniform(all);
    // Runs of tiles: a workgroup each, at most one per tile; neighbours, which
    // may read the same K and V, on one XCD where every workgroup has a run.
    const int64_t groups = min((int64_t)gridDim.x, all);
    const int me = all >= gridDim.x ? xcd_remap(blockIdx.x, gridDim.x) : (int)blockIdx.x;
    if (blockIdx.x == 0 && tid == 0) *a.unit_count = (int)min(all_units, (int64_t)a.units);
    if (me >= groups) return;
    int64_t at = all * me / groups;
    const int64_t end = all * (me + 1) / groups;
    if (at >= t_at && at < t_at + tiles) {
        int r = r0;
        for (; r < r1 - 1; ++r) {
            const Need d = need_of<R>(a, r);
            const int64_t n = (int64_t)d.blocks * heads * d.tiles;
            if (at < t_at + n) break;
            t_at += n, u_at += (int64_t)d.blocks * heads;
        }
        found = r, found_at = t_at, found_units = u_at;
    }
    __syncthreads();
    int r = uniform(found);
    int64_t start = uniform(found_at), u0 = uniform(found_units);  // of the request
    while (at < end) {
        const Need d = need_of<R>(a, r);
        const int64_t n = (int64_t)d.blocks * heads * d.tiles;
        if (at >= start + n) {
            start += n, u0 += (int64_t)d.blocks * heads, ++r;
            continue;
        }
        const int u = (int)((at - start) / d.tiles);
        const int first = (int)((at - start) - (int64_t)u * d.tiles);
        const int count = (int)min((int64_t)(d.tiles - first), end - at);
        int slot = -1;
        if (first > 0) slot = 2 * me;
        else if (count < d.tiles) slot = 2 * me + 1;
        if (first == 0 && tid == 0 && u0 + u < a.units) {
            // The workgroup that has the unit's last tile ends it.
            const int64_t last = ((at + d.tiles) * groups - 1) / all;
            a.joins[u0 + u] = int4{me, (int)(last - me) + 1, r, u};
        }
        const int h = u / d.blocks;
        run_unit<HD, CODES, R, false>(a, d, r, h, u - h * d.blocks, first, count,
                                      slot < 0 ? -1 : (int64_t)slot * 16 * R, lds);
        at += count;
    }
}

// One workgroup per unit that was cut: per pair, its parts' sums brought to
// their common maximum and added, by a wavefront where they are few, else by
// all four.
template <int HD, int R>
__global__ __launch_bounds__(256) void kv_attention_join_kernel(AttnArgs a) {
    if ((int)blockIdx.x >= *a.unit_count) return;
    const int4 j = a.joins[blockIdx.x];
    const int parts = j.y;
    if (parts < 2) return;
    const Need d = need_of<R>(a, j.z);
    const int h = j.w / d.blocks, block = j.w - h * d.blocks;
    const int pairs = min(16 * R, d.q.n * a.group - block * 16 * R);
    constexpr int L = HD / 4;  // lanes of a part
    const bool few = parts <= 16;
    const int span = few ? 64 : 256, mine = threadIdx.x % span;
    const int lanes = mine % L, k0 = mine / L, step = span / L;
    __shared__ f32x4_t so[256];
    __shared__ float sm[256], sl[256];
    const int rows = 256 / span;
    for (int base = blockIdx.y * rows; base < pairs; base += gridDim.y * rows) {
        const int pr = base + threadIdx.x / span;
        float m = kNoMax, l = 0.0f;
        f32x4_t o = {0.0f, 0.0f, 0.0f, 0.0f};
        if (pr < pairs) {
#pragma unroll 4
            for (int k = k0; k < parts; k += step) {
                const int64_t at = (int64_t)(k == 0 ? 2 * j.x + 1 : 2 * (j.x + k)) * 16 * R + pr;
                const float2 ml = a.part_ml[at];
                const f32x4_t v = *(const f32x4_t*)(a.part_o + at * HD + 4 * lanes);
                const float top = fmaxf(m, ml.x);
                const float f = __builtin_amdgcn_exp2f(m - top), e = __builtin_amdgcn_exp2f(ml.x - top);
                l = l * f + ml.y * e;
                o = o * f + v * e;
                m = top;
            }
        }
        so[threadIdx.x] = o, sm[threadIdx.x] = m, sl[threadIdx.x] = l;
        __syncthreads();
        if (k0 == 0 && pr < pairs) {
            for (int k = 1; k < step; ++k) {
                const int x = threadIdx.x + k * L;
                const float top = fmaxf(m, sm[x]);
                const float f = __builtin_amdgcn_exp2f(m - top), e = __builtin_amdgcn_exp2f(sm[x] - top);
                l = l * f + sl[x] * e;
                o = o * f + so[x] * e;
                m = top;
            }
            const int pair = block * 16 * R + pr;
            const int row = pair / a.group, head = h * a.group + pair - row * a.group;
            const float inv = l == 0.0f ? 0.0f : 1.0f / l;
            const u32x2_t b = {bf16x2_bits_rne(o[0] * inv, o[1] * inv),
                               bf16x2_bits_rne(o[2] * inv, o[3] * inv)};
            *(u32x2_t*)(a.out + (d.q.o0 + row) * a.out_stride + (int64_t)head * HD + 4 * lanes) = b;
        }
        __syncthreads();
    }
}

// How a step is laid out: by its sizes alone, so that the workspace's size and
// the launch agree.
struct Layout {
    int r16;            // R
    int64_t units;      // at most
    int64_t groups;     // workgroups
    bool cut;           // whether a unit can be
    int64_t some;       // requests that may have rows
    size_t joins, ml, o, bytes;  // offsets in the workspace
};

Layout layout_of(const ncm_kv_cache_t& c, const ncm_kv_batch_t& b, int q_heads) {
    Layout s;
    const int64_t group = q_heads / c.kv_heads, pairs = b.rows * group;
    const int64_t some = std::max<int64_t>(1, std::min(b.requests, b.rows));
    // 16 R pairs a unit. R = 2 where requests have more than 16 on average: each
    // token's codes are loaded and widened once for twice the pairs. R = 1 and 2:
    // 38 and 34 us for 8 trees of up to 25 rows and 4 heads over up to 4000 tokens,
    // int8, 212 and 129 for chunks of 256 and 186 rows over 8000 and 2160, bf16;
    // with one row a request, 101 and 112 for 64 of them, fp8, 7.5 and 9.6 for one
    // over 777 tokens. (R = 4, one wavefront a SIMD, when R = 2 took 36 and 143: 53
    // for the trees, 148 for the chunks.)
    s.r16 = pairs <= 16 * some ? 1 : 2;
    s.some = some;
    s.units = (pairs / (16 * s.r16) + some) * c.kv_heads;
    const int64_t tiles = std::max<int64_t>(1, ((b.table_width * c.page_size) + kTile - 1) / kTile);
    s.cut = tiles > 1;
    s.groups = std::min<int64_t>(s.units * tiles, 2 * kCus);
    const size_t slots = 2 * (size_t)s.groups * 16 * s.r16;
    s.joins = 16;
    s.ml = s.joins + 16 * (size_t)s.units;
    s.o = s.ml + (slots * 8 + 15) / 16 * 16;
    s.bytes = s.o + slots * c.head_dim * 4;
    return s;
}

template <int HD, int CODES, int R>
hipError_t launch(const AttnArgs& a, const Layout& s, hipStream_t st) {
    kv_attention_kernel<HD, CODES, R><<<(uint32_t)s.groups, 256, 0, st>>>(a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || !s.cut) return e;
    // A workgroup per pair where few units are cut into many parts, else per
    // four; of the pairs that a request has on average (the others' wait).
    const int64_t pairs = std::min<int64_t>(16 * R, (a.batch.rows * a.group + s.some - 1) / s.some);
    const uint32_t y = (uint32_t)(s.units * 8 <= s.groups ? pairs : (pairs + 3) / 4);
    kv_attention_join_kernel<HD, R><<<dim3((uint32_t)s.units, y), 256, 0, st>>>(a);
    return hipGetLastError();
}

template <int HD, int CODES>
hipError_t launch_r(const AttnArgs& a, const Layout& s, hipStream_t st) {
    return s.r16 == 1 ? launch<HD, CODES, 1>(a, s, st) : launch<HD, CODES, 2>(a, s, st);
}

int check_attention(const ncm_kv_cache_t* cache, const ncm_kv_batch_t* batch, int q_heads,
                    AttnArgs* a) {
    int rc = check_cache(cache, &a->cache);
    if (rc) return rc;
    rc = check_batch(batch, a->cache.page_log2, &a->batch);
    if (rc) return rc;
    if (q_heads < 1 || q_heads > 65535 || q_heads % cache->kv_heads ||
        batch->rows * q_heads > 0x7FFFFFFF)
        return NCM_E_SHAPE;
    // The join's launch has a workgroup per unit.
    if (layout_of(*cache, *batch, q_heads).units > kMaxBlocks) return NCM_E_SHAPE;
    a->q_heads = q_heads;
    a->group = q_heads / cache->kv_heads;
    return NCM_OK;
}

}  // namespace
}  // namespace ncm

extern "C" int ncm_kv_attention_workspace(const ncm_kv_cache_t* cache,
                                          const ncm_kv_batch_t* batch, int q_heads,
                                          size_t* bytes) {
    using namespace ncm;
    if (!bytes) return NCM_E_NULL;
    *bytes = 0;
    AttnArgs a = {};
    const int rc = check_attention(cache, batch, q_heads, &a);
    if (rc) return rc;
    if (batch->rows > 0 && batch->requests > 0) *bytes = layout_of(*cache, *batch, q_heads).bytes;
    return NCM_OK;
}

extern "C" int ncm_kv_attention_dev(ncm_ctx_t* ctx, const ncm_kv_cache_t* cache,
                                    const ncm_kv_batch_t* batch, const uint16_t* q, uint16_t* out,
                                    int q_heads, int64_t q_stride, int64_t out_stride,
                                    float scale, int64_t window, const int32_t* positions,
                                    const uint64_t* tree_mask, int64_t mask_words,
                                    void* workspace, size_t workspace_bytes) {
    using namespace ncm;
    if (!ctx) return NCM_E_NULL;
    AttnArgs a = {};
    int rc = check_attention(cache, batch, q_heads, &a);
    if (rc) return rc;
    if (window < 0 || mask_words < 0 || mask_words > kMaxRows / 2) return NCM_E_SHAPE;
    if (batch->rows == 0 || batch->requests == 0) return NCM_OK;
    const int64_t width = (int64_t)q_heads * cache->head_dim;
    rc = check_rows(q, q_stride, width);
    if (!rc) rc = check_rows(out, out_stride, width);
    if (rc) return rc;
    const Layout s = layout_of(*cache, *batch, q_heads);
    // Offsets may give every request all rows: the tiles must still be counted
    // in 64 bits, times the workgroups.
    const double most = ((double)batch->rows * q_heads / 16 + cache->kv_heads) * batch->requests *
                        ((double)a.batch.capacity / kTile + 1);
    if (most > 0x1p50) return NCM_E_SHAPE;
    if (!workspace) return NCM_E_NULL;
    if (workspace_bytes < s.bytes) return NCM_E_LENGTH;
    if ((uintptr_t)workspace % 16) return NCM_E_ARG;
    char* ws = (char*)workspace;
    a.q = q, a.out = out, a.positions = positions, a.tree_mask = (const uint32_t*)tree_mask;
    a.q_stride = q_stride, a.out_stride = out_stride, a.window = window;
    a.mask_words = mask_words, a.scale = scale;
    a.units = (int)s.units;
    a.unit_count = (int*)ws;
    a.joins = (int4*)(ws + s.joins);
    a.part_ml = (float2*)(ws + s.ml);
    a.part_o = (float*)(ws + s.o);
    const DeviceScope scope(ncm_ctx_device(ctx));
    rc = step_hip(scope.error(), "kv_attention device");
    if (rc) return rc;
    const hipStream_t st = ncm_ctx_stream(ctx);
    const bool wide = cache->head_dim == 128;
    hipError_t e;
    switch (cache->codes) {
        case NCM_KV_BF16:
            e = wide ? launch_r<128, NCM_KV_BF16>(a, s, st) : launch_r<64, NCM_KV_BF16>(a, s, st);
            break;
        case NCM_KV_FP8:
            e = wide ? launch_r<128, NCM_KV_FP8>(a, s, st) : launch_r<64, NCM_KV_FP8>(a, s, st);
            break;
        default:
            e = wide ? launch_r<128, NCM_KV_INT8>(a, s, st) : launch_r<64, NCM_KV_INT8>(a, s, st);
    }
    return step_hip(e, "kv_attention launch");
}
