// Attention over the paged cache of requests that share prefixes
// (ncm_kv_attention_shared_dev). The products and the softmax are in
// kv_attention.h.
//
// A group's requests hold the same tokens up to shared[g]. The rows of all of
// them against those tokens are one problem, which reads the prefix once for 16
// RP (row, head) pairs, whoever's they are, and has the matrix cores' columns
// full; each request's rows against its own tokens are another. Both give
// unnormalised sums with their maxima, which the join brings together.
//
// Work: units of (K/V head, block of pairs), the groups' first and the requests'
// behind them, of tiles of 128 tokens; all tiles in a row are cut into equal
// runs, one per workgroup. Every unit that is not whole in one run, and every
// unit of rows that have a prefix, goes to the workspace in parts.
#include "kv_attention.h"

namespace ncm {
namespace {

struct SharedArgs {
    AttnArgs a;
    const int32_t* groups;  // [n_groups + 1]
    const int32_t* shared;  // [n_groups]
    int n_groups;
    int prefix_units, own_units;  // there is room for
    int* counts;                  // units there are: the groups', the requests'
    int* unit_base;               // of a group
    int4* joins;                  // {first workgroup, parts, segment, unit of the segment}
    int64_t whole_prefix, whole_own;  // rows of the parts of units in one run
};

// Group g's requests [r0, r1) and the tokens that they share; none where there
// is nothing to share them with.
struct Group {
    int r0, r1, tokens;
};
__device__ __forceinline__ Group group_of(const SharedArgs& s, int g) {
    Group q;
    q.r0 = min(max(s.groups[g], 0), s.a.batch.requests);
    q.r1 = min(max(s.groups[g + 1], q.r0), s.a.batch.requests);
    q.tokens = q.r1 - q.r0 < 2
                   ? 0
                   : (int)min((int64_t)max(s.shared[g], 0), s.a.batch.capacity);
    return q;
}
// The group of request r, or -1.
__device__ __forceinline__ int group_with(const SharedArgs& s, int r) {
    int lo = 0, hi = s.n_groups;  // the first group that ends behind r
    while (lo < hi) {
        const int mid = (lo + hi) / 2;
        if (s.groups[mid + 1] > r) hi = mid;
        else lo = mid + 1;
    }
    return lo < s.n_groups && s.groups[lo] <= r ? lo : -1;
}

// Tokens of request r that it reads through its group.
__device__ __forceinline__ int prefix_of(const SharedArgs& s, int r, int before) {
    const int g = group_with(s, r);
    return g < 0 ? 0 : min(group_of(s, g).tokens, before);
}

template <int RP>
__device__ __forceinline__ Need group_need(const SharedArgs& s, int g) {
    const Group q = group_of(s, g);
    const AttnArgs& a = s.a;
    Need d;
    d.q.o0 = d.q.n = 0;
    d.q.before = d.end = d.before = q.tokens;
    d.base = d.floor = d.tile0 = 0;
    if (q.tokens > 0) {
        d.q.o0 = min(max(a.batch.offsets[q.r0], 0), a.batch.rows);
        d.q.n = max(min(a.batch.offsets[q.r1], a.batch.rows) - d.q.o0, 0);
        if (a.window > 0) {
            int least = q.tokens;
            for (int r = q.r0; r < q.r1; ++r) least = min(least, max(a.batch.starts[r], 0));
            d.tile0 = (int)(max((int64_t)least - a.window + 1, (int64_t)0) / kTile);
        }
    }
    d.tiles = max((d.end + kTile - 1) / kTile - d.tile0, 1);
    d.blocks = (int)(((int64_t)d.q.n * a.group + 16 * RP - 1) / (16 * RP));
    return d;
}

template <int RO>
__device__ __forceinline__ Need own_need(const SharedArgs& s, int r) {
    const AttnArgs& a = s.a;
    const int64_t cap = a.batch.capacity;
    Need d;
    d.q = request_of(a.batch, r);
    d.end = (int)min((int64_t)d.q.before + d.q.n, cap);
    d.before = (int)min((int64_t)d.q.before, cap);
    d.floor = prefix_of(s, r, d.before);
    const int64_t low = a.window > 0 ? max((int64_t)d.q.before - a.window + 1, (int64_t)0) : 0;
    d.base = (int)max((int64_t)d.floor, min(low, cap)) & ~15;
    d.tile0 = 0;
    d.tiles = max((d.end - d.base + kTile - 1) / kTile, 1);
    d.blocks = (int)(((int64_t)d.q.n * a.group + 16 * RO - 1) / (16 * RO));
    return d;
}

template <int RP, int RO>
__device__ __forceinline__ Need segment_need(const SharedArgs& s, int seg) {
    return seg < s.n_groups ? group_need<RP>(s, seg) : own_need<RO>(s, seg - s.n_groups);
}

// RP and RO: 16 pairs of a group's and of a request's unit.
template <int HD, int CODES, int RP, int RO>
__global__ __launch_bounds__(256, 2) void kv_attention_shared_kernel(SharedArgs s) {
    static_assert(RP >= RO, "one unit's LDS and parts hold the other's");
    __shared__ Lds<HD, RP> lds;
    __shared__ int64_t wave_tiles[4], wave_units[4], wave_prefix[4], found_at, found_units;
    __shared__ int found;
    const AttnArgs& a = s.a;
    const int tid = threadIdx.x, lane = tid & 63, heads = a.cache.kv_heads;
    const int segments = s.n_groups + a.batch.requests;

    // Tiles and units ahead of each thread's share of the segments.
    const int per = (segments + 255) / 256, s0 = min(tid * per, segments);
    const int s1 = min(s0 + per, segments);
    int64_t tiles = 0, units = 0, prefix = 0;
    for (int x = s0; x < s1; ++x) {
        const Need d = segment_need<RP, RO>(s, x);
        units += (int64_t)d.blocks * heads;
        prefix += x < s.n_groups ? (int64_t)d.blocks * heads : 0;
        tiles += (int64_t)d.blocks * heads * d.tiles;
    }
    int64_t t_sum = tiles, u_sum = units, p_sum = prefix;
    for (int x = 1; x < 64; x <<= 1) {
        const int64_t t = __shfl_up(t_sum, x), u = __shfl_up(u_sum, x);
        if (lane >= x) t_sum += t, u_sum += u;
    }
    for (int x = 32; x; x >>= 1) p_sum += __shfl_xor(p_sum, x);
    if (lane == 63) wave_tiles[tid >> 6] = t_sum, wave_units[tid >> 6] = u_sum, wave_prefix[tid >> 6] = p_sum;
    __syncthreads();
    int64_t all = 0, t_at = t_sum - tiles, all_units = 0, u_at = u_sum - units, all_prefix = 0;
    for (int w = 0; w < 4; ++w) {
        if (w < (tid >> 6)) t_at += wave_tiles[w], u_at += wave_units[w];
        all += wave_tiles[w], all_units += wave_units[w], all_prefix += wave_prefix[w];
    }
    all = uniform(all);
    all_prefix = uniform(all_prefix);
    const int64_t groups = min((int64_t)gridDim.x, all);
    const int me = all >= gridDim.x ? xcd_remap(blockIdx.x, gridDim.x) : (int)blockIdx.x;
    if (blockIdx.x == 0) {
        if (tid == 0) {
            s.counts[0] = (int)min(all_prefix, (int64_t)s.prefix_units);
            s.counts[1] = (int)min(all_units - all_prefix, (int64_t)s.own_units);
        }
        int64_t u = u_at;
        for (int x = s0; x < min(s1, s.n_groups); ++x) {
            s.unit_base[x] = (int)min(u, (int64_t)s.prefix_units);
            u += (int64_t)group_need<RP>(s, x).blocks * heads;
        }
    }
    if (me >= groups) return;
    int64_t at = all * me / groups;
    const int64_t end = all * (me + 1) / groups;
    if (at >= t_at && at < t_at + tiles) {
        int x = s0;
        for (; x < s1 - 1; ++x) {
            const Need d = segment_need<RP, RO>(s, x);
            const int64_t n = (int64_t)d.blocks * heads * d.tiles;
            if (at < t_at + n) break;
            t_at += n, u_at += (int64_t)d.blocks * heads;
        }
        found = x, found_at = t_at, found_units = u_at;
    }
    __syncthreads();
    int seg = uniform(found);
    int64_t start = uniform(found_at), u0 = uniform(found_units);  // of the segment
    while (at < end) {
        const Need d = segment_need<RP, RO>(s, seg);
        const int64_t n = (int64_t)d.blocks * heads * d.tiles;
        if (at >= start + n) {
            start += n, u0 += (int64_t)d.blocks * heads, ++seg;
            continue;
        }
        const bool is_group = seg < s.n_groups;
        const int u = (int)((at - start) / d.tiles);
        const int first = (int)((at - start) - (int64_t)u * d.tiles);
        const int count = (int)min((int64_t)(d.tiles - first), end - at);
        // The unit's place among its kind, and its record's.
        const int64_t mine = u0 + u - (is_group ? 0 : all_prefix);
        const bool room = mine < (is_group ? s.prefix_units : s.own_units);
        int64_t part = -1;
        if (first > 0) part = (int64_t)2 * me * 16 * RP;
        else if (count < d.tiles) part = (int64_t)(2 * me + 1) * 16 * RP;
        else if (is_group) part = s.whole_prefix + mine * 16 * RP;
        else if (d.floor > 0) part = s.whole_own + mine * 16 * RO;
        if (first == 0 && tid == 0 && room) {
            // The workgroup that has the unit's last tile ends it.
            const int64_t last = ((at + d.tiles) * groups - 1) / all;
            s.joins[(is_group ? 0 : s.prefix_units) + mine] = int4{me, (int)(last - me) + 1, seg, u};
        }
        const int h = u / d.blocks, block = u - h * d.blocks;
        if (!room) {
            // Offsets that give rows to several requests: no record, no result.
        } else if (is_group) {
            run_unit<HD, CODES, RP, true>(a, d, group_of(s, seg).r0, h, block, first, count, part, lds);
        } else {
            run_unit<HD, CODES, RO, false>(a, d, seg - s.n_groups, h, block, first, count, part,
                                           reinterpret_cast<Lds<HD, RO>&>(lds));
        }
        at += count;
    }
}

// One workgroup per unit of a request: per pair, the parts of its own tokens
// and those of its group's prefix, brought to their common maximum and added.
template <int HD, int RP, int RO>
__global__ __launch_bounds__(256) void kv_attention_shared_join_kernel(SharedArgs s) {
    const AttnArgs& a = s.a;
    if ((int)blockIdx.x >= s.counts[1]) return;
    const int4 j = s.joins[s.prefix_units + blockIdx.x];
    const int r = j.z - s.n_groups;
    const Need d = own_need<RO>(s, r);
    if (j.y < 2 && d.floor == 0) return;
    const int h = j.w / d.blocks, block = j.w - h * d.blocks;
    const int pairs = min(16 * RO, d.q.n * a.group - block * 16 * RO);
    const int g = d.floor > 0 ? group_with(s, r) : 0;
    Need p = {};
    if (d.floor > 0) p = group_need<RP>(s, g);
    constexpr int L = HD / 4;  // lanes of a part
    const bool few = j.y <= 16;
    const int span = few ? 64 : 256, mine = threadIdx.x % span;
    const int lanes = mine % L, k0 = mine / L, step = span / L;
    __shared__ f32x4_t so[256];
    __shared__ float sm[256], sl[256];
    const int rows = 256 / span;
    for (int base = blockIdx.y * rows; base < pairs; base += gridDim.y * rows) {
        const int pr = base + threadIdx.x / span;
        const int pair = block * 16 * RO + pr;
        float m = kNoMax, l = 0.0f;
        f32x4_t o = {0.0f, 0.0f, 0.0f, 0.0f};
        auto take = [&](int64_t at) {
            const float2 ml = a.part_ml[at];
            const f32x4_t v = *(const f32x4_t*)(a.part_o + at * HD + 4 * lanes);
            const float top = fmaxf(m, ml.x);
            const float f = __builtin_amdgcn_exp2f(m - top), e = __builtin_amdgcn_exp2f(ml.x - top);
            l = l * f + ml.y * e;
            o = o * f + v * e;
            m = top;
        };
        auto parts = [&](int4 u, int64_t whole, int64_t at) {
            for (int k = k0; k < u.y; k += step)
                take((u.y == 1 ? whole : (int64_t)(k == 0 ? 2 * u.x + 1 : 2 * (u.x + k)) * 16 * RP) + at);
        };
        if (pr < pairs) {
            parts(j, s.whole_own + (int64_t)blockIdx.x * 16 * RO, pr);
            if (d.floor > 0) {
                const int64_t its = (int64_t)(d.q.o0 - p.q.o0) * a.group + pair;
                const int64_t unit = s.unit_base[g] + (int64_t)h * p.blocks + its / (16 * RP);
                if (its >= 0 && unit < s.counts[0])
                    parts(s.joins[unit], s.whole_prefix + unit * 16 * RP, its % (16 * RP));
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
struct SharedLayout {
    int rp, ro;                     // RP and RO
    int64_t prefix_units, own_units;  // at most
    int64_t runs;                   // workgroups
    int64_t some;                   // requests that may have rows
    int64_t whole_prefix, whole_own;  // rows of parts
    size_t base, joins, ml, o, bytes;  // offsets in the workspace
};

SharedLayout shared_layout(const ncm_kv_cache_t& c, const ncm_kv_batch_t& b, int64_t n_groups,
                           int q_heads) {
    SharedLayout s;
    const int64_t group = q_heads / c.kv_heads, pairs = b.rows * group;
    s.some = std::max<int64_t>(1, std::min(b.requests, b.rows));
    s.ro = pairs <= 16 * s.some ? 1 : 2;
    s.rp = pairs <= 16 * std::max<int64_t>(1, std::min(n_groups, s.some)) ? 1 : 2;
    s.own_units = (pairs / (16 * s.ro) + s.some) * c.kv_heads;
    s.prefix_units = n_groups ? (pairs / (16 * s.rp) + n_groups) * c.kv_heads : 0;
    const int64_t tiles = std::max<int64_t>(1, (b.table_width * c.page_size + kTile - 1) / kTile);
    s.runs = std::min<int64_t>((s.own_units + s.prefix_units) * tiles, 2 * kCus);
    s.whole_prefix = 2 * s.runs * 16 * s.rp;
    s.whole_own = s.whole_prefix + s.prefix_units * 16 * s.rp;
    const size_t rows = (size_t)(s.whole_own + s.own_units * 16 * s.ro);
    s.base = 16;
    s.joins = s.base + ((size_t)n_groups * 4 + 15) / 16 * 16;
    s.ml = s.joins + 16 * (size_t)(s.prefix_units + s.own_units);
    s.o = s.ml + (rows * 8 + 15) / 16 * 16;
    s.bytes = s.o + rows * c.head_dim * 4;
    return s;
}

template <int HD, int CODES, int RP, int RO>
hipError_t launch_shared(const SharedArgs& a, const SharedLayout& s, hipStream_t st) {
    kv_attention_shared_kernel<HD, CODES, RP, RO><<<(uint32_t)s.runs, 256, 0, st>>>(a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    // A workgroup per pair where few units are cut into many parts, else per
    // four; of the pairs that a request has on average (the others' wait).
    const int64_t pairs =
        std::min<int64_t>(16 * RO, (a.a.batch.rows * a.a.group + s.some - 1) / s.some);
    const uint32_t y = (uint32_t)(s.own_units * 8 <= s.runs ? pairs : (pairs + 3) / 4);
    kv_attention_shared_join_kernel<HD, RP, RO><<<dim3((uint32_t)s.own_units, y), 256, 0, st>>>(a);
    return hipGetLastError();
}

template <int HD, int CODES>
hipError_t launch_shared_r(const SharedArgs& a, const SharedLayout& s, hipStream_t st) {
    if (s.ro == 2) return launch_shared<HD, CODES, 2, 2>(a, s, st);
    return s.rp == 2 ? launch_shared<HD, CODES, 2, 1>(a, s, st) : launch_shared<HD, CODES, 1, 1>(a, s, st);
}

int check_shared(const ncm_kv_cache_t* cache, const ncm_kv_batch_t* batch, int64_t n_groups,
                 int q_heads, AttnArgs* a) {
    int rc = check_cache(cache, &a->cache);
    if (rc) return rc;
    rc = check_batch(batch, a->cache.page_log2, &a->batch);
    if (rc) return rc;
    if (q_heads < 1 || q_heads > 65535 || q_heads % cache->kv_heads ||
        batch->rows * q_heads > 0x7FFFFFFF || n_groups < 0 || n_groups > batch->requests)
        return NCM_E_SHAPE;
    // The join's launch has a workgroup per unit.
    const SharedLayout s = shared_layout(*cache, *batch, n_groups, q_heads);
    if (s.own_units + s.prefix_units > kMaxBlocks) return NCM_E_SHAPE;
    a->q_heads = q_heads;
    a->group = q_heads / cache->kv_heads;
    return NCM_OK;
}

}  // namespace
}  // namespace ncm

extern "C" int ncm_kv_attention_shared_workspace(const ncm_kv_cache_t* cache,
                                                 const ncm_kv_batch_t* batch, int64_t n_groups,
                                                 int q_heads, size_t* bytes) {
    using namespace ncm;
    if (!bytes) return NCM_E_NULL;
    *bytes = 0;
    AttnArgs a = {};
    const int rc = check_shared(cache, batch, n_groups, q_heads, &a);
    if (rc) return rc;
    if (batch->rows > 0 && batch->requests > 0)
        *bytes = shared_layout(*cache, *batch, n_groups, q_heads).bytes;
    return NCM_OK;
}

extern "C" int ncm_kv_attention_shared_dev(ncm_ctx_t* ctx, const ncm_kv_cache_t* cache,
                                           const ncm_kv_batch_t* batch, const int32_t* groups,
                                           const int32_t* shared, int64_t n_groups,
                                           const uint16_t* q, uint16_t* out, int q_heads,
                                           int64_t q_stride, int64_t out_stride, float scale,
                                           int64_t window, const int32_t* positions,
                                           const uint64_t* tree_mask, int64_t mask_words,
                                           void* workspace, size_t workspace_bytes) {
    using namespace ncm;
    if (!ctx) return NCM_E_NULL;
    SharedArgs s = {};
    AttnArgs& a = s.a;
    int rc = check_shared(cache, batch, n_groups, q_heads, &a);
    if (rc) return rc;
    if (window < 0 || mask_words < 0 || mask_words > kMaxRows / 2) return NCM_E_SHAPE;
    if (batch->rows == 0 || batch->requests == 0) return NCM_OK;
    if (n_groups > 0 && (!groups || !shared)) return NCM_E_NULL;
    const int64_t width = (int64_t)q_heads * cache->head_dim;
    rc = check_rows(q, q_stride, width);
    if (!rc) rc = check_rows(out, out_stride, width);
    if (rc) return rc;
    const SharedLayout l = shared_layout(*cache, *batch, n_groups, q_heads);
    // Offsets may give every request, and groups every group, all rows: the
    // tiles must still be counted in 64 bits, times the workgroups.
    const double most = ((double)batch->rows * q_heads / 16 + cache->kv_heads) *
                        (double)(batch->requests + n_groups) * ((double)a.batch.capacity / kTile + 1);
    if (most > 0x1p50) return NCM_E_SHAPE;
    if (!workspace) return NCM_E_NULL;
    if (workspace_bytes < l.bytes) return NCM_E_LENGTH;
    if ((uintptr_t)workspace % 16) return NCM_E_ARG;
    char* ws = (char*)workspace;
    a.q = q, a.out = out, a.positions = positions, a.tree_mask = (const uint32_t*)tree_mask;
    a.q_stride = q_stride, a.out_stride = out_stride, a.window = window;
    a.mask_words = mask_words, a.scale = scale;
    a.part_ml = (float2*)(ws + l.ml);
    a.part_o = (float*)(ws + l.o);
    s.groups = groups, s.shared = shared, s.n_groups = (int)n_groups;
    s.prefix_units = (int)l.prefix_units, s.own_units = (int)l.own_units;
    s.counts = (int*)ws;
    s.unit_base = (int*)(ws + l.base);
    s.joins = (int4*)(ws + l.joins);
    s.whole_prefix = l.whole_prefix, s.whole_own = l.whole_own;
    const DeviceScope scope(ncm_ctx_device(ctx));
    rc = step_hip(scope.error(), "kv_attention_shared device");
    if (rc) return rc;
    const hipStream_t st = ncm_ctx_stream(ctx);
    const bool wide = cache->head_dim == 128;
    hipError_t e;
    switch (cache->codes) {
        case NCM_KV_BF16:
            e = wide ? launch_shared_r<128, NCM_KV_BF16>(s, l, st) : launch_shared_r<64, NCM_KV_BF16>(s, l, st);
            break;
        case NCM_KV_FP8:
            e = wide ? launch_shared_r<128, NCM_KV_FP8>(s, l, st) : launch_shared_r<64, NCM_KV_FP8>(s, l, st);
            break;
        default:
            e = wide ? launch_shared_r<128, NCM_KV_INT8>(s, l, st) : launch_shared_r<64, NCM_KV_INT8>(s, l, st);
    }
    return step_hip(e, "kv_attention_shared launch");
}
