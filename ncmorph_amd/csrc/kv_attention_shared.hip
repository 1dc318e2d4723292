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
//
// Groups of many pairs are bound by products and softmax instead of the prefix's
// bytes, and have a kernel of their own (kv_attention_prefix_kernel): wavefronts
// of 32 pairs each, which share tiles of K and V as bf16 in LDS. It does the tiles
// that every row of the group sees whole, the units above the prefix's rest.
//
// Measured, 32 heads over 8 of 128, 64 requests behind 8192 tokens, e4m3: 4.8 + 34.6
// + 24 + 8.5 us for plan, prefix, own tokens and join; 256 requests behind 16000,
// bf16: 4.7 + 131 (510 TFLOP/s) + 62 + 13. The prefix kernel spends
// 4 us a tile of 64 tokens and 256 pairs, a third of it in the matrix cores: products
// and softmax of one wavefront hardly overlap those of the other on its SIMD.
#include "kv_attention.h"

namespace ncm {
namespace {

// What is known of a group before its units are cut: its first request and its
// rows (none where there is no prefix), the prefix's tokens, those of them that
// the kernel for many pairs does, and the tile that the narrow units begin with.
struct GroupPlan {
    int r0, r1, o0, n;
    int tokens, done, tile0, pad;
};

struct SharedArgs {
    AttnArgs a;
    const int32_t* groups;  // [n_groups + 1]
    const int32_t* shared;  // [n_groups]
    int n_groups;
    int prefix_units, own_units;  // there is room for
    GroupPlan* plans;
    int* floors;         // of each request: tokens that it reads through its group
    // The kernel for groups of many pairs, its units, their pairs (0: it does not
    // run) and parts.
    int wide_units, wide_pairs;
    int* wide_base;
    int4* wide_joins;
    int64_t wide_cut, whole_wide;
    int* counts;                  // units there are: the groups', the requests', the wide ones
    int* unit_base;               // of a group
    int4* joins;                  // {first workgroup, parts, segment, unit of the segment}
    // Rows of the parts of units in one run. Those of the others begin at row 0: two
    // of 16 RP rows a workgroup, of groups' units and requests' alike.
    int64_t whole_prefix, whole_own;
};

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

constexpr int kWideTile = 64;   // tokens of a tile of the kernel for many pairs
// Groups have that kernel from so many pairs each and (row, head) pairs x tokens x
// head_dim in all on, the tokens those that the table has room for: it is a launch
// more, whose workgroups start for 6 us. With it and without, head_dim 128, 8 K/V
// heads, us: one group behind 8192 tokens and 64 own ones each, 64 pairs 43.6, 42.7,
// 128 49, 56, 256 58, 87; with 512 own ones, 128 60, 50, 256 73, 69; behind 1024, 256
// 43, 30. Eight groups behind 4096, 32 pairs 68, 59, 48 81, 94, 128 144, 175. The
// prefixes' lengths are on the device, the table's width stands for them: in a table
// much wider than the step a short prefix takes this kernel too (one group behind
// 1024, 64 requests, 256 pairs: 29 us in a table of 1100 tokens, 49 in one of 32768).
constexpr int kWidePairs = 48;
constexpr double kWideWork = 5 * 0x1p28;

// The plans, a wavefront per group, and behind them the floors, a thread per
// request: once, instead of by every workgroup of the kernels that cut the units.
__global__ __launch_bounds__(256) void kv_attention_plan_kernel(SharedArgs s, int group_blocks) {
    const BatchView& b = s.a.batch;
    auto tokens_of = [&](int g, int r0, int r1) {
        return r1 - r0 < 2 ? 0 : (int)min((int64_t)max(s.shared[g], 0), b.capacity);
    };
    auto first_of = [&](int g) { return min(max(s.groups[g], 0), b.requests); };
    if ((int)blockIdx.x >= group_blocks) {
        const int r = ((int)blockIdx.x - group_blocks) * 256 + (int)threadIdx.x;
        if (r >= b.requests) return;
        const int before = (int)min((int64_t)max(b.starts[r], 0), b.capacity);
        const int g = group_with(s, r);
        int floor = 0;
        if (g >= 0) {
            const int r0 = first_of(g);
            floor = min(tokens_of(g, r0, min(max(s.groups[g + 1], r0), b.requests)), before);
        }
        s.floors[r] = floor;
        return;
    }
    const int g = (int)(blockIdx.x * 4 + (threadIdx.x >> 6)), lane = threadIdx.x & 63;
    if (g >= s.n_groups) return;
    GroupPlan p = {};
    p.r0 = first_of(g);
    p.r1 = min(max(s.groups[g + 1], p.r0), b.requests);
    p.tokens = tokens_of(g, p.r0, p.r1);
    if (p.tokens > 0) {
        p.o0 = min(max(b.offsets[p.r0], 0), b.rows);
        p.n = max(min(b.offsets[p.r1], b.rows) - p.o0, 0);
        int least = p.tokens;  // before its requests with rows
        for (int r = p.r0 + lane; r < p.r1; r += 64) {
            const Request one = request_of(b, r);
            least = min(least, one.n > 0 ? one.before : p.tokens);
        }
        for (int x = 32; x; x >>= 1) least = min(least, __shfl_xor(least, x));
        if (s.wide_pairs) p.done = least / kWideTile * kWideTile;
        if (s.a.window > 0)
            p.tile0 = (int)(max((int64_t)least - s.a.window + 1, (int64_t)0) / kTile);
    }
    if (lane == 0) s.plans[g] = p;
}

template <int RP>
__device__ __forceinline__ Need group_need(const SharedArgs& s, const GroupPlan& p) {
    Need d;
    d.q.o0 = p.o0;
    d.q.n = p.tokens > p.done ? p.n : 0;
    d.q.before = d.end = d.before = p.tokens;
    d.base = d.floor = p.done;
    d.tile0 = p.tile0;
    d.tiles = max((d.end - d.base + kTile - 1) / kTile - d.tile0, 1);
    d.blocks = (int)(((int64_t)d.q.n * s.a.group + 16 * RP - 1) / (16 * RP));
    return d;
}

template <int RO>
__device__ __forceinline__ Need own_need(const SharedArgs& s, int r) {
    const AttnArgs& a = s.a;
    const int64_t cap = a.batch.capacity;
    Need d;
    d.floor = s.floors[r];
    d.q = request_of(a.batch, r);
    d.end = (int)min((int64_t)d.q.before + d.q.n, cap);
    d.before = (int)min((int64_t)d.q.before, cap);
    const int64_t low = a.window > 0 ? max((int64_t)d.q.before - a.window + 1, (int64_t)0) : 0;
    d.base = (int)max((int64_t)d.floor, min(low, cap)) & ~15;
    d.tile0 = 0;
    d.tiles = max((d.end - d.base + kTile - 1) / kTile, 1);
    d.blocks = (int)(((int64_t)d.q.n * a.group + 16 * RO - 1) / (16 * RO));
    return d;
}

template <int RP, int RO>
__device__ __forceinline__ Need segment_need(const SharedArgs& s, int seg) {
    return seg < s.n_groups ? group_need<RP>(s, s.plans[seg]) : own_need<RO>(s, seg - s.n_groups);
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
            u += (int64_t)group_need<RP>(s, s.plans[x]).blocks * heads;
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
    Need d = segment_need<RP, RO>(s, seg);
    while (at < end) {
        const int64_t n = (int64_t)d.blocks * heads * d.tiles;
        if (at >= start + n) {
            start += n, u0 += (int64_t)d.blocks * heads, ++seg;
            d = segment_need<RP, RO>(s, seg);
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
            const GroupPlan& of = s.plans[seg];
            run_unit<HD, CODES, RP, true>(a, d, of.r0, h, block, first, count, part, lds, of.r1);
        } else {
            run_unit<HD, CODES, RO, false>(a, d, seg - s.n_groups, h, block, first, count, part,
                                           reinterpret_cast<Lds<HD, RO>&>(lds));
        }
        at += count;
    }
}

// ------------------------------------------------------- groups of many pairs

// A tile of K and V as bf16, rows of HD values; 16-byte chunk c of row r of K is
// at chunk c ^ (r % 16) (HD 64: c ^ (r / 2 % 8)), so that the sixteen rows of an
// operand's reads fall into different banks.
template <int HD>
struct WideTile {
    u32x4_t k[kWideTile][HD / 8];
    u32x4_t v[kWideTile][HD / 8];
    float ks[kWideTile], vs[kWideTile];
    static __device__ __forceinline__ int place(int row, int chunk) {
        return HD == 128 ? chunk ^ (row & 15) : chunk ^ ((row >> 1) & 7);
    }
};
template <int HD>
struct WideLds {
    WideTile<HD> tile[2];
    uint64_t gone[4];        // of four tiles in turn: tokens that are not there
    float m[4][2][64], l[4][2][64];
};

// What a thread brings of a tile: eight threads a token, codes of 16 bytes.
template <int HD, int CODES>
struct WideLoad {
    static constexpr int ES = CODES == NCM_KV_BF16 ? 2 : 1, N = HD * ES / 128;  // of 16 bytes
    static constexpr bool HALF = HD * ES < 128;  // 64 codes: every second thread
    u32x4_t k[N ? N : 1], v[N ? N : 1];
    float ks, vs;
    bool ok;

    __device__ __forceinline__ void load(const KvView& cache, int h, int token, int page) {
        const int lane = threadIdx.x & 7;
        ok = page >= 0;
        const int64_t at = ((int64_t)h << cache.page_log2) + (token & ((1 << cache.page_log2) - 1));
        const int64_t p = max(page, 0);
        if (!HALF || lane < 4) {
#pragma unroll
            for (int i = 0; i < (N ? N : 1); ++i) {
                k[i] = *(const u32x4_t*)(cache.k + (p * cache.k_stride + at * HD) * ES + 16 * (lane + 8 * i));
                v[i] = *(const u32x4_t*)(cache.v + (p * cache.v_stride + at * HD) * ES + 16 * (lane + 8 * i));
            }
        }
        if constexpr (CODES != NCM_KV_BF16)
            if (lane == 0) ks = cache.ks[p * cache.ks_stride + at], vs = cache.vs[p * cache.vs_stride + at];
    }

    // Into the tile, zeros for a token that is not there.
    __device__ __forceinline__ void store(WideTile<HD>& tile, uint64_t* gone) {
        const int row = threadIdx.x >> 3, lane = threadIdx.x & 7;
        const u32x4_t zero = {0, 0, 0, 0};
        if (!HALF || lane < 4) {
#pragma unroll
            for (int i = 0; i < (N ? N : 1); ++i) {
                const u32x4_t x = ok ? k[i] : zero, y = ok ? v[i] : zero;
                if constexpr (CODES == NCM_KV_BF16) {
                    const int chunk = lane + 8 * i;
                    tile.k[row][WideTile<HD>::place(row, chunk)] = x;
                    tile.v[row][chunk] = y;
                } else {
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        u32x4_t a, b;
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            uint32_t lo, hi;
                            widen4<CODES>(x[2 * half + j], lo, hi);
                            a[2 * j] = lo, a[2 * j + 1] = hi;
                            widen4<CODES>(y[2 * half + j], lo, hi);
                            b[2 * j] = lo, b[2 * j + 1] = hi;
                        }
                        const int chunk = 2 * (lane + 8 * i) + half;
                        tile.k[row][WideTile<HD>::place(row, chunk)] = a;
                        tile.v[row][chunk] = b;
                    }
                }
            }
        }
        if (lane == 0) {
            if constexpr (CODES != NCM_KV_BF16) tile.ks[row] = ok ? ks : 0.0f, tile.vs[row] = ok ? vs : 0.0f;
            if (!ok) atomicOr((unsigned long long*)gone, 1ull << row);
        }
    }
};

// Adds 32 tokens of a tile, from row `base` on, to a wavefront's 32 pairs, which
// all see them; gone: those that are not there. The arithmetic is add_tokens'.
template <int HD, int CODES>
__device__ __forceinline__ void add_wide(State<HD, 2, false>& st,
                                         const bf16x8_t (&q)[2][HD / 32], const WideTile<HD>& tile,
                                         int base, uint32_t gone,
                                         float to_log2, float lag) {
    const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
    float s[2][8];
    {
        f32x4_t sc[2][2];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int row = base + 16 * half + c;
#pragma unroll
            for (int rr = 0; rr < 2; ++rr) sc[rr][half] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int k = 0; k < HD / 32; ++k) {
                const bf16x8_t op = __builtin_bit_cast(bf16x8_t, tile.k[row][WideTile<HD>::place(row, 4 * k + g)]);
#pragma unroll
                for (int rr = 0; rr < 2; ++rr)
                    sc[rr][half] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(op, q[rr][k], sc[rr][half], 0, 0, 0);
            }
        }
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            f32x4_t ks = {1.0f, 1.0f, 1.0f, 1.0f};
            if constexpr (CODES != NCM_KV_BF16) ks = *(const f32x4_t*)&tile.ks[base + 16 * half + 4 * g];
#pragma unroll
            for (int rr = 0; rr < 2; ++rr)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    s[rr][4 * half + i] = sc[rr][half][i];
                    if constexpr (CODES != NCM_KV_BF16) s[rr][4 * half + i] *= ks[i] * to_log2;
                }
        }
    }
    if (gone)
#pragma unroll
        for (int rr = 0; rr < 2; ++rr)
#pragma unroll
            for (int i = 0; i < 8; ++i)
                s[rr][i] = (gone >> (16 * (i / 4) + 4 * g + i % 4)) & 1u ? -INFINITY : s[rr][i];
    f32x4_t vs[2] = {{1.0f, 1.0f, 1.0f, 1.0f}, {1.0f, 1.0f, 1.0f, 1.0f}};
    if constexpr (CODES != NCM_KV_BF16)
#pragma unroll
        for (int half = 0; half < 2; ++half) vs[half] = *(const f32x4_t*)&tile.vs[base + 16 * half + 4 * g];
    bf16x8_t p[2], rest[2];
#pragma unroll
    for (int rr = 0; rr < 2; ++rr) {
        float top = s[rr][0];
#pragma unroll
        for (int i = 1; i < 8; ++i) top = fmaxf(top, s[rr][i]);
        top = max_over_groups(top);
        if (__any(top > st.m[rr] + (CODES == NCM_KV_BF16 ? lag : 8.0f))) {
            top = fmaxf(top, st.m[rr]);
            const float d = st.m[rr] - top;
            const float f = __builtin_amdgcn_exp2f(CODES == NCM_KV_BF16 ? d * to_log2 : d);
            st.m[rr] = top;
            st.l[rr] *= f;
#pragma unroll
            for (int n = 0; n < HD / 16; ++n) st.o[rr][n] *= f;
        }
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float d = s[rr][i] - st.m[rr];
            s[rr][i] = __builtin_amdgcn_exp2f(CODES == NCM_KV_BF16 ? d * to_log2 : d);
            sum += s[rr][i];
            if constexpr (CODES != NCM_KV_BF16) s[rr][i] = s[rr][i] * vs[i / 4][i % 4];
        }
        st.l[rr] += sum;
        u32x4_t hi, lo;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t x = __float_as_uint(s[rr][2 * i]), y = __float_as_uint(s[rr][2 * i + 1]);
            hi[i] = __builtin_amdgcn_perm(y, x, 0x07060302u);
            lo[i] = bf16x2_rne(fmaf(s[rr][2 * i], 1.00000095367431640625f,
                                    -__uint_as_float(x & 0xFFFF0000u)),
                               fmaf(s[rr][2 * i + 1], 1.00000095367431640625f,
                                    -__uint_as_float(y & 0xFFFF0000u)));
        }
        p[rr] = __builtin_bit_cast(bf16x8_t, hi);
        rest[rr] = __builtin_bit_cast(bf16x8_t, lo);
    }
    // Not read ahead of the softmax: there are no registers for them beside its own.
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    typedef uint32_t vec __attribute__((ext_vector_type(HD / 32)));
    vec raw[8];
#pragma unroll
    for (int i = 0; i < 8; ++i)
        raw[i] = ((const vec*)tile.v[base + 16 * (i / 4) + 4 * g + i % 4])[c];
#pragma unroll
    for (int f = 0; f < HD / 64; ++f) {
#pragma unroll
        for (int n = 0; n < 4; ++n) {
            u32x4_t w;
#pragma unroll
            for (int j = 0; j < 4; ++j)
                w[j] = __builtin_amdgcn_perm(raw[2 * j + 1][2 * f + n / 2], raw[2 * j][2 * f + n / 2],
                                             n % 2 ? 0x07060302u : 0x05040100u);
            const bf16x8_t v = __builtin_bit_cast(bf16x8_t, w);
#pragma unroll
            for (int rr = 0; rr < 2; ++rr)
                st.o[rr][4 * f + n] =
                    __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, p[rr], st.o[rr][4 * f + n], 0, 0, 0);
#pragma unroll
            for (int rr = 0; rr < 2; ++rr)
                st.o[rr][4 * f + n] =
                    __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, rest[rr], st.o[rr][4 * f + n], 0, 0, 0);
        }
    }
}

// What the kernel does of a group.
struct Wide {
    int r0, o0, rows, tiles, blocks;
};
__device__ __forceinline__ Wide wide_of(const SharedArgs& s, int g) {
    const GroupPlan& p = s.plans[g];
    const int rows = p.done > 0 ? p.n : 0;
    return {p.r0, p.o0, rows, max(p.done / kWideTile, 1),
            (int)(((int64_t)rows * s.a.group + s.wide_pairs - 1) / s.wide_pairs)};
}

// Tiles [first, first + count) of a group's unit, into the part that begins at row
// `part`: NP wavefronts of 32 pairs each, and 8 / NP of such sets, which take
// halves of the tiles and every other tile.
template <int HD, int CODES, int NP>
__device__ __forceinline__ void run_wide(const SharedArgs& s, const Wide& d, int h, int block,
                                         int first, int count, int64_t part, WideLds<HD>& lds) {
    constexpr int NS = 8 / NP, NR = NS < 2 ? 1 : 2;  // wavefronts of a tile's rounds
    const AttnArgs& a = s.a;
    const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
    const int c = lane & 15, g = lane >> 4, np = wave % NP, ns = wave / NP;
    const int pairs = d.rows * a.group - block * 32 * NP;
    const int key0 = first * kWideTile, mine = key0 + (tid >> 3);
    auto page = [&](int t) {  // of the thread's token of tile t
        return t < count ? page_of(a.batch, a.cache, d.r0, mine + t * kWideTile) : -1;
    };
    WideLoad<HD, CODES> next;
    const int page0 = page(0);
    int page2 = page(1);
    if (tid < 4) lds.gone[tid] = 0;
    State<HD, 2, false> st;
    bf16x8_t q[2][HD / 32];
    const uint32_t sign = a.scale < 0.0f ? 0x80008000u : 0u;
    const float to_log2 = a.scale == 0.0f ? 1.4e-45f : fabsf(a.scale) * 1.4426950408889634f;
    const float lag = fminf(8.0f / to_log2, 1e30f);
#pragma unroll
    for (int rr = 0; rr < 2; ++rr) {
        const int pair = block * 32 * NP + min(32 * np + 16 * rr + c, pairs - 1);
        const int row = pair / a.group, head = h * a.group + pair - row * a.group;
        const uint16_t* from = a.q + (d.o0 + row) * a.q_stride + (int64_t)head * HD + 8 * g;
#pragma unroll
        for (int k = 0; k < HD / 32; ++k)
            q[rr][k] = __builtin_bit_cast(bf16x8_t, *(const u32x4_t*)(from + 32 * k) ^ sign);
#pragma unroll
        for (int n = 0; n < HD / 16; ++n) st.o[rr][n] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
        st.m[rr] = kNoMax;
        st.l[rr] = 0.0f;
    }
    next.load(a.cache, h, mine, page0);
    __syncthreads();
    next.store(lds.tile[0], &lds.gone[0]);
    if (count > 1) next.load(a.cache, h, mine + kWideTile, page2);
    page2 = page(2);
    lds_barrier();
    // Tile t is in one buffer, t + 1 in registers on its way to the other, and the
    // page of t + 2 known.
    for (int t = 0; t < count; ++t) {
        const WideTile<HD>& tile = lds.tile[t & 1];
        const uint64_t gone = uniform((int64_t)lds.gone[t & 3]);
#pragma unroll 1
        for (int round = 0; round < kWideTile / 32 / NR; ++round) {
            const int base = 32 * (round * NR + ns % NR);
            if (NS <= 2 || (t & 1) == ns / 2)
                add_wide<HD, CODES>(st, q, tile, base, (uint32_t)(gone >> base), to_log2, lag);
        }
        if (tid == 0) lds.gone[(t + 2) & 3] = 0;
        if (t + 1 < count) {
            next.store(lds.tile[(t + 1) & 1], &lds.gone[(t + 1) & 3]);
            if (t + 2 < count) next.load(a.cache, h, mine + (t + 2) * kWideTile, page2);
            page2 = page(t + 3);
        }
        lds_barrier();  // the loads stay in flight
    }
    // The states of one NP wavefronts' pairs into those of the first NP: by halves,
    // through the tiles' LDS, in chunks of a row of lanes.
    float m[2], l[2];
#pragma unroll
    for (int rr = 0; rr < 2; ++rr) {
        l[rr] = sum_over_groups(st.l[rr]);
        m[rr] = st.m[rr];
        if (CODES == NCM_KV_BF16 && m[rr] > kNoMax) m[rr] = fmaxf(m[rr] * to_log2, kNoMax);
    }
    f32x4_t* mem = (f32x4_t*)lds.tile;
    static_assert(sizeof(lds.tile) >= 4 * 2 * (HD / 16) * 64 * 16, "four states");
#pragma unroll
    for (int half = NS / 2; half >= 1; half /= 2) {
        if (ns >= half && ns < 2 * half) {
            const int at = (wave - half * NP) * 2;
#pragma unroll
            for (int rr = 0; rr < 2; ++rr) {
#pragma unroll
                for (int n = 0; n < HD / 16; ++n) mem[((at + rr) * (HD / 16) + n) * 64 + lane] = st.o[rr][n];
                lds.m[wave - half * NP][rr][lane] = m[rr], lds.l[wave - half * NP][rr][lane] = l[rr];
            }
        }
        __syncthreads();
        if (ns < half) {
#pragma unroll
            for (int rr = 0; rr < 2; ++rr) {
                const float m2 = lds.m[wave][rr][lane], l2 = lds.l[wave][rr][lane];
                const float top = fmaxf(m[rr], m2);
                const float f = __builtin_amdgcn_exp2f(m[rr] - top), e = __builtin_amdgcn_exp2f(m2 - top);
                l[rr] = l[rr] * f + l2 * e;
                m[rr] = top;
#pragma unroll
                for (int n = 0; n < HD / 16; ++n)
                    st.o[rr][n] = st.o[rr][n] * f + mem[((wave * 2 + rr) * (HD / 16) + n) * 64 + lane] * e;
            }
        }
        __syncthreads();
    }
    if (ns == 0) {
#pragma unroll
        for (int rr = 0; rr < 2; ++rr) {
            const int pr = 32 * np + 16 * rr + c;
            if (pr >= pairs) continue;
            const int64_t at = part + pr;
            if (g == 0) a.part_ml[at] = float2{m[rr], l[rr]};
#pragma unroll
            for (int x = 0; x < 4; ++x)
#pragma unroll
                for (int n = 0; n < HD / 16; n += 4) {
                    f32x4_t v;
#pragma unroll
                    for (int i = 0; i < 4; ++i) v[i] = st.o[rr][n + i][x];
                    *(f32x4_t*)(a.part_o + at * HD + (HD / 16) * (4 * g + x) + n) = v;
                }
        }
    }
    __syncthreads();
}

template <int HD, int CODES, int NP>
__global__ __launch_bounds__(512, 2) void kv_attention_prefix_kernel(SharedArgs s) {
    __shared__ WideLds<HD> lds;
    __shared__ int64_t wave_tiles[8], wave_units[8], found_at, found_units;
    __shared__ int found;
    const AttnArgs& a = s.a;
    const int tid = threadIdx.x, lane = tid & 63, heads = a.cache.kv_heads;
    // Tiles and units ahead of each thread's share of the groups.
    const int per = (s.n_groups + 511) / 512, g0 = min(tid * per, s.n_groups);
    const int g1 = min(g0 + per, s.n_groups);
    int64_t tiles = 0, units = 0;
    for (int x = g0; x < g1; ++x) {
        const Wide d = wide_of(s, x);
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
    for (int w = 0; w < 8; ++w) {
        if (w < (tid >> 6)) t_at += wave_tiles[w], u_at += wave_units[w];
        all += wave_tiles[w], all_units += wave_units[w];
    }
    all = uniform(all);
    const int64_t groups = min((int64_t)gridDim.x, all);
    const int me = all >= gridDim.x ? xcd_remap(blockIdx.x, gridDim.x) : (int)blockIdx.x;
    if (blockIdx.x == 0) {
        if (tid == 0) s.counts[2] = (int)min(all_units, (int64_t)s.wide_units);
        int64_t u = u_at;
        for (int x = g0; x < g1; ++x) {
            s.wide_base[x] = (int)min(u, (int64_t)s.wide_units);
            u += (int64_t)wide_of(s, x).blocks * heads;
        }
    }
    if (me >= groups) return;
    int64_t at = all * me / groups;
    const int64_t end = all * (me + 1) / groups;
    if (at >= t_at && at < t_at + tiles) {
        int x = g0;
        for (; x < g1 - 1; ++x) {
            const Wide d = wide_of(s, x);
            const int64_t n = (int64_t)d.blocks * heads * d.tiles;
            if (at < t_at + n) break;
            t_at += n, u_at += (int64_t)d.blocks * heads;
        }
        found = x, found_at = t_at, found_units = u_at;
    }
    __syncthreads();
    int seg = uniform(found);
    int64_t start = uniform(found_at), u0 = uniform(found_units);  // of the group
    Wide d = wide_of(s, seg);
    while (at < end) {
        const int64_t n = (int64_t)d.blocks * heads * d.tiles;
        if (at >= start + n) {
            start += n, u0 += (int64_t)d.blocks * heads, ++seg;
            d = wide_of(s, seg);
            continue;
        }
        const int u = (int)((at - start) / d.tiles);
        const int first = (int)((at - start) - (int64_t)u * d.tiles);
        const int count = (int)min((int64_t)(d.tiles - first), end - at);
        const bool room = u0 + u < s.wide_units;
        int64_t part = s.whole_wide + (u0 + u) * s.wide_pairs;
        if (first > 0) part = s.wide_cut + 2 * (int64_t)me * s.wide_pairs;
        else if (count < d.tiles) part = s.wide_cut + (2 * (int64_t)me + 1) * s.wide_pairs;
        if (first == 0 && tid == 0 && room) {
            // The workgroup that has the unit's last tile ends it.
            const int64_t last = ((at + d.tiles) * groups - 1) / all;
            s.wide_joins[u0 + u] = int4{me, (int)(last - me) + 1, seg, u};
        }
        const int h = u / d.blocks;
        if (room)
            run_wide<HD, CODES, NP>(s, d, h, u - h * d.blocks, first, count, part, lds);
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
    Wide w = {};
    if (d.floor > 0) {
        p = group_need<RP>(s, s.plans[g]);
        if (s.wide_pairs) w = wide_of(s, g);
    }
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
        if (pr < pairs) {
            const int64_t whole = s.whole_own + (int64_t)blockIdx.x * 16 * RO;
            for (int k = k0; k < j.y; k += step)
                take((j.y == 1 ? whole : (int64_t)(k == 0 ? 2 * j.x + 1 : 2 * (j.x + k)) * 16 * RP) + pr);
            auto group_parts = [&](int64_t its, int64_t unit, int units, int unit_pairs, const int4* joins,
                                   int64_t cut, int64_t whole) {
                if (its < 0 || unit >= units) return;
                const int4 u = joins[unit];
                for (int k = k0; k < u.y; k += step) {
                    const int64_t slot = k == 0 ? 2 * (int64_t)u.x + 1 : 2 * ((int64_t)u.x + k);
                    take((u.y == 1 ? whole + unit * unit_pairs : cut + slot * unit_pairs) + its % unit_pairs);
                }
            };
            if (p.blocks > 0) {
                const int64_t its = (int64_t)(d.q.o0 - p.q.o0) * a.group + pair;
                group_parts(its, s.unit_base[g] + (int64_t)h * p.blocks + its / (16 * RP), s.counts[0],
                            16 * RP, s.joins, 0, s.whole_prefix);
            }
            if (w.blocks > 0) {
                const int64_t its = (int64_t)(d.q.o0 - w.o0) * a.group + pair;
                group_parts(its, s.wide_base[g] + (int64_t)h * w.blocks + its / s.wide_pairs, s.counts[2],
                            s.wide_pairs, s.wide_joins, s.wide_cut, s.whole_wide);
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
    int rp, ro;                       // RP and RO
    int wide;                         // NP of the groups' own kernel, or 0
    int64_t prefix_units, own_units, wide_units;  // at most
    int64_t runs, wide_runs;          // workgroups
    int64_t some;                     // requests that may have rows
    int64_t whole_prefix, whole_own, wide_cut, whole_wide;  // rows of parts
    size_t plans, floors, base, wide_base, joins, ml, o, bytes;     // offsets in the workspace
};

SharedLayout shared_layout(const ncm_kv_cache_t& c, const ncm_kv_batch_t& b, int64_t n_groups,
                           int q_heads, bool window) {
    SharedLayout s;
    const int64_t group = q_heads / c.kv_heads, pairs = b.rows * group;
    s.some = std::max<int64_t>(1, std::min(b.requests, b.rows));
    s.ro = pairs <= 16 * s.some ? 1 : 2;
    const int64_t per_group = pairs / std::max<int64_t>(1, std::min(n_groups, s.some));
    s.rp = std::max(s.ro, per_group <= 16 ? 1 : 2);
    const int64_t tokens = std::max<int64_t>(1, b.table_width * c.page_size);
    const bool many = (double)pairs * c.kv_heads * tokens * c.head_dim >= kWideWork && per_group >= kWidePairs;
    // Two wavefronts of pairs where a group fills no more (eight groups of 48 pairs
    // behind 4096 tokens: 81 us, 88 with four; of 128: 159, 144).
    s.wide = n_groups == 0 || window || !many ? 0 : per_group <= 64 ? 2 : 4;
    // Eight wavefronts of pairs, each tile of the prefix brought once for 256, where
    // that leaves a workgroup tiles enough to be worth the state that it writes and
    // the join reads (1024 pairs behind 16000 tokens, 31 tiles each: 136 us, 158
    // with four; 256 behind 8192, 4 tiles each: 35 and a join of 11.8 us, 36 and 8.6).
    if (s.wide == 4 && per_group > 128 &&
        (pairs / 256 + n_groups) * c.kv_heads * (tokens / kWideTile) >= 12 * kCus)
        s.wide = 8;
    s.own_units = (pairs / (16 * s.ro) + s.some) * c.kv_heads;
    s.prefix_units = n_groups ? (pairs / (16 * s.rp) + n_groups) * c.kv_heads : 0;
    s.wide_units = s.wide ? (pairs / (32 * s.wide) + n_groups) * c.kv_heads : 0;
    const int64_t tiles = (tokens + kTile - 1) / kTile;
    s.runs = std::min<int64_t>((s.own_units + s.prefix_units) * tiles, 2 * kCus);
    s.wide_runs = std::min<int64_t>(s.wide_units * ((tokens + kWideTile - 1) / kWideTile), kCus);
    s.whole_prefix = 2 * s.runs * 16 * s.rp;
    s.whole_own = s.whole_prefix + s.prefix_units * 16 * s.rp;
    s.wide_cut = s.whole_own + s.own_units * 16 * s.ro;
    s.whole_wide = s.wide_cut + 2 * s.wide_runs * 32 * s.wide;
    const size_t rows = (size_t)(s.whole_wide + s.wide_units * 32 * s.wide);
    auto up = [](size_t bytes) { return (bytes + 15) / 16 * 16; };
    s.plans = 16;
    s.floors = s.plans + sizeof(GroupPlan) * (size_t)n_groups;
    s.base = s.floors + up(4 * (size_t)b.requests);
    s.wide_base = s.base + up(4 * (size_t)n_groups);
    s.joins = s.wide_base + up(4 * (size_t)n_groups);
    s.ml = s.joins + 16 * (size_t)(s.prefix_units + s.own_units + s.wide_units);
    s.o = s.ml + up(rows * 8);
    s.bytes = s.o + rows * c.head_dim * 4;
    return s;
}

template <int HD, int CODES, int RP, int RO>
hipError_t launch_shared(const SharedArgs& a, const SharedLayout& s, hipStream_t st) {
    const int group_blocks = (a.n_groups + 3) / 4;
    kv_attention_plan_kernel<<<(uint32_t)(group_blocks + (a.a.batch.requests + 255) / 256), 256, 0, st>>>(
        a, group_blocks);
    if (s.wide == 2) kv_attention_prefix_kernel<HD, CODES, 2><<<(uint32_t)s.wide_runs, 512, 0, st>>>(a);
    if (s.wide == 4) kv_attention_prefix_kernel<HD, CODES, 4><<<(uint32_t)s.wide_runs, 512, 0, st>>>(a);
    if (s.wide == 8) kv_attention_prefix_kernel<HD, CODES, 8><<<(uint32_t)s.wide_runs, 512, 0, st>>>(a);
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
    for (bool window : {false, true}) {
        const SharedLayout s = shared_layout(*cache, *batch, n_groups, q_heads, window);
        if (s.own_units + s.prefix_units + s.wide_units > kMaxBlocks) return NCM_E_SHAPE;
    }
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
    if (batch->rows > 0 && batch->requests > 0)  // with a window or without
        *bytes = std::max(shared_layout(*cache, *batch, n_groups, q_heads, false).bytes,
                          shared_layout(*cache, *batch, n_groups, q_heads, true).bytes);
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
    const SharedLayout l = shared_layout(*cache, *batch, n_groups, q_heads, window > 0);
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
    s.plans = (GroupPlan*)(ws + l.plans);
    s.floors = (int*)(ws + l.floors);
    s.unit_base = (int*)(ws + l.base);
    s.wide_base = (int*)(ws + l.wide_base);
    s.joins = (int4*)(ws + l.joins);
    s.wide_joins = s.joins + l.prefix_units + l.own_units;
    s.whole_prefix = l.whole_prefix, s.whole_own = l.whole_own;
    s.wide_cut = l.wide_cut, s.whole_wide = l.whole_wide;
    s.wide_units = (int)l.wide_units, s.wide_pairs = 32 * l.wide;
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
