// Attention of a step's rows over the paged cache (ncm_kv_attention_dev).
//
// One pass with a running maximum and sum of the softmax:
//   s_j = scale q.k_j (times the scale of k_j), m' >= max(m, max s_j) - 8,
//   l' = l 2^(m - m') + sum 2^(s_j - m'), o' = o 2^(m - m') + sum 2^(s_j - m') v_j
// with log2(e) folded into the scale (which for bf16 caches multiplies the
// differences s_j - m in place of the products). The query heads of a K/V head
// and the rows of a request stand together: R times 16 (row, head) pairs are
// the columns of v_mfma_f32_16x16x32_bf16 products, tokens the rows of S^T =
// K Q^T and the summed index of O^T = V^T P^T.
//
// Bound by the cache's bytes for one token a request, so K and V go from
// memory to registers, each read once, without LDS between: the lane layout of
// S^T (a column's four tokens 4 g .. 4 g + 3 in lane group g) is that of the
// second product's P^T operand if its summed index runs over the tokens in the
// order the lanes hold them, and a lane then needs of V those same tokens'
// values of its own dims, which are its own rows' loads, their 16-bit halves
// regrouped with v_perm_b32. 8-bit codes are widened to bf16 in registers
// (exact); their scales multiply scores and probabilities, not values. The
// queries, which all four wavefronts read, are in LDS.
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
#include "step.h"

namespace ncm {
namespace {

constexpr int kTile = 128;     // tokens of a tile, 32 per wavefront
constexpr int kCus = 256;
// No score is below this start but -inf, and 2^(-inf - m) stays 0 as it is finite.
constexpr float kNoMax = -3.40282347e38f;

struct AttnArgs {
    KvView cache;
    BatchView batch;
    const uint16_t* q;
    uint16_t* out;
    const int32_t* positions;
    const uint32_t* tree_mask;  // pairs of words
    int64_t q_stride, out_stride, window, mask_words;
    float scale;
    int q_heads, group;
    // Workspace: the number of units, a join record per unit, and two parts
    // per workgroup (the end of a unit that an earlier one began, and the
    // beginning of one that a later one ends): m and l, then o, per pair.
    int units;          // records there is room for
    int* unit_count;
    int4* joins;        // {first workgroup, parts, request, unit of the request}
    float2* part_ml;
    float* part_o;
};

// What a request asks for, in units and tiles.
struct Need {
    Request q;
    int end;           // tokens that its rows can see lie in [.., end)
    int before;        // tokens before its rows, at most the table's
    int tile0, tiles;  // of a unit
    int blocks;        // of 16 R pairs
};
template <int R>
__device__ __forceinline__ Need need_of(const AttnArgs& a, int r) {
    Need d;
    d.q = request_of(a.batch, r);
    const int64_t cap = a.batch.capacity;
    d.end = (int)min((int64_t)d.q.before + d.q.n, cap);
    d.before = (int)min((int64_t)d.q.before, cap);
    const int64_t low = a.window > 0 ? max((int64_t)d.q.before - a.window + 1, (int64_t)0) : 0;
    d.tile0 = (int)(min(low, cap) / kTile);
    d.tiles = max((d.end + kTile - 1) / kTile - d.tile0, 1);
    d.blocks = (int)(((int64_t)d.q.n * a.group + 16 * R - 1) / (16 * R));
    return d;
}

__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ int64_t uniform(int64_t v) {
    const uint32_t lo = (uint32_t)uniform((int)v), hi = (uint32_t)uniform((int)(v >> 32));
    return (int64_t)(((uint64_t)hi << 32) | lo);
}

// Four codes of a dword as two dwords of bf16 pairs.
template <int CODES>
__device__ __forceinline__ void widen4(uint32_t w, uint32_t& lo, uint32_t& hi) {
    if constexpr (CODES == NCM_KV_FP8) {
        lo = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)w, 1.0f, false));
        hi = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)w, 1.0f, true));
    } else {
        // Integers to 127 are exact in bf16: the high halves of their floats.
        uint32_t f[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = __float_as_uint((float)(int8_t)(w >> (8 * i)));
        lo = __builtin_amdgcn_perm(f[1], f[0], 0x07060302u);
        hi = __builtin_amdgcn_perm(f[3], f[2], 0x07060302u);
    }
}

// 32 tokens of K and V in a wavefront's registers. Lane l: c = l % 16, g = l /
// 16. k[half]: token 16 half + c, 16 bytes at 64 j + 16 g of its row; v[4 half
// + i]: token 16 half + 4 g + i, its values at dims HD / 16 * c onwards.
template <int HD, int CODES>
struct Tile {
    static constexpr int ES = CODES == NCM_KV_BF16 ? 2 : 1;
    static constexpr int KL = HD * ES / 64, VW = HD * ES / 64;
    typedef uint32_t vec __attribute__((ext_vector_type(VW)));
    u32x4_t k[2][KL];
    vec v[8];
    f32x4_t ks[2], vs[2];

    // page: those of tokens key .. key + 15 and key + 16 .. key + 31, at
    // least 0; tokens of a page past what the request has are loaded too.
    __device__ __forceinline__ void load_k(const KvView& cache, int h, int key, int page0,
                                           int page1, int lane) {
        const int c = lane & 15, g = lane >> 4, mask = (1 << cache.page_log2) - 1;
        const uint32_t off = (uint32_t)(c * HD * ES + g * 16);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int64_t page = half ? page1 : page0;
            const int64_t at = ((int64_t)h << cache.page_log2) + ((key + 16 * half) & mask);
            const char* base = cache.k + (page * cache.k_stride + at * HD) * ES;
#pragma unroll
            for (int j = 0; j < KL; ++j) k[half][j] = *(const u32x4_t*)(base + off + 64 * j);
            if constexpr (CODES != NCM_KV_BF16)
                ks[half] = *(const f32x4_t*)(cache.ks + page * cache.ks_stride + at + 4 * g);
        }
    }
    __device__ __forceinline__ void load_v(const KvView& cache, int h, int key, int page0,
                                           int page1, int lane) {
        const int c = lane & 15, g = lane >> 4, mask = (1 << cache.page_log2) - 1;
        const uint32_t off = (uint32_t)(4 * g * HD * ES + c * (HD / 16) * ES);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int64_t page = half ? page1 : page0;
            const int64_t at = ((int64_t)h << cache.page_log2) + ((key + 16 * half) & mask);
            const char* base = cache.v + (page * cache.v_stride + at * HD) * ES;
#pragma unroll
            for (int i = 0; i < 4; ++i) v[4 * half + i] = *(const vec*)(base + off + i * HD * ES);
            if constexpr (CODES != NCM_KV_BF16)
                vs[half] = *(const f32x4_t*)(cache.vs + page * cache.vs_stride + at + 4 * g);
        }
    }
    // The bf16 operand of k-step s (32 dims) of 16 tokens.
    __device__ __forceinline__ bf16x8_t k_operand(int half, int s) const {
        if constexpr (CODES == NCM_KV_BF16) {
            return __builtin_bit_cast(bf16x8_t, k[half][s]);
        } else {
            u32x4_t w;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                uint32_t lo, hi;
                widen4<CODES>(k[half][s / 2][2 * (s % 2) + j], lo, hi);
                w[2 * j] = lo, w[2 * j + 1] = hi;
            }
            return __builtin_bit_cast(bf16x8_t, w);
        }
    }
    // The dims of a head that k-step s takes from lane group g.
    static __device__ __forceinline__ int k_dims(int s, int g) {
        return CODES == NCM_KV_BF16 ? 32 * s + 8 * g : 64 * (s / 2) + 16 * g + 8 * (s % 2);
    }
    // The operands of V^T for dims 4 f + n of the lane's HD / 16: w[n][j] holds
    // the bf16 of tokens 2 j and 2 j + 1 of the lane's eight.
    __device__ __forceinline__ void v_operands(int f, uint32_t (&w)[4][4]) const {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if constexpr (CODES == NCM_KV_BF16) {
#pragma unroll
                for (int n = 0; n < 4; ++n)
                    w[n][j] = __builtin_amdgcn_perm(v[2 * j + 1][2 * f + n / 2], v[2 * j][2 * f + n / 2],
                                                    n % 2 ? 0x07060302u : 0x05040100u);
            } else if constexpr (CODES == NCM_KV_FP8) {
                // The two tokens' bytes side by side, then widened in pairs.
                const uint32_t lo = __builtin_amdgcn_perm(v[2 * j + 1][f], v[2 * j][f], 0x05010400u);
                const uint32_t hi = __builtin_amdgcn_perm(v[2 * j + 1][f], v[2 * j][f], 0x07030602u);
                widen4<CODES>(lo, w[0][j], w[1][j]);
                widen4<CODES>(hi, w[2][j], w[3][j]);
            } else {
#pragma unroll
                for (int n = 0; n < 4; ++n)
                    w[n][j] = __builtin_amdgcn_perm(
                        __float_as_uint((float)(int8_t)(v[2 * j + 1][f] >> (8 * n))),
                        __float_as_uint((float)(int8_t)(v[2 * j][f] >> (8 * n))), 0x07060302u);
            }
        }
    }
};

// Which values of a dword of V are not finite: all ones in their places.
template <int CODES>
__device__ __forceinline__ uint32_t not_finite(uint32_t x) {
    if constexpr (CODES == NCM_KV_BF16) {
        const uint32_t e = x & 0x7F807F80u;
        return ((e & 0xFFFFu) == 0x7F80u ? 0xFFFFu : 0u) | ((e >> 16) == 0x7F80u ? 0xFFFF0000u : 0u);
    } else if constexpr (CODES == NCM_KV_FP8) {
        return ((((x & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u) >> 7) * 0xFFu;
    } else {
        return 0u;
    }
}

__device__ __forceinline__ float max_over_groups(float v) {
    u32x2_t p = swap16(__float_as_uint(v));
    v = fmaxf(__uint_as_float(p[0]), __uint_as_float(p[1]));
    p = swap32(__float_as_uint(v));
    return fmaxf(__uint_as_float(p[0]), __uint_as_float(p[1]));
}
__device__ __forceinline__ float sum_over_groups(float v) {
    u32x2_t p = swap16(__float_as_uint(v));
    v = __uint_as_float(p[0]) + __uint_as_float(p[1]);
    p = swap32(__float_as_uint(v));
    return __uint_as_float(p[0]) + __uint_as_float(p[1]);
}

// The unit's queries, in the order of the products' operands (element [rr][s]
// [lane] is lane's operand of k-step s), which the four wavefronts share; and
// at a unit's end their states.
template <int HD, int R>
struct Lds {
    static constexpr int PITCH = HD + 4;
    union {
        u32x4_t q[R][HD / 32][64];
        float o[2][16 * R][PITCH];
    };
    float m[4][16 * R], l[4][16 * R];
};

// A wavefront's softmax state for 16 R pairs, and what it needs of them: lane
// l holds pair l % 16 of each sixteen.
template <int HD, int R>
struct State {
    f32x4_t o[R][HD / 16];
    float m[R], l[R];  // l: of the lane group's own tokens
    int row[R];        // the pair's row of the request
    int near[R];       // it sees tokens above this
};

// Which of a tile's 32 tokens the lane's pair sees: bit 4 half + i for token 16
// half + 4 g + i. there: bit t, token key + t exists.
__device__ __forceinline__ uint32_t seen_tokens(const AttnArgs& a, const Need& d, int row, int near,
                                                int key, uint32_t there, int g) {
    const int j0 = key - d.before, word = j0 >> 5, words = (int)a.mask_words * 2;
    uint32_t bits = 0;  // of new tokens
    if (a.tree_mask) {
        const uint32_t* m = a.tree_mask + (int64_t)(d.q.o0 + row) * words;
        const uint32_t lo = word >= 0 && word < words ? m[word] : 0;
        const uint32_t hi = word >= -1 && word + 1 < words ? m[word + 1] : 0;
        bits = (uint32_t)((((uint64_t)hi << 32) | lo) >> (j0 & 31));
    }
    uint32_t see = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int at = 16 * (i / 4) + 4 * g + i % 4, token = key + at;
        const bool old = token < d.before;
        const bool ok = old || !a.tree_mask ? token > near && (old || j0 + at <= row)
                                            : (bits >> at) & 1u;
        see |= (ok && ((there >> at) & 1u) ? 1u : 0u) << i;
    }
    return see;
}

// V where some tokens are not there, or hold a value that is not finite: 0
// times either must stay 0 for a pair that does not see them. Tokens that are
// not there become zero, whatever their places hold. Infinities and NaN become
// zero too, and are added to the outputs of the pairs that see them from their
// token's row in the cache, one such token after another.
template <int HD, int CODES, int R>
__device__ __forceinline__ void clean_values(const AttnArgs& a, int h, int key, int page0, int page1,
                                             Tile<HD, CODES>& t, const uint32_t (&see)[R],
                                             uint32_t there, int lane, State<HD, R>& st) {
    typedef Tile<HD, CODES> T;
    const int c = lane & 15, g = lane >> 4;
    uint32_t bad = 0;  // bit i: the lane's token i holds one
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const bool ok = (there >> (16 * (i / 4) + 4 * g + i % 4)) & 1u;
#pragma unroll
        for (int u = 0; u < T::VW; ++u) {
            t.v[i][u] = ok ? t.v[i][u] : 0u;
            const uint32_t m = not_finite<CODES>(t.v[i][u]);
            t.v[i][u] &= ~m;
            bad |= m ? 1u << i : 0u;
        }
    }
    if constexpr (CODES == NCM_KV_INT8) return;
    if (!__any(bad != 0)) return;
    for (int at = 0; at < 32; ++at) {
        const int i = 4 * (at / 16) + at % 4, tg = (at % 16) / 4;
        const uint64_t in_lanes = __ballot(g == tg && ((bad >> i) & 1u));
        if (!in_lanes) continue;
        const int64_t page = at < 16 ? page0 : page1;
        const int64_t row = ((int64_t)h << a.cache.page_log2) +
                            ((key + at) & ((1 << a.cache.page_log2) - 1));
        const char* p = a.cache.v + (page * a.cache.v_stride + row * HD) * T::ES;
        bool sees[R];
#pragma unroll
        for (int rr = 0; rr < R; ++rr) sees[rr] = (__shfl((int)see[rr], 16 * tg + c) >> i) & 1;
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            const typename T::vec v = *(const typename T::vec*)(p + (4 * g + x) * (HD / 16) * T::ES);
#pragma unroll
            for (int u = 0; u < T::VW; ++u) {
                const uint32_t odd = v[u] & not_finite<CODES>(v[u]);
#pragma unroll
                for (int k = 0; k < 4 / T::ES; ++k) {
                    // Where it is not finite, the value; else 0.
                    const uint32_t bits = odd >> (8 * T::ES * k);
                    const float add = T::ES == 2 ? __uint_as_float(bits << 16)
                                                 : (bits & 0x7Fu) ? __builtin_nanf("") : 0.0f;
#pragma unroll
                    for (int rr = 0; rr < R; ++rr)
                        st.o[rr][4 / T::ES * u + k][x] += sees[rr] ? add : 0.0f;
                }
            }
        }
    }
}

// Adds a tile's 32 tokens and loads the next tile's into its registers, K once
// the scores are formed and V once the outputs are: each load has the other
// half of a round to arrive in, and a wavefront needs one tile's registers.
// FULL: every pair sees every token.
template <bool FULL, int HD, int CODES, int R, typename NextK, typename NextV>
__device__ __forceinline__ void add_tokens(const AttnArgs& a, const Need& d, int h,
                                           Tile<HD, CODES>& t, State<HD, R>& st, int key, int page0,
                                           int page1, uint32_t there, float to_log2, float lag,
                                           int lane, const Lds<HD, R>& lds, NextK next_k,
                                           NextV next_v) {
    const int g = lane >> 4;
    float s[R][8];
    // The queries are read from LDS each round: hoisted out of the loop they
    // would take the registers that a second or third wavefront runs on.
    asm volatile("" ::: "memory");
    {
        f32x4_t sc[R][2];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
#pragma unroll
            for (int rr = 0; rr < R; ++rr) sc[rr][half] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int k = 0; k < HD / 32; ++k) {
                const bf16x8_t op = t.k_operand(half, k);
#pragma unroll
                for (int rr = 0; rr < R; ++rr)
                    sc[rr][half] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                        op, __builtin_bit_cast(bf16x8_t, lds.q[rr][k][lane]), sc[rr][half], 0, 0, 0);
            }
        }
#pragma unroll
        for (int rr = 0; rr < R; ++rr)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                s[rr][i] = sc[rr][i / 4][i % 4];
                if constexpr (CODES != NCM_KV_BF16) s[rr][i] = s[rr][i] * (t.ks[i / 4][i % 4] * to_log2);
            }
    }
    next_k();
    uint32_t see[R];
    if constexpr (!FULL) {
#pragma unroll
        for (int rr = 0; rr < R; ++rr) {
            see[rr] = seen_tokens(a, d, st.row[rr], st.near[rr], key, there, g);
#pragma unroll
            for (int i = 0; i < 8; ++i) s[rr][i] = (see[rr] >> i) & 1u ? s[rr][i] : -INFINITY;
        }
    }
    bf16x8_t p[R], rest[R];
#pragma unroll
    for (int rr = 0; rr < R; ++rr) {
        float top = s[rr][0];
#pragma unroll
        for (int i = 1; i < 8; ++i) top = fmaxf(top, s[rr][i]);
        top = max_over_groups(top);
        // m follows the maximum once that has grown by 2^8: sums in fp32 and
        // the rounding of p, a relative one, are as good to 2^8 as to 1, and o
        // is seldom touched after the first tiles. The comparison fails for a
        // pair that has seen nothing yet. bf16 caches: s and m are plain
        // products, their difference takes the scale: scaled first, two large
        // scores would differ by their products' roundings, and 2^31 is enough
        // for that to leave the exponent's range.
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
            // A scale of 0 times -inf, and 0 times a V scale that is NaN.
            if constexpr (!FULL) s[rr][i] = (see[rr] >> i) & 1u ? s[rr][i] : 0.0f;
            sum += s[rr][i];
            if constexpr (CODES != NCM_KV_BF16) s[rr][i] = s[rr][i] * t.vs[i / 4][i % 4];
            if constexpr (CODES != NCM_KV_BF16 && !FULL)
                s[rr][i] = (see[rr] >> i) & 1u ? s[rr][i] : 0.0f;
        }
        st.l[rr] += sum;
        // As two bf16 terms for the product, the upper 8 bits and the rest: one
        // bf16 alone would add an error as large as the output's own rounding.
        u32x4_t hi, lo;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t x = __float_as_uint(s[rr][2 * i]), y = __float_as_uint(s[rr][2 * i + 1]);
            hi[i] = __builtin_amdgcn_perm(y, x, 0x07060302u);
            // (1 + 2^-20) p less the upper term: above 0 wherever p is, so that
            // an infinite value times it is no NaN.
            lo[i] = bf16x2_rne(fmaf(s[rr][2 * i], 1.00000095367431640625f,
                                    -__uint_as_float(x & 0xFFFF0000u)),
                               fmaf(s[rr][2 * i + 1], 1.00000095367431640625f,
                                    -__uint_as_float(y & 0xFFFF0000u)));
        }
        p[rr] = __builtin_bit_cast(bf16x8_t, hi);
        rest[rr] = __builtin_bit_cast(bf16x8_t, lo);
    }
    if constexpr (!FULL) clean_values<HD, CODES, R>(a, h, key, page0, page1, t, see, there, lane, st);
#pragma unroll
    for (int f = 0; f < HD / 64; ++f) {
        uint32_t w[4][4];
        t.v_operands(f, w);
#pragma unroll
        for (int n = 0; n < 4; ++n) {
            const bf16x8_t v = __builtin_bit_cast(bf16x8_t, u32x4_t{w[n][0], w[n][1], w[n][2], w[n][3]});
#pragma unroll
            for (int rr = 0; rr < R; ++rr)
                st.o[rr][4 * f + n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                    v, p[rr], st.o[rr][4 * f + n], 0, 0, 0);
#pragma unroll
            for (int rr = 0; rr < R; ++rr)
                st.o[rr][4 * f + n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                    v, rest[rr], st.o[rr][4 * f + n], 0, 0, 0);
        }
    }
    next_v();
}


// Tiles [first, first + count) of a unit, by the whole workgroup: into `out`
// where slot < 0, else as a part.
template <int HD, int CODES, int R>
__device__ __forceinline__ void run_unit(const AttnArgs& a, const Need& d, int r, int h, int block,
                                         int first, int count, int slot, Lds<HD, R>& lds) {
    const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
    const int c = lane & 15, g = lane >> 4;
    const int pairs = d.q.n * a.group - block * 16 * R;  // of the unit, in all
    typedef Tile<HD, CODES> T;
    State<HD, R> st;
    int far = -1;  // the largest `near`
    // A negative scale turns the queries' signs, so that the maximum of the
    // products is that of the scores.
    const uint32_t sign = a.scale < 0.0f ? 0x80008000u : 0u;
    // For a scale of 0 the least above it: the difference of m's start to a large
    // product is an infinity, which 0 would turn into NaN.
    const float to_log2 = a.scale == 0.0f ? 1.4e-45f : fabsf(a.scale) * 1.4426950408889634f;
    // 2^8 in plain products; low enough for the first of them to move m, whatever
    // the scale: no product less the start may leave fp32's range upwards.
    const float lag = fminf(8.0f / to_log2, 1e30f);
#pragma unroll
    for (int rr = 0; rr < R; ++rr) {
        const int pair = block * 16 * R + min(16 * rr + c, pairs - 1);
        const int row = pair / a.group, head = h * a.group + pair - row * a.group;
        const uint16_t* q = a.q + (d.q.o0 + row) * a.q_stride + (int64_t)head * HD;
#pragma unroll
        for (int s = 0; s < HD / 32; ++s)  // a quarter of them by each wavefront
            if ((rr * (HD / 32) + s) % 4 == wave)
                lds.q[rr][s][lane] = *(const u32x4_t*)(q + T::k_dims(s, g)) ^ sign;
#pragma unroll
        for (int n = 0; n < HD / 16; ++n) st.o[rr][n] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
        st.m[rr] = kNoMax;
        st.l[rr] = 0.0f;
        st.row[rr] = row;
        st.near[rr] = -1;
        if (a.window > 0) {
            int64_t pos = (int64_t)d.q.before + row;
            if (a.positions) pos = max(a.positions[d.q.o0 + row], d.q.before);
            st.near[rr] = (int)min(max(pos - a.window, (int64_t)-1), kMaxTokens);
            far = max(far, st.near[rr]);
        }
    }
    if (a.window > 0)
#pragma unroll
        for (int x = 1; x < 16; x <<= 1) far = max(far, __shfl_xor(far, x));
    far = uniform(far);

    // Pages of 16 tokens each, 32 tiles' worth at a time: lane 2 s + half.
    const int key0 = (d.tile0 + first) * kTile + 32 * wave;
    int pages = -1;
    auto look_up = [&](int s) {
        const int t = key0 + (s + (lane >> 1)) * kTile + 16 * (lane & 1);
        pages = (s + (lane >> 1)) < count && t < d.end ? page_of(a.batch, a.cache, r, t) : -1;
    };
    auto page = [&](int s, int half) { return __builtin_amdgcn_readlane(pages, 2 * (s & 31) + half); };
    auto tokens_there = [&](int key, int p0, int p1) {
        const int n = min(max(d.end - key, 0), 32);
        uint32_t m = n >= 32 ? 0xFFFFFFFFu : (1u << n) - 1u;
        if (p0 < 0) m &= 0xFFFF0000u;
        if (p1 < 0) m &= 0x0000FFFFu;
        return m;
    };
    __syncthreads();  // the queries
    T t;
    look_up(0);
    int p0 = page(0, 0), p1 = page(0, 1);
    t.load_k(a.cache, h, key0, max(p0, 0), max(p1, 0), lane);
    t.load_v(a.cache, h, key0, max(p0, 0), max(p1, 0), lane);
    // A round: 32 tokens, their K and V in t, their pages in p0 and p1.
    int s = 0;
    auto round = [&](auto full) {
        const int key = key0 + s * kTile, q0 = p0, q1 = p1;
        const uint32_t there = decltype(full)::value ? 0u : tokens_there(key, p0, p1);
        // The last round loads its own tokens again: no branch around the loads.
        const int s2 = min(s + 1, count - 1), key2 = key0 + s2 * kTile;
        if (s2 != s && (s2 & 31) == 0) look_up(s2);
        p0 = page(s2, 0), p1 = page(s2, 1);
        add_tokens<decltype(full)::value, HD, CODES, R>(
            a, d, h, t, st, key, max(q0, 0), max(q1, 0), there, to_log2, lag, lane, lds,
            [&] { t.load_k(a.cache, h, key2, max(p0, 0), max(p1, 0), lane); },
            [&] { t.load_v(a.cache, h, key2, max(p0, 0), max(p1, 0), lane); });
        ++s;
    };
    while (s < count) {
        while (s < count && (p0 | p1) >= 0 && key0 + s * kTile + 32 <= d.before &&
               key0 + s * kTile > far)
            round(std::true_type());
        if (s < count) round(std::false_type());
    }

    // The four wavefronts' states, joined; the queries are done with.
#pragma unroll
    for (int rr = 0; rr < R; ++rr) {
        st.l[rr] = sum_over_groups(st.l[rr]);
        // Maxima of plain products to exponents of 2, but for a pair that saw nothing.
        if (CODES == NCM_KV_BF16 && st.m[rr] > kNoMax)
            st.m[rr] = fmaxf(st.m[rr] * to_log2, kNoMax);
        if (g == 0) lds.m[wave][16 * rr + c] = st.m[rr];
    }
    __syncthreads();
    // The upper two wavefronts' outputs to the lower two, then those to all.
    auto put = [&] {
#pragma unroll
        for (int rr = 0; rr < R; ++rr)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int n = 0; n < HD / 16; n += 4) {
                    f32x4_t v;
#pragma unroll
                    for (int x = 0; x < 4; ++x) v[x] = st.o[rr][n + x][i];
                    *(f32x4_t*)&lds.o[wave & 1][16 * rr + c][(HD / 16) * (4 * g + i) + n] = v;
                }
    };
#pragma unroll
    for (int rr = 0; rr < R; ++rr) {
        const int pr = 16 * rr + c;
        const float top = fmaxf(fmaxf(lds.m[0][pr], lds.m[1][pr]), fmaxf(lds.m[2][pr], lds.m[3][pr]));
        const float f = __builtin_amdgcn_exp2f(st.m[rr] - top);
        if (g == 0) lds.l[wave][pr] = st.l[rr] * f;
#pragma unroll
        for (int n = 0; n < HD / 16; ++n) st.o[rr][n] *= f;
    }
    if (wave >= 2) put();
    __syncthreads();
    if (wave < 2) {
#pragma unroll
        for (int rr = 0; rr < R; ++rr)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int n = 0; n < HD / 16; n += 4) {
                    const f32x4_t v =
                        *(const f32x4_t*)&lds.o[wave][16 * rr + c][(HD / 16) * (4 * g + i) + n];
#pragma unroll
                    for (int x = 0; x < 4; ++x) st.o[rr][n + x][i] += v[x];
                }
        put();  // where it has just read
    }
    __syncthreads();
    constexpr int CH = HD / 8;
    const int dim = 8 * (tid % CH);
    for (int pr = tid / CH; pr < min(16 * R, pairs); pr += 256 / CH) {
        float l = 0.0f;
#pragma unroll
        for (int w = 0; w < 4; ++w) l += lds.l[w][pr];
        const f32x4_t v0 = *(const f32x4_t*)&lds.o[0][pr][dim] + *(const f32x4_t*)&lds.o[1][pr][dim];
        const f32x4_t v1 =
            *(const f32x4_t*)&lds.o[0][pr][dim + 4] + *(const f32x4_t*)&lds.o[1][pr][dim + 4];
        if (slot < 0) {
            const int pair = block * 16 * R + pr;
            const int row = pair / a.group, head = h * a.group + pair - row * a.group;
            const float inv = l == 0.0f ? 0.0f : 1.0f / l;
            u32x4_t b;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                b[i] = bf16x2_bits_rne(v0[2 * i] * inv, v0[2 * i + 1] * inv);
                b[2 + i] = bf16x2_bits_rne(v1[2 * i] * inv, v1[2 * i + 1] * inv);
            }
            *(u32x4_t*)(a.out + (d.q.o0 + row) * a.out_stride + (int64_t)head * HD + dim) = b;
        } else {
            const int64_t at = (int64_t)slot * 16 * R + pr;
            if (dim == 0) {
                const float top = fmaxf(fmaxf(lds.m[0][pr], lds.m[1][pr]),
                                        fmaxf(lds.m[2][pr], lds.m[3][pr]));
                a.part_ml[at] = float2{top, l};
            }
            *(f32x4_t*)(a.part_o + at * HD + dim) = v0;
            *(f32x4_t*)(a.part_o + at * HD + dim + 4) = v1;
        }
    }
    __syncthreads();
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
        run_unit<HD, CODES, R>(a, d, r, h, u - h * d.blocks, first, count, slot, lds);
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
