// The pick of a token from given random numbers (ncm_sample_dev).
//
// Tokens stand in the order (logit descending, id ascending), a token's weight
// is w = exp((x - max) / T). Top-k, top-p and min-p each keep the beginning of
// that order, and the token is the first whose cumulative weight passes u times
// the kept tokens' sum. Weights are integers, exp in 64-bit floats times 2^43
// rounded, so that sums (of at most 2^20 tokens) neither round nor depend on
// the order in which they are made, and a cut or a draw next to a border falls
// where 64-bit arithmetic puts it.
//
// Few tokens matter to a row: those next to its cuts and to its draw. Where they
// stand is found from sums over 2048 bins of (max - x) / T, equally wide over the
// row's range or over the 31 units in which tokens have weights:
//   1. the largest logit of every segment (1 KB) of a row, by many workgroups;
//   2. weights (and numbers, for top-k) of its bins, in LDS, then added to the
//      row's in memory; segments whose largest logit is behind the k-th largest
//      of the segments', or too weak for min-p, are left out;
//   3. the bins that a cut or the draw can fall into, from the row's bins, and
//      their tokens into a list, from the segments that can have some;
//   4. each listed token's cumulative weight, exactly, from its bin's and the
//      listed tokens of its bin; cuts and draw are minima over these.
// Bound by the four launches' chains of loads for few rows: 4.6 + 6.5 + 8.4 + 6.0 us
// for 4 rows of 128256 with all rules in use. For many by the operations of step 2 (an
// exp in 64 bits and two LDS atomics a token) and the two later reads, which L2 serves
// in part: 151 rows of 151936, half of the logits masked, all rules in use by some rows,
// 19 (4.9 TB/s) + 32 + 22 + 7. Step 4 compares every pair of listed tokens: the same
// rows where one lists 515 take 127 us in place of 78.
//
// A row that lists more than 1024 is done digit by digit of the token's 52-bit place
// in the order (32 bits of the logit, 20 of the id): sums of the tokens by their next
// digit, then the digit where the target is passed. One workgroup reads the row once
// and five times a cut and the draw for that. It happens where the tokens of a bin are
// many: bf16 logits away from zero (about 20 they are 1/8 apart), equal logits, and a
// flat row whose range a finite mask stretches, so that its bins are 1/64 T wide. One
// row of 128256, us, without rules and with top_p 0.95: bf16 about 20 with a standard
// deviation of 2, 484 and 892 (64 rows 517 and 935), about 0 with top_p 46; fp32 with a
// deviation of 1 and some logits at -1e9, with top_p 705, without those 51; all equal
// 1010 and 1925. top_k keeps the lists short (50 and the mask: 21).
#include "step.h"

namespace ncm {
namespace {

constexpr double kOne = 0x1p43;  // the largest weight
constexpr int64_t kMaxVocab = int64_t(1) << 20;
constexpr int kThreads = 1024, kWavesOf = kThreads / 64;
// Of the row's last kernel: few enough for its rare part to have all the registers
// that it wants (1024 threads of 128: scratch memory, 12 us in place of 5 for 4
// rows that have no use for that part).
constexpr int kPickThreads = 256, kPickWaves = kPickThreads / 64;
constexpr int kBins = 2048, kList = 1024;

struct SampleArgs {
    ncm_sample_rules_t rules;
    const void* logits;
    const void* uniform;
    int32_t* tokens;
    float* probabilities;
    int64_t stride;
    int rows, vocab;
    bool wide_uniform;
    char* space;
    int64_t row_bytes;
    int slices;
};

// What a row is drawn by.
struct RowRule {
    double per;      // 32 log2(e) / T
    double top_p;    // 1: off
    double min_p;    // 0: off
    double uniform;
    float bins;      // bins a unit of half a logit, at least; above 0
    int top_k;       // 0: off
    int greedy;
    int request;     // -1: none
};

// Ranges of bins that hold a cut or the draw, whatever the tokens inside them
// decide, and what is known ahead of that.
struct Ranges {
    int lo[4], hi[4];   // top-k, top-p, min-p, draw; empty where lo > hi
    uint64_t all;       // the sum behind top-k where its range is empty
    uint64_t sure;      // the sum of the bins below `strong`
    int strong;         // bins below it hold only tokens of at least min_p
    int pad;

    __device__ __forceinline__ int first() const { return min(min(lo[0], lo[1]), min(lo[2], lo[3])); }
    __device__ __forceinline__ int last() const { return max(max(hi[0], hi[1]), max(hi[2], hi[3])); }
    __device__ __forceinline__ bool has(int b) const {
        bool in = false;
#pragma unroll
        for (int i = 0; i < 4; ++i) in |= b >= lo[i] && b <= hi[i];
        return in;
    }
};

// A row's part of the workspace.
struct RowSpace {
    RowRule* rule;
    uint64_t* sums;     // [kBins]
    uint32_t* counts;   // [kBins]
    uint2* ends;        // [slices]: the first and the last key of a slice
    Ranges* ranges;
    uint64_t* list;     // [kList]: places
    uint64_t* below;    // [kList]: the sum of the bins below the place's
    uint32_t* ahead;    // [kList]: their number
    uint32_t* listed;   // places there are for the list
    uint32_t* firsts;   // [segments]: the first key of a segment
};

__device__ __forceinline__ RowSpace row_space(const SampleArgs& a, int row) {
    char* p = a.space + row * a.row_bytes;
    RowSpace r;
    r.rule = (RowRule*)p;
    r.ranges = (Ranges*)(p + sizeof(RowRule));
    r.sums = (uint64_t*)(r.ranges + 1);
    r.list = r.sums + kBins;
    r.below = r.list + kList;
    r.ends = (uint2*)(r.below + kList);
    r.counts = (uint32_t*)(r.ends + a.slices);
    r.ahead = r.counts + kBins;
    r.listed = r.ahead + kList;
    r.firsts = r.listed + 1;
    return r;
}

// The request of a row, by each wavefront: 64 boundaries at a time.
__device__ __forceinline__ int request_row(const ncm_sample_rules_t& u, int row) {
    if (!u.offsets) return row;
    const int lane = threadIdx.x & 63;
    int lo = 0, hi = (int)u.requests;  // the first request that ends behind the row
    while (hi > lo) {
        const int step = (hi - lo + 63) / 64, at = min(lo + (lane + 1) * step, hi) - 1;
        const uint64_t behind = __ballot(u.offsets[at + 1] > row);
        if (!behind) return -1;
        const int first = __ffsll((unsigned long long)behind) - 1;
        const int end = min(lo + (first + 1) * step, hi);
        lo += first * step;
        hi = end;
        if (hi - lo == 1) break;
    }
    return hi > lo && u.offsets[lo] <= row ? lo : -1;
}

__device__ __forceinline__ RowRule rule_of(const SampleArgs& a, int row) {
    const ncm_sample_rules_t& u = a.rules;
    RowRule q = {};
    const int r = q.request = request_row(u, row);
    if (r < 0) return q;
    const float t = u.temperature ? u.temperature[r] : 1.0f;
    q.greedy = !(t > 0.0f);
    q.per = 32.0 * 1.44269504088896340736 / (double)fmaxf(t, 0x1p-96f);
    q.bins = 128.0f / fminf(fmaxf(t, 0x1p-96f), 3.40282347e38f);
    q.top_k = u.top_k ? max(u.top_k[r], 0) : 0;
    q.top_p = u.top_p ? (double)u.top_p[r] : 1.0;
    if (!(q.top_p < 1.0)) q.top_p = 1.0;
    q.min_p = u.min_p ? (double)u.min_p[r] : 0.0;
    q.min_p = q.min_p > 0.0 ? fmin(q.min_p, 1.0) : 0.0;
    q.uniform = a.wide_uniform ? ((const double*)a.uniform)[row] : (double)((const float*)a.uniform)[row];
    q.uniform = q.uniform > 0.0 ? fmin(q.uniform, 1.0 - 0x1p-53) : 0.0;
    return q;
}

// A logit as the order has it: infinity the largest finite value, zeros one
// value, NaN and -infinity not there (-infinity).
__device__ __forceinline__ float value_of(float x) {
    x = x == x ? fminf(x, 3.40282347e38f) : -INFINITY;
    return x == 0.0f ? 0.0f : x;
}
// A logit's key, and with its id its place: both ascending in the order. No key
// is kNoKey, that of the NaN of all ones.
constexpr uint32_t kNoKey = 0xFFFFFFFFu;
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t b = __float_as_uint(x);
    return b & 0x80000000u ? b : ~(b | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t key) {
    return __uint_as_float(key & 0x80000000u ? key : ~key & 0x7FFFFFFFu);
}
__device__ __forceinline__ uint64_t place_of(float x, int id) {
    return ((uint64_t)key_of(x) << 20) | (uint32_t)id;
}
__device__ __forceinline__ float place_value(uint64_t p) { return key_value((uint32_t)(p >> 20)); }
__device__ __forceinline__ int place_id(uint64_t p) { return (int)(p & 0xFFFFFu); }

// 2^(j / 32), and in LDS.
__device__ const double kPowers[32] = {
    1.0, 1.0218971486541166, 1.0442737824274138, 1.0671404006768237,
    1.0905077326652577, 1.1143867425958924, 1.1387886347566916, 1.1637248587775775,
    1.189207115002721, 1.215247359980469, 1.241857812073484, 1.2690509571917332,
    1.2968395546510096, 1.3252366431597413, 1.3542555469368927, 1.383909881963832,
    1.4142135623730951, 1.4451808069770467, 1.4768261459394993, 1.5091644275934228,
    1.5422108254079407, 1.5759808451078865, 1.6104903319492543, 1.645755478153965,
    1.681792830507429, 1.718619298122478, 1.7562521603732995, 1.7947090750031072,
    1.8340080864093424, 1.8741676341103, 1.9152065613971474, 1.9571441241754002};
typedef double Powers[32];
__device__ __forceinline__ void fill(Powers& powers) {
    if (threadIdx.x < 32) powers[threadIdx.x] = kPowers[threadIdx.x];
}

// rint(2^43 exp((x - top) / T)), per = 32 log2(e) / T: a power of 2^(1 / 32) times
// the exponential of the rest, at most ln(2) / 64 = 0.0108 to either side, by its
// Taylor polynomial of degree 5, good to 0.0108^6 / 720 = 2^-48.
__device__ __forceinline__ uint64_t weight_of(float x, float top, double per, const Powers& powers) {
    const double y = fmax(((double)x - (double)top) * per, -1600.0);
    const double n = rint(y), r = (y - n) * (0.693147180559945309417 / 32.0);
    const int i = (int)n;
    double p = fma(r, 1.0 / 120.0, 1.0 / 24.0);
    p = fma(p, r, 1.0 / 6.0);
    p = fma(p, r, 0.5);
    p = fma(p, r, 1.0);
    p = fma(p, r, 1.0);
    // times 2^(i / 32 + 43), and 2^52 for the rounding: the integer is in the low
    // bits (0 from 44 bits below the largest on).
    const double scale =
        __longlong_as_double(__double_as_longlong(powers[i & 31]) + (int64_t)((uint64_t)((i >> 5) + 43) << 52));
    return (uint64_t)__double_as_longlong(fma(p, scale, 0x1p52)) & ((uint64_t(1) << 52) - 1);
}

// floor(f * total) and whether it is more than that, exactly: the product of f's 53
// bits, f = m 2^-s, and the total's 64. f in [0, 1].
__device__ __forceinline__ uint64_t share_of(double f, uint64_t total, bool& more) {
    const uint64_t bits = (uint64_t)__double_as_longlong(f), e = (bits >> 52) & 0x7FF;
    const uint64_t m = (bits & ((uint64_t(1) << 52) - 1)) | (e ? uint64_t(1) << 52 : 0);
    const int s = 1075 - max((int)e, 1);  // 52 at least
    const uint64_t lo = m * total, hi = __umul64hi(m, total);
    if (s < 64) {
        more = (lo & ((uint64_t(1) << s) - 1)) != 0;
        return (hi << (64 - s)) | (lo >> s);
    }
    const int t = min(s - 64, 63);  // hi is below 2^53
    more = lo != 0 || (hi & ((uint64_t(1) << t) - 1)) != 0;
    return hi >> t;
}

// The cumulative weight at which a part p of `total` is reached, and a draw's.
__device__ __forceinline__ uint64_t cut_at(double p, uint64_t total) {
    bool more;
    const uint64_t target = share_of(fmax(p, 0.0), total, more);
    return max(target + (more ? 1 : 0), (uint64_t)1);
}
__device__ __forceinline__ uint64_t draw_at(double u, uint64_t total) {
    bool more;
    return share_of(u, total, more) + 1;
}

__device__ __forceinline__ void put_token(const SampleArgs& a, int row, uint64_t place,
                                          uint64_t weight, uint64_t kept) {
    a.tokens[row] = place_id(place);
    if (a.probabilities) a.probabilities[row] = (float)((double)weight / (double)kept);
}

// A row in accesses of 16 bytes, aligned in memory, N logits each, and in segments
// of 64 such accesses; the first and the last access may hold values that are not
// the row's.
template <bool BF16>
struct Row {
    static constexpr int SIZE = BF16 ? 2 : 4, N = 16 / SIZE;
    const char* base;
    int skip;      // values ahead of the row in its first access
    int vocab;
    int segments;

    __device__ __forceinline__ Row(const SampleArgs& a, int row) {
        base = (const char*)a.logits + (int64_t)row * a.stride * SIZE;
        skip = (int)((uintptr_t)base % 16) / SIZE;
        vocab = a.vocab;
        segments = (vocab + skip + 64 * N - 1) / (64 * N);
    }
    // The id of the lane's first value of a segment.
    __device__ __forceinline__ int first(int segment) const {
        return (segment * 64 + (int)(threadIdx.x & 63)) * N - skip;
    }
    __device__ __forceinline__ bool whole(int segment) const {
        return first(segment) >= 0 && first(segment) + N <= vocab;
    }
    __device__ __forceinline__ u32x4_t load(int segment) const {
        u32x4_t raw = {0, 0, 0, 0};
        if (whole(segment)) raw = *(const u32x4_t*)(base + (int64_t)first(segment) * SIZE);
        return raw;
    }
    static __device__ __forceinline__ float raw_value(const u32x4_t& raw, int i) {
        return BF16 ? __uint_as_float(i % 2 ? raw[i / 2] & 0xFFFF0000u : raw[i / 2] << 16)
                    : __uint_as_float(raw[BF16 ? 0 : i]);
    }
    __device__ __forceinline__ float one(int id) const {
        return value_of(BF16 ? __uint_as_float((uint32_t)((const uint16_t*)base)[id] << 16)
                             : ((const float*)base)[id]);
    }
    // -infinity where there is no value of the row.
    __device__ __forceinline__ void values(int segment, const u32x4_t& raw, float (&x)[N]) const {
        if (whole(segment)) {
#pragma unroll
            for (int i = 0; i < N; ++i)
                x[i] = value_of(raw_value(raw, i));
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int id = first(segment) + i;
                x[i] = id >= 0 && id < vocab ? one(id) : -INFINITY;
            }
        }
    }
    // f(values, the lane's first id, segment) for segments s0 .. s1 - 1, one of
    // every wavefront at a time and AHEAD of them loaded together.
    template <int AHEAD, int WAVES, typename F>
    __device__ __forceinline__ void each(int s0, int s1, F f) const {
        for (int s = s0 + (int)(threadIdx.x >> 6); s < s1; s += WAVES * AHEAD) {
            u32x4_t raw[AHEAD];
#pragma unroll
            for (int k = 0; k < AHEAD; ++k)
                if (s + k * WAVES < s1) raw[k] = load(s + k * WAVES);
#pragma unroll
            for (int k = 0; k < AHEAD; ++k) {
                const int at = s + k * WAVES;
                if (at >= s1) break;
                float x[N];
                values(at, raw[k], x);
                f(x, first(at), at);
            }
        }
    }
};

// Sums and numbers by a place's next digit.
struct Digits {
    uint64_t sums[2048];
    uint32_t counts[2048];
    uint64_t wave_sums[kPickWaves];
    uint64_t wave_counts[kPickWaves];
    uint64_t place, sum, count;
    int found;
};

// The first place whose cumulative weight (COUNT: number) is at least `target`;
// sum: the cumulative weight there. False where all together is less.
template <bool BF16, bool COUNT>
__device__ bool find_place(const Row<BF16>& logits, float top, const RowRule& q,
                           const Powers& powers, uint64_t target, Digits& s, uint64_t& place,
                           uint64_t& sum) {
    constexpr int PER = 2048 / kPickThreads;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    uint64_t prefix = 0, done_sum = 0, done_count = 0;
    int low = 52;  // digits above it are fixed
    while (low > 0) {
        const int bits = low > 30 ? 11 : 10, next = low - bits;
        __syncthreads();
        for (int i = tid; i < 2048; i += kPickThreads) s.sums[i] = 0, s.counts[i] = 0;
        if (tid == 0) s.found = 0;
        __syncthreads();
        logits.template each<4, kPickWaves>(0, logits.segments, [&](const auto& x, int first, int) {
#pragma unroll
            for (int i = 0; i < Row<BF16>::N; ++i) {
                const uint64_t p = place_of(x[i], first + i);
                if (x[i] == -INFINITY || (p >> low) != prefix) continue;
                const int digit = (int)((p >> next) & ((1 << bits) - 1));
                atomicAdd(&s.counts[digit], 1u);
                const uint64_t w = weight_of(x[i], top, q.per, powers);
                if (w) atomicAdd((unsigned long long*)&s.sums[digit], (unsigned long long)w);
            }
        });
        __syncthreads();
        uint64_t c = 0, w = 0;
        for (int i = 0; i < PER; ++i) c += s.counts[PER * tid + i], w += s.sums[PER * tid + i];
        uint64_t c_at = c, w_at = w;
        for (int x = 1; x < 64; x <<= 1) {
            const uint64_t oc = __shfl_up((unsigned long long)c_at, x);
            const uint64_t ow = __shfl_up((unsigned long long)w_at, x);
            if (lane >= x) c_at += oc, w_at += ow;
        }
        if (lane == 63) s.wave_sums[wave] = w_at, s.wave_counts[wave] = c_at;
        __syncthreads();
        c_at += done_count - c, w_at += done_sum - w;
        for (int v = 0; v < wave; ++v) c_at += s.wave_counts[v], w_at += s.wave_sums[v];
        // The thread's digits from here on, the target among them or not.
        for (int i = 0; i < PER; ++i) {
            const uint64_t n = s.counts[PER * tid + i], m = s.sums[PER * tid + i];
            const uint64_t before = COUNT ? c_at : w_at, after = before + (COUNT ? n : m);
            if (before < target && target <= after) {
                s.found = 1;
                s.place = (prefix << bits) | (uint64_t)(PER * tid + i);
                s.sum = w_at;
                s.count = c_at;
            }
            c_at += n, w_at += m;
        }
        __syncthreads();
        if (!s.found) return false;
        prefix = s.place, done_sum = s.sum, done_count = s.count;
        low = next;
    }
    place = prefix;
    sum = done_sum + weight_of(place_value(place), top, q.per, powers);
    return true;
}

__device__ __forceinline__ uint64_t wave_least(uint64_t v) {
    for (int x = 32; x; x >>= 1) v = min(v, (uint64_t)__shfl_xor((unsigned long long)v, x));
    return v;
}
__device__ __forceinline__ uint64_t wave_total(uint64_t v) {
    for (int x = 32; x; x >>= 1) v += __shfl_xor((unsigned long long)v, x);
    return v;
}
// Of a workgroup's values.
__device__ __forceinline__ uint64_t least_of(uint64_t v, uint64_t (&waves)[kPickWaves]) {
    v = wave_least(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = v;
    __syncthreads();
    for (int w = 0; w < kPickWaves; ++w) v = min(v, waves[w]);
    return v;
}
__device__ __forceinline__ uint64_t total_of(uint64_t v, uint64_t (&waves)[kPickWaves]) {
    v = wave_total(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0;
    for (int w = 0; w < kPickWaves; ++w) v += waves[w];
    return v;
}

// The least weight that min_p keeps.
__device__ __forceinline__ uint64_t least_weight(const RowRule& q) {
    return max((uint64_t)ceil(q.min_p * kOne), (uint64_t)1);
}

// A row by its places' digits.
template <bool BF16>
__device__ void pick_by_digits(const SampleArgs& a, int row, const RowRule& q, float top,
                               const Powers& powers, Digits& s) {
    const uint64_t least = least_weight(q);
    uint64_t all = 0, strong = 0;  // all weights, and those of at least min_p
    const Row<BF16> logits(a, row);
    logits.template each<4, kPickWaves>(0, logits.segments, [&](const auto& x, int, int) {
#pragma unroll
        for (int i = 0; i < Row<BF16>::N; ++i) {
            const uint64_t w = weight_of(x[i], top, q.per, powers);
            all += w;
            strong += w >= least ? w : 0;
        }
    });
    all = total_of(all, s.wave_sums);
    strong = total_of(strong, s.wave_counts);
    uint64_t place, sum;
    if (q.top_k && find_place<BF16, true>(logits, top, q, powers, q.top_k, s, place, sum)) all = sum;
    uint64_t kept = all;
    if (q.top_p < 1.0 &&
        find_place<BF16, false>(logits, top, q, powers, cut_at(q.top_p, all), s, place, sum))
        kept = min(kept, sum);
    kept = min(kept, strong);
    find_place<BF16, false>(logits, top, q, powers, draw_at(q.uniform, kept), s, place, sum);
    if (threadIdx.x == 0)
        put_token(a, row, place, weight_of(place_value(place), top, q.per, powers), kept);
}

// The row's bins: at least 64 a unit of (max - x) / T, or 2047 over all its
// values where these lie closer. By halves, whose differences fp32 holds for any
// two values; `per` is above 0, so that only what is no token gives a NaN.
struct Bins {
    float half;  // of the largest value
    float top, per;
    // Bins from the largest value to x: negative for +infinity, which counts as
    // the largest finite value.
    __device__ __forceinline__ float distance(float x) const { return fmaf(x, -0.5f, half) * per; }
    __device__ __forceinline__ int of(float x) const {
        return (int)fminf(distance(x), (float)(kBins - 1));
    }
};

// What all of a row's slices say: its first and its last value.
__device__ __forceinline__ uint2 ends_of(const RowSpace& sp, int slices) {
    const int lane = threadIdx.x & 63;
    const uint2 e = lane < slices ? sp.ends[lane] : make_uint2(kNoKey, 0u);
    return make_uint2(wave_min_xor(e.x), ~wave_min_xor(~e.y));
}
__device__ __forceinline__ Bins bins_of(uint2 ends, const RowRule& q) {
    const float top = key_value(ends.x), half = 0.5f * top;
    const float range = half - 0.5f * key_value(ends.y);
    return {half, top, range > 0.0f ? fmaxf(q.bins, fminf(2047.0f / range, 0x1p101f)) : q.bins};
}

// The bin where weights fall below the least that min_p keeps: as they are
// rounded, those from half a unit below it on reach it.
__device__ __forceinline__ int weak_bin(const Bins& bins, const RowRule& q) {
    // The logarithm times T: the logits' distance from the largest, in bins.
    const double border = ((double)least_weight(q) - 0.5) / kOne;
    const double d = -log(border) * (16.0 * 1.44269504088896340736) / q.per * (double)bins.per;
    return (int)fmin(d, (double)kBins);
}

template <bool BF16>
__global__ __launch_bounds__(kThreads) void sample_first_kernel(SampleArgs a) {
    __shared__ uint2 waves[kWavesOf];
    const int row = (int)(blockIdx.x / (uint32_t)a.slices), slice = (int)(blockIdx.x % (uint32_t)a.slices);
    const int lane = threadIdx.x & 63;
    const RowSpace sp = row_space(a, row);
    // What the row's next kernels start from.
    if (a.slices > 1)
        for (int i = slice * kThreads + (int)threadIdx.x; i < kBins; i += a.slices * kThreads)
            sp.sums[i] = 0, sp.counts[i] = 0;
    if (slice == 0 && threadIdx.x < 64) {
        const RowRule q = rule_of(a, row);
        if (threadIdx.x == 0) *sp.rule = q, *sp.listed = 0;
    }
    const Row<BF16> logits(a, row);
    uint32_t first = kNoKey, last = 0;
    logits.template each<4, kWavesOf>((int)((int64_t)logits.segments * slice / a.slices),
                            (int)((int64_t)logits.segments * (slice + 1) / a.slices),
                            [&](const auto& x, int, int segment) {
        uint32_t least = kNoKey;
#pragma unroll
        for (int i = 0; i < Row<BF16>::N; ++i) {
            const uint32_t key = key_of(x[i]);
            const bool there = x[i] != -INFINITY;
            least = min(least, there ? key : kNoKey);
            last = max(last, there ? key : 0u);
        }
        least = wave_min_xor(least);
        if (lane == 0) sp.firsts[segment] = least;
        first = min(first, least);
    });
    last = ~wave_min_xor(~last);
    if (lane == 0) waves[threadIdx.x >> 6] = make_uint2(first, last);
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < kWavesOf; ++w) first = min(first, waves[w].x), last = max(last, waves[w].y);
        sp.ends[slice] = make_uint2(first, last);
    }
}

// The bin that holds the target'th of `counts` (kBins - 1 where there are fewer),
// by one wavefront.
__device__ __forceinline__ int bin_reaching(const uint32_t* counts, uint32_t target) {
    const int lane = threadIdx.x & 63;
    uint32_t n = 0;
    for (int i = 0; i < 32; ++i) n += counts[32 * lane + (i + lane) % 32];
    uint32_t at = n;
    for (int x = 1; x < 64; x <<= 1) {
        const uint32_t o = __shfl_up(at, x);
        if (lane >= x) at += o;
    }
    const uint64_t there = __ballot(at >= target);
    if (!there) return kBins - 1;
    const int l = __ffsll((unsigned long long)there) - 1;
    uint32_t c = lane < 32 ? counts[32 * l + lane] : 0;
    for (int x = 1; x < 32; x <<= 1) {
        const uint32_t o = __shfl_up(c, x);
        if (lane >= x) c += o;
    }
    const uint32_t before = __shfl(at - n, l);
    return 32 * l + __ffsll((unsigned long long)__ballot(lane < 32 && before + c >= target)) - 1;
}

// Segments that are looked at, in any order.
struct Wanted {
    int n;
    uint16_t at[kMaxVocab / 256 + 1];

    // Those of s0 .. s1 - 1 that begin at bin `far` or ahead of it; n is 0 before.
    __device__ __forceinline__ void fill(const RowSpace& sp, const Bins& bins, int s0, int s1, int far) {
        for (int i = s0 + (int)threadIdx.x; i < s1; i += kThreads) {
            const uint32_t key = sp.firsts[i];
            if (key != kNoKey && bins.of(key_value(key)) <= far) at[atomicAdd(&n, 1)] = (uint16_t)i;
        }
    }
    // f(values, the lane's first id), as Row::each, of segments where some lane's
    // access has ok(value).
    template <int AHEAD, bool BF16, typename Ok, typename F>
    __device__ __forceinline__ void each(const Row<BF16>& logits, Ok ok, F f) const {
        for (int i = threadIdx.x >> 6; i < n; i += kWavesOf * AHEAD) {
            u32x4_t raw[AHEAD];
            int segment[AHEAD];
#pragma unroll
            for (int k = 0; k < AHEAD; ++k)
                if (i + k * kWavesOf < n) {
                    segment[k] = __builtin_amdgcn_readfirstlane(at[i + k * kWavesOf]);
                    raw[k] = logits.load(segment[k]);
                }
#pragma unroll
            for (int k = 0; k < AHEAD; ++k) {
                if (i + k * kWavesOf >= n) break;
                bool some = !logits.whole(segment[k]);
#pragma unroll
                for (int e = 0; e < Row<BF16>::N; ++e) some |= ok(Row<BF16>::raw_value(raw[k], e));
                if (!__any(some)) continue;
                float x[Row<BF16>::N];
                logits.values(segment[k], raw[k], x);
                f(x, logits.first(segment[k]));
            }
        }
    }
};

template <bool BF16>
__global__ __launch_bounds__(kThreads, 8) void sample_bins_kernel(SampleArgs a) {
    __shared__ uint64_t sums[kBins];
    __shared__ uint32_t counts[kBins];
    __shared__ Powers powers;
    __shared__ int reach;
    __shared__ Wanted wanted;
    const int row = (int)(blockIdx.x / (uint32_t)a.slices), slice = (int)(blockIdx.x % (uint32_t)a.slices);
    const RowSpace sp = row_space(a, row);
    const RowRule q = *sp.rule;
    const uint2 ends = ends_of(sp, a.slices);
    if (q.request < 0 || q.greedy || ends.x == kNoKey) return;
    const Bins bins = bins_of(ends, q);
    const Row<BF16> logits(a, row);
    fill(powers);
    for (int i = threadIdx.x; i < kBins; i += kThreads) sums[i] = 0, counts[i] = 0;
    if (threadIdx.x == 0) wanted.n = 0;
    __syncthreads();
    // Segments that begin behind bin `far` have nothing that counts.
    int far = kBins;
    if (q.top_k && q.top_k < logits.segments) {
        // The k first of the segments' first tokens are k tokens: the k-th of all
        // is not behind them.
        for (int i = threadIdx.x; i < logits.segments; i += kThreads) {
            const uint32_t key = sp.firsts[i];
            if (key != kNoKey) atomicAdd(&counts[bins.of(key_value(key))], 1u);
        }
        __syncthreads();
        if (threadIdx.x < 64) {
            const int b = bin_reaching(counts, (uint32_t)q.top_k);
            if (threadIdx.x == 0) reach = b;
        }
        __syncthreads();
        far = reach;
        for (int i = threadIdx.x; i < kBins; i += kThreads) counts[i] = 0;
        __syncthreads();
    } else if (q.min_p > 0.0 && !q.top_k && q.top_p == 1.0) {
        far = weak_bin(bins, q) + 1;
    }
    wanted.fill(sp, bins, (int)((int64_t)logits.segments * slice / a.slices),
                (int)((int64_t)logits.segments * (slice + 1) / a.slices), far);
    __syncthreads();
    wanted.template each<BF16 ? 1 : 2>(logits, [](float) { return true; }, [&](const auto& x, int) {
        // Four weights side by side.
#pragma unroll
        for (int h = 0; h < Row<BF16>::N; h += 4) {
            uint64_t w[4];
            int b[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = weight_of(x[h + i], bins.top, q.per, powers);
#pragma unroll
            for (int i = 0; i < 4; ++i) b[i] = bins.of(x[h + i]);
            if (q.top_k)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (x[h + i] != -INFINITY) atomicAdd(&counts[b[i]], 1u);
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (w[i]) atomicAdd((unsigned long long*)&sums[b[i]], (unsigned long long)w[i]);
        }
    });
    __syncthreads();
    for (int i = threadIdx.x; i < kBins; i += kThreads) {
        if (a.slices == 1) {
            sp.sums[i] = sums[i], sp.counts[i] = counts[i];
        } else {
            if (sums[i]) atomicAdd((unsigned long long*)&sp.sums[i], (unsigned long long)sums[i]);
            if (counts[i]) atomicAdd(&sp.counts[i], counts[i]);
        }
    }
}

// Cumulative bins of a row.
struct Cumulative {
    uint64_t sums[kBins + 1];  // [b]: of the bins below b
    uint32_t counts[kBins + 1];
    uint64_t wave_sums[4];
    uint32_t wave_counts[4];

    // By the workgroup's first four wavefronts, from what fetch() has read.
    static constexpr int PER = kBins / 256;
    struct Part {
        uint64_t s[PER];
        uint32_t n[PER];
    };
    static __device__ __forceinline__ Part fetch(const RowSpace& sp) {
        Part f = {};
        if (threadIdx.x < 256) {
#pragma unroll
            for (int i = 0; i < PER; ++i) f.s[i] = sp.sums[threadIdx.x * PER + i];
#pragma unroll
            for (int i = 0; i < PER; ++i) f.n[i] = sp.counts[threadIdx.x * PER + i];
        }
        return f;
    }
    __device__ __forceinline__ void load(const Part& f) {
        const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
        uint64_t w = 0, w_at = 0;
        uint32_t c = 0, c_at = 0;
        if (tid < 256) {
#pragma unroll
            for (int i = 0; i < PER; ++i) w += f.s[i], c += f.n[i];
            w_at = w, c_at = c;
            for (int x = 1; x < 64; x <<= 1) {
                const uint64_t ow = __shfl_up((unsigned long long)w_at, x);
                const uint32_t oc = __shfl_up(c_at, x);
                if (lane >= x) w_at += ow, c_at += oc;
            }
            if (lane == 63) wave_sums[wave] = w_at, wave_counts[wave] = c_at;
        }
        __syncthreads();
        if (tid < 256) {
            w_at -= w, c_at -= c;
            for (int v = 0; v < wave; ++v) w_at += wave_sums[v], c_at += wave_counts[v];
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                sums[tid * PER + i] = w_at, counts[tid * PER + i] = c_at;
                w_at += f.s[i], c_at += f.n[i];
            }
            if (tid == 255) sums[kBins] = w_at, counts[kBins] = c_at;
        }
        __syncthreads();
    }
    // The first bin whose tokens reach the target (kBins: none does), by each
    // wavefront: lane l looks at the end of 32 bins, then at one of these.
    template <typename T>
    static __device__ __forceinline__ int reach(const T* below, T target) {
        const int lane = threadIdx.x & 63;
        uint64_t there = __ballot(below[32 * lane + 32] >= target);
        if (!there) return kBins;
        const int b = 32 * (__ffsll((unsigned long long)there) - 1);
        there = __ballot(below[b + (lane & 31) + 1] >= target);
        return b + __ffsll((unsigned long long)there) - 1;
    }
};

__device__ __forceinline__ Ranges ranges_of(const Cumulative& c, const Bins& bins, const RowRule& q) {
    typedef Cumulative C;
    Ranges g;
#pragma unroll
    for (int i = 0; i < 4; ++i) g.lo[i] = kBins, g.hi[i] = -1;
    // The kept tokens' sum lies in [least, most].
    const uint64_t one = (uint64_t)kOne;
    uint64_t least = c.sums[kBins], most = least;
    if (q.top_k && (uint32_t)q.top_k < c.counts[kBins]) {
        const int b = C::reach(c.counts, (uint32_t)q.top_k);
        most = least = c.sums[b + 1];
        if (c.counts[b + 1] != (uint32_t)q.top_k && c.sums[b] != c.sums[b + 1]) {
            g.lo[0] = g.hi[0] = b;
            least = max(c.sums[b], one);
        }
    }
    g.all = most;
    if (q.top_p < 1.0) {
        const uint64_t t0 = cut_at(q.top_p, least), t1 = cut_at(q.top_p, most);
        g.lo[1] = C::reach(c.sums, t0), g.hi[1] = C::reach(c.sums, t1);
        least = max(t0, c.sums[g.lo[1]]);
        most = min(most, c.sums[g.hi[1] + 1]);
    }
    g.strong = kBins, g.sure = 0, g.pad = 0;
    if (q.min_p > 0.0) {
        // A bin to either side for the rounding of weights, logarithm and bins.
        const int b = weak_bin(bins, q);
        const int low = max(b - 1, 0), high = min(b + 1, kBins - 1);
        if (c.sums[low] < most) {
            g.lo[2] = low, g.hi[2] = high, g.strong = low, g.sure = c.sums[low];
            least = min(least, max(c.sums[low], one));
            most = min(most, c.sums[high + 1]);
        }
    }
    g.lo[3] = C::reach(c.sums, draw_at(q.uniform, least));
    g.hi[3] = C::reach(c.sums, draw_at(q.uniform, most));
    return g;
}

template <bool BF16>
__global__ __launch_bounds__(kThreads, 8) void sample_list_kernel(SampleArgs a) {
    __shared__ Cumulative sums;
    __shared__ Ranges ranges;
    __shared__ Wanted wanted;
    const int row = (int)(blockIdx.x / (uint32_t)a.slices), slice = (int)(blockIdx.x % (uint32_t)a.slices);
    const RowSpace sp = row_space(a, row);
    const Cumulative::Part part = Cumulative::fetch(sp);
    const RowRule q = *sp.rule;
    const uint2 ends = ends_of(sp, a.slices);
    if (q.request < 0 || q.greedy || ends.x == kNoKey) return;
    const Row<BF16> logits(a, row);
    const Bins bins = bins_of(ends, q);
    if (threadIdx.x == 0) wanted.n = 0;
    sums.load(part);
    if (threadIdx.x < 64) {
        const Ranges g = ranges_of(sums, bins, q);
        if (threadIdx.x == 0) {
            ranges = g;
            if (slice == 0) *sp.ranges = g;
        }
    }
    __syncthreads();
    const Ranges g = ranges;
    wanted.fill(sp, bins, (int)((int64_t)logits.segments * slice / a.slices),
                (int)((int64_t)logits.segments * (slice + 1) / a.slices), g.last());
    __syncthreads();
    // Distances that can be in one of the ranges; infinity's, which counts as the
    // largest, is -infinity here.
    const float near = g.first() > 0 ? (float)g.first() : -INFINITY, far = (float)(g.last() + 1);
    auto ok = [&](float x) {
        const float d = bins.distance(x);
        return d >= near && (d < far || far == (float)kBins);
    };
    wanted.template each<BF16 ? 2 : 4>(logits, ok, [&](const auto& x, int first) {
#pragma unroll
        for (int e = 0; e < Row<BF16>::N; ++e) {
            const int bin = bins.of(x[e]);
            if (x[e] == -INFINITY || !g.has(bin)) continue;
            const uint32_t at = atomicAdd(sp.listed, 1u);
            if (at < kList)
                sp.list[at] = place_of(x[e], first + e), sp.below[at] = sums.sums[bin],
                sp.ahead[at] = sums.counts[bin];
        }
    });
}

struct Listed {
    uint64_t place;  // the bin in its upper 12 bits
    uint64_t weight;
};

template <bool BF16>
__global__ __launch_bounds__(kPickThreads) void sample_pick_kernel(SampleArgs a) {
    __shared__ union Space {
        struct {
            Listed list[kList];
            uint64_t sums[kList];
            uint32_t counts[kList];
        } p;
        Digits digits;
    } s;
    __shared__ Powers powers;
    const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 63;
    const RowSpace sp = row_space(a, row);
    const uint32_t listed = *sp.listed;
    const RowRule q = *sp.rule;
    const Ranges g = *sp.ranges;
    const uint2 ends = ends_of(sp, a.slices);
    fill(powers);
    if (q.request < 0) return;
    if (ends.x == kNoKey) {
        if (tid == 0) {
            a.tokens[row] = -1;
            if (a.probabilities) a.probabilities[row] = 0.0f;
        }
        return;
    }
    const Row<BF16> logits(a, row);
    if (q.greedy) {
        // The first segment that begins with the row's first key.
        uint64_t at = ~0ull;
        for (int i = tid; i < logits.segments; i += kPickThreads)
            if (sp.firsts[i] == ends.x) at = min(at, (uint64_t)i);
        at = least_of(at, s.digits.wave_sums);
        if (tid >= 64) return;
        float x[Row<BF16>::N];
        logits.values((int)at, logits.load((int)at), x);
        uint32_t id = 0xFFFFFFFFu;
#pragma unroll
        for (int i = Row<BF16>::N - 1; i >= 0; --i)
            if (key_of(x[i]) == ends.x && x[i] != -INFINITY) id = (uint32_t)(logits.first((int)at) + i);
        id = wave_min_xor(id);
        if (tid == 0) {
            a.tokens[row] = (int)id;
            if (a.probabilities) a.probabilities[row] = 1.0f;
        }
        return;
    }
    const Bins bins = bins_of(ends, q);
    __syncthreads();
    if (listed > kList) {
        pick_by_digits<BF16>(a, row, q, bins.top, powers, s.digits);
        return;
    }
    const int n = (int)listed;
    for (int t = tid; t < n; t += kPickThreads) {
        const uint64_t place = sp.list[t];
        const float x = place_value(place);
        s.p.list[t] = Listed{(uint64_t)bins.of(x) << 52 | place, weight_of(x, bins.top, q.per, powers)};
    }
    __syncthreads();
    // The listed token's cumulative weight and number: its bin's tokens up to it
    // are those at most its place in the bin below it.
    for (int t = tid; t < n; t += kPickThreads) {
        uint64_t sum = sp.below[t];
        uint32_t count = sp.ahead[t];
        const uint64_t mine = s.p.list[t].place, reach = mine & ((uint64_t(1) << 52) - 1);
#pragma unroll 8
        for (int i = 0; i < n; ++i) {
            const Listed other = s.p.list[i];
            const bool in = mine - other.place <= reach;
            sum += in ? other.weight : 0;
            count += in;
        }
        s.p.sums[t] = sum, s.p.counts[t] = count;
    }
    __syncthreads();
    // The rest by one wavefront, without barriers.
    if (tid >= 64) return;
    const uint64_t none = ~0ull;
    auto reaches = [&](uint64_t target) {  // the least sum of at least that
        uint64_t v = none;
        for (int i = lane; i < n; i += 64) v = s.p.sums[i] >= target ? min(v, s.p.sums[i]) : v;
        return wave_least(v);
    };
    uint64_t kept = g.all;
    if (g.lo[0] <= g.hi[0]) {
        uint64_t v = none;
        for (int i = lane; i < n; i += 64) v = s.p.counts[i] == (uint32_t)q.top_k ? s.p.sums[i] : v;
        kept = wave_least(v);
    }
    if (q.top_p < 1.0) kept = min(kept, reaches(cut_at(q.top_p, kept)));
    if (g.strong < kBins) {
        const uint64_t least = least_weight(q);
        uint64_t v = 0;
        for (int i = lane; i < n; i += 64) {
            const Listed l = s.p.list[i];
            const int bin = (int)(l.place >> 52);
            v += bin >= g.lo[2] && bin <= g.hi[2] && l.weight >= least ? l.weight : 0;
        }
        kept = min(kept, g.sure + wave_total(v));
    }
    const uint64_t drawn = reaches(draw_at(q.uniform, kept));
    for (int i = lane; i < n; i += 64) {
        const Listed l = s.p.list[i];
        // One token of a weight has this sum.
        if (s.p.sums[i] == drawn && l.weight)
            put_token(a, row, l.place & ((uint64_t(1) << 52) - 1), l.weight, kept);
    }
}

// How many slices a row is cut into: up to 256 workgroups in all as long as a
// slice has 8192 logits, up to 512 as long as it has 16384; at most one per lane
// of ends_of. In a graph, top-k 64 and top-p 0.95: one row of 128256 20.6 us, 22.1 in
// slices of 16384; 24 rows 25.7, 29.4 in slices of 8192 up to 512 workgroups; 150 rows
// of 151936 48.9, 54.9 with up to 256 workgroups, 61.5 with up to 1024. Without rules
// one row 19.4, 23.0; 150 rows 83, 124 and 85.
constexpr int64_t kMaxSlices = 64;
int64_t slices_of(int64_t rows, int64_t vocab) {
    rows = std::max<int64_t>(rows, 1);
    const int64_t fine = std::min((vocab + 8191) / 8192, 256 / rows);
    const int64_t coarse = std::min((vocab + 16383) / 16384, 512 / rows);
    return std::clamp<int64_t>(std::max(fine, coarse), 1, kMaxSlices);
}
int64_t row_bytes_of(int64_t slices, int64_t vocab) {
    const int64_t segments = vocab / 256 + 2;
    return (sizeof(RowRule) + sizeof(Ranges) + kBins * 12 + kList * 20 + slices * 8 + (segments + 1) * 4 + 15) / 16 * 16;
}

template <bool BF16>
hipError_t launch_sample(const SampleArgs& a, hipStream_t st) {
    const uint32_t blocks = (uint32_t)((int64_t)a.rows * a.slices);
    sample_first_kernel<BF16><<<blocks, kThreads, 0, st>>>(a);
    sample_bins_kernel<BF16><<<blocks, kThreads, 0, st>>>(a);
    sample_list_kernel<BF16><<<blocks, kThreads, 0, st>>>(a);
    sample_pick_kernel<BF16><<<(uint32_t)a.rows, kPickThreads, 0, st>>>(a);
    return hipGetLastError();
}

}  // namespace
}  // namespace ncm

extern "C" int ncm_sample_workspace(int64_t rows, int64_t vocab, size_t* bytes) {
    using namespace ncm;
    if (!bytes) return NCM_E_NULL;
    *bytes = 0;
    if (rows < 0 || rows >= kMaxBlocks / 4 || vocab < 0 || vocab > kMaxVocab) return NCM_E_SHAPE;
    if (rows > 0) *bytes = (size_t)rows * row_bytes_of(slices_of(rows, vocab), vocab);
    return NCM_OK;
}

extern "C" int ncm_sample_dev(ncm_ctx_t* ctx, const ncm_sample_rules_t* rules, const void* logits,
                              int64_t rows, int64_t vocab, int64_t stride, int dtype,
                              const void* uniform, int uniform_bits, int32_t* tokens,
                              float* probabilities, void* workspace, size_t workspace_bytes) {
    using namespace ncm;
    if (!ctx || !rules) return NCM_E_NULL;
    size_t need;
    int rc = ncm_sample_workspace(rows, vocab, &need);
    if (rc) return rc;
    if (stride < vocab || stride > (int64_t(1) << 40) || rules->requests < 0 ||
        (rules->offsets ? rules->requests > kMaxRequests : rules->requests != rows))
        return NCM_E_SHAPE;
    if ((dtype != NCM_OUT_F32 && dtype != NCM_OUT_BF16) || (uniform_bits != 32 && uniform_bits != 64))
        return NCM_E_ARG;
    if (rows == 0 || rules->requests == 0) return NCM_OK;
    if ((!logits && vocab > 0) || !uniform || !tokens || (need && !workspace)) return NCM_E_NULL;
    if (workspace_bytes < need) return NCM_E_LENGTH;
    const int size = dtype == NCM_OUT_BF16 ? 2 : 4;
    if ((uintptr_t)logits % size || (uintptr_t)uniform % (uniform_bits / 8) ||
        (need && (uintptr_t)workspace % 16))
        return NCM_E_ARG;
    const int64_t slices = slices_of(rows, vocab);
    const SampleArgs a = {*rules, logits, uniform, tokens, probabilities, stride, (int)rows, (int)vocab,
                          uniform_bits == 64, (char*)workspace, row_bytes_of(slices, vocab), (int)slices};
    const DeviceScope scope(ncm_ctx_device(ctx));
    rc = step_hip(scope.error(), "sample device");
    if (rc) return rc;
    const hipStream_t st = ncm_ctx_stream(ctx);
    return step_hip(dtype == NCM_OUT_BF16 ? launch_sample<true>(a, st) : launch_sample<false>(a, st),
                    "sample launch");
}
