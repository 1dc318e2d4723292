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
// stand is found from sums over 2048 bins of 1/64 of (max - x) / T, the last of
// them for what is too far below to have a weight:
//   1. the first token of each slice of a row;
//   2. weights (and numbers, for top-k) of its bins, in LDS, then added to the
//      row's in memory;
//   3. the bins that a cut or the draw can fall into, from the row's bins, and
//      their tokens into a list;
//   4. each listed token's cumulative weight, exactly, from its bin's and the
//      listed tokens of its bin; cuts and draw are minima over these.
// A row whose list would be longer than 1024 (many equal logits, a temperature
// that puts thousands of tokens into a bin) is done digit by digit of the
// token's 52-bit place in the order (32 bits of the logit, 20 of the id): sums of
// the tokens by their next digit, then the digit where the target is passed.
#include "step.h"

namespace ncm {
namespace {

constexpr double kOne = 0x1p43;  // the largest weight
constexpr int64_t kMaxVocab = int64_t(1) << 20;
constexpr int kThreads = 1024, kWavesOf = kThreads / 64;
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
    float bins;      // 64 / T: bins a unit of logit
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
    uint64_t* list;     // [kList]: places
    uint64_t* below;    // [kList]: the sum of the bins below the place's
    uint32_t* ahead;    // [kList]: their number
    Ranges* ranges;
    uint64_t* firsts;   // [slices]: each slice's first place
    uint32_t* counts;   // [kBins]
    uint32_t* listed;   // places there are for the list
};

__device__ __forceinline__ RowSpace row_space(const SampleArgs& a, int row) {
    char* p = a.space + row * a.row_bytes;
    RowSpace r;
    r.rule = (RowRule*)p;
    r.sums = (uint64_t*)(p + sizeof(RowRule));
    r.list = r.sums + kBins;
    r.below = r.list + kList;
    r.firsts = r.below + kList;
    r.ranges = (Ranges*)(r.firsts + a.slices);
    r.counts = (uint32_t*)(r.ranges + 1);
    r.ahead = r.counts + kBins;
    r.listed = r.ahead + kList;
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
    q.bins = 64.0f / fmaxf(t, 0x1p-96f);
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
// Ascending in the order.
__device__ __forceinline__ uint64_t place_of(float x, int id) {
    const uint32_t b = __float_as_uint(x);
    const uint32_t up = b & 0x80000000u ? ~b : b | 0x80000000u;
    return ((uint64_t)~up << 20) | (uint32_t)id;
}
constexpr uint64_t kNowhere = (uint64_t)0xFFFFFFFFu << 20;  // above every place: NaN's bits
__device__ __forceinline__ float place_value(uint64_t p) {
    const uint32_t up = ~(uint32_t)(p >> 20);
    return __uint_as_float(up & 0x80000000u ? up & 0x7FFFFFFFu : ~up);
}
__device__ __forceinline__ int place_id(uint64_t p) { return (int)(p & 0xFFFFFu); }

// 2^(j / 32), in LDS.
typedef double Powers[32];
__device__ __forceinline__ void fill(Powers& powers) {
    if (threadIdx.x < 32) powers[threadIdx.x] = exp2((double)threadIdx.x / 32.0);
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

// floor(f * total) and whether it is more than that; f in [0, 1].
__device__ __forceinline__ uint64_t share_of(double f, uint64_t total, bool& more) {
    const uint64_t m = (uint64_t)(f * 0x1p53);  // f < 1 has no bit behind but below 2^-53
    const uint64_t lo = m * total, hi = __umul64hi(m, total);
    more = (lo & ((uint64_t(1) << 53) - 1)) != 0 || (double)m != f * 0x1p53;
    return (hi << 11) | (lo >> 53);
}

template <bool BF16>
__device__ __forceinline__ float load_logit(const SampleArgs& a, int row, int i) {
    const int64_t at = (int64_t)row * a.stride + i;
    const float x = BF16 ? __uint_as_float((uint32_t)((const uint16_t*)a.logits)[at] << 16)
                         : ((const float*)a.logits)[at];
    return value_of(x);
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

// Accesses ahead: 16 logits.
template <bool BF16>
constexpr int kAhead = BF16 ? 2 : 4;

// The logits of a slice of a row, N of a 16-byte access at a time: f(values, id
// of the first); values that are not the row's are -infinity.
template <bool BF16, int AHEAD, typename F>
__device__ __forceinline__ void each_logit(const SampleArgs& a, int row, int slice, int slices, F f) {
    constexpr int SIZE = BF16 ? 2 : 4, N = 16 / SIZE;
    const char* base = (const char*)a.logits + (int64_t)row * a.stride * SIZE;
    const int skip = (int)((uintptr_t)base % 16) / SIZE;  // values ahead of the row in its first access
    const int vectors = (a.vocab + skip + N - 1) / N;
    const int v0 = (int)((int64_t)vectors * slice / slices);
    const int v1 = (int)((int64_t)vectors * (slice + 1) / slices);
    for (int v = v0 + (int)threadIdx.x; v < v1; v += kThreads * AHEAD) {
        u32x4_t raw[AHEAD];
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) {
            const int at = v + k * kThreads, first = at * N - skip;
            if (at < v1 && first >= 0 && first + N <= a.vocab)
                raw[k] = *(const u32x4_t*)(base + (int64_t)first * SIZE);
        }
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) {
            const int at = v + k * kThreads, first = at * N - skip;
            if (at >= v1) break;
            float x[N];
            if (first >= 0 && first + N <= a.vocab) {
#pragma unroll
                for (int i = 0; i < N; ++i)
                    x[i] = value_of(BF16 ? __uint_as_float(i % 2 ? raw[k][i / 2] & 0xFFFF0000u
                                                                 : raw[k][i / 2] << 16)
                                         : __uint_as_float(raw[k][BF16 ? 0 : i]));
            } else {
#pragma unroll
                for (int i = 0; i < N; ++i)
                    x[i] = first + i >= 0 && first + i < a.vocab ? load_logit<BF16>(a, row, first + i)
                                                                 : -INFINITY;
            }
            f(x, first);
        }
    }
}

// Sums and numbers by a place's next digit.
struct Digits {
    uint64_t sums[2048];
    uint32_t counts[2048];
    uint64_t wave_sums[kWavesOf];
    uint64_t wave_counts[kWavesOf];
    uint64_t place, sum, count;
    int found;
};

// The first place whose cumulative weight (COUNT: number) is at least `target`;
// sum: the cumulative weight there. False where all together is less.
template <bool BF16, bool COUNT>
__device__ bool find_place(const SampleArgs& a, int row, float top, const RowRule& q,
                           const Powers& powers, uint64_t target, Digits& s, uint64_t& place,
                           uint64_t& sum) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    uint64_t prefix = 0, done_sum = 0, done_count = 0;
    int low = 52;  // digits above it are fixed
    while (low > 0) {
        const int bits = low > 30 ? 11 : 10, next = low - bits;
        __syncthreads();
        for (int i = tid; i < 2048; i += kThreads) s.sums[i] = 0, s.counts[i] = 0;
        if (tid == 0) s.found = 0;
        __syncthreads();
        each_logit<BF16, kAhead<BF16>>(a, row, 0, 1, [&](const auto& x, int first) {
            constexpr int N = sizeof(x) / sizeof(float);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const uint64_t p = place_of(x[i], first + i);
                if (x[i] == -INFINITY || (p >> low) != prefix) continue;
                const int digit = (int)((p >> next) & ((1 << bits) - 1));
                atomicAdd(&s.counts[digit], 1u);
                const uint64_t w = weight_of(x[i], top, q.per, powers);
                if (w) atomicAdd((unsigned long long*)&s.sums[digit], (unsigned long long)w);
            }
        });
        __syncthreads();
        const uint64_t c0 = s.counts[2 * tid], c1 = s.counts[2 * tid + 1];
        const uint64_t s0 = s.sums[2 * tid], s1 = s.sums[2 * tid + 1];
        uint64_t c = c0 + c1, w = s0 + s1;
        for (int x = 1; x < 64; x <<= 1) {
            const uint64_t oc = __shfl_up((unsigned long long)c, x), ow = __shfl_up((unsigned long long)w, x);
            if (lane >= x) c += oc, w += ow;
        }
        if (lane == 63) s.wave_sums[wave] = w, s.wave_counts[wave] = c;
        __syncthreads();
        c += done_count, w += done_sum;
        for (int v = 0; v < wave; ++v) c += s.wave_counts[v], w += s.wave_sums[v];
        // Cumulative values ahead of, between and behind the thread's two digits.
        const uint64_t c_at = c - c0 - c1, w_at = w - s0 - s1;
        const uint64_t before = COUNT ? c_at : w_at, mid = COUNT ? c_at + c0 : w_at + s0;
        if (before < target && target <= (COUNT ? c : w)) {
            const bool second = mid < target;
            s.found = 1;
            s.place = (prefix << bits) | (uint64_t)(2 * tid + second);
            s.sum = second ? w_at + s0 : w_at;
            s.count = second ? c_at + c0 : c_at;
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
__device__ __forceinline__ uint64_t least_of(uint64_t v, uint64_t (&waves)[kWavesOf]) {
    v = wave_least(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = v;
    __syncthreads();
    for (int w = 0; w < kWavesOf; ++w) v = min(v, waves[w]);
    return v;
}
__device__ __forceinline__ uint64_t total_of(uint64_t v, uint64_t (&waves)[kWavesOf]) {
    v = wave_total(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0;
    for (int w = 0; w < kWavesOf; ++w) v += waves[w];
    return v;
}

// The least weight that min_p keeps.
__device__ __forceinline__ uint64_t least_weight(const RowRule& q) {
    return max((uint64_t)ceil(q.min_p * kOne), (uint64_t)1);
}

// A row by its places' digits.
template <bool BF16>
__device__ __noinline__ void pick_by_digits(const SampleArgs& a, int row, const RowRule& q, float top,
                               const Powers& powers, Digits& s) {
    const uint64_t least = least_weight(q);
    uint64_t all = 0, strong = 0;  // all weights, and those of at least min_p
    each_logit<BF16, kAhead<BF16>>(a, row, 0, 1, [&](const auto& x, int) {
        constexpr int N = sizeof(x) / sizeof(float);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const uint64_t w = weight_of(x[i], top, q.per, powers);
            all += w;
            strong += w >= least ? w : 0;
        }
    });
    all = total_of(all, s.wave_sums);
    strong = total_of(strong, s.wave_counts);
    uint64_t place, sum;
    if (q.top_k && find_place<BF16, true>(a, row, top, q, powers, q.top_k, s, place, sum)) all = sum;
    uint64_t kept = all;
    if (q.top_p < 1.0 &&
        find_place<BF16, false>(a, row, top, q, powers, cut_at(q.top_p, all), s, place, sum))
        kept = min(kept, sum);
    kept = min(kept, strong);
    find_place<BF16, false>(a, row, top, q, powers, draw_at(q.uniform, kept), s, place, sum);
    if (threadIdx.x == 0)
        put_token(a, row, place, weight_of(place_value(place), top, q.per, powers), kept);
}

__device__ __forceinline__ int bin_of(float x, float top, const RowRule& q) {
    return (int)fminf((top - x) * q.bins, (float)(kBins - 1));
}

template <bool BF16>
__global__ __launch_bounds__(kThreads) void sample_first_kernel(SampleArgs a) {
    __shared__ uint64_t waves[kWavesOf];
    const int row = (int)(blockIdx.x / (uint32_t)a.slices), slice = (int)(blockIdx.x % (uint32_t)a.slices);
    const RowSpace sp = row_space(a, row);
    // What the row's next kernels start from.
    if (a.slices > 1)
        for (int i = slice * kThreads + (int)threadIdx.x; i < kBins; i += a.slices * kThreads)
            sp.sums[i] = 0, sp.counts[i] = 0;
    if (slice == 0 && threadIdx.x < 64) {
        const RowRule q = rule_of(a, row);
        if (threadIdx.x == 0) *sp.rule = q, *sp.listed = 0;
    }
    float top = -INFINITY;
    int id = 0x7FFFFFFF;
    each_logit<BF16, kAhead<BF16>>(a, row, slice, a.slices, [&](const auto& x, int first) {
        constexpr int N = sizeof(x) / sizeof(float);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            id = x[i] > top ? first + i : id;
            top = fmaxf(top, x[i]);
        }
    });
    const uint64_t place = least_of(top == -INFINITY ? kNowhere : place_of(top, id), waves);
    if (threadIdx.x == 0) sp.firsts[slice] = place;
}

// The row's first place, from its slices'.
__device__ __forceinline__ uint64_t first_of(const RowSpace& sp, int slices) {
    const int lane = threadIdx.x & 63;
    return wave_least(lane < slices ? sp.firsts[lane] : kNowhere);
}

template <bool BF16>
__global__ __launch_bounds__(kThreads, 8) void sample_bins_kernel(SampleArgs a) {
    __shared__ uint64_t sums[kBins];
    __shared__ uint32_t counts[kBins];
    __shared__ Powers powers;
    const int row = (int)(blockIdx.x / (uint32_t)a.slices), slice = (int)(blockIdx.x % (uint32_t)a.slices);
    const RowSpace sp = row_space(a, row);
    const RowRule q = *sp.rule;
    const uint64_t place = first_of(sp, a.slices);
    if (q.request < 0 || q.greedy || place == kNowhere) return;
    const float top = place_value(place);
    fill(powers);
    for (int i = threadIdx.x; i < kBins; i += kThreads) sums[i] = 0, counts[i] = 0;
    __syncthreads();
    each_logit<BF16, kAhead<BF16> / 2>(a, row, slice, a.slices, [&](const auto& x, int) {
        constexpr int N = sizeof(x) / sizeof(float);
        uint64_t w[N];
        int b[N];
#pragma unroll
        for (int i = 0; i < N; ++i) w[i] = weight_of(x[i], top, q.per, powers);
#pragma unroll
        for (int i = 0; i < N; ++i) b[i] = bin_of(x[i], top, q);
        if (q.top_k)
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (x[i] != -INFINITY) atomicAdd(&counts[b[i]], 1u);
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (w[i]) atomicAdd((unsigned long long*)&sums[b[i]], (unsigned long long)w[i]);
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

    // By the workgroup's first four wavefronts.
    __device__ __forceinline__ void load(const RowSpace& sp) {
        constexpr int PER = kBins / 256;
        const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
        uint64_t s[PER], w = 0, w_at = 0;
        uint32_t n[PER], c = 0, c_at = 0;
        if (tid < 256) {
#pragma unroll
            for (int i = 0; i < PER; ++i) s[i] = sp.sums[tid * PER + i];
#pragma unroll
            for (int i = 0; i < PER; ++i) n[i] = sp.counts[tid * PER + i];
#pragma unroll
            for (int i = 0; i < PER; ++i) w += s[i], c += n[i];
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
                w_at += s[i], c_at += n[i];
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

__device__ __forceinline__ Ranges ranges_of(const Cumulative& c, const RowRule& q) {
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
        // A bin to either side for the rounding of logarithm and bins.
        const int b = (int)fminf(-logf((float)q.min_p) * 64.0f, (float)kBins);
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
    __shared__ Cumulative bins;
    __shared__ Ranges ranges;
    const int row = (int)(blockIdx.x / (uint32_t)a.slices), slice = (int)(blockIdx.x % (uint32_t)a.slices);
    const RowSpace sp = row_space(a, row);
    const RowRule q = *sp.rule;
    const uint64_t first = first_of(sp, a.slices);
    if (q.request < 0 || q.greedy || first == kNowhere) return;
    const float top = place_value(first);
    bins.load(sp);
    if (threadIdx.x < 64) {
        const Ranges g = ranges_of(bins, q);
        if (threadIdx.x == 0) {
            ranges = g;
            if (slice == 0) *sp.ranges = g;
        }
    }
    __syncthreads();
    const Ranges g = ranges;
    each_logit<BF16, kAhead<BF16>>(a, row, slice, a.slices, [&](const auto& x, int id) {
        constexpr int N = sizeof(x) / sizeof(float);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int bin = bin_of(x[i], top, q);
            if (x[i] == -INFINITY || !g.has(bin)) continue;
            const uint32_t at = atomicAdd(sp.listed, 1u);
            if (at < kList)
                sp.list[at] = place_of(x[i], id + i), sp.below[at] = bins.sums[bin],
                sp.ahead[at] = bins.counts[bin];
        }
    });
}

struct Listed {
    uint64_t place;  // the bin in its upper 12 bits
    uint64_t weight;
};

template <bool BF16>
__global__ __launch_bounds__(kThreads) void sample_pick_kernel(SampleArgs a) {
    __shared__ union Space {
        struct {
            Listed list[kList];
            uint64_t sums[kList];
            uint32_t counts[kList];
        } p;
        Digits digits;
    } s;
    __shared__ Powers powers;
    const int row = blockIdx.x, tid = threadIdx.x;
    const RowSpace sp = row_space(a, row);
    const RowRule q = *sp.rule;
    const uint64_t first = first_of(sp, a.slices);
    const int n = (int)min(*sp.listed, (uint32_t)kList + 1);
    const Ranges g = *sp.ranges;
    if (q.request < 0) return;
    if (q.greedy || first == kNowhere) {
        if (tid == 0) {
            a.tokens[row] = first == kNowhere ? -1 : place_id(first);
            if (a.probabilities) a.probabilities[row] = first == kNowhere ? 0.0f : 1.0f;
        }
        return;
    }
    const float top = place_value(first);
    fill(powers);
    __syncthreads();
    if (n > kList) {
        pick_by_digits<BF16>(a, row, q, top, powers, s.digits);
        return;
    }
    uint64_t sum = 0, mine = 0;
    uint32_t count = 0;
    if (tid < n) {
        const uint64_t place = sp.list[tid];
        sum = sp.below[tid], count = sp.ahead[tid];
        const float x = place_value(place);
        mine = (uint64_t)bin_of(x, top, q) << 52 | place;
        s.p.list[tid] = Listed{mine, weight_of(x, top, q.per, powers)};
    }
    __syncthreads();
    // The listed token's cumulative weight and number: its bin's tokens up to it
    // are those at most its place in the bin below it.
    if (tid < n) {
        const uint64_t reach = mine & ((uint64_t(1) << 52) - 1);
#pragma unroll 8
        for (int i = 0; i < n; ++i) {
            const Listed other = s.p.list[i];
            const bool in = mine - other.place <= reach;
            sum += in ? other.weight : 0;
            count += in;
        }
        s.p.sums[tid] = sum, s.p.counts[tid] = count;
    }
    __syncthreads();
    // The rest by one wavefront, without barriers.
    if (tid >= 64) return;
    const uint64_t none = ~0ull;
    auto reaches = [&](uint64_t target) {  // the least sum of at least that
        uint64_t v = none;
        for (int i = tid; i < n; i += 64) v = s.p.sums[i] >= target ? min(v, s.p.sums[i]) : v;
        return wave_least(v);
    };
    uint64_t kept = g.all;
    if (g.lo[0] <= g.hi[0]) {
        uint64_t v = none;
        for (int i = tid; i < n; i += 64) v = s.p.counts[i] == (uint32_t)q.top_k ? s.p.sums[i] : v;
        kept = wave_least(v);
    }
    if (q.top_p < 1.0) kept = min(kept, reaches(cut_at(q.top_p, kept)));
    if (g.strong < kBins) {
        const uint64_t least = least_weight(q);
        uint64_t v = 0;
        for (int i = tid; i < n; i += 64) {
            const Listed l = s.p.list[i];
            const int bin = (int)(l.place >> 52);
            v += bin >= g.lo[2] && bin <= g.hi[2] && l.weight >= least ? l.weight : 0;
        }
        kept = min(kept, g.sure + wave_total(v));
    }
    const uint64_t drawn = reaches(draw_at(q.uniform, kept));
    for (int i = tid; i < n; i += 64) {
        const Listed l = s.p.list[i];
        // One token of a weight has this sum.
        if (s.p.sums[i] == drawn && l.weight)
            put_token(a, row, l.place & ((uint64_t(1) << 52) - 1), l.weight, kept);
    }
}

// How many slices a row is cut into: 512 workgroups in all where that leaves a
// slice 16384 logits.
int64_t slices_of(int64_t rows, int64_t vocab) {
    return std::max<int64_t>(1, std::min<int64_t>((vocab + 16383) / 16384, 512 / std::max<int64_t>(rows, 1)));
}
static_assert(kMaxVocab / 16384 <= 64, "first_of has a lane per slice");
int64_t row_bytes_of(int64_t slices) {
    return (sizeof(RowRule) + sizeof(Ranges) + kBins * 12 + kList * 20 + slices * 8 + 4 + 15) / 16 * 16;
}

template <bool BF16>
hipError_t launch_sample(const SampleArgs& a, hipStream_t st) {
    const uint32_t blocks = (uint32_t)((int64_t)a.rows * a.slices);
    sample_first_kernel<BF16><<<blocks, kThreads, 0, st>>>(a);
    sample_bins_kernel<BF16><<<blocks, kThreads, 0, st>>>(a);
    sample_list_kernel<BF16><<<blocks, kThreads, 0, st>>>(a);
    sample_pick_kernel<BF16><<<(uint32_t)a.rows, kThreads, 0, st>>>(a);
    return hipGetLastError();
}

}  // namespace
}  // namespace ncm

extern "C" int ncm_sample_workspace(int64_t rows, int64_t vocab, size_t* bytes) {
    using namespace ncm;
    if (!bytes) return NCM_E_NULL;
    *bytes = 0;
    if (rows < 0 || rows >= kMaxBlocks / 4 || vocab < 0 || vocab > kMaxVocab) return NCM_E_SHAPE;
    if (rows > 0) *bytes = (size_t)rows * row_bytes_of(slices_of(rows, vocab));
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
                          uniform_bits == 64, (char*)workspace, row_bytes_of(slices), (int)slices};
    const DeviceScope scope(ncm_ctx_device(ctx));
    rc = step_hip(scope.error(), "sample device");
    if (rc) return rc;
    const hipStream_t st = ncm_ctx_stream(ctx);
    return step_hip(dtype == NCM_OUT_BF16 ? launch_sample<true>(a, st) : launch_sample<false>(a, st),
                    "sample launch");
}
