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
constexpr int kDigits = 2048;

struct SampleArgs {
    ncm_sample_rules_t rules;
    const void* logits;
    const void* uniform;
    int32_t* tokens;
    float* probabilities;
    int64_t stride;
    int rows, vocab;
    bool wide_uniform;
};

// What a row is drawn by.
struct RowRule {
    bool greedy;
    double per;      // log2(e) / T
    float bins;      // 64 / T: bins a unit of logit
    int top_k;       // 0: off
    double top_p;    // 1: off
    double min_p;    // 0: off
    double uniform;
};

__device__ __forceinline__ int request_row(const ncm_sample_rules_t& u, int row) {
    if (!u.offsets) return row;
    int lo = 0, hi = (int)u.requests;  // the first request that ends behind the row
    while (lo < hi) {
        const int mid = (lo + hi) / 2;
        if (u.offsets[mid + 1] > row) hi = mid;
        else lo = mid + 1;
    }
    return lo < u.requests && u.offsets[lo] <= row ? lo : -1;
}

__device__ __forceinline__ RowRule rule_of(const SampleArgs& a, int r, int row) {
    const ncm_sample_rules_t& u = a.rules;
    RowRule q;
    const float t = u.temperature ? u.temperature[r] : 1.0f;
    q.greedy = !(t > 0.0f);
    q.per = 1.44269504088896340736 / (double)fmaxf(t, 0x1p-96f);
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

// rint(2^43 exp((x - top) / T)), per = log2(e) / T: 2^f of the exponent's part
// from 1/2 below to 1/2 above an integer by its Taylor polynomial of degree 11,
// good to (ln 2 / 2)^12 / 12! = 2^-47.
__device__ __forceinline__ uint64_t weight_of(float x, float top, double per) {
    const double y = ((double)x - (double)top) * per;
    if (!(y > -45.0)) return 0;
    const double n = rint(y), r = (y - n) * 0.693147180559945309417;
    double p = 1.0 / 39916800.0;
    p = fma(p, r, 1.0 / 3628800.0);
    p = fma(p, r, 1.0 / 362880.0);
    p = fma(p, r, 1.0 / 40320.0);
    p = fma(p, r, 1.0 / 5040.0);
    p = fma(p, r, 1.0 / 720.0);
    p = fma(p, r, 1.0 / 120.0);
    p = fma(p, r, 1.0 / 24.0);
    p = fma(p, r, 1.0 / 6.0);
    p = fma(p, r, 0.5);
    p = fma(p, r, 1.0);
    p = fma(p, r, 1.0);
    // times 2^(n + 43), and 2^52 for the rounding: the integer is in the low bits.
    const double scale = __longlong_as_double((long long)((int)n + 43 + 1023) << 52);
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

__device__ __forceinline__ void put_token(const SampleArgs& a, int row, uint64_t place, float top,
                                          const RowRule& q, uint64_t kept) {
    a.tokens[row] = place_id(place);
    if (a.probabilities)
        a.probabilities[row] =
            (float)((double)weight_of(place_value(place), top, q.per) / (double)kept);
}

// A workgroup's view of a row, and what it finds there.
struct Shared {
    uint64_t sums[kDigits];
    uint32_t counts[kDigits];
    uint64_t wave_sums[16];
    uint64_t wave_counts[16];
    uint64_t place, sum;
    uint64_t count;
    int found;
};

// The first place whose cumulative weight (COUNT: number) is at least `target`;
// sum: the cumulative weight there. False where all together is less.
template <bool BF16, bool COUNT>
__device__ bool find_place(const SampleArgs& a, int row, float top, double per, uint64_t target,
                           Shared& s, uint64_t& place, uint64_t& sum) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    uint64_t prefix = 0, done_sum = 0, done_count = 0;
    int low = 52;  // digits above it are fixed
    while (low > 0) {
        const int bits = low > 30 ? 11 : 10, next = low - bits;
        __syncthreads();
        for (int i = tid; i < kDigits; i += 1024) s.sums[i] = 0, s.counts[i] = 0;
        if (tid == 0) s.found = 0;
        __syncthreads();
        for (int i = tid; i < a.vocab; i += 1024) {
            const float x = load_logit<BF16>(a, row, i);
            const uint64_t p = place_of(x, i);
            if (x == -INFINITY || (p >> low) != prefix) continue;
            const int digit = (int)((p >> next) & ((1 << bits) - 1));
            atomicAdd(&s.counts[digit], 1u);
            const uint64_t w = weight_of(x, top, per);
            if (w) atomicAdd((unsigned long long*)&s.sums[digit], (unsigned long long)w);
        }
        __syncthreads();
        const uint64_t c0 = s.counts[2 * tid], c1 = s.counts[2 * tid + 1];
        const uint64_t s0 = s.sums[2 * tid], s1 = s.sums[2 * tid + 1];
        uint64_t c = c0 + c1, w = s0 + s1;
        for (int x = 1; x < 64; x <<= 1) {
            const uint64_t oc = __shfl_up(c, x), ow = __shfl_up(w, x);
            if (lane >= x) c += oc, w += ow;
        }
        if (lane == 63) s.wave_sums[wave] = w, s.wave_counts[wave] = c;
        __syncthreads();
        uint64_t ac = done_count, aw = done_sum;
        for (int v = 0; v < wave; ++v) ac += s.wave_counts[v], aw += s.wave_sums[v];
        c += ac, w += aw;
        // Cumulative values ahead of and behind the thread's two digits.
        const uint64_t b0c = c - c0 - c1, b0w = w - s0 - s1;
        const uint64_t before = COUNT ? b0c : b0w, mid = COUNT ? b0c + c0 : b0w + s0;
        const uint64_t after = COUNT ? c : w;
        if (before < target && target <= after) {
            const bool second = mid < target;
            s.found = 1;
            s.place = (prefix << bits) | (uint64_t)(2 * tid + second);
            s.sum = second ? b0w + s0 : b0w;
            s.count = second ? b0c + c0 : b0c;
        }
        __syncthreads();
        if (!s.found) return false;
        prefix = s.place, done_sum = s.sum, done_count = s.count;
        low = next;
    }
    place = prefix;
    sum = done_sum + weight_of(place_value(place), top, per);
    return true;
}

// A row by its places' digits.
template <bool BF16>
__device__ void pick_by_digits(const SampleArgs& a, int row, const RowRule& q, float top, Shared& s) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    // All weights, and those of at least min_p.
    const uint64_t least = max((uint64_t)ceil(q.min_p * kOne), (uint64_t)1);
    uint64_t all = 0, strong = 0;
    for (int i = tid; i < a.vocab; i += 1024) {
        const uint64_t w = weight_of(load_logit<BF16>(a, row, i), top, q.per);
        all += w;
        strong += w >= least ? w : 0;
    }
    for (int x = 32; x; x >>= 1) all += __shfl_xor(all, x), strong += __shfl_xor(strong, x);
    __syncthreads();
    if (lane == 0) s.wave_sums[wave] = all, s.wave_counts[wave] = strong;
    __syncthreads();
    all = strong = 0;
    for (int v = 0; v < 16; ++v) all += s.wave_sums[v], strong += s.wave_counts[v];
    uint64_t place, sum;
    if (q.top_k && find_place<BF16, true>(a, row, top, q.per, q.top_k, s, place, sum)) all = sum;
    uint64_t kept = all;
    if (q.top_p < 1.0 &&
        find_place<BF16, false>(a, row, top, q.per, cut_at(q.top_p, all), s, place, sum))
        kept = min(kept, sum);
    kept = min(kept, strong);
    find_place<BF16, false>(a, row, top, q.per, draw_at(q.uniform, kept), s, place, sum);
    if (tid == 0) put_token(a, row, place, top, q, kept);
}

// ------------------------------------------------------------------- bins

constexpr int kBins = 2048, kList = 1024, kSliceThreads = 256;

__device__ __forceinline__ int bin_of(float x, float top, const RowRule& q) {
    return (int)fminf((top - x) * q.bins, (float)(kBins - 1));
}

// Per row in the workspace.
struct RowSpace {
    uint64_t* firsts;   // [slices]: each slice's first place
    uint64_t* sums;     // [kBins]
    uint32_t* counts;   // [kBins]
    uint32_t* listed;   // places there are for the list
    uint64_t* list;     // [kList]
};

struct SliceArgs {
    SampleArgs s;
    char* space;
    int64_t row_bytes;
    int slices;
};

__device__ __forceinline__ RowSpace row_space(const SliceArgs& a, int row) {
    char* p = a.space + row * a.row_bytes;
    RowSpace r;
    r.sums = (uint64_t*)p;
    r.list = r.sums + kBins;
    r.firsts = r.list + kList;
    r.counts = (uint32_t*)(r.firsts + a.slices);
    r.listed = r.counts + kBins;
    return r;
}

// The logits of a slice of a row, N of a 16-byte access at a time: f(values, id
// of the first); values that are not the row's are -infinity.
template <bool BF16, typename F>
__device__ __forceinline__ void each_logit(const SampleArgs& a, int row, int slice, int slices, F f) {
    constexpr int SIZE = BF16 ? 2 : 4, N = 16 / SIZE, AHEAD = 4;
    const char* base = (const char*)a.logits + (int64_t)row * a.stride * SIZE;
    const int skip = (int)((uintptr_t)base % 16) / SIZE;  // values ahead of the row in its first access
    const int vectors = (a.vocab + skip + N - 1) / N;
    const int v0 = (int)((int64_t)vectors * slice / slices);
    const int v1 = (int)((int64_t)vectors * (slice + 1) / slices);
    for (int v = v0 + (int)threadIdx.x; v < v1; v += kSliceThreads * AHEAD) {
        u32x4_t raw[AHEAD];
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) {
            const int at = v + k * kSliceThreads, first = at * N - skip;
            if (at < v1 && first >= 0 && first + N <= a.vocab)
                raw[k] = *(const u32x4_t*)(base + (int64_t)first * SIZE);
        }
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) {
            const int at = v + k * kSliceThreads, first = at * N - skip;
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

template <bool BF16>
__global__ __launch_bounds__(kSliceThreads) void sample_first_kernel(SliceArgs a) {
    __shared__ uint64_t waves[kSliceThreads / 64];
    const int row = (int)(blockIdx.x / (uint32_t)a.slices), slice = (int)(blockIdx.x % (uint32_t)a.slices);
    const RowSpace sp = row_space(a, row);
    // The row's bins start from zero.
    if (a.slices > 1)
        for (int i = slice * kSliceThreads + (int)threadIdx.x; i < kBins; i += a.slices * kSliceThreads)
            sp.sums[i] = 0, sp.counts[i] = 0;
    if (slice == 0 && threadIdx.x == 0) *sp.listed = 0;
    float top = -INFINITY;
    int id = 0x7FFFFFFF;
    each_logit<BF16>(a.s, row, slice, a.slices, [&](const auto& x, int first) {
        constexpr int N = sizeof(x) / sizeof(float);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            id = x[i] > top ? first + i : id;
            top = fmaxf(top, x[i]);
        }
    });
    uint64_t place = top == -INFINITY ? kNowhere : place_of(top, id);
    for (int x = 32; x; x >>= 1) place = min(place, (uint64_t)__shfl_xor((unsigned long long)place, x));
    if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = place;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < kSliceThreads / 64; ++w) place = min(place, waves[w]);
        sp.firsts[slice] = place;
    }
}

// The row's first place, from its slices'.
__device__ __forceinline__ uint64_t first_of(const RowSpace& sp, int slices) {
    const int lane = threadIdx.x & 63;
    uint64_t place = kNowhere;
    for (int i = lane; i < slices; i += 64) place = min(place, sp.firsts[i]);
    for (int x = 32; x; x >>= 1) place = min(place, (uint64_t)__shfl_xor((unsigned long long)place, x));
    return place;
}

template <bool BF16>
__global__ __launch_bounds__(kSliceThreads) void sample_bins_kernel(SliceArgs a) {
    __shared__ uint64_t sums[kBins];
    __shared__ uint32_t counts[kBins];
    const int row = (int)(blockIdx.x / (uint32_t)a.slices), slice = (int)(blockIdx.x % (uint32_t)a.slices);
    const int r = request_row(a.s.rules, row);
    if (r < 0) return;
    const RowRule q = rule_of(a.s, r, row);
    if (q.greedy) return;
    const RowSpace sp = row_space(a, row);
    const uint64_t place = first_of(sp, a.slices);
    if (place == kNowhere) return;
    const float top = place_value(place);
    for (int i = threadIdx.x; i < kBins; i += kSliceThreads) sums[i] = 0, counts[i] = 0;
    __syncthreads();
    each_logit<BF16>(a.s, row, slice, a.slices, [&](const auto& x, int) {
        constexpr int N = sizeof(x) / sizeof(float);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if (x[i] == -INFINITY) continue;
            const int b = bin_of(x[i], top, q);
            if (q.top_k) atomicAdd(&counts[b], 1u);
            const uint64_t w = weight_of(x[i], top, q.per);
            if (w) atomicAdd((unsigned long long*)&sums[b], (unsigned long long)w);
        }
    });
    __syncthreads();
    for (int i = threadIdx.x; i < kBins; i += kSliceThreads) {
        if (a.slices == 1) {
            sp.sums[i] = sums[i], sp.counts[i] = counts[i];
        } else {
            if (sums[i]) atomicAdd((unsigned long long*)&sp.sums[i], (unsigned long long)sums[i]);
            if (counts[i]) atomicAdd(&sp.counts[i], counts[i]);
        }
    }
}

// Cumulative bins of a row, by a workgroup of THREADS.
template <int THREADS>
struct Cumulative {
    uint64_t sums[kBins + 1];   // [b]: of the bins below b
    uint32_t counts[kBins + 1];
    uint64_t wave_sums[THREADS / 64];
    uint32_t wave_counts[THREADS / 64];

    __device__ __forceinline__ void load(const RowSpace& sp) {
        constexpr int PER = kBins / THREADS;
        const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
        uint64_t s[PER], w = 0;
        uint32_t n[PER], c = 0;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            s[i] = sp.sums[tid * PER + i], n[i] = sp.counts[tid * PER + i];
            w += s[i], c += n[i];
        }
        uint64_t w_at = w;
        uint32_t c_at = c;
        for (int x = 1; x < 64; x <<= 1) {
            const uint64_t ow = __shfl_up((unsigned long long)w_at, x);
            const uint32_t oc = __shfl_up(c_at, x);
            if (lane >= x) w_at += ow, c_at += oc;
        }
        if (lane == 63) wave_sums[wave] = w_at, wave_counts[wave] = c_at;
        __syncthreads();
        w_at -= w, c_at -= c;
        for (int v = 0; v < wave; ++v) w_at += wave_sums[v], c_at += wave_counts[v];
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            sums[tid * PER + i] = w_at, counts[tid * PER + i] = c_at;
            w_at += s[i], c_at += n[i];
        }
        if (tid == THREADS - 1) sums[kBins] = w_at, counts[kBins] = c_at;
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
        there = __ballot(lane >= 32 || below[b + lane + 1] >= target);
        return b + __ffsll((unsigned long long)there) - 1;
    }
};

// Ranges of bins that hold a cut or the draw, whatever the tokens inside them
// decide, and what is known ahead of that.
struct Ranges {
    int lo[4], hi[4];   // top-k, top-p, min-p, draw; empty where lo > hi
    uint64_t all;       // the sum behind top-k where its range is empty
    int strong;         // bins below it hold only tokens of at least min_p

    __device__ __forceinline__ bool has(int b) const {
        bool in = false;
#pragma unroll
        for (int i = 0; i < 4; ++i) in |= b >= lo[i] && b <= hi[i];
        return in;
    }
};

template <int THREADS>
__device__ __forceinline__ Ranges ranges_of(const Cumulative<THREADS>& c, const RowRule& q) {
    typedef Cumulative<THREADS> C;
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
    g.strong = kBins;
    if (q.min_p > 0.0) {
        // A bin to either side for the rounding of logarithm and bins.
        const double at = -log(q.min_p) * 64.0;
        const int b = at < kBins ? (int)at : kBins;
        const int low = max(b - 1, 0), high = min(b + 1, kBins - 1);
        if (low < kBins && c.sums[low] < most) {
            g.lo[2] = low, g.hi[2] = high, g.strong = low;
            least = min(least, max(c.sums[low], one));
            most = min(most, c.sums[high + 1]);
        }
    }
    g.lo[3] = C::reach(c.sums, draw_at(q.uniform, least));
    g.hi[3] = C::reach(c.sums, draw_at(q.uniform, most));
    return g;
}

template <bool BF16>
__global__ __launch_bounds__(kSliceThreads) void sample_list_kernel(SliceArgs a) {
    __shared__ Cumulative<kSliceThreads> bins;
    const int row = (int)(blockIdx.x / (uint32_t)a.slices), slice = (int)(blockIdx.x % (uint32_t)a.slices);
    const int r = request_row(a.s.rules, row);
    if (r < 0) return;
    const RowRule q = rule_of(a.s, r, row);
    if (q.greedy) return;
    const RowSpace sp = row_space(a, row);
    const uint64_t place = first_of(sp, a.slices);
    if (place == kNowhere) return;
    const float top = place_value(place);
    bins.load(sp);
    const Ranges g = ranges_of(bins, q);
    each_logit<BF16>(a.s, row, slice, a.slices, [&](const auto& x, int first) {
        constexpr int N = sizeof(x) / sizeof(float);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if (x[i] == -INFINITY || !g.has(bin_of(x[i], top, q))) continue;
            const uint32_t at = atomicAdd(sp.listed, 1u);
            if (at < kList) sp.list[at] = place_of(x[i], first + i);
        }
    });
}

// The smallest of a workgroup's values.
__device__ __forceinline__ uint64_t least_of(uint64_t v, uint64_t (&waves)[16]) {
    for (int x = 32; x; x >>= 1) v = min(v, (uint64_t)__shfl_xor((unsigned long long)v, x));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = v;
    __syncthreads();
    for (int w = 0; w < 16; ++w) v = min(v, waves[w]);
    return v;
}
__device__ __forceinline__ uint64_t sum_of(uint64_t v, uint64_t (&waves)[16]) {
    for (int x = 32; x; x >>= 1) v += __shfl_xor((unsigned long long)v, x);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0;
    for (int w = 0; w < 16; ++w) v += waves[w];
    return v;
}

struct PickSpace {
    Cumulative<1024> bins;
    uint64_t places[kList], weights[kList];
    uint16_t bin[kList];
    uint64_t waves[16];
};

template <bool BF16>
__global__ __launch_bounds__(1024) void sample_pick_kernel(SliceArgs a) {
    __shared__ union Space {
        PickSpace p;
        Shared digits;
    } s;
    const int row = blockIdx.x, tid = threadIdx.x;
    const int r = request_row(a.s.rules, row);
    if (r < 0) return;
    const RowRule q = rule_of(a.s, r, row);
    const RowSpace sp = row_space(a, row);
    const uint64_t first = first_of(sp, a.slices);
    if (first == kNowhere || q.greedy) {
        if (tid == 0) {
            a.s.tokens[row] = first == kNowhere ? -1 : place_id(first);
            if (a.s.probabilities) a.s.probabilities[row] = first == kNowhere ? 0.0f : 1.0f;
        }
        return;
    }
    const float top = place_value(first);
    const int n = (int)min(*sp.listed, (uint32_t)kList + 1);
    if (n > kList) {
        pick_by_digits<BF16>(a.s, row, q, top, s.digits);
        return;
    }
    PickSpace& p = s.p;
    uint64_t place = kNowhere, weight = 0;
    int bin = -1;
    if (tid < n) {
        place = sp.list[tid];
        const float x = place_value(place);
        weight = weight_of(x, top, q.per);
        bin = bin_of(x, top, q);
        p.places[tid] = place, p.weights[tid] = weight, p.bin[tid] = (uint16_t)bin;
    }
    p.bins.load(sp);
    const Ranges g = ranges_of(p.bins, q);
    // The listed token's cumulative weight and number.
    uint64_t sum = ~0ull, count = 0;
    if (tid < n) {
        sum = p.bins.sums[bin], count = p.bins.counts[bin];
        for (int i = 0; i < n; ++i) {
            const bool ahead = p.bin[i] == bin && p.places[i] <= place;
            sum += ahead ? p.weights[i] : 0;
            count += ahead;
        }
    }
    const uint64_t none = ~0ull;
    uint64_t kept = g.all;
    if (g.lo[0] <= g.hi[0]) kept = least_of(tid < n && count == (uint64_t)q.top_k ? sum : none, p.waves);
    if (q.top_p < 1.0) {
        const uint64_t target = cut_at(q.top_p, kept);
        kept = min(kept, least_of(tid < n && sum >= target ? sum : none, p.waves));
    }
    if (g.strong < kBins) {
        const uint64_t least = max((uint64_t)ceil(q.min_p * kOne), (uint64_t)1);
        const bool mine = tid < n && bin >= g.lo[2] && bin <= g.hi[2] && weight >= least;
        kept = min(kept, p.bins.sums[g.strong] + sum_of(mine ? weight : 0, p.waves));
    }
    const uint64_t target = draw_at(q.uniform, kept);
    const uint64_t drawn = least_of(tid < n && sum >= target ? sum : none, p.waves);
    // One token has this sum: every weight in the way of one is more than 0.
    if (tid < n && sum == drawn && weight) put_token(a.s, row, place, top, q, kept);
}

// How many slices a row is cut into: 1024 workgroups in all where that leaves a
// slice 4096 logits.
int64_t slices_of(int64_t rows, int64_t vocab) {
    return std::max<int64_t>(1, std::min<int64_t>({(vocab + 4095) / 4096, 64, (1024 + rows - 1) / rows}));
}
int64_t row_bytes_of(int64_t slices) {
    return (kBins * 12 + kList * 8 + slices * 8 + 4 + 15) / 16 * 16;
}

template <bool BF16>
hipError_t launch_sample(const SliceArgs& a, hipStream_t st) {
    const uint32_t blocks = (uint32_t)((int64_t)a.s.rows * a.slices);
    sample_first_kernel<BF16><<<blocks, kSliceThreads, 0, st>>>(a);
    sample_bins_kernel<BF16><<<blocks, kSliceThreads, 0, st>>>(a);
    sample_list_kernel<BF16><<<blocks, kSliceThreads, 0, st>>>(a);
    sample_pick_kernel<BF16><<<(uint32_t)a.s.rows, 1024, 0, st>>>(a);
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
    SampleArgs a = {*rules, logits, uniform, tokens, probabilities, stride, (int)rows, (int)vocab,
                    uniform_bits == 64};
    const DeviceScope scope(ncm_ctx_device(ctx));
    rc = step_hip(scope.error(), "sample device");
    if (rc) return rc;
    const hipStream_t st = ncm_ctx_stream(ctx);
    const int64_t slices = slices_of(rows, vocab);
    const SliceArgs s = {a, (char*)workspace, row_bytes_of(slices), (int)slices};
    return step_hip(dtype == NCM_OUT_BF16 ? launch_sample<true>(s, st) : launch_sample<false>(s, st),
                    "sample launch");
}
