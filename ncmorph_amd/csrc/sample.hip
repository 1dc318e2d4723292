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
// A cut is found digit by digit of the token's 52-bit place in the order (32
// bits of the logit, 20 of the id): counts and sums of the tokens by their next
// digit, in LDS, then the digit where the count or the sum passes its target.
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
    double per;      // 1 / T
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
    q.per = (double)fmaxf(t, 0x1p-96f);
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

__device__ __forceinline__ uint64_t weight_of(float x, float top, double t) {
    if (x == -INFINITY) return 0;
    const double d = ((double)x - (double)top) / t;
    return d < -31.0 ? 0 : (uint64_t)__double2ull_rn(exp(d) * kOne);
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
__device__ bool find_place(const SampleArgs& a, int row, float top, double t, uint64_t target,
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
            const uint64_t w = weight_of(x, top, t);
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
    sum = done_sum + weight_of(place_value(place), top, t);
    return true;
}

template <bool BF16>
__global__ __launch_bounds__(1024) void sample_kernel(SampleArgs a) {
    __shared__ Shared s;
    const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int r = request_row(a.rules, row);
    if (r < 0) return;
    const RowRule q = rule_of(a, r, row);
    uint64_t first = kNowhere;
    for (int i = tid; i < a.vocab; i += 1024) {
        const float x = load_logit<BF16>(a, row, i);
        if (x != -INFINITY) first = min(first, place_of(x, i));
    }
    for (int x = 32; x; x >>= 1) first = min(first, (uint64_t)__shfl_xor((unsigned long long)first, x));
    if (lane == 0) s.wave_sums[wave] = first;
    __syncthreads();
    for (int v = 0; v < 16; ++v) first = min(first, s.wave_sums[v]);
    if (first == kNowhere || q.greedy) {
        if (tid == 0) {
            a.tokens[row] = first == kNowhere ? -1 : place_id(first);
            if (a.probabilities) a.probabilities[row] = first == kNowhere ? 0.0f : 1.0f;
        }
        return;
    }
    const float top = place_value(first);
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
    bool more;
    if (q.top_p < 1.0) {
        uint64_t target = share_of(fmax(q.top_p, 0.0), all, more);
        target = max(target + (more ? 1 : 0), (uint64_t)1);
        if (find_place<BF16, false>(a, row, top, q.per, target, s, place, sum)) kept = min(kept, sum);
    }
    kept = min(kept, strong);
    const uint64_t target = share_of(q.uniform, kept, more) + 1;
    find_place<BF16, false>(a, row, top, q.per, target, s, place, sum);
    if (tid == 0) {
        a.tokens[row] = place_id(place);
        if (a.probabilities)
            a.probabilities[row] =
                (float)((double)weight_of(place_value(place), top, q.per) / (double)kept);
    }
}

}  // namespace
}  // namespace ncm

extern "C" int ncm_sample_workspace(int64_t rows, int64_t vocab, size_t* bytes) {
    using namespace ncm;
    if (!bytes) return NCM_E_NULL;
    *bytes = 0;
    if (rows < 0 || rows > kMaxBlocks / 4 || vocab < 0 || vocab > kMaxVocab) return NCM_E_SHAPE;
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
    if (dtype == NCM_OUT_BF16) sample_kernel<true><<<(uint32_t)rows, 1024, 0, st>>>(a);
    else sample_kernel<false><<<(uint32_t)rows, 1024, 0, st>>>(a);
    return step_hip(hipGetLastError(), "sample launch");
}
