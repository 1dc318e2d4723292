// Penalties, biases and grammar masks on logits (ncm_adjust_logits_dev).
//
// A workgroup takes a slice of a row's vocabulary. It counts the history and
// the row's drafted path into one 32-bit LDS word per token of the slice
// (integer atomics: the result does not depend on their order), then streams
// the logits through once. Biased tokens are marked in their words, left out
// of the stream and done by the thread that owns their first list entry, so
// that entries of one token are summed in list order.
//
// Memory bound: logits in and out and a bit a token; the history is read once
// per slice, from the L2 after the first. 143 rows of 151936 float32 with
// histories of 4000, masks and 300 biases: 47 us (3.7 TB/s).
#include "step.h"

namespace ncm {
namespace {

constexpr uint32_t kInPrompt = 0x80000000u, kBiased = 0x40000000u, kCount = 0x3FFFFFFFu;

struct LogitArgs {
    ncm_logit_rules_t rules;
    const void* in;
    void* out;
    int64_t in_stride, out_stride;
    int rows, vocab, slices, words;
};

template <bool BF16> struct Logit;
template <> struct Logit<false> {
    typedef float T;
    static constexpr int N = 4;
    static __device__ __forceinline__ float get(const float* p) { return *p; }
    static __device__ __forceinline__ void put(float* p, float v) { *p = v; }
};
template <> struct Logit<true> {
    typedef uint16_t T;
    static constexpr int N = 8;
    static __device__ __forceinline__ float get(const uint16_t* p) {
        return __uint_as_float((uint32_t)*p << 16);
    }
    static __device__ __forceinline__ void put(uint16_t* p, float v) { *p = (uint16_t)bf16_bits_rne(v); }
};

struct RowRules {
    float rep, freq, pres;
    const uint32_t* allowed;
};

__device__ __forceinline__ float adjusted(float x, uint32_t word, const RowRules& r) {
    if (word & ~kBiased) {
        const uint32_t count = word & kCount;
        x = x > 0.0f ? x / r.rep : x * r.rep;
        x = x - r.freq * (float)count;
        x = count ? x - r.pres : x;
    }
    return x;
}

__device__ __forceinline__ bool token_allowed(const RowRules& r, int t) {
    return !r.allowed || (r.allowed[t >> 5] >> (t & 31)) & 1u;
}

constexpr int threads_of(bool bf16, int slice) { return slice == 8192 && !bf16 ? 512 : 256; }

// COUNTS: the row has a history, a drafted path or biases. WIDE: 16-byte
// accesses, in and out equally far past a 16-byte boundary; the slice's logits
// are then loaded ahead of the counting, into registers.
template <bool BF16, bool COUNTS, bool WIDE, int SLICE>
__global__ __launch_bounds__(threads_of(BF16, SLICE)) void adjust_logits_kernel(LogitArgs a) {
    typedef Logit<BF16> L;
    typedef typename L::T T;
    constexpr int TH = threads_of(BF16, SLICE);
    __shared__ __attribute__((aligned(16))) uint32_t word[COUNTS ? SLICE : 4];
    __shared__ int twice;  // a token stands in two entries of the bias list
    const ncm_logit_rules_t& u = a.rules;
    const int row = (int)(blockIdx.x / (uint32_t)a.slices), tid = threadIdx.x;
    int r = row, o0 = 0, n = 1;
    if (u.offsets) {
        // The request of the row: as many as end at or before it.
        int c = 0;
        for (int j = tid; j < u.requests; j += TH) c += u.offsets[j + 1] <= row;
        r = __syncthreads_count(c > 0);  // all of them, if one a thread
        if (u.requests > TH) {
            __shared__ int sum;
            if (tid == 0) sum = 0;
            __syncthreads();
            atomicAdd(&sum, c);
            __syncthreads();
            r = sum;
        }
        if (r >= u.requests) return;
        o0 = min(max(u.offsets[r], 0), a.rows);
        n = min(u.offsets[r + 1], a.rows) - o0;
        if (row < o0 || row >= o0 + n) return;
    } else if (row >= u.requests) {
        return;
    }
    const T* in = (const T*)a.in + row * a.in_stride;
    T* out = (T*)a.out + row * a.out_stride;
    // The slice starts at a 16-byte boundary: the first one's may lie `shift`
    // values ahead of the row.
    const int shift = WIDE ? (int)(((uintptr_t)in % 16) / sizeof(T)) : 0;
    const int from = (int)(blockIdx.x % (uint32_t)a.slices) * SLICE - shift;
    const int lo = max(from, 0), hi = min(from + SLICE, a.vocab);
    RowRules rr;
    rr.rep = u.repetition ? u.repetition[r] : 1.0f;
    rr.freq = u.frequency ? u.frequency[r] : 0.0f;
    rr.pres = u.presence ? u.presence[r] : 0.0f;
    rr.allowed = u.allowed ? u.allowed + (int64_t)row * a.words : nullptr;
    const int32_t* ids = u.bias_ids ? u.bias_ids + r * u.bias_count : nullptr;
    const int nb = ids ? (int)u.bias_count : 0;

    constexpr int N = WIDE ? L::N : 1, VECS = WIDE ? SLICE / (TH * N) : 1;
    // Whole groups of N values lie in [first, last).
    const int first = from < 0 ? min(from + N, hi) : lo;
    const int last = first + (hi - first) / N * N;
    u32x4_t raw[VECS];
    if constexpr (WIDE) {
#pragma unroll
        for (int k = 0; k < VECS; ++k) {
            const int t = first + (k * TH + tid) * N;
            if (t < last) raw[k] = *(const u32x4_t*)(in + t);
        }
    }
    if constexpr (COUNTS) {
        for (int i = tid * 4; i < SLICE; i += 4 * TH) *(u32x4_t*)(word + i) = u32x4_t{0, 0, 0, 0};
        if (tid == 0) twice = 0;
        __syncthreads();
        if (u.history) {
            const int width = (int)u.history_width;
            const int32_t* h = u.history + r * u.history_width;
            const int all = u.history_lens ? min(max(u.history_lens[r], 0), width) : width;
            const int p = u.prompt_lens ? min(max(u.prompt_lens[r], 0), width) : 0;
            for (int i = tid; i < max(all, p); i += TH) {
                const int t = h[i];
                if (t < lo || t >= hi) continue;
                if (i < p) atomicOr(&word[t - from], kInPrompt);
                else atomicAdd(&word[t - from], 1u);
            }
        }
        if (u.draft_tokens) {
            const uint64_t* bits = u.tree_mask ? u.tree_mask + row * u.mask_words : nullptr;
            for (int j = tid; j < n; j += TH) {
                const int t = u.draft_tokens[o0 + j];
                if (t < lo || t >= hi) continue;
                const bool on = bits ? (j >> 6) < u.mask_words && ((bits[j >> 6] >> (j & 63)) & 1u)
                                     : j <= row - o0;
                if (on) atomicAdd(&word[t - from], 1u);
            }
        }
        for (int e = tid; e < nb; e += TH) {
            const int t = ids[e];
            if (t < lo || t >= hi) continue;
            if (atomicOr(&word[t - from], kBiased) & kBiased) twice = 1;
        }
        __syncthreads();
    }

    auto one = [&](int t) {
        const uint32_t w = COUNTS ? word[t - from] : 0u;
        if (w & kBiased) return;
        const float x = L::get(in + t);
        L::put(out + t, token_allowed(rr, t) ? adjusted(x, w, rr) : -INFINITY);
    };
    if constexpr (!WIDE) {
        for (int t = lo + tid; t < hi; t += TH) one(t);
    } else {
        for (int t = lo + tid; t < first; t += TH) one(t);
        for (int t = last + tid; t < hi; t += TH) one(t);
#pragma unroll
        for (int k = 0; k < VECS; ++k) {
            const int t = first + (k * TH + tid) * N;
            if (t >= last) break;
            float x[N];
            uint32_t w[N];
            uint32_t any = 0;
#pragma unroll
            for (int i = 0; i < N; ++i)
                x[i] = BF16 ? __uint_as_float((i % 2) ? raw[k][(i / 2) % 4] & 0xFFFF0000u
                                                      : raw[k][(i / 2) % 4] << 16)
                            : __uint_as_float(raw[k][i % 4]);
            if constexpr (COUNTS) {
#pragma unroll
                for (int i = 0; i < N; i += 4) {
                    const u32x4_t c = *(const u32x4_t*)(word + (t - from) + i);
#pragma unroll
                    for (int j = 0; j < 4; ++j) w[i + j] = c[j], any |= c[j];
                }
                if (any) {
#pragma unroll
                    for (int i = 0; i < N; ++i) x[i] = adjusted(x[i], w[i], rr);
                }
            }
            if (rr.allowed) {
                const uint32_t w0 = rr.allowed[t >> 5], w1 = rr.allowed[(t + N - 1) >> 5];
                const uint32_t bits = (uint32_t)(((((uint64_t)w1) << 32) | w0) >> (t & 31));
#pragma unroll
                for (int i = 0; i < N; ++i) x[i] = (bits >> i) & 1u ? x[i] : -INFINITY;
            }
            if (any & kBiased) {
#pragma unroll
                for (int i = 0; i < N; ++i)
                    if (!(w[i] & kBiased)) L::put(out + t + i, x[i]);
            } else {
                u32x4_t o;
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    o[i] = BF16 ? bf16x2_bits_rne(x[(2 * i) % N], x[(2 * i + 1) % N])
                                : __float_as_uint(x[i]);
                // Large outputs past the caches: 51 us against 54 for 143 rows
                // of 151936 float32.
                if constexpr (SLICE == 8192) __builtin_nontemporal_store(o, (u32x4_t*)(out + t));
                else *(u32x4_t*)(out + t) = o;
            }
        }
    }
    if constexpr (COUNTS) {
        const float* values = u.bias_values + r * u.bias_count;
        for (int e = tid; e < nb; e += TH) {
            const int t = ids[e];
            if (t < lo || t >= hi) continue;
            float b = values[e];
            if (twice) {
                bool later = false;
                for (int j = 0; j < e; ++j) later |= ids[j] == t;
                if (later) continue;
                for (int j = e + 1; j < nb; ++j)
                    if (ids[j] == t) b = b + values[j];
            }
            const float x = adjusted(L::get(in + t), word[t - from], rr) + b;
            L::put(out + t, token_allowed(rr, t) ? x : -INFINITY);
        }
    }
}

// Slices of 8192 tokens where that leaves four workgroups a CU: the history is
// read once a slice. 8192 and 2048: 48 and 70 us for 143 rows of 151936 float32,
// 7.4 and 6.1 for 4 rows of 128256.
int slice_of(int64_t rows, int64_t vocab) {
    return rows * (vocab / 8192 + 1) >= 1024 ? 8192 : 2048;
}

template <bool BF16, bool COUNTS, bool WIDE>
void launch(const LogitArgs& a, int slice, uint32_t blocks, hipStream_t st) {
    const int threads = threads_of(BF16, slice);
    if (slice == 8192) adjust_logits_kernel<BF16, COUNTS, WIDE, 8192><<<blocks, threads, 0, st>>>(a);
    else adjust_logits_kernel<BF16, COUNTS, WIDE, 2048><<<blocks, threads, 0, st>>>(a);
}

}  // namespace
}  // namespace ncm

extern "C" int ncm_adjust_logits_dev(ncm_ctx_t* ctx, const ncm_logit_rules_t* rules,
                                     const void* logits, void* out, int64_t rows, int64_t vocab,
                                     int64_t in_stride, int64_t out_stride, int dtype) {
    using namespace ncm;
    if (!ctx || !rules) return NCM_E_NULL;
    const ncm_logit_rules_t& u = *rules;
    if (rows < 0 || rows > kMaxRows || vocab < 0 || vocab > (1 << 30) || in_stride < vocab ||
        out_stride < vocab || in_stride > (int64_t(1) << 40) || out_stride > (int64_t(1) << 40) ||
        u.requests < 0 || u.requests > kMaxRows || u.history_width < 0 ||
        u.history_width > kMaxRows || u.bias_count < 0 || u.bias_count > kMaxRows ||
        u.mask_words < 0 || u.mask_words > kMaxRows)
        return NCM_E_SHAPE;
    // A token that stands in every entry still leaves the word's marks alone.
    if ((u.history ? u.history_width : 0) + (u.draft_tokens ? rows : 0) > (int64_t)kCount)
        return NCM_E_SHAPE;
    if (dtype != NCM_OUT_F32 && dtype != NCM_OUT_BF16) return NCM_E_ARG;
    if (u.offsets ? u.requests > kMaxRequests : u.requests != rows) return NCM_E_SHAPE;
    if ((u.draft_tokens && !u.offsets) || !u.bias_ids != !u.bias_values) return NCM_E_NULL;
    const bool bf16 = dtype == NCM_OUT_BF16;
    const int size = bf16 ? 2 : 4, slice = slice_of(rows, vocab);
    const int slices = (int)((vocab + 16 / size - 1 + slice - 1) / slice);
    if (rows * slices > kMaxThreads / threads_of(bf16, slice)) return NCM_E_SHAPE;
    if (rows == 0 || vocab == 0 || u.requests == 0) return NCM_OK;
    if (!logits || !out) return NCM_E_NULL;
    if ((uintptr_t)logits % size || (uintptr_t)out % size) return NCM_E_ARG;
    if (logits == out && in_stride != out_stride) return NCM_E_ARG;
    const bool wide = ((uintptr_t)logits - (uintptr_t)out) % 16 == 0 &&
                      (in_stride - out_stride) * size % 16 == 0;
    const bool counts = (u.history && u.history_width > 0) || u.draft_tokens ||
                        (u.bias_ids && u.bias_count > 0);
    LogitArgs a = {u, logits, out, in_stride, out_stride, (int)rows, (int)vocab, slices,
                   (int)((vocab + 31) / 32)};
    const uint32_t blocks = (uint32_t)(rows * slices);
    const DeviceScope scope(ncm_ctx_device(ctx));
    const int rc = step_hip(scope.error(), "adjust_logits device");
    if (rc) return rc;
    const hipStream_t st = ncm_ctx_stream(ctx);
    auto go = [&](auto b, auto c, auto w) {
        launch<decltype(b)::value, decltype(c)::value, decltype(w)::value>(a, slice, blocks, st);
    };
    const std::true_type yes;
    const std::false_type no;
    if (bf16) counts ? (wide ? go(yes, yes, yes) : go(yes, yes, no))
                     : (wide ? go(yes, no, yes) : go(yes, no, no));
    else counts ? (wide ? go(no, yes, yes) : go(no, yes, no))
                : (wide ? go(no, no, yes) : go(no, no, no));
    return step_hip(hipGetLastError(), "adjust_logits launch");
}
