// The paged K/V cache: writing a step's K and V rows, quantised
// (ncm_kv_write_dev), and reading them back (ncm_kv_read_dev).
//
// A head of a token is head_dim / 8 lanes of eight values each. fp8 scales are
// powers of two: they cost a floating format no precision, and make both
// x / scale and, in bf16, code * scale exact. int8 codes are rint(x * 127 / m)
// of a correctly rounded quotient of exact operands (a bf16 value times 127 has
// 15 bits), so x = m / 2, a tie, rounds as it does in real numbers.
//
// Memory bound: a bf16 value in and its code out, or the other way.
#include "step.h"

namespace ncm {
namespace {

// The request of a row: the number of requests that end at or before it, each
// lane of the head counting its share of them.
template <int LANES>
__device__ __forceinline__ int request_of_row(const BatchView& b, int row, int lane) {
    int n = 0;
    for (int r = lane; r < b.requests; r += LANES) n += b.offsets[r + 1] <= row;
#pragma unroll
    for (int d = 1; d < LANES; d <<= 1) n += __shfl_xor(n, d);
    return n;
}

// Where a head of a row's token lies: page and token in the page; false where
// the row is nobody's.
struct Place {
    int page, at;
};
template <int LANES>
__device__ __forceinline__ bool place_of(const BatchView& b, const KvView& c, int row, int lane,
                                         Place& p) {
    const int r = request_of_row<LANES>(b, row, lane);
    if (r >= b.requests) return false;
    const Request q = request_of(b, r);
    if (row < q.o0 || row >= q.o0 + q.n) return false;
    const int64_t t = (int64_t)q.before + (row - q.o0);
    p.page = page_of(b, c, r, t);
    p.at = (int)(t & ((1 << c.page_log2) - 1));
    return true;
}

// Eight codes of eight values from two dwords of four.
__device__ __forceinline__ uint32_t fp8x4(float a, float b, float c, float d) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
}

struct WriteArgs {
    KvView cache;
    BatchView batch;
    const uint16_t* k;
    const uint16_t* v;
    int64_t k_stride, v_stride;
};

template <int HD, int CODES>
__global__ __launch_bounds__(256) void kv_write_kernel(WriteArgs a) {
    constexpr int LANES = HD / 8, PER = 256 / LANES;
    const int lane = threadIdx.x % LANES;
    const int heads = a.cache.kv_heads;
    const int64_t item = (int64_t)blockIdx.x * PER + threadIdx.x / LANES;
    const int64_t row64 = item / (2 * heads);
    if (row64 >= a.batch.rows) return;
    const int row = (int)row64, which = (int)(item % (2 * heads));
    const bool is_v = which >= heads;
    const int h = is_v ? which - heads : which;
    const uint16_t* src = (is_v ? a.v + row * a.v_stride : a.k + row * a.k_stride) + h * HD + 8 * lane;
    const u32x4_t w = *(const u32x4_t*)src;
    Place p;
    if (!place_of<LANES>(a.batch, a.cache, row, lane, p) || p.page < 0) return;
    const int64_t in_page = ((int64_t)h << a.cache.page_log2) + p.at;
    char* base = is_v ? a.cache.v : a.cache.k;
    const int64_t at = p.page * (is_v ? a.cache.v_stride : a.cache.k_stride) + in_page * HD + 8 * lane;
    if constexpr (CODES == NCM_KV_BF16) {
        *(u32x4_t*)(base + 2 * at) = w;
        return;
    }
    // Largest magnitude as bits: above every finite one where it is not finite.
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) m = max(m, max(w[i] & 0x7FFFu, (w[i] >> 16) & 0x7FFFu));
#pragma unroll
    for (int d = 1; d < LANES; d <<= 1) m = max(m, (uint32_t)__shfl_xor((int)m, d));
    float f[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) f[2 * i] = bf16_lo_to_f32(w[i]), f[2 * i + 1] = bf16_hi_to_f32(w[i]);
    float scale;
    u32x2_t q = {0, 0};
    if (m >= 0x7F80u) {
        scale = __uint_as_float(0x7FC00000u);
    } else if constexpr (CODES == NCM_KV_FP8) {
        // m = 1.f * 2^(E - 127) <= 1.75 * 2^8 * 2^e: e = E - 135, one more where
        // its fraction is above .75 (448 = 1.75 * 2^8).
        const int e = max((int)(m >> 7) - 135 + ((m & 0x7Fu) > 0x60u ? 1 : 0), -126);
        scale = __uint_as_float((uint32_t)(e + 127) << 23);
        const float inv = __uint_as_float((uint32_t)(127 - e) << 23);
        q[0] = fp8x4(f[0] * inv, f[1] * inv, f[2] * inv, f[3] * inv);
        q[1] = fp8x4(f[4] * inv, f[5] * inv, f[6] * inv, f[7] * inv);
    } else {
        const float top = __uint_as_float(m << 16);
        scale = top / 127.0f;
        if (m != 0) {
            // Both sides of the quotient 2^-32 smaller where x * 127 could pass
            // the fp32 range.
            const float down = m >= 0x7000u ? 0x1p-32f : 1.0f;
            const float up = 127.0f * down, den = top * down;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int c = (int)rintf((f[i] * up) / den);
                q[i / 4] |= ((uint32_t)c & 0xFFu) << (8 * (i % 4));
            }
        }
    }
    *(u32x2_t*)(base + at) = q;
    if (lane == 0) {
        if (is_v) a.cache.vs[p.page * a.cache.vs_stride + in_page] = scale;
        else a.cache.ks[p.page * a.cache.ks_stride + in_page] = scale;
    }
}

struct ReadArgs {
    KvView cache;
    BatchView batch;
    uint16_t* k;
    uint16_t* v;
    int64_t k_stride, v_stride;
};

template <int HD, int CODES>
__global__ __launch_bounds__(256) void kv_read_kernel(ReadArgs a) {
    constexpr int LANES = HD / 8, PER = 256 / LANES;
    const int lane = threadIdx.x % LANES;
    const int heads = a.cache.kv_heads;
    const int64_t item = (int64_t)blockIdx.x * PER + threadIdx.x / LANES;
    const int64_t row64 = item / (2 * heads);
    if (row64 >= a.batch.rows) return;
    const int row = (int)row64, which = (int)(item % (2 * heads));
    const bool is_v = which >= heads;
    const int h = is_v ? which - heads : which;
    Place p;
    if (!place_of<LANES>(a.batch, a.cache, row, lane, p)) return;
    u32x4_t w = {0, 0, 0, 0};
    if (p.page >= 0) {
        const int64_t in_page = ((int64_t)h << a.cache.page_log2) + p.at;
        const char* base = is_v ? a.cache.v : a.cache.k;
        const int64_t at =
            p.page * (is_v ? a.cache.v_stride : a.cache.k_stride) + in_page * HD + 8 * lane;
        if constexpr (CODES == NCM_KV_BF16) {
            w = *(const u32x4_t*)(base + 2 * at);
        } else {
            const u32x2_t q = *(const u32x2_t*)(base + at);
            const float scale = is_v ? a.cache.vs[p.page * a.cache.vs_stride + in_page]
                                     : a.cache.ks[p.page * a.cache.ks_stride + in_page];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int d = (int)q[i / 2];
                float lo, hi;
                if constexpr (CODES == NCM_KV_FP8) {
                    const f32x2_t t = (i % 2) ? __builtin_amdgcn_cvt_pk_f32_fp8(d, true)
                                              : __builtin_amdgcn_cvt_pk_f32_fp8(d, false);
                    lo = t[0], hi = t[1];
                } else {
                    lo = (float)(int8_t)(d >> (16 * (i % 2)));
                    hi = (float)(int8_t)(d >> (16 * (i % 2) + 8));
                }
                w[i] = bf16x2_bits_rne(lo * scale, hi * scale);
            }
        }
    }
    uint16_t* dst = (is_v ? a.v + row * a.v_stride : a.k + row * a.k_stride) + h * HD + 8 * lane;
    *(u32x4_t*)dst = w;
}

template <typename F>
void by_codes(int codes, F f) {
    switch (codes) {
        case NCM_KV_BF16: f(std::integral_constant<int, NCM_KV_BF16>()); break;
        case NCM_KV_FP8: f(std::integral_constant<int, NCM_KV_FP8>()); break;
        default: f(std::integral_constant<int, NCM_KV_INT8>()); break;
    }
}

// Checks that the write and the read share, then the launch for the cache's
// head_dim and codes.
template <typename Args, typename Ptr, typename Launch>
int move_rows(ncm_ctx_t* ctx, const ncm_kv_cache_t* cache, const ncm_kv_batch_t* batch, Ptr k,
              Ptr v, int64_t k_stride, int64_t v_stride, const char* what, Launch go) {
    if (!ctx) return NCM_E_NULL;
    Args a;
    int rc = check_cache(cache, &a.cache);
    if (rc) return rc;
    rc = check_batch(batch, a.cache.page_log2, &a.batch);
    if (rc) return rc;
    if (batch->rows == 0 || batch->requests == 0) return NCM_OK;
    const int64_t width = (int64_t)cache->kv_heads * cache->head_dim;
    rc = check_rows(k, k_stride, width);
    if (!rc) rc = check_rows(v, v_stride, width);
    if (rc) return rc;
    a.k = k, a.v = v, a.k_stride = k_stride, a.v_stride = v_stride;
    const int per = 256 / (cache->head_dim / 8);
    const int64_t blocks = (batch->rows * 2 * cache->kv_heads + per - 1) / per;
    if (blocks > 0x7FFFFFFF) return NCM_E_SHAPE;
    const DeviceScope scope(ncm_ctx_device(ctx));
    rc = step_hip(scope.error(), what);
    if (rc) return rc;
    go(a, (uint32_t)blocks, ncm_ctx_stream(ctx));
    return step_hip(hipGetLastError(), what);
}

}  // namespace
}  // namespace ncm

extern "C" int ncm_kv_write_dev(ncm_ctx_t* ctx, const ncm_kv_cache_t* cache,
                                const ncm_kv_batch_t* batch, const uint16_t* k,
                                const uint16_t* v, int64_t k_stride, int64_t v_stride) {
    using namespace ncm;
    return move_rows<WriteArgs>(
        ctx, cache, batch, k, v, k_stride, v_stride, "kv_write",
        [&](const WriteArgs& a, uint32_t blocks, hipStream_t st) {
            by_codes(cache->codes, [&](auto c) {
                if (cache->head_dim == 128)
                    kv_write_kernel<128, decltype(c)::value><<<blocks, 256, 0, st>>>(a);
                else
                    kv_write_kernel<64, decltype(c)::value><<<blocks, 256, 0, st>>>(a);
            });
        });
}

extern "C" int ncm_kv_read_dev(ncm_ctx_t* ctx, const ncm_kv_cache_t* cache,
                               const ncm_kv_batch_t* batch, uint16_t* k, uint16_t* v,
                               int64_t k_stride, int64_t v_stride) {
    using namespace ncm;
    return move_rows<ReadArgs>(
        ctx, cache, batch, k, v, k_stride, v_stride, "kv_read",
        [&](const ReadArgs& a, uint32_t blocks, hipStream_t st) {
            by_codes(cache->codes, [&](auto c) {
                if (cache->head_dim == 128)
                    kv_read_kernel<128, decltype(c)::value><<<blocks, 256, 0, st>>>(a);
                else
                    kv_read_kernel<64, decltype(c)::value><<<blocks, 256, 0, st>>>(a);
            });
        });
}
