// The paged K/V cache: writing a step's K and V rows, quantised
// (ncm_kv_write_dev), and reading them back (ncm_kv_read_dev).
//
// A head of a token is head_dim / 8 lanes of eight values each. fp8 scales are
// powers of two: they cost a floating format no precision, and make both
// x / scale and, in bf16, code * scale exact. int8 codes are rint(x * 127 / m)
// of a correctly rounded quotient of exact operands (a bf16 value times 127 has
// 15 bits), so x = m / 2, a tie, rounds as it does in real numbers.
//
// Memory bound: a bf16 value in and its code out, or the other way. 14720 rows of
// 8 heads of 128, e4m3: written in 23 us (4.0 TB/s of values, codes and scales),
// read in 19 (4.9).
#include "step.h"

namespace ncm {
namespace {

// Where a row's token lies: its page, -1 where the token is not there, and its
// place in the page; page kNobody where the row is no request's.
constexpr int kNobody = -2;
struct Place {
    int page, at;
};

// By a whole wavefront: the request of a row is the number of requests that end
// at or before it, 64 of them a step.
__device__ __forceinline__ Place place_of(const BatchView& b, const KvView& c, int row, int lane) {
    int r = 0;
    for (int j = 0; j < b.requests; j += 64)
        r += __popcll(__ballot(j + lane < b.requests && b.offsets[min(j + lane, b.requests - 1) + 1] <= row));
    if (r >= b.requests) return {kNobody, 0};
    const Request q = request_of(b, r);
    if (row < q.o0 || row >= q.o0 + q.n) return {kNobody, 0};
    const int64_t t = (int64_t)q.before + (row - q.o0);
    return {page_of(b, c, r, t), (int)(t & ((1 << c.page_log2) - 1))};
}

// A workgroup moves ROWS rows: their places first, a wavefront each, then their
// heads, HD / 8 lanes each, K's and V's of a row after one another. f(row,
// place, is_v, head, lane of the head).
template <int HD, int ROWS, typename F>
__device__ __forceinline__ void for_heads(const BatchView& b, const KvView& c, F f) {
    __shared__ Place places[ROWS];
    constexpr int LANES = HD / 8;
    const int tid = threadIdx.x, first = (int)blockIdx.x * ROWS, heads = c.kv_heads;
    for (int i = tid >> 6; i < ROWS; i += 4)
        if (first + i < b.rows) {
            const Place p = place_of(b, c, first + i, tid & 63);
            if ((tid & 63) == 0) places[i] = p;
        }
    __syncthreads();
    const int lane = tid % LANES, items = min(ROWS, b.rows - first) * 2 * heads;
    int i = 0, which = tid / LANES;
    while (which >= 2 * heads) which -= 2 * heads, ++i;
    for (int item = tid / LANES; item < items; item += 256 / LANES) {
        const Place p = places[i];
        const bool is_v = which >= heads;
        if (p.page != kNobody) f(first + i, p, is_v, is_v ? which - heads : which, lane);
        which += 256 / LANES;
        while (which >= 2 * heads) which -= 2 * heads, ++i;
    }
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

// One head of one row.
template <int HD, int CODES>
__device__ __forceinline__ void write_head(const WriteArgs& a, int row, Place p, bool is_v, int h,
                                           int lane) {
    constexpr int LANES = HD / 8;
    const uint16_t* src =
        (is_v ? a.v + row * a.v_stride : a.k + row * a.k_stride) + h * HD + 8 * lane;
    const u32x4_t w = *(const u32x4_t*)src;
    if (p.page < 0) return;
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
__device__ __forceinline__ void read_head(const ReadArgs& a, int row, Place p, bool is_v, int h,
                                          int lane) {
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

template <int HD, int CODES, int ROWS>
__global__ __launch_bounds__(256) void kv_write_kernel(WriteArgs a) {
    for_heads<HD, ROWS>(a.batch, a.cache, [&](int row, Place p, bool is_v, int h, int lane) {
        write_head<HD, CODES>(a, row, p, is_v, h, lane);
    });
}
template <int HD, int CODES, int ROWS>
__global__ __launch_bounds__(256) void kv_read_kernel(ReadArgs a) {
    for_heads<HD, ROWS>(a.batch, a.cache, [&](int row, Place p, bool is_v, int h, int lane) {
        read_head<HD, CODES>(a, row, p, is_v, h, lane);
    });
}

template <int HD, int CODES, int ROWS>
void start(const WriteArgs& a, uint32_t blocks, hipStream_t st) {
    kv_write_kernel<HD, CODES, ROWS><<<blocks, 256, 0, st>>>(a);
}
template <int HD, int CODES, int ROWS>
void start(const ReadArgs& a, uint32_t blocks, hipStream_t st) {
    kv_read_kernel<HD, CODES, ROWS><<<blocks, 256, 0, st>>>(a);
}

// Rows a workgroup: four where that leaves four workgroups a CU, for one search
// and its chain of loads for four times the bytes. One and four: 88 and 74 us for
// 53607 rows of 8 heads of 128, int8, read back (143 with a search by every head,
// 77 with eight rows), 25.5 and 23 for 14720 rows, e4m3, written (25 with eight);
// 3.6 and 6.3 us for 48 rows written.
template <int HD, int CODES, typename Args>
void start_rows(const Args& a, hipStream_t st) {
    const int64_t rows = a.batch.rows;
    if (rows >= 4 * 1024) start<HD, CODES, 4>(a, (uint32_t)((rows + 3) / 4), st);
    else start<HD, CODES, 1>(a, (uint32_t)rows, st);
}
template <int HD, typename Args>
void start_codes(const Args& a, int codes, hipStream_t st) {
    switch (codes) {
        case NCM_KV_BF16: start_rows<HD, NCM_KV_BF16>(a, st); break;
        case NCM_KV_FP8: start_rows<HD, NCM_KV_FP8>(a, st); break;
        default: start_rows<HD, NCM_KV_INT8>(a, st);
    }
}

// The checks and the launch of a write or a read.
template <typename Args, typename Ptr>
int move_rows(ncm_ctx_t* ctx, const ncm_kv_cache_t* cache, const ncm_kv_batch_t* batch, Ptr k,
              Ptr v, int64_t k_stride, int64_t v_stride, const char* what) {
    if (!ctx) return NCM_E_NULL;
    Args a;
    int rc = check_cache(cache, &a.cache);
    if (rc) return rc;
    rc = check_batch(batch, a.cache.page_log2, &a.batch);
    if (rc) return rc;
    if (batch->rows > 4 * kMaxBlocks) return NCM_E_SHAPE;  // four rows a workgroup
    if (batch->rows == 0 || batch->requests == 0) return NCM_OK;
    const int64_t width = (int64_t)cache->kv_heads * cache->head_dim;
    rc = check_rows(k, k_stride, width);
    if (!rc) rc = check_rows(v, v_stride, width);
    if (rc) return rc;
    a.k = k, a.v = v, a.k_stride = k_stride, a.v_stride = v_stride;
    const DeviceScope scope(ncm_ctx_device(ctx));
    rc = step_hip(scope.error(), what);
    if (rc) return rc;
    if (cache->head_dim == 128) start_codes<128>(a, cache->codes, ncm_ctx_stream(ctx));
    else start_codes<64>(a, cache->codes, ncm_ctx_stream(ctx));
    return step_hip(hipGetLastError(), what);
}

}  // namespace
}  // namespace ncm

extern "C" int ncm_kv_write_dev(ncm_ctx_t* ctx, const ncm_kv_cache_t* cache,
                                const ncm_kv_batch_t* batch, const uint16_t* k,
                                const uint16_t* v, int64_t k_stride, int64_t v_stride) {
    return ncm::move_rows<ncm::WriteArgs>(ctx, cache, batch, k, v, k_stride, v_stride, "kv_write");
}

extern "C" int ncm_kv_read_dev(ncm_ctx_t* ctx, const ncm_kv_cache_t* cache,
                               const ncm_kv_batch_t* batch, uint16_t* k, uint16_t* v,
                               int64_t k_stride, int64_t v_stride) {
    return ncm::move_rows<ncm::ReadArgs>(ctx, cache, batch, k, v, k_stride, v_stride, "kv_read");
}
