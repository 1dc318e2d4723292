// Attention of a step's rows over the paged cache (ncm_kv_attention_dev).
//
// One workgroup per row and query head: its four wavefronts take every fourth
// token, a lane two (head_dim 128) or one of its values, and keep a running
// maximum and sum of the softmax; the four are joined through LDS.
#include "step.h"

namespace ncm {
namespace {

struct AttnArgs {
    KvView cache;
    BatchView batch;
    const uint16_t* q;
    uint16_t* out;
    const int32_t* positions;
    const uint64_t* tree_mask;
    int64_t q_stride, out_stride, window, mask_words;
    float scale;
    int q_heads;
};

template <int CODES>
__device__ __forceinline__ float value_of(const char* p, int64_t i) {
    if constexpr (CODES == NCM_KV_BF16) return __uint_as_float((uint32_t)((const uint16_t*)p)[i] << 16);
    else if constexpr (CODES == NCM_KV_FP8) return __builtin_amdgcn_cvt_f32_fp8(((const uint8_t*)p)[i], 0);
    else return (float)((const int8_t*)p)[i];
}

template <int HD, int CODES>
__global__ __launch_bounds__(256) void kv_attention_kernel(AttnArgs a) {
    constexpr int PER = HD / 64;
    const int row = blockIdx.x, head = blockIdx.y, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int h = head / (a.q_heads / a.cache.kv_heads);
    int r = 0;
    for (int j = 0; j < a.batch.requests; ++j) r += a.batch.offsets[j + 1] <= row;
    if (r >= a.batch.requests) return;
    const Request rq = request_of(a.batch, r);
    if (row < rq.o0 || row >= rq.o0 + rq.n) return;
    const int i = row - rq.o0;
    const int64_t pos = a.positions ? max(a.positions[row], rq.before) : (int64_t)rq.before + i;
    float q[PER], o[PER];
    for (int d = 0; d < PER; ++d) {
        q[d] = __uint_as_float((uint32_t)a.q[row * a.q_stride + head * HD + lane + 64 * d] << 16);
        o[d] = 0.0f;
    }
    float m = -1e30f, l = 0.0f;
    for (int64_t t = wave; t < (int64_t)rq.before + rq.n; t += 4) {
        const int64_t j = t - rq.before;
        bool see;
        if (j < 0 || !a.tree_mask) see = j <= i && (a.window <= 0 || t > pos - a.window);
        else see = (j >> 6) < a.mask_words &&
                   ((a.tree_mask[row * a.mask_words + (j >> 6)] >> (j & 63)) & 1u);
        if (!see) continue;
        const int page = page_of(a.batch, a.cache, r, t);
        if (page < 0) continue;
        const int64_t in_page = ((int64_t)h << a.cache.page_log2) + (t & ((1 << a.cache.page_log2) - 1));
        const int64_t kb = page * a.cache.k_stride + in_page * HD, vb = page * a.cache.v_stride + in_page * HD;
        float s = 0.0f;
        for (int d = 0; d < PER; ++d) s = fmaf(q[d], value_of<CODES>(a.cache.k, kb + lane + 64 * d), s);
        s = wave_sum_xor(s) * a.scale;
        float vs = 1.0f;
        if constexpr (CODES != NCM_KV_BF16) {
            s *= a.cache.ks[page * a.cache.ks_stride + in_page];
            vs = a.cache.vs[page * a.cache.vs_stride + in_page];
        }
        const float mn = fmaxf(m, s), al = expf(m - mn), p = expf(s - mn);
        l = l * al + p;
        for (int d = 0; d < PER; ++d)
            o[d] = fmaf(p * vs, value_of<CODES>(a.cache.v, vb + lane + 64 * d), o[d] * al);
        m = mn;
    }
    __shared__ float sm[4], sl[4], so[4][HD];
    if (lane == 0) sm[wave] = m, sl[wave] = l;
    for (int d = 0; d < PER; ++d) so[wave][lane + 64 * d] = o[d];
    __syncthreads();
    if (threadIdx.x >= HD) return;
    const float top = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
    float total = 0.0f, acc = 0.0f;
    for (int w = 0; w < 4; ++w) {
        const float f = expf(sm[w] - top);
        total = fmaf(sl[w], f, total);
        acc = fmaf(so[w][threadIdx.x], f, acc);
    }
    a.out[row * a.out_stride + head * HD + threadIdx.x] =
        (uint16_t)bf16_bits_rne(total == 0.0f ? 0.0f : acc / total);
}

int check_attention(const ncm_kv_cache_t* cache, const ncm_kv_batch_t* batch, int q_heads,
                    AttnArgs* a) {
    int rc = check_cache(cache, &a->cache);
    if (rc) return rc;
    rc = check_batch(batch, a->cache.page_log2, &a->batch);
    if (rc) return rc;
    if (q_heads < 1 || q_heads > 65535 || q_heads % cache->kv_heads) return NCM_E_SHAPE;
    a->q_heads = q_heads;
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
    return check_attention(cache, batch, q_heads, &a);
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
    if (window < 0 || mask_words < 0 || mask_words > kMaxRows) return NCM_E_SHAPE;
    if (batch->rows == 0 || batch->requests == 0) return NCM_OK;
    const int64_t width = (int64_t)q_heads * cache->head_dim;
    rc = check_rows(q, q_stride, width);
    if (!rc) rc = check_rows(out, out_stride, width);
    if (rc) return rc;
    a.q = q, a.out = out, a.positions = positions, a.tree_mask = tree_mask;
    a.q_stride = q_stride, a.out_stride = out_stride, a.window = window;
    a.mask_words = mask_words, a.scale = scale;
    const DeviceScope scope(ncm_ctx_device(ctx));
    rc = step_hip(scope.error(), "kv_attention device");
    if (rc) return rc;
    const hipStream_t st = ncm_ctx_stream(ctx);
    const dim3 grid((uint32_t)batch->rows, (uint32_t)q_heads);
    const bool wide = cache->head_dim == 128;
    switch (cache->codes) {
        case NCM_KV_BF16:
            wide ? kv_attention_kernel<128, NCM_KV_BF16><<<grid, 256, 0, st>>>(a)
                 : kv_attention_kernel<64, NCM_KV_BF16><<<grid, 256, 0, st>>>(a);
            break;
        case NCM_KV_FP8:
            wide ? kv_attention_kernel<128, NCM_KV_FP8><<<grid, 256, 0, st>>>(a)
                 : kv_attention_kernel<64, NCM_KV_FP8><<<grid, 256, 0, st>>>(a);
            break;
        default:
            wide ? kv_attention_kernel<128, NCM_KV_INT8><<<grid, 256, 0, st>>>(a)
                 : kv_attention_kernel<64, NCM_KV_INT8><<<grid, 256, 0, st>>>(a);
    }
    return step_hip(hipGetLastError(), "kv_attention launch");
}
