// Shared by the entry points that continue sequences (rope_positions.hip,
// kv_cache.hip, kv_attention.hip, logits.hip): the device's view of a paged
// cache and of a step's requests, and the host side's checks of both.
#pragma once

#include <string>

#include "common.h"
#include "status.h"

hipStream_t ncm_ctx_stream(ncm_ctx_t* ctx);
int ncm_ctx_device(ncm_ctx_t* ctx);

namespace ncm {

// The context's device for the length of a call; the calling thread's own
// device is current again afterwards, so a call for another device leaves the
// caller's allocations and streams where they were.
class DeviceScope {
  public:
    explicit DeviceScope(int device) {
        err_ = hipGetDevice(&before_);
        if (err_ == hipSuccess && before_ != device) {
            err_ = hipSetDevice(device);
            moved_ = err_ == hipSuccess;
        }
    }
    ~DeviceScope() {
        if (moved_) (void)hipSetDevice(before_);
    }
    DeviceScope(const DeviceScope&) = delete;
    DeviceScope& operator=(const DeviceScope&) = delete;
    hipError_t error() const { return err_; }

  private:
    hipError_t err_ = hipSuccess;
    int before_ = 0;
    bool moved_ = false;
};

inline int step_hip(hipError_t e, const char* what) {
    if (e == hipSuccess) return NCM_OK;
    ncm_set_error_detail(std::string(what) + ": " + hipGetErrorString(e));
    return NCM_E_HIP;
}

// A cache as the kernels take it: bases, strides in elements, log2 page size.
struct KvView {
    char* k;
    char* v;
    float* ks;
    float* vs;
    int64_t k_stride, v_stride, ks_stride, vs_stride;
    int32_t pages, kv_heads, page_log2;
};

// A step's requests; width counts tokens that the table reaches.
struct BatchView {
    const int32_t* offsets;
    const int32_t* starts;
    const int32_t* table;
    int64_t table_stride;
    int64_t capacity;
    int32_t requests;
    int32_t rows;
};

// Request r's rows [o0, o0 + n) and the tokens before them.
struct Request {
    int32_t o0, n;
    int32_t before;
};

__device__ __forceinline__ Request request_of(const BatchView& b, int r) {
    Request q;
    q.o0 = min(max(b.offsets[r], 0), b.rows);
    q.n = max(min(b.offsets[r + 1], b.rows) - q.o0, 0);
    q.before = max(b.starts[r], 0);
    return q;
}

// The page of token t of request r, or -1 where the token is not there.
__device__ __forceinline__ int page_of(const BatchView& b, const KvView& c, int64_t r,
                                       int64_t t) {
    if (t >= b.capacity) return -1;
    const int id = b.table[r * b.table_stride + (t >> c.page_log2)];
    return (uint32_t)id < (uint32_t)c.pages ? id : -1;
}

constexpr int64_t kMaxRequests = 65535;
constexpr int64_t kMaxRows = int64_t(1) << 30;
constexpr int64_t kMaxTokens = int64_t(1) << 30;  // of a sequence
constexpr int64_t kMaxThreads = 0xFFFFFFFF;       // of a launch, along x
constexpr int64_t kMaxBlocks = kMaxThreads / 256;

inline int check_cache(const ncm_kv_cache_t* c, KvView* view) {
    if (!c) return NCM_E_NULL;
    if (c->codes < NCM_KV_BF16 || c->codes > NCM_KV_INT8) return NCM_E_ARG;
    if (c->head_dim != 64 && c->head_dim != 128) return NCM_E_SHAPE;
    if (c->kv_heads < 1 || c->kv_heads > 4096 || c->pages < 1 || c->pages > 0x7FFFFFFF)
        return NCM_E_SHAPE;
    int log2 = 4;
    while (log2 < 10 && (1 << log2) != c->page_size) ++log2;
    if ((1 << log2) != c->page_size) return NCM_E_SHAPE;
    if (!c->k || !c->v) return NCM_E_NULL;
    const bool scaled = c->codes != NCM_KV_BF16;
    if (scaled != (c->k_scale != nullptr) || scaled != (c->v_scale != nullptr))
        return NCM_E_NULL;
    const int64_t rows = (int64_t)c->kv_heads * c->page_size, size = scaled ? 1 : 2;
    for (int64_t st : {c->k_stride, c->v_stride}) {
        if (st < rows * c->head_dim || st > (int64_t(1) << 40)) return NCM_E_SHAPE;
        if (st * size % 16) return NCM_E_ARG;
    }
    if ((uintptr_t)c->k % 16 || (uintptr_t)c->v % 16) return NCM_E_ARG;
    if (scaled) {
        for (int64_t st : {c->k_scale_stride, c->v_scale_stride}) {
            if (st < rows || st > (int64_t(1) << 40)) return NCM_E_SHAPE;
            if (st % 4) return NCM_E_ARG;
        }
        if ((uintptr_t)c->k_scale % 16 || (uintptr_t)c->v_scale % 16) return NCM_E_ARG;
    }
    if (view)
        *view = {(char*)c->k, (char*)c->v, c->k_scale, c->v_scale, c->k_stride, c->v_stride,
                 c->k_scale_stride, c->v_scale_stride, (int32_t)c->pages, c->kv_heads, log2};
    return NCM_OK;
}

inline int check_batch(const ncm_kv_batch_t* b, int page_log2, BatchView* view) {
    if (!b) return NCM_E_NULL;
    if (b->requests < 0 || b->requests > kMaxRequests || b->rows < 0 || b->rows > kMaxRows ||
        b->table_width < 0 || b->table_width > 0x7FFFFFFF || b->table_stride < b->table_width ||
        b->table_stride > (int64_t(1) << 40) || b->table_width << page_log2 > kMaxTokens)
        return NCM_E_SHAPE;
    if (b->requests > 0 && b->rows > 0 &&
        (!b->offsets || !b->starts || (!b->page_table && b->table_width > 0)))
        return NCM_E_NULL;
    if (view)
        *view = {b->offsets, b->starts, b->page_table, b->table_stride,
                 b->table_width << page_log2, (int32_t)b->requests, (int32_t)b->rows};
    return NCM_OK;
}

// Rows of `heads` heads of a step's tensor for the 16-byte accesses.
inline int check_rows(const void* p, int64_t stride, int64_t width) {
    if (stride < width || stride > (int64_t(1) << 40)) return NCM_E_SHAPE;
    if (!p) return NCM_E_NULL;
    if (stride % 8 || (uintptr_t)p % 16) return NCM_E_ARG;
    return NCM_OK;
}

}  // namespace ncm
