// Rotation of q and k heads at given positions (ncm_rope_positions_dev).
//
// The angle is formed in 64 bits, in turns: t = position * inv_freq / 2 pi,
// less its nearest integer, so a position of a million keeps an angle good to
// 1e-10 turns (a 32-bit product would be off by up to 0.01). What is left of
// it, less the nearest quarter turn, is at most pi / 4, where the Taylor sums
// of sine and cosine to x^9 and x^10 are exact to 2^-25. Pairs are turned in
// fp32 with one rounding at the end.
//
// Memory bound: rows * heads * head_dim values in and out. A thread turns 32
// bytes of one head, sines and all: sharing them among eight heads of a row gave
// nothing for 8192 rows of 40 heads of 128, bf16, interleaved (33.3 us, 5.0 TB/s; a
// copy runs at 5.1), and took 6.6 us against 3.5 for 4 rows.
#include "step.h"

namespace ncm {
namespace {

__device__ __forceinline__ void sincos_turns(double turns, float scale, float& c, float& s) {
    const double r = turns - rint(turns);
    const double n = rint(4.0 * r);
    const float x = (float)((r - 0.25 * n) * 6.283185307179586);
    const float x2 = x * x;
    // Taylor: sin x = x - x^3/3! + ... + x^9/9!, cos x = 1 - x^2/2! + ... - x^10/10!.
    float a = 2.7557319e-6f;
    a = fmaf(a, x2, -1.9841270e-4f);
    a = fmaf(a, x2, 8.3333333e-3f);
    a = fmaf(a, x2, -0.16666667f);
    const float sn = fmaf(a * x2, x, x);
    float b = -2.7557319e-7f;
    b = fmaf(b, x2, 2.4801587e-5f);
    b = fmaf(b, x2, -1.3888889e-3f);
    b = fmaf(b, x2, 4.1666667e-2f);
    b = fmaf(b, x2, -0.5f);
    const float cs = fmaf(b, x2, 1.0f);
    const int q = (int)n & 3;
    const float u = (q & 1) ? cs : sn, v = (q & 1) ? sn : cs;
    s = scale * ((q & 2) ? -u : u);
    c = scale * ((q == 1 || q == 2) ? -v : v);
}

struct RopeArgs {
    const void* x;
    void* y;
    const int32_t* positions;
    const float* inv_freq;
    int64_t rows, x_stride, y_stride;
    int heads, head_dim, half;
    int units;        // threads that cover a head: turned ones, then copied ones
    int turn_units;
    float scale;
};

// Sixteen bytes of a head as floats.
template <bool BF16> struct Vec;
template <> struct Vec<true> {
    static constexpr int N = 8;
    typedef uint16_t elem;
    static __device__ __forceinline__ void load(const uint16_t* p, float (&f)[8]) {
        const u32x4_t w = *(const u32x4_t*)p;
#pragma unroll
        for (int i = 0; i < 4; ++i) f[2 * i] = bf16_lo_to_f32(w[i]), f[2 * i + 1] = bf16_hi_to_f32(w[i]);
    }
    static __device__ __forceinline__ void store(uint16_t* p, const float (&f)[8]) {
        u32x4_t w;
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = bf16x2_bits_rne(f[2 * i], f[2 * i + 1]);
        *(u32x4_t*)p = w;
    }
    static __device__ __forceinline__ float get(const uint16_t* p) {
        return __uint_as_float((uint32_t)*p << 16);
    }
    static __device__ __forceinline__ void put(uint16_t* p, float v) { *p = (uint16_t)bf16_bits_rne(v); }
};
template <> struct Vec<false> {
    static constexpr int N = 4;
    typedef float elem;
    static __device__ __forceinline__ void load(const float* p, float (&f)[4]) {
        const f32x4_t w = *(const f32x4_t*)p;
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = w[i];
    }
    static __device__ __forceinline__ void store(float* p, const float (&f)[4]) {
        f32x4_t w;
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = f[i];
        *(f32x4_t*)p = w;
    }
    static __device__ __forceinline__ float get(const float* p) { return *p; }
    static __device__ __forceinline__ void put(float* p, float v) { *p = v; }
};

// WIDE: a unit is two 16-byte pieces of a head, its first and second elements
// of N pairs (half layout) or 2 N neighbours (interleaved); copied units are
// one piece. Otherwise a unit is one pair, or one copied value.
template <bool BF16, bool INTERLEAVED, bool WIDE>
__global__ __launch_bounds__(256) void rope_positions_kernel(RopeArgs a) {
    typedef Vec<BF16> V;
    typedef typename V::elem T;
    constexpr int N = WIDE ? V::N : 1;
    // In 32 bits, whose division is far shorter: 33.5 us against 35.8.
    const uint32_t id = blockIdx.x * 256 + threadIdx.x, rest = id / (uint32_t)a.units;
    const int u = (int)(id % (uint32_t)a.units);
    const int64_t row = rest / (uint32_t)a.heads;
    if (row >= a.rows) return;
    const int64_t head = (int64_t)(rest % (uint32_t)a.heads) * a.head_dim;
    const T* x = (const T*)a.x + row * a.x_stride + head;
    T* y = (T*)a.y + row * a.y_stride + head;
    if (u >= a.turn_units) {  // behind the rotated part: copied
        const int at = 2 * a.half + (u - a.turn_units) * N;
        if constexpr (WIDE) *(u32x4_t*)(y + at) = *(const u32x4_t*)(x + at);
        else y[at] = x[at];
        return;
    }
    const int p0 = u * N;
    const double pos = (double)a.positions[row];
    float c[N], s[N];
#pragma unroll
    for (int i = 0; i < N; ++i)
        sincos_turns(pos * (double)a.inv_freq[p0 + i] * 0.15915494309189535, a.scale, c[i], s[i]);
    const int first = INTERLEAVED ? 2 * p0 : p0;
    const int second = INTERLEAVED ? (WIDE ? 2 * p0 + N : 2 * p0 + 1) : a.half + p0;
    if constexpr (WIDE) {
        float f[N], g[N];
        V::load(x + first, f);
        V::load(x + second, g);
        if constexpr (INTERLEAVED) {
#pragma unroll
            for (int i = 0; i < N / 2; ++i) {
                const float e = f[2 * i], d = f[2 * i + 1];
                f[2 * i] = fmaf(e, c[i], -(d * s[i]));
                f[2 * i + 1] = fmaf(d, c[i], e * s[i]);
                const int j = N / 2 + i;
                const float e2 = g[2 * i], d2 = g[2 * i + 1];
                g[2 * i] = fmaf(e2, c[j], -(d2 * s[j]));
                g[2 * i + 1] = fmaf(d2, c[j], e2 * s[j]);
            }
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float e = f[i], d = g[i];
                f[i] = fmaf(e, c[i], -(d * s[i]));
                g[i] = fmaf(d, c[i], e * s[i]);
            }
        }
        V::store(y + first, f);
        V::store(y + second, g);
    } else {
        const float e = V::get(x + first), d = V::get(x + second);
        V::put(y + first, fmaf(e, c[0], -(d * s[0])));
        V::put(y + second, fmaf(d, c[0], e * s[0]));
    }
}

template <bool BF16>
void launch(const RopeArgs& a, bool interleaved, bool wide, int64_t blocks, hipStream_t st) {
    const dim3 grid((uint32_t)blocks), block(256);
    if (interleaved)
        wide ? rope_positions_kernel<BF16, true, true><<<grid, block, 0, st>>>(a)
             : rope_positions_kernel<BF16, true, false><<<grid, block, 0, st>>>(a);
    else
        wide ? rope_positions_kernel<BF16, false, true><<<grid, block, 0, st>>>(a)
             : rope_positions_kernel<BF16, false, false><<<grid, block, 0, st>>>(a);
}

}  // namespace
}  // namespace ncm

extern "C" int ncm_rope_positions_dev(ncm_ctx_t* ctx, const void* x, void* y,
                                      const int32_t* positions, const float* inv_freq,
                                      int64_t rows, int heads, int head_dim, int rot_dim,
                                      int64_t x_stride, int64_t y_stride, int layout, float scale,
                                      int dtype) {
    using namespace ncm;
    if (!ctx) return NCM_E_NULL;
    if (rows < 0 || rows > kMaxRows || heads < 0 || heads > 65535 || head_dim <= 0 ||
        head_dim > 65536 || rot_dim <= 0 || rot_dim % 2 || rot_dim > head_dim)
        return NCM_E_SHAPE;
    const int64_t width = (int64_t)heads * head_dim;
    if (width > 0 && rows > (int64_t(1) << 32) / width) return NCM_E_SHAPE;
    if (x_stride < width || y_stride < width || x_stride > (int64_t(1) << 40) ||
        y_stride > (int64_t(1) << 40))
        return NCM_E_SHAPE;
    if (layout != NCM_ROPE_HALF && layout != NCM_ROPE_INTERLEAVED) return NCM_E_ARG;
    if (dtype != NCM_OUT_F32 && dtype != NCM_OUT_BF16) return NCM_E_ARG;
    if (rows == 0 || heads == 0) return NCM_OK;
    if (!x || !y || !positions || !inv_freq) return NCM_E_NULL;
    if (x == y && x_stride != y_stride) return NCM_E_ARG;
    const bool bf16 = dtype == NCM_OUT_BF16;
    const int n = bf16 ? 8 : 4, half = rot_dim / 2;
    const bool wide = !(((uintptr_t)x | (uintptr_t)y) % 16) && x_stride % n == 0 &&
                      y_stride % n == 0 && head_dim % n == 0 && half % n == 0;
    RopeArgs a = {x, y, positions, inv_freq, rows, x_stride, y_stride, heads, head_dim, half,
                  0, 0, scale};
    const int step = wide ? n : 1;
    a.turn_units = half / step;
    a.units = a.turn_units + (x == y ? 0 : (head_dim - rot_dim) / step);
    const int64_t blocks = (rows * a.units * heads + 255) / 256;
    const DeviceScope scope(ncm_ctx_device(ctx));
    int rc = step_hip(scope.error(), "rope_positions device");
    if (rc) return rc;
    const bool il = layout == NCM_ROPE_INTERLEAVED;
    if (bf16) launch<true>(a, il, wide, blocks, ncm_ctx_stream(ctx));
    else launch<false>(a, il, wide, blocks, ncm_ctx_stream(ctx));
    return step_hip(hipGetLastError(), "rope_positions launch");
}
