// Products with 4-bit weights (ncm_linear_int4) and what makes them.
//
//   y[m, n] = sum_g s[n, g] sum_{k in g} (q[n, k] - z[n, g]) x[m, k]
//
// A code becomes the bf16 value 128 + q by setting its four bits into 0x4300,
// one operation for two codes, and enters v_mfma_f32_16x16x32_bf16 with the
// bf16 rows of x, weights the rows and tokens the columns of the product. A
// product with ones gives the sum of x over the same k, so that per group
//   y += s (sum (128 + q) x - (128 + z) sum x)
// in fp32: scales and zero points meet fp32 sums, and nothing is rounded to 16
// bits but the output. The difference costs a factor of 143 / 8 of the rounding
// of a plain fp32 sum at most.
//
// Bound by the weights' bytes for few rows. They are packed once in the order
// of the lanes: 16 outputs and 128 inputs are 1 KB, a wavefront's 16-byte load.
// A workgroup makes 16 outputs of up to 16 rows, its eight wavefronts taking
// every eighth 128 inputs; their sums are added in order through LDS. 28672 x 4096
// in groups of 128, weights from HBM: one row 17 us (3.6 TB/s), 4 rows 21, 8 26; in
// groups of 32 with zeros, a scale and two fp32 operations an output, row and group:
// 19, 24 and 27. More rows (linear_int4_rows_kernel; here from 10 on) are bound by the
// unpacking and the group sums, repeated for every 32 rows: 16 rows 24 and 30 us, 256
// rows 112 (540 TFLOP/s) and 149.
#include "step.h"

namespace ncm {
namespace {

constexpr int kWaves = 8;

struct Int4Args {
    const uint16_t* x;
    const u32x4_t* codes;
    const char* scales;
    const uint16_t* bias;
    const float* residual;
    void* y;
    int64_t x_stride;
    int m, n, k, blocks;  // of 128 inputs
    bool wide;            // 4 outputs of a row in one access
    float* parts;         // [splits][m][n] where the inputs are split, else NULL
    int splits;
};

// Scales of 16 outputs, a block of 128 inputs: [128 / GROUP][16], two bytes, or
// with zero points four: 128 + z in the low half, both bf16.
template <int GROUP, bool ZEROS>
constexpr int scale_bytes() { return 128 / GROUP * 16 * (ZEROS ? 4 : 2); }

// What a wavefront loads of 128 inputs.
template <bool HELD>
struct Stage {
    u32x4_t w;
    u32x4_t x[HELD ? 1 : 4];
    uint32_t s;  // a dword of the tile's scales, by lane
};

// Four outputs of a row, from column `col` on.
template <int OUT>
__device__ __forceinline__ void store_block(const Int4Args& a, f32x4_t v, int row, int64_t col) {
    if (row >= a.m) return;
    int64_t at = (int64_t)row * a.n + col;
    const int left = (int)min((int64_t)4, a.n - col);
    if (left <= 0) return;
    if (a.wide) {
        if (a.bias) {
            const u32x2_t bits = *(const u32x2_t*)(a.bias + col);
#pragma unroll
            for (int j = 0; j < 4; ++j)
                v[j] += __uint_as_float(j % 2 ? bits[j / 2] & 0xFFFF0000u : bits[j / 2] << 16);
        }
        if (a.residual) v += *(const f32x4_t*)(a.residual + at);
        if constexpr (OUT == NCM_OUT_BF16) {
            *(u32x2_t*)((uint16_t*)a.y + at) =
                u32x2_t{bf16x2_bits_rne(v[0], v[1]), bf16x2_bits_rne(v[2], v[3])};
        } else {
            if constexpr (OUT == NCM_OUT_BF16_F32)
#pragma unroll
                for (int j = 0; j < 4; ++j) v[j] = __uint_as_float(bf16_bits_rne(v[j]) << 16);
            *(f32x4_t*)((float*)a.y + at) = v;
        }
    } else {
        for (int j = 0; j < left; ++j) {
            float f = v[j];
            if (a.bias) f += __uint_as_float((uint32_t)a.bias[col + j] << 16);
            if (a.residual) f += a.residual[at + j];
            if constexpr (OUT == NCM_OUT_BF16) ((uint16_t*)a.y)[at + j] = (uint16_t)bf16_bits_rne(f);
            else ((float*)a.y)[at + j] =
                OUT == NCM_OUT_F32 ? f : __uint_as_float(bf16_bits_rne(f) << 16);
        }
    }
}

// DEPTH: blocks of 128 inputs that a wavefront loads ahead. HELD: all of x is in
// LDS, [m][blocks][16] chunks, which leaves registers for more wavefronts.
template <int GROUP, bool ZEROS, int DEPTH, bool HELD, int OUT>
__global__ __launch_bounds__(64 * kWaves) void linear_int4_kernel(Int4Args a) {
    typedef Stage<HELD> S;
    constexpr int G = 128 / GROUP, STEPS = 4 / G;  // MFMA steps of a group
    constexpr int SB = scale_bytes<GROUP, ZEROS>() / 4;
    __shared__ f32x4_t parts[kWaves][64];
    // Each wavefront's scales on their way from one coalesced load to the lanes
    // that need them (loaded by those lanes: 36 us in place of 25 for 28672 x 4096
    // in groups of 32 with zero points).
    __shared__ __attribute__((aligned(16))) uint32_t scales[kWaves][SB];
    extern __shared__ u32x4_t held[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c = lane & 15, g = lane >> 4;
    const int64_t tile = blockIdx.x;

    auto load = [&](S& s, int b) {
        const int64_t at = tile * a.blocks + b;
        s.w = a.codes[at * 64 + lane];
        s.s = ((const uint32_t*)a.scales)[at * SB + min(lane, SB - 1)];
        if constexpr (!HELD)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int k = 128 * b + 32 * i + 8 * g;
                s.x[i] = u32x4_t{0, 0, 0, 0};
                if (c < a.m && k < a.k) s.x[i] = *(const u32x4_t*)(a.x + c * a.x_stride + k);
            }
    };

    f32x4_t sum = {0.0f, 0.0f, 0.0f, 0.0f};
    const u32x4_t one_bits = {0x3F803F80u, 0x3F803F80u, 0x3F803F80u, 0x3F803F80u};
    const bf16x8_t ones = __builtin_bit_cast(bf16x8_t, one_bits);
    auto add = [&](const S& s, int b) {
        bf16x8_t x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (HELD) {
                u32x4_t bits = {0, 0, 0, 0};
                if (c < a.m) bits = held[(c * a.blocks + b) * 16 + 4 * i + g];
                x[i] = __builtin_bit_cast(bf16x8_t, bits);
            } else {
                x[i] = __builtin_bit_cast(bf16x8_t, s.x[i]);
            }
        }
        if (lane < SB) scales[wave][lane] = s.s;
#pragma unroll
        for (int i = 0; i < G; ++i) {
            f32x4_t of_x = {0.0f, 0.0f, 0.0f, 0.0f}, of_q = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int e = STEPS * i; e < STEPS * (i + 1); ++e) {
                of_x = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, x[e], of_x, 0, 0, 0);
                u32x4_t q;
#pragma unroll
                for (int j = 0; j < 4; ++j) q[j] = ((s.w[e] >> (4 * j)) & 0x000F000Fu) | 0x43004300u;
                of_q = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, q), x[e], of_q,
                                                               0, 0, 0);
            }
            const uint32_t* words = &scales[wave][i * (ZEROS ? 16 : 8) + g * (ZEROS ? 4 : 2)];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t word = words[ZEROS ? j : j / 2];
                const float scale = __uint_as_float(!ZEROS && j % 2 == 0 ? word << 16 : word & 0xFFFF0000u);
                const float zero = ZEROS ? __uint_as_float(word << 16) : 136.0f;
                sum[j] = fmaf(scale, fmaf(-zero, of_x[j], of_q[j]), sum[j]);
            }
        }
        asm volatile("" ::: "memory");  // the next block's scales stay behind these reads
    };

    S now[DEPTH], next[DEPTH];
#pragma unroll
    for (int i = 0; i < DEPTH; ++i)
        if (wave + i * kWaves < a.blocks) load(now[i], wave + i * kWaves);
    if constexpr (HELD) {
        for (int i = threadIdx.x; i < a.m * a.blocks * 16; i += 64 * kWaves) {
            const int row = i / (a.blocks * 16), k = 8 * (i - row * a.blocks * 16);
            held[i] = k < a.k ? *(const u32x4_t*)(a.x + row * a.x_stride + k) : u32x4_t{0, 0, 0, 0};
        }
        lds_barrier();
    }
    for (int b = wave; b < a.blocks; b += DEPTH * kWaves) {
#pragma unroll
        for (int i = 0; i < DEPTH; ++i) {
            const int after = b + (DEPTH + i) * kWaves;
            if (after < a.blocks) load(next[i], after);
        }
#pragma unroll
        for (int i = 0; i < DEPTH; ++i)
            if (b + i * kWaves < a.blocks) add(now[i], b + i * kWaves);
#pragma unroll
        for (int i = 0; i < DEPTH; ++i) now[i] = next[i];
    }

    parts[wave][lane] = sum;
    __syncthreads();
    if (wave > 0) return;
    f32x4_t v = parts[0][lane];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) {
        const f32x4_t p = parts[w][lane];
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = v[j] + p[j];
    }
    store_block<OUT>(a, v, c, tile * 16 + 4 * g);
}

// More rows, 32 a workgroup: they are shared by NW wavefronts of 32 outputs each,
// in LDS, and 8 / NW sets of these take every 8 / NW-th 128 inputs. Weights go from
// memory to registers a block ahead; scales through LDS, which gives each lane its
// four outputs' without 64 registers for them. 16-byte chunk c of row r of x is at
// chunk c ^ (r % 16), so that an operand's sixteen rows fall into different banks.
// 32 rows leave room for two workgroups a CU, of which one computes while the other
// waits: 28672 x 4096 in groups of 128, 256 rows 112 us, 136 with 64 rows a
// workgroup and half the reads of the weights; 96 rows 55, 67; 4096 x 14336,
// 128 rows 36.5, 43.
constexpr int kRowsOf = 32;
template <int GROUP, bool ZEROS, int OUT>
__global__ __launch_bounds__(512, 2) void linear_int4_rows_kernel(Int4Args a) {
    constexpr int NW = 4, KW = 8 / NW, G = 128 / GROUP, STEPS = 4 / G, NT = 2;
    constexpr int ROWS = kRowsOf, MT = ROWS / 16;
    constexpr int SB = scale_bytes<GROUP, ZEROS>() / 4;  // dwords of a tile's block
    constexpr int PER = KW * ROWS * 16 / 512;            // chunks of x a thread brings
    __shared__ u32x4_t xs[2][KW][ROWS][16];
    __shared__ __attribute__((aligned(16))) uint32_t scales[2][8][NT * SB];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int c = lane & 15, g = lane >> 4, nw = wave % NW, kw = wave / NW;
    const int64_t tile0 = ((int64_t)blockIdx.x * NW + nw) * NT;
    const int tiles = (a.n + 15) / 16, m0 = blockIdx.y * ROWS;
    // The workgroup's steps of KW blocks.
    const int all = (a.blocks + KW - 1) / KW;
    const int step0 = (int)((int64_t)all * blockIdx.z / a.splits);
    const int steps = (int)((int64_t)all * (blockIdx.z + 1) / a.splits) - step0;

    u32x4_t w[NT], x[PER];
    uint32_t s[(NT * SB + 63) / 64];
    auto load_w = [&](int step) {
        const int b = min((step0 + step) * KW + kw, a.blocks - 1);
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const int64_t at = min(tile0 + t, (int64_t)tiles - 1) * a.blocks + b;
            w[t] = a.codes[at * 64 + lane];
        }
#pragma unroll
        for (int i = 0; i < (NT * SB + 63) / 64; ++i) {
            const int d = min(i * 64 + lane, NT * SB - 1);
            const int64_t at = min(tile0 + d / SB, (int64_t)tiles - 1) * a.blocks + b;
            s[i] = ((const uint32_t*)a.scales)[at * SB + d % SB];
        }
    };
    auto load_x = [&](int step) {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int chunk = tid + 512 * i, row = chunk / 16 % ROWS, set = chunk / (16 * ROWS);
            const int64_t k = 128 * ((int64_t)(step0 + step) * KW + set) + 8 * (chunk % 16);
            x[i] = u32x4_t{0, 0, 0, 0};
            if (m0 + row < a.m && k < a.k) x[i] = *(const u32x4_t*)(a.x + (m0 + row) * a.x_stride + k);
        }
    };
    auto put = [&](int buffer) {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int chunk = tid + 512 * i, row = chunk / 16 % ROWS, set = chunk / (16 * ROWS);
            xs[buffer][set][row][(chunk ^ row) & 15] = x[i];
        }
#pragma unroll
        for (int i = 0; i < (NT * SB + 63) / 64; ++i)
            if (i * 64 + lane < NT * SB) scales[buffer][wave][i * 64 + lane] = s[i];
    };

    f32x4_t sum[NT][MT];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int r = 0; r < MT; ++r) sum[t][r] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
    const u32x4_t one_bits = {0x3F803F80u, 0x3F803F80u, 0x3F803F80u, 0x3F803F80u};
    const bf16x8_t ones = __builtin_bit_cast(bf16x8_t, one_bits);

    load_w(0);
    load_x(0);
    put(0);
    u32x4_t now[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) now[t] = w[t];
    if (steps > 1) load_w(1), load_x(1);
    lds_barrier();
    for (int step = 0; step < steps; ++step) {
        const int b = step & 1;
        if ((step0 + step) * KW + kw < a.blocks) {
#pragma unroll
            for (int i = 0; i < G; ++i) {
                f32x4_t of_x[MT], of_q[NT][MT];
#pragma unroll
                for (int r = 0; r < MT; ++r) {
                    of_x[r] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int t = 0; t < NT; ++t) of_q[t][r] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
                }
#pragma unroll
                for (int e = STEPS * i; e < STEPS * (i + 1); ++e) {
                    bf16x8_t q[NT];
#pragma unroll
                    for (int t = 0; t < NT; ++t) {
                        u32x4_t bits;
#pragma unroll
                        for (int j = 0; j < 4; ++j) bits[j] = ((now[t][e] >> (4 * j)) & 0x000F000Fu) | 0x43004300u;
                        q[t] = __builtin_bit_cast(bf16x8_t, bits);
                    }
#pragma unroll
                    for (int r = 0; r < MT; ++r) {
                        const bf16x8_t rows =
                            __builtin_bit_cast(bf16x8_t, xs[b][kw][16 * r + c][(4 * e + g) ^ c]);
                        of_x[r] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, rows, of_x[r], 0, 0, 0);
#pragma unroll
                        for (int t = 0; t < NT; ++t)
                            of_q[t][r] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(q[t], rows, of_q[t][r], 0, 0, 0);
                    }
                }
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    const uint32_t* p = &scales[b][wave][t * SB + i * (ZEROS ? 16 : 8) + g * (ZEROS ? 4 : 2)];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const uint32_t word = p[ZEROS ? j : j / 2];
                        const float scale =
                            __uint_as_float(!ZEROS && j % 2 == 0 ? word << 16 : word & 0xFFFF0000u);
                        const float zero = ZEROS ? __uint_as_float(word << 16) : 136.0f;
#pragma unroll
                        for (int r = 0; r < MT; ++r)
                            sum[t][r][j] = fmaf(scale, fmaf(-zero, of_x[r][j], of_q[t][r][j]), sum[t][r][j]);
                    }
                }
            }
        }
        if (step + 1 < steps) {
            put(b ^ 1);
#pragma unroll
            for (int t = 0; t < NT; ++t) now[t] = w[t];
            if (step + 2 < steps) load_w(step + 2), load_x(step + 2);
        }
        lds_barrier();
    }
    // The sets' sums, added in order.
    f32x4_t* parts = (f32x4_t*)xs;
    static_assert(sizeof(xs) >= (KW - 1) * NW * NT * MT * 1024, "the other sets' sums");
    if (kw > 0)
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int r = 0; r < MT; ++r)
                parts[((((kw - 1) * NW + nw) * NT + t) * MT + r) * 64 + lane] = sum[t][r];
    __syncthreads();
    if (kw == 0)
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int r = 0; r < MT; ++r) {
                f32x4_t v = sum[t][r];
#pragma unroll
                for (int other = 0; other < KW - 1; ++other) {
                    const f32x4_t p = parts[(((other * NW + nw) * NT + t) * MT + r) * 64 + lane];
#pragma unroll
                    for (int j = 0; j < 4; ++j) v[j] = v[j] + p[j];
                }
                const int row = m0 + 16 * r + c;
                const int64_t col = (tile0 + t) * 16 + 4 * g;
                if (!a.parts) store_block<OUT>(a, v, row, col);
                else if (row < a.m) {
                    float* p = a.parts + ((int64_t)blockIdx.z * a.m + row) * a.n + col;
                    if (a.n % 4 == 0 && col < a.n) *(f32x4_t*)p = v;
                    else
                        for (int j = 0; j < min((int64_t)4, a.n - col); ++j) p[j] = v[j];
                }
            }
}

// The splits' sums, added in order.
template <int OUT>
__global__ __launch_bounds__(256) void linear_int4_join_kernel(Int4Args a) {
    const int64_t quads = (a.n + 3) / 4, i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= quads * a.m) return;
    const int row = (int)(i / quads);
    const int64_t col = (i - row * quads) * 4, at = (int64_t)row * a.n + col;
    f32x4_t v = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int s = 0; s < a.splits; ++s) {
        const float* p = a.parts + (int64_t)s * a.m * a.n + at;
        if (a.n % 4 == 0) {
            const f32x4_t x = *(const f32x4_t*)p;
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = v[j] + x[j];
        } else {
            for (int j = 0; j < min((int64_t)4, a.n - col); ++j) v[j] = v[j] + p[j];
        }
    }
    store_block<OUT>(a, v, row, col);
}

// Codes, a byte each, into the products' order; outputs past n and inputs past
// k as codes 0 with scales 0.
__global__ __launch_bounds__(256) void int4_pack_kernel(const uint8_t* codes, const uint16_t* scales,
                                                        const uint8_t* zeros, int64_t n, int64_t k,
                                                        int group, int64_t blocks, uint32_t* to,
                                                        char* scales_to) {
    const int64_t block = (int64_t)blockIdx.x;  // 16 outputs, 128 inputs
    const int64_t tile = block / blocks, b = block - tile * blocks;
    const int lane = threadIdx.x & 63, e = threadIdx.x >> 6;
    const int64_t row = 16 * tile + (lane & 15), k0 = 128 * b + 32 * e + 8 * (lane >> 4);
    uint32_t word = 0;
    for (int i = 0; i < 8; ++i) {
        const uint32_t q = row < n && k0 + i < k ? codes[row * k + k0 + i] & 15u : 0u;
        word |= q << (4 * (i / 2) + 16 * (i % 2));
    }
    to[(block * 64 + lane) * 4 + e] = word;
    const int per = 128 / group, all = (int)((k + group - 1) / group);
    if ((int)threadIdx.x < per * 16) {
        const int i = threadIdx.x / 16;
        const int64_t r = 16 * tile + threadIdx.x % 16, at = b * per + i;
        const bool in = r < n && at < all;
        const uint32_t s = in ? scales[r * all + at] : 0u;
        const int64_t slot = block * per * 16 + threadIdx.x;
        if (zeros) {
            const float z = 128.0f + (in ? (float)(zeros[r * all + at] & 15) : 0.0f);
            ((uint32_t*)scales_to)[slot] = s << 16 | __float_as_uint(z) >> 16;
        } else {
            ((uint16_t*)scales_to)[slot] = (uint16_t)s;
        }
    }
}

// A wavefront per group of a row.
__global__ __launch_bounds__(256) void int4_quantise_kernel(const uint16_t* w, int64_t n, int64_t k,
                                                            int64_t stride, int group, uint8_t* codes,
                                                            uint16_t* scales, uint8_t* zeros) {
    const int64_t all = (k + group - 1) / group;
    const int64_t at = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    if (at >= n * all) return;
    const int64_t row = at / all, k0 = (at - row * all) * group;
    const int len = (int)min((int64_t)group, k - k0);
    float v[2], lo = 0.0f, hi = 0.0f;
    bool bad = false;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int j = lane + 64 * i;
        v[i] = j < len ? __uint_as_float((uint32_t)w[row * stride + k0 + j] << 16) : 0.0f;
        bad |= !(fabsf(v[i]) <= 3.40282347e38f);
        lo = fminf(lo, v[i]), hi = fmaxf(hi, v[i]);
    }
    for (int x = 32; x; x >>= 1) lo = fminf(lo, __shfl_xor(lo, x)), hi = fmaxf(hi, __shfl_xor(hi, x));
    bad = __any(bad);
    // Divided before they are added: the range of the largest values has no float.
    const float unit = zeros ? hi / 15.0f - lo / 15.0f : fmaxf(hi, -lo) / 7.0f;
    const uint32_t bits = bad ? 0x7FC0u : bf16_bits_rne(unit);
    const float s = __uint_as_float(bits << 16);
    const bool none = bad || s == 0.0f;
    const float z = none ? 8.0f : zeros ? fminf(fmaxf(rintf(-lo / s), 0.0f), 15.0f) : 8.0f;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int j = lane + 64 * i;
        if (j < len)
            codes[row * k + k0 + j] =
                (uint8_t)(none ? z : fminf(fmaxf(rintf(v[i] / s) + z, 0.0f), 15.0f));
    }
    if (lane == 0) {
        scales[at] = (uint16_t)bits;
        if (zeros) zeros[at] = (uint8_t)z;
    }
}

int check_int4(int64_t n, int64_t k, int group) {
    if (n < 0 || n > (1 << 26) || k < 8 || k > (1 << 24) || k % 8 ||
        (group != 32 && group != 64 && group != 128))
        return NCM_E_SHAPE;
    // A workgroup per 16 outputs and 128 inputs packs them.
    return (n + 15) / 16 * ((k + 127) / 128) > kMaxBlocks ? NCM_E_SHAPE : NCM_OK;
}

template <typename F>
void with_out(int out, F f) {
    if (out == NCM_OUT_F32) f(std::integral_constant<int, NCM_OUT_F32>());
    else if (out == NCM_OUT_BF16) f(std::integral_constant<int, NCM_OUT_BF16>());
    else f(std::integral_constant<int, NCM_OUT_BF16_F32>());
}

// How a product is laid out, by its sizes.
struct Int4Layout {
    bool few;      // rows: the kernel without shared ones
    int splits;    // of the inputs
    size_t bytes;  // of the workspace
};
// A workgroup of the kernel of few rows reads all of x for 16 outputs, one of the
// other for 128, which counts where there are many of both. us in the one and the
// other, groups of 128: 4096 x 4096, 16 rows 7.3, 11.9; 16384 x 4096, 16 19.0, 16.8;
// 28672 x 4096, 8 25.5, 22.7 (groups of 32: 27.7, 29.9), 12 29.8, 23.2 (31.6, 30.2);
// 65536 x 4096, 2 31, 35, 5 43, 35 (52, 49); 128256 x 2048, 4 37, 37, 8 49, 37.
bool few_rows(int64_t m, int64_t n) { return m <= 4 || (m <= 16 && m * n <= (1 << 18)); }

Int4Layout int4_layout(int64_t m, int64_t n, int64_t k) {
    Int4Layout l = {few_rows(m, n), 1, 0};
    if (l.few) return l;
    // Workgroups of 128 outputs. Where they leave a CU without two, the inputs are
    // split, with at least four steps of 256 each; where they leave one without any,
    // with at least two (every output tile reads all of x, so narrower tiles would
    // only move the load to that). 28672 x 4096, 32 rows: 28 us, 30 without a split;
    // 4096 x 14336, 64: 25 in 8, 29 in 4 parts, unsplit 71; 4096 x 4096, 64: 13.8 in
    // 4, 15.6 in 8 parts of two steps, but 32 rows 12.6 in 8 of two, 12.8 in 4.
    // More than 8 parts lose: 4096 x 14336, 17 rows in 16 20.7 us, in 8 19.6.
    const int64_t groups = std::max<int64_t>(1, (n + 127) / 128 * ((m + kRowsOf - 1) / kRowsOf));
    const int64_t steps = (k + 255) / 256;
    const int64_t parts = std::max(std::min(512 / groups, steps / 4), std::min(256 / groups, steps / 2));
    l.splits = (int)std::clamp<int64_t>(parts, 1, 8);
    if (l.splits > 1) l.bytes = (size_t)l.splits * m * n * 4;
    return l;
}

template <int GROUP, bool ZEROS>
void launch(const Int4Args& a, const Int4Layout& l, int out, hipStream_t st) {
    const int64_t tiles = (a.n + 15) / 16;
    with_out(out, [&](auto mode) {
        constexpr int OUT = decltype(mode)::value;
        if (l.few) {
            const uint32_t blocks = (uint32_t)tiles;
            const size_t held = (size_t)a.m * a.blocks * 256;
            // Two blocks ahead where there are few wavefronts to wait on each other
            // (4096 x 14336: 13.4 us, 15.5 one ahead; 28672 x 4096: 24, 22), else x in
            // LDS where that is little (28672 x 4096, one row: 16.8 us, 22.4 without;
            // four: 21.2, 25; six, 48 KB of x: 26.4, 25.5).
            if (tiles < 512) linear_int4_kernel<GROUP, ZEROS, 2, false, OUT><<<blocks, 64 * kWaves, 0, st>>>(a);
            else if (held <= 32 * 1024) linear_int4_kernel<GROUP, ZEROS, 1, true, OUT><<<blocks, 64 * kWaves, held, st>>>(a);
            else linear_int4_kernel<GROUP, ZEROS, 1, false, OUT><<<blocks, 64 * kWaves, 0, st>>>(a);
            return;
        }
        const dim3 grid((uint32_t)((tiles + 7) / 8), (uint32_t)((a.m + kRowsOf - 1) / kRowsOf), (uint32_t)l.splits);
        linear_int4_rows_kernel<GROUP, ZEROS, OUT><<<grid, 512, 0, st>>>(a);
        if (l.splits > 1) {
            const int64_t quads = ((int64_t)a.n + 3) / 4 * a.m;
            linear_int4_join_kernel<OUT><<<(uint32_t)((quads + 255) / 256), 256, 0, st>>>(a);
        }
    });
}

}  // namespace
}  // namespace ncm

extern "C" int ncm_int4_bytes(int64_t n, int64_t k, int group, int has_zeros, size_t* codes,
                              size_t* scales) {
    using namespace ncm;
    if (!codes || !scales) return NCM_E_NULL;
    *codes = *scales = 0;
    const int rc = check_int4(n, k, group);
    if (rc) return rc;
    const size_t blocks = (size_t)((n + 15) / 16) * (size_t)((k + 127) / 128);
    *codes = blocks * 1024;
    *scales = blocks * (128 / group) * 16 * (has_zeros ? 4 : 2);
    return NCM_OK;
}

extern "C" int ncm_int4_quantise_dev(ncm_ctx_t* ctx, const uint16_t* w, int64_t n, int64_t k,
                                     int64_t stride, int group, uint8_t* codes, uint16_t* scales,
                                     uint8_t* zeros) {
    using namespace ncm;
    if (!ctx) return NCM_E_NULL;
    int rc = check_int4(n, k, group);
    if (rc) return rc;
    if (stride < k || stride > (int64_t(1) << 40)) return NCM_E_SHAPE;
    const int64_t groups = (k + group - 1) / group;
    if ((n * groups + 3) / 4 > kMaxBlocks) return NCM_E_SHAPE;
    if (n == 0) return NCM_OK;
    if (!w || !codes || !scales) return NCM_E_NULL;
    const DeviceScope scope(ncm_ctx_device(ctx));
    rc = step_hip(scope.error(), "int4_quantise device");
    if (rc) return rc;
    int4_quantise_kernel<<<(uint32_t)((n * groups + 3) / 4), 256, 0, ncm_ctx_stream(ctx)>>>(
        w, n, k, stride, group, codes, scales, zeros);
    return step_hip(hipGetLastError(), "int4_quantise launch");
}

extern "C" int ncm_int4_pack_dev(ncm_ctx_t* ctx, const uint8_t* codes, const uint16_t* scales,
                                 const uint8_t* zeros, int64_t n, int64_t k, int group,
                                 void* packed_codes, void* packed_scales) {
    using namespace ncm;
    if (!ctx) return NCM_E_NULL;
    int rc = check_int4(n, k, group);
    if (rc || n == 0) return rc;
    if (!codes || !scales || !packed_codes || !packed_scales) return NCM_E_NULL;
    if ((uintptr_t)packed_codes % 16 || (uintptr_t)packed_scales % 16) return NCM_E_ARG;
    const DeviceScope scope(ncm_ctx_device(ctx));
    rc = step_hip(scope.error(), "int4_pack device");
    if (rc) return rc;
    const int64_t blocks = (k + 127) / 128;
    int4_pack_kernel<<<(uint32_t)((n + 15) / 16 * blocks), 256, 0, ncm_ctx_stream(ctx)>>>(
        codes, scales, zeros, n, k, group, blocks, (uint32_t*)packed_codes, (char*)packed_scales);
    return step_hip(hipGetLastError(), "int4_pack launch");
}

extern "C" int ncm_linear_int4_workspace(int64_t m, int64_t n, int64_t k, size_t* bytes) {
    using namespace ncm;
    if (!bytes) return NCM_E_NULL;
    *bytes = 0;
    const int rc = check_int4(n, k, 32);
    if (rc) return rc;
    if (m < 0 || m > (1 << 20)) return NCM_E_SHAPE;
    *bytes = int4_layout(m, n, k).bytes;
    return NCM_OK;
}

extern "C" int ncm_linear_int4(ncm_ctx_t* ctx, const uint16_t* x, int64_t x_stride,
                               const ncm_int4_weight_t* w, const uint16_t* bias,
                               const float* residual, void* y, int64_t m, int out_mode,
                               void* workspace, size_t workspace_bytes) {
    using namespace ncm;
    if (!ctx || !w) return NCM_E_NULL;
    int rc = check_int4(w->n, w->k, w->group);
    if (rc) return rc;
    if (m < 0 || m > (1 << 20)) return NCM_E_SHAPE;
    if (out_mode != NCM_OUT_F32 && out_mode != NCM_OUT_BF16 && out_mode != NCM_OUT_BF16_F32)
        return NCM_E_ARG;
    if (m == 0 || w->n == 0) return NCM_OK;
    rc = check_rows(x, x_stride, w->k);
    if (rc) return rc;
    if (!w->codes || !w->scales || !y) return NCM_E_NULL;
    const int size = out_mode == NCM_OUT_BF16 ? 2 : 4;
    if ((uintptr_t)w->codes % 16 || (uintptr_t)w->scales % 16 || (uintptr_t)y % size ||
        (uintptr_t)bias % 2 || (uintptr_t)residual % 4)
        return NCM_E_ARG;
    if (residual == y && size == 2) return NCM_E_ARG;
    const Int4Layout l = int4_layout(m, w->n, w->k);
    if (l.bytes && !workspace) return NCM_E_NULL;
    if (workspace_bytes < l.bytes) return NCM_E_LENGTH;
    if (l.bytes && (uintptr_t)workspace % 16) return NCM_E_ARG;
    const bool wide = w->n % 4 == 0 && (uintptr_t)y % (4 * size) == 0 && (uintptr_t)bias % 8 == 0 &&
                      (uintptr_t)residual % 16 == 0;
    const Int4Args a = {x, (const u32x4_t*)w->codes, (const char*)w->scales, bias, residual, y,
                        x_stride, (int)m, (int)w->n, (int)w->k, (int)((w->k + 127) / 128), wide,
                        l.bytes ? (float*)workspace : nullptr, l.splits};
    const DeviceScope scope(ncm_ctx_device(ctx));
    rc = step_hip(scope.error(), "linear_int4 device");
    if (rc) return rc;
    const hipStream_t st = ncm_ctx_stream(ctx);
    auto go = [&](auto group) {
        constexpr int GROUP = decltype(group)::value;
        w->has_zeros ? launch<GROUP, true>(a, l, out_mode, st) : launch<GROUP, false>(a, l, out_mode, st);
    };
    if (w->group == 32) go(std::integral_constant<int, 32>());
    else if (w->group == 64) go(std::integral_constant<int, 64>());
    else go(std::integral_constant<int, 128>());
    return step_hip(hipGetLastError(), "linear_int4 launch");
}
