// Linear layers with 4-bit weights: y = x W^T + bias, W[o][c] = s[o][g] (q[o][c] - z[o][g]), with a
// scale s (and a zero point z, 8 where there is none) for every `group` columns.  HBM-bound on the
// weights for few rows of x.
//
// The weights are the M dimension of mma.sync (16 outputs x 16 columns), up to 32 rows of x its N
// dimension: a warp reads 16 outputs' words straight into the fragments' registers, each word once,
// with no shared memory between.  A product's sum does not depend on the order of the columns, so
// the fragments take them as the words hold them: lane t of a quad has 32 neighbouring columns of
// its output, and columns i and i + 4 of a word are one register (one shift and one and-or give
// both as bf16 128 + q), which the x fragments match by two byte permutations.  q - 8 is exact in
// bf16 and the group's sum is kept in fp32; scale and zero are applied to the sum:
//   s (sum (q - 8) x - (z - 8) sum x), the second sum by an MMA with a matrix of ones.
// So nothing is rounded before y is.
//
// The warps of a CTA take the columns in turn, 128 at a time, and add their sums through shared
// memory in a fixed order.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "qw_sm100.cuh"

namespace {

constexpr int kWarps = 8;
constexpr uint32_t kChunk = 128;  // columns of a warp's step

struct Params {
    const uint16_t *x;
    const uint32_t *w;
    const uint16_t *scales, *zeros, *bias;
    uint16_t *y;
    uint32_t rows, k, n, group;
};

__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
        "{%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Columns i and i + 4 of a word, less 8, as a pair of bf16: 0x4300 | q is 128 + q.
__device__ __forceinline__ uint32_t pair_of(uint32_t word, int i) {
    uint32_t r;
    asm("lop3.b32 %0, %1, 0x000f000f, 0x43004300, 0xea;" : "=r"(r) : "r"(word >> (4 * i)));
    const __nv_bfloat162 minus = __halves2bfloat162(__ushort_as_bfloat16(0xc308), __ushort_as_bfloat16(0xc308));
    const __nv_bfloat162 v = __hadd2(*reinterpret_cast<const __nv_bfloat162 *>(&r), minus);
    return *reinterpret_cast<const uint32_t *>(&v);
}

__device__ __forceinline__ float widened(uint16_t bits) { return __uint_as_float((uint32_t)bits << 16); }

// The four words of an output that a lane has of a chunk.  Groups of 128 columns and more: words
// 4t .. 4t + 3, one load; narrower ones, whose columns must not meet in one MMA: words t, 4 + t, ...
template <bool kWide>
__device__ __forceinline__ void load_words(uint32_t (&w)[4], const uint32_t *row, uint32_t words,
                                           uint32_t chunk, uint32_t t) {
    if constexpr (kWide) {
        const uint4 v = __ldg(reinterpret_cast<const uint4 *>(row + chunk * 16) + t);
        w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t at = chunk * 16 + 4 * j + t;
            w[j] = at < words ? __ldg(row + at) : 0u;
        }
    }
}

// kFold: words of a lane after which a group ends (1: 32 columns, 2: 64, 4: 128 and more).
template <int kTilesN, int kTilesM, int kFold, bool kZeros>
__global__ void __launch_bounds__(kWarps * 32) qw_linear_w4_kernel(const Params p) {
    constexpr int kRows = 8 * kTilesN, kOutputs = 16 * kTilesM;
    constexpr bool kWide = kFold == 4;
    __shared__ float sums[kWarps][kRows][kOutputs + 1];
    sm100::grid_launch_dependents();
    sm100::grid_wait();
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u, g = lane >> 2, t = lane & 3u;
    const uint32_t out0 = blockIdx.x * kOutputs, row0 = blockIdx.y * kRows;
    const uint32_t words = p.k / 8, groups = p.k / p.group, chunks = (p.k + kChunk - 1) / kChunk;

    // Outputs past the end are the last one's once more and not stored.
    const uint32_t *w_row[kTilesM][2];
    size_t s_row[kTilesM][2];
#pragma unroll
    for (int m = 0; m < kTilesM; ++m)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const uint32_t o = min(out0 + 16 * m + 8 * r + g, p.n - 1);
            w_row[m][r] = p.w + (size_t)o * words;
            s_row[m][r] = (size_t)o * groups;
        }
    float total[kTilesM][kTilesN][4] = {};
    uint32_t next[kTilesM][2][4];
    if (warp < chunks) {
#pragma unroll
        for (int m = 0; m < kTilesM; ++m)
#pragma unroll
            for (int r = 0; r < 2; ++r) load_words<kWide>(next[m][r], w_row[m][r], words, warp, t);
    }
    for (uint32_t chunk = warp; chunk < chunks; chunk += kWarps) {
        uint32_t w[kTilesM][2][4];
#pragma unroll
        for (int m = 0; m < kTilesM; ++m)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
#pragma unroll
                for (int j = 0; j < 4; ++j) w[m][r][j] = next[m][r][j];
                if (chunk + kWarps < chunks)
                    load_words<kWide>(next[m][r], w_row[m][r], words, chunk + kWarps, t);
            }
        float acc[kTilesM][kTilesN][4], of_x[kTilesN][4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (j % kFold == 0) {
#pragma unroll
                for (int n = 0; n < kTilesN; ++n) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) of_x[n][i] = 0.0f;
#pragma unroll
                    for (int m = 0; m < kTilesM; ++m)
#pragma unroll
                        for (int i = 0; i < 4; ++i) acc[m][n][i] = 0.0f;
                }
            }
            const uint32_t column = chunk * kChunk + (kWide ? 32 * t + 8 * j : 32 * j + 8 * t);
            uint32_t b[kTilesN][4];
#pragma unroll
            for (int n = 0; n < kTilesN; ++n) {
                const uint32_t row = row0 + 8 * n + g;
                uint4 v = make_uint4(0, 0, 0, 0);
                if (row < p.rows && column < p.k)
                    v = __ldg(reinterpret_cast<const uint4 *>(p.x + (size_t)row * p.k + column));
                b[n][0] = __byte_perm(v.x, v.z, 0x5410);
                b[n][1] = __byte_perm(v.x, v.z, 0x7632);
                b[n][2] = __byte_perm(v.y, v.w, 0x5410);
                b[n][3] = __byte_perm(v.y, v.w, 0x7632);
            }
#pragma unroll
            for (int half = 0; half < 2; ++half) {
#pragma unroll
                for (int m = 0; m < kTilesM; ++m) {
                    const uint32_t a[4] = {pair_of(w[m][0][j], 2 * half), pair_of(w[m][1][j], 2 * half),
                                           pair_of(w[m][0][j], 2 * half + 1),
                                           pair_of(w[m][1][j], 2 * half + 1)};
#pragma unroll
                    for (int n = 0; n < kTilesN; ++n)
                        mma(acc[m][n], a, b[n][2 * half], b[n][2 * half + 1]);
                }
                if constexpr (kZeros) {
                    const uint32_t ones[4] = {0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u};
#pragma unroll
                    for (int n = 0; n < kTilesN; ++n)
                        mma(of_x[n], ones, b[n][2 * half], b[n][2 * half + 1]);
                }
            }
            if (j % kFold == kFold - 1) {
                // (a group past the last column has sums of zero)
                const uint32_t group =
                    min(kWide ? chunk * kChunk / p.group : (chunk * kChunk + 32 * j) / p.group, groups - 1);
#pragma unroll
                for (int m = 0; m < kTilesM; ++m)
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        const float s = widened(__ldg(p.scales + s_row[m][r] + group));
                        float z = 0.0f;
                        if constexpr (kZeros) z = widened(__ldg(p.zeros + s_row[m][r] + group)) - 8.0f;
#pragma unroll
                        for (int n = 0; n < kTilesN; ++n)
#pragma unroll
                            for (int i = 0; i < 2; ++i) {
                                float v = acc[m][n][2 * r + i];
                                if constexpr (kZeros) v = fmaf(-z, of_x[n][2 * r + i], v);
                                total[m][n][2 * r + i] = fmaf(s, v, total[m][n][2 * r + i]);
                            }
                    }
            }
        }
    }
#pragma unroll
    for (int m = 0; m < kTilesM; ++m)
#pragma unroll
        for (int n = 0; n < kTilesN; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                sums[warp][8 * n + 2 * t + (i & 1)][16 * m + 8 * (i >> 1) + g] = total[m][n][i];
    __syncthreads();
    for (uint32_t e = threadIdx.x; e < kRows * kOutputs; e += kWarps * 32) {
        const uint32_t row = e / kOutputs, o = e - row * kOutputs;
        if (row0 + row >= p.rows || out0 + o >= p.n) continue;
        float v = p.bias ? widened(__ldg(p.bias + out0 + o)) : 0.0f;
#pragma unroll
        for (int i = 0; i < kWarps; ++i) v += sums[i][row][o];
        p.y[(size_t)(row0 + row) * p.n + out0 + o] =
            (uint16_t)(sm100::pack_bf16(v, 0.0f) & 0xffffu);
    }
}

template <int kTilesN, int kTilesM>
int launch_tiles(const Params &p, cudaStream_t stream) {
    void (*kernel)(const Params);
    if (p.group >= kChunk)
        kernel = p.zeros ? qw_linear_w4_kernel<kTilesN, kTilesM, 4, true>
                         : qw_linear_w4_kernel<kTilesN, kTilesM, 4, false>;
    else if (p.group == 64)
        kernel = p.zeros ? qw_linear_w4_kernel<kTilesN, kTilesM, 2, true>
                         : qw_linear_w4_kernel<kTilesN, kTilesM, 2, false>;
    else
        kernel = p.zeros ? qw_linear_w4_kernel<kTilesN, kTilesM, 1, true>
                         : qw_linear_w4_kernel<kTilesN, kTilesM, 1, false>;
    const dim3 grid((p.n + 16 * kTilesM - 1) / (16 * kTilesM), (p.rows + 8 * kTilesN - 1) / (8 * kTilesN));
    return sm100::launch(kernel, grid, kWarps * 32, 0, 1, stream, p);
}

}  // namespace

extern "C" int qwcu_linear_w4_launch(const qwcu_linear_w4_args *a, int sm_count, qwcu_stream stream_) {
    (void)sm_count;
    cudaStream_t stream = static_cast<cudaStream_t>(stream_);
    const bool whole = a->group == 32 || a->group == 64 || (a->group && a->group % kChunk == 0);
    if (!a->rows || !a->n || !a->k || !whole || a->k % a->group) return (int)cudaErrorInvalidValue;
    if (((uintptr_t)a->x | (uintptr_t)a->w) & 15u) return (int)cudaErrorMisalignedAddress;
    Params p;
    p.x = static_cast<const uint16_t *>(a->x);
    p.w = a->w;
    p.scales = static_cast<const uint16_t *>(a->scales);
    p.zeros = static_cast<const uint16_t *>(a->zeros);
    p.bias = static_cast<const uint16_t *>(a->bias);
    p.y = static_cast<uint16_t *>(a->y);
    p.rows = a->rows;
    p.k = a->k;
    p.n = a->n;
    p.group = a->group;
    if (a->rows <= 8) return launch_tiles<1, 1>(p, stream);
    if (a->rows <= 16) return launch_tiles<2, 1>(p, stream);
    return launch_tiles<4, 2>(p, stream);
}
