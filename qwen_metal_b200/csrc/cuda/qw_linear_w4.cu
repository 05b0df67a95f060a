// Linear layers with 4-bit weights for few rows of x: y = x W^T + bias, W[o][c] = s[o][g] (q[o][c] -
// z[o][g]), with a scale s (and a zero point z, 8 where there is none) for every `group` columns.
//
// The weights are the M dimension of mma.sync (16 outputs x 16 columns), 8 or 16 rows of x its N
// dimension: a warp reads 16 outputs' words straight into the fragments' registers, each word once,
// with no shared memory between.  A product's sum does not depend on the order of the columns, so
// the fragments take them as the words hold them: lane t of a quad has 32 neighbouring columns of
// its output, and columns i and i + 4 of a word are one register (one shift and one and-or give
// both as bf16 128 + q, exactly), which the x fragments match by two byte permutations.  A group's
// sums are kept in fp32; scale and zero are applied to them:
//   s (sum (128 + q) x - (128 + z) sum x), the second sum by an MMA with a matrix of ones.
// So nothing is rounded before y is, and taking 128 away costs an fp32 sum 2^-24 of 136 |x|, where
// a rounded weight would cost up to 2^-8 of its own.
//
// The warps of a CTA take the columns in turn, 128 at a time, and add their sums through shared
// memory in a fixed order.
//
// What bounds it: the weights' bytes only in the limit.  One row through 4096 -> 32768 (67 MB, groups of
// 128) takes 19 us in a chain of layers, 3.6 TB/s; through 4096 -> 6144 (12.6 MB) 5.5 us, 2.4 TB/s: a launch
// reads its code and first operands (4 us), then a warp has four or eight chunks to go.  13 rows of
// 4096 -> 12288, groups of 32, take 17 us (tensor pipe 19 %, issue 28 %): the warps wait for loads, of words two
// chunks ahead and of x, from L2, where it is used.
//
// The shape of a CTA follows the tiles of 16 outputs that an SM gets, so that all are there at once and the
// few columns a warp has left do not wait for few warps.  (It does not look at the columns: the figures are those of
// 4096 but for one line, and with 1024 half of sixteen warps have no chunk.)  Passes of four layers of 4096 columns,
// groups of 128 / 32, us (warps x tiles of outputs, CTAs that an SM must hold):
//   up to 8 rows     2048 outputs   16x1 1  26.0 / 27.9    12x1 2  25.7 / 29.9     8x1 3  26.1 / 33.3
//                    4096           12x1 2  26.5 / 32.6     8x1 3  27.2 / 38.8    16x1 1  30.5 / 42.0
//                    6144            8x1 3  30.1 / 39.3     8x2 2  30.9 / 46.5    12x1 2  35.3 / 53.0
//                    8192            8x2 2  31.0 / 47.2     8x1 3  40.9 / 64.2     4x1 4  35.0 / 56.0
//                   12288            8x2 2  45.1 / 81.8     8x1 3  47.8 / 68.9
//   9 to 16 rows     2048           16x1 1  24.4 / 28.2     8x1 1  27.7 / 36.7     4x2 3  40.9 / 62.3
//                    4096            8x2 1  33.1 / 42.8     8x1 1  36.0 / 40.0     4x2 3  40.0 / 64.8
//                    8192            6x2 2  44.2 / 61.8     4x2 3  54.1 / 77.0     8x2 1  55.2 / 73.5
//                   12288            4x2 3  56.7 / 82.0     6x2 2  75.5 / 113      8x2 1  75.2 / 101
// (12288 columns -> 4096, 13 rows: 8x2 1 66.5 / 109, 8x1 1 76.0 / 97.7, 4x2 3 99.2 / 209.)
// The CTA's weights are asked for in L2 before the wait for the kernel in front: 12288 -> 4096, 16 rows,
// groups of 64: 176 us, without 183.  x through shared memory and words through rings of cp.async were
// slower than either (one row, 6144 outputs, eight layers: 53 us, with rings 71 to 90).
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "qw_sm100.cuh"

namespace {

constexpr uint32_t kChunk = 128;  // columns of a warp's step

struct Params {
    const uint16_t *x;
    const uint32_t *w;
    const uint16_t *scales, *zeros, *bias;
    uint16_t *y;
    uint32_t rows, k, n, group;
    uint32_t per_group;  // groups of more than 128 columns: 2^32 over their chunks, rounded up
};

__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
        "{%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Columns i and i + 4 of a word as a pair of bf16: 0x4300 | q is 128 + q.
__device__ __forceinline__ uint32_t pair_of(uint32_t word, int i) {
    uint32_t r;
    asm("lop3.b32 %0, %1, 0x000f000f, 0x43004300, 0xea;" : "=r"(r) : "r"(word >> (4 * i)));
    return r;
}

__device__ __forceinline__ float widened(uint16_t bits) { return __uint_as_float((uint32_t)bits << 16); }

__device__ __forceinline__ uint4 load_stream(const uint32_t *p) {
    uint4 v;  // weights pass once; L1 is for x
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "l"(p));
    return v;
}

// Word i of lane t becomes word t of lane i, in each quad.
__device__ __forceinline__ void transpose_quad(uint32_t (&w)[4], uint32_t t) {
#pragma unroll
    for (int step = 1; step <= 2; step <<= 1) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (i & step) continue;
            const uint32_t mine = (t & step) ? w[i] : w[i | step];
            const uint32_t theirs = __shfl_xor_sync(0xffffffffu, mine, step);
            if (t & step) w[i] = theirs;
            else w[i | step] = theirs;
        }
    }
}

// Packed fp32 pairs (one issue slot for two).
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("{\n\t.reg .b64 ra, rb, rc, rd;\n\t"
        "mov.b64 ra, {%2, %3};\n\tmov.b64 rb, {%4, %5};\n\tmov.b64 rc, {%6, %7};\n\t"
        "fma.rn.f32x2 rd, ra, rb, rc;\n\tmov.b64 {%0, %1}, rd;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}

// Asks for [p, p + bytes) in L2, less what is not whole 16-byte pieces of it.
__device__ __forceinline__ void prefetch_l2(const void *p, size_t bytes) {
    const uintptr_t from = ((uintptr_t)p + 15) & ~(uintptr_t)15, to = ((uintptr_t)p + bytes) & ~(uintptr_t)15;
    if (from < to)
        asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(from), "r"((uint32_t)(to - from))
                     : "memory");
}

// What a lane holds of a chunk: words 4t .. 4t + 3 of its outputs, a scale and a zero point.
template <int kTilesM>
struct Stage {
    uint4 w[kTilesM][2];
    uint16_t s[kTilesM][2], z[kTilesM][2];
};

// kTilesN: 8 rows of x each; kTilesM: 16 outputs each.  kFold: words of a lane after which a group ends
// (1: 32 columns, 2: 64, 4: 128 and more).  kAhead: chunks of a warp in flight.
template <int kWarps, int kTilesN, int kTilesM, int kFold, bool kZeros, int kAhead, int kCtas>
__global__ void __launch_bounds__(kWarps * 32, kCtas) qw_linear_w4_kernel(const Params p) {
    constexpr int kRows = 8 * kTilesN, kOutputs = 16 * kTilesM;
    constexpr bool kWide = kFold == 4;
    __shared__ float sums[kWarps][kRows][kOutputs + 1];
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u, g = lane >> 2, t = lane & 3u;
    const uint32_t out0 = blockIdx.x * kOutputs, row0 = blockIdx.y * kRows;
    const uint32_t words = p.k / 8, groups = p.k / p.group, parts = p.k / 32;
    const uint32_t chunks = (p.k + kChunk - 1) / kChunk;
    // The CTA's weights and scales lie together.  Asking for them in L2 reads nothing that could be
    // out of date later, so it may run under the kernel before.
    sm100::grid_launch_dependents();
    if (threadIdx.x == 0) {
        const uint32_t outs = min((uint32_t)kOutputs, p.n - out0);
        prefetch_l2(p.w + (size_t)out0 * words, (size_t)outs * words * 4);
        prefetch_l2(p.scales + (size_t)out0 * groups, (size_t)outs * groups * 2);
        if constexpr (kZeros) prefetch_l2(p.zeros + (size_t)out0 * groups, (size_t)outs * groups * 2);
    }
    // Rows and outputs past the end are the last one's once more, and not stored: loads need no
    // conditions.  So are chunks past the end, which are loaded ahead and not used.
    const uint32_t *w_row[kTilesM][2];
    const uint16_t *s_row[kTilesM][2];
    const size_t zeros_from_scales = kZeros ? (size_t)(p.zeros - p.scales) : 0;
#pragma unroll
    for (int m = 0; m < kTilesM; ++m)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const uint32_t o = min(out0 + 16 * m + 8 * r + g, p.n - 1);
            w_row[m][r] = p.w + (size_t)o * words;
            s_row[m][r] = p.scales + (size_t)o * groups;
        }
    const uint16_t *x_row[kTilesN];
#pragma unroll
    for (int n = 0; n < kTilesN; ++n)
        x_row[n] = p.x + (size_t)min(row0 + 8 * n + g, p.rows - 1) * p.k;

    using Ring = Stage<kTilesM>;
    const auto fetch = [&](Ring &st, uint32_t chunk) __attribute__((always_inline)) {
        chunk = min(chunk, chunks - 1);
        uint32_t at, group;
        if constexpr (kWide) {
            at = chunk * 16 + 4 * t;
            group = p.per_group ? __umulhi(chunk, p.per_group) : chunk;
        } else {
            const uint32_t part = min(chunk * 4 + t, parts - 1);  // of 32 columns
            at = part * 4;
            group = part / kFold;
        }
#pragma unroll
        for (int m = 0; m < kTilesM; ++m)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                st.w[m][r] = load_stream(w_row[m][r] + at);
                st.s[m][r] = __ldg(s_row[m][r] + group);
                if constexpr (kZeros) st.z[m][r] = __ldg(s_row[m][r] + zeros_from_scales + group);
            }
    };
    float2 total[kTilesM][kTilesN][2] = {};
    const auto consume = [&](const Ring &st, uint32_t chunk) __attribute__((always_inline)) {
        uint4 x[kTilesN][4];
#pragma unroll
        for (int n = 0; n < kTilesN; ++n)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t column =
                    kWide ? chunk * kChunk + 32 * t + 8 * j : min(chunk * 4 + j, parts - 1) * 32 + 8 * t;
                x[n][j] = __ldg(reinterpret_cast<const uint4 *>(x_row[n] + column));
            }
        uint32_t w[kTilesM][2][4];
#pragma unroll
        for (int m = 0; m < kTilesM; ++m)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                w[m][r][0] = st.w[m][r].x, w[m][r][1] = st.w[m][r].y;
                w[m][r][2] = st.w[m][r].z, w[m][r][3] = st.w[m][r].w;
                // Narrow groups' columns must not meet in one MMA with another group's.
                if constexpr (!kWide) transpose_quad(w[m][r], t);
            }
        float acc[kTilesM][kTilesN][4], of_x[kTilesN][4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (!kWide && chunk * 4 + j >= parts) break;
            if (j % kFold == 0) {
#pragma unroll
                for (int n = 0; n < kTilesN; ++n)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        of_x[n][i] = 0.0f;
#pragma unroll
                        for (int m = 0; m < kTilesM; ++m) acc[m][n][i] = 0.0f;
                    }
            }
            uint32_t b[kTilesN][4];
#pragma unroll
            for (int n = 0; n < kTilesN; ++n) {
                b[n][0] = __byte_perm(x[n][j].x, x[n][j].z, 0x5410);
                b[n][1] = __byte_perm(x[n][j].x, x[n][j].z, 0x7632);
                b[n][2] = __byte_perm(x[n][j].y, x[n][j].w, 0x5410);
                b[n][3] = __byte_perm(x[n][j].y, x[n][j].w, 0x7632);
            }
            const uint32_t ones[4] = {0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u};
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
#pragma unroll
                for (int n = 0; n < kTilesN; ++n)
                    mma(of_x[n], ones, b[n][2 * half], b[n][2 * half + 1]);
            }
            if (j % kFold == kFold - 1) {
#pragma unroll
                for (int m = 0; m < kTilesM; ++m)
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        // (a narrow group's scale is with the lane whose load it was)
                        uint32_t s = st.s[m][r], z = kZeros ? st.z[m][r] : 0u;
                        if constexpr (!kWide) {
                            if constexpr (kZeros) s |= z << 16;
                            s = __shfl_sync(0xffffffffu, s, j, 4);
                            if constexpr (kZeros) z = s >> 16;
                        }
                        const float scale = __uint_as_float(s << 16);
                        const float less = kZeros ? -128.0f - __uint_as_float(z << 16) : -136.0f;
                        const float2 scale2 = make_float2(scale, scale), less2 = make_float2(less, less);
#pragma unroll
                        for (int n = 0; n < kTilesN; ++n) {
                            const float2 v = fma2(less2, make_float2(of_x[n][2 * r], of_x[n][2 * r + 1]),
                                                  make_float2(acc[m][n][2 * r], acc[m][n][2 * r + 1]));
                            total[m][n][r] = fma2(scale2, v, total[m][n][r]);
                        }
                    }
            }
        }
    };
    sm100::grid_wait();
    Ring ring[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) fetch(ring[i], warp + i * kWarps);
    for (uint32_t chunk = warp; chunk < chunks; chunk += kAhead * kWarps) {
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const uint32_t at = chunk + i * kWarps;
            if (at >= chunks) break;
            consume(ring[i], at);
            if (at + kAhead * kWarps < chunks) fetch(ring[i], at + kAhead * kWarps);
        }
    }
#pragma unroll
    for (int m = 0; m < kTilesM; ++m)
#pragma unroll
        for (int n = 0; n < kTilesN; ++n)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                sums[warp][8 * n + 2 * t][16 * m + 8 * r + g] = total[m][n][r].x;
                sums[warp][8 * n + 2 * t + 1][16 * m + 8 * r + g] = total[m][n][r].y;
            }
    __syncthreads();
    for (uint32_t e = threadIdx.x; e < kRows * kOutputs; e += kWarps * 32) {
        const uint32_t row = e / kOutputs, o = e - row * kOutputs;
        if (row0 + row >= p.rows || out0 + o >= p.n) continue;
        float v = p.bias ? widened(__ldg(p.bias + out0 + o)) : 0.0f;
#pragma unroll
        for (int i = 0; i < kWarps; ++i) v += sums[i][row][o];
        p.y[(size_t)(row0 + row) * p.n + out0 + o] = (uint16_t)(sm100::pack_bf16(v, 0.0f) & 0xffffu);
    }
}

template <int kWarps, int kTilesN, int kTilesM, int kFold, int kAhead, int kCtas>
int launch_fold(const Params &p, cudaStream_t stream) {
    const auto kernel = p.zeros ? qw_linear_w4_kernel<kWarps, kTilesN, kTilesM, kFold, true, kAhead, kCtas>
                                : qw_linear_w4_kernel<kWarps, kTilesN, kTilesM, kFold, false, kAhead, kCtas>;
    const dim3 grid((p.n + 16 * kTilesM - 1) / (16 * kTilesM), (p.rows + 8 * kTilesN - 1) / (8 * kTilesN));
    return sm100::launch(kernel, grid, kWarps * 32, 0, 1, stream, p);
}
template <int kWarps, int kTilesN, int kTilesM, int kAhead, int kCtas>
int launch_narrow(const Params &p, cudaStream_t stream) {
    return p.group == 64 ? launch_fold<kWarps, kTilesN, kTilesM, 2, kAhead, kCtas>(p, stream)
                         : launch_fold<kWarps, kTilesN, kTilesM, 1, kAhead, kCtas>(p, stream);
}
template <int kWarps, int kTilesN, int kTilesM, int kAhead, int kCtas>
int launch_tiles(const Params &p, cudaStream_t stream) {
    return p.group >= kChunk ? launch_fold<kWarps, kTilesN, kTilesM, 4, kAhead, kCtas>(p, stream)
                             : launch_narrow<kWarps, kTilesN, kTilesM, kAhead, kCtas>(p, stream);
}

}  // namespace

extern "C" int qwcu_linear_w4_launch(const qwcu_linear_w4_args *a, int sm_count, qwcu_stream stream_) {
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
    const uint32_t of_group = a->group / kChunk;
    p.per_group = of_group > 1 ? (uint32_t)((0x100000000ull + of_group - 1) / of_group) : 0u;
    const unsigned tiles = a->n / 16 + (a->n % 16 != 0), sms = (unsigned)(sm_count > 0 ? sm_count : 148);
    const bool wide = a->group >= kChunk;
    if (a->rows <= 8) {
        if (tiles <= sms) return launch_tiles<16, 1, 1, 2, 1>(p, stream);
        if (tiles <= 2 * sms) return launch_tiles<12, 1, 1, 2, 2>(p, stream);
        if (tiles <= 3 * sms) return launch_tiles<8, 1, 1, 2, 3>(p, stream);
        if (wide || tiles <= 4 * sms) return launch_tiles<8, 1, 2, 2, 2>(p, stream);
        return launch_narrow<8, 1, 1, 2, 3>(p, stream);
    }
    if (tiles <= sms) return launch_tiles<16, 2, 1, 2, 1>(p, stream);
    if (tiles <= 2 * sms)
        return wide ? launch_fold<8, 2, 2, 4, 2, 1>(p, stream) : launch_narrow<8, 2, 1, 2, 1>(p, stream);
    if (tiles <= 4 * sms) return launch_tiles<6, 2, 2, 2, 2>(p, stream);
    return launch_tiles<4, 2, 2, 2, 3>(p, stream);
}
