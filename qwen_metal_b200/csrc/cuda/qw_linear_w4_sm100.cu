// Linear layers with 4-bit weights for many rows, on the tensor cores (tcgen05).
//
//   y = x W^T + bias, W[o][c] = s[o][g] (q[o][c] - z[o][g])
//
// The weights are the A operand, 128 outputs in the lanes of TMEM, and up to 256 rows of x the B
// operand in shared memory.  A thread owns half of an output's columns of a step: it takes their words, makes
// s (q - z) in bf16 of them and stores them into TMEM, where the MMAs read A from; nothing of the expanded
// weights goes through shared memory, whose bandwidth the MMAs need for B.  q - z is exact for whole z of up to
// 8 bits (z = 8 without zero points) and rounded to bf16 otherwise; the weight is rounded once more, to half a
// step, as it would be in a layer of bf16 weights.  All of a tile's products are summed in fp32 in TMEM.
//
// Warps (384 threads):
//   0      TMA producer: 128 columns of x and of the weights' words a step
//   1      MMA issuer, TMEM allocation
//   4..11  weights: words -> bf16 -> TMEM; at the end TMEM -> the result
// What bounds it: for tiles of up to 128 rows the weights' integer work, a step of 128 columns about 1000 clocks
// against 512 of MMA; a tile of 256 rows half hides it (4000 rows through 4096 x 12288: 337 us, 1.19 PFLOP/s).
// 412 rows of 4096 x 4096: 30 us, begin to submit; 300 rows, a layer of a chain, 20 us.
// With whole q - z as A and every group's sums taken out of TMEM and scaled in fp32 no weight is rounded, but
// four warps do nothing else and every group is a hand-over: 4 layers of those 300 rows took 115 us (groups of
// 128) and 278 us (of 32), as here 88 and 95; 4000 rows 574 and 1404 us, as here 423 and 441 (tiles of 128).
// A few tiles would leave SMs idle: up to eight CTAs of a cluster then take a share of the columns each
// and add their sums through each other's shared memory, in the order of the CTAs (30 rows of 4096 x 4096:
// 8 us a layer).
//
// Every wait is bounded (status words, abort flag), and a CTA leaves no copy or MMA in flight.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "qw_sm100.cuh"

namespace {

using namespace sm100;

constexpr int kThreads = 384;
constexpr int kOutputs = 128;         // of a tile: TMEM lanes
constexpr uint32_t kChunk = 128;      // columns of a step
constexpr int kMaxStages = 8;
constexpr int kMostSmem = 227 * 1024;
// More than half an SM's: a second CTA there would wait for the first one's TMEM, while that one may wait, by
// its cluster or by the order of launches, for the second.
constexpr size_t kLeastSmem = 116 * 1024;
constexpr int kABuffers = 4;          // expanded weights of a step each, 64 columns of TMEM
constexpr uint32_t kTmemCols = 512, kTmemA = 256;  // sums at 0, weights from 256
constexpr int kWordBytes = kOutputs * 64;  // words of 128 outputs x 128 columns
constexpr int kWeightWarp = 4;  // first of eight

enum Barrier : int {
    kBarFull = 0,                        // x and words of a stage landed
    kBarEmpty = kBarFull + kMaxStages,   // words taken (8 warps) and x consumed (MMA)
    kBarAFull = kBarEmpty + kMaxStages,  // weights in TMEM (8 warps)
    kBarAEmpty = kBarAFull + kABuffers,
    kBarDone = kBarAEmpty + kABuffers,   // every MMA of the CTA is done
    kBarCount = kBarDone + 1
};

struct __align__(16) Control {
    Mbar bars[kBarCount];
    uint32_t tmem_base;
    volatile uint32_t abort_flag;
};

struct Params {
    const uint16_t *scales, *zeros, *bias;
    uint16_t *y;
    uint32_t rows, k, n, groups;
    uint32_t tile_rows;    // rows of x of a tile, a multiple of 16: the MMA's N
    uint32_t idesc;
    uint32_t group_steps;  // steps of a group of 128 columns and more
    uint32_t stages;       // of the ring, at most kMaxStages
    uint32_t splits;       // CTAs of a cluster, over the columns
    uint32_t *status;
    long long wait_cycles;
    int probes;            // the same budget for the MMA warp's waits
    uint32_t withhold;     // step (>= 1) from which the producer loads nothing, 0: none
};

__device__ __forceinline__ float widened(uint16_t bits) { return __uint_as_float((uint32_t)bits << 16); }
__device__ __forceinline__ uint32_t mul_bf16x2(uint32_t a, uint32_t b) {
    const __nv_bfloat162 v = __hmul2(*reinterpret_cast<const __nv_bfloat162 *>(&a),
                                     *reinterpret_cast<const __nv_bfloat162 *>(&b));
    return *reinterpret_cast<const uint32_t *>(&v);
}
__device__ __forceinline__ uint32_t add_bf16x2(uint32_t a, uint32_t b) {
    const __nv_bfloat162 v = __hadd2(*reinterpret_cast<const __nv_bfloat162 *>(&a),
                                     *reinterpret_cast<const __nv_bfloat162 *>(&b));
    return *reinterpret_cast<const uint32_t *>(&v);
}

// Scales or zero points of half a step's columns of an output, a step ahead of their use.  kUnits: groups of
// a step (1: a group is a step or several).
template <int kUnits>
struct Ahead {
    static constexpr uint32_t kHere = kUnits == 4 ? 2 : 1;
    const uint16_t *row;
    uint32_t group, last, left, steps;  // left: steps that the group has still to go
    uint16_t next[kHere];
    __device__ __forceinline__ Ahead(const Params &p, const uint16_t *values, uint32_t output, uint32_t step,
                                     uint32_t half)
        : row(values + (size_t)output * p.groups), last(p.groups - 1), steps(p.group_steps) {
        if constexpr (kUnits == 1) {
            group = step / steps;
            left = steps - (step - group * steps);
        } else {
            group = step * kUnits + half * kHere;
        }
        read();
    }
    // (Groups past the end are the last one's once more: their columns of x are zeros.)
    __device__ __forceinline__ void read() {
#pragma unroll
        for (uint32_t u = 0; u < kHere; ++u) next[u] = __ldg(row + min(group + u, last));
    }
    __device__ __forceinline__ void advance() {
        if constexpr (kUnits == 1) {
            if (--left == 0) ++group, left = steps;
        } else {
            group += kUnits;
        }
        read();
    }
};

// Eight 4-bit columns of a word as four pairs of bf16 in their order, less the zero point.  0x4300 | q
// is 128 + q; taking 128 away first leaves q, from which a zero of any value is taken with one rounding.
template <bool kZeros>
__device__ __forceinline__ void expand(uint32_t word, uint32_t minus_zero, uint32_t (&out)[4]) {
    const uint32_t odd = word >> 4;
#pragma unroll
    for (int i = 0; i < 4; ++i) {  // columns 2i and 2i + 1: byte i of the word and of the shifted word
        uint32_t v = __byte_perm(word, odd, 0x4400 + 0x1111 * i);
        asm("lop3.b32 %0, %0, 0x000f000f, 0x43004300, 0xea;" : "+r"(v));
        if constexpr (kZeros) out[i] = add_bf16x2(add_bf16x2(v, 0xc300c300u), minus_zero);
        else out[i] = add_bf16x2(v, 0xc308c308u);
    }
}

__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
        "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
        "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
        "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]),
        "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]),
        "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
        : "memory");
}

// The bounded wait in line, for warps whose registers are full: a call would have them saved around it.
__device__ __forceinline__ bool wait_in_line(const Waiter &w, Mbar *bar, uint32_t parity, uint32_t where,
                                             uint32_t step) {
    bool ok = mbar_try(bar, parity);
    if (!ok) {
        const long long start = clock64();
        do {
            ok = mbar_try(bar, parity);
            if (!ok && *w.abort_flag) break;
            if (!ok && clock64() - start > w.budget) {
                *w.abort_flag = 1;
                if (atomicCAS(w.status, 0u, (uint32_t)QWCU_STATUS_WAIT_TIMEOUT) == 0u) {
                    w.status[1] = where;
                    w.status[2] = step;
                    w.status[3] = blockIdx.x;
                }
                __threadfence_system();
                break;
            }
        } while (!ok);
    }
    return __all_sync(0xffffffffu, ok) != 0;
}

// The wait of the MMA warp, bounded by a number of probes that the host makes of the budget: each clock
// between two groups' MMAs is one in which the tensor cores, which take four MMAs ahead, may run dry, so
// the loop holds nothing else.  A probe that fails suspends the warp for up to 7800 clocks.
constexpr long long kProbeCycles = 10000;
__device__ __forceinline__ bool probe(uint32_t bar, uint32_t parity, int probes) {
    bool ok = false;
#pragma unroll 1
    for (int i = 0; i < probes && !ok; ++i) ok = mbar_try(bar, parity);
    return __all_sync(0xffffffffu, ok) != 0;
}
static __device__ __noinline__ void gave_up(const Waiter w, uint32_t bar, uint32_t step) {
    *w.abort_flag = 1;
    if (atomicCAS(w.status, 0u, (uint32_t)QWCU_STATUS_WAIT_TIMEOUT) == 0u) {
        w.status[1] = (2u << 16) | bar;
        w.status[2] = step;
        w.status[3] = blockIdx.x;
    }
    __threadfence_system();
}

// A value the compiler knows to be the same in all lanes of the (converged) warp.
template <typename T>
__device__ __forceinline__ T uniform(T v) {
    return __shfl_sync(0xffffffffu, v, 0);
}

// The MMAs of a step.  Unrolled, on operands in uniform registers: in a loop over them an MMA took 150 clocks
// to issue, more than twice its execution.
__device__ __forceinline__ void issue_step(uint32_t d, uint32_t a, uint32_t x_lo, uint32_t box, uint32_t idesc,
                                           uint32_t accumulate) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
        mma_ts(d, a + (uint32_t)i * 8u, x_lo + (uint32_t)(i >> 2) * box + (uint32_t)(i & 3) * 2u, idesc,
               i > 0 ? 1u : accumulate);
}

__device__ __forceinline__ float4 ld_cluster4(uint32_t cluster_addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                 : "r"(cluster_addr)
                 : "memory");
    return v;
}

// kUnits: groups of a step (1: a group is a step or several).
template <int kUnits, bool kZeros>
__global__ void __launch_bounds__(kThreads, 1)
qw_linear_w4_sm100_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w,
                          const Params p) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    const uint32_t box_bytes = p.tile_rows * 128u, stage_bytes = 2 * box_bytes + kWordBytes;
    Control *ctl = reinterpret_cast<Control *>(smem + p.stages * stage_bytes);
    const int warp = warp_index();
    const uint32_t lane = threadIdx.x & 31u;
    const uint32_t rank = blockIdx.x % p.splits;
    const uint32_t tile = blockIdx.x / p.splits;
    const uint32_t out0 = tile * kOutputs, row0 = blockIdx.y * p.tile_rows;
    const uint32_t steps = (p.k + kChunk - 1) / kChunk;
    const uint32_t first = (uint32_t)((unsigned long long)steps * rank / p.splits);
    const uint32_t end = (uint32_t)((unsigned long long)steps * (rank + 1) / p.splits);
    Mbar *bars = ctl->bars;

    if (warp == 0 && lane == 0) {
        for (int i = 0; i < kMaxStages; ++i) {
            mbar_init(&bars[kBarFull + i], 1);
            mbar_init(&bars[kBarEmpty + i], 9);
        }
        for (int i = 0; i < kABuffers; ++i) {
            mbar_init(&bars[kBarAFull + i], 8);
            mbar_init(&bars[kBarAEmpty + i], 1);
        }
        mbar_init(&bars[kBarDone], 1);
        ctl->abort_flag = 0;
        mbar_init_fence();
    }
    if (warp == 1) tmem_alloc<1>(&ctl->tmem_base, kTmemCols);
    grid_launch_dependents();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    grid_wait();
    const uint32_t tmem = ctl->tmem_base;
    const Waiter w = {&ctl->abort_flag, p.status, p.wait_cycles > 0 ? p.wait_cycles : kWaitCycles};
    float *staged = reinterpret_cast<float *>(smem);  // the tile's totals [row of x][output], where the ring was

    if (warp >= kWeightWarp) {
        // A thread has half of a step's columns of an output.
        const uint32_t half = (uint32_t)(warp - kWeightWarp) >> 2, row = (uint32_t)(warp & 3) * 32 + lane;
        const uint32_t lanes = (uint32_t)(warp & 3) * 32 << 16;
        uint32_t s = 0, phase = 0, t = 0;
        bool ok = true;
        const uint32_t output = min(out0 + row, p.n - 1);
        Ahead<kUnits> scales(p, p.scales, output, first, half);
        // (without zero points the scales stand in for them, unused)
        Ahead<kUnits> zeros(p, kZeros ? p.zeros : p.scales, output, first, half);
        for (uint32_t step = first; step < end; ++step, ++t) {
            const uint32_t a = t % kABuffers;
            constexpr uint32_t kHere = Ahead<kUnits>::kHere;
            uint32_t scale[kHere], minus_zero[kHere];
#pragma unroll
            for (uint32_t u = 0; u < kHere; ++u) {
                scale[u] = (uint32_t)scales.next[u] * 0x10001u;
                minus_zero[u] = kZeros ? (uint32_t)(zeros.next[u] ^ 0x8000u) * 0x10001u : 0u;
            }
            scales.advance();
            if constexpr (kZeros) zeros.advance();
            ok = wait_in_line(w, &bars[kBarFull + s], phase, (3u << 16) | (kBarFull + s), step);
            if (!ok) break;
            // 64 bytes of an output, 16-byte pieces swizzled by the TMA over pairs of rows.
            const uint32_t words = smem_u32(smem + s * stage_bytes + 2 * box_bytes) + row * 64u;
            uint4 v[2];
#pragma unroll
            for (uint32_t i = 0; i < 2; ++i) v[i] = ld_shared16(words + (((2 * half + i) ^ ((row >> 1) & 3u)) << 4));
            __syncwarp();
            if (lane == 0) mbar_arrive(&bars[kBarEmpty + s]);
            if (++s == p.stages) s = 0, phase ^= 1u;
            uint32_t r[32];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const uint4 &q = v[i >> 2];
                const uint32_t word = (i & 3) == 0 ? q.x : (i & 3) == 1 ? q.y : (i & 3) == 2 ? q.z : q.w;
                const uint32_t unit = kHere == 2 ? i >> 2 : 0;
                uint32_t e[4];
                expand<kZeros>(word, minus_zero[unit], e);
#pragma unroll
                for (int c = 0; c < 4; ++c) r[4 * i + c] = mul_bf16x2(e[c], scale[unit]);
            }
            ok = wait_in_line(w, &bars[kBarAEmpty + a], ((t / kABuffers) & 1u) ^ 1u, (3u << 16) | (kBarAEmpty + a),
                              step);
            if (!ok) break;
            tc_fence_after();
            tmem_st32(tmem + lanes + kTmemA + a * 64 + half * 32, r);
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&bars[kBarAFull + a]);
        }
        // When all MMAs are done, so are all loads and whoever reads them.
        if (ok) ok = wait_in_line(w, &bars[kBarDone], 0, (3u << 16) | kBarDone, end);
        tc_fence_after();
#pragma unroll 1
        for (uint32_t row0 = 32 * half; ok && row0 < p.tile_rows; row0 += 64) {
            uint32_t r[32];
            tmem_ld32(r, tmem + lanes + row0);
            tmem_wait_ld32(r);
#pragma unroll
            for (uint32_t i = 0; i < 32; ++i)
                if (row0 + i < p.tile_rows) staged[(row0 + i) * kOutputs + row] = __uint_as_float(r[i]);
        }
    }
    if (warp == 0) {
        uint32_t s = 0, phase = 0, t = 0;
        for (uint32_t step = first; step < end; ++step, ++t) {
            if (p.withhold && t >= p.withhold) break;  // nothing is issued, nothing is in flight
            if (!mbar_wait_warp(w, &bars[kBarEmpty + s], phase ^ 1u, (1u << 16) | (kBarEmpty + s), step)) break;
            if (elect_one()) {
                uint8_t *to = smem + s * stage_bytes;
                const uint32_t bar = smem_u32(&bars[kBarFull + s]);
                mbar_expect_tx(&bars[kBarFull + s], stage_bytes);
                tma_load_2d<1>(to + 2 * box_bytes, &map_w, bar, (int)(step * (kChunk / 8)), (int)out0);
                tma_load_2d<1>(to, &map_x, bar, (int)(step * kChunk), (int)row0);
                tma_load_2d<1>(to + box_bytes, &map_x, bar, (int)(step * kChunk + 64), (int)row0);
            }
            __syncwarp();
            if (++s == p.stages) s = 0, phase ^= 1u;
        }
        // Leave no copy in flight: the last round's, and of the round before those not yet loaded over.
        for (uint32_t i = 0; i < p.stages; ++i) {
            if (i < s) mbar_drain(&bars[kBarFull + i], phase, w.budget);
            else if (t >= p.stages) mbar_drain(&bars[kBarFull + i], phase ^ 1u, w.budget);
        }
    } else if (warp == 1) {
        bool ok = true;
        uint32_t s = 0, t = 0;
        const uint32_t d_tmem = uniform(tmem), x0 = uniform(smem_u32(smem) >> 4) | kDescKMajor;
        const uint32_t bar0 = uniform(smem_u32(bars)), box = box_bytes >> 4;
        const auto at = [&](uint32_t which) { return bar0 + which * (uint32_t)sizeof(Mbar); };
        for (uint32_t step = first; step < end && ok; ++step, ++t) {
            const uint32_t a = t % kABuffers;
            // (The weights' warps have seen the stage: so has, through their arrivals, this one.)
            ok = probe(at(kBarAFull + a), (t / kABuffers) & 1u, p.probes);
            if (!ok) {
                gave_up(w, kBarAFull + a, step);
                break;
            }
            const uint32_t x_lo = x0 + s * (stage_bytes >> 4), a_tmem = d_tmem + kTmemA + a * 64;
            tc_fence_after();
            if (elect_one()) {
                issue_step(d_tmem, a_tmem, x_lo, box, p.idesc, t > 0 ? 1u : 0u);
                tc_commit<1>(at(kBarEmpty + s));
                tc_commit<1>(at(kBarAEmpty + a));
            }
            __syncwarp();
            if (++s == p.stages) s = 0;
        }
        if (elect_one()) tc_commit<1>(&bars[kBarDone]);
        __syncwarp();
        mbar_drain(&bars[kBarDone], 0, w.budget);
    }
    tc_fence_before();
    if (p.splits > 1) cluster_sync();
    else __syncthreads();
    const uint32_t rows = min(p.tile_rows, p.rows - row0);
    for (uint32_t e = threadIdx.x; e < rows * (kOutputs / 4); e += kThreads) {
        const uint32_t r = e / (kOutputs / 4), o = (e - r * (kOutputs / 4)) * 4;
        if (r % p.splits != rank || out0 + o >= p.n) continue;
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (p.splits > 1) {
            for (uint32_t c = 0; c < p.splits; ++c) {
                const float4 x = ld_cluster4(map_to_rank(staged + r * kOutputs + o, c));
                v.x += x.x, v.y += x.y, v.z += x.z, v.w += x.w;
            }
        } else {
            v = *reinterpret_cast<const float4 *>(staged + r * kOutputs + o);
        }
        const float f[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) {
            if (out0 + o + i >= p.n) break;
            const float bias = p.bias ? widened(__ldg(p.bias + out0 + o + i)) : 0.0f;
            p.y[(size_t)(row0 + r) * p.n + out0 + o + i] = (uint16_t)(pack_bf16(f[i] + bias, 0.0f) & 0xffffu);
        }
    }
    if (p.splits > 1) cluster_sync();  // (nobody leaves while its totals are read)
    if (warp == 1) tmem_dealloc<1>(tmem, kTmemCols);
}

// [n][k / 8] words, boxes of 16 words x 128 outputs, 16-byte pieces swizzled within 64 bytes.
int make_words_map(CUtensorMap *map, const void *base, uint32_t n, uint32_t words) {
    EncodeTiledFn fn = encode_tiled_fn();
    if (!fn) return (int)cudaErrorNotSupported;
    const cuuint64_t dims[2] = {words, n}, strides[1] = {(cuuint64_t)words * 4};
    const cuuint32_t box[2] = {kChunk / 8, kOutputs}, elem[2] = {1, 1};
    const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT32, 2, const_cast<void *>(base), dims, strides, box,
                          elem, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_64B,
                          CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? 0 : (int)cudaErrorInvalidValue;
}

template <int kUnits, bool kZeros>
int launch_kernel(const Params &p, const CUtensorMap &map_x, const CUtensorMap &map_w, cudaStream_t stream) {
    // The opt-in to the shared memory is an attribute of the device: set on first use.
    static bool ready[64];
    const auto kernel = qw_linear_w4_sm100_kernel<kUnits, kZeros>;
    int dev = 0;
    cudaError_t code = cudaGetDevice(&dev);
    if (code != cudaSuccess) return (int)code;
    const bool tracked = dev >= 0 && dev < 64;
    if (!tracked || !ready[dev]) {
        code = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostSmem);
        if (code != cudaSuccess) return (int)code;
        if (tracked) ready[dev] = true;
    }
    const dim3 grid((p.n + kOutputs - 1) / kOutputs * p.splits, (p.rows + p.tile_rows - 1) / p.tile_rows);
    const size_t needed = p.stages * (p.tile_rows * 256u + kWordBytes) + sizeof(Control) + 1024;
    return launch(kernel, grid, kThreads, needed > kLeastSmem ? needed : kLeastSmem, (int)p.splits, stream, map_x,
                  map_w, p);
}
// Clusters of `size` CTAs that the device holds at once, asked for once.  (One CTA per SM, by its shared memory,
// in all variants.)
unsigned clusters_at_once(unsigned size) {
    static unsigned known[64][9];
    int dev = 0, count = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return 0;
    const bool tracked = dev >= 0 && dev < 64;
    if (tracked && known[dev][size]) return known[dev][size];
    const auto kernel = qw_linear_w4_sm100_kernel<1, false>;
    cudaLaunchConfig_t config = {};
    cudaLaunchAttribute cluster;
    cluster.id = cudaLaunchAttributeClusterDimension;
    cluster.val.clusterDim.x = size;
    cluster.val.clusterDim.y = cluster.val.clusterDim.z = 1;
    config.gridDim = dim3(size);
    config.blockDim = dim3(kThreads);
    config.dynamicSmemBytes = kMostSmem;
    config.attrs = &cluster;
    config.numAttrs = 1;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostSmem) != cudaSuccess ||
        cudaOccupancyMaxActiveClusters(&count, kernel, &config) != cudaSuccess) {
        cudaGetLastError();
        return 0;
    }
    if (tracked) known[dev][size] = (unsigned)count;
    return (unsigned)count;
}

}  // namespace

extern "C" int qwcu_linear_w4_sm100_launch(const qwcu_linear_w4_args *a, int sm_count, qwcu_stream stream_) {
    cudaStream_t stream = static_cast<cudaStream_t>(stream_);
    const bool whole = a->group == 32 || a->group == 64 || (a->group && a->group % kChunk == 0);
    if (!a->rows || !a->n || !a->k || !whole || a->k % a->group) return (int)cudaErrorInvalidValue;
    if (((uintptr_t)a->x | (uintptr_t)a->w) & 15u) return (int)cudaErrorMisalignedAddress;
    Params p;
    p.scales = static_cast<const uint16_t *>(a->scales);
    p.zeros = static_cast<const uint16_t *>(a->zeros);
    p.bias = static_cast<const uint16_t *>(a->bias);
    p.y = static_cast<uint16_t *>(a->y);
    p.rows = a->rows;
    p.k = a->k;
    p.n = a->n;
    p.groups = a->k / a->group;
    p.group_steps = a->group / kChunk;
    p.status = a->status;
    p.wait_cycles = a->wait_cycles;
    // (At least 32 probes; kProbeCycles is more than a probe takes, so that this role, which waits for the
    // cause itself, gives up before those that wait behind it.)
    p.probes = 32 + (int)((a->wait_cycles > 0 ? a->wait_cycles : kWaitCycles) / kProbeCycles);
    p.withhold = a->withhold_from;
    // Tiles of equal height.  With 128 rows and less of a tile there may be few enough for several CTAs to a
    // tile's columns, of at least four steps each.  Room is what the device says: clusters do not reach over
    // its parts, so SMs are left over (24 rows of 4096, a pass of four layers: 2048 outputs are 16 clusters of
    // eight, of which 14 fit: 55.2 us, with clusters of four 39.4; 4608 outputs are 36 of four, 70.9 us, of two
    // 54.5).
    const unsigned sms = (unsigned)(sm_count > 0 ? sm_count : 148);
    const uint32_t steps = (a->k + kChunk - 1) / kChunk, low = (a->rows + 127) / 128;
    const unsigned long long columns = (a->n + kOutputs - 1) / kOutputs;
    const auto height = [&](uint32_t tiles) { return ((a->rows + tiles - 1) / tiles + 15) / 16 * 16; };
    uint32_t tiles = low;
    p.splits = 1;
    while (p.splits < 8 && steps / (p.splits * 2) >= 4 && columns * tiles <= clusters_at_once(p.splits * 2))
        p.splits *= 2;
    // Otherwise as many tiles as make the waves cheapest, up to 256 rows each: a CTA's time goes as 170 + rows,
    // of which the 170 are the weights.  4096 -> 4096, 500 rows: 21 us in tiles of 128, 26 of 256 (two CTAs
    // each); 1000 rows, where 256 save the second wave, 40 and 29; 4000 rows to 12288 outputs 420 and 327.
    if (p.splits == 1) {
        const auto cost = [&](uint32_t count) {
            return (columns * count + sms - 1) / sms * (170 + height(count));
        };
        for (uint32_t count = low - low / 2, step = 1 + low / 32; count < low; count += step)
            if (columns * count * 2 > sms && cost(count) < cost(tiles)) tiles = count;
    }
    p.tile_rows = height(tiles);
    // As many stages as there is room for, up to eight (412 rows of 4096: no difference between four and six).
    const uint32_t fit = (kMostSmem - 1024 - (uint32_t)sizeof(Control)) / (p.tile_rows * 256u + kWordBytes);
    p.stages = fit < (uint32_t)kMaxStages ? fit : (uint32_t)kMaxStages;
    p.idesc = instr_desc(kOutputs, p.tile_rows, false);
    CUtensorMap map_x, map_w;
    int rc;
    if ((rc = make_map_2d(&map_x, a->x, a->rows, a->k, p.tile_rows))) return rc;
    if ((rc = make_words_map(&map_w, a->w, a->n, a->k / 8))) return rc;
    if (p.zeros)
        return a->group == 32   ? launch_kernel<4, true>(p, map_x, map_w, stream)
               : a->group == 64 ? launch_kernel<2, true>(p, map_x, map_w, stream)
                                : launch_kernel<1, true>(p, map_x, map_w, stream);
    return a->group == 32   ? launch_kernel<4, false>(p, map_x, map_w, stream)
           : a->group == 64 ? launch_kernel<2, false>(p, map_x, map_w, stream)
                            : launch_kernel<1, false>(p, map_x, map_w, stream);
}
