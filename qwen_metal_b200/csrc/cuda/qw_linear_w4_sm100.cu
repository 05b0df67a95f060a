// Linear layers with 4-bit weights for many rows, on the tensor cores (tcgen05).
//
//   y = x W^T + bias, W[o][c] = s[o][g] (q[o][c] - z[o][g])
//
// The weights are the A operand, 128 outputs in the lanes of TMEM, and up to 256 rows of x the B
// operand in shared memory.  A thread owns half of an output's columns of a step: it takes their words, makes
// s (q - z) of them and stores them into TMEM, where the MMAs read A from; nothing of the expanded weights goes
// through shared memory, whose bandwidth the MMAs need for B.  A weight is the sum of two bf16 numbers, and each
// is an A operand of its own, so that no weight is rounded: s (q - 8) has 12 bits and is held whole, as is
// s (q - z) for whole z; other zero points cost at most 3 * 2^-16 of the weight.  (One bf16 number, 2^-8 of the
// weight off, is half of the MMAs, but a layer then answers otherwise than with few rows: 412 rows of 4096 x 4096
// 28 us between a chain's events, as here 36; a sum of random weights' products 0.0022 of its size off and 0.0017,
// which is the result's own rounding.)  All of a tile's products are summed in fp32 in TMEM.
//
// Warps (384 threads):
//   0      TMA producer: 128 columns of x and of the weights' words a step
//   1      MMA issuer, TMEM allocation
//   4..11  weights: words -> two parts in bf16 -> TMEM; at the end TMEM -> the result
// What bounds it: up to 128 rows of a tile a step's chain of waits, words, expansion, TMEM stores and MMAs, which
// run beside one another only in part: 1400 clocks for 112 rows (412 of 4096 x 4096: tensor pipe 55 % active, issue
// 38 %, ALU 32 %; 36 us between the events of a chain, 49 from its begin to its submit's end; 300 rows, a layer of
// a chain, 29).  With 256 rows the MMAs, 16 to a step of 128 columns: 2800 clocks (4000 rows through 4096 x 12288
// 593 us, 0.68 PFLOP/s of the layer, 1.36 of the MMAs).
// With whole q - z as A and every group's sums taken out of TMEM and scaled in fp32 four warps do nothing else and
// every group is a hand-over: 4 layers of those 300 rows took 115 us (groups of 128) and 278 us (of 32), as here
// 121 and 126; 4000 rows 574 and 1404 us, as here 593 and 618; and a zero point that is not whole is rounded.
// A few tiles would leave SMs idle: up to eight CTAs of a cluster then take a share of the columns each
// and add their sums through each other's shared memory, in the order of the CTAs (30 rows of 4096 x 4096:
// 9 us a layer).
//
// Every wait is bounded (status words, abort flag), and a CTA leaves no copy or MMA in flight.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <type_traits>

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
// TMEM: sums in the first 128 or 256 columns, behind them three or two buffers of a step's weights, 64 columns of
// first parts and 64 of second ones.
constexpr int kMaxABuffers = 3;
constexpr uint32_t kTmemCols = 512, kACols = 128;
constexpr int kWordBytes = kOutputs * 64;  // words of 128 outputs x 128 columns
constexpr int kWeightWarp = 4;  // first of eight

enum Barrier : int {
    kBarFull = 0,                        // x and words of a stage landed
    kBarEmpty = kBarFull + kMaxStages,   // words taken (8 warps) and x consumed (MMA)
    kBarAFull = kBarEmpty + kMaxStages,  // weights in TMEM (8 warps)
    kBarAEmpty = kBarAFull + kMaxABuffers,
    kBarDone = kBarAEmpty + kMaxABuffers,  // every MMA of the CTA is done
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
    uint32_t tmem_a, a_buffers;  // where the weights' buffers begin, and how many there are
    uint32_t group_steps;  // steps of a group of 128 columns and more
    uint32_t stages;       // of the ring, at most kMaxStages
    uint32_t splits;       // CTAs of a cluster, over the columns
    uint32_t *status;
    long long wait_cycles;
    int probes;            // the same budget for the MMA warp's waits
    uint32_t withhold;     // step (>= 1) from which the producer loads nothing, 0: none
};

__device__ __forceinline__ float widened(uint16_t bits) { return __uint_as_float((uint32_t)bits << 16); }
__device__ __forceinline__ uint32_t fma_bf16x2(uint32_t a, uint32_t b, uint32_t c) {
    const __nv_bfloat162 v =
        __hfma2(*reinterpret_cast<const __nv_bfloat162 *>(&a), *reinterpret_cast<const __nv_bfloat162 *>(&b),
                *reinterpret_cast<const __nv_bfloat162 *>(&c));
    return *reinterpret_cast<const uint32_t *>(&v);
}
__device__ __forceinline__ uint32_t mul_bf16x2(uint32_t a, uint32_t b) {
    const __nv_bfloat162 v = __hmul2_rn(*reinterpret_cast<const __nv_bfloat162 *>(&a),
                                     *reinterpret_cast<const __nv_bfloat162 *>(&b));
    return *reinterpret_cast<const uint32_t *>(&v);
}
__device__ __forceinline__ uint32_t add_bf16x2(uint32_t a, uint32_t b) {
    const __nv_bfloat162 v = __hadd2_rn(*reinterpret_cast<const __nv_bfloat162 *>(&a),
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

constexpr uint32_t kSigns = 0x80008000u;

// The two bf16 parts of a group's weights s (q - z), from v = 16 + q: `first` and `second` add up to a weight.
//   without zero points   first = h (q - 8), second = l (q - 8) with h + l = s of four bits each: both have eight
//                         bits at most, and (16 + q) h - 24 h is one instruction without a rounding.
//   |z| <= 64             z = n + f, n whole: d = q - n is exact, and first = d s - c rounded, c the first part of
//                         s f = c + e.  t = d s - first is exact: for d = 0 it is c; otherwise |first| is at least
//                         half of s, so t, which is c but for half a step of `first`, is a multiple of 2^-8 (of
//                         s's binade) below 1, or with |first| > 1 of 2^-7 below 2.  second = (t - c) - e: what
//                         the rounding left, less the rest of s f, 2^-7 of the weight at most; its two roundings
//                         cost 2^-16 and 2^-15 of the weight.
//   any other             q - z as d and its error, by the two-sum of six additions that Knuth gives; first = d s
//                         rounded, second what that left and the error's product.  (24 h may not overflow either.)
template <bool kZeros>
struct Group {
    uint32_t scale, minus_zero;  // bf16 pairs
    uint32_t a, b, c, d;         // h, l, -24 h, -24 l; or -(16 + n), -c, -e
    bool near;
    __device__ __forceinline__ Group(uint16_t s, uint16_t z) {
        scale = (uint32_t)s * 0x10001u;
        if constexpr (kZeros) {
            minus_zero = (uint32_t)(z ^ 0x8000u) * 0x10001u;
            const float zero = widened(z), whole = rintf(zero), rest = widened(s) * (whole - zero);
            near = fabsf(zero) <= 64.0f;
            a = pack_bf16(-16.0f - whole, -16.0f - whole);
            b = pack_bf16(rest, rest);
            const float more = rest - __uint_as_float(b & 0xffff0000u);
            c = pack_bf16(more, more);
        } else {
            minus_zero = 0xc100c100u;  // -8
            near = (s & 0x7fffu) < 0x7b80u;  // 2^120
            a = scale & 0xfff0fff0u;
            b = add_bf16x2(scale, a ^ kSigns);
            c = mul_bf16x2(a, 0xc1c0c1c0u);
            d = mul_bf16x2(b, 0xc1c0c1c0u);
        }
    }
    // Eight columns of a word as four pairs in their order.  0x4180 | q << 3 is 16 + q.
    template <bool kNear>
    __device__ __forceinline__ void expand(uint32_t word, uint32_t *first, uint32_t *second) const {
        const uint32_t even = word << 3, odd = word >> 1;
#pragma unroll
        for (int i = 0; i < 4; ++i) {  // columns 2i and 2i + 1: the same byte of both
            uint32_t v = __byte_perm(even, odd, 0x4400 + 0x1111 * i);
            asm("lop3.b32 %0, %0, 0x00780078, 0x41804180, 0xea;" : "+r"(v));
            if constexpr (!kNear) {
                const uint32_t q = add_bf16x2(v, 0xc180c180u), sum = add_bf16x2(q, minus_zero);
                const uint32_t y = add_bf16x2(sum, q ^ kSigns), x = add_bf16x2(sum, y ^ kSigns);
                const uint32_t err = add_bf16x2(add_bf16x2(q, x ^ kSigns), add_bf16x2(minus_zero, y ^ kSigns));
                first[i] = mul_bf16x2(sum, scale);
                second[i] = fma_bf16x2(err, scale, fma_bf16x2(sum, scale, first[i] ^ kSigns));
            } else if constexpr (kZeros) {
                const uint32_t x = add_bf16x2(v, a);
                first[i] = fma_bf16x2(x, scale, b);
                second[i] = add_bf16x2(add_bf16x2(fma_bf16x2(x, scale, first[i] ^ kSigns), b), c);
            } else {
                first[i] = fma_bf16x2(v, a, c);
                second[i] = fma_bf16x2(v, b, d);
            }
        }
    }
};

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

// The MMAs of half a step's A, 128 columns of one part.  Unrolled, on operands in uniform registers: in a loop
// over them an MMA took 150 clocks to issue, more than twice its execution.
__device__ __forceinline__ void issue_part(uint32_t d, uint32_t a, uint32_t x_lo, uint32_t box, uint32_t idesc,
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
        for (int i = 0; i < kMaxABuffers; ++i) {
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
        uint32_t s = 0, phase = 0, a = 0, a_phase = 1;
        bool ok = true;
        const uint32_t output = min(out0 + row, p.n - 1);
        Ahead<kUnits> scales(p, p.scales, output, first, half);
        // (without zero points the scales stand in for them, unused)
        Ahead<kUnits> zeros(p, kZeros ? p.zeros : p.scales, output, first, half);
        for (uint32_t step = first; step < end; ++step) {
            constexpr uint32_t kHere = Ahead<kUnits>::kHere;
            // (where there is one, the second is not made)
            const Group<kZeros> groups[2] = {{scales.next[0], zeros.next[0]},
                                             {scales.next[kHere - 1], zeros.next[kHere - 1]}};
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
            uint32_t r[2][32];
            const auto expand = [&](auto near) __attribute__((always_inline)) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const uint4 &q = v[i >> 2];
                    const uint32_t word = (i & 3) == 0 ? q.x : (i & 3) == 1 ? q.y : (i & 3) == 2 ? q.z : q.w;
                    groups[kHere == 2 ? i >> 2 : 0].template expand<decltype(near)::value>(word, r[0] + 4 * i,
                                                                                          r[1] + 4 * i);
                }
            };
            if (__all_sync(0xffffffffu, groups[0].near && groups[kHere - 1].near)) expand(std::true_type());
            else expand(std::false_type());
            ok = wait_in_line(w, &bars[kBarAEmpty + a], a_phase, (3u << 16) | (kBarAEmpty + a), step);
            if (!ok) break;
            tc_fence_after();
            const uint32_t to = tmem + lanes + p.tmem_a + a * kACols + half * 32;
            tmem_st32(to, r[0]);
            tmem_st32(to + kACols / 2, r[1]);
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&bars[kBarAFull + a]);
            if (++a == p.a_buffers) a = 0, a_phase ^= 1u;
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
        uint32_t s = 0, a = 0, a_phase = 0;
        const uint32_t d_tmem = uniform(tmem), x0 = uniform(smem_u32(smem) >> 4) | kDescKMajor;
        const uint32_t bar0 = uniform(smem_u32(bars)), box = box_bytes >> 4;
        const auto at = [&](uint32_t which) { return bar0 + which * (uint32_t)sizeof(Mbar); };
        for (uint32_t step = first; step < end && ok; ++step) {
            // (The weights' warps have seen the stage: so has, through their arrivals, this one.)
            ok = probe(at(kBarAFull + a), a_phase, p.probes);
            if (!ok) {
                gave_up(w, kBarAFull + a, step);
                break;
            }
            const uint32_t x_lo = x0 + s * (stage_bytes >> 4), a_tmem = d_tmem + p.tmem_a + a * kACols;
            tc_fence_after();
            if (elect_one()) {
                issue_part(d_tmem, a_tmem, x_lo, box, p.idesc, step > first ? 1u : 0u);
                issue_part(d_tmem, a_tmem + kACols / 2, x_lo, box, p.idesc, 1u);
                tc_commit<1>(at(kBarEmpty + s));
                tc_commit<1>(at(kBarAEmpty + a));
            }
            __syncwarp();
            if (++s == p.stages) s = 0;
            if (++a == p.a_buffers) a = 0, a_phase ^= 1u;
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
    const long long budget = a->wait_cycles > 0 ? a->wait_cycles : kWaitCycles;
    p.probes = 32 + (int)(budget / kProbeCycles < 1ll << 30 ? budget / kProbeCycles : 1ll << 30);
    p.withhold = a->withhold_from;
    // Tiles of equal height.  With 128 rows and less of a tile there may be few enough for several CTAs to a
    // tile's columns, of at least four steps each.  Room is what the device says: clusters do not reach over
    // its parts, so SMs are left over (24 rows of 4096, a pass of four layers: 2048 outputs are 16 clusters of
    // eight, of which 14 fit: 58.2 us, with clusters of four 42.4; 4608 outputs are 36 of four, 74.6 us, of two
    // 59.1).
    const unsigned sms = (unsigned)(sm_count > 0 ? sm_count : 148);
    const uint32_t steps = (a->k + kChunk - 1) / kChunk, low = (a->rows + 127) / 128;
    const unsigned long long columns = (a->n + kOutputs - 1) / kOutputs;
    const auto height = [&](uint32_t tiles) { return ((a->rows + tiles - 1) / tiles + 15) / 16 * 16; };
    uint32_t tiles = low;
    p.splits = 1;
    while (p.splits < 8 && steps / (p.splits * 2) >= 4 && columns * tiles <= clusters_at_once(p.splits * 2))
        p.splits *= 2;
    // Otherwise as many tiles as make the waves cheapest, up to 256 rows each: a CTA's time goes as 60 + rows, with
    // zero points 120 + rows, for which 90 + rows stands (60 or 170 there: 1 to 10 % slower or equal where it
    // chooses otherwise).  A layer 4096 -> 4096, 500 rows: 32 us in tiles of 128, 50 of 256; 1000 rows, where 256
    // save the second wave, 60 and 51; 4000 rows to 12288 outputs 685 and 593.
    if (p.splits == 1) {
        const auto cost = [&](uint32_t count) {
            return (columns * count + sms - 1) / sms * (90 + height(count));
        };
        for (uint32_t count = low - low / 2, step = 1 + low / 32; count < low; count += step)
            if (columns * count * 2 > sms && cost(count) < cost(tiles)) tiles = count;
    }
    p.tile_rows = height(tiles);
    // As many stages as there is room for, up to eight (412 rows of 4096, four layers: 123 us with
    // six, 128 with four).
    const uint32_t fit = (kMostSmem - 1024 - (uint32_t)sizeof(Control)) / (p.tile_rows * 256u + kWordBytes);
    p.stages = fit < (uint32_t)kMaxStages ? fit : (uint32_t)kMaxStages;
    p.idesc = instr_desc(kOutputs, p.tile_rows, false);
    p.tmem_a = p.tile_rows <= 128 ? 128 : 256;
    p.a_buffers = (kTmemCols - p.tmem_a) / kACols;
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
