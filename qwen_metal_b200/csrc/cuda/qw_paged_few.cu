// Attention of a few new tokens of each sequence over a paged K/V cache (HBM-bound: every visible K
// and V row is read once for all the heads and tokens that share it).
//
//   o = softmax(scale * q K^T) V over the cache rows a token sees: those before it and its own.
//
// A unit is a (sequence, kv head, 8 or 16 query rows): the query heads of a kv head, token by token,
// are its rows.  Both products run on mma.sync with the keys, then the value's dimensions, as M and
// the query rows as N, so that one tile of 16 keys and 8 rows costs 16 MMAs and all accumulators of a
// warp are 32 registers:
//   S^T = K Q^T    a lane reads 16 bytes of a key; which dimension of the sum a register of a
//                  fragment holds is free as long as K and Q agree, so they go in as they are loaded;
//   O^T = V^T P^T  a lane reads 16 bytes of four keys, and a byte permutation makes pairs of keys of
//                  them; S^T becomes P^T by movmatrix.
// So K and V go from global memory to registers to the tensor cores: no shared memory, no barrier.
// Cache rows past the sequence's end are not read (what they hold may be anything); masked scores
// are -inf.  Running maximum and sum are fp32 in the exp2 domain, P is rounded to bf16 for P V: 2^-8 of a
// weight at most, as in the library's other attention.  (What that leaves as a second operand, which would
// make it 2^-16, spills registers: 64 sequences of up to 4096 keys, two layers, 240 -> 251 us, 1000 of up to 64,
// four layers, 208 -> 234.)
//
// What bounds it: HBM, once there are some MB to read.  One sequence of 131072 keys (537 MB): 97 us,
// 5.5 TB/s, 85 % of a plain copy's rate; 64 of up to 4096 keys 120 us (5.6 TB/s).  One of 2000 keys: 20 us
// between the events of a chain, 28 to 32 from its begin to its submit's end; 1000 sequences of up to 64 keys 58 us,
// twice what their bytes take:
// a unit of four tiles is a chain of their loads' latencies.  168 registers a thread keep a tile of K and V
// of each of 12 warps in flight.
//
// All key tiles of all units are numbered through and dealt out evenly, a run of them to a CTA,
// whose warps take tiles in turn and merge at the end of a unit, or, of several short units, a unit
// each.  A unit that lies in several CTAs' runs is merged by the last of them to finish, from partial
// results in the workspace in the order of the CTAs, so that results do not depend on who is last.
#include <cuda_runtime.h>
#include <stdint.h>

#include "qw_paged.cuh"
#include "qw_sm100.cuh"

namespace {

using sm100::pack_bf16;

constexpr int kDim = 128;
constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kCtasPerSm = 3;
constexpr int kKeys = 16;         // keys of a tile; a page holds whole tiles
// Tiles of a CTA: below, launch and merge cost more than they gain (8 sequences of 300 keys: 31.0 us, with
// 4 tiles 31.8, 16 36.2, 24 41.7, 40 54.3).
constexpr uint32_t kLeast = 8;
// Tiles of the warps without a unit that a merge may cost.  Single tokens of 1000 sequences of up to 64 keys
// 58.0 us, 256 of up to 200 49.7, of up to 1000 128; with 0 62.4, 53.5, 128; with 48 58.1, 51.4, 136; all
// units merged 99.3, 58.4, 130, but 64 sequences of 4 tokens over up to 1000 keys 61.0 instead of 62.1.
constexpr uint32_t kAlone = 16;
constexpr int kMostRows = 16;     // query rows of a unit
constexpr int kPartial = kMostRows * (kDim + 2);  // floats of a partial result: rows, then (m, l)
constexpr int kStride = kDim + 4;                 // floats of a row of a warp's result in shared memory
// CTAs of a launch, so parts of a unit: their weights, a row after the other, take the place of the warps'
// rows (176 SMs' CTAs; with one or two rows the last warp's place holds sums).
constexpr unsigned kMostCtas = kWarps * kStride;
static_assert(2 * kMostCtas <= (kWarps - 1) * 8 * kStride, "weights of two rows reach into the sums");

struct Params {
    const uint16_t *q, *k_pages, *v_pages;
    uint16_t *out;
    uint32_t heads, kv_heads, share;  // share: query heads of a kv head
    uint32_t most_rows;               // sequences with more query rows are another kernel's
    int beside;                       // that kernel is the one in front of this one in the stream
    float scale_log2;
    float *partials;     // two of each CTA
    uint32_t *counters;  // one of each CTA, zero between launches
    paged::Cache cache;
};

__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                    uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
        "{%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transposed(uint32_t v) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
__device__ __forceinline__ float fast_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// 1 / sum: 0 for a row that has seen nothing, NaN for a NaN sum.
__device__ __forceinline__ float inverse(float sum) { return sum == 0.0f ? 0.0f : 1.0f / sum; }
__device__ __forceinline__ uint4 load16(const uint16_t *p, bool there) {
    return there ? __ldg(reinterpret_cast<const uint4 *>(p)) : make_uint4(0, 0, 0, 0);
}
__device__ __forceinline__ uint32_t word(const uint4 &v, int i) {
    return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w;
}

// What a sequence gives to do: units (row tiles of a kv head) and key tiles of each.
struct Work {
    uint32_t row_tiles, tiles;
};
template <int kRows>
__device__ __forceinline__ Work work_of(const Params &p, const paged::Sequence &s) {
    const unsigned long long rows = (unsigned long long)s.fresh * p.share;
    Work w;
    w.row_tiles = rows > p.most_rows ? 0u : (uint32_t)((rows + kRows - 1) / kRows);  // (kRows: a power of two)
    w.tiles = max(1u, ((uint32_t)s.length + kKeys - 1) / kKeys);  // (no key: zeros are still written)
    return w;
}

template <int kTilesN>
__global__ void __launch_bounds__(kThreads, kTilesN == 1 ? kCtasPerSm : 2)
qw_paged_few_kernel(const Params p) {
    constexpr int kRows = 8 * kTilesN;
    __shared__ float merge_o[kWarps][kRows][kStride];
    __shared__ float merge_m[kWarps][kRows], merge_l[kWarps][kRows];
    __shared__ unsigned long long scan[kWarps], found_rest;
    __shared__ uint32_t found_b, last_one;
    // The kernel for chunks starts this one when it has itself waited for all that was before it, and the two
    // read and write nothing of each other's: this one waits for it only at its end, so that whoever waits for
    // this one has waited for both.
    sm100::grid_launch_dependents();
    if (!p.beside) sm100::grid_wait();
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u, g = lane >> 2, t = lane & 3u;

    // The tiles of every sequence, summed over the batch; a thread has a run of sequences.
    const uint32_t batch = p.cache.batch, per = (batch + kThreads - 1) / kThreads;
    const uint32_t b_first = min(tid * per, batch), b_end = min(b_first + per, batch);
    unsigned long long mine = 0;
    for (uint32_t b = b_first; b < b_end; ++b) {
        const Work w = work_of<kRows>(p, paged::sequence(p.cache, b));
        mine += (unsigned long long)w.row_tiles * w.tiles * p.kv_heads;
    }
    unsigned long long before = mine;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
        const unsigned long long v = __shfl_up_sync(0xffffffffu, before, off);
        if (lane >= off) before += v;
    }
    if (lane == 31) scan[warp] = before;
    before -= mine;
    __syncthreads();
    unsigned long long total = 0;
#pragma unroll
    for (int i = 0; i < kWarps; ++i) {
        if (i < (int)warp) before += scan[i];
        total += scan[i];
    }
    // (Divisions in 32 bits where they are enough: a launch reads its code anew, line by line from L2, and one in
    // 64 bits is long.)
    const unsigned long long even =
        total >> 31 ? (total + gridDim.x - 1) / gridDim.x : ((uint32_t)total + gridDim.x - 1) / gridDim.x;
    const unsigned long long run = even > kLeast ? even : kLeast;
    unsigned long long at = run * blockIdx.x;
    const unsigned long long end = at + run < total ? at + run : total;
    if (at >= total) {
        if (p.beside) sm100::grid_wait();
        return;
    }
    if (at >= before && at < before + mine) {
        unsigned long long rest = at - before;
        for (uint32_t b = b_first;; ++b) {
            const Work w = work_of<kRows>(p, paged::sequence(p.cache, b));
            const unsigned long long here = (unsigned long long)w.row_tiles * w.tiles * p.kv_heads;
            if (rest < here) {
                found_b = b;
                break;
            }
            rest -= here;
        }
        found_rest = rest;
    }
    __syncthreads();
    uint32_t b = found_b;
    unsigned long long rest = found_rest;  // tile of sequence b that this CTA is at
    const size_t row_elements = (size_t)p.kv_heads * kDim;

    while (at < end) {
        const paged::Sequence s = paged::sequence(p.cache, b);
        const Work w = work_of<kRows>(p, s);
        const unsigned long long here = (unsigned long long)w.row_tiles * w.tiles * p.kv_heads;
        if (rest >= here) {
            rest -= here;
            ++b;
            continue;
        }
        uint32_t unit = rest >> 32 ? (uint32_t)(rest / w.tiles) : (uint32_t)rest / w.tiles;
        const uint32_t tile0 = (uint32_t)(rest - (unsigned long long)unit * w.tiles);
        const uint32_t left = (uint32_t)min(end - at, 0xffffffffull);
        // Whole units that follow one another in a sequence: a warp takes one alone, which saves the merge
        // (with fewer units than warps it must be worth the warps that have none).
        uint32_t units = 1;
        if (tile0 == 0 && w.tiles <= left / 2)
            units = min(min((uint32_t)kWarps, left / w.tiles), w.row_tiles * p.kv_heads - unit);
        const bool alone = units > 1 && w.tiles * (kWarps - units) <= kAlone;
        if (alone) unit += min(warp, units - 1);
        else units = 1;
        const uint32_t h = unit / w.row_tiles, row0 = (unit - h * w.row_tiles) * kRows;
        const uint32_t count = alone ? (warp < units ? w.tiles : 0u) : min(w.tiles - tile0, left);
        const uint32_t first = alone ? 0u : warp, stride = alone ? 1u : (uint32_t)kWarps;
        const uint32_t rows = (uint32_t)s.fresh * p.share;
        const int seen0 = s.length - s.fresh + 1;  // keys that the first token sees

        uint32_t q[kTilesN][16];
        int limit[kTilesN][2];
#pragma unroll
        for (int n = 0; n < kTilesN; ++n) {
            const uint32_t r = row0 + 8 * n + g, token = r / p.share;
            const uint16_t *from =
                p.q + ((size_t)(s.start + token) * p.heads + h * p.share + (r - token * p.share)) * kDim + 8 * t;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint4 v = load16(from + 32 * i, r < rows);
                q[n][4 * i] = v.x, q[n][4 * i + 1] = v.y, q[n][4 * i + 2] = v.z, q[n][4 * i + 3] = v.w;
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const uint32_t x = row0 + 8 * n + 2 * t + i;
                limit[n][i] = x < rows ? seen0 + (int)(x / p.share) : 0;
            }
        }

        float o[kTilesN][8][4] = {};
        float m[kTilesN][2], l[kTilesN][2];
#pragma unroll
        for (int n = 0; n < kTilesN; ++n)
#pragma unroll
            for (int i = 0; i < 2; ++i) m[n][i] = -INFINITY, l[n][i] = 0.0f;

        uint4 k[2][4];
        size_t pool = 0;
        const auto load_k = [&](uint32_t tile) {
            const uint32_t key = tile * kKeys;
            if (key < (uint32_t)s.length) pool = paged::pool_row(p.cache, b, key) * row_elements + h * kDim;
#pragma unroll
            for (int r = 0; r < 2; ++r)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    k[r][i] = load16(p.k_pages + pool + (g + 8 * r) * row_elements + 8 * t + 32 * i,
                                     (int)(key + g + 8 * r) < s.length);
        };
        if (first < count) load_k(tile0 + first);
        for (uint32_t i_tile = first; i_tile < count; i_tile += stride) {
            const int key0 = (int)((tile0 + i_tile) * kKeys);
            uint4 v[4][2];  // keys 2t, 2t + 1, 2t + 8, 2t + 9; dimensions 8g.. and 64 + 8g..
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int key = 2 * t + (i & 1) + 8 * (i >> 1);
#pragma unroll
                for (int d = 0; d < 2; ++d)
                    v[i][d] = load16(p.v_pages + pool + key * row_elements + 64 * d + 8 * g,
                                     key0 + key < s.length);
            }
            float sc[kTilesN][4] = {};
#pragma unroll
            for (int i = 0; i < 8; ++i)
#pragma unroll
                for (int n = 0; n < kTilesN; ++n)
                    mma(sc[n], word(k[0][i >> 1], 2 * (i & 1)), word(k[1][i >> 1], 2 * (i & 1)),
                        word(k[0][i >> 1], 2 * (i & 1) + 1), word(k[1][i >> 1], 2 * (i & 1) + 1),
                        q[n][2 * i], q[n][2 * i + 1]);
            if (i_tile + stride < count) load_k(tile0 + i_tile + stride);

            uint32_t pr[kTilesN][2];
#pragma unroll
            for (int n = 0; n < kTilesN; ++n) {
                float alpha[2];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    // row 2t + i: keys g and g + 8
                    float lo = key0 + (int)g < limit[n][i] ? sc[n][i] * p.scale_log2 : -INFINITY;
                    float hi = key0 + 8 + (int)g < limit[n][i] ? sc[n][2 + i] * p.scale_log2 : -INFINITY;
                    float top = fmaxf(lo, hi);
#pragma unroll
                    for (int off = 4; off < 32; off <<= 1)
                        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
                    const float m_new = fmaxf(m[n][i], top), ref = m_new == -INFINITY ? 0.0f : m_new;
                    alpha[i] = fast_exp2(m[n][i] - ref);
                    m[n][i] = m_new;
                    lo = fast_exp2(lo - ref);
                    hi = fast_exp2(hi - ref);
                    l[n][i] = fmaf(l[n][i], alpha[i], lo + hi);
                    sc[n][i] = lo;
                    sc[n][2 + i] = hi;
                }
                pr[n][0] = transposed(pack_bf16(sc[n][0], sc[n][1]));
                pr[n][1] = transposed(pack_bf16(sc[n][2], sc[n][3]));
                if (__any_sync(0xffffffffu, alpha[0] != 1.0f || alpha[1] != 1.0f)) {
#pragma unroll
                    for (int i = 0; i < 8; ++i)
#pragma unroll
                        for (int e = 0; e < 4; ++e) o[n][i][e] *= alpha[e & 1];
                }
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const uint32_t sel = (i & 1) ? 0x7632u : 0x5410u;
                const uint32_t a0 = __byte_perm(word(v[0][0], i >> 1), word(v[1][0], i >> 1), sel);
                const uint32_t a1 = __byte_perm(word(v[0][1], i >> 1), word(v[1][1], i >> 1), sel);
                const uint32_t a2 = __byte_perm(word(v[2][0], i >> 1), word(v[3][0], i >> 1), sel);
                const uint32_t a3 = __byte_perm(word(v[2][1], i >> 1), word(v[3][1], i >> 1), sel);
#pragma unroll
                for (int n = 0; n < kTilesN; ++n) mma(o[n][i], a0, a1, a2, a3, pr[n][0], pr[n][1]);
            }
        }

        if (alone) {
            if (warp < units) {
#pragma unroll
                for (int n = 0; n < kTilesN; ++n)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        float sum = l[n][i];
#pragma unroll
                        for (int off = 4; off < 32; off <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
                        const uint32_t r = row0 + 8 * n + 2 * t + i;
                        if (r >= rows) continue;
                        const float inv = inverse(sum);
                        const uint32_t token = r / p.share, head = r - token * p.share;
                        uint16_t *to =
                            p.out + ((size_t)(s.start + token) * p.heads + h * p.share + head) * kDim + 8 * g;
#pragma unroll
                        for (int d = 0; d < 2; ++d)
                            *reinterpret_cast<uint4 *>(to + 64 * d) =
                                make_uint4(pack_bf16(o[n][0][2 * d + i] * inv, o[n][1][2 * d + i] * inv),
                                           pack_bf16(o[n][2][2 * d + i] * inv, o[n][3][2 * d + i] * inv),
                                           pack_bf16(o[n][4][2 * d + i] * inv, o[n][5][2 * d + i] * inv),
                                           pack_bf16(o[n][6][2 * d + i] * inv, o[n][7][2 * d + i] * inv));
                    }
            }
            at += (unsigned long long)units * w.tiles;
            rest += (unsigned long long)units * w.tiles;
            continue;
        }
        // The warps' results, merged by all threads.
#pragma unroll
        for (int n = 0; n < kTilesN; ++n)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int r = 8 * n + 2 * t + i;
                float sum = l[n][i];
#pragma unroll
                for (int off = 4; off < 32; off <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
                if (g == 0) merge_m[warp][r] = m[n][i], merge_l[warp][r] = sum;
#pragma unroll
                for (int d = 0; d < 2; ++d)
#pragma unroll
                    for (int e = 0; e < 8; e += 4)
                        *reinterpret_cast<float4 *>(&merge_o[warp][r][64 * d + 8 * g + e]) =
                            make_float4(o[n][e][2 * d + i], o[n][e + 1][2 * d + i],
                                        o[n][e + 2][2 * d + i], o[n][e + 3][2 * d + i]);
            }
        __syncthreads();
        // A unit that this CTA has from end to end is written out; a part goes to the workspace: the
        // CTA's second slot if the unit starts here, the first if it started in an earlier CTA.
        const unsigned long long unit_at = at - tile0;
        const unsigned long long unit_end = unit_at + w.tiles - 1;
        const bool wide = (unit_end | run) >> 32;
        const uint32_t cta0 = wide ? (uint32_t)(unit_at / run) : (uint32_t)unit_at / (uint32_t)run;
        const uint32_t cta1 = wide ? (uint32_t)(unit_end / run) : (uint32_t)unit_end / (uint32_t)run;
        const bool whole = cta0 == cta1;
        float *part = p.partials + (size_t)(2 * blockIdx.x + (tile0 == 0)) * kPartial;
        for (uint32_t r = warp; r < (uint32_t)kRows && row0 + r < rows; r += kWarps) {
            float top = merge_m[0][r];
#pragma unroll
            for (int i = 1; i < kWarps; ++i) top = fmaxf(top, merge_m[i][r]);
            const float ref = top == -INFINITY ? 0.0f : top;
            float sum = 0.0f;
            float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int i = 0; i < kWarps; ++i) {
                const float f = fast_exp2(merge_m[i][r] - ref);
                const float4 y = *reinterpret_cast<const float4 *>(&merge_o[i][r][4 * lane]);
                sum = fmaf(f, merge_l[i][r], sum);
                x.x = fmaf(f, y.x, x.x), x.y = fmaf(f, y.y, x.y);
                x.z = fmaf(f, y.z, x.z), x.w = fmaf(f, y.w, x.w);
            }
            if (whole) {
                const float inv = inverse(sum);
                const uint32_t token = (row0 + r) / p.share, head = row0 + r - token * p.share;
                *reinterpret_cast<uint2 *>(
                    p.out + ((size_t)(s.start + token) * p.heads + h * p.share + head) * kDim + 4 * lane) =
                    make_uint2(pack_bf16(x.x * inv, x.y * inv), pack_bf16(x.z * inv, x.w * inv));
            } else {
                __stcg(reinterpret_cast<float4 *>(part + r * kDim) + lane, x);
                if (lane == 0)
                    __stcg(reinterpret_cast<float2 *>(part + kMostRows * kDim) + r, make_float2(top, sum));
            }
        }
        if (!whole) {
            __threadfence();
            __syncthreads();
            if (tid == 0) {
                const uint32_t arrived = atomicAdd(p.counters + cta0, 1u);
                last_one = arrived == cta1 - cta0;
                if (last_one) p.counters[cta0] = 0;
            }
            __syncthreads();
            if (last_one) {
                __threadfence();
                // First the weights of all parts, a lane for each: loads behind a running maximum would
                // wait for one another (55 parts: 25 us).  Then their sum; with fewer rows than warps,
                // several warps share a row's parts.  No part is left out for a weight of 0: what is NaN in it
                // (all its scores, of which the maximum knows nothing, or a value) is NaN in the result.  Nor is
                // there a branch around one, behind which loads would wait for one another: four layers
                // of one sequence of 8000 keys 78 us, with a branch 86, where it leaves the loop 108.
                const uint32_t parts = cta1 - cta0 + 1, here_rows = min((uint32_t)kRows, rows - row0);
                float *weights = &merge_o[0][0][0];  // [row][part]: room for kMostCtas parts of every row
                const auto part_of = [&](uint32_t c) {
                    return p.partials + (size_t)(2 * (cta0 + c) + (c == 0)) * kPartial;
                };
                for (uint32_t r = warp; r < here_rows; r += kWarps) {
                    float top = -INFINITY, sum = 0.0f;
                    for (uint32_t c = lane; c < parts; c += 32) {
                        const float2 ml =
                            __ldcg(reinterpret_cast<const float2 *>(part_of(c) + kMostRows * kDim) + r);
                        weights[r * parts + c] = ml.x;
                        const float m_new = fmaxf(top, ml.x), ref = m_new == -INFINITY ? 0.0f : m_new;
                        sum = sum * fast_exp2(top - ref) + ml.y * fast_exp2(ml.x - ref);
                        top = m_new;
                    }
                    float all = top;
#pragma unroll
                    for (int off = 1; off < 32; off <<= 1)
                        all = fmaxf(all, __shfl_xor_sync(0xffffffffu, all, off));
                    const float ref = all == -INFINITY ? 0.0f : all;
                    sum *= fast_exp2(top - ref);
#pragma unroll
                    for (int off = 1; off < 32; off <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
                    for (uint32_t c = lane; c < parts; c += 32)
                        weights[r * parts + c] = fast_exp2(weights[r * parts + c] - ref);
                    if (lane == 0) merge_l[0][r] = inverse(sum);
                }
                __syncthreads();
                const uint32_t sharers = here_rows < (uint32_t)kWarps ? kWarps / here_rows : 1u;
                float4 *shared_sums = reinterpret_cast<float4 *>(&merge_o[kWarps - 1][0][0]);  // [warp][lane]
                for (uint32_t r0 = 0; r0 < here_rows; r0 += kWarps / sharers) {
                    const uint32_t r = r0 + warp / sharers, share = warp % sharers;
                    const bool mine = r < here_rows && warp / sharers < kWarps / sharers;
                    float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    if (mine) {
                        constexpr uint32_t kAhead = 8;
                        for (uint32_t c = share; c < parts; c += kAhead * sharers) {
                            float4 y[kAhead];
#pragma unroll
                            for (uint32_t i = 0; i < kAhead; ++i)
                                y[i] = __ldcg(reinterpret_cast<const float4 *>(
                                                  part_of(min(c + i * sharers, parts - 1)) + r * kDim) +
                                              lane);
#pragma unroll
                            for (uint32_t i = 0; i < kAhead; ++i) {
                                const uint32_t from = c + i * sharers;
                                const float f = from < parts ? weights[r * parts + from] : 0.0f;
                                if (from >= parts) y[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                                x.x = fmaf(f, y[i].x, x.x), x.y = fmaf(f, y[i].y, x.y);
                                x.z = fmaf(f, y[i].z, x.z), x.w = fmaf(f, y[i].w, x.w);
                            }
                        }
                    }
                    if (sharers > 1) {
                        __syncthreads();  // (the weights have been read)
                        shared_sums[tid] = x;
                        __syncthreads();
                        if (mine && share == 0)
                            for (uint32_t i = 1; i < sharers; ++i) {
                                const float4 y = shared_sums[tid + 32 * i];
                                x.x += y.x, x.y += y.y, x.z += y.z, x.w += y.w;
                            }
                    }
                    if (mine && share == 0) {
                        const float inv = merge_l[0][r];
                        const uint32_t token = (row0 + r) / p.share, head = row0 + r - token * p.share;
                        *reinterpret_cast<uint2 *>(p.out +
                                                   ((size_t)(s.start + token) * p.heads + h * p.share + head) * kDim +
                                                   4 * lane) =
                            make_uint2(pack_bf16(x.x * inv, x.y * inv), pack_bf16(x.z * inv, x.w * inv));
                    }
                }
            }
        }
        __syncthreads();  // (merge_* are written anew)
        at += count;
        rest += count;
    }
    if (p.beside) sm100::grid_wait();
}

unsigned most_ctas(int sm_count) {
    const unsigned ctas = (unsigned)(sm_count > 0 ? sm_count : 148) * kCtasPerSm;
    return ctas < kMostCtas ? ctas : kMostCtas;
}

}  // namespace

extern "C" size_t qwcu_paged_few_workspace_bytes(int sm_count) {
    const size_t ctas = most_ctas(sm_count);
    return ctas * 2 * kPartial * sizeof(float) + ctas * sizeof(uint32_t);
}

extern "C" int qwcu_paged_few_launch(const qwcu_paged_args *a, uint32_t most_rows, int beside_chunks,
                                     void *workspace, int sm_count, qwcu_stream stream_) {
    cudaStream_t stream = static_cast<cudaStream_t>(stream_);
    if (!a->tokens || !a->cache.batch || !a->heads || !a->kv_heads || a->heads % a->kv_heads ||
        a->cache.page_shift < 4 || !a->cache.pool_pages)
        return (int)cudaErrorInvalidValue;
    const unsigned ctas = most_ctas(sm_count);
    Params p;
    p.q = static_cast<const uint16_t *>(a->q);
    p.k_pages = static_cast<const uint16_t *>(a->k_pages);
    p.v_pages = static_cast<const uint16_t *>(a->v_pages);
    p.out = static_cast<uint16_t *>(a->out);
    p.heads = a->heads;
    p.kv_heads = a->kv_heads;
    p.share = a->heads / a->kv_heads;
    p.most_rows = most_rows;
    p.beside = beside_chunks;
    p.scale_log2 = a->scale * 1.4426950408889634f;
    p.partials = static_cast<float *>(workspace);
    p.counters = reinterpret_cast<uint32_t *>(p.partials + (size_t)ctas * 2 * kPartial);
    p.cache = {a->cache.page_table, a->cache.token_start, a->cache.cache_len, a->cache.batch, a->tokens,
               a->cache.table_width, a->cache.page_shift, a->cache.pool_pages, a->cache.status};
    const bool narrow = (unsigned long long)a->max_new * p.share <= 8 || most_rows <= 8;
    return sm100::launch(narrow ? qw_paged_few_kernel<1> : qw_paged_few_kernel<2>,
                         narrow ? ctas : ctas / kCtasPerSm * 2, kThreads, 0, 1, stream, p);
}
