// Attention of chunks of new tokens over a paged K/V cache, on the tensor cores (tcgen05).
//
//   o = softmax(scale * q K^T) V over the cache rows a token sees: those before it and its own.
//
// The softmax, the MMAs and the CTA's form are those of qw_attn_sm100.cu (running maximum; P rounded to bf16
// for P V, 2^-8 of a weight at most: what that leaves as a second operand would be half as many MMAs again, and
// longer in the softmax that bounds the kernel).  What is different here:
//   rows   The query heads of a kv head, token by token, are the rows of a 128-row sub-tile (as many
//          whole tokens as fit): K and V are read once for all of them, the causal edge of a chunk cuts
//          128 / share tokens' tiles and not 128 tokens', and a chunk of 16 tokens fills a sub-tile.
//          One TMA box of 64 columns x share heads x tokens brings them in that order.
//   keys   A tile of 128 keys is fetched page by page, a lane of the producer warp for each page, the
//          page table's entries for the next tile read ahead.  Pages past the sequence's end are not
//          read, and rows past it in its last page may hold anything: masked scores need no care,
//          but 0 * NaN would reach the result through P V, so a warp of its own zeroes those rows of
//          the last V tile between its arrival and its release to the MMAs.
//   parts  A unit is a (sequence, kv head, two sub-tiles of rows).  Where there are fewer units than SMs,
//          a unit's key tiles are divided over several CTAs, whose results are merged by a second kernel.
//          A unit of one sub-tile's rows runs in split form, half of its tiles for each warpgroup.
// Sequence lengths are device data: every CTA works out from them which unit is its own.
//
// What bounds it: the softmax, as in qw_attn_sm100.cu: 1.95 us for a step of 256 rows x 128 keys, the tensor
// pipe 60 % active.  2048 tokens over 16384 keys, 32 heads: 459 us (1.12 PFLOP/s), of which the second wave
// of 256 units on 148 SMs is a part; 4096 tokens over nothing 143 us; 300 over 8000 72 us; 100 over 3000
// 40 us.  Not kept: CTAs that stay and take even runs of key tiles (447, 189 and 88 us for the first three),
// parts chosen by each sequence's own length (58 for the last); both pay for code in front of the first load.
#include <cuda_bf16.h>
#include <stdint.h>

#include "qw_attn_tile.cuh"
#include "qw_paged.cuh"

namespace {

using namespace attn;

constexpr int kFixWarp = 10;
constexpr int kLeastTiles = 6;  // key tiles of a part: a CTA's fixed part costs as much
constexpr int kWarps = kThreads / 32;

struct Params {
    uint32_t *status;
    float scale_log2;
    int mma_probes;
    long long wait_cycles;
    int withhold_from;
    __nv_bfloat16 *out;
    uint32_t heads, kv_heads, share, tile_tokens;  // tokens of a sub-tile
    uint32_t least_rows;  // sequences with fewer query rows are another kernel's
    uint32_t sms;
    int divide;  // units may be divided over CTAs (the merging kernel follows)
    float *part_o;   // [CTA][256][128]
    float2 *part_ml; // [CTA][256]
    paged::Cache cache;
};

struct Unit {
    uint32_t b, block, h;   // block: the rows' place in the sequence
    uint32_t parts;         // CTAs that share the launch's units, P of each
    int active;
    int more;               // kSeveral: this CTA has another one
};

struct __align__(16) Extra {
    Mbar fix;              // V of the sequence's last tile has landed
    uint32_t fix_slot;     // in this ring slot
    unsigned long long scan[kWarps];
    Unit unit;
};

constexpr size_t kSmem = kSmemBytes + sizeof(Extra) + 16;

// Blocks of rows that a sequence gives.
__device__ __forceinline__ uint32_t blocks_of(const Params &p, const paged::Sequence &s) {
    if ((unsigned long long)s.fresh * p.share < p.least_rows) return 0;
    return ((uint32_t)s.fresh + 2 * p.tile_tokens - 1) / (2 * p.tile_tokens);
}

// Unit of CTA `index` when every unit has P CTAs, with P so that all SMs have one; by all threads
// of the CTA.  Units of a sequence stand together, its last blocks, which see the most keys, first.
template <int kCtaWarps, bool kSeveral>
__device__ __forceinline__ void find_unit(const Params &p, uint32_t index, unsigned long long *scan,
                                          Unit *unit) {
    const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5;
    const uint32_t batch = p.cache.batch, per = (batch + kCtaWarps * 32 - 1) / (kCtaWarps * 32);
    const uint32_t first = min(tid * per, batch), end = min(first + per, batch);
    unsigned long long mine = 0;
    for (uint32_t b = first; b < end; ++b)
        mine += (unsigned long long)blocks_of(p, paged::sequence(p.cache, b)) * p.kv_heads;
    unsigned long long before = mine;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
        const unsigned long long v = __shfl_up_sync(0xffffffffu, before, off);
        if (lane >= off) before += v;
    }
    if (lane == 31) scan[warp] = before;
    before -= mine;
    if (tid == 0) unit->active = 0;
    __syncthreads();
    unsigned long long total = 0;
#pragma unroll
    for (int i = 0; i < kCtaWarps; ++i) {
        if (i < (int)warp) before += scan[i];
        total += scan[i];
    }
    const uint32_t parts = p.divide && total && total < p.sms ? p.sms / (uint32_t)total : 1u;
    const unsigned long long mine_unit = index / parts;
    if (kSeveral && tid == 0) unit->more = mine_unit + gridDim.x < total;
    if (mine_unit >= before && mine_unit < before + mine) {
        unsigned long long rest = mine_unit - before;
        for (uint32_t b = first;; ++b) {
            const uint32_t blocks = blocks_of(p, paged::sequence(p.cache, b));
            const unsigned long long here = (unsigned long long)blocks * p.kv_heads;
            if (rest < here) {
                unit->b = b;
                unit->block = blocks - 1 - (uint32_t)(rest / p.kv_heads);
                unit->h = (uint32_t)(rest % p.kv_heads);
                unit->parts = parts;
                unit->active = 1;
                break;
            }
            rest -= here;
        }
    }
    __syncthreads();
}

// The same for a batch of one sequence, by each thread for itself.  (A launch reads its code anew, line by line
// from L2: what a CTA runs once in front of its first load costs more than its instructions.)
template <bool kSeveral>
__device__ __forceinline__ Unit unit_of_one(const Params &p, uint32_t index, const paged::Sequence &s) {
    const uint32_t blocks = blocks_of(p, s), total = blocks * p.kv_heads;
    Unit u;
    u.b = 0;
    u.parts = p.divide && total && total < p.sms ? p.sms / total : 1u;
    const uint32_t at = index / u.parts;
    u.active = at < total;
    u.more = kSeveral && at + gridDim.x < total;
    u.block = blocks - 1 - at / p.kv_heads;
    u.h = at % p.kv_heads;
    return u;
}

// What a unit has to do: its tokens and the key tiles that any of its rows sees.
struct Plan {
    uint32_t token0;      // within the sequence
    uint32_t tokens;
    int tiles, parts;     // parts: CTAs that take some of the tiles
    bool split;
};
__device__ __forceinline__ Plan plan_of(const Params &p, const Unit &u, const paged::Sequence &s) {
    Plan x;
    x.token0 = u.block * 2 * p.tile_tokens;
    x.tokens = min(2 * p.tile_tokens, (uint32_t)s.fresh - x.token0);
    const int seen = max(0, s.length - s.fresh + (int)(x.token0 + x.tokens));
    x.tiles = (seen + kTileN - 1) / kTileN;
    x.parts = max(1, min((int)u.parts, x.tiles / kLeastTiles));
    x.split = x.tokens <= p.tile_tokens;
    return x;
}

// Row r of a sub-tile whose first token is `token0`: its token, or none.
__device__ __forceinline__ bool row_token(const Params &p, uint32_t r, uint32_t token0, uint32_t fresh,
                                          uint32_t &token) {
    const uint32_t t = r / p.share;
    token = token0 + t;
    return t < p.tile_tokens && token < fresh;
}

// 32 rows of a warp out of TMEM, as write_rows does it: final ones to their tokens' heads, parts as
// fp32 in the order of the rows.  where: for each of a lane's four rows the element of `out`, or < 0.
__device__ __noinline__ void write_tokens(uint32_t tmem_own, uint32_t tmem_other, float w_own,
                                          float w_other, float inv, uint32_t box, __nv_bfloat16 *out,
                                          longlong2 where01, longlong2 where23) {
    const uint32_t lane = threadIdx.x & 31u, first = lane >> 2, piece = lane & 3u;
#pragma unroll 1
    for (uint32_t c = 0; c < (uint32_t)kHeadDim; c += 32) {
        const uint32_t at = box + (c & 32u) * 64u;
        uint32_t o[32];
        if (tmem_own != kNoTmem) {
            QW_TMEM_LD32(tmem_own + c, o);
            QW_TMEM_WAIT_LD32(o);
        } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = 0u;
        }
        if (tmem_other != kNoTmem) {
            uint32_t x[32];
            QW_TMEM_LD32(tmem_other + c, x);
            QW_TMEM_WAIT_LD32(x);
#pragma unroll
            for (int i = 0; i < 32; ++i)
                o[i] = __float_as_uint(
                    fmaf(__uint_as_float(x[i]), w_other, __uint_as_float(o[i]) * w_own));
        } else if (w_own != 1.0f) {
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * w_own);
        }
#pragma unroll
        for (uint32_t c16 = 0; c16 < 4; ++c16) {
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
                w[i] = pack_bf16(__uint_as_float(o[8 * c16 + 2 * i]) * inv,
                                 __uint_as_float(o[8 * c16 + 2 * i + 1]) * inv);
            st_shared16(at + lane * 64u + ((c16 ^ ((lane >> 1) & 3u)) << 4), w[0], w[1], w[2], w[3]);
        }
        __syncwarp();
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) {
            const uint32_t r = 8u * i + first;
            const uint4 x = ld_shared16(at + r * 64u + ((piece ^ ((r >> 1) & 3u)) << 4));
            const long long to = i == 0 ? where01.x : i == 1 ? where01.y : i == 2 ? where23.x : where23.y;
            if (to >= 0) *reinterpret_cast<uint4 *>(out + to + c + piece * 8u) = x;
        }
    }
}
__device__ __noinline__ void write_part(uint32_t tmem_own, uint32_t tmem_other, float w_own,
                                        float w_other, uint32_t box, float *out) {
    const uint32_t lane = threadIdx.x & 31u, first = lane >> 3, piece = lane & 7u;
#pragma unroll 1
    for (uint32_t c = 0; c < (uint32_t)kHeadDim; c += 32) {
        uint32_t o[32];
        if (tmem_own != kNoTmem) {
            QW_TMEM_LD32(tmem_own + c, o);
            QW_TMEM_WAIT_LD32(o);
        } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = 0u;
        }
        if (tmem_other != kNoTmem) {
            uint32_t x[32];
            QW_TMEM_LD32(tmem_other + c, x);
            QW_TMEM_WAIT_LD32(x);
#pragma unroll
            for (int i = 0; i < 32; ++i)
                o[i] = __float_as_uint(
                    fmaf(__uint_as_float(x[i]), w_other, __uint_as_float(o[i]) * w_own));
        } else if (w_own != 1.0f) {
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * w_own);
        }
        __syncwarp();  // (the columns before have been read)
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i)
            st_shared16(box + lane * 128u + ((i ^ (lane & 7u)) << 4), o[4 * i], o[4 * i + 1],
                        o[4 * i + 2], o[4 * i + 3]);
        __syncwarp();
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i) {
            const uint32_t r = 4u * i + first;
            const uint4 x = ld_shared16(box + r * 128u + ((piece ^ (r & 7u)) << 4));
            *reinterpret_cast<uint4 *>(out + r * kHeadDim + c + piece * 4u) = x;
        }
    }
}

// Producer: the whole warp, a lane for each page of a tile.
__device__ __forceinline__ void tma_warp(const Params &p, SharedControl *ctl, Extra *extra,
                                         uint8_t *smem_kv, const CUtensorMap *map_k,
                                         const CUtensorMap *map_v, const Unit &unit, int length,
                                         int begin, bool split) {
    const uint32_t where = 3u << 16, lane = threadIdx.x & 31u;
    const uint32_t shift = p.cache.page_shift;
    const int box_rows = shift < 7 ? 1 << shift : kTileN, boxes = kTileN / box_rows;
    const int col = (int)(unit.h * kHeadDim);
    const int la = ctl->tile_count[0], lb = ctl->tile_count[1];
    const int pairs = split ? la + lb : max(la, lb);
    // The i-th pair of tiles (K, V) to be loaded; split form: a0 b0 a1 b1 ..., the first half's alone
    // where the second has one less.
    const auto tile_of = [&](int i) {
        if (!split) return i;
        return (i & 1) && (i >> 1) < lb ? la + (i >> 1) : (i >> 1);
    };
    // Pool row of a lane's box of a tile, or -1 past the sequence's end.
    const auto pool_row = [&](int u) {
        const int key = (begin + u) * kTileN + (int)lane * box_rows;
        if (u < 0 || (int)lane >= boxes || key >= length) return -1;
        return (int)paged::pool_row(p.cache, unit.b, (uint32_t)key);
    };
    uint32_t t = 0;
    bool ok = true, fixed = false;
    int next = pairs > 0 ? pool_row(tile_of(0)) : -1;
    for (int i = 0; i < pairs && ok; ++i) {
        const int u = tile_of(i), row = next, key0 = (begin + u) * kTileN;
        if (i + 1 < pairs) next = pool_row(tile_of(i + 1));
        if (p.withhold_from >= 0 && u >= p.withhold_from) {
            ok = false;  // the tile stays away: nothing is issued, nothing is in flight
            break;
        }
        const uint32_t bytes =
            (uint32_t)__popc(__ballot_sync(0xffffffffu, row >= 0)) * (uint32_t)box_rows * kHeadDim * 2;
        const bool last = key0 + kTileN > length;  // rows past the end: V goes to the fixing warp first
        for (int which = 0; which < 2 && ok; ++which, ++t) {
            const uint32_t slot = t % kStages, par = ((t / kStages) & 1u) ^ 1u;
            ok = __all_sync(0xffffffffu,
                            mbar_wait(ctl, smem_u32(&ctl->bars[kBarKvEmpty + slot]), par, p.status,
                                      where | (kBarKvEmpty + slot), (uint32_t)u)) != 0;
            if (!ok) break;
            Mbar *bar = &ctl->bars[kBarKvFull + slot];
            if (which && last) {
                bar = &extra->fix;
                fixed = true;
                if (lane == 0) extra->fix_slot = slot;
            }
            if (lane == 0) mbar_expect_tx(bar, bytes);
            __syncwarp();
            if (row >= 0) {
                uint8_t *dst = smem_kv + (size_t)slot * kTileBytes + lane * (uint32_t)box_rows * 128u;
                const CUtensorMap *map = which ? map_v : map_k;
                tma_load_2d<1>(dst, map, smem_u32(bar), col, row);
                tma_load_2d<1>(dst + kHalfTileBytes, map, smem_u32(bar), col + 64, row);
            }
            __syncwarp();
        }
    }
    // Leave no copy in flight (bounded like every other wait).
    if (lane == 0) {
        if (fixed) mbar_drain(&extra->fix, 0, ctl->wait_cycles);
        const uint32_t first = t > (uint32_t)kStages ? t - kStages : 0;
        for (uint32_t u = first; u < t; ++u)
            mbar_drain(&ctl->bars[kBarKvFull + u % kStages], (u / kStages) & 1u, ctl->wait_cycles);
    }
}

// Rows of the sequence's last V tile past its end become zeros.
__device__ __forceinline__ void fix_warp(const Params &p, SharedControl *ctl, Extra *extra,
                                         uint8_t *smem_kv, int length, int tiles) {
    const uint32_t lane = threadIdx.x & 31u;
    // This tile comes after all others: a wait's budget for each.  (Where one of them stays away, the
    // roles that wait for it raise the flag.)
    const long long start = clock64();
    while (!mbar_try(&extra->fix, 0)) {
        if (ctl->abort_flag) break;
        if (clock64() - start > ctl->wait_cycles * (tiles + 1)) {
            record_expiry(ctl, p.status, 4u << 16, 0);
            break;
        }
    }
    if (!__all_sync(0xffffffffu, mbar_try(&extra->fix, 0))) return;
    const uint32_t slot = extra->fix_slot;
    const uint32_t tile = smem_u32(smem_kv + (size_t)slot * kTileBytes);
    const uint32_t from = (uint32_t)(length % kTileN) * 8u;  // 16-byte pieces of 128-byte rows
    for (uint32_t i = from + lane; i < (uint32_t)kTileN * 8u; i += 32) {
        st_shared16(tile + i * 16u, 0, 0, 0, 0);
        st_shared16(tile + kHalfTileBytes + i * 16u, 0, 0, 0, 0);
    }
    fence_async_shared();
    __syncwarp();
    if (lane == 0) mbar_arrive(&ctl->bars[kBarKvFull + slot]);
}

__device__ __forceinline__ void init_barriers(SharedControl *ctl, Extra *extra) {
    for (int i = 0; i < 2; ++i) mbar_init(&ctl->bars[kBarQFull + i], 1);
    for (int i = 0; i < kStages; ++i) {
        mbar_init(&ctl->bars[kBarKvFull + i], 1);
        mbar_init(&ctl->bars[kBarKvEmpty + i], 1);
    }
    for (int i = 0; i < 2; ++i) {
        mbar_init(&ctl->bars[kBarSFull + i], 1);
        mbar_init(&ctl->bars[kBarPFirst + i], kTileM / 32);
        mbar_init(&ctl->bars[kBarPFull + i], kTileM / 32);
        mbar_init(&ctl->bars[kBarOFinal + i], 1);
    }
    mbar_init(&ctl->bars[kBarMerge], kTileM / 32);
    mbar_init(&extra->fix, 1);
    mbar_init_fence();
}

// kSeveral: there may be more units than CTAs, so that a CTA takes several; without it the code is 1 to 3 %
// faster (2048 tokens over 16384 keys: 464 us and 470).
template <bool kSeveral>
__global__ void __launch_bounds__(kThreads, 1)
qw_paged_chunk_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                      const __grid_constant__ CUtensorMap map_v, const Params p) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    uint8_t *smem_q = smem;
    uint8_t *smem_kv = smem + 2 * kTileBytes;
    SharedControl *ctl = reinterpret_cast<SharedControl *>(smem + kSmemData);
    Extra *extra = reinterpret_cast<Extra *>(ctl + 1);

    const int tid = threadIdx.x;
    const int warp = warp_index();
    const int lane = tid & 31;
    if (warp == kTmaWarp && lane == 0) {
        init_barriers(ctl, extra);
        ctl->abort_flag = 0;
        ctl->wait_cycles = p.wait_cycles > 0 ? p.wait_cycles : kWaitCycles;
    }
    if (warp == kMmaWarp) tmem_alloc<1>(&ctl->tmem_base, kTmemCols);
    // Always in this order, unlike in other kernels: the kernel for few rows, which the host launches directly behind
    // this one, reads and writes from its start on and relies on this kernel having waited for all that was before
    // both.  With the trigger ahead of the wait, or another kernel between the two, it would race with that.
    grid_wait();
    grid_launch_dependents();
    uint32_t index = blockIdx.x;
    bool again;
    do {
        Unit unit;
        paged::Sequence s = {0, 0, 0};
        if (p.cache.batch == 1) {
            s = paged::sequence(p.cache, 0);
            unit = unit_of_one<kSeveral>(p, index, s);
        } else {
            find_unit<kWarps, kSeveral>(p, index, extra->scan, &extra->unit);
            unit = extra->unit;
            if (unit.active) s = paged::sequence(p.cache, unit.b);
        }
        Plan plan = {0, 0, 0, 0, false};
        int part = 0;
        if (unit.active) {
            plan = plan_of(p, unit, s);
            part = (int)(index % unit.parts);
        }
        const bool active = unit.active && part < plan.parts;  // the same in all threads
        const int begin = active ? (int)((long long)plan.tiles * part / plan.parts) : 0;
        const int end = active ? (int)((long long)plan.tiles * (part + 1) / plan.parts) : 0;
        const bool split = plan.split;

        int my_limit = 0, sub = 0, tid_in_group = 0;
        uint32_t my_token0 = 0;
        if (active) {
            if (warp == kTmaWarp && lane == 0) {
                for (int i = 0; i < (split ? 1 : 2); ++i) {
                    Mbar *bar = &ctl->bars[kBarQFull + i];
                    mbar_expect_tx(bar, p.tile_tokens * p.share * kHeadDim * 2);
                    uint8_t *dst = smem_q + (size_t)i * kTileBytes;
                    const int head = (int)(unit.h * p.share);
                    const int token = (int)(s.start + plan.token0 + (uint32_t)i * p.tile_tokens);
                    tma_load_3d(dst, &map_q, bar, 0, head, token);
                    tma_load_3d(dst + kHalfTileBytes, &map_q, bar, 64, head, token);
                }
            }
            if (tid < kSoftmaxThreads) {
                sub = tid >> 7;
                tid_in_group = tid & 127;
                my_token0 = plan.token0 + (split ? 0u : (uint32_t)sub * p.tile_tokens);
                uint32_t token;
                const bool real = row_token(p, (uint32_t)tid_in_group, my_token0, (uint32_t)s.fresh, token);
                // (A row of no token is computed like its neighbours and never stored.)
                my_limit = real ? max(0, s.length - s.fresh + (int)token + 1) : 0x7fffffff;
            }
            if (tid < 2) {
                // A sub-tile's last token sees the most.
                const uint32_t first = split ? plan.token0 : plan.token0 + (uint32_t)tid * p.tile_tokens;
                const uint32_t past = min(first + p.tile_tokens, (uint32_t)s.fresh);
                const int tiles = min((max(0, s.length - s.fresh + (int)past) + kTileN - 1) / kTileN, end);
                const int mine = max(0, tiles - begin);
                // Tiles are numbered from the part's first.
                ctl->skip_lo = 0;
                ctl->skip_hi = begin;
                if (!split) {
                    ctl->tile_first[tid] = 0;
                    ctl->tile_count[tid] = mine;
                } else {
                    const int half = (mine + 1) / 2;
                    ctl->tile_first[tid] = tid ? half : 0;
                    ctl->tile_count[tid] = tid ? mine - half : half;
                }
            }
        }
        tc_fence_before();
        __syncthreads();
        tc_fence_after();

        if (active) {
            if (tid < kSoftmaxThreads) {
                asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
                const uint32_t warp_row0 = (uint32_t)(tid_in_group >> 5) * 32u;
                const uint32_t box = smem_u32(smem_q + (size_t)sub * kTileBytes) + warp_row0 * 128u;
                const auto has_rows = []() __attribute__((always_inline)) { return true; };
                const auto store = [&p, &s, &unit, &plan, index, box, warp_row0, tid_in_group, sub, my_token0,
                                    lane](
                                       uint32_t tmem_own, uint32_t tmem_other, float w_own, float w_other,
                                       float inv, float m_row, float l_row) __attribute__((always_inline)) {
                    if (plan.parts > 1) {
                        const size_t row = (size_t)index * (2 * kTileM) + (uint32_t)sub * kTileM;
                        p.part_ml[row + (uint32_t)tid_in_group] = make_float2(m_row, l_row);
                        write_part(tmem_own, tmem_other, w_own, w_other, box,
                                   p.part_o + (row + warp_row0) * kHeadDim);
                        return;
                    }
                    long long where[4];
    #pragma unroll
                    for (uint32_t i = 0; i < 4; ++i) {
                        const uint32_t r = warp_row0 + 8u * i + ((uint32_t)lane >> 2);
                        uint32_t token;
                        const bool real = row_token(p, r, my_token0, (uint32_t)s.fresh, token);
                        where[i] = real ? (long long)(((size_t)(s.start + token) * p.heads +
                                                       unit.h * p.share + r % p.share) *
                                                      kHeadDim)
                                        : -1ll;
                    }
                    write_tokens(tmem_own, tmem_other, w_own, w_other, inv, box, p.out,
                                 make_longlong2(where[0], where[1]), make_longlong2(where[2], where[3]));
                };
                softmax_role<false, true>(p, ctl, sub, tid_in_group, my_limit, 0, 0, split, 0.0f, has_rows,
                                          store);
                if (kSeveral && unit.more) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kLaunchRegs));
            } else {
                asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
            }
            if (tid < kSoftmaxThreads) {
            } else if (warp == kMmaWarp) {
                if (split) mma_role_split(p, ctl, smem_q, smem_kv);
                else mma_role(p, ctl, smem_q, smem_kv);
            } else if (warp == kTmaWarp) {
                tma_warp(p, ctl, extra, smem_kv, &map_k, &map_v, unit, s.length, begin, split);
                // The loads of Q must have landed as well.
                if (lane == 0)
                    for (int i = 0; i < (split ? 1 : 2); ++i)
                        mbar_drain(&ctl->bars[kBarQFull + i], 0, ctl->wait_cycles);
            } else if (warp == kFixWarp) {
                // The tile that holds the end, if it is one of this CTA's and the end is inside it.
                const int visited =
                    split ? ctl->tile_count[0] + ctl->tile_count[1] : max(ctl->tile_count[0], ctl->tile_count[1]);
                const int last = s.length / kTileN;
                if (s.length % kTileN && last >= begin && last < begin + visited)
                    fix_warp(p, ctl, extra, smem_kv, s.length, visited);
            }
            if (kSeveral && tid >= kSoftmaxThreads && unit.more) {
                __syncwarp();
                asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kLaunchRegs));
            }
        }

        if (kSeveral && unit.more) fence_async_shared();  // (the rows' staging is where the next Q lands)
        tc_fence_before();
        __syncthreads();
        // The next unit, with everything as at the start.
        again = kSeveral && unit.more && !ctl->abort_flag;
        if (again) {
            index += gridDim.x;
            if (warp == kTmaWarp && lane == 0) {
                for (int i = 0; i < kBarCount; ++i) mbar_inval(&ctl->bars[i]);
                mbar_inval(&extra->fix);
                init_barriers(ctl, extra);
            }
            tc_fence_after();
        }
    } while (again);
    if (warp == kMmaWarp) {
        tc_fence_after();
        tmem_dealloc<1>(ctl->tmem_base, kTmemCols);
    }
}

// Units whose keys were divided: a warp for a row, its parts in their order.
constexpr int kMergeWarps = 8;
constexpr uint32_t kMergeSlices = 8;  // CTAs of a unit, 32 of its rows each
__global__ void __launch_bounds__(kMergeWarps * 32) qw_paged_merge_kernel(const Params p) {
    __shared__ unsigned long long scan[kMergeWarps];
    __shared__ Unit shared_unit;
    grid_launch_dependents();
    grid_wait();
    const uint32_t index = blockIdx.x / kMergeSlices, slice = blockIdx.x % kMergeSlices;
    // (unit `index` of a launch of at most sms CTAs: its first CTA)
    Unit unit;
    paged::Sequence s;
    if (p.cache.batch == 1) {
        s = paged::sequence(p.cache, 0);
        unit = unit_of_one<false>(p, 0, s);
        if (!unit.active || unit.parts == 1) return;
        unit = unit_of_one<false>(p, index * unit.parts, s);
        if (!unit.active) return;
    } else {
        find_unit<kMergeWarps, false>(p, 0, scan, &shared_unit);
        if (!shared_unit.active || shared_unit.parts == 1) return;
        const uint32_t at = index * shared_unit.parts;
        __syncthreads();
        find_unit<kMergeWarps, false>(p, at, scan, &shared_unit);
        unit = shared_unit;
        if (!unit.active) return;
        s = paged::sequence(p.cache, unit.b);
    }
    const uint32_t parts_of_all = unit.parts;
    const Plan plan = plan_of(p, unit, s);
    if (plan.parts == 1) return;
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
    const uint32_t per = 2 * kTileM / kMergeSlices;
    for (uint32_t r = slice * per + warp; r < (slice + 1) * per; r += kMergeWarps) {
        const uint32_t sub = r / kTileM, in_tile = r % kTileM;
        if (plan.split && sub) break;
        uint32_t token;
        if (!row_token(p, in_tile, plan.token0 + sub * p.tile_tokens, (uint32_t)s.fresh, token)) continue;
        float top = -INFINITY, sum = 0.0f;
        float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        constexpr int kAhead = 4;
        for (int c = 0; c < plan.parts; c += kAhead) {
            float4 y[kAhead];
            float2 ml[kAhead];
#pragma unroll
            for (int i = 0; i < kAhead; ++i) {
                const size_t row =
                    (size_t)(index * parts_of_all + (uint32_t)min(c + i, plan.parts - 1)) * (2 * kTileM) + r;
                y[i] = __ldcg(reinterpret_cast<const float4 *>(p.part_o + row * kHeadDim) + lane);
                ml[i] = __ldcg(p.part_ml + row);
            }
#pragma unroll
            for (int i = 0; i < kAhead; ++i) {
                if (c + i >= plan.parts) break;
                const float m_new = fmaxf(top, ml[i].x), ref = m_new == -INFINITY ? 0.0f : m_new;
                const float f = fast_exp2(top - ref), g = fast_exp2(ml[i].x - ref);
                sum = fmaf(sum, f, ml[i].y * g);
                x.x = fmaf(x.x, f, y[i].x * g), x.y = fmaf(x.y, f, y[i].y * g);
                x.z = fmaf(x.z, f, y[i].z * g), x.w = fmaf(x.w, f, y[i].w * g);
                top = m_new;
            }
        }
        const float inv = sum > 0.0f ? 1.0f / sum : 0.0f;
        *reinterpret_cast<uint2 *>(
            p.out + ((size_t)(s.start + token) * p.heads + unit.h * p.share + in_tile % p.share) * kHeadDim +
            4 * lane) = make_uint2(pack_bf16(x.x * inv, x.y * inv), pack_bf16(x.z * inv, x.w * inv));
    }
}

// [tokens][heads][128], boxes of 64 columns x share heads x tile_tokens tokens.
int make_query_map(CUtensorMap *map, const void *base, uint32_t tokens, uint32_t heads, uint32_t share,
                   uint32_t tile_tokens) {
    EncodeTiledFn fn = encode_tiled_fn();
    if (!fn) return (int)cudaErrorNotSupported;
    const cuuint64_t dims[3] = {kHeadDim, heads, tokens};
    const cuuint64_t strides[2] = {kHeadDim * 2, (cuuint64_t)heads * kHeadDim * 2};
    const cuuint32_t box[3] = {64, share, tile_tokens}, elem[3] = {1, 1, 1};
    const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void *>(base), dims, strides,
                          box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                          CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? 0 : (int)cudaErrorInvalidValue;
}

unsigned sms_of(int sm_count) { return (unsigned)(sm_count > 0 ? sm_count : 148); }

// The opt-in to the shared memory is an attribute of the device: set on first use.
int make_ready() {
    static bool ready[64];
    int dev = 0;
    cudaError_t code = cudaGetDevice(&dev);
    if (code != cudaSuccess) return (int)code;
    const bool tracked = dev >= 0 && dev < 64;
    if (tracked && ready[dev]) return 0;
    for (const auto kernel : {qw_paged_chunk_kernel<false>, qw_paged_chunk_kernel<true>})
        if (code == cudaSuccess)
            code = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmem);
    if (code == cudaSuccess && tracked) ready[dev] = true;
    return (int)code;
}

}  // namespace

extern "C" size_t qwcu_paged_chunk_workspace_bytes(int sm_count) {
    return (size_t)sms_of(sm_count) * 2 * kTileM * (kHeadDim * sizeof(float) + sizeof(float2));
}

namespace {

// Everything but the tensor maps; 0 or a CUDA error.
int make_params(const qwcu_paged_args *a, uint32_t least_rows, void *workspace, int sm_count, Params &p) {
    const uint32_t share = a->kv_heads ? a->heads / a->kv_heads : 0;
    if (!a->tokens || !a->cache.batch || !share || share > (uint32_t)kTileM || a->heads % a->kv_heads ||
        a->cache.page_shift < 4 || !a->cache.pool_pages ||
        ((unsigned long long)a->cache.pool_pages << a->cache.page_shift) > 0x7fffffffull)
        return (int)cudaErrorInvalidValue;
    p.status = a->cache.status;
    p.scale_log2 = a->scale * 1.4426950408889634f;
    p.wait_cycles = a->wait_cycles;
    p.withhold_from = a->withhold_from > 0 ? a->withhold_from : -1;
    const long long budget = p.wait_cycles > 0 ? p.wait_cycles : kWaitCycles;
    p.mma_probes = 32 + (int)min(budget / kProbeCycles, 1ll << 30);
    p.out = static_cast<__nv_bfloat16 *>(a->out);
    p.heads = a->heads;
    p.kv_heads = a->kv_heads;
    p.share = share;
    p.tile_tokens = (uint32_t)kTileM / share;
    p.least_rows = least_rows;
    p.sms = sms_of(sm_count);
    p.part_o = static_cast<float *>(workspace);
    p.part_ml = reinterpret_cast<float2 *>(p.part_o + (size_t)p.sms * 2 * kTileM * kHeadDim);
    p.cache = {a->cache.page_table, a->cache.token_start, a->cache.cache_len, a->cache.batch, a->tokens,
               a->cache.table_width, a->cache.page_shift, a->cache.pool_pages, a->cache.status};
    // A single sequence whose rows, if it has them all, give more units than half the SMs needs no
    // second kernel.
    const uint32_t unit_tokens = 2 * p.tile_tokens;
    p.divide = p.sms > 1 && !(a->cache.batch == 1 && a->max_new >= a->tokens &&
                              2ull * a->kv_heads * ((a->tokens + unit_tokens - 1) / unit_tokens) > p.sms);
    return 0;
}

}  // namespace

extern "C" int qwcu_paged_chunk_launch(const qwcu_paged_args *a, uint32_t least_rows, void *workspace,
                                       int sm_count, qwcu_stream stream) {
    Params p;
    int rc = make_params(a, least_rows, workspace, sm_count, p);
    if (rc || (rc = make_ready())) return rc;
    CUtensorMap map_q, map_k, map_v;
    const uint32_t box_rows = a->cache.page_shift < 7 ? 1u << a->cache.page_shift : (uint32_t)kTileN;
    const uint32_t cols = a->kv_heads * kHeadDim, pool_rows = a->cache.pool_pages << a->cache.page_shift;
    if ((rc = make_query_map(&map_q, a->q, a->tokens, a->heads, p.share, p.tile_tokens))) return rc;
    if ((rc = make_map_2d(&map_k, a->k_pages, pool_rows, cols, box_rows))) return rc;
    if ((rc = make_map_2d(&map_v, a->v_pages, pool_rows, cols, box_rows))) return rc;
    // Units: full ones, and a last, partly filled block of each sequence that is not the other kernel's.
    // Most sequences may well be that one's, and CTAs without a unit cost 2.5 us each: where their number
    // could pass two of every SM, one of every SM is all there are, and CTAs with several units take them
    // one after the other (255 single tokens over 200 keys beside a chunk of 128: 59.9 us, with a CTA for
    // every unit there can be 77.6; 999 over 64 beside one of 32: 128 and 236).
    const uint32_t unit_tokens = 2 * p.tile_tokens, least = (least_rows + p.share - 1) / p.share;
    const uint32_t most = least ? a->tokens / least : a->tokens;
    const unsigned long long sequences = a->cache.batch < most ? a->cache.batch : most;
    const unsigned long long whole = (unsigned long long)(a->tokens / unit_tokens) * a->kv_heads;
    const unsigned long long last = sequences * a->kv_heads;
    if (whole + last > 0x3fffffffull) return (int)cudaErrorInvalidValue;
    const bool several = last > 2 * p.sms;
    const unsigned units = (unsigned)(whole + (several ? p.sms : last));
    const unsigned grid = units > p.sms ? units : p.sms;
    const auto kernel = several ? qw_paged_chunk_kernel<true> : qw_paged_chunk_kernel<false>;
    return launch(kernel, grid, kThreads, kSmem, 1, static_cast<cudaStream_t>(stream), map_q,
                  map_k, map_v, p);
}

extern "C" int qwcu_paged_merge_launch(const qwcu_paged_args *a, uint32_t least_rows, void *workspace,
                                       int sm_count, qwcu_stream stream, int *launched) {
    Params p;
    *launched = 0;
    const int rc = make_params(a, least_rows, workspace, sm_count, p);
    if (rc || !p.divide) return rc;
    *launched = 1;
    // (units of two parts and more: at most one for every two SMs)
    return launch(qw_paged_merge_kernel, p.sms / 2 * kMergeSlices, kMergeWarps * 32, 0, 1,
                  static_cast<cudaStream_t>(stream), p);
}
