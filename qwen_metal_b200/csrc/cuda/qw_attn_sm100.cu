// Block-causal (prefix-visible) flash-attention forward for sm_100a.
//
// One CTA owns 256 query rows of one (batch, head): two 128-row sub-tiles that
// ping-pong on the tensor pipe.  Q/K/V tiles arrive through TMA (128B swizzle)
// into shared memory; S = Q K^T and O += P V run as tcgen05.mma with fp32
// accumulators in tensor memory (TMEM); the softmax is fp32 in the exp2 domain,
// one thread per query row, and writes P back to TMEM as bf16 over the S
// columns so P V reads its A operand straight from TMEM.
//
// Warp roles (384 threads = 3 warpgroups; registers are moved from the third
// warpgroup to the two softmax warpgroups with setmaxnreg):
//   warps 0-3   softmax + epilogue of sub-tile 0 (TMEM lanes 0..127)
//   warps 4-7   softmax + epilogue of sub-tile 1
//   warp  8     MMA issue (all lanes run the loop, one is elected per issue), TMEM allocation
//   warp  9     TMA producer (one elected lane)
//   warps 10-11 idle (they only complete the third warpgroup)
//
// Mask: every row has an integer key limit (prefix) and the batch item may have
// a key-padding window.  Key tiles past the largest limit of a sub-tile are
// never issued, key tiles that lie completely inside the padding window are
// skipped by all roles, interior tiles run without a compare, boundary tiles have their
// scores masked (see mask_scores).
//
// Epilogue: O / l is rounded to bf16 and goes through the (by then dead) Q tile in shared
// memory to global memory, every warp its own 32 rows (write_rows).  When the heads
// are sharded over several GPUs the rows go to this rank's head columns of a
// full-width output (the kernel can address several such destinations, peer-
// mapped ones included); the multi-GPU group writes the rank's own buffer here
// and carries the columns to the peers with a push kernel under the next layer,
// because with a single wave of CTAs all peer stores would leave at the kernel's
// end as one exposed burst.  At its start the kernel then opens the output slot's
// next epoch for the peers' pushes.
//
// Softmax.  Callers that promise bounded row norms (the DiT layer's QK-norm) get
// P = exp2(score*c - bound) against one fixed exponent: no row maximum, no
// rescaling, scores streamed out of TMEM in 32-column chunks.  Other callers get the
// running maximum with lazy rescaling.
//
// Wave tail.  The grid is one CTA per (batch, head, 256-row block), heaviest
// blocks first, and rarely a multiple of the SM count.  The units that would
// form the last, partly filled wave are therefore run in split form, two CTAs per
// unit: a CTA takes 128 of the rows and gives each of its two sub-tiles half of
// the key tiles; at the end warpgroup 0 merges the two accumulators (both sit in
// the same TMEM lanes) with the usual exp2 reweighting.  Twice the CTAs of half
// the length fill the idle SMs, and nothing leaves the CTA unmerged.
//
// Every wait is bounded: when one runs out the CTA records where in the status
// words, raises a shared abort flag that the other waits poll, drains its TMA
// loads, frees its TMEM and returns.  (The MMA warp's waits do not poll it: they count
// probes, and end within the same budget.)
//
// Semantics follow the reference prefix kernel (h3_shaders.metal:3061-3272):
// scale applied to fp32 scores, P rounded to bf16 before P V, fp32 accumulate,
// output acc / l rounded to bf16; rows without a visible key store zeros.

#include <stdio.h>
#include <stdlib.h>
#include <string.h>

#include "qw_sm100.cuh"

namespace {

struct KernelParams {
    const int32_t *kv_limit;
    uint32_t *status;
#ifdef QW_ATTN_TRACE
    unsigned long long *trace;  // event log of block (0,0,0), dumped to $QW_CUDA_ATTN_TRACE
#endif
    int per_batch_limits;
    int causal;
    uint32_t causal_offset;
    uint32_t batch, q_rows, kv_rows, heads, kv_heads;
    uint32_t text_len[8];
    uint32_t text_pad;
    float scale_log2;  // scale * log2(e)
    // Optional promise by the caller (two floats in device memory): every query row
    // has a 2-norm of at most score_bound[0] and every key row of at most
    // score_bound[1], so |q.k| <= their product and the softmax can use one fixed
    // reference exponent instead of a running row maximum.
    const float *score_bound;
    int head_major_out;
    // Sharded runs: the rows are stored at this rank's head columns of n_out
    // full-width outputs (peer-mapped pointers allowed).  out_heads_total is the
    // head count of the destination rows and out_head_offset this rank's first head.
    __nv_bfloat16 *out_peers[8];
    uint32_t n_out, out_heads_total, out_head_offset;
    // Launch geometry: CTA c < total_units - tail_units runs unit c whole; the
    // last tail_units units run in split form, two CTAs each.
    uint32_t n_qblocks, total_units, tail_units;
    // Gather by a separate push: epoch counter of the output slot and the peers'
    // flag words that receive the new epoch when this kernel starts.
    uint32_t *slot_use;
    uint32_t *freed_peer[8];
    uint32_t n_freed;
    // Bounded-wait exercise (tests only): budget in SM cycles (0 = the default) and
    // the first visited key tile the producer does NOT load (< 0: loads everything),
    // so that the waits downstream of it run out and the CTA takes its clean exit.
    long long wait_cycles;
    int withhold_from;
    int mma_probes;  // the same budget for the MMA warp's waits, in probes
};

// Pipeline event log, compiled in only with -DQW_ATTN_TRACE (a debugging build).
#ifdef QW_ATTN_TRACE
// Event log for pipeline analysis: (role, event, tile) and the SM clock, written
// by one thread per role of block (0, 0, 0) when a trace buffer is attached.
constexpr int kTraceSlots = 4096;
__device__ __forceinline__ void trace_event(const KernelParams &p, int role, int event, int tile,
                                            uint32_t &cursor) {
    // One private region per role and a register cursor: a plain store, no
    // round trip, so the log barely perturbs what it measures.  (The MMA warp runs its
    // loop with all lanes: one writes.)
    if (p.trace && (threadIdx.x & 31) == 0 && blockIdx.x == 0 && blockIdx.y == 0 && blockIdx.z == 0 && cursor < 1000) {
        p.trace[1 + role * 1024 + cursor] =
            ((unsigned long long)(role << 20 | event << 12 | (tile & 0xfff)) << 40) |
            ((unsigned long long)clock64() & 0xffffffffffull);
        ++cursor;
    }
}
#define QW_TRACE(role, event, tile) trace_event(p, role, event, tile, trace_cursor)
#else
#define QW_TRACE(role, event, tile) ((void)0)
#endif

}  // namespace

#include "qw_attn_tile.cuh"

namespace {

using namespace attn;

__device__ __forceinline__ int row_limit(const KernelParams &p, uint32_t b, uint32_t r) {
    if (r >= p.q_rows) return 0;
    if (p.text_pad && r >= p.text_len[b] && r < p.text_pad) return 0;  // padding query row
    int limit;
    if (p.kv_limit) {
        limit = p.kv_limit[p.per_batch_limits ? (size_t)b * p.q_rows + r : r];
        limit = max(limit, 0);
    } else if (p.causal) {
        unsigned long long c = (unsigned long long)r + 1ull + p.causal_offset;
        limit = (int)min(c, (unsigned long long)p.kv_rows);
    } else {
        limit = (int)p.kv_rows;
    }
    return min(limit, (int)p.kv_rows);
}

// ---------------------------------------------------------------------------
// TMA producer role (one thread).
// ---------------------------------------------------------------------------
__device__ void tma_role(const KernelParams &p, SharedControl *ctl, uint8_t *smem_kv,
                         const CUtensorMap *map_k, const CUtensorMap *map_v, uint32_t b,
                         uint32_t kvh, bool split) {
    const uint32_t where = 3u << 16;
    // K and V of the first visited tile are already on their way (ring slots 0, 1):
    // the kernel body issued them before the row limits were known.
    uint32_t t = 2;
    bool ok = true;
    const int col = (int)(kvh * kHeadDim);
    // One (K, V) pair of visited tile u into the next two ring slots.
    auto load_pair = [&](int u) {
        if (p.withhold_from >= 0 && u >= p.withhold_from) {
            ok = false;  // the tile stays away: nothing is issued, nothing is in flight
            return;
        }
        const int j = phys_tile(ctl, u);
        for (int which = 0; which < 2 && ok; ++which) {
            uint32_t slot = t % kStages, par = ((t / kStages) & 1u) ^ 1u;
            ok = mbar_wait(ctl, smem_u32(&ctl->bars[kBarKvEmpty + slot]), par, p.status,
                           where | (kBarKvEmpty + slot), (uint32_t)j);
            if (!ok) break;
            ++t;
            uint8_t *dst = smem_kv + (size_t)slot * kTileBytes;
            Mbar *bar = &ctl->bars[kBarKvFull + slot];
            mbar_expect_tx(bar, kTileBytes);
            const CUtensorMap *map = which ? map_v : map_k;
            tma_load_3d(dst, map, bar, col, j * kTileN, (int)b);
            tma_load_3d(dst + kHalfTileBytes, map, bar, col + 64, j * kTileN, (int)b);
        }
    };
    if (!split) {
        const int n_max = max(ctl->tile_count[0], ctl->tile_count[1]);
        for (int u = 1; u < n_max && ok; ++u) load_pair(u);
    } else {
        // pairs in the order a0 (under way), b0, a1, b1, ...
        const int la = ctl->tile_count[0], lb = ctl->tile_count[1];
        for (int s = 0; s < la && ok; ++s) {
            if (s > 0) load_pair(s);
            if (s < lb && ok) load_pair(la + s);
        }
    }
    // Leave no copy in flight: every issued load must have landed before the
    // CTA may release its shared memory (bounded like every other wait).
    uint32_t first = t > (uint32_t)kStages ? t - kStages : 0;
    for (uint32_t u = first; u < t; ++u) {
        uint32_t slot = u % kStages, par = (u / kStages) & 1u;
        long long start = clock64();
        while (!mbar_try(&ctl->bars[kBarKvFull + slot], par))
            if (clock64() - start > ctl->wait_cycles) break;
    }
}

__device__ __forceinline__ void issue_q_loads(const KernelParams &p, SharedControl *ctl,
                                              uint8_t *smem_q, const CUtensorMap *map_q, uint32_t b,
                                              uint32_t h, uint32_t row0, int tiles) {
    for (int i = 0; i < tiles; ++i) {
        uint32_t r = row0 + (uint32_t)i * kTileM;
        if (r >= p.q_rows) continue;  // inactive sub-tile: n_tiles is 0, nobody waits
        Mbar *bar = &ctl->bars[kBarQFull + i];
        mbar_expect_tx(bar, kTileBytes);
        uint8_t *dst = smem_q + (size_t)i * kTileBytes;
        tma_load_3d(dst, map_q, bar, (int)(h * kHeadDim), (int)r, (int)b);
        tma_load_3d(dst + kHalfTileBytes, map_q, bar, (int)(h * kHeadDim) + 64, (int)r, (int)b);
    }
}

template <bool kMayBound>
__global__ void __launch_bounds__(kThreads, 1)
qw_attn_sm100_kernel(const __grid_constant__ CUtensorMap map_q,
                     const __grid_constant__ CUtensorMap map_k,
                     const __grid_constant__ CUtensorMap map_v, const KernelParams p) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    uint8_t *smem_q = smem;
    uint8_t *smem_kv = smem + 2 * kTileBytes;
    SharedControl *ctl = reinterpret_cast<SharedControl *>(smem + kSmemData);

    const int tid = threadIdx.x;
    const int warp = warp_index();
    const int lane = tid & 31;
    // CTA -> unit.  Units are numbered batch-major, then head, then query block
    // with the heaviest blocks first (rows late in the joint sequence see the most
    // keys).  The last tail_units units run in split form, two CTAs each.
    const uint32_t whole_units = p.total_units - p.tail_units;
    const bool split = blockIdx.x >= whole_units;
    const uint32_t unit = split ? whole_units + ((blockIdx.x - whole_units) >> 1) : blockIdx.x;
    const uint32_t half = split ? (blockIdx.x - whole_units) & 1u : 0u;
    const uint32_t bh = unit / p.n_qblocks;
    const uint32_t b = bh / p.heads;
    const uint32_t h = bh - b * p.heads;
    const uint32_t kvh = (uint32_t)((unsigned long long)h * p.kv_heads / p.heads);
    const uint32_t qblock = p.n_qblocks - 1 - (unit - bh * p.n_qblocks);
    const uint32_t row0 = qblock * (2 * kTileM) + half * kTileM;

    // The producer thread sets the barriers up itself and starts Q and the first
    // K/V tile at once, under the row-limit loads of the softmax threads.
    if (warp == kTmaWarp && lane == 0) {
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
        ctl->abort_flag = 0;
        ctl->wait_cycles = p.wait_cycles > 0 ? p.wait_cycles : kWaitCycles;
        int lo = 0, hi = 0;
        if (p.text_pad && p.text_len[b] < p.text_pad) {
            lo = ((int)p.text_len[b] + kTileN - 1) / kTileN;
            hi = (int)p.text_pad / kTileN;
            if (hi < lo) hi = lo;
        }
        ctl->skip_lo = lo;
        ctl->skip_hi = hi;
        mbar_init_fence();
    }
    if (warp == kMmaWarp) {
        tmem_alloc<1>(&ctl->tmem_base, kTmemCols);
    }
    // What stands above may run under the tail of the kernel before this one; all that
    // reads or writes global memory stands below.
    grid_launch_dependents();
    grid_wait();
    if (warp == kTmaWarp && lane == 0) {
        const int lo = ctl->skip_lo, hi = ctl->skip_hi;
        issue_q_loads(p, ctl, smem_q, &map_q, b, h, row0, split ? 1 : 2);
        // First visited key tile, assuming the unit has one (if it has none the
        // tile is simply never consumed; the producer drains it before exit).
        const int j0 = lo == 0 ? hi : 0;
        for (int which = 0; which < 2; ++which) {
            uint8_t *dst = smem_kv + (size_t)which * kTileBytes;
            Mbar *bar = &ctl->bars[kBarKvFull + which];
            mbar_expect_tx(bar, kTileBytes);
            const CUtensorMap *map = which ? &map_v : &map_k;
            const int col = (int)(kvh * kHeadDim);
            tma_load_3d(dst, map, bar, col, j0 * kTileN, (int)b);
            tma_load_3d(dst + kHalfTileBytes, map, bar, col + 64, j0 * kTileN, (int)b);
        }
    }
    if (blockIdx.x == 0 && warp == 10 && lane == 0 && p.slot_use) {
        // Sharded heads: whatever read this output slot's previous contents was
        // enqueued before this kernel, so the peers may store the new epoch now.
        const uint32_t epoch = *p.slot_use + 1u;
        *p.slot_use = epoch;
        __threadfence_system();
        for (uint32_t d = 0; d < p.n_freed; ++d)
            asm volatile("st.release.sys.global.u32 [%0], %1;" ::"l"(p.freed_peer[d]), "r"(epoch)
                         : "memory");
    }

    // Row limits: each softmax thread owns one row; the largest limit of a
    // sub-tile bounds its key-tile loop.
    int my_limit = 0;
    int sub = 0, tid_in_group = 0;
    // Fixed reference exponent (log2 units, an integer so that P is the exact
    // power-of-two multiple of what any other reference would give), or < 0 for
    // the running-maximum softmax: no promise given, or one too loose to keep
    // exp2(score*c - bound) >= 2^-2*bound inside the normal fp32 range.
    float bound = -1.0f;
    if (kMayBound && p.score_bound) {  // every role needs to know which softmax runs
        const float limit = ceilf(p.score_bound[0] * p.score_bound[1] * p.scale_log2);
        if (limit >= 0.0f && limit <= 60.0f) bound = limit;
    }
    if (tid < kSoftmaxThreads) {
        sub = tid >> 7;
        tid_in_group = tid & 127;
        // (split form: both warpgroups work on the same 128 rows)
        const uint32_t my_row = row0 + (split ? 0u : (uint32_t)sub * kTileM) + (uint32_t)tid_in_group;
        my_limit = row_limit(p, b, my_row);
        int warp_max = my_limit;
        // A row past the end is computed like its neighbours and never stored: with a
        // limit of 0 it would send its whole warp through the masked path on every tile
        // (600 -> 1500 clocks a tile for the row maximum alone).
        if (my_row >= p.q_rows) my_limit = 0x7fffffff;
#pragma unroll
        for (int off = 16; off > 0; off >>= 1)
            warp_max = max(warp_max, __shfl_xor_sync(0xffffffffu, warp_max, off));
        if (lane == 0) ctl->warp_max[warp] = warp_max;
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (tid < 2) {
        int m = 0;
        for (int w = 0; w < 4; ++w) m = max(m, ctl->warp_max[tid * 4 + w]);
        const int tiles = (m + kTileN - 1) / kTileN;
        ctl->n_tiles[tid] = tiles;
        const int visited = visited_tiles(tiles, ctl->skip_lo, ctl->skip_hi);
        if (!split) {
            ctl->tile_first[tid] = 0;
            ctl->tile_count[tid] = visited;
        } else {
            // both warpgroups saw the same rows: the first half (rounded up) and the rest
            const int first_half = (visited + 1) / 2;
            ctl->tile_first[tid] = tid ? first_half : 0;
            ctl->tile_count[tid] = tid ? visited - first_half : first_half;
        }
    }
    __syncthreads();

    if (tid < kSoftmaxThreads) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
        uint8_t *stage = smem_q + (size_t)sub * kTileBytes;
        const uint32_t tile_row0 = split ? row0 : row0 + (uint32_t)sub * kTileM;
        const int pad_lo = p.text_pad ? (int)p.text_len[b] : 0, pad_hi = (int)p.text_pad;
        // (Captured by name: with [&] the kernel spills 36 bytes instead of 12.)
        const auto store = [&p, stage, tid_in_group, tile_row0, b, h](
                               uint32_t tmem_own, uint32_t tmem_other, float w_own, float w_other,
                               float inv, float, float) __attribute__((always_inline)) {
            const int warp_in_group = tid_in_group >> 5;
            const uint32_t warp_row0 = tile_row0 + (uint32_t)warp_in_group * 32u;
            if (warp_row0 >= p.q_rows) return;
            const uint32_t row_stride = (p.head_major_out ? 1u : p.out_heads_total) * kHeadDim;
            const size_t first = p.head_major_out
                                     ? (((size_t)b * p.heads + h) * p.q_rows + warp_row0) * kHeadDim
                                     : ((size_t)b * p.q_rows + warp_row0) * row_stride +
                                           (size_t)(p.out_head_offset + h) * kHeadDim;
#pragma unroll 1
            for (uint32_t d = 0; d < p.n_out; ++d)
                write_rows(tmem_own, tmem_other, w_own, w_other, inv,
                           smem_u32(stage + warp_in_group * (32 * 128)), p.out_peers[d] + first,
                           row_stride, min(32u, p.q_rows - warp_row0));
        };
        const auto has_rows = [&p, tile_row0]() __attribute__((always_inline)) { return tile_row0 < p.q_rows; };
        if (kMayBound && bound >= 0.0f)
            softmax_role<kMayBound, false>(p, ctl, sub, tid_in_group, my_limit, pad_lo, pad_hi, split,
                                           bound, has_rows, store);
        else
            softmax_role<false, false>(p, ctl, sub, tid_in_group, my_limit, pad_lo, pad_hi, split, 0.0f,
                                       has_rows, store);
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
    }
    if (tid < kSoftmaxThreads) {
    } else if (warp == kMmaWarp) {
        if (split) mma_role_split(p, ctl, smem_q, smem_kv);
        else mma_role(p, ctl, smem_q, smem_kv);
    } else if (warp == kTmaWarp && lane == 0) {
        tma_role(p, ctl, smem_kv, &map_k, &map_v, b, kvh, split);
        // Q loads of active sub-tiles must have landed as well.
        for (int i = 0; i < (split ? 1 : 2); ++i) {
            if (row0 + (uint32_t)i * kTileM >= p.q_rows) continue;
            long long start = clock64();
            while (!mbar_try(&ctl->bars[kBarQFull + i], 0))
                if (clock64() - start > ctl->wait_cycles) break;
        }
    }

    tc_fence_before();
    __syncthreads();
    if (warp == kMmaWarp) {
        tc_fence_after();
        tmem_dealloc<1>(ctl->tmem_base, kTmemCols);
    }
}

// [batch][rows][heads*128] bf16, boxes of 128 rows x 64 columns.
int make_map_3d(CUtensorMap *map, const void *base, uint32_t batch, uint32_t rows, uint32_t heads) {
    const cuuint64_t dims[3] = {(cuuint64_t)heads * kHeadDim, rows, batch};
    const cuuint64_t strides[2] = {(cuuint64_t)heads * kHeadDim * 2,
                                   (cuuint64_t)rows * heads * kHeadDim * 2};
    return make_map(map, base, 3, dims, strides, kTileN);
}

#ifdef QW_ATTN_TRACE
// QW_CUDA_ATTN_TRACE=<file>: attach an event log to every launch and dump it after
// each one (synchronous; a debugging aid, never set in production runs).
unsigned long long *trace_buffer() {
    static unsigned long long *buffer = nullptr;
    static bool looked = false;
    if (!looked) {
        looked = true;
        const char *path = getenv("QW_CUDA_ATTN_TRACE");
        if (path && *path) {
            if (cudaMalloc(&buffer, kTraceSlots * 8) != cudaSuccess) buffer = nullptr;
            else cudaMemset(buffer, 0, kTraceSlots * 8);
        }
    }
    return buffer;
}

void trace_dump(cudaStream_t stream) {
    unsigned long long *buffer = trace_buffer();
    if (!buffer) return;
    static unsigned long long host[kTraceSlots];
    cudaStreamSynchronize(stream);
    cudaMemcpy(host, buffer, sizeof(host), cudaMemcpyDeviceToHost);
    cudaMemset(buffer, 0, kTraceSlots * 8);
    FILE *f = fopen(getenv("QW_CUDA_ATTN_TRACE"), "a");
    if (!f) return;
    fprintf(f, "launch\n");
    for (int i = 1; i < kTraceSlots; ++i) {
        unsigned long long w = host[i];
        if (!w) continue;
        unsigned tag = (unsigned)(w >> 40);
        fprintf(f, "%u %u %u %llu\n", tag >> 20, (tag >> 12) & 0xff, tag & 0xfff,
                w & 0xffffffffffull);
    }
    fclose(f);
}
#endif

typedef void (*AttnKernel)(const CUtensorMap, const CUtensorMap, const CUtensorMap,
                           const KernelParams);

int sm_count_of_current_device() {
    static int sms[64];
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64) return 148;
    if (!sms[dev]) {
        cudaDeviceGetAttribute(&sms[dev], cudaDevAttrMultiProcessorCount, dev);
        if (sms[dev] <= 0) sms[dev] = 148;
    }
    return sms[dev];
}

// QW_CUDA_ATTN_TAIL=whole: never split the last wave's units (comparison runs).
bool whole_units_forced() {
    static int forced = -1;
    if (forced < 0) {
        const char *env = getenv("QW_CUDA_ATTN_TAIL");
        forced = env && !strcmp(env, "whole") ? 1 : 0;
    }
    return forced != 0;
}

// The kernel with or without the fixed-exponent softmax, for callers that pass a score
// bound or not.  The opt-in to ~197 KB of dynamic shared memory is a per-device
// attribute: it is set on first use on every device a process drives.
AttnKernel pick_kernel(bool may_bound) {
    static bool ready[64][2];
    AttnKernel chosen = may_bound ? qw_attn_sm100_kernel<true> : qw_attn_sm100_kernel<false>;
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return nullptr;
    const bool tracked = dev >= 0 && dev < 64;
    if (!tracked || !ready[dev][may_bound ? 1 : 0]) {
        if (cudaFuncSetAttribute(chosen, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 (int)kSmemBytes) != cudaSuccess)
            return nullptr;
        if (tracked) ready[dev][may_bound ? 1 : 0] = true;
    }
    return chosen;
}

}  // namespace

// Units of the last, partly filled wave that run in split form: all of them when
// the doubled CTAs still fit the SMs (a sixteenth over is tolerated: block-causal
// layouts always have a few near-empty units that retire at once), none otherwise
// -- two half-length waves would take as long as the one they replace.
extern "C" uint32_t qwcu_attn_sm100_tail_units(uint32_t units, uint32_t sm_count) {
    if (!sm_count) return 0;
    const uint32_t rest = units % sm_count;
    return rest && 2 * rest <= sm_count + sm_count / 16 ? rest : 0u;
}

extern "C" int qwcu_attn_sm100_launch(const qwcu_attn_args *a, qwcu_stream stream_) {
    cudaStream_t stream = static_cast<cudaStream_t>(stream_);
    if (a->batch == 0 || a->batch > 8 || !a->q_rows || !a->kv_rows || !a->heads || !a->kv_heads)
        return (int)cudaErrorInvalidValue;
    // TMA needs 16-byte aligned bases; cudaMalloc gives 256.
    if (((uintptr_t)a->q | (uintptr_t)a->k | (uintptr_t)a->v | (uintptr_t)a->out) & 15u)
        return (int)cudaErrorMisalignedAddress;
    AttnKernel kernel = pick_kernel(a->score_bound != nullptr);
    if (!kernel) return (int)cudaGetLastError();
    CUtensorMap map_q, map_k, map_v;
    int rc;
    if ((rc = make_map_3d(&map_q, a->q, a->batch, a->q_rows, a->heads))) return rc;
    if ((rc = make_map_3d(&map_k, a->k, a->batch, a->kv_rows, a->kv_heads))) return rc;
    if ((rc = make_map_3d(&map_v, a->v, a->batch, a->kv_rows, a->kv_heads))) return rc;
    KernelParams p;
    p.kv_limit = a->kv_limit;
    p.status = a->status;
#ifdef QW_ATTN_TRACE
    p.trace = trace_buffer();
#endif
    p.per_batch_limits = a->per_batch_limits;
    p.causal = a->causal;
    p.causal_offset = a->causal_offset;
    p.batch = a->batch;
    p.q_rows = a->q_rows;
    p.kv_rows = a->kv_rows;
    p.heads = a->heads;
    p.kv_heads = a->kv_heads;
    for (int i = 0; i < 8; ++i) p.text_len[i] = a->text_len[i];
    p.text_pad = a->text_pad;
    p.scale_log2 = a->scale * 1.4426950408889634f;
    p.score_bound = a->score_bound;
    p.head_major_out = a->head_major_out;
    if (a->n_out_peers > 0) {
        if (a->n_out_peers > 8 || a->head_major_out) return (int)cudaErrorInvalidValue;
        p.n_out = a->n_out_peers;
        for (uint32_t d = 0; d < p.n_out; ++d) {
            if ((uintptr_t)a->out_peers[d] & 15u) return (int)cudaErrorMisalignedAddress;
            p.out_peers[d] = static_cast<__nv_bfloat16 *>(a->out_peers[d]);
        }
        p.out_heads_total = a->out_heads_total;
        p.out_head_offset = a->out_head_offset;
    } else {
        p.n_out = 1;
        p.out_peers[0] = static_cast<__nv_bfloat16 *>(a->out);
        p.out_heads_total = a->heads;
        p.out_head_offset = 0;
    }
    p.wait_cycles = a->wait_cycles;
    // (At least 32 probes, like the other waits.  kProbeCycles is more than a probe takes: this
    // role, which waits for the cause itself, gives up before those that wait behind it.)
    const long long budget = p.wait_cycles > 0 ? p.wait_cycles : kWaitCycles;
    p.mma_probes = 32 + (int)min(budget / kProbeCycles, 1ll << 30);
    p.withhold_from = a->withhold_from > 0 ? a->withhold_from : -1;
    p.slot_use = a->slot_use;
    p.n_freed = a->slot_use ? a->n_freed : 0;
    if (p.n_freed > 8) return (int)cudaErrorInvalidValue;
    for (uint32_t d = 0; d < 8; ++d) p.freed_peer[d] = d < p.n_freed ? a->freed_peer[d] : nullptr;
    // One CTA per unit; the units of the last, partly filled wave run split in two
    // (half the rows each, the key tiles divided between the sub-tiles) when the
    // doubled CTAs still fit the idle SMs, give or take a few light units.
    const unsigned long long units =
        (unsigned long long)((a->q_rows + 2 * kTileM - 1) / (2 * kTileM)) * a->heads * a->batch;
    if (units > 0x3fffffffull) return (int)cudaErrorInvalidValue;
    p.n_qblocks = (a->q_rows + 2 * kTileM - 1) / (2 * kTileM);
    p.total_units = (uint32_t)units;
    p.tail_units = (a->whole_units || whole_units_forced())
                       ? 0u
                       : qwcu_attn_sm100_tail_units(p.total_units,
                                                    (uint32_t)sm_count_of_current_device());
    const unsigned grid = p.total_units + p.tail_units;
    rc = launch(kernel, grid, kThreads, kSmemBytes, 1, stream, map_q, map_k, map_v, p);
#ifdef QW_ATTN_TRACE
    if (p.trace && !rc) trace_dump(stream);
#endif
    return rc;
}
