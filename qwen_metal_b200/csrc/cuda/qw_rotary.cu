// Rotary positions for grouped heads, alone or into a paged K/V cache (HBM-bound).
//
// Pair (a, b) number i of a head's rotated part, at position p:
//   a' = m (a cos(p f_i) - b sin(p f_i)),  b' = m (a sin(p f_i) + b cos(p f_i)),
// the pairs being neighbours (2i, 2i + 1) or halves (i, i + rotary_dim / 2); what lies behind the
// rotated part is copied.  The angle is taken in turns: p * (f_i / 2 pi) minus its nearest whole
// number, in 64 bits (positions of a million leave 2^-4 of a turn in 32), and only the remainder
// goes to sincospi in 32.
//
// A CTA takes one or a few tokens.  Their cosines and sines are worked out once, a thread per
// pair, into shared memory (each costs as much as rotating a dozen pairs); then a thread takes
// kVec pairs of a token in registers and walks the heads of q, of k and, into a cache, of v.
#include <cuda_runtime.h>
#include <stdint.h>

#include "qw_paged.cuh"
#include "qw_sm100.cuh"

namespace {

using sm100::pack_bf16;

constexpr int kThreads = 256;
constexpr uint32_t kMaxTokens = 4;  // of a CTA
// Heads that a thread has in flight: 16384 rows of 40 heads 62.0 us, with four 63.5, with eight 67.0.
constexpr int kTrip = 2;

struct Params {
    const uint16_t *q_in, *k_in, *v_in;
    uint16_t *q_out, *k_out, *v_out;
    const uint32_t *positions;  // or NULL: the cache row
    const float *frequencies;
    uint32_t tokens, heads, kv_heads;
    uint32_t head_dim, pairs;  // pairs = rotary_dim / 2
    uint32_t cta_tokens;       // tokens of a CTA
    uint32_t slots, lanes;     // threads of a token: slots = head_dim / (2 kVec) times lanes
    float magnitude;
    int into_cache;
    paged::Cache cache;
};

template <int kVec>
struct Vec {
    uint32_t w[(kVec + 1) / 2];
};

template <int kVec>
__device__ __forceinline__ Vec<kVec> load(const uint16_t *p) {
    Vec<kVec> v;
    if constexpr (kVec == 8) {
        const uint4 x = __ldcs(reinterpret_cast<const uint4 *>(p));
        v.w[0] = x.x, v.w[1] = x.y, v.w[2] = x.z, v.w[3] = x.w;
    } else if constexpr (kVec == 4) {
        const uint2 x = __ldcs(reinterpret_cast<const uint2 *>(p));
        v.w[0] = x.x, v.w[1] = x.y;
    } else if constexpr (kVec == 2) {
        v.w[0] = __ldcs(reinterpret_cast<const uint32_t *>(p));
    } else {
        v.w[0] = __ldcs(p);
    }
    return v;
}

template <int kVec>
__device__ __forceinline__ void store(uint16_t *p, const Vec<kVec> &v) {
    if constexpr (kVec == 8)
        *reinterpret_cast<uint4 *>(p) = make_uint4(v.w[0], v.w[1], v.w[2], v.w[3]);
    else if constexpr (kVec == 4)
        *reinterpret_cast<uint2 *>(p) = make_uint2(v.w[0], v.w[1]);
    else if constexpr (kVec == 2)
        *reinterpret_cast<uint32_t *>(p) = v.w[0];
    else
        *p = (uint16_t)v.w[0];
}

// Two neighbouring vectors of eight, 32 bytes in one access: the same rows, neighbouring pairs, 64.8 -> 63.4 us.
__device__ __forceinline__ void load_pair(const uint16_t *p, Vec<8> &a, Vec<8> &b) {
    asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(a.w[0]), "=r"(a.w[1]), "=r"(a.w[2]), "=r"(a.w[3]), "=r"(b.w[0]), "=r"(b.w[1]),
                   "=r"(b.w[2]), "=r"(b.w[3])
                 : "l"(p));
}
__device__ __forceinline__ void store_pair(uint16_t *p, const Vec<8> &a, const Vec<8> &b) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(a.w[0]),
                 "r"(a.w[1]), "r"(a.w[2]), "r"(a.w[3]), "r"(b.w[0]), "r"(b.w[1]), "r"(b.w[2]), "r"(b.w[3])
                 : "memory");
}

template <int kVec>
__device__ __forceinline__ float get(const Vec<kVec> &v, int i) {
    return __uint_as_float((i & 1) ? v.w[i / 2] & 0xffff0000u : v.w[i / 2] << 16);
}

// Two vectors of kVec elements: the first and second elements of kVec pairs (halves) or kVec pairs
// as they lie (neighbours).
template <int kVec, bool kHalf>
__device__ __forceinline__ void rotate(Vec<kVec> &a, Vec<kVec> &b, const float (&c)[kVec],
                                       const float (&s)[kVec]) {
    float x[2 * kVec];
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
        const int at = kHalf ? i : 2 * i, to = kHalf ? i + kVec : 2 * i + 1;
        const float u = at < kVec ? get(a, at) : get(b, at - kVec);
        const float v = to < kVec ? get(a, to) : get(b, to - kVec);
        x[at] = fmaf(u, c[i], -(v * s[i]));
        x[to] = fmaf(u, s[i], v * c[i]);
    }
    if constexpr (kVec == 1) {
        a.w[0] = pack_bf16(x[0], 0.0f);
        b.w[0] = pack_bf16(x[1], 0.0f);
    } else {
#pragma unroll
        for (int i = 0; i < kVec / 2; ++i) {
            a.w[i] = pack_bf16(x[2 * i], x[2 * i + 1]);
            b.w[i] = pack_bf16(x[kVec + 2 * i], x[kVec + 2 * i + 1]);
        }
    }
}

template <int kVec, bool kHalf>
__global__ void __launch_bounds__(kThreads) qw_rotary_kernel(const Params p) {
    extern __shared__ float table[];  // [cta_tokens][pairs] cosines, then sines
    __shared__ long long row_of[kMaxTokens];  // cache row in the pool, or -1; position
    __shared__ uint32_t sequence_of[kMaxTokens], position_of[kMaxTokens];
    sm100::grid_launch_dependents();
    sm100::grid_wait();
    const uint32_t token0 = blockIdx.x * p.cta_tokens;
    const uint32_t count = min(p.cta_tokens, p.tokens - token0);
    if (p.into_cache) {
        // Whose tokens they are: every thread looks at some sequences.  Tokens of one that does not fit its
        // tensors have no row that can be told, and are left out like padding.
        if (threadIdx.x < kMaxTokens) sequence_of[threadIdx.x] = 0xffffffffu;
        __syncthreads();
        for (uint32_t b = threadIdx.x; b < p.cache.batch; b += kThreads) {
            const paged::Sequence s = paged::sequence(p.cache, b);
            for (uint32_t i = 0; i < count; ++i)
                if (s.fits && token0 + i - s.start < (uint32_t)s.fresh) sequence_of[i] = b;
        }
        __syncthreads();
        if (threadIdx.x < count) {
            const uint32_t b = sequence_of[threadIdx.x], token = token0 + threadIdx.x;
            long long at = -1;
            uint32_t position = 0;
            if (b != 0xffffffffu) {
                const paged::Sequence s = paged::sequence(p.cache, b);
                const int row = s.length - s.fresh + (int)(token - s.start);
                if (row >= 0) {
                    at = paged::pool_row_or_none(p.cache, b, (uint32_t)row);
                    position = p.positions ? p.positions[token] : (uint32_t)row;
                }
            }
            row_of[threadIdx.x] = at;
            position_of[threadIdx.x] = position;
        }
        __syncthreads();
    }
    for (uint32_t j = threadIdx.x; j < count * p.pairs; j += kThreads) {
        const uint32_t i = j / p.pairs, pair = j - i * p.pairs;
        const uint32_t position = p.into_cache ? position_of[i] : __ldg(p.positions + token0 + i);
        const double turns =
            (double)position * ((double)__ldg(p.frequencies + pair) * 0.15915494309189535);
        float sine, cosine;
        sincospif(2.0f * (float)(turns - rint(turns)), &sine, &cosine);
        table[j] = cosine * p.magnitude;
        table[p.cta_tokens * p.pairs + j] = sine * p.magnitude;
    }
    __syncthreads();

    const uint32_t each = p.slots * p.lanes;
    const uint32_t i = threadIdx.x / each, rest = threadIdx.x - i * each;
    if (i >= count) return;
    const uint32_t lane = rest / p.slots, slot = rest - lane * p.slots;
    const long long row = p.into_cache ? row_of[i] : 0;
    if (row < 0) return;  // padding behind the last sequence, in front of the cache, or without a page
    const bool turn = slot * kVec < p.pairs;
    float c[kVec], s[kVec];
    // Where the two vectors lie in a head.
    uint32_t first = 2 * slot * kVec, second = first + kVec;
    if (turn) {
        if (kHalf) first = slot * kVec, second = first + p.pairs;
#pragma unroll
        for (int v = 0; v < kVec; ++v) {
            c[v] = table[i * p.pairs + slot * kVec + v];
            s[v] = table[(p.cta_tokens + i) * p.pairs + slot * kVec + v];
        }
    }
    const size_t token = token0 + i;
    const uint32_t all = p.heads + p.kv_heads * (p.into_cache ? 2u : 1u);
    // kTrip heads at a time, all their loads ahead of the first store: the compiler cannot know
    // that a store is not to a head that has still to be loaded.
    for (uint32_t h0 = lane; h0 < all; h0 += kTrip * p.lanes) {
        Vec<kVec> a[kTrip], b[kTrip];
        uint16_t *out[kTrip];
        bool turn_it[kTrip];
#pragma unroll
        for (int u = 0; u < kTrip; ++u) {
            const uint32_t h = h0 + u * p.lanes;
            if (h >= all) break;
            const uint16_t *in;
            turn_it[u] = turn;
            if (h < p.heads) {
                const size_t at = (token * p.heads + h) * p.head_dim;
                in = p.q_in + at, out[u] = p.q_out + at;
            } else {
                uint32_t g = h - p.heads;
                const bool value = g >= p.kv_heads;
                if (value) g -= p.kv_heads, turn_it[u] = false;
                in = (value ? p.v_in : p.k_in) + (token * p.kv_heads + g) * p.head_dim;
                out[u] = (value ? p.v_out : p.k_out) +
                         ((p.into_cache ? (size_t)row : token) * p.kv_heads + g) * p.head_dim;
            }
            if constexpr (kVec == 8 && !kHalf) load_pair(in + first, a[u], b[u]);
            else a[u] = load<kVec>(in + first), b[u] = load<kVec>(in + second);
        }
#pragma unroll
        for (int u = 0; u < kTrip; ++u) {
            if (h0 + u * p.lanes >= all) break;
            if (turn_it[u]) rotate<kVec, kHalf>(a[u], b[u], c, s);
            if constexpr (kVec == 8 && !kHalf) {
                store_pair(out[u] + first, a[u], b[u]);
            } else {
                store<kVec>(out[u] + first, a[u]);
                store<kVec>(out[u] + second, b[u]);
            }
        }
    }
}

template <int kVec>
int launch_vec(const Params &p, bool half, cudaStream_t stream) {
    const unsigned grid = (p.tokens + p.cta_tokens - 1) / p.cta_tokens;
    const size_t smem = (size_t)p.cta_tokens * p.pairs * 2 * sizeof(float);
    return sm100::launch(half ? qw_rotary_kernel<kVec, true> : qw_rotary_kernel<kVec, false>, grid,
                         kThreads, smem, 1, stream, p);
}

}  // namespace

extern "C" int qwcu_rotary_launch(const qwcu_rotary_args *a, int sm_count, qwcu_stream stream_) {
    cudaStream_t stream = static_cast<cudaStream_t>(stream_);
    const uint32_t dim = a->head_dim, rotary = a->rotary_dim;
    if (!a->tokens || !a->heads || !dim || dim % 2 || dim > 512 || !rotary || rotary % 2 || rotary > dim)
        return (int)cudaErrorInvalidValue;
    Params p;
    p.q_in = static_cast<const uint16_t *>(a->q_in);
    p.k_in = static_cast<const uint16_t *>(a->k_in);
    p.v_in = static_cast<const uint16_t *>(a->v_in);
    p.q_out = static_cast<uint16_t *>(a->q_out);
    p.k_out = static_cast<uint16_t *>(a->k_out);
    p.v_out = static_cast<uint16_t *>(a->v_out);
    p.positions = a->positions;
    p.frequencies = a->frequencies;
    p.tokens = a->tokens;
    p.heads = a->heads;
    p.kv_heads = a->k_in ? a->kv_heads : 0;
    p.head_dim = dim;
    p.pairs = rotary / 2;
    p.magnitude = a->magnitude;
    p.into_cache = a->v_in != nullptr;
    p.cache = {a->cache.page_table, a->cache.token_start, a->cache.cache_len, a->cache.batch, a->tokens,
               a->cache.table_width, a->cache.page_shift, a->cache.pool_pages, a->cache.status};
    // The widest vectors that neither straddle the rotated part's end nor, in halves, its middle.
    int vec = 8;
    while (vec > 1 && ((rotary / 2) % vec || (dim - rotary) % (2 * vec))) vec /= 2;
    p.slots = dim / (2 * vec);
    const unsigned sms = (unsigned)(sm_count > 0 ? sm_count : 148);
    p.cta_tokens = kMaxTokens;
    while (p.cta_tokens > 1 && (p.cta_tokens * p.slots > (uint32_t)kThreads ||
                                a->tokens < sms * 4u * p.cta_tokens))
        p.cta_tokens /= 2;
    p.lanes = kThreads / (p.cta_tokens * p.slots);
    switch (vec) {
        case 8: return launch_vec<8>(p, a->half != 0, stream);
        case 4: return launch_vec<4>(p, a->half != 0, stream);
        case 2: return launch_vec<2>(p, a->half != 0, stream);
        default: return launch_vec<1>(p, a->half != 0, stream);
    }
}
