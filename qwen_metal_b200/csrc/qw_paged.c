/* The ops of a text tower that is served token by token (no counterpart in the reference, whose
 * tower runs whole prompts): rotary positions for grouped heads, alone or into a paged K/V cache,
 * and attention of new tokens over that cache.  Validation as in qw_ops.c, then one launch. */
#include "qw_internal.h"

#include <math.h>
#include <string.h>

/* Elements of a tensor that must be there; geometry is at most 2^32 * 2^32 * 512, so the product is
 * checked on the way. */
static int elements_of(size_t *count, uint32_t a, uint32_t b, uint32_t c) {
    return !__builtin_mul_overflow((size_t)a, (size_t)b, count) &&
           !__builtin_mul_overflow(*count, (size_t)c, count) && *count <= SIZE_MAX / 4;
}

/* The tensor holds `elements` of the type and lies on this context's device. */
static int require(h3_gpu *gpu, const h3_gpu_tensor *tensor, size_t elements, h3_gpu_dtype dtype,
                   const char *label) {
    if (!qw_require_dtype(gpu, tensor, elements, dtype, label)) return 0;
    if (tensor->owner->device != gpu->device) {
        qw_set_error(gpu, "%s tensor lies on another device", label);
        return 0;
    }
    return 1;
}

static int overlap(h3_gpu *gpu, const char *what) {
    qw_set_error(gpu, "%s: an output is also an input of another place", what);
    return 0;
}

/* The cache's page table, its sequences and its pools. */
static int require_cache(h3_gpu *gpu, qwcu_cache_args *cache, const h3_gpu_tensor *key_pages,
                         const h3_gpu_tensor *value_pages, const h3_gpu_tensor *page_table,
                         const h3_gpu_tensor *token_start, const h3_gpu_tensor *cache_len,
                         uint32_t batch, uint32_t table_width, uint32_t page_rows,
                         uint32_t kv_heads, uint32_t head_dim, const char *what) {
    if (!batch || !table_width || page_rows < 16 || page_rows > 4096 || (page_rows & (page_rows - 1)) ||
        (uint64_t)table_width * page_rows > 0x7fffff00u || batch > 0x7fffffffu) {
        qw_set_error(gpu, "%s: unsupported cache geometry (pages of 16 to 4096 rows, a power of two)",
                     what);
        return 0;
    }
    size_t entries, page;
    if (!elements_of(&entries, batch, table_width, 1) ||
        !elements_of(&page, page_rows, kv_heads, head_dim)) {
        qw_set_error(gpu, "%s: geometry too large", what);
        return 0;
    }
    if (!require(gpu, page_table, entries, H3_GPU_U32, "page table") ||
        !require(gpu, token_start, (size_t)batch + 1, H3_GPU_U32, "token start") ||
        !require(gpu, cache_len, batch, H3_GPU_U32, "cache length") ||
        !require(gpu, key_pages, page, H3_GPU_BF16, "key pages") ||
        !require(gpu, value_pages, page, H3_GPU_BF16, "value pages"))
        return 0;
    if (key_pages == value_pages) return overlap(gpu, what);
    size_t pages = key_pages->elements / page, value = value_pages->elements / page;
    if (value < pages) pages = value;
    cache->page_table = page_table->dev;
    cache->token_start = token_start->dev;
    cache->cache_len = cache_len->dev;
    cache->batch = batch;
    cache->table_width = table_width;
    cache->page_shift = (uint32_t)__builtin_ctz(page_rows);
    cache->pool_pages = pages > UINT32_MAX ? UINT32_MAX : (uint32_t)pages;
    cache->status = gpu->status_dev;
    return 1;
}

/* What the two rotations share. */
static int require_rotation(h3_gpu *gpu, qwcu_rotary_args *args, const h3_gpu_tensor *frequencies,
                            uint32_t tokens, uint32_t heads, uint32_t kv_heads, uint32_t head_dim,
                            uint32_t rotary_dim, uint32_t layout, float magnitude, const char *what) {
    if (!tokens || !heads || !head_dim || head_dim % 2 || head_dim > 512 || !rotary_dim ||
        rotary_dim % 2 || rotary_dim > head_dim) {
        qw_set_error(gpu, "%s: unsupported geometry (even head_dim up to 512, even rotary_dim within it)",
                     what);
        return 0;
    }
    if (layout != QW_ROTARY_NEIGHBOURS && layout != QW_ROTARY_HALVES) {
        qw_set_error(gpu, "%s: unknown layout %u", what, layout);
        return 0;
    }
    if (!isfinite(magnitude)) {
        qw_set_error(gpu, "%s: the magnitude is not finite", what);
        return 0;
    }
    if (!require(gpu, frequencies, rotary_dim / 2, H3_GPU_F32, "rotary frequencies")) return 0;
    if (tokens > 0x7fffffffu || kv_heads > 0x1fffffffu || heads > 0x1fffffffu) {
        qw_set_error(gpu, "%s: geometry too large", what);
        return 0;
    }
    memset(args, 0, sizeof(*args));
    args->frequencies = frequencies->dev;
    args->tokens = tokens;
    args->heads = heads;
    args->kv_heads = kv_heads;
    args->head_dim = head_dim;
    args->rotary_dim = rotary_dim;
    args->half = layout == QW_ROTARY_HALVES;
    args->magnitude = magnitude;
    return 1;
}

static int launch_rotary(h3_gpu *gpu, const qwcu_rotary_args *args, const char *what) {
    if (!qw_bind(gpu)) return 0;
    int rc = qwcu_rotary_launch(args, qwcu_device_sm_count(gpu->device), gpu->stream);
    qw_count_launch(gpu, rc, what);
    return rc == 0;
}

int qw_gpu_rotary_bf16(h3_gpu *gpu, h3_gpu_tensor *query_output, h3_gpu_tensor *key_output,
                       const h3_gpu_tensor *query_input, const h3_gpu_tensor *key_input,
                       const h3_gpu_tensor *positions, const h3_gpu_tensor *frequencies,
                       uint32_t tokens, uint32_t heads, uint32_t kv_heads, uint32_t head_dim,
                       uint32_t rotary_dim, uint32_t layout, float magnitude) {
    static const char what[] = "rotary";
    if (!gpu) return 0;
    size_t q_count, k_count;
    if (!elements_of(&q_count, tokens, heads, head_dim) ||
        !elements_of(&k_count, tokens, kv_heads, head_dim)) {
        qw_set_error(gpu, "%s: geometry too large", what);
        return 0;
    }
    const int with_key = key_input || key_output;
    if (!require(gpu, query_input, q_count, H3_GPU_BF16, "rotary query") ||
        !require(gpu, query_output, q_count, H3_GPU_BF16, "rotary query output") ||
        (with_key && (!require(gpu, key_input, k_count, H3_GPU_BF16, "rotary key") ||
                      !require(gpu, key_output, k_count, H3_GPU_BF16, "rotary key output"))) ||
        !require(gpu, positions, tokens, H3_GPU_U32, "rotary positions"))
        return 0;
    if (!qw_require_command(gpu)) return 0;
    qwcu_rotary_args args;
    if (!require_rotation(gpu, &args, frequencies, tokens, heads, kv_heads, head_dim, rotary_dim, layout,
                          magnitude, what))
        return 0;
    if (with_key && !kv_heads) {
        qw_set_error(gpu, "%s: unsupported geometry (a key without heads)", what);
        return 0;
    }
    if (with_key && (query_output == key_output || query_output == key_input || key_output == query_input))
        return overlap(gpu, what);
    args.q_in = query_input->dev;
    args.q_out = query_output->dev;
    args.k_in = with_key ? key_input->dev : NULL;
    args.k_out = with_key ? key_output->dev : NULL;
    args.positions = positions->dev;
    return launch_rotary(gpu, &args, what);
}

int qw_gpu_rotary_append_bf16(h3_gpu *gpu, h3_gpu_tensor *query_output, h3_gpu_tensor *key_pages,
                              h3_gpu_tensor *value_pages, const h3_gpu_tensor *query_input,
                              const h3_gpu_tensor *key_new, const h3_gpu_tensor *value_new,
                              const h3_gpu_tensor *positions, const h3_gpu_tensor *frequencies,
                              const h3_gpu_tensor *page_table, const h3_gpu_tensor *token_start,
                              const h3_gpu_tensor *cache_len, uint32_t batch, uint32_t tokens,
                              uint32_t table_width, uint32_t page_rows, uint32_t heads,
                              uint32_t kv_heads, uint32_t head_dim, uint32_t rotary_dim,
                              uint32_t layout, float magnitude) {
    static const char what[] = "rotary append";
    if (!gpu) return 0;
    size_t q_count, k_count;
    if (!elements_of(&q_count, tokens, heads, head_dim) ||
        !elements_of(&k_count, tokens, kv_heads, head_dim)) {
        qw_set_error(gpu, "%s: geometry too large", what);
        return 0;
    }
    if (!require(gpu, query_input, q_count, H3_GPU_BF16, "rotary append query") ||
        !require(gpu, query_output, q_count, H3_GPU_BF16, "rotary append query output") ||
        !require(gpu, key_new, k_count, H3_GPU_BF16, "rotary append key") ||
        !require(gpu, value_new, k_count, H3_GPU_BF16, "rotary append value") ||
        (positions && !require(gpu, positions, tokens, H3_GPU_U32, "rotary append positions")))
        return 0;
    if (!qw_require_command(gpu)) return 0;
    qwcu_rotary_args args;
    if (!require_rotation(gpu, &args, frequencies, tokens, heads, kv_heads, head_dim, rotary_dim, layout,
                          magnitude, what))
        return 0;
    if (!kv_heads) {
        qw_set_error(gpu, "%s: unsupported geometry (a key without heads)", what);
        return 0;
    }
    if (!require_cache(gpu, &args.cache, key_pages, value_pages, page_table, token_start, cache_len,
                       batch, table_width, page_rows, kv_heads, head_dim, what))
        return 0;
    if (key_pages == query_input || key_pages == key_new || key_pages == value_new ||
        key_pages == query_output || value_pages == query_input || value_pages == key_new ||
        value_pages == value_new || value_pages == query_output || query_output == key_new ||
        query_output == value_new)
        return overlap(gpu, what);
    args.q_in = query_input->dev;
    args.q_out = query_output->dev;
    args.k_in = key_new->dev;
    args.k_out = key_pages->dev;
    args.v_in = value_new->dev;
    args.v_out = value_pages->dev;
    args.positions = positions ? positions->dev : NULL;
    return launch_rotary(gpu, &args, what);
}

/* The paged attention's workspaces: of one size for every call on a device, made by the first. */
static char *paged_workspace(h3_gpu *gpu, size_t few_bytes, size_t chunk_bytes) {
    if (gpu->paged_work) return gpu->paged_work;
    if (gpu->capturing) {
        qw_set_error(gpu, "paged attention: run it once before capturing it into a graph (it makes its "
                          "workspace)");
        gpu->chain_failed = 1;
        return NULL;
    }
    void *block = NULL;
    if (cudaMallocAsync(&block, few_bytes + chunk_bytes, gpu->stream) != cudaSuccess) {
        cudaGetLastError();
        qw_set_error(gpu, "cannot allocate %zu bytes of workspace", few_bytes + chunk_bytes);
        return NULL;
    }
    if (!qw_cuda_ok(gpu, cudaMemsetAsync(block, 0, few_bytes, gpu->stream), "workspace")) {
        cudaFreeAsync(block, gpu->stream);
        return NULL;
    }
    gpu->paged_work = block;
    return block;
}

/* Query rows (new tokens x query heads of a kv head) up to which a sequence goes to the kernel for
 * few: one of its units.  With 8 instead of 16, 64 sequences of 4 tokens of 4 heads over 1000 keys take
 * 110 us instead of 87 and 8 over 16000 keys 123 instead of 87; a mixed batch of 20 single tokens and 4
 * chunks 121 instead of 126. */
#define QW_PAGED_FEW_ROWS 16u

int qw_gpu_paged_attention_bf16(h3_gpu *gpu, h3_gpu_tensor *output, const h3_gpu_tensor *query,
                                const h3_gpu_tensor *key_pages, const h3_gpu_tensor *value_pages,
                                const h3_gpu_tensor *page_table, const h3_gpu_tensor *token_start,
                                const h3_gpu_tensor *cache_len, uint32_t batch, uint32_t tokens,
                                uint32_t max_new, uint32_t table_width, uint32_t page_rows,
                                uint32_t heads, uint32_t kv_heads, uint32_t head_dim, float scale) {
    static const char what[] = "paged attention";
    if (!gpu) return 0;
    size_t count;
    if (head_dim != 128 || !heads || !kv_heads || heads % kv_heads || !tokens || !max_new) {
        qw_set_error(gpu, "%s: unsupported geometry (head_dim 128, whole groups of heads)", what);
        return 0;
    }
    if (!elements_of(&count, tokens, heads, head_dim) || (uint64_t)tokens * heads > 0x7fffffffu) {
        qw_set_error(gpu, "%s: geometry too large", what);
        return 0;
    }
    if (!(scale > 0.0f) || !isfinite(scale * 1.4426950408889634f)) { /* (the kernels' exponents are powers of two) */
        qw_set_error(gpu, "%s: the scale must be positive and, times log2(e), finite", what);
        return 0;
    }
    if (!require(gpu, query, count, H3_GPU_BF16, "paged attention query") ||
        !require(gpu, output, count, H3_GPU_BF16, "paged attention output") || !qw_require_command(gpu))
        return 0;
    qwcu_paged_args args;
    memset(&args, 0, sizeof(args));
    if (!require_cache(gpu, &args.cache, key_pages, value_pages, page_table, token_start, cache_len,
                       batch, table_width, page_rows, kv_heads, head_dim, what))
        return 0;
    if (output == query || output == key_pages || output == value_pages) return overlap(gpu, what);
    if (!qw_bind(gpu)) return 0;
    args.q = query->dev;
    args.k_pages = key_pages->dev;
    args.v_pages = value_pages->dev;
    args.out = output->dev;
    args.tokens = tokens;
    args.heads = heads;
    args.kv_heads = kv_heads;
    args.max_new = max_new;
    args.scale = scale;
    args.wait_cycles = gpu->attn_wait_cycles;
    args.withhold_from = gpu->attn_withhold_tile;
    const int sms = qwcu_device_sm_count(gpu->device);
    const size_t few_bytes = (qwcu_paged_few_workspace_bytes(sms) + 255) / 256 * 256;
    char *workspace = paged_workspace(gpu, few_bytes, qwcu_paged_chunk_workspace_bytes(sms));
    if (!workspace) return 0;
    /* Each kernel skips the other's sequences; one sequence alone needs no second kernel.  Where both run, the one
     * for few rows follows the one for chunks directly: it relies on that one's wait for what was before. */
    const uint32_t share = heads / kv_heads;
    const int chunks = share <= 128 && (uint64_t)max_new * share > QW_PAGED_FEW_ROWS;
    const uint32_t least_rows = batch == 1 ? 0u : QW_PAGED_FEW_ROWS + 1u;
    int rc = 0;
    if (chunks) {
        rc = qwcu_paged_chunk_launch(&args, least_rows, workspace + few_bytes, sms, gpu->stream);
        qw_count_launch(gpu, rc, what);
    }
    if (!rc && (!chunks || batch > 1)) {
        rc = qwcu_paged_few_launch(&args, chunks ? QW_PAGED_FEW_ROWS : UINT32_MAX, chunks, workspace, sms,
                                   gpu->stream);
        qw_count_launch(gpu, rc, what);
    }
    if (!rc && chunks) {
        int launched;
        rc = qwcu_paged_merge_launch(&args, least_rows, workspace + few_bytes, sms, gpu->stream, &launched);
        if (rc || launched) qw_count_launch(gpu, rc, what);
    }
    return rc == 0;
}
