// Entry points of the attention over the quantised cache (kernels: attention_rows.cuh, attention_tiles.cuh).
#include "attention_launch.cuh"

#include <new>

extern "C" {

tf_status tf_attention_workspace_create(tf_context* ctx, uint32_t head_dim, tf_attention_workspace** out) {
    const char* name = "tf_attention_workspace_create";
    TF_REQUIRE(ctx, ctx != nullptr && out != nullptr, TF_ERR_INVALID_ARGUMENT, "%s: NULL argument", name);
    *out = nullptr;
    TF_REQUIRE(ctx, head_dim == 64 || head_dim == 128 || head_dim == 256 || head_dim == 512, TF_ERR_UNSUPPORTED,
               "%s: head_dim %u is not 64, 128, 256 or 512", name, head_dim);
    const tf::DeviceScope scope(ctx->device);
    tf_attention_workspace* ws = new (std::nothrow) tf_attention_workspace();
    TF_REQUIRE(ctx, ws != nullptr, TF_ERR_OUT_OF_MEMORY, "%s: out of host memory", name);
    ws->device = ctx->device;
    ws->head_dim = head_dim;
    ws->row_capacity = (uint32_t)ctx->sm_count * 128;          // per SM: a block with a unit of 128 rows, or 16 workers with units of eight
    ws->max_workers = (uint32_t)ctx->sm_count * 16;
    const uint64_t partial = (uint64_t)2 * ws->row_capacity * (head_dim + 4) * sizeof(float), info = (uint64_t)ws->max_workers * sizeof(tf::ShareInfo);
    cudaError_t e = cudaMalloc(&ws->partial, partial);
    if (e == cudaSuccess) e = cudaMalloc(&ws->info, info);
    const uint64_t tickets = (uint64_t)3 * 4 * ws->max_workers * sizeof(uint32_t);      // kJoin^3 shares are more than there are workers
    if (e == cudaSuccess) e = cudaMalloc(&ws->tickets, tickets);
    if (e == cudaSuccess) e = cudaMemset(ws->tickets, 0, tickets);
    if (e == cudaSuccess) e = cudaStreamSynchronize(cudaStreamLegacy);                  // calls may come on streams that do not wait for this one
    if (e != cudaSuccess) {
        cudaGetLastError();
        tf_attention_workspace_destroy(ws);
        return tf::fail(ctx, TF_ERR_OUT_OF_MEMORY, "%s: %s", name, cudaGetErrorString(e));
    }
    ws->bytes = partial + info + tickets;
    *out = ws;
    return TF_OK;
}

void tf_attention_workspace_destroy(tf_attention_workspace* ws) {
    if (!ws) return;
    const tf::DeviceScope scope(ws->device);
    if (ws->partial) cudaFree(ws->partial);
    if (ws->info) cudaFree(ws->info);
    if (ws->tickets) cudaFree(ws->tickets);
    delete ws;
}

uint64_t tf_attention_workspace_bytes(const tf_attention_workspace* ws) { return ws ? ws->bytes : 0; }

tf_status tf_tree_attention(tf_context* ctx, void* stream, const void* q, uint32_t q_stride, void* out, uint32_t out_stride,
                            const tf_kv_cache* cache, const tf_kv_batch* batch, const uint64_t* tree_mask, uint32_t mask_words, uint32_t window,
                            float scale, uint32_t q_heads, tf_dtype act_dtype, tf_attention_workspace* ws) {
    const char* name = "tf_tree_attention";
    TF_REQUIRE(ctx, ctx != nullptr, TF_ERR_INVALID_ARGUMENT, "%s: ctx is NULL", name);
    TF_REQUIRE(ctx, (q && out) || (batch && batch->rows == 0), TF_ERR_INVALID_ARGUMENT, "%s: NULL buffer", name);
    tf_status s = tf::check_kv_cache(ctx, name, cache);
    if (s == TF_OK) s = tf::check_kv_batch(ctx, name, batch);
    if (s != TF_OK) return s;
    TF_REQUIRE(ctx, ws != nullptr, TF_ERR_INVALID_ARGUMENT, "%s: workspace is NULL", name);
    TF_REQUIRE(ctx, ws->device == ctx->device, TF_ERR_INVALID_ARGUMENT, "%s: the workspace belongs to device %d, the context to %d", name, ws->device, ctx->device);
    TF_REQUIRE(ctx, ws->head_dim == cache->head_dim, TF_ERR_DIMENSION_MISMATCH, "%s: the workspace is for heads of %u, the cache has %u", name, ws->head_dim,
               cache->head_dim);
    TF_REQUIRE(ctx, act_dtype == TF_FP16 || act_dtype == TF_BF16, TF_ERR_UNSUPPORTED, "%s: rows are fp16 or bf16", name);
    TF_REQUIRE(ctx, q_heads > 0 && q_heads <= 65535 && q_heads % cache->kv_heads == 0, TF_ERR_INVALID_ARGUMENT,
               "%s: %u query heads do not share %u kv heads", name, q_heads, cache->kv_heads);
    const uint64_t row = (uint64_t)q_heads * cache->head_dim;
    TF_REQUIRE(ctx, q_stride >= row && out_stride >= row, TF_ERR_INVALID_ARGUMENT, "%s: a row stride is smaller than its row", name);
    TF_REQUIRE(ctx, tf::aligned(q, 16) && tf::aligned(out, 16) && (q_stride | out_stride) % 8 == 0, TF_ERR_ALIGNMENT,
               "%s: rows must be 16-byte aligned and strides multiples of 8 elements", name);
    TF_REQUIRE(ctx, q != out || q_stride == out_stride || batch->rows <= 1, TF_ERR_INVALID_ARGUMENT, "%s: out may be q only with the same stride", name);
    TF_REQUIRE(ctx, tree_mask == nullptr || mask_words > 0, TF_ERR_INVALID_ARGUMENT, "%s: mask_words is 0", name);
    TF_REQUIRE(ctx, tf::aligned(tree_mask, 8), TF_ERR_ALIGNMENT, "%s: tree_mask must be 8-byte aligned", name);
    TF_REQUIRE(ctx, tree_mask == nullptr || window == 0 || batch->positions != nullptr || batch->rows == 0, TF_ERR_INVALID_ARGUMENT,
               "%s: a tree with a window needs positions", name);
    TF_REQUIRE(ctx, window <= 0x7FFFFFFFu, TF_ERR_INVALID_ARGUMENT, "%s: window must be below 2^31", name);
    TF_REQUIRE(ctx, scale - scale == 0.0f, TF_ERR_INVALID_ARGUMENT, "%s: scale must be finite", name);
    if (batch->rows == 0 || batch->sequences == 0) return TF_OK;
    const uint32_t group = q_heads / cache->kv_heads;
    TF_REQUIRE(ctx, (uint64_t)batch->rows * group <= 0x7FFFFFFFu, TF_ERR_UNSUPPORTED, "%s: rows times query heads per kv head must be below 2^31", name);
    tf::AttnArgs a = {};
    a.q = static_cast<const uint16_t*>(q); a.out = static_cast<uint16_t*>(out);
    a.k = {static_cast<uint8_t*>(cache->k_codes), static_cast<uint16_t*>(cache->k_scales), static_cast<uint16_t*>(cache->k_biases)};
    a.v = {static_cast<uint8_t*>(cache->v_codes), static_cast<uint16_t*>(cache->v_scales), static_cast<uint16_t*>(cache->v_biases)};
    a.table = {batch->page_table, batch->page_table_stride, cache->num_pages, tf::log2_of(cache->page_size)};
    a.row_offsets = batch->row_offsets; a.context_lengths = batch->context_lengths; a.positions = batch->positions;
    a.mask = reinterpret_cast<const unsigned long long*>(tree_mask); a.mask_words = mask_words;
    a.partial = ws->partial; a.info = static_cast<tf::ShareInfo*>(ws->info); a.tickets = ws->tickets; a.ticket_stride = 4 * ws->max_workers;
    a.error = ctx->device_error;
    a.q_stride = q_stride; a.out_stride = out_stride;
    a.sequences = batch->sequences; a.rows = batch->rows; a.kv_heads = cache->kv_heads; a.group = group;
    a.window = window; a.scale = scale; a.head_parts = 1;
    const tf::DeviceScope scope(ctx->device);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const bool bf16 = act_dtype == TF_BF16;
    if (cache->bits == 8) {
        switch (cache->head_dim) {
            case 64: return tf::attend<64, 8>(ctx, st, a, ws, bf16);
            case 128: return tf::attend<128, 8>(ctx, st, a, ws, bf16);
            case 256: return tf::attend<256, 8>(ctx, st, a, ws, bf16);
            default: return tf::attend<512, 8>(ctx, st, a, ws, bf16);
        }
    }
    switch (cache->head_dim) {
        case 64: return tf::attend<64, 4>(ctx, st, a, ws, bf16);
        case 128: return tf::attend<128, 4>(ctx, st, a, ws, bf16);
        case 256: return tf::attend<256, 4>(ctx, st, a, ws, bf16);
        default: return tf::attend<512, 4>(ctx, st, a, ws, bf16);
    }
}

}  // extern "C"
