// Head norms with rotation and the quantised cache write of a layer's QKV rows, and the cache read.
#include "kv_cache.cuh"

namespace tf {

tf_status check_kv_cache(tf_context* ctx, const char* name, const tf_kv_cache* c) {
    TF_REQUIRE(ctx, c != nullptr, TF_ERR_INVALID_ARGUMENT, "%s: cache is NULL", name);
    TF_REQUIRE(ctx, c->k_codes && c->k_scales && c->k_biases && c->v_codes && c->v_scales && c->v_biases, TF_ERR_INVALID_ARGUMENT,
               "%s: NULL cache plane", name);
    TF_REQUIRE(ctx, c->bits == 4 || c->bits == 8, TF_ERR_UNSUPPORTED, "%s: cache codes have 4 or 8 bits, not %u", name, c->bits);
    TF_REQUIRE(ctx, c->head_dim == 64 || c->head_dim == 128 || c->head_dim == 256 || c->head_dim == 512, TF_ERR_UNSUPPORTED,
               "%s: head_dim %u is not 64, 128, 256 or 512", name, c->head_dim);
    TF_REQUIRE(ctx, c->page_size >= 16 && c->page_size <= 65536 && (c->page_size & (c->page_size - 1)) == 0, TF_ERR_UNSUPPORTED,
               "%s: page_size %u is not a power of two from 16 to 65536", name, c->page_size);
    TF_REQUIRE(ctx, c->num_pages > 0 && c->num_pages <= 0x7FFFFFFFu && c->kv_heads > 0 && c->kv_heads <= 65535, TF_ERR_INVALID_ARGUMENT,
               "%s: num_pages and kv_heads must be positive (num_pages below 2^31, kv_heads below 65536)", name);
    TF_REQUIRE(ctx, (uint64_t)c->num_pages * c->kv_heads * c->page_size < 0xFFFFFFFFull, TF_ERR_UNSUPPORTED,
               "%s: pages times heads times page size must be below 2^32", name);
    TF_REQUIRE(ctx, aligned(c->k_codes, 16) && aligned(c->k_scales, 16) && aligned(c->k_biases, 16) && aligned(c->v_codes, 16) &&
                        aligned(c->v_scales, 16) && aligned(c->v_biases, 16), TF_ERR_ALIGNMENT, "%s: cache planes must be 16-byte aligned", name);
    return TF_OK;
}

tf_status check_kv_batch(tf_context* ctx, const char* name, const tf_kv_batch* b) {
    TF_REQUIRE(ctx, b != nullptr, TF_ERR_INVALID_ARGUMENT, "%s: batch is NULL", name);
    if (b->rows == 0 || b->sequences == 0) return TF_OK;
    TF_REQUIRE(ctx, b->row_offsets && b->context_lengths && b->page_table, TF_ERR_INVALID_ARGUMENT, "%s: NULL array in the batch", name);
    TF_REQUIRE(ctx, b->page_table_stride > 0, TF_ERR_INVALID_ARGUMENT, "%s: page_table_stride is 0", name);
    TF_REQUIRE(ctx, b->rows <= 0x7FFFFFFFu && b->sequences < 0x7FFFFFFFu, TF_ERR_INVALID_ARGUMENT, "%s: rows and sequences must be below 2^31", name);
    TF_REQUIRE(ctx, aligned(b->row_offsets, 4) && aligned(b->context_lengths, 4) && aligned(b->page_table, 4) && aligned(b->positions, 4),
               TF_ERR_ALIGNMENT, "%s: batch arrays must be 4-byte aligned", name);
    return TF_OK;
}

// ---------------------------------------------------------------------------
// head norms, rotation, cache write
// ---------------------------------------------------------------------------

constexpr int kEpilogueThreads = 256;
constexpr int kEpilogueWarps = kEpilogueThreads / kWarp;
constexpr uint16_t kBf16NaN = 0x7FC0;

struct EpilogueArgs {
    const uint16_t *q, *k, *v, *q_weight, *k_weight;
    const float* frequencies;
    uint16_t *q_out, *k_out, *v_out;
    const int32_t *row_offsets, *context_lengths, *positions;
    KvTable table;
    KvPlanes k_cache, v_cache;
    uint32_t* error;
    uint32_t q_stride, k_stride, v_stride, q_out_stride, k_out_stride, v_out_stride;
    uint32_t rows, sequences, q_heads, kv_heads, pairs;
    float eps;
    int norm_v, bits, has_cache;
};

template <bool BF16>
__device__ __forceinline__ float2 pair_to_float(uint32_t v) {
    if constexpr (BF16) return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&v));
    else return __half22float2(*reinterpret_cast<const __half2*>(&v));
}
template <bool BF16>
__device__ __forceinline__ uint32_t float_to_pair(float a, float b) {
    if constexpr (BF16) {
        const __nv_bfloat162 r = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&r);
    } else {
        const __half2 r = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&r);
    }
}

template <int WORDS>
__device__ __forceinline__ void store_words(void* p, const uint32_t (&w)[WORDS]) {
    if constexpr (WORDS == 1) *static_cast<uint32_t*>(p) = w[0];
    else if constexpr (WORDS == 2) *static_cast<uint2*>(p) = make_uint2(w[0], w[1]);
    else {
#pragma unroll
        for (int i = 0; i < WORDS / 4; ++i) static_cast<uint4*>(p)[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
    }
}

// One head's values, VEC per lane, as codes and planes of their groups of 64 at row `row` of the planes (a row is one token of one head).
template <int D>
__device__ __forceinline__ void quantise_head(const float (&f)[D / 32], const KvPlanes& planes, size_t row, int bits, int lane) {
    constexpr int VEC = D / 32, LANES = 64 / VEC;            // lanes of a group
    float low = f[0], high = f[0];
    bool bad = false;
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
        low = fminf(low, f[e]);
        high = fmaxf(high, f[e]);
        bad |= !(fabsf(f[e]) <= 3.402823466e38f);
    }
#pragma unroll
    for (int off = LANES / 2; off >= 1; off >>= 1) {
        low = fminf(low, __shfl_xor_sync(kFullMask, low, off));
        high = fmaxf(high, __shfl_xor_sync(kFullMask, high, off));
    }
    const int group = lane / LANES;
    const unsigned lanes = (LANES == 32 ? kFullMask : ((1u << (LANES % 32)) - 1u)) << (group * LANES % 32);
    bad = (__ballot_sync(kFullMask, bad) & lanes) != 0;
    const float top = bits == 8 ? 255.0f : 15.0f;
    uint16_t s16 = __bfloat16_as_ushort(__float2bfloat16_rn(high == low ? 1.0f : __fdiv_rn(high - low, top)));
    uint16_t o16 = __bfloat16_as_ushort(__float2bfloat16_rn(low));
    if (bad || (s16 & 0x7F80) == 0x7F80 || (o16 & 0x7F80) == 0x7F80) s16 = o16 = kBf16NaN;
    const float scale = bf16_bits_to_float(s16), bias = bf16_bits_to_float(o16);
    const float inv = scale == 0.0f ? 0.0f : __fdiv_rn(1.0f, scale);
    uint32_t code[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) code[e] = (uint32_t)fminf(fmaxf(floorf(__fadd_rn(__fmul_rn(f[e] - bias, inv), 0.5f)), 0.0f), top);   // a NaN becomes 0
    if (bits == 8) {
        uint8_t* at = planes.codes + row * D + lane * VEC;
        if constexpr (VEC == 2) {
            *reinterpret_cast<uint16_t*>(at) = (uint16_t)(code[0] | code[1] << 8);
        } else {
            uint32_t w[VEC / 4];
#pragma unroll
            for (int i = 0; i < VEC / 4; ++i) w[i] = code[4 * i] | code[4 * i + 1] << 8 | code[4 * i + 2] << 16 | code[4 * i + 3] << 24;
            store_words(at, w);
        }
    } else {
        uint8_t* at = planes.codes + row * (D / 2) + lane * (VEC / 2);
        if constexpr (VEC == 2) *at = (uint8_t)(code[0] | code[1] << 4);
        else if constexpr (VEC == 4) *reinterpret_cast<uint16_t*>(at) = (uint16_t)(code[0] | code[1] << 4 | code[2] << 8 | code[3] << 12);
        else {
            uint32_t w[VEC / 8];
#pragma unroll
            for (int i = 0; i < VEC / 8; ++i) {
                w[i] = 0;
#pragma unroll
                for (int e = 0; e < 8; ++e) w[i] |= code[8 * i + e] << (4 * e);
            }
            store_words(at, w);
        }
    }
    if (lane % LANES == 0) {
        planes.scales[row * (D / 64) + group] = s16;
        planes.biases[row * (D / 64) + group] = o16;
    }
}

// A block takes one row and up to 8 * HPW of its heads (q heads, then k, then v), a warp HPW of them, VEC = D / 32 consecutive elements per
// lane. The row's angles are computed once per block and kept in shared memory; a pair's partner is a whole number of lanes away.
template <int D, bool BF16, int HPW>
__global__ void __launch_bounds__(kEpilogueThreads)
qkv_epilogue_kernel(const EpilogueArgs a) {
    constexpr int VEC = D / 32;
    __shared__ float2 turn[D / 2];                            // (cos, sin) of the row's angles
    __shared__ int32_t s_page;
    __shared__ uint32_t s_slot;
    __shared__ int s_state;                                   // 0: a row of no sequence, 1: its page is missing, 2: fine
    const int warp = threadIdx.x / kWarp, lane = threadIdx.x % kWarp;
    const uint32_t row = blockIdx.x, heads = a.q_heads + 2 * a.kv_heads;
    const uint32_t first = blockIdx.y * (kEpilogueWarps * HPW) + warp;

    uint32_t x[HPW][VEC / 2];
#pragma unroll
    for (int n = 0; n < HPW; ++n) {
        const uint32_t h = first + n * kEpilogueWarps;
        if (h >= heads) break;
        const uint16_t* src = h < a.q_heads ? a.q + (size_t)row * a.q_stride + (size_t)h * D
                              : h < a.q_heads + a.kv_heads ? a.k + (size_t)row * a.k_stride + (size_t)(h - a.q_heads) * D
                                                           : a.v + (size_t)row * a.v_stride + (size_t)(h - a.q_heads - a.kv_heads) * D;
        load_words(x[n], src + lane * VEC);
    }
    if (threadIdx.x == 0) s_state = a.has_cache ? 0 : 2;
    __syncthreads();
    if (a.has_cache) {
        for (uint32_t b = threadIdx.x; b < a.sequences; b += kEpilogueThreads) {
            const int64_t begin = a.row_offsets[b], end = a.row_offsets[b + 1];
            if (begin <= (int64_t)row && (int64_t)row < end) {
                const int64_t token = (int64_t)a.context_lengths[b] + ((int64_t)row - begin);
                const int32_t page = a.context_lengths[b] < 0 ? -1 : a.table.page(b, token);
                s_page = page;
                s_slot = (uint32_t)token & ((1u << a.table.page_log2) - 1u);
                s_state = page < 0 ? 1 : 2;
                if (page < 0) *a.error = kErrKvPage;
            }
            if (row == 0 && (begin < 0 || begin > end || end > (int64_t)a.rows)) *a.error = kErrKvOffsets;
        }
    }
    for (uint32_t j = threadIdx.x; j < a.pairs; j += kEpilogueThreads) {
        // in turns: the whole ones are dropped in 64 bits, what is left is at most half a turn
        const double turns = (double)a.positions[row] * (double)a.frequencies[j] * 0.15915494309189533577;
        float s, c;
        sincospif(2.0f * (float)(turns - rint(turns)), &s, &c);
        turn[j] = make_float2(c, s);
    }
    __syncthreads();
    if (s_state == 0) return;

#pragma unroll
    for (int n = 0; n < HPW; ++n) {
        const uint32_t h = first + n * kEpilogueWarps;
        if (h >= heads) break;
        const bool is_q = h < a.q_heads, is_v = h >= a.q_heads + a.kv_heads;
        float f[VEC];
#pragma unroll
        for (int i = 0; i < VEC / 2; ++i) {
            const float2 t = pair_to_float<BF16>(x[n][i]);
            f[2 * i] = t.x;
            f[2 * i + 1] = t.y;
        }
        if (!is_v || a.norm_v) {
            float sum = 0.0f;
#pragma unroll
            for (int e = 0; e < VEC; ++e) sum = fmaf(f[e], f[e], sum);
            const float inv = rsqrtf(warp_sum(sum) / (float)D + a.eps);
            const uint16_t* weight = is_q ? a.q_weight : is_v ? nullptr : a.k_weight;
            uint32_t w[VEC / 2];
            if (weight) load_words(w, weight + lane * VEC);
#pragma unroll
            for (int i = 0; i < VEC / 2; ++i) {
                f[2 * i] *= inv;
                f[2 * i + 1] *= inv;
                if (weight) {
                    f[2 * i] *= bf16_bits_to_float((uint16_t)w[i]);
                    f[2 * i + 1] *= bf16_bits_to_float((uint16_t)(w[i] >> 16));
                }
            }
        }
        if (!is_v && a.pairs) {
            const int apart = (int)a.pairs / VEC;              // lanes between the elements of a pair
            const bool lower = lane < apart, turned = lane < 2 * apart;
            const int from = lower ? lane + apart : turned ? lane - apart : lane;
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const float other = __shfl_sync(kFullMask, f[e], from);
                if (turned) {
                    const float2 t = turn[(lower ? lane : from) * VEC + e];
                    f[e] = lower ? fmaf(-other, t.y, f[e] * t.x) : fmaf(other, t.y, f[e] * t.x);
                }
            }
        }
        uint32_t y[VEC / 2];
#pragma unroll
        for (int i = 0; i < VEC / 2; ++i) y[i] = float_to_pair<BF16>(f[2 * i], f[2 * i + 1]);
        if (is_q) {
            store_words(a.q_out + (size_t)row * a.q_out_stride + (size_t)h * D + lane * VEC, y);
            continue;
        }
        const uint32_t kv = is_v ? h - a.q_heads - a.kv_heads : h - a.q_heads;
        uint16_t* out = is_v ? a.v_out : a.k_out;
        if (out) store_words(out + (size_t)row * (is_v ? a.v_out_stride : a.k_out_stride) + (size_t)kv * D + lane * VEC, y);
        if (a.has_cache && s_state == 2)
            quantise_head<D>(f, is_v ? a.v_cache : a.k_cache, (((size_t)s_page * a.kv_heads + kv) << a.table.page_log2) + s_slot, a.bits, lane);
    }
}

template <int D, bool BF16>
static void launch_epilogue(cudaStream_t st, const EpilogueArgs& a, uint32_t rows) {
    const uint32_t heads = a.q_heads + 2 * a.kv_heads;
    // One head per warp while that leaves few blocks: a lone row's heads go through side by side. With four the angles are computed
    // for four times as many heads.
    if ((uint64_t)rows * ((heads + 7) / 8) <= 1184) qkv_epilogue_kernel<D, BF16, 1><<<dim3(rows, (heads + 7) / 8), kEpilogueThreads, 0, st>>>(a);
    else qkv_epilogue_kernel<D, BF16, 4><<<dim3(rows, (heads + 31) / 32), kEpilogueThreads, 0, st>>>(a);
}

// ---------------------------------------------------------------------------
// cache read
// ---------------------------------------------------------------------------

constexpr int kReadThreads = 256, kReadRows = 8;

struct ReadArgs {
    KvPlanes planes[2];
    uint16_t* out[2];
    uint32_t out_stride[2];
    const int32_t *row_offsets, *context_lengths;
    KvTable table;
    uint32_t* error;
    uint32_t sequences, rows, kv_heads, head_dim;
};

// A block takes eight rows; its warps find the rows' tokens, then every thread turns eight codes at a time into one 16-byte store.
template <int BITS, bool BF16>
__global__ void __launch_bounds__(kReadThreads)
kv_cache_read_kernel(const ReadArgs a) {
    __shared__ int32_t s_page[kReadRows];
    __shared__ uint32_t s_slot[kReadRows];
    const int warp = threadIdx.x / kWarp, lane = threadIdx.x % kWarp;
    const uint32_t row0 = blockIdx.x * kReadRows;
    if (lane == 0) s_page[warp] = -1;
    __syncwarp();
    const int64_t row = (int64_t)row0 + warp;
    for (uint32_t b = lane; row < a.rows && b < a.sequences; b += kWarp) {
        const int64_t begin = a.row_offsets[b], end = a.row_offsets[b + 1];
        if (begin <= row && row < end) {
            const int64_t token = (int64_t)a.context_lengths[b] + (row - begin);
            const int32_t page = a.context_lengths[b] < 0 ? -1 : a.table.page(b, token);
            s_page[warp] = page;
            s_slot[warp] = (uint32_t)token & ((1u << a.table.page_log2) - 1u);
            if (page < 0) *a.error = kErrKvPage;
        }
        if (row == 0 && (begin < 0 || begin > end || end > (int64_t)a.rows)) *a.error = kErrKvOffsets;
    }
    __syncthreads();
    const uint32_t per_head = a.head_dim / 8, per_row = a.kv_heads * per_head, groups = a.head_dim / 64;
    const int kv = blockIdx.y;                                 // keys or values
    if (!a.out[kv]) return;
    const KvPlanes p = a.planes[kv];
    const uint32_t total = per_row * kReadRows;
    for (uint32_t i = threadIdx.x; i < total; i += kReadThreads) {
        const uint32_t r = i / per_row, c = i - r * per_row, h = c / per_head, e = c - h * per_head;
        const int32_t page = s_page[r];
        if (page < 0) continue;
        const size_t at = (((size_t)page * a.kv_heads + h) << a.table.page_log2) + s_slot[r];
        const float scale = bf16_bits_to_float(p.scales[at * groups + e / 8]), bias = bf16_bits_to_float(p.biases[at * groups + e / 8]);
        uint32_t y[4];
        if constexpr (BITS == 8) {
            uint32_t w[2];
            load_words(w, p.codes + at * a.head_dim + e * 8);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t v = w[j / 2] >> (16 * (j % 2));
                y[j] = float_to_pair<BF16>(fmaf((float)(v & 255u), scale, bias), fmaf((float)(v >> 8 & 255u), scale, bias));
            }
        } else {
            const uint32_t v = *reinterpret_cast<const uint32_t*>(p.codes + at * (a.head_dim / 2) + e * 4);
#pragma unroll
            for (int j = 0; j < 4; ++j)
                y[j] = float_to_pair<BF16>(fmaf((float)(v >> (8 * j) & 15u), scale, bias), fmaf((float)(v >> (8 * j + 4) & 15u), scale, bias));
        }
        store_words(a.out[kv] + (size_t)(row0 + r) * a.out_stride[kv] + (size_t)c * 8, y);
    }
}

static KvTable table_of(const tf_kv_cache* c, const tf_kv_batch* b) {
    return {b->page_table, b->page_table_stride, c->num_pages, log2_of(c->page_size)};
}

}  // namespace tf

extern "C" {

tf_status tf_qkv_epilogue(tf_context* ctx, void* stream, const void* q, uint32_t q_stride, const void* k, uint32_t k_stride, const void* v,
                          uint32_t v_stride, const void* q_weight, const void* k_weight, int norm_v, const float* frequencies,
                          uint32_t rotated_pairs, float eps, void* q_out, uint32_t q_out_stride, void* k_out, uint32_t k_out_stride,
                          void* v_out, uint32_t v_out_stride, const tf_kv_batch* batch, const tf_kv_cache* cache, uint32_t q_heads,
                          uint32_t kv_heads, uint32_t head_dim, tf_dtype act_dtype) {
    const char* name = "tf_qkv_epilogue";
    TF_REQUIRE(ctx, ctx != nullptr, TF_ERR_INVALID_ARGUMENT, "%s: ctx is NULL", name);
    TF_REQUIRE(ctx, q && k && v && q_out, TF_ERR_INVALID_ARGUMENT, "%s: NULL buffer", name);
    TF_REQUIRE(ctx, batch != nullptr, TF_ERR_INVALID_ARGUMENT, "%s: batch is NULL", name);
    TF_REQUIRE(ctx, cache || (k_out && v_out), TF_ERR_INVALID_ARGUMENT, "%s: without a cache k_out and v_out are needed", name);
    TF_REQUIRE(ctx, act_dtype == TF_FP16 || act_dtype == TF_BF16, TF_ERR_UNSUPPORTED, "%s: rows are fp16 or bf16", name);
    TF_REQUIRE(ctx, head_dim == 64 || head_dim == 128 || head_dim == 256 || head_dim == 512, TF_ERR_UNSUPPORTED,
               "%s: head_dim %u is not 64, 128, 256 or 512", name, head_dim);
    TF_REQUIRE(ctx, q_heads > 0 && kv_heads > 0 && q_heads <= 65535 && kv_heads <= 65535, TF_ERR_INVALID_ARGUMENT,
               "%s: head counts must be from 1 to 65535", name);
    if (cache) {
        const tf_status s = tf::check_kv_cache(ctx, name, cache);
        if (s != TF_OK) return s;
        TF_REQUIRE(ctx, cache->kv_heads == kv_heads && cache->head_dim == head_dim, TF_ERR_DIMENSION_MISMATCH,
                   "%s: the cache has %u heads of %u, the rows %u of %u", name, cache->kv_heads, cache->head_dim, kv_heads, head_dim);
        const tf_status t = tf::check_kv_batch(ctx, name, batch);
        if (t != TF_OK) return t;
    }
    const uint64_t q_row = (uint64_t)q_heads * head_dim, kv_row = (uint64_t)kv_heads * head_dim;
    TF_REQUIRE(ctx, q_stride >= q_row && k_stride >= kv_row && v_stride >= kv_row && q_out_stride >= q_row && (!k_out || k_out_stride >= kv_row) &&
                        (!v_out || v_out_stride >= kv_row), TF_ERR_INVALID_ARGUMENT, "%s: a row stride is smaller than its row", name);
    TF_REQUIRE(ctx, tf::aligned(q, 16) && tf::aligned(k, 16) && tf::aligned(v, 16) && tf::aligned(q_out, 16) && tf::aligned(k_out, 16) &&
                        tf::aligned(v_out, 16) && tf::aligned(q_weight, 16) && tf::aligned(k_weight, 16) &&
                        (q_stride | k_stride | v_stride | q_out_stride | (k_out ? k_out_stride : 0) | (v_out ? v_out_stride : 0)) % 8 == 0,
               TF_ERR_ALIGNMENT, "%s: rows and weights must be 16-byte aligned and strides multiples of 8 elements", name);
    TF_REQUIRE(ctx, rotated_pairs <= head_dim / 2 && rotated_pairs % (head_dim / 32) == 0, TF_ERR_UNSUPPORTED,
               "%s: rotated_pairs %u is not a multiple of %u up to %u", name, rotated_pairs, head_dim / 32, head_dim / 2);
    TF_REQUIRE(ctx, rotated_pairs == 0 || (frequencies && batch->positions), TF_ERR_INVALID_ARGUMENT, "%s: a rotation needs frequencies and positions", name);
    TF_REQUIRE(ctx, tf::aligned(frequencies, 4) && tf::aligned(batch->positions, 4), TF_ERR_ALIGNMENT,
               "%s: frequencies and positions must be 4-byte aligned", name);
    TF_REQUIRE(ctx, !(k == v && (k_out == k || v_out == k)), TF_ERR_INVALID_ARGUMENT, "%s: k_out or v_out may not overwrite rows that are both k and v", name);
    TF_REQUIRE(ctx, eps >= 0.0f && eps <= 3.4e38f, TF_ERR_INVALID_ARGUMENT, "%s: eps must be finite and not negative", name);
    if (batch->rows == 0 || (cache && batch->sequences == 0)) return TF_OK;
    TF_REQUIRE(ctx, batch->rows <= 0x7FFFFFFFu, TF_ERR_INVALID_ARGUMENT, "%s: rows must be below 2^31", name);
    tf::EpilogueArgs a = {};
    a.q = static_cast<const uint16_t*>(q); a.k = static_cast<const uint16_t*>(k); a.v = static_cast<const uint16_t*>(v);
    a.q_weight = static_cast<const uint16_t*>(q_weight); a.k_weight = static_cast<const uint16_t*>(k_weight);
    a.frequencies = frequencies;
    a.q_out = static_cast<uint16_t*>(q_out); a.k_out = static_cast<uint16_t*>(k_out); a.v_out = static_cast<uint16_t*>(v_out);
    a.row_offsets = batch->row_offsets; a.context_lengths = batch->context_lengths; a.positions = batch->positions;
    a.error = ctx->device_error;
    a.q_stride = q_stride; a.k_stride = k_stride; a.v_stride = v_stride;
    a.q_out_stride = q_out_stride; a.k_out_stride = k_out_stride; a.v_out_stride = v_out_stride;
    a.rows = batch->rows; a.sequences = batch->sequences; a.q_heads = q_heads; a.kv_heads = kv_heads; a.pairs = rotated_pairs;
    a.eps = eps; a.norm_v = norm_v != 0;
    if (cache) {
        a.has_cache = 1;
        a.bits = (int)cache->bits;
        a.table = tf::table_of(cache, batch);
        a.k_cache = {static_cast<uint8_t*>(cache->k_codes), static_cast<uint16_t*>(cache->k_scales), static_cast<uint16_t*>(cache->k_biases)};
        a.v_cache = {static_cast<uint8_t*>(cache->v_codes), static_cast<uint16_t*>(cache->v_scales), static_cast<uint16_t*>(cache->v_biases)};
    }
    const tf::DeviceScope scope(ctx->device);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const bool bf16 = act_dtype == TF_BF16;
    switch (head_dim) {
        case 64: bf16 ? tf::launch_epilogue<64, true>(st, a, batch->rows) : tf::launch_epilogue<64, false>(st, a, batch->rows); break;
        case 128: bf16 ? tf::launch_epilogue<128, true>(st, a, batch->rows) : tf::launch_epilogue<128, false>(st, a, batch->rows); break;
        case 256: bf16 ? tf::launch_epilogue<256, true>(st, a, batch->rows) : tf::launch_epilogue<256, false>(st, a, batch->rows); break;
        default: bf16 ? tf::launch_epilogue<512, true>(st, a, batch->rows) : tf::launch_epilogue<512, false>(st, a, batch->rows); break;
    }
    return tf::check_launch(ctx, name);
}

tf_status tf_kv_cache_read(tf_context* ctx, void* stream, const tf_kv_cache* cache, const tf_kv_batch* batch, void* k_out,
                           uint32_t k_out_stride, void* v_out, uint32_t v_out_stride, tf_dtype act_dtype) {
    const char* name = "tf_kv_cache_read";
    TF_REQUIRE(ctx, ctx != nullptr, TF_ERR_INVALID_ARGUMENT, "%s: ctx is NULL", name);
    tf_status s = tf::check_kv_cache(ctx, name, cache);
    if (s == TF_OK) s = tf::check_kv_batch(ctx, name, batch);
    if (s != TF_OK) return s;
    TF_REQUIRE(ctx, k_out || v_out, TF_ERR_INVALID_ARGUMENT, "%s: NULL buffer", name);
    TF_REQUIRE(ctx, act_dtype == TF_FP16 || act_dtype == TF_BF16, TF_ERR_UNSUPPORTED, "%s: rows are fp16 or bf16", name);
    const uint64_t row = (uint64_t)cache->kv_heads * cache->head_dim;
    TF_REQUIRE(ctx, (!k_out || k_out_stride >= row) && (!v_out || v_out_stride >= row), TF_ERR_INVALID_ARGUMENT,
               "%s: a row stride is smaller than its row", name);
    TF_REQUIRE(ctx, tf::aligned(k_out, 16) && tf::aligned(v_out, 16) && ((k_out ? k_out_stride : 0) | (v_out ? v_out_stride : 0)) % 8 == 0,
               TF_ERR_ALIGNMENT, "%s: rows must be 16-byte aligned and strides multiples of 8 elements", name);
    if (batch->rows == 0 || batch->sequences == 0) return TF_OK;
    tf::ReadArgs a = {};
    a.planes[0] = {static_cast<uint8_t*>(cache->k_codes), static_cast<uint16_t*>(cache->k_scales), static_cast<uint16_t*>(cache->k_biases)};
    a.planes[1] = {static_cast<uint8_t*>(cache->v_codes), static_cast<uint16_t*>(cache->v_scales), static_cast<uint16_t*>(cache->v_biases)};
    a.out[0] = static_cast<uint16_t*>(k_out); a.out[1] = static_cast<uint16_t*>(v_out);
    a.out_stride[0] = k_out_stride; a.out_stride[1] = v_out_stride;
    a.row_offsets = batch->row_offsets; a.context_lengths = batch->context_lengths;
    a.table = tf::table_of(cache, batch);
    a.error = ctx->device_error;
    a.sequences = batch->sequences; a.rows = batch->rows; a.kv_heads = cache->kv_heads; a.head_dim = cache->head_dim;
    const tf::DeviceScope scope(ctx->device);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const dim3 grid((batch->rows + tf::kReadRows - 1) / tf::kReadRows, 2);
    const bool bf16 = act_dtype == TF_BF16;
    if (cache->bits == 8) {
        if (bf16) tf::kv_cache_read_kernel<8, true><<<grid, tf::kReadThreads, 0, st>>>(a);
        else tf::kv_cache_read_kernel<8, false><<<grid, tf::kReadThreads, 0, st>>>(a);
    } else {
        if (bf16) tf::kv_cache_read_kernel<4, true><<<grid, tf::kReadThreads, 0, st>>>(a);
        else tf::kv_cache_read_kernel<4, false><<<grid, tf::kReadThreads, 0, st>>>(a);
    }
    return tf::check_launch(ctx, name);
}

}  // extern "C"
