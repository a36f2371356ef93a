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

// Minimum and maximum that keep a NaN of either side.
__device__ __forceinline__ float min_nan(float a, float b) { float r; asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b)); return r; }
__device__ __forceinline__ float max_nan(float a, float b) { float r; asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b)); return r; }

// One head's values, VEC per lane, as codes and planes of their groups of 64 at row `row` of the planes (a row is one token of one head). The planes
// are rounded to bf16, as the cache holds them, and the codes are those of the rounded planes: a value is off by half a code step where no rounding of
// the bias or scale pushes it past the ends. A group that holds a NaN or an infinity, or whose planes have no bf16 value, gets NaN planes.
template <int D>
__device__ __forceinline__ void quantise_head(const float (&f)[D / 32], const KvPlanes& planes, size_t row, int bits, int lane) {
    constexpr int VEC = D / 32, LANES = 64 / VEC;            // lanes of a group
    float low = f[0], high = f[0];
#pragma unroll
    for (int e = 1; e < VEC; ++e) {
        low = min_nan(low, f[e]);
        high = max_nan(high, f[e]);
    }
#pragma unroll
    for (int off = LANES / 2; off >= 1; off >>= 1) {
        low = min_nan(low, __shfl_xor_sync(kFullMask, low, off));
        high = max_nan(high, __shfl_xor_sync(kFullMask, high, off));
    }
    const float top = bits == 8 ? 255.0f : 15.0f, part = bits == 8 ? 1.0f / 255.0f : 1.0f / 15.0f, range = high - low;
    const float about = range * part, step = fmaf(fmaf(-about, top, range), part, about);      // range / top, rounded once more
    // at least 2^-126, bf16's and fp32's least normal number, whose quotient is finite
    uint16_t s16 = (uint16_t)max(0x0080u, (uint32_t)__bfloat16_as_ushort(__float2bfloat16_rn(high == low ? 1.0f : step)));
    uint16_t o16 = __bfloat16_as_ushort(__float2bfloat16_rn(low));
    const bool finite = low >= -3.402823466e38f && high <= 3.402823466e38f && (s16 & 0x7F80) != 0x7F80 && (o16 & 0x7F80) != 0x7F80;
    if (!finite) s16 = o16 = kBf16NaN;
    const float scale = bf16_bits_to_float(s16), bias = bf16_bits_to_float(o16);
    const float inv = __frcp_rn(scale);
    uint32_t code[VEC];                                       // in the low byte, under the bits of 2^23: added toward zero it leaves the whole part
#pragma unroll
    for (int e = 0; e < VEC; ++e)
        code[e] = __float_as_uint(__fadd_rz(fminf(fmaxf(__fadd_rn(__fmul_rn(f[e] - bias, inv), 0.5f), 0.0f), top), 8388608.0f));      // a NaN becomes 0
    if (bits == 8) {
        uint8_t* at = planes.codes + row * D + lane * VEC;
        if constexpr (VEC == 2) {
            *reinterpret_cast<uint16_t*>(at) = (uint16_t)__byte_perm(code[0], code[1], 0x0040);
        } else {
            uint32_t w[VEC / 4];
#pragma unroll
            for (int i = 0; i < VEC / 4; ++i)
                w[i] = __byte_perm(__byte_perm(code[4 * i], code[4 * i + 1], 0x0040), __byte_perm(code[4 * i + 2], code[4 * i + 3], 0x0040), 0x5410);
            store_words(at, w);
        }
    } else {
#pragma unroll
        for (int e = 0; e < VEC; e += 2) code[e] = (code[e] & 15u) | (code[e + 1] & 15u) << 4;
        uint8_t* at = planes.codes + row * (D / 2) + lane * (VEC / 2);
        if constexpr (VEC == 2) *at = (uint8_t)code[0];
        else if constexpr (VEC == 4) *reinterpret_cast<uint16_t*>(at) = (uint16_t)(code[0] | code[2] << 8);
        else {
            uint32_t w[VEC / 8];
#pragma unroll
            for (int i = 0; i < VEC / 8; ++i) w[i] = code[8 * i] | code[8 * i + 2] << 8 | code[8 * i + 4] << 16 | code[8 * i + 6] << 24;
            store_words(at, w);
        }
    }
    if (lane % LANES == 0) {
        const size_t at = row * (D / 64) + lane / LANES;
        planes.scales[at] = s16;
        planes.biases[at] = o16;
    }
}

// (cos, sin) of a position's turn at one frequency. In turns: the whole ones are dropped in 64 bits, what is left is at most half a turn. (The hardware's
// sine and cosine are off by 2^-21, which moves planes and codes of the cache that stand near a tie: 4 us less at 4096 rows are not worth it.)
__device__ __forceinline__ float2 turn_of(int32_t position, float frequency) {
    const double turns = (double)position * (double)frequency * 0.15915494309189533577;
    float s, c;
    sincospif(2.0f * (float)(turns - rint(turns)), &s, &c);
    return make_float2(c, s);
}

// Where a row's token lies. state: 0: a row of no sequence, 1: its page is missing, 2: fine.
struct RowPlace {
    int state;
    int32_t page;
    uint32_t slot;
};
__device__ __forceinline__ bool place_row(const EpilogueArgs& a, uint32_t b, uint32_t row, RowPlace& place) {
    const int64_t begin = a.row_offsets[b], end = a.row_offsets[b + 1];
    if (row == 0 && (begin < 0 || begin > end || end > (int64_t)a.rows)) *a.error = kErrKvOffsets;
    if (!(begin <= (int64_t)row && (int64_t)row < end)) return false;
    const int64_t token = (int64_t)a.context_lengths[b] + ((int64_t)row - begin);
    place.page = a.context_lengths[b] < 0 ? -1 : a.table.page(b, token);
    place.slot = (uint32_t)token & ((1u << a.table.page_log2) - 1u);
    place.state = place.page < 0 ? 1 : 2;
    if (place.page < 0) *a.error = kErrKvPage;
    return true;
}

// Heads of one kind: those of q, k or v.
struct HeadKind {
    const uint16_t *source, *weight;                           // of head 0 of the row; nullptr: no weight
    uint16_t* out;                                             // head 0 of the row, or nullptr
    KvPlanes cache;
    uint32_t heads;
    bool norm, turned, cached;
};
__device__ __forceinline__ HeadKind kind_of(const EpilogueArgs& a, int kind, uint32_t row) {
    HeadKind r;
    r.source = kind == 0 ? a.q + (size_t)row * a.q_stride : kind == 1 ? a.k + (size_t)row * a.k_stride : a.v + (size_t)row * a.v_stride;
    r.weight = kind == 0 ? a.q_weight : kind == 1 ? a.k_weight : nullptr;
    r.out = kind == 0 ? a.q_out : kind == 1 ? a.k_out : a.v_out;
    if (r.out) r.out += (size_t)row * (kind == 0 ? a.q_out_stride : kind == 1 ? a.k_out_stride : a.v_out_stride);
    r.cache.codes = kind == 2 ? a.v_cache.codes : a.k_cache.codes;
    r.cache.scales = kind == 2 ? a.v_cache.scales : a.k_cache.scales;
    r.cache.biases = kind == 2 ? a.v_cache.biases : a.k_cache.biases;
    r.heads = kind == 0 ? a.q_heads : a.kv_heads;
    r.norm = kind != 2 || a.norm_v;
    r.turned = kind != 2 && a.pairs;
    r.cached = kind != 0 && a.has_cache;
    return r;
}

// What a lane's elements y of the normed head become: y[e] * own[e] + partner's y * other[e]; weight and rotation in one. A pair's partner is a whole
// number of lanes away. turn(j): (cos, sin) of pair j.
template <int VEC>
struct HeadTurn {
    float own[VEC], other[VEC];
    int from;
};
template <int VEC, typename Turn>
__device__ __forceinline__ void make_turn(HeadTurn<VEC>& t, const uint16_t* weight, uint32_t pairs, int lane, Turn turn) {
    const int apart = (int)pairs / VEC;                        // lanes between the elements of a pair
    const bool lower = lane < apart, turned = lane < 2 * apart;
    t.from = lower ? lane + apart : turned ? lane - apart : lane;
    uint32_t w[VEC / 2], u[VEC / 2];
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) w[i] = u[i] = 0x3F803F80u;
    if (weight) {
        load_words(w, weight + lane * VEC);
        load_words(u, weight + t.from * VEC);
    }
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
        const float mine = __uint_as_float(e % 2 ? w[e / 2] & 0xFFFF0000u : w[e / 2] << 16), theirs = __uint_as_float(e % 2 ? u[e / 2] & 0xFFFF0000u : u[e / 2] << 16);
        t.own[e] = mine;
        t.other[e] = 0.0f;
        if (turned) {
            const float2 cs = turn((lower ? lane : t.from) * VEC + e);
            t.own[e] = mine * cs.x;
            t.other[e] = (lower ? -theirs : theirs) * cs.y;
        }
    }
}

// The head's values f times `inv`, weighed, turned and stored, with its row of the cache.
template <int D, bool BF16>
__device__ __forceinline__ void finish_head(float (&f)[D / 32], float inv, const HeadKind& kind, const HeadTurn<D / 32>& t, uint32_t h, size_t cache_row, int bits, int lane) {
    constexpr int VEC = D / 32;
    if (kind.norm) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) f[e] *= inv;
    }
    if (kind.turned) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) f[e] = fmaf(__shfl_sync(kFullMask, f[e], t.from), t.other[e], f[e] * t.own[e]);
    } else if (kind.weight) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) f[e] *= t.own[e];
    }
    if (kind.out) {
        uint32_t y[VEC / 2];
#pragma unroll
        for (int i = 0; i < VEC / 2; ++i) y[i] = float_to_pair<BF16>(f[2 * i], f[2 * i + 1]);
        store_words(kind.out + (size_t)h * D + lane * VEC, y);
    }
    if (kind.cached) quantise_head<D>(f, kind.cache, cache_row, bits, lane);
}

template <int D, bool BF16>
__device__ __forceinline__ float unpack_head(float (&f)[D / 32], const uint32_t (&x)[D / 64]) {      // and this lane's sum of squares
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < D / 64; ++i) {
        const float2 t = pair_to_float<BF16>(x[i]);
        f[2 * i] = t.x;
        f[2 * i + 1] = t.y;
        sum = fmaf(t.x, t.x, sum);
        sum = fmaf(t.y, t.y, sum);
    }
    return sum;
}

// Heads [first, last) of one kind of a row, by one warp, VEC = D / 32 consecutive elements of a head per lane. BATCH heads are requested while BATCH are
// worked on; their sums of squares are added up together: at each of the first steps a lane hands on the half of the heads that it does not keep.
template <int D, bool BF16, int BATCH, typename Place, typename Turn>
__device__ __forceinline__ void epilogue_heads(const EpilogueArgs& a, HeadKind& kind, uint32_t first, uint32_t last, int lane, Place find_place, Turn turn) {
    constexpr int VEC = D / 32;
    uint32_t x[BATCH][VEC / 2];
#pragma unroll
    for (int n = 0; n < BATCH; ++n) load_words(x[n], kind.source + (size_t)min(first + n, last - 1) * D + lane * VEC);
    const RowPlace place = find_place();
    if (place.state == 0) return;
    if (place.state == 1) kind.cached = false;
    HeadTurn<VEC> t;
    make_turn<VEC>(t, kind.weight, kind.turned ? a.pairs : 0, lane, turn);
#pragma unroll 1
    for (uint32_t h0 = first; h0 < last; h0 += BATCH) {
        float f[BATCH][VEC], sum[BATCH];
#pragma unroll
        for (int n = 0; n < BATCH; ++n) sum[n] = unpack_head<D, BF16>(f[n], x[n]);
        if (BATCH > 1) {
#pragma unroll
            for (int n = 0; n < BATCH; ++n) load_words(x[n], kind.source + (size_t)min(h0 + BATCH + n, last - 1) * D + lane * VEC);
        }
        int off = 16;
#pragma unroll
        for (int left = BATCH / 2; left >= 1; left /= 2, off /= 2)
#pragma unroll
            for (int n = 0; n < left; ++n) {
                const bool upper = lane & off;                 // keeps the upper heads
                sum[n] = __fadd_rn(upper ? sum[n + left] : sum[n], __shfl_xor_sync(kFullMask, upper ? sum[n] : sum[n + left], off));
            }
#pragma unroll
        for (int o = 16 / BATCH; o >= 1; o /= 2) sum[0] = __fadd_rn(sum[0], __shfl_xor_sync(kFullMask, sum[0], o));
        const float inv = rsqrtf(fmaf(sum[0], 1.0f / (float)D, a.eps));
#pragma unroll
        for (int n = 0; n < BATCH; ++n) {
            const float mine = BATCH == 1 ? inv : __shfl_sync(kFullMask, inv, n * (kWarp / BATCH));       // a lane's highest bit is its head's highest
            if (h0 + n < last)
                finish_head<D, BF16>(f[n], mine, kind, t, h0 + n, (((size_t)place.page * a.kv_heads + h0 + n) << a.table.page_log2) + place.slot, a.bits, lane);
        }
    }
}

// Few rows: a block takes one row and eight of its heads (q heads, then k, then v), a warp per head. The row's place and angles are found once per block.
// One row of 32 heads of 256 takes 5.5 us, a chain of latencies: offsets, table, angles, norm, stores.
template <int D, bool BF16>
__global__ void __launch_bounds__(kEpilogueThreads)
qkv_epilogue_kernel(const EpilogueArgs a) {
    __shared__ float2 s_turn[D / 2];                          // (cos, sin) of the row's angles
    __shared__ RowPlace s_place;
    const uint32_t row = blockIdx.x;
    uint32_t h = min(blockIdx.y * kEpilogueWarps + threadIdx.x / kWarp, a.q_heads + 2 * a.kv_heads - 1);       // the last head may be done twice
    int which = 0;
    if (h >= a.q_heads) { which = 1; h -= a.q_heads; }
    if (which && h >= a.kv_heads) { which = 2; h -= a.kv_heads; }
    HeadKind kind = kind_of(a, which, row);
    epilogue_heads<D, BF16, 1>(a, kind, h, h + 1, threadIdx.x % kWarp, [&]() {
        if (threadIdx.x == 0) s_place = {a.has_cache ? 0 : 2, 0, 0};
        __syncthreads();
        if (a.has_cache)
            for (uint32_t b = threadIdx.x; b < a.sequences; b += kEpilogueThreads) {
                RowPlace p;
                if (place_row(a, b, row, p)) s_place = p;
            }
        for (uint32_t j = threadIdx.x; j < a.pairs; j += kEpilogueThreads) s_turn[j] = turn_of(a.positions[row], a.frequencies[j]);
        __syncthreads();
        return s_place; }, [&](int j) { return s_turn[j]; });
}

// Many rows: a block takes eight rows and up to eight heads of one kind, a warp per row. So the kind is known to the whole block (its branches and
// addresses cost no lane's instructions), weights and angles of a lane's elements stay in registers, and no warp waits for another. 4096 rows of 32
// heads of 256 into an 8-bit cache: 45 us, 2.6 TB/s; it is bound by issuing some 235 instructions per head. With warps of mixed kinds it was 76 us; heads two
// by two at half the registers are 5 us faster than four by four.
constexpr uint32_t kBlockHeads = 8;
template <int D, bool BF16>
__global__ void __launch_bounds__(kEpilogueThreads, D == 512 ? 2 : 4)
qkv_epilogue_rows_kernel(const EpilogueArgs a) {
    const int lane = threadIdx.x % kWarp;
    const uint32_t q_chunks = (a.q_heads + kBlockHeads - 1) / kBlockHeads, kv_chunks = (a.kv_heads + kBlockHeads - 1) / kBlockHeads;
    const uint32_t group = blockIdx.x / (q_chunks + 2 * kv_chunks), row = group * kEpilogueWarps + threadIdx.x / kWarp;
    uint32_t chunk = blockIdx.x - group * (q_chunks + 2 * kv_chunks);
    if (row >= a.rows) return;
    int which = 0;
    if (chunk >= q_chunks) { which = 1; chunk -= q_chunks; }
    if (which && chunk >= kv_chunks) { which = 2; chunk -= kv_chunks; }
    HeadKind kind = kind_of(a, which, row);
    const uint32_t first = chunk * kBlockHeads;
    const int32_t position = kind.turned ? a.positions[row] : 0;
    epilogue_heads<D, BF16, 2>(a, kind, first, min(first + kBlockHeads, kind.heads), lane, [&]() {
        RowPlace place = {a.has_cache ? 0 : 2, 0, 0};
        if (a.has_cache)
            for (uint32_t b0 = 0; b0 < a.sequences; b0 += kWarp) {
                RowPlace p = {0, 0, 0};
                const bool mine = b0 + lane < a.sequences && place_row(a, b0 + lane, row, p);
                const uint32_t owner = __ballot_sync(kFullMask, mine);
                if (owner) {
                    const int from = __ffs(owner) - 1;
                    place.state = __shfl_sync(kFullMask, p.state, from);
                    place.page = __shfl_sync(kFullMask, p.page, from);
                    place.slot = __shfl_sync(kFullMask, p.slot, from);
                    if (row != 0) break;                       // the first row's warps look at all offsets
                }
            }
        return place; }, [&](int j) { return turn_of(position, a.frequencies[j]); });
}

static uint64_t row_blocks(uint32_t rows, uint32_t q_heads, uint32_t kv_heads) {
    return ((uint64_t)rows + kEpilogueWarps - 1) / kEpilogueWarps * (((uint64_t)q_heads + kBlockHeads - 1) / kBlockHeads + 2 * (((uint64_t)kv_heads + kBlockHeads - 1) / kBlockHeads));
}

template <int D, bool BF16>
static void launch_epilogue(cudaStream_t st, const EpilogueArgs& a, uint32_t rows) {
    const uint32_t heads = a.q_heads + 2 * a.kv_heads;
    // A warp per head while those are few: a lone row's heads go through side by side. Measured in us, a warp per head / a warp per eight heads: heads of 512, 300
    // blocks of the first kind 12.3 / 12.3, 444: 14.3 / 12.3, 111: 8.2 / 12.3; of 256, 592: 10.2 / 12.3, 1200: 14.3 / 14.3, 4000: 28.6 / 18.5; of 128,
    // 1332: 10.2 / 12.3, 3600: 16.4 / 14.3.
    const uint64_t blocks = (uint64_t)rows * ((heads + 7) / 8);
    if (blocks * D <= 196608) qkv_epilogue_kernel<D, BF16><<<dim3(rows, (heads + 7) / 8), kEpilogueThreads, 0, st>>>(a);
    else qkv_epilogue_rows_kernel<D, BF16><<<(uint32_t)row_blocks(rows, a.q_heads, a.kv_heads), kEpilogueThreads, 0, st>>>(a);
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
    uint32_t sequences, rows, kv_heads, head_log2;
};

// A block takes eight rows of keys or values; its warps find the rows' tokens, then every thread turns eight codes at a time into one 16-byte store.
// Four places are requested before the first is stored: 65536 tokens of 8 heads of 256, 8 bits, 146 us, 5.6 TB/s, bound by HBM (one by one: 166).
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
    const int kv = blockIdx.y;                                 // keys or values
    if (!a.out[kv]) return;
    const KvPlanes p = a.planes[kv];
    const uint32_t per_head_log2 = a.head_log2 - 3, per_row = a.kv_heads << per_head_log2, groups_log2 = a.head_log2 - 6;
    // Eight values a time; a thread's next place is a fixed number of rows and values on. Four places are requested before the first is stored.
    uint32_t r = threadIdx.x / per_row, c = threadIdx.x % per_row;
    const uint32_t step_r = kReadThreads / per_row, step_c = kReadThreads % per_row;
    constexpr int BATCH = 4;
    while (r < kReadRows) {
        uint32_t w[BATCH][BITS / 4], rr[BATCH], cc[BATCH];
        uint16_t s16[BATCH], o16[BATCH];
        bool is[BATCH];
#pragma unroll
        for (int n = 0; n < BATCH; ++n) {
            rr[n] = r;
            cc[n] = c;
            is[n] = r < kReadRows && s_page[r] >= 0;
            if (is[n]) {
                const uint32_t h = c >> per_head_log2, e = c & ((1u << per_head_log2) - 1u);
                const size_t at = (((size_t)s_page[r] * a.kv_heads + h) << a.table.page_log2) + s_slot[r];
                load_words(w[n], p.codes + (at << a.head_log2) * BITS / 8 + e * BITS);
                s16[n] = p.scales[(at << groups_log2) + e / 8];
                o16[n] = p.biases[(at << groups_log2) + e / 8];
            }
            r += step_r;
            c += step_c;
            if (c >= per_row) { c -= per_row; ++r; }
        }
#pragma unroll
        for (int n = 0; n < BATCH; ++n) {
            if (!is[n]) continue;
            const float scale = bf16_bits_to_float(s16[n]), bias = bf16_bits_to_float(o16[n]);
            uint32_t y[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                uint32_t c0, c1;
                if constexpr (BITS == 8) { c0 = w[n][j / 2] >> (16 * (j % 2)) & 255u; c1 = w[n][j / 2] >> (16 * (j % 2) + 8) & 255u; }
                else { c0 = w[n][0] >> (8 * j) & 15u; c1 = w[n][0] >> (8 * j + 4) & 15u; }
                y[j] = float_to_pair<BF16>(fmaf((float)c0, scale, bias), fmaf((float)c1, scale, bias));
            }
            store_words(a.out[kv] + (size_t)(row0 + rr[n]) * a.out_stride[kv] + (size_t)cc[n] * 8, y);
        }
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
    const bool empty = batch && batch->rows == 0;
    TF_REQUIRE(ctx, empty || (q && k && v && q_out), TF_ERR_INVALID_ARGUMENT, "%s: NULL buffer", name);
    TF_REQUIRE(ctx, batch != nullptr, TF_ERR_INVALID_ARGUMENT, "%s: batch is NULL", name);
    TF_REQUIRE(ctx, empty || cache || (k_out && v_out), TF_ERR_INVALID_ARGUMENT, "%s: without a cache k_out and v_out are needed", name);
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
    TF_REQUIRE(ctx, empty || rotated_pairs == 0 || (frequencies && batch->positions), TF_ERR_INVALID_ARGUMENT, "%s: a rotation needs frequencies and positions", name);
    TF_REQUIRE(ctx, tf::aligned(frequencies, 4) && tf::aligned(batch->positions, 4), TF_ERR_ALIGNMENT,
               "%s: frequencies and positions must be 4-byte aligned", name);
    TF_REQUIRE(ctx, batch->rows <= 1 || ((q_out != q || q_out_stride == q_stride) && (k_out != k || k_out_stride == k_stride) && (v_out != v || v_out_stride == v_stride)),
               TF_ERR_INVALID_ARGUMENT, "%s: an output may be its input only with the same stride", name);
    TF_REQUIRE(ctx, empty || !(k == v && (k_out == k || v_out == k)), TF_ERR_INVALID_ARGUMENT, "%s: k_out or v_out may not overwrite rows that are both k and v", name);
    TF_REQUIRE(ctx, eps >= 0.0f && eps <= 3.4e38f, TF_ERR_INVALID_ARGUMENT, "%s: eps must be finite and not negative", name);
    if (batch->rows == 0 || (cache && batch->sequences == 0)) return TF_OK;
    TF_REQUIRE(ctx, batch->rows <= 0x7FFFFFFFu, TF_ERR_INVALID_ARGUMENT, "%s: rows must be below 2^31", name);
    TF_REQUIRE(ctx, tf::row_blocks(batch->rows, q_heads, kv_heads) <= 0x7FFFFFFFu, TF_ERR_UNSUPPORTED, "%s: too many rows for the number of heads", name);
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
    TF_REQUIRE(ctx, k_out || v_out || batch->rows == 0, TF_ERR_INVALID_ARGUMENT, "%s: NULL buffer", name);
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
    a.sequences = batch->sequences; a.rows = batch->rows; a.kv_heads = cache->kv_heads; a.head_log2 = tf::log2_of(cache->head_dim);
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
