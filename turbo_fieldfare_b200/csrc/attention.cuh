// Attention of the newest rows of every sequence (one token, a tree of drafted tokens, a chain) over the quantised, paged cache.
//
// With s_j = scale * q . k_j over the visible tokens j and any m, out = sum_j 2^((s_j - m) log2 e) v_j / sum_j 2^((s_j - m) log2 e): one
// pass over the tokens with the running maximum, rescaling what was summed when it grows.
//
// Work. The query heads that share a kv head are rows of one product: row f of a sequence's kv head is (token f / group, head f % group).
// A unit is MT such rows of one kv head of one sequence over all the tokens that they may see, in tiles of 64; the tiles of all units in
// a row are cut into equal shares, one per block of a grid that fills the device, so one long context, a ragged batch and many
// short ones load the device alike. The lengths are read on the device. A unit that more than one block works on
// leaves (maximum, sum, product) of each share in the workspace and attention_combine_kernel joins them in the blocks' order, which is a
// property of the lengths alone: repeats give the same bits.
//
// A tile. K and V codes and planes come by cp.async into a ring of stages (16-byte pieces swizzled so that the reads below meet no bank
// twice). Logits: warp w takes tokens 8w to 8w + 7 against all rows (mma.sync m16n8k16, rows as A). An 8-bit code c enters as the fp16
// subnormal c * 2^-24, a 4-bit one as c * 2^-24 or c * 2^-20 against a q pre-scaled by 1/16, so a pair costs one PRMT or AND; scale and
// bias come in fp32 per group, s * (q . c) + b * sum(q), so the logits carry no rounding beyond q's own. The q rows are brought to one
// power-of-two range first (bf16 rows may be outside of fp16's). After the softmax the warps take slices of the head's
// elements (and shares of the tokens where a head has few): codes of two tokens become (c - 128) * s + (b + 128 s) in fp16, the planes
// divided by a power of two that follows the largest of the tile, so no cache leaves fp16's range; its rounding, 2^-11 of the largest
// value in the group, is below the 16-bit output's. Sums are fp32.
#pragma once

#include "attention_rows.cuh"
#include "mma_gemv.cuh"

namespace tf {

constexpr int kTile = 64;                                      // tokens

constexpr int kAttnThreads = 256, kAttnWarps = kAttnThreads / kWarp;
constexpr int kCombineThreads = 128;
constexpr float kLog2e = 1.4426950408889634f;

template <int D, int BITS, int MT>
struct AttnShape {
    static constexpr int G = D / 64, ROW = D * BITS / 8, PIECES = ROW / 16, M = MT / 16;
    // warps over the second product: slices of the head's elements x shares of the tokens
    static constexpr bool NARROW = BITS == 4 && D == 64;       // a lane takes 16 bits of codes at a time, not 32
    static constexpr int UNIT = BITS == 8 || NARROW ? 32 : 64; // elements that one load per lane covers
    static constexpr int SLICE = D / 8 > UNIT ? D / 8 : UNIT, SLICES = D / SLICE, SHARES = kAttnWarps / SLICES, LOADS = SLICE / UNIT;
    static constexpr int NT = SLICE / 8;                       // n8 tiles of a slice
    static constexpr int CODES = kTile * ROW, PLANE = kTile * G * 2, STAGE = 2 * CODES + 4 * PLANE;
    static constexpr int P_PITCH = kTile + 8;                  // halves: rows of ldmatrix on distinct banks
    static constexpr int O_PITCH = D + 4;
    static constexpr int OFF_Q = 0, OFF_P = OFF_Q + MT * D * 2, OFF_SV = OFF_P + MT * P_PITCH * 2, OFF_BV = OFF_SV + G * kTile * 2,
                         OFF_QS = OFF_BV + G * kTile * 2, OFF_RF = OFF_QS + MT * G * 4, OFF_RED = OFF_RF + MT * 4,
                         OFF_VRED = OFF_RED + MT * kAttnWarps * 4, OFF_LSUM = OFF_VRED + G * kAttnWarps * 4,
                         OFF_LOW = OFF_LSUM + MT * kAttnWarps * 4, OFF_O = OFF_LOW + MT * 4,
                         OFF_STAGE = (OFF_O + (SHARES > 1 ? MT * O_PITCH * 4 : 0) + 127) / 128 * 128;
    static constexpr int stages(int budget) { return (budget - OFF_STAGE) / STAGE; }
    static constexpr int TWO = (226 * 1024) / 2 - 1024 - 512, ONE = 226 * 1024;
    // two blocks per SM where at least two stages fit beside each other, else one; four stages at most
    static constexpr int STAGES = stages(TWO) >= 2 ? (stages(TWO) > 4 ? 4 : stages(TWO)) : stages(ONE) > 4 ? 4 : stages(ONE);
    static constexpr int SMEM = OFF_STAGE + STAGES * STAGE;
    static_assert(STAGES >= 2, "a ring needs two stages");
    static __host__ __device__ __forceinline__ uint32_t k_at(uint32_t row, uint32_t byte) {
        uint32_t at = row * ROW + byte;
        if constexpr (BITS == 8) { if constexpr (ROW >= 128) at ^= (row & 1u) << 6; }
        else if constexpr (ROW >= 128) at ^= (row & 3u) << 5;
        else if constexpr (ROW == 64) at ^= ((row >> 1) & 1u) << 5;
        return at;
    }
    static __host__ __device__ __forceinline__ uint32_t v_at(uint32_t row, uint32_t byte) { return (row * ROW + byte) ^ (((row >> 1) & 3u) << 5); }
};

__device__ __forceinline__ void cp_async_16(uint32_t dst, const void* src, bool there) {
    const uint32_t bytes = there ? 16u : 0u;                   // the rest is filled with zeros
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ uint32_t h2_bits(__half2 v) { return *reinterpret_cast<uint32_t*>(&v); }
__device__ __forceinline__ __half2 bits_h2(uint32_t v) { return *reinterpret_cast<__half2*>(&v); }

__device__ __forceinline__ void attn_mma(float (&c)[4], const uint4& a, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldmatrix_x4(uint4& r, uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "r"(addr) : "memory");
}

// Exponent e of a positive finite v (v in [2^e, 2^(e+1)), subnormals as -126), within what a power of two below can be made of.
__device__ __forceinline__ int exponent_of(float v) {
    const int e = (int)((__float_as_uint(v) >> 23) & 255u) - 127;
    return max(-126, min(e, 126));
}
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float((uint32_t)(max(-126, min(e, 127)) + 127) << 23); }

template <int D, int BITS, int MT, bool BF16>
__global__ void __launch_bounds__(kAttnThreads, MT == 16 && D <= 256 ? 2 : 1)
tree_attention_kernel(const __grid_constant__ AttnArgs a) {
    using S = AttnShape<D, BITS, MT>;
    constexpr int G = S::G, M = S::M;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ unsigned long long s_scan[kAttnWarps];
    __shared__ uint32_t s_start[4];
    const uint32_t smem_base = (uint32_t)__cvta_generic_to_shared(smem);
    const int tid = threadIdx.x, warp = tid / kWarp, lane = tid % kWarp, g = lane / 4, t = lane % 4;

    // ---- this block's share of the tiles ----
    Cursor<MT, kTile> now;
    uint64_t total, item, stop;
    Shares shares;
    {
        const uint32_t per = (a.sequences + kAttnThreads - 1) / kAttnThreads, b0 = min((uint64_t)per * tid, (uint64_t)a.sequences),
                       b1 = min((uint64_t)b0 + per, (uint64_t)a.sequences);
        uint64_t mine = 0;
        for (uint32_t b = b0; b < b1; ++b) {
            Sequence s;
            s.load(a, b, blockIdx.x == 0);
            mine += sequence_tiles<MT, kTile>(a, s) * a.kv_heads;
        }
        uint64_t upto = mine;
#pragma unroll
        for (int off = 1; off < kWarp; off <<= 1) {
            const uint64_t o = __shfl_up_sync(kFullMask, upto, off);
            if (lane >= off) upto += o;
        }
        if (lane == kWarp - 1) s_scan[warp] = upto;
        __syncthreads();
        total = 0;
        uint64_t before = 0;
#pragma unroll
        for (int w = 0; w < kAttnWarps; ++w) {
            if (w == warp) before = total;
            total += s_scan[w];
        }
        before += upto - mine;
        shares.set(total, gridDim.x);
        if (tid == 0) a.info[blockIdx.x].active = 0;
        if (blockIdx.x >= shares.workers) return;
        item = shares.begin(blockIdx.x);
        stop = shares.begin(blockIdx.x + 1);
        if (item >= before && item < before + mine) {
            uint64_t left = item - before;
            for (uint32_t b = b0; b < b1; ++b) {
                Sequence s;
                s.load(a, b, false);
                const uint64_t n = sequence_tiles<MT, kTile>(a, s) * a.kv_heads;
                if (left < n) {
                    uint32_t place[3];
                    place_in_sequence<MT, kTile>(a, s, left, place);
                    s_start[0] = b; s_start[1] = place[0]; s_start[2] = place[1]; s_start[3] = place[2];
                    break;
                }
                left -= n;
            }
        }
        __syncthreads();
        now.b = s_start[0]; now.head = s_start[1]; now.flat0 = s_start[2]; now.tile = s_start[3];
        now.seq.load(a, now.b, false);
        now.range.set(a, now.seq, now.flat0, MT, kTile);
    }

    // ---- loads of a tile ----
    Cursor<MT, kTile> next = now;
    uint64_t next_item = item;
    // pages of the four runs of 16 tokens of a tile, as this thread's rows need them; -1: left out
    auto load_tile = [&](uint32_t stage) {
        const int64_t token0 = next.token0();
        int32_t page[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) page[i] = token0 + 16 * i < next.range.end ? a.table.page(next.b, token0 + 16 * i) : -1;
        const uint32_t base = smem_base + S::OFF_STAGE + stage * S::STAGE, in_page = (1u << a.table.page_log2) - 1u;
        auto row_of = [&](uint32_t r, bool& there) -> size_t {
            const uint32_t part = r >> 4;
            const int32_t p = part & 2 ? (part & 1 ? page[3] : page[2]) : (part & 1 ? page[1] : page[0]);
            there = p >= 0 && token0 + r < next.range.end;
            return there ? ((((size_t)p * a.kv_heads + next.head) << a.table.page_log2) + ((uint32_t)(token0 + r) & in_page)) : 0;
        };
#pragma unroll
        for (int i = 0; i < (kTile * S::PIECES + kAttnThreads - 1) / kAttnThreads; ++i) {
            const uint32_t id = tid + i * kAttnThreads, r = id / S::PIECES, piece = id % S::PIECES;
            if (kTile * S::PIECES % kAttnThreads != 0 && r >= kTile) break;
            bool there;
            const size_t at = row_of(r, there) * S::ROW + piece * 16;
            cp_async_16(base + S::k_at(r, piece * 16), a.k.codes + at, there);
            cp_async_16(base + S::CODES + S::v_at(r, piece * 16), a.v.codes + at, there);
        }
        // planes: 16 bytes are 8 / G rows of a plane, within one run of 16 tokens
        if (tid < 4 * 8 * G) {
            const uint32_t plane = tid / (8 * G), c = tid % (8 * G), r = c * 8 / G;
            bool there;
            const size_t at = row_of(r, there) * G;
            const uint16_t* src = plane == 0 ? a.k.scales : plane == 1 ? a.k.biases : plane == 2 ? a.v.scales : a.v.biases;
            cp_async_16(base + 2 * S::CODES + plane * S::PLANE + c * 16, src + at, there);
        }
        cp_async_commit();
    };
    // the runs of 16 tokens of the current tile that have a page
    auto runs_of = [&](const Cursor<MT, kTile>& c) -> uint32_t {
        const int64_t token0 = c.token0();
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (token0 + 16 * i < c.range.end) {
                if (a.table.page(c.b, token0 + 16 * i) >= 0) m |= 1u << i;
                else if (tid == 0) *a.error = kErrKvPage;
            }
        return m;
    };
#pragma unroll 1
    for (int i = 0; i < S::STAGES - 1; ++i) {
        if (next_item < stop) {
            load_tile(i);
            if (++next_item < stop) next.advance(a);
        } else {
            cp_async_commit();
        }
    }

    float* row_factor = reinterpret_cast<float*>(smem + S::OFF_RF);      // logits in base 2 per unit of the raw product
    float* q_sums = reinterpret_cast<float*>(smem + S::OFF_QS);          // [G][MT]
    float* red = reinterpret_cast<float*>(smem + S::OFF_RED);            // [MT][warps]
    float* v_red = reinterpret_cast<float*>(smem + S::OFF_VRED);         // [G][warps]
    float* l_sum = reinterpret_cast<float*>(smem + S::OFF_LSUM);         // [warps][MT]
    int32_t* row_low = reinterpret_cast<int32_t*>(smem + S::OFF_LOW);    // first token a row sees, from the unit's first tile on
    __half* p_rows = reinterpret_cast<__half*>(smem + S::OFF_P);
    __half* sv = reinterpret_cast<__half*>(smem + S::OFF_SV);            // [G][kTile]
    __half* bv = reinterpret_cast<__half*>(smem + S::OFF_BV);
    const int slice = warp % S::SLICES, share = warp / S::SLICES;
    constexpr int SHARE_TOKENS = kTile / S::SHARES;
    static_assert(SHARE_TOKENS % 16 == 0 && S::SLICES * S::SHARES == kAttnWarps, "warps over slices and tokens");
    const int my_group = slice * S::SLICE / 64;
    constexpr float kCentre = BITS == 8 ? 128.0f : 8.0f;

    uint32_t stage = 0;
    while (item < stop) {
        // ---- a unit's segment: q rows ----
        const uint64_t flat_rows = now.flat_rows(a);
        const uint32_t valid = (uint32_t)min((uint64_t)MT, flat_rows - now.flat0);
        const bool from_start = now.tile == 0;
        const uint32_t segment = (uint32_t)min((uint64_t)(now.range.tiles - now.tile), stop - item);
        const bool to_end = now.tile + segment == now.range.tiles;
        __syncthreads();                                       // the segment before may still read what is written here
        for (int r = warp; r < MT; r += kAttnWarps) {
            constexpr int VEC = D / 32;
            float f[VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e) f[e] = 0.0f;
            int32_t low = 0;
            if (r < (int)valid) {
                const uint32_t flat = now.flat0 + r, token = flat / a.group, h = now.head * a.group + flat % a.group;
                const uint16_t* src = a.q + (size_t)(now.seq.row0 + token) * a.q_stride + (size_t)h * D + lane * VEC;
#pragma unroll
                for (int e = 0; e < VEC; e += 2) {
                    const uint32_t w = *reinterpret_cast<const uint32_t*>(src + e);
                    if constexpr (BF16) {
                        f[e] = bf16_bits_to_float((uint16_t)w);
                        f[e + 1] = bf16_bits_to_float((uint16_t)(w >> 16));
                    } else {
                        f[e] = f16_bits_to_float((uint16_t)w);
                        f[e + 1] = f16_bits_to_float((uint16_t)(w >> 16));
                    }
                }
                if (a.window) {
                    const int64_t pos = a.mask ? max((int64_t)a.positions[now.seq.row0 + token], (int64_t)now.seq.context) : (int64_t)now.seq.context + token;
                    const int64_t l = pos - (int64_t)a.window + 1 - (int64_t)now.range.tile0 * kTile;
                    low = (int32_t)max((int64_t)0, min(l, (int64_t)0x7FFFFFFF));
                }
            }
            float most = 0.0f;
#pragma unroll
            for (int e = 0; e < VEC; ++e) most = fmaxf(most, fabsf(f[e]));
#pragma unroll
            for (int off = 16; off >= 1; off >>= 1) most = fmaxf(most, __shfl_xor_sync(kFullMask, most, off));
            const int e2 = most > 0.0f ? max(exponent_of(most) - 7, -126) : 0;      // the largest element to [128, 256)
            const float down = power_of_two(-e2);
            float sum = 0.0f;
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const int d = lane * VEC + e, dd = d % 64, tt = dd / 16, j = dd % 16;
                int ks, reg, half;
                float v = f[e] * down;
                if constexpr (BITS == 8) {
                    ks = j / 4; reg = (j % 4) / 2; half = j % 2;
                } else {
                    const int n = j % 8;
                    ks = 2 * (j / 8) + (n % 4) / 2; reg = n % 2; half = n / 4;
                }
                const bool sixteenth = BITS == 4 && (j % 2);
                const __half hv = __float2half_rn(sixteenth ? v * 0.0625f : v);
                sum += __half2float(hv) * (sixteenth ? 16.0f : 1.0f);
                const int at = ((((r / 16) * (D / 16) + (d / 64) * 4 + ks) * 32 + (r % 8) * 4 + tt) * 4 + reg * 2 + (r % 16) / 8) * 2 + half;
                reinterpret_cast<__half*>(smem + S::OFF_Q)[at] = hv;
            }
            constexpr int LANES = 64 / VEC;                    // lanes of a group
#pragma unroll
            for (int off = LANES / 2; off >= 1; off >>= 1) sum += __shfl_xor_sync(kFullMask, sum, off);
            if (lane % LANES == 0) q_sums[(lane / LANES) * MT + r] = sum * 5.9604644775390625e-8f;   // 2^-24, as the products
            if (lane == 0) {
                row_factor[r] = 16777216.0f * power_of_two(e2) * a.scale * kLog2e;
                row_low[r] = low;
            }
        }
        float m[M][2], l[M][2], o[M][S::NT][4];
#pragma unroll
        for (int i = 0; i < M; ++i) {
            m[i][0] = m[i][1] = -INFINITY;
            l[i][0] = l[i][1] = 0.0f;
#pragma unroll
            for (int j = 0; j < S::NT; ++j) o[i][j][0] = o[i][j][1] = o[i][j][2] = o[i][j][3] = 0.0f;
        }
        int e_mine = -126, e_prep = -126;                      // exponents of the value planes so far: of this warp's group, of the prepared one
        int32_t low_most = 0;                                  // the last of the rows' first tokens
        __syncthreads();
        if (a.window)
            for (uint32_t r = 0; r < valid; ++r) low_most = max(low_most, row_low[r]);

        for (uint32_t done = 0; done < segment; ++done, ++item) {
            const uint32_t runs = runs_of(now);
            const int64_t token0 = now.token0();
            const int32_t rel0 = now.tile * kTile;             // of the tile's first token, as row_low counts
            cp_async_wait<S::STAGES - 2>();
            __syncthreads();                                   // the tile has landed for all
            if (next_item < stop) {
                load_tile((stage + S::STAGES - 1) % S::STAGES);
                if (++next_item < stop) next.advance(a);
            } else {
                cp_async_commit();
            }
            const uint8_t* st = smem + S::OFF_STAGE + stage * S::STAGE;

            // ---- logits of 8 tokens ----
            float x[M][4];
#pragma unroll
            for (int i = 0; i < M; ++i) x[i][0] = x[i][1] = x[i][2] = x[i][3] = 0.0f;
            const uint16_t* ks16 = reinterpret_cast<const uint16_t*>(st + 2 * S::CODES);
            const uint16_t* kb16 = reinterpret_cast<const uint16_t*>(st + 2 * S::CODES + S::PLANE);
#pragma unroll
            for (int grp = 0; grp < G; ++grp) {
                uint32_t w[4];
                if constexpr (BITS == 8) {
                    const uint4 c = *reinterpret_cast<const uint4*>(st + S::k_at(8 * warp + g, grp * 64 + 16 * t));
                    w[0] = c.x; w[1] = c.y; w[2] = c.z; w[3] = c.w;
                } else {
                    const uint2 c = *reinterpret_cast<const uint2*>(st + S::k_at(8 * warp + g, grp * 32 + 8 * t));
                    w[0] = c.x; w[1] = c.x >> 8; w[2] = c.y; w[3] = c.y >> 8;
                }
                float acc[M][4];
#pragma unroll
                for (int i = 0; i < M; ++i) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.0f;
#pragma unroll
                for (int ks = 0; ks < 4; ++ks) {
                    uint32_t b0, b1;
                    if constexpr (BITS == 8) {
                        b0 = gm_prmt(w[ks], 0, 0x4140);
                        b1 = gm_prmt(w[ks], 0, 0x4342);
                    } else {
                        b0 = w[ks] & 0x000F000Fu;
                        b1 = w[ks] & 0x00F000F0u;
                    }
#pragma unroll
                    for (int i = 0; i < M; ++i) {
                        const uint4 qa = *reinterpret_cast<const uint4*>(smem + S::OFF_Q + (((i * (D / 16) + grp * 4 + ks) * 32 + lane) << 4));
                        attn_mma(acc[i], qa, b0, b1);
                    }
                }
                const int key = 8 * warp + 2 * t;
                const float s0 = bf16_bits_to_float(ks16[key * G + grp]), s1 = bf16_bits_to_float(ks16[(key + 1) * G + grp]);
                const float b0 = bf16_bits_to_float(kb16[key * G + grp]), b1 = bf16_bits_to_float(kb16[(key + 1) * G + grp]);
#pragma unroll
                for (int i = 0; i < M; ++i) {
                    const float q0 = q_sums[grp * MT + 16 * i + g], q1 = q_sums[grp * MT + 16 * i + g + 8];
                    x[i][0] = fmaf(s0, acc[i][0], fmaf(b0, q0, x[i][0]));
                    x[i][1] = fmaf(s1, acc[i][1], fmaf(b1, q0, x[i][1]));
                    x[i][2] = fmaf(s0, acc[i][2], fmaf(b0, q1, x[i][2]));
                    x[i][3] = fmaf(s1, acc[i][3], fmaf(b1, q1, x[i][3]));
                }
            }
            // ---- mask; the rows' maxima over this warp's tokens ----
            const bool open = runs == 15u && rel0 >= low_most && token0 + kTile <= now.seq.context;     // rows behind the valid ones are zeros
#pragma unroll
            for (int i = 0; i < M; ++i) {
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const int r = 16 * i + g + (c >= 2 ? 8 : 0), key = 8 * warp + 2 * t + (c & 1);
                    x[i][c] *= row_factor[r];
                    if (!open) {
                        const int64_t token = token0 + key;
                        bool seen = r < (int)valid && (runs >> (key >> 4) & 1u) && token < now.range.end;
                        if (seen) {
                            if (token < now.seq.context) {
                                seen = rel0 + key >= row_low[r];
                            } else {
                                const uint32_t j = (uint32_t)(token - now.seq.context), row = (now.flat0 + r) / a.group;
                                if (a.mask) seen = (a.mask[(size_t)(now.seq.row0 + row) * a.mask_words + (j >> 6)] >> (j & 63u)) & 1ull;
                                else seen = j <= row && (!a.window || row - j < a.window);
                            }
                        }
                        if (!seen) x[i][c] = -INFINITY;
                    }
                }
                float m0 = fmaxf(x[i][0], x[i][1]), m1 = fmaxf(x[i][2], x[i][3]);
                m0 = fmaxf(m0, __shfl_xor_sync(kFullMask, m0, 1));
                m1 = fmaxf(m1, __shfl_xor_sync(kFullMask, m1, 1));
                m0 = fmaxf(m0, __shfl_xor_sync(kFullMask, m0, 2));
                m1 = fmaxf(m1, __shfl_xor_sync(kFullMask, m1, 2));
                if (t == 0) {
                    red[(16 * i + g) * kAttnWarps + warp] = m0;
                    red[(16 * i + g + 8) * kAttnWarps + warp] = m1;
                }
            }
            // ---- value planes of this warp's tokens, centred: (c - centre) * s + (b + centre * s) ----
            constexpr int PREP = 8 * G > 32 ? 2 : 1;
            const uint16_t* vs16 = reinterpret_cast<const uint16_t*>(st + 2 * S::CODES + 2 * S::PLANE);
            const uint16_t* vb16 = reinterpret_cast<const uint16_t*>(st + 2 * S::CODES + 3 * S::PLANE);
            float ps[PREP], pb[PREP], most = 0.0f;
            bool broken = false;
#pragma unroll
            for (int n = 0; n < PREP; ++n) {
                const int idx = lane + 32 * n, key = 8 * warp + idx / G;
                ps[n] = pb[n] = 0.0f;
                if (idx < 8 * G && (runs >> (key >> 4) & 1u) && token0 + key < now.range.end) {
                    ps[n] = bf16_bits_to_float(vs16[key * G + idx % G]);
                    pb[n] = fmaf(kCentre, ps[n], bf16_bits_to_float(vb16[key * G + idx % G]));
                    const float mag = fmaxf(kCentre * fabsf(ps[n]), fabsf(pb[n]));
                    if (ps[n] - ps[n] == 0.0f && pb[n] - pb[n] == 0.0f) most = fmaxf(most, mag);
                    else broken = true;
                }
            }
            const bool any_broken = __any_sync(kFullMask, broken);
#pragma unroll
            for (int off = G; off < kWarp; off <<= 1) most = fmaxf(most, __shfl_xor_sync(kFullMask, most, off));
            if (lane < G) v_red[lane * kAttnWarps + warp] = any_broken ? -most : most;      // the sign: a plane here is not finite
            __syncthreads();

            // ---- probabilities ----
            float alpha[M][2];
#pragma unroll
            for (int i = 0; i < M; ++i) {
#pragma unroll
                for (int hi = 0; hi < 2; ++hi) {
                    const int r = 16 * i + g + 8 * hi;
                    const float4 u = *reinterpret_cast<const float4*>(red + r * kAttnWarps), v = *reinterpret_cast<const float4*>(red + r * kAttnWarps + 4);
                    const float top = fmaxf(fmaxf(fmaxf(u.x, u.y), fmaxf(u.z, u.w)), fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w)));
                    const float m_new = fmaxf(m[i][hi], top), base = m_new == -INFINITY ? 0.0f : m_new;
                    alpha[i][hi] = exp2f(m[i][hi] - base);
                    m[i][hi] = m_new;
                    const __half2 p = __floats2half2_rn(exp2f(x[i][2 * hi] - base), exp2f(x[i][2 * hi + 1] - base));
                    const float2 pf = __half22float2(p);       // the sum takes what the product takes
                    l[i][hi] = fmaf(l[i][hi], alpha[i][hi], pf.x + pf.y);
                    *reinterpret_cast<__half2*>(p_rows + r * S::P_PITCH + 8 * warp + 2 * t) = p;
                }
            }
            bool tile_broken = false;
            {
                auto exponent = [&](int grp, int before) {
                    const float4 u = *reinterpret_cast<const float4*>(v_red + grp * kAttnWarps), v = *reinterpret_cast<const float4*>(v_red + grp * kAttnWarps + 4);
                    const uint32_t signs = (__float_as_uint(u.x) | __float_as_uint(u.y) | __float_as_uint(u.z) | __float_as_uint(u.w) |
                                            __float_as_uint(v.x) | __float_as_uint(v.y) | __float_as_uint(v.z) | __float_as_uint(v.w)) >> 31;
                    tile_broken |= signs != 0;
                    const float top = fmaxf(fmaxf(fmaxf(fabsf(u.x), fabsf(u.y)), fmaxf(fabsf(u.z), fabsf(u.w))),
                                            fmaxf(fmaxf(fabsf(v.x), fabsf(v.y)), fmaxf(fabsf(v.z), fabsf(v.w))));
                    return max(before, exponent_of(top) - 7);  // |(c - centre) * s| and |b + centre * s| below 2^8
                };
                e_prep = exponent(lane % G, e_prep);
                const float down = power_of_two(-e_prep);
#pragma unroll
                for (int n = 0; n < PREP; ++n) {
                    const int idx = lane + 32 * n;
                    if (idx < 8 * G) {
                        sv[(idx % G) * kTile + 8 * warp + idx / G] = __float2half_rn(ps[n] * down);
                        bv[(idx % G) * kTile + 8 * warp + idx / G] = __float2half_rn(pb[n] * down);
                    }
                }
                const int e_new = exponent(my_group, e_mine);
                const float fit = power_of_two(e_mine - e_new);
                e_mine = e_new;
#pragma unroll
                for (int i = 0; i < M; ++i) {
                    const float a0 = alpha[i][0] * fit, a1 = alpha[i][1] * fit;
#pragma unroll
                    for (int j = 0; j < S::NT; ++j) { o[i][j][0] *= a0; o[i][j][1] *= a0; o[i][j][2] *= a1; o[i][j][3] *= a1; }
                }
            }
            __syncthreads();

            // ---- values ----
            {
                const uint8_t* vt = st + S::CODES;
#pragma unroll
                for (int k0 = 0; k0 < SHARE_TOKENS; k0 += 16) {
                    const int key = share * SHARE_TOKENS + k0 + 2 * t;
                    __half2 s_lo = *reinterpret_cast<const __half2*>(sv + my_group * kTile + key), s_hi = *reinterpret_cast<const __half2*>(sv + my_group * kTile + key + 8);
                    __half2 b_lo = *reinterpret_cast<const __half2*>(bv + my_group * kTile + key), b_hi = *reinterpret_cast<const __half2*>(bv + my_group * kTile + key + 8);
                    uint4 pa[M];
#pragma unroll
                    for (int i = 0; i < M; ++i)
                        ldmatrix_x4(pa[i], smem_base + S::OFF_P + ((16 * i + lane % 16) * S::P_PITCH + share * SHARE_TOKENS + k0 + lane / 16 * 8) * 2);
                    if (tile_broken) {
                        // planes that are not finite count as zeros, and the rows whose probability there is not zero become NaN
                        const float ok[4] = {__low2float(s_lo) * 0.0f + __low2float(b_lo) * 0.0f, __high2float(s_lo) * 0.0f + __high2float(b_lo) * 0.0f,
                                             __low2float(s_hi) * 0.0f + __low2float(b_hi) * 0.0f, __high2float(s_hi) * 0.0f + __high2float(b_hi) * 0.0f};
                        const __half zero = __float2half_rn(0.0f);
                        if (ok[0] != 0.0f) { s_lo = __halves2half2(zero, __high2half(s_lo)); b_lo = __halves2half2(zero, __high2half(b_lo)); }
                        if (ok[1] != 0.0f) { s_lo = __halves2half2(__low2half(s_lo), zero); b_lo = __halves2half2(__low2half(b_lo), zero); }
                        if (ok[2] != 0.0f) { s_hi = __halves2half2(zero, __high2half(s_hi)); b_hi = __halves2half2(zero, __high2half(b_hi)); }
                        if (ok[3] != 0.0f) { s_hi = __halves2half2(__low2half(s_hi), zero); b_hi = __halves2half2(__low2half(b_hi), zero); }
                        for (int kk = 0; kk < 16; ++kk) {
                            const int at = share * SHARE_TOKENS + k0 + kk;
                            const float f = __half2float(sv[my_group * kTile + at]) * 0.0f + __half2float(bv[my_group * kTile + at]) * 0.0f;
                            if (f == 0.0f) continue;
#pragma unroll
                            for (int i = 0; i < M; ++i) {
#pragma unroll
                                for (int hi = 0; hi < 2; ++hi)
                                    if (__half2float(p_rows[(16 * i + g + 8 * hi) * S::P_PITCH + at]) > 0.0f) {
#pragma unroll
                                        for (int j = 0; j < S::NT; ++j) o[i][j][2 * hi] = o[i][j][2 * hi + 1] = __int_as_float(0x7FC00000);
                                    }
                            }
                        }
                    }
#pragma unroll
                    for (int n = 0; n < S::LOADS; ++n) {
                        const uint32_t col = slice * (S::SLICE * BITS / 8) + n * (S::UNIT * BITS / 8);
                        uint32_t lo_pairs[8], hi_pairs[8];     // (token, token + 1) and (token + 8, token + 9) of each element
                        auto unpack = [&](uint32_t wa, uint32_t wb, __half2 s2, __half2 b2, uint32_t (&out)[8]) {
                            if constexpr (BITS == 8) {
                                const uint32_t t0 = gm_prmt(wa, wb, 0x5140), t1 = gm_prmt(wa, wb, 0x7362);
                                const __half2 off = __half2half2(__float2half_rn(-1152.0f));     // 1024 from the bits, 128 the centre
                                const uint32_t c[4] = {gm_prmt(t0, 0x64646464u, 0x4140), gm_prmt(t0, 0x64646464u, 0x4342),
                                                       gm_prmt(t1, 0x64646464u, 0x4140), gm_prmt(t1, 0x64646464u, 0x4342)};
#pragma unroll
                                for (int j = 0; j < 4; ++j) out[j] = h2_bits(__hfma2(__hadd2(bits_h2(c[j]), off), s2, b2));
                            } else {
                                const __half2 off = __half2half2(__float2half_rn(-1032.0f)), off16 = __half2half2(__float2half_rn(-1152.0f));
                                const __half2 s16 = __hmul2(s2, __half2half2(__float2half_rn(0.0625f)));
#pragma unroll
                                for (int half = 0; half < (S::NARROW ? 1 : 2); ++half) {
                                    const uint32_t u = gm_prmt(wa, wb, half ? 0x7632 : 0x5410), u8 = u >> 8;
                                    out[4 * half + 0] = h2_bits(__hfma2(__hadd2(bits_h2((u & 0x000F000Fu) | 0x64006400u), off), s2, b2));
                                    out[4 * half + 1] = h2_bits(__hfma2(__hadd2(bits_h2((u & 0x00F000F0u) | 0x64006400u), off16), s16, b2));
                                    out[4 * half + 2] = h2_bits(__hfma2(__hadd2(bits_h2((u8 & 0x000F000Fu) | 0x64006400u), off), s2, b2));
                                    out[4 * half + 3] = h2_bits(__hfma2(__hadd2(bits_h2((u8 & 0x00F000F0u) | 0x64006400u), off16), s16, b2));
                                }
                            }
                        };
                        auto word = [&](int row) -> uint32_t {
                            if constexpr (S::NARROW) return *reinterpret_cast<const uint16_t*>(vt + S::v_at(row, col + 2 * g));
                            else return *reinterpret_cast<const uint32_t*>(vt + S::v_at(row, col + 4 * g));
                        };
                        unpack(word(key), word(key + 1), s_lo, b_lo, lo_pairs);
                        unpack(word(key + 8), word(key + 9), s_hi, b_hi, hi_pairs);
                        constexpr int PER = S::UNIT / 8;
#pragma unroll
                        for (int j = 0; j < PER; ++j) {
#pragma unroll
                            for (int i = 0; i < M; ++i) attn_mma(o[i][n * PER + j], pa[i], lo_pairs[j], hi_pairs[j]);
                        }
                    }
                }
            }
            stage = stage + 1 == S::STAGES ? 0 : stage + 1;
            if (done + 1 < segment) ++now.tile;
        }

        // ---- the segment's result ----
#pragma unroll
        for (int i = 0; i < M; ++i) {
#pragma unroll
            for (int hi = 0; hi < 2; ++hi) {
                float s = l[i][hi];
                s += __shfl_xor_sync(kFullMask, s, 1);
                s += __shfl_xor_sync(kFullMask, s, 2);
                if (t == 0) l_sum[warp * MT + 16 * i + g + 8 * hi] = s;
            }
        }
        const float up = power_of_two(e_mine);
        constexpr int PER = S::UNIT / 8;                       // elements of one code word: a thread ends up with 2 * PER neighbours
        float* o_rows = reinterpret_cast<float*>(smem + S::OFF_O);
        const bool whole = from_start && to_end;
        float* part = a.partial + (size_t)(2 * blockIdx.x + (from_start ? 1 : 0)) * MT * (D + 2);
        auto row_sum = [&](int r) {
            float s = 0.0f;
#pragma unroll
            for (int w = 0; w < kAttnWarps; ++w) s += l_sum[w * MT + r];
            return s;
        };
        auto out_row = [&](int r) -> uint16_t* {
            const uint32_t flat = now.flat0 + r;
            return a.out + (size_t)(now.seq.row0 + flat / a.group) * a.out_stride + (size_t)(now.head * a.group + flat % a.group) * D;
        };
        auto store_run = [&](int r, int d, const float* v, int n, float inv) {     // n: 8 or 16 neighbours
            if (whole) {
                uint16_t* dst = out_row(r) + d;
                for (int e = 0; e < n; e += 8) {
                    uint32_t w[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float y0 = v[e + 2 * j] * inv, y1 = v[e + 2 * j + 1] * inv;
                        if constexpr (BF16) { const __nv_bfloat162 b = __floats2bfloat162_rn(y0, y1); w[j] = *reinterpret_cast<const uint32_t*>(&b); }
                        else w[j] = h2_bits(__floats2half2_rn(y0, y1));
                    }
                    *reinterpret_cast<uint4*>(dst + e) = make_uint4(w[0], w[1], w[2], w[3]);
                }
            } else {
                float* dst = part + 2 * MT + (size_t)r * D + d;
                for (int e = 0; e < n; e += 4) *reinterpret_cast<float4*>(dst + e) = make_float4(v[e], v[e + 1], v[e + 2], v[e + 3]);
            }
        };
        if constexpr (S::SHARES == 1) {
            __syncthreads();                                   // l_sum
#pragma unroll
            for (int i = 0; i < M; ++i) {
#pragma unroll
                for (int hi = 0; hi < 2; ++hi) {
                    const int r = 16 * i + g + 8 * hi;
                    if (r < (int)valid) {
                        const float s = row_sum(r), inv = s == 0.0f ? 0.0f : 1.0f / s;
#pragma unroll
                        for (int n = 0; n < S::LOADS; ++n) {
                            float v[2 * PER];
#pragma unroll
                            for (int j = 0; j < PER; ++j) {
                                v[j] = o[i][n * PER + j][2 * hi] * up;
                                v[PER + j] = o[i][n * PER + j][2 * hi + 1] * up;
                            }
                            store_run(r, slice * S::SLICE + n * S::UNIT + 2 * PER * t, v, 2 * PER, inv);
                        }
                    }
                }
            }
        } else {
            // shares of the tokens meet in shared memory, one after the other
#pragma unroll 1
            for (int turn = 0; turn < S::SHARES; ++turn) {
                if (share == turn) {
#pragma unroll
                    for (int i = 0; i < M; ++i) {
#pragma unroll
                        for (int hi = 0; hi < 2; ++hi) {
#pragma unroll
                            for (int n = 0; n < S::LOADS; ++n) {
                                float* dst = o_rows + (16 * i + g + 8 * hi) * S::O_PITCH + slice * S::SLICE + n * S::UNIT + 2 * PER * t;
#pragma unroll
                                for (int j = 0; j < PER; ++j) {
                                    const float v0 = o[i][n * PER + j][2 * hi] * up, v1 = o[i][n * PER + j][2 * hi + 1] * up;
                                    dst[j] = turn ? dst[j] + v0 : v0;
                                    dst[PER + j] = turn ? dst[PER + j] + v1 : v1;
                                }
                            }
                        }
                    }
                }
                __syncthreads();
            }
            for (int idx = tid; idx < (int)valid * (D / 8); idx += kAttnThreads) {
                const int r = idx / (D / 8), d = idx % (D / 8) * 8;
                const float s = row_sum(r), inv = s == 0.0f ? 0.0f : 1.0f / s;
                float v[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = o_rows[r * S::O_PITCH + d + e];
                store_run(r, d, v, 8, inv);
            }
        }
        if (!whole) {
            if (warp == 0) {
#pragma unroll
                for (int i = 0; i < M; ++i) {
#pragma unroll
                    for (int hi = 0; hi < 2; ++hi) {
                        const int r = 16 * i + g + 8 * hi;
                        if (t == 0 && r < (int)valid) {
                            part[r] = m[i][hi];
                            part[MT + r] = row_sum(r);
                        }
                    }
                }
            }
            if (from_start && tid == 0) {
                const uint64_t end_item = item - segment + now.range.tiles;      // of the unit; it begins in this share
                ShareInfo& info = a.info[blockIdx.x];
                info.last = shares.of(end_item - 1);
                info.row0 = now.seq.row0;
                info.flat0 = now.flat0;
                info.valid = valid;
                info.head = now.head;
                info.active = 1;
            }
        }
        if (item < stop) now.next_unit(a);
    }
    cp_async_wait<0>();
}

// Joins the shares of a unit that blocks c to last_block worked on: a warp per row, lanes over the head's elements.
template <int D, int MT, bool BF16>
__global__ void __launch_bounds__(kCombineThreads)
attention_combine_kernel(const AttnArgs a) {
    constexpr int VEC = D / 32;
    pdl_wait();
    const uint32_t c = blockIdx.x;
    const ShareInfo info = a.info[c];
    const uint32_t warp = threadIdx.x / kWarp, lane = threadIdx.x % kWarp, r = blockIdx.y * (kCombineThreads / kWarp) + warp;
    if (!info.active || r >= info.valid) return;
    const uint32_t parts = info.last - c + 1;
    constexpr size_t kSlot = (size_t)MT * (D + 2);
    auto slot = [&](uint32_t p) { return a.partial + (size_t)(p == 0 ? 2 * c + 1 : 2 * (c + p)) * kSlot; };
    float top = -INFINITY;
    for (uint32_t p = lane; p < parts; p += kWarp) top = fmaxf(top, slot(p)[r]);
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) top = fmaxf(top, __shfl_xor_sync(kFullMask, top, off));
    const float base = top == -INFINITY ? 0.0f : top;
    float sum = 0.0f, v[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) v[e] = 0.0f;
    for (uint32_t p0 = 0; p0 < parts; p0 += kWarp) {
        float w = 0.0f, l = 0.0f;
        if (p0 + lane < parts) {
            const float* s = slot(p0 + lane);
            w = exp2f(s[r] - base);
            l = s[MT + r];
        }
        const uint32_t n = min(parts - p0, (uint32_t)kWarp);
#pragma unroll 4
        for (uint32_t j = 0; j < n; ++j) {
            const float wj = __shfl_sync(kFullMask, w, j), lj = __shfl_sync(kFullMask, l, j);
            const float* src = slot(p0 + j) + 2 * MT + (size_t)r * D + lane * VEC;
            sum = fmaf(wj, lj, sum);
#pragma unroll
            for (int e = 0; e < VEC; e += 2) {
                const float2 x = *reinterpret_cast<const float2*>(src + e);
                v[e] = fmaf(wj, x.x, v[e]);
                v[e + 1] = fmaf(wj, x.y, v[e + 1]);
            }
        }
    }
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    const uint32_t flat = info.flat0 + r;
    uint16_t* dst = a.out + (size_t)(info.row0 + flat / a.group) * a.out_stride + (size_t)(info.head * a.group + flat % a.group) * D + lane * VEC;
#pragma unroll
    for (int e = 0; e < VEC; e += 2) {
        uint32_t w;
        if constexpr (BF16) { const __nv_bfloat162 b = __floats2bfloat162_rn(v[e] * inv, v[e + 1] * inv); w = *reinterpret_cast<const uint32_t*>(&b); }
        else w = h2_bits(__floats2half2_rn(v[e] * inv, v[e + 1] * inv));
        *reinterpret_cast<uint32_t*>(dst + e) = w;
    }
}

template <int D, int BITS, int MT, bool BF16>
static tf_status launch_attention(tf_context* ctx, cudaStream_t st, const AttnArgs& a, const tf_attention_workspace* ws) {
    using S = AttnShape<D, BITS, MT>;
    auto kernel = tree_attention_kernel<D, BITS, MT, BF16>;
    static DeviceSmemCache smem_cache;
    static ResidentBlocksCache blocks_cache;
    const tf_status s = ensure_dynamic_smem(ctx, kernel, smem_cache, S::SMEM);
    if (s != TF_OK) return s;
    uint32_t blocks = resident_blocks(ctx, kernel, blocks_cache, kAttnThreads, S::SMEM);
    if (blocks > ws->row_capacity / MT) blocks = ws->row_capacity / MT;
    if (blocks > ws->max_workers) blocks = ws->max_workers;
    TF_REQUIRE(ctx, blocks > 0, TF_ERR_CUDA, "tf_tree_attention: the kernel does not fit on the device");
    kernel<<<blocks, kAttnThreads, S::SMEM, st>>>(a);
    const tf_status t = check_launch(ctx, "tf_tree_attention");
    if (t != TF_OK) return t;
    TF_CUDA(ctx, launch_pdl(attention_combine_kernel<D, MT, BF16>, dim3(blocks, MT / (kCombineThreads / kWarp)), dim3(kCombineThreads), 0, st, a));
    return check_launch(ctx, "tf_tree_attention (combine)");
}

template <int D, int BITS>
tf_status attend(tf_context* ctx, cudaStream_t st, const AttnArgs& a, const tf_attention_workspace* ws, bool bf16) {
    // Rows of one kv head in a mean sequence: units of 16 rows while they hold them, else of 64, which read a tile once for four times as many.
    const uint64_t mean = ((uint64_t)a.rows + a.sequences - 1) / a.sequences * a.group;
    if (mean <= 8) return bf16 ? launch_rows<D, BITS, 8, true>(ctx, st, a, ws) : launch_rows<D, BITS, 8, false>(ctx, st, a, ws);
    if (mean <= 16) return bf16 ? launch_attention<D, BITS, 16, true>(ctx, st, a, ws) : launch_attention<D, BITS, 16, false>(ctx, st, a, ws);
    return bf16 ? launch_attention<D, BITS, 64, true>(ctx, st, a, ws) : launch_attention<D, BITS, 64, false>(ctx, st, a, ws);
}

}  // namespace tf

