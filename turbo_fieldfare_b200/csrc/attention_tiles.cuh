// Attention over the quantised, paged cache for units of up to 128 rows (trees and chains): tcgen05 with tensor-memory accumulators.
//
// With this many rows the products bound it, 4 * 128 * D FLOP per token and unit, next to the unpacking, which a unit pays once for its 128 rows.
// One persistent block per SM; 8 warps unpack, one issues the MMAs, 4 do the softmax, a thread per row. For tile i of TILE tokens:
//   unpack:  codes and planes from global memory (requested a tile ahead) -> K_i, V_i in fp16, [64 elements][token][128 bytes] with the 128-byte
//            swizzle, two buffers each
//   MMA:     S_i = Q K_i^T into tensor memory (two buffers), then O += P_(i-1) V_(i-1); K is K-major, V, as it lies, MN-major
//   softmax: S_i -> registers -> mask, 2^(x - m), P_i as fp16 into tensor memory (the A operand of the second product)
// K_i and V_i carry (code - centre) s + (bias + centre s) rounded to fp16, 2^-11 of the value: logits see it as an error of about 2^-12 |q||k| / sqrt(D),
// of the size of the output's own rounding to 16 bits. The planes are divided by powers of two that follow the largest of the tile (K) or
// of all tiles so far (V), so caches outside of fp16's range work; a token's values keep their precision beside others up to 2^20 times as large.
// m is raised only when a logit exceeds it by 8, and what O holds is rescaled only then, or when V's exponent grows. TILE * D is 16384 but for heads of 64,
// so the buffers of all head sizes have the same size; heads of 512, whose product would fill tensor memory alone, are two units
// with half of the values each.
#pragma once

#include "async_copy.cuh"
#include "attention_rows.cuh"

namespace tf {

constexpr uint32_t kErrAttentionWait = 0x7F000053u;           // a bounded wait of attention_tiles_kernel ran out

template <int D, int BITS>
struct TilesShape {
    static constexpr int MT = 128, TILE = D == 512 ? 32 : D == 256 ? 64 : 128, DV = D < 256 ? D : 256, PARTS = D / DV, G = D / 64, GV = DV / 64;
    static constexpr int SOFT_WARPS = 4, UNPACK_WARPS = 8, WARPS = SOFT_WARPS + UNPACK_WARPS + 1, THREADS = WARPS * kWarp, UNPACK = UNPACK_WARPS * kWarp;
    static constexpr int ROW_BYTES = D * BITS / 8, PIECE = 2 * BITS;          // bytes of 16 codes
    static constexpr int K_ROW = D / 16, V_ROW = DV / 16;                     // pieces of a token
    static constexpr int K_EACH = TILE * K_ROW / UNPACK, V_EACH = TILE * V_ROW / UNPACK;
    static constexpr int RUNS = TILE / 16;
    static constexpr int Q_BYTES = MT * D * 2, K_BYTES = TILE * D * 2, V_BYTES = TILE * DV * 2;
    static constexpr int OFF_K = Q_BYTES, OFF_V = OFF_K + 2 * K_BYTES, OFF_META = OFF_V + 2 * V_BYTES, META = 1024, SMEM = OFF_META + META + 1024;
    // tensor memory, in columns
    static constexpr int COL_S = 0, COL_P = 2 * TILE, COL_O = 3 * TILE, COLS = 512;
    static_assert(COL_O + DV <= COLS && SMEM <= 227 * 1024 && K_EACH * UNPACK == TILE * K_ROW && V_EACH * UNPACK == TILE * V_ROW, "sizes");
    // a 16-byte chunk (eight elements) of an operand row: [64 elements][rows][128 bytes], chunks swizzled by the row
    static __host__ __device__ __forceinline__ uint32_t chunk_at(uint32_t rows, uint32_t row, uint32_t chunk) {
        return (chunk >> 3) * (rows * 128) + row * 128 + (((chunk & 7u) ^ (row & 7u)) << 4);
    }
};

// What the unpacking warps tell the softmax about a tile, and the rest of the block's small things.
struct TilesMeta {
    unsigned long long bars[16];
    uint32_t tmem, dead;
    float largest[2][2][8];        // [tile parity][K, V][warp]
    int32_t e_k[2], e_v[2];
    uint32_t runs[2], any_bad[2];
    uint32_t bad[2][4][4];         // value planes that are not finite: [tile parity][group][32 tokens]
};
static_assert(sizeof(TilesMeta) <= 1024, "meta");

__device__ __forceinline__ uint64_t tiles_desc(uint32_t addr, uint32_t leading, uint32_t stride) {     // 128-byte swizzle
    return (uint64_t)((addr & 0x3FFFFu) >> 4) | ((uint64_t)(leading >> 4) << 16) | ((uint64_t)(stride >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
__device__ __forceinline__ void tiles_mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void tiles_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
                 ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void tiles_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void tiles_ld32(uint32_t addr, uint32_t (&r)[32]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 "
                 "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
                   "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]),
                   "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
                 : "r"(addr) : "memory");
}
__device__ __forceinline__ void tiles_st32(uint32_t addr, const uint32_t (&r)[32]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
                 "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};"
                 ::"r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
                   "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]),
                   "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]) : "memory");
}
__device__ __forceinline__ void tiles_st16(uint32_t addr, const uint32_t (&r)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
                 ::"r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
                   "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]) : "memory");
}
__device__ __forceinline__ void tiles_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tiles_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tiles_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tiles_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// Sixteen codes as (code - centre) s + b in fp16, two 16-byte chunks of eight elements. 4-bit codes of eight elements come in the order
// (0, 4, 1, 5, 2, 6, 3, 7), as one mask yields them: the rows of q are laid out alike, and the product's columns are put back at the end.
template <int BITS>
__device__ __forceinline__ void tiles_unpack(const uint32_t (&w)[BITS / 2], float scale, float bias, uint4 (&out)[2]) {
    const __half2 s = __float2half2_rn(scale), b = __float2half2_rn(bias);
    uint32_t h[8];
    auto put = [&](int i, uint32_t bits, float off, __half2 by) {
        const __half2 v = __hfma2(__hadd2(*reinterpret_cast<const __half2*>(&bits), __float2half2_rn(off)), by, b);
        h[i] = *reinterpret_cast<const uint32_t*>(&v);
    };
    if constexpr (BITS == 8) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            put(2 * i, gm_prmt(w[i], 0x64646464u, 0x4140), -1152.0f, s);             // 1024 from the bits, 128 the centre
            put(2 * i + 1, gm_prmt(w[i], 0x64646464u, 0x4342), -1152.0f, s);
        }
    } else {
        const __half2 s16 = __float2half2_rn(scale * 0.0625f);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint32_t v = w[i] >> 8;
            put(4 * i, (w[i] & 0x000F000Fu) | 0x64006400u, -1032.0f, s);
            put(4 * i + 1, (w[i] & 0x00F000F0u) | 0x64006400u, -1152.0f, s16);
            put(4 * i + 2, (v & 0x000F000Fu) | 0x64006400u, -1032.0f, s);
            put(4 * i + 3, (v & 0x00F000F0u) | 0x64006400u, -1152.0f, s16);
        }
    }
    out[0] = make_uint4(h[0], h[1], h[2], h[3]);
    out[1] = make_uint4(h[4], h[5], h[6], h[7]);
}

template <int D, int BITS, bool BF16>
__global__ void __launch_bounds__(TilesShape<D, BITS>::THREADS, 1)
attention_tiles_kernel(const __grid_constant__ AttnArgs a) {
    using S = TilesShape<D, BITS>;
    constexpr int MT = S::MT, TILE = S::TILE;
    constexpr float kCentre = BITS == 8 ? 128.0f : 8.0f;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    const uint32_t base = ((uint32_t)__cvta_generic_to_shared(smem_raw) + 1023u) & ~1023u;      // the swizzle goes by the address
    uint8_t* smem = smem_raw + (base - (uint32_t)__cvta_generic_to_shared(smem_raw));
    TilesMeta& meta = *reinterpret_cast<TilesMeta*>(smem + S::OFF_META);
    const uint32_t bars = base + S::OFF_META;
    const int tid = threadIdx.x, warp = tid / kWarp, lane = tid % kWarp;
    // barriers of tile i: buffer i % 2, phase i / 2 % 2
    auto k_full = [&](uint32_t i) { return bars + (i & 1) * 8; };
    auto v_full = [&](uint32_t i) { return bars + 16 + (i & 1) * 8; };
    auto k_free = [&](uint32_t i) { return bars + 32 + (i & 1) * 8; };      // S_i is there
    auto v_free = [&](uint32_t i) { return bars + 48 + (i & 1) * 8; };      // O holds tile i
    auto s_free = [&](uint32_t i) { return bars + 64 + (i & 1) * 8; };      // S_i and what is told about tile i have been read
    auto p_full = [&](uint32_t i) { return bars + 80 + (i & 1) * 8; };
    const uint32_t q_full = bars + 96, all_done = bars + 104;
    volatile uint32_t* dead = &meta.dead;
    auto wait_lane = [&](uint32_t bar, uint32_t phase) -> bool {
        for (uint32_t round = 0; round < kMbarSpinLimit / 1024; ++round) {
            for (uint32_t i = 0; i < 1024; ++i) {
                uint32_t ok;
                asm volatile("{ .reg .pred p; mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2; selp.u32 %0, 1, 0, p; }" : "=r"(ok) : "r"(bar), "r"(phase) : "memory");
                if (ok) return true;
            }
            if (*dead) return false;
        }
        *dead = 1;
        *a.error = kErrAttentionWait;
        return false;
    };
    // of a whole warp
    auto wait = [&](uint32_t bar, uint32_t phase) -> bool { return __all_sync(kFullMask, wait_lane(bar, phase)); };
    auto phase = [](uint32_t i) { return (i >> 1) & 1u; };
    auto phase_before = [](uint32_t i) { return ((i >> 1) & 1u) ^ 1u; };    // of the buffer's use by tile i - 2

    if (tid == 0) {
        for (uint32_t i = 0; i < 2; ++i) {
            mbar_init(k_full(i), S::UNPACK_WARPS);
            mbar_init(v_full(i), S::UNPACK_WARPS);
            mbar_init(k_free(i), 1);
            mbar_init(v_free(i), 1);
            mbar_init(s_free(i), S::SOFT_WARPS);
            mbar_init(p_full(i), S::SOFT_WARPS);
        }
        mbar_init(q_full, S::SOFT_WARPS);
        mbar_init(all_done, 1);
        meta.dead = 0;
        a.info[blockIdx.x].active = 0;
        fence_proxy_async();
    }
    if (warp == S::WARPS - 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"((uint32_t)__cvta_generic_to_shared(&meta.tmem)), "r"((uint32_t)S::COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    Cursor<MT, TILE> now;
    Shares shares;
    uint64_t item = 0, stop = 0;
    const bool busy = find_share<MT, TILE>(a, blockIdx.x, gridDim.x, lane, blockIdx.x == 0, now, shares, item, stop);
    tiles_fence_before();
    __syncthreads();
    tiles_fence_after();
    const uint32_t tmem = meta.tmem, count = busy ? (uint32_t)(stop - item) : 0;

    if (warp >= S::SOFT_WARPS && warp < S::WARPS - 1) {
        // ===================== unpacking =====================
        const uint32_t u = tid - S::SOFT_WARPS * kWarp, uw = u / kWarp;
        uint32_t kr[S::K_EACH][BITS / 2], vr[S::V_EACH][BITS / 2];
        uint16_t ks[S::K_EACH], kb[S::K_EACH], vs[S::V_EACH], vb[S::V_EACH];
        uint32_t runs = 0;
        Cursor<MT, TILE> next = now;
        // rows of tile `next`, which the pieces of this thread belong to; a piece without one is zeros
        auto row_of = [&](uint32_t key, bool& there) -> size_t {
            const uint32_t token = next.token0() + key;
            int32_t page = -1;
            if (token < next.range.end) {
                page = a.table.table[(size_t)next.b * a.table.stride + (token >> a.table.page_log2)];
                if (page >= 0 && (uint32_t)page >= a.table.pages) page = -1;
            }
            there = page >= 0;
            return there ? (((size_t)page * a.kv_heads + next.head / S::PARTS) << a.table.page_log2) + (token & ((1u << a.table.page_log2) - 1u)) : 0;
        };
        auto load_piece = [&](uint32_t (&r)[BITS / 2], uint16_t& s, uint16_t& b, const KvPlanes& p, uint32_t key, uint32_t piece) {
            bool there;
            const size_t row = row_of(key, there);
#pragma unroll
            for (int j = 0; j < BITS / 2; ++j) r[j] = 0;
            s = b = 0;
            if (there) {
                load_words(r, p.codes + row * S::ROW_BYTES + piece * S::PIECE);
                s = p.scales[row * S::G + piece / 4];
                b = p.biases[row * S::G + piece / 4];
            }
        };
        auto load_k = [&] {
#pragma unroll
            for (int j = 0; j < S::K_EACH; ++j) load_piece(kr[j], ks[j], kb[j], a.k, (u + j * S::UNPACK) / S::K_ROW, u % S::K_ROW);
        };
        auto load_v = [&] {
#pragma unroll
            for (int j = 0; j < S::V_EACH; ++j)
                load_piece(vr[j], vs[j], vb[j], a.v, (u + j * S::UNPACK) / S::V_ROW, u % S::V_ROW + next.head % S::PARTS * S::V_ROW);
            bool there = false;
            if (lane < S::RUNS) row_of(lane * 16, there);
            runs = __ballot_sync(kFullMask, there);
        };
        if (count) { load_k(); load_v(); }
        int e_v = -126;
        uint32_t segment = busy ? (uint32_t)lesser((uint64_t)(now.range.tiles - now.tile), stop - item) : 0;      // tiles left of the unit at hand
        for (uint32_t i = 0; i < count; ++i) {
            const uint32_t st = i & 1;
            // A wait that runs out is told to all, whose later waits end at once: every warp goes through all tiles, since they meet at a barrier in each.
            if (i >= 2 && wait(k_free(i), phase_before(i))) wait(s_free(i), phase_before(i));
            // ---- the planes' largest magnitudes ----
            float most_k = 0.0f, most_v = 0.0f;
            uint32_t broken = 0;
            auto measure = [&](uint16_t s16, uint16_t b16, float& most) -> bool {
                const float s = bf16_bits_to_float(s16), b = fmaf(kCentre, s, bf16_bits_to_float(b16)), mag = fmaxf(kCentre * fabsf(s), fabsf(b));
                const bool fine = s - s == 0.0f && b - b == 0.0f;
                if (fine) most = fmaxf(most, mag);
                return fine;
            };
#pragma unroll
            for (int j = 0; j < S::K_EACH; ++j) measure(ks[j], kb[j], most_k);
#pragma unroll
            for (int j = 0; j < S::V_EACH; ++j)
                if (!measure(vs[j], vb[j], most_v)) broken |= 1u << j;
            most_k = __uint_as_float(__reduce_max_sync(kFullMask, __float_as_uint(most_k)));
            most_v = __uint_as_float(__reduce_max_sync(kFullMask, __float_as_uint(most_v)));
            if (lane == 0) {
                meta.largest[st][0][uw] = most_k;
                meta.largest[st][1][uw] = most_v;
            }
            if (uw == 0) {
                if (lane < 16) meta.bad[st][lane / 4][lane % 4] = 0;
                if (lane == 0) {
                    meta.any_bad[st] = 0;
                    meta.runs[st] = runs;
                }
            }
            asm volatile("bar.sync 1, %0;" ::"n"(S::UNPACK) : "memory");
            float top_k = 0.0f, top_v = 0.0f;
#pragma unroll
            for (int w = 0; w < 8; ++w) {
                top_k = fmaxf(top_k, meta.largest[st][0][w]);
                top_v = fmaxf(top_v, meta.largest[st][1][w]);
            }
            const int e_k = min(max(rows_exponent(top_k) - 7, -126), 119);           // both parts of a value below 2^8
            e_v = min(max(e_v, rows_exponent(top_v) - 7), 119);
            if (u == 0) {
                meta.e_k[st] = e_k;
                meta.e_v[st] = e_v;
            }
            if (broken) {
#pragma unroll
                for (int j = 0; j < S::V_EACH; ++j)
                    if (broken >> j & 1u) {
                        const uint32_t key = (u + j * S::UNPACK) / S::V_ROW;
                        atomicOr(&meta.bad[st][u % S::V_ROW / 4][key / 32], 1u << (key % 32));
                        meta.any_bad[st] = 1;
                        vs[j] = vb[j] = 0;
                    }
            }
            // ---- K ----
            auto store = [&](uint32_t buffer, const uint32_t (&r)[BITS / 2], uint16_t s16, uint16_t b16, float down, uint32_t key, uint32_t piece) {
                const float s = bf16_bits_to_float(s16);
                uint4 h[2];
                tiles_unpack<BITS>(r, s * down, fmaf(kCentre, s, bf16_bits_to_float(b16)) * down, h);
                // the two chunks in the order in which eight lanes meet eight different banks
                const uint32_t odd = S::K_ROW >= 8 ? piece / 4 & 1u : 0u, at = buffer + key * 128 + (piece / 4) * (TILE * 128);
                const uint4 first = odd ? h[1] : h[0], second = odd ? h[0] : h[1];
                const uint32_t c0 = (piece % 4 * 2 + odd) ^ (key & 7u);
                *reinterpret_cast<uint4*>(smem + at + c0 * 16) = first;
                *reinterpret_cast<uint4*>(smem + at + (c0 ^ 1u) * 16) = second;
            };
            const float down_k = rows_power(-e_k), down_v = rows_power(-e_v);
#pragma unroll
            for (int j = 0; j < S::K_EACH; ++j)
                store(S::OFF_K + st * S::K_BYTES, kr[j], ks[j], kb[j], down_k, (u + j * S::UNPACK) / S::K_ROW, u % S::K_ROW);
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(k_full(i));
            const bool more = i + 1 < count;
            if (more) {
                if (--segment == 0) {
                    next.next_unit(a);
                    segment = (uint32_t)lesser((uint64_t)next.range.tiles, (uint64_t)(count - i - 1));
                } else {
                    ++next.tile;
                }
                load_k();
            }
            // ---- V ----
            if (i >= 2) wait(v_free(i), phase_before(i));
#pragma unroll
            for (int j = 0; j < S::V_EACH; ++j)
                store(S::OFF_V + st * S::V_BYTES, vr[j], vs[j], vb[j], down_v, (u + j * S::UNPACK) / S::V_ROW, u % S::V_ROW);
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(v_full(i));
            if (more) load_v();
        }
    } else if (warp == S::WARPS - 1) {
        // ===================== MMA issuer =====================
        constexpr uint32_t idesc_s = (1u << 4) | ((uint32_t)(TILE >> 3) << 17) | ((uint32_t)(MT >> 4) << 24);
        constexpr uint32_t idesc_o = (1u << 4) | (1u << 16) | ((uint32_t)(S::DV >> 3) << 17) | ((uint32_t)(MT >> 4) << 24);      // B: MN-major
        uint32_t segment = 0, segments = 0;
        bool opens = false;                                    // tile i - 1 is its unit's first here: its product starts O anew
        auto logits = [&](uint32_t i) -> bool {
            if (!wait(k_full(i), phase(i)) || (i >= 2 && !wait(s_free(i), phase_before(i)))) return false;
            tiles_fence_after();
            if (lane == 0) {
                const uint64_t q0 = tiles_desc(base, 16, 1024), k0 = tiles_desc(base + S::OFF_K + (i & 1) * S::K_BYTES, 16, 1024);
#pragma unroll
                for (int e = 0; e < D / 16; ++e)
                    tiles_mma_ss(tmem + S::COL_S + (i & 1) * TILE, q0 + (((e / 4) * (MT * 128) + e % 4 * 32) >> 4), k0 + (((e / 4) * (TILE * 128) + e % 4 * 32) >> 4),
                                 idesc_s, e > 0);
                tiles_commit(k_free(i));
            }
            __syncwarp();
            return true;
        };
        auto values = [&](uint32_t j) -> bool {
            if (!wait(p_full(j), phase(j)) || !wait(v_full(j), phase(j))) return false;
            tiles_fence_after();
            if (lane == 0) {
                const uint64_t v0 = tiles_desc(base + S::OFF_V + (j & 1) * S::V_BYTES, TILE * 128, 1024);
#pragma unroll
                for (int e = 0; e < TILE / 16; ++e)
                    tiles_mma_ts(tmem + S::COL_O, tmem + S::COL_P + (j & 1) * (TILE / 2) + e * 8, v0 + (e * 2048 >> 4), idesc_o, e > 0 || !opens);
                tiles_commit(v_free(j));
            }
            __syncwarp();
            return true;
        };
        for (uint32_t i = 0; i <= count; ++i) {
            // Within a unit the logits of tile i go ahead of the values of tile i - 1; at a unit's end the softmax waits for those values before it
            // lays out the next rows of q.
            const bool new_unit = i < count && segment == 0;
            if (new_unit || i == count) {
                if (i > 0 && !values(i - 1)) break;
                if (i == count) break;
                if (i) now.next_unit(a);
                segment = (uint32_t)lesser((uint64_t)(now.range.tiles - now.tile), (uint64_t)(count - i));
                if (!wait(q_full, segments++ & 1u) || !logits(i)) break;
            } else if (!logits(i) || !values(i - 1)) {
                break;
            }
            opens = new_unit;
            --segment;
        }
        // nothing is in flight when the block leaves
        if (lane == 0) tiles_commit(all_done);
        __syncwarp();
        for (uint32_t i = 0; i < kMbarSpinLimit; ++i) {
            uint32_t ok;
            asm volatile("{ .reg .pred p; mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2; selp.u32 %0, 1, 0, p; }" : "=r"(ok) : "r"(all_done), "r"(0u) : "memory");
            if (ok) break;
        }
    } else {
        // ===================== softmax: a thread per row =====================
        const uint32_t r = tid, lanes = tmem + ((uint32_t)warp * 32u << 16);
        uint32_t i = 0;
        bool ok = true;
        while (ok && i < count) {
            // ---- the unit's rows of q: fp16 in the operand's layout, brought to one range by a power of two ----
            const uint32_t valid = lesser((uint32_t)MT, now.flat_rows(a) - now.flat0), first_tile = now.tile;
            const uint32_t segment = (uint32_t)lesser((uint64_t)(now.range.tiles - first_tile), (uint64_t)(count - i));
            const bool is = r < valid, from_start = first_tile == 0, whole = from_start && segment == now.range.tiles;
            const uint32_t flat = now.flat0 + (is ? r : 0), node = flat / a.group, head = now.head / S::PARTS;
            const uint16_t* src = a.q + (size_t)(now.seq.row0 + node) * a.q_stride + (size_t)(head * a.group + flat % a.group) * D;
            uint32_t most = 0;
            if (is)
#pragma unroll 4
                for (int c = 0; c < D / 8; ++c) {
                    const uint4 v = reinterpret_cast<const uint4*>(src)[c];
                    most = __vmaxu2(__vmaxu2(__vmaxu2(most, v.x & 0x7FFF7FFFu), __vmaxu2(v.y & 0x7FFF7FFFu, v.z & 0x7FFF7FFFu)), v.w & 0x7FFF7FFFu);
                }
            most = max(most & 0xFFFFu, most >> 16);
            const float q_top = BF16 ? bf16_bits_to_float((uint16_t)most) : f16_bits_to_float((uint16_t)most);
            const int e_q = q_top > 0.0f && q_top <= 3.402823466e38f ? max(rows_exponent(q_top), -126) : 0;      // the largest element to [1, 2)
            const float down = rows_power(-e_q), factor = rows_power(e_q) * a.scale * 1.4426950408889634f;
#pragma unroll 2
            for (int c = 0; c < D / 8; ++c) {
                const uint4 v = is ? reinterpret_cast<const uint4*>(src)[c] : make_uint4(0, 0, 0, 0);
                const uint32_t w[4] = {v.x, v.y, v.z, v.w};
                uint32_t h[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float lo = BF16 ? __uint_as_float(w[j] << 16) : f16_bits_to_float((uint16_t)w[j]);
                    const float hi = BF16 ? __uint_as_float(w[j] & 0xFFFF0000u) : f16_bits_to_float((uint16_t)(w[j] >> 16));
                    h[j] = rows_half2(lo * down, hi * down);
                }
                const uint4 out = BITS == 8 ? make_uint4(h[0], h[1], h[2], h[3])
                                            : make_uint4(gm_prmt(h[0], h[2], 0x5410), gm_prmt(h[0], h[2], 0x7632), gm_prmt(h[1], h[3], 0x5410), gm_prmt(h[1], h[3], 0x7632));
                *reinterpret_cast<uint4*>(smem + S::chunk_at(MT, r, c)) = out;
            }
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(q_full);
            uint32_t low = 0;                                  // first token that the row sees
            if (a.window && is) {
                const int64_t pos = a.mask ? max((int64_t)a.positions[now.seq.row0 + node], (int64_t)now.seq.context) : (int64_t)now.seq.context + node;
                low = (uint32_t)max((int64_t)0, lesser(pos - (int64_t)a.window + 1, (int64_t)kMostTokens));
            }
            const uint32_t low_most = __reduce_max_sync(kFullMask, low), open_end = lesser(now.seq.context, now.range.end);
            float m = -INFINITY, l = 0.0f;
            int e_o = -126;                                    // exponent of what O holds
            uint32_t poison = 0;                               // groups that are not a number
            const uint32_t stop_i = i + segment;
            uint32_t token0 = now.token0();
            for (; i < stop_i; ++i, token0 += TILE) {
                const uint32_t st = i & 1;
                ok = wait(k_free(i), phase(i)) && wait(k_full(i), phase(i));         // S_i; what is told about the tile
                if (!ok) break;
                tiles_fence_after();
                const int e_k = meta.e_k[st], e_v = meta.e_v[st];
                const uint32_t runs = meta.runs[st], any_bad = meta.any_bad[st];
                const float f = factor * rows_power(e_k);
                // ---- what the row sees ----
                const bool open = runs == (1u << S::RUNS) - 1u && token0 >= low_most && token0 + TILE <= open_end;
                uint32_t seen[TILE / 32];
#pragma unroll
                for (int w = 0; w < TILE / 32; ++w) seen[w] = 0xFFFFFFFFu;
                if (!open) {
#pragma unroll
                    for (int w = 0; w < TILE / 32; ++w) {
                        const uint32_t t0 = token0 + 32 * w;
                        auto below = [&](uint32_t end) { return end <= t0 ? 0u : end - t0 >= 32 ? 0xFFFFFFFFu : (1u << (end - t0)) - 1u; };      // tokens before `end`
                        uint32_t see = below(open_end) & ~below(low);
                        const uint32_t drafted = below(now.range.end) & ~below(now.seq.context);
                        if (drafted) {
                            const uint32_t shift = t0 < now.seq.context ? now.seq.context - t0 : 0, j = t0 + shift - now.seq.context;      // row j at bit `shift`
                            if (a.mask) {
                                const unsigned long long* bits = a.mask + (size_t)(now.seq.row0 + node) * a.mask_words;
                                const uint32_t word = j >> 6, off = j & 63u;
                                unsigned long long b = word < a.mask_words ? bits[word] >> off : 0ull;
                                if (off && word + 1 < a.mask_words) b |= bits[word + 1] << (64 - off);
                                see |= (uint32_t)b << shift & drafted;
                            } else {
                                uint32_t chain = below(now.seq.context + node + 1);
                                if (a.window && node + 1 > a.window) chain &= ~below(now.seq.context + node + 1 - a.window);
                                see |= chain & drafted;
                            }
                        }
                        if (!(runs >> (2 * w) & 1u)) see &= 0xFFFF0000u;
                        if (!(runs >> (2 * w + 1) & 1u)) see &= 0x0000FFFFu;
                        seen[w] = is ? see : 0u;
                    }
                    if (tid == 0) {
                        const uint32_t held = token0 >= now.range.end ? 0u : lesser((now.range.end - token0 + 15) / 16, (uint32_t)S::RUNS);
                        if (runs != (1u << held) - 1u) *a.error = kErrKvPage;
                    }
                }
                // the logits of 32 tokens, in base 2
                auto load_logits = [&](int w, float (&x)[32]) {
                    uint32_t raw[32];
                    tiles_ld32(lanes + S::COL_S + st * TILE + w * 32, raw);
                    tiles_wait_ld();
#pragma unroll
                    for (int j = 0; j < 32; ++j) x[j] = __uint_as_float(raw[j]) * f;
                    if (!open) {
#pragma unroll
                        for (int j = 0; j < 32; ++j) x[j] = seen[w] >> j & 1u ? x[j] : -INFINITY;
                    }
                };
                // ---- maximum ----
                float top = -INFINITY;
#pragma unroll
                for (int w = 0; w < TILE / 32; ++w) {
                    float x[32];
                    load_logits(w, x);
#pragma unroll
                    for (int j = 0; j < 32; ++j) top = fmaxf(top, x[j]);
                }
                float alpha = 1.0f;
                if (top > m + 8.0f) {
                    alpha = rows_exp2(m - top);                // m = -inf: zero
                    m = top;
                }
                l *= alpha;
                alpha *= rows_power(e_o - e_v);
                e_o = e_v;
                const float shift = m == -INFINITY ? 0.0f : m;
                // ---- O, when a maximum or the exponent moved ----
                if (i > stop_i - segment && __any_sync(kFullMask, alpha != 1.0f)) {
                    ok = wait(v_free(i - 1), phase(i - 1));
                    if (!ok) break;
                    tiles_fence_after();
#pragma unroll 1
                    for (int c = 0; c < S::DV; c += 32) {
                        uint32_t o[32];
                        tiles_ld32(lanes + S::COL_O + c, o);
                        tiles_wait_ld();
#pragma unroll
                        for (int j = 0; j < 32; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * alpha);
                        tiles_st32(lanes + S::COL_O + c, o);
                    }
                    tiles_wait_st();
                }
                // ---- probabilities, at most 2^8, two to a column ----
                if (i >= 2) {
                    ok = wait(v_free(i), phase_before(i));     // P's buffer has been read
                    if (!ok) break;
                }
                float sum = 0.0f;
#pragma unroll
                for (int w = 0; w < TILE / 32; ++w) {
                    float x[32];
                    uint32_t p[16];
                    load_logits(w, x);
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        const float p0 = rows_exp2(x[2 * j] - shift), p1 = rows_exp2(x[2 * j + 1] - shift);
                        sum += p0 + p1;
                        p[j] = rows_half2(p0, p1);
                    }
                    tiles_st16(lanes + S::COL_P + st * (TILE / 2) + w * 16, p);
                    if (any_bad) {
                        // a row that gives a token weight whose planes are not finite in a group becomes NaN there
                        uint32_t live = 0;
#pragma unroll
                        for (int j = 0; j < 16; ++j) live |= (p[j] & 0x7FFFu ? 1u : 0u) << (2 * j) | (p[j] & 0x7FFF0000u ? 2u : 0u) << (2 * j);
#pragma unroll
                        for (int g = 0; g < S::GV; ++g) poison |= live & meta.bad[st][g][w] ? 1u << g : 0u;
                    }
                }
                l += sum;
                tiles_wait_st();
                tiles_fence_before();
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(s_free(i));
                    mbar_arrive(p_full(i));
                }
            }
            if (!ok) break;
            // ---- the segment's result ----
            if (!wait(v_free(i - 1), phase(i - 1))) break;
            tiles_fence_after();
            float* part = a.partial + (size_t)(2 * blockIdx.x + (from_start ? 1 : 0)) * MT * (S::DV + 2);
            if (!whole && is) {
                part[r] = m;
                part[MT + r] = l;
            }
            const float up = rows_power(e_o), inv = whole ? (l == 0.0f ? 0.0f : 1.0f / l) * up : up;
            uint16_t* dst = a.out + (size_t)(now.seq.row0 + node) * a.out_stride + (size_t)(head * a.group + flat % a.group) * D + now.head % S::PARTS * S::DV;
            float* pdst = part + 2 * MT + (size_t)r * S::DV;
#pragma unroll 1
            for (int c = 0; c < S::DV; c += 32) {
                uint32_t o[32];
                tiles_ld32(lanes + S::COL_O + c, o);
                tiles_wait_ld();
                const float by = poison >> (c / 64) & 1u ? __int_as_float(0x7FC00000) : inv;
                if (is) {
#pragma unroll
                    for (int e = 0; e < 32; e += 8) {
                        float v[8];
#pragma unroll
                        for (int j = 0; j < 8; ++j) v[BITS == 8 ? j : (j / 2) + (j % 2) * 4] = __uint_as_float(o[e + j]) * by;
                        if (whole) {
                            *reinterpret_cast<uint4*>(dst + c + e) = make_uint4(rows_pair<BF16>(v[0], v[1]), rows_pair<BF16>(v[2], v[3]), rows_pair<BF16>(v[4], v[5]),
                                                                                rows_pair<BF16>(v[6], v[7]));
                        } else {
                            *reinterpret_cast<float4*>(pdst + c + e) = make_float4(v[0], v[1], v[2], v[3]);
                            *reinterpret_cast<float4*>(pdst + c + e + 4) = make_float4(v[4], v[5], v[6], v[7]);
                        }
                    }
                }
            }
            tiles_fence_before();
            if (!whole && from_start && tid == 0) {
                ShareInfo& info = a.info[blockIdx.x];
                info.last = shares.of(item + stop_i - 1 + (now.range.tiles - segment));
                info.row0 = now.seq.row0;
                info.flat0 = now.flat0;
                info.valid = valid;
                info.head = now.head;
                info.active = 1;
            }
            if (i < count) now.next_unit(a);
        }
    }
    tiles_fence_before();
    __syncthreads();
    if (warp == S::WARPS - 1) {
        tiles_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"((uint32_t)S::COLS) : "memory");
    }
}

// Joins the shares of the unit that block c's share ends in: a warp per row, lanes over the elements.
constexpr int kTilesJoinThreads = 128;
template <int D, int DV, bool BF16>
__global__ void __launch_bounds__(kTilesJoinThreads)
attention_tiles_join_kernel(const AttnArgs a) {
    constexpr int VEC = DV / 32, MT = 128, PARTS = D / DV;
    pdl_wait();
    const uint32_t c = blockIdx.x;
    const ShareInfo info = a.info[c];
    const uint32_t warp = threadIdx.x / kWarp, lane = threadIdx.x % kWarp, r = blockIdx.y * (kTilesJoinThreads / kWarp) + warp;
    if (!info.active || r >= info.valid) return;
    const uint32_t parts = info.last - c + 1;
    constexpr size_t kSlot = (size_t)MT * (DV + 2);
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
            w = rows_exp2(s[r] - base);
            l = s[MT + r];
        }
        const uint32_t n = min(parts - p0, (uint32_t)kWarp);
#pragma unroll 4
        for (uint32_t j = 0; j < n; ++j) {
            const float wj = __shfl_sync(kFullMask, w, j), lj = __shfl_sync(kFullMask, l, j);
            const float* src = slot(p0 + j) + 2 * MT + (size_t)r * DV + lane * VEC;
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
    uint16_t* dst = a.out + (size_t)(info.row0 + flat / a.group) * a.out_stride + (size_t)(info.head / PARTS * a.group + flat % a.group) * D + info.head % PARTS * DV + lane * VEC;
#pragma unroll
    for (int e = 0; e < VEC; e += 2) *reinterpret_cast<uint32_t*>(dst + e) = rows_pair<BF16>(v[e] * inv, v[e + 1] * inv);
}

template <int D, int BITS, bool BF16>
static tf_status launch_tiles(tf_context* ctx, cudaStream_t st, const AttnArgs& args, const tf_attention_workspace* ws) {
    using S = TilesShape<D, BITS>;
    AttnArgs a = args;
    a.head_parts = S::PARTS;
    auto kernel = attention_tiles_kernel<D, BITS, BF16>;
    static DeviceSmemCache smem_cache;
    const tf_status s = ensure_dynamic_smem(ctx, kernel, smem_cache, S::SMEM);
    if (s != TF_OK) return s;
    const uint32_t blocks = lesser((uint32_t)ctx->sm_count, ws->row_capacity / S::MT);
    kernel<<<blocks, S::THREADS, S::SMEM, st>>>(a);
    const tf_status t = check_launch(ctx, "tf_tree_attention");
    if (t != TF_OK) return t;
    TF_CUDA(ctx, launch_pdl(attention_tiles_join_kernel<D, S::DV, BF16>, dim3(blocks, S::MT / (kTilesJoinThreads / kWarp)), dim3(kTilesJoinThreads), 0, st, a));
    return check_launch(ctx, "tf_tree_attention (join)");
}

template <int D, int BITS>
tf_status attend(tf_context* ctx, cudaStream_t st, const AttnArgs& a, const tf_attention_workspace* ws, bool bf16) {
    // Rows of one kv head in a mean sequence. Units of eight rows read the cache once each, units of 128 once for all.
    const uint64_t mean = ((uint64_t)a.rows + a.sequences - 1) / a.sequences * a.group;
    if (mean <= 32) return bf16 ? launch_rows<D, BITS, 8, true>(ctx, st, a, ws) : launch_rows<D, BITS, 8, false>(ctx, st, a, ws);
    return bf16 ? launch_tiles<D, BITS, true>(ctx, st, a, ws) : launch_tiles<D, BITS, false>(ctx, st, a, ws);
}

}  // namespace tf
