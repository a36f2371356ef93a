// Attention over the quantised, paged cache for units of up to 128 rows (trees and chains): tcgen05 with tensor-memory accumulators.
//
// With this many rows the products bound it, 4 * 128 * D FLOP per token and unit, next to the unpacking, which a unit pays once for its 128 rows.
// One persistent block per SM; 8 warps unpack, one issues the MMAs, 4 do the softmax, a thread per row. For tile i of TILE tokens:
//   unpack:  codes and planes, by cp.async a tile ahead into places of the thread's own -> K_i, V_i in fp16, [64 elements][token][128 bytes] with the
//            128-byte swizzle (K in one buffer: it is free again when its logits are there, long before the next ones are wanted)
//   MMA:     S_i = Q K_i^T into tensor memory (two buffers), then O += P_(i-1) V_(i-1); K is K-major, V, as it lies, MN-major
//   softmax: S_i -> registers -> mask, 2^(x - m), P_i as fp16 into tensor memory (the A operand of the second product)
// The loops are rolled where registers allow it: three kinds of warps share an SM's instruction caches, and straight-line code of all of them
// waited for instructions most of the time (9600 clocks a tile instead of what the notes of the measurements give).
// K_i and V_i carry (code - centre) s + (bias + centre s) rounded to fp16, 2^-11 of the value: logits see it as an error of about 2^-12 |q||k| / sqrt(D),
// of the size of the output's own rounding to 16 bits. A token's values are divided by a power of two of its own first; K's comes back with the
// logits, V's into the probabilities, p' = 2^(x - m - E) * 2^e, where E is a row's own and follows the largest p' so far: tokens that a row
// does not see have no say, and no cache leaves fp16's range. m is raised only when a logit exceeds it by 8, and what O holds is
// rescaled only when m or E moves. TILE * D is 16384 but for heads of 64; heads of 512, whose product would fill tensor memory alone,
// are two units with half of the values each.
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
    static constexpr int V_BUFS = D == 512 ? 1 : 2;
    static constexpr bool SAME = K_ROW == V_ROW;                              // a thread's pieces of K and V are of the same tokens
    static constexpr int Q_BYTES = MT * D * 2, K_BYTES = TILE * D * 2, V_BYTES = TILE * DV * 2;
    static constexpr int OFF_K = Q_BYTES, OFF_V = OFF_K + K_BYTES;
    // what the unpacking threads have requested, [piece][thread]: codes; (scale, bias) words, of V for two tiles; pages of the next tiles
    static constexpr int OFF_KC = OFF_V + V_BUFS * V_BYTES, OFF_VC = OFF_KC + K_EACH * UNPACK * PIECE, OFF_KS = OFF_VC + V_EACH * UNPACK * PIECE,
                         OFF_VS = OFF_KS + K_EACH * UNPACK * 8, OFF_KP = OFF_VS + 2 * V_EACH * UNPACK * 8, OFF_VP = SAME ? OFF_KP : OFF_KP + K_EACH * UNPACK * 4,
                         OFF_META = OFF_VP + 2 * V_EACH * UNPACK * 4;
    static constexpr int META = (256 + 2 * TILE * 9 + 127) / 128 * 128, SMEM = OFF_META + META + 1024;
    // tensor memory, in columns
    static constexpr int COL_S = 0, COL_P = 2 * TILE, COL_O = 3 * TILE, COLS = 512;
    static_assert(COL_O + DV <= COLS && SMEM <= 227 * 1024 && K_EACH * UNPACK == TILE * K_ROW && V_EACH * UNPACK == TILE * V_ROW, "sizes");
    // a 16-byte chunk (eight elements) of an operand row: [64 elements][rows][128 bytes], chunks swizzled by the row
    static __host__ __device__ __forceinline__ uint32_t chunk_at(uint32_t rows, uint32_t row, uint32_t chunk) {
        return (chunk >> 3) * (rows * 128) + row * 128 + (((chunk & 7u) ^ (row & 7u)) << 4);
    }
};

// What the unpacking warps tell the softmax about tiles (two of them), and the block's barriers.
template <int TILE>
struct TilesMeta {
    unsigned long long bars[24];
    uint32_t tmem, dead;
    uint8_t flags[2][8];           // per unpacking warp: something in `bad`
    alignas(16) float k_up[2][TILE];           // what a token's logits are multiplied with: its power of two, the scale, log2 e
    alignas(16) float v_up[2][TILE];           // a token's power of two
    uint8_t bad[2][TILE];          // bit g: value planes of group g are not finite; bit 7: the token's page is missing
};

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

__device__ __forceinline__ void tiles_cp_async(uint32_t dst, const void* src, uint32_t bytes, bool there) {      // 16, 8 or 4 bytes; zeros if not there
    const uint32_t n = there ? bytes : 0u;
    if (bytes == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
    else if (bytes == 8) asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}

template <int D, int BITS, bool BF16>
__global__ void __launch_bounds__(TilesShape<D, BITS>::THREADS, 1)
attention_tiles_kernel(const __grid_constant__ AttnArgs a) {
    using S = TilesShape<D, BITS>;
    using Meta = TilesMeta<S::TILE>;
    constexpr int MT = S::MT, TILE = S::TILE;
    constexpr float kCentre = BITS == 8 ? 128.0f : 8.0f;
    static_assert(sizeof(Meta) <= S::META, "meta");
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    const uint32_t base = ((uint32_t)__cvta_generic_to_shared(smem_raw) + 1023u) & ~1023u;      // the swizzle goes by the address
    uint8_t* smem = smem_raw + (base - (uint32_t)__cvta_generic_to_shared(smem_raw));
    Meta& meta = *reinterpret_cast<Meta*>(smem + S::OFF_META);
    const uint32_t bars = base + S::OFF_META;
    const int tid = threadIdx.x, warp = tid / kWarp, lane = tid % kWarp;
    // Barriers of tile i and the phase in which they are done with it, by the number of their buffers.
    auto k_full = [&] { return bars; };
    auto k_free = [&] { return bars + 8; };                                 // K's buffer: the logits of tile i are there
    auto v_full = [&](uint32_t i) { return bars + 16 + (i % S::V_BUFS) * 8; };
    auto v_free = [&](uint32_t i) { return bars + 32 + (i % S::V_BUFS) * 8; };
    auto s_full = [&](uint32_t i) { return bars + 48 + (i & 1) * 8; };
    auto s_free = [&](uint32_t i) { return bars + 64 + (i & 1) * 8; };      // S_i and what is told about tile i have been read
    auto p_full = [&](uint32_t i) { return bars + 80 + (i & 1) * 8; };
    auto o_done = [&](uint32_t i) { return bars + 96 + (i & 1) * 8; };      // O holds tile i, P_i has been read
    auto told = [&](uint32_t i) { return bars + 128 + (i & 1) * 8; };       // as K_i is, for the softmax: K's own barrier may be past it
    const uint32_t q_full = bars + 112, all_done = bars + 120;
    auto one = [](uint32_t i) { return i & 1u; };
    auto two = [](uint32_t i) { return i >> 1 & 1u; };
    auto of_v = [](uint32_t i) { return i / S::V_BUFS & 1u; };
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

    if (tid == 0) {
        mbar_init(k_full(), S::UNPACK_WARPS);
        mbar_init(k_free(), 1);
        for (uint32_t i = 0; i < 2; ++i) {
            mbar_init(bars + 16 + i * 8, S::UNPACK_WARPS);
            mbar_init(bars + 32 + i * 8, 1);
            mbar_init(s_full(i), 1);
            mbar_init(s_free(i), S::SOFT_WARPS);
            mbar_init(p_full(i), S::SOFT_WARPS);
            mbar_init(o_done(i), 1);
            mbar_init(told(i), S::UNPACK_WARPS);
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
        // A thread's piece j of K (V) is sixteen elements of one token; what it requests lies in places that it alone reads, so a wait for its own
        // copies is all it takes. While tile i is unpacked, tile i + 1 is requested, by page numbers that were requested a tile before.
        const uint32_t u = tid - S::SOFT_WARPS * kWarp, uw = u / kWarp;
        const uint32_t k_piece = u % S::K_ROW, v_piece = u % S::V_ROW;
        const uint32_t page_mask = (1u << a.table.page_log2) - 1u;
        struct Tile { uint32_t token0, end, head; const int32_t* table; };
        auto tile_of = [&](const Cursor<MT, TILE>& c) { return Tile{c.token0(), c.range.end, c.head, a.table.table + (size_t)c.b * a.table.stride}; };
        auto k_key = [&](uint32_t j) { return (u + j * S::UNPACK) / S::K_ROW; };
        auto v_key = [&](uint32_t j) { return (u + j * S::UNPACK) / S::V_ROW; };
        // places of page numbers: of V for even and odd tiles, of K the same ones or (heads of 512) one
        auto v_page = [&](uint32_t i, uint32_t j) { return S::OFF_VP + (((i & 1) * S::V_EACH + j) * S::UNPACK + u) * 4; };
        auto k_page = [&](uint32_t i, uint32_t j) { return S::SAME ? v_page(i, j) : S::OFF_KP + (j * S::UNPACK + u) * 4; };
        auto page_at = [&](uint32_t off) { return *reinterpret_cast<const int32_t*>(smem + off); };
        auto ask_page = [&](const Tile& t, uint32_t key, uint32_t off) {
            const uint32_t token = t.token0 + key;
            if (token < t.end) tiles_cp_async(base + off, t.table + (token >> a.table.page_log2), 4, true);
        };
        // the cache's row of a token (a number below 2^32, as the entry point has checked), and whether there is one
        auto row_at = [&](const Tile& t, uint32_t key, int32_t page, bool& there) -> uint32_t {
            const uint32_t token = t.token0 + key;
            there = token < t.end && page >= 0 && (uint32_t)page < a.table.pages;
            return there ? (((uint32_t)page * a.kv_heads + t.head / S::PARTS) << a.table.page_log2) + (token & page_mask) : 0u;
        };
        // the 32-bit word that holds a group's 16-bit scale (bias), and which half of it
        auto ask_planes = [&](const KvPlanes& p, uint32_t row, uint32_t grp, bool there, uint32_t off) {
            const size_t at = ((size_t)row * S::G + grp) & ~(size_t)1;
            tiles_cp_async(base + off, p.scales + at, 4, there);
            tiles_cp_async(base + off + 4, p.biases + at, 4, there);
        };
        const uint32_t k_half = S::G == 1 ? k_key(0) & 1u : k_piece / 4 & 1u, v_half = S::G == 1 ? v_key(0) & 1u : v_piece / 4 & 1u;
        auto read_planes = [&](uint32_t off, uint32_t half, float& s, float& b) {        // the bias centred
            const uint2 w = *reinterpret_cast<const uint2*>(smem + off);
            s = __uint_as_float(half ? w.x & 0xFFFF0000u : w.x << 16);
            b = fmaf(kCentre, s, __uint_as_float(half ? w.y & 0xFFFF0000u : w.y << 16));
        };
        auto ask_k = [&](const Tile& t, uint32_t i, uint32_t j) {
            bool there;
            const uint32_t row = row_at(t, k_key(j), page_at(k_page(i, j)), there);
            tiles_cp_async(base + S::OFF_KC + (j * S::UNPACK + u) * S::PIECE, a.k.codes + (size_t)row * S::ROW_BYTES + k_piece * S::PIECE, S::PIECE, there);
            ask_planes(a.k, row, k_piece / 4, there, S::OFF_KS + (j * S::UNPACK + u) * 8);
        };
        auto ask_v_planes = [&](const Tile& t, uint32_t i, uint32_t j) {
            bool there;
            const uint32_t row = row_at(t, v_key(j), page_at(v_page(i, j)), there);
            ask_planes(a.v, row, v_piece / 4 + t.head % S::PARTS * S::GV, there, S::OFF_VS + (((i & 1) * S::V_EACH + j) * S::UNPACK + u) * 8);
        };
        auto ask_v = [&](const Tile& t, uint32_t i, uint32_t j) {
            bool there;
            const uint32_t row = row_at(t, v_key(j), page_at(v_page(i, j)), there);
            tiles_cp_async(base + S::OFF_VC + (j * S::UNPACK + u) * S::PIECE, a.v.codes + (size_t)row * S::ROW_BYTES + (v_piece + t.head % S::PARTS * S::V_ROW) * S::PIECE, S::PIECE,
                           there);
        };
        auto commit = [] { asm volatile("cp.async.commit_group;" ::: "memory"); };
        auto landed = [] { asm volatile("cp.async.wait_group 1;" ::: "memory"); };
        // the largest of a token's lanes
        auto token_most = [&](float v, int lanes) {
            for (int off = lanes / 2; off >= 1; off >>= 1) v = fmaxf(v, __shfl_xor_sync(kFullMask, v, off));
            return v;
        };
        auto magnitude = [&](float s, float b) { return fmaxf(kCentre * fabsf(s), fabsf(b)); };
        auto exponent = [&](float most) { return min(max(rows_exponent(most) - 7, -126), 119); };      // both parts of a value below 2^8
        auto store = [&](uint32_t buffer, const uint32_t (&r)[BITS / 2], float s, float b, uint32_t key, uint32_t piece) {
            uint4 h[2];
            tiles_unpack<BITS>(r, s, b, h);
            // the two chunks in the order in which eight lanes meet eight different banks
            const uint32_t odd = S::K_ROW >= 8 ? piece / 4 & 1u : 0u, at = buffer + key * 128 + (piece / 4) * (TILE * 128), c0 = (piece % 4 * 2 + odd) ^ (key & 7u);
            *reinterpret_cast<uint4*>(smem + at + c0 * 16) = odd ? h[1] : h[0];
            *reinterpret_cast<uint4*>(smem + at + (c0 ^ 1u) * 16) = odd ? h[0] : h[1];
        };
        Cursor<MT, TILE> next = now;                           // of the tile that pages are asked for
        uint32_t left = busy ? (uint32_t)lesser((uint64_t)(now.range.tiles - now.tile), stop - item) : 0, ahead = 0;
        Tile t0 = {}, t1 = {}, t2 = {};                        // tiles i, i + 1, i + 2
        auto step = [&] {                                      // `next` one tile on, if there is one
            if (++ahead >= count) return;
            if (--left == 0) {
                next.next_unit(a);
                left = (uint32_t)lesser((uint64_t)next.range.tiles, (uint64_t)(count - ahead));
            } else {
                ++next.tile;
            }
        };
        if (count) {
            t0 = t1 = tile_of(next);
            for (int j = 0; j < S::K_EACH; ++j) ask_page(t0, k_key(j), k_page(0, j));
            if (!S::SAME)
                for (int j = 0; j < S::V_EACH; ++j) ask_page(t0, v_key(j), v_page(0, j));
            asm volatile("cp.async.wait_all;" ::: "memory");
            for (int j = 0; j < S::K_EACH; ++j) ask_k(t0, 0, j);
            for (int j = 0; j < S::V_EACH; ++j) ask_v_planes(t0, 0, j);
            step();
            t1 = tile_of(next);
            if (count > 1) {
                for (int j = 0; j < S::K_EACH; ++j) ask_page(t1, k_key(j), k_page(1, j));
                if (!S::SAME)
                    for (int j = 0; j < S::V_EACH; ++j) ask_page(t1, v_key(j), v_page(1, j));
            }
            commit();
            for (int j = 0; j < S::V_EACH; ++j) ask_v(t0, 0, j);
            commit();
            step();
            t2 = tile_of(next);
        }
        // A wait that runs out is told to all, whose later waits end at once; every warp goes through all tiles.
#pragma unroll 1
        for (uint32_t i = 0; i < count; ++i) {
            // ---- K_i, what is told about tile i; K_(i+1) and the planes of V_(i+1) are requested, and the pages of tile i + 2 ----
            landed();
            if (i >= 1) wait(k_free(), one(i - 1));
            if (i >= 2) wait(s_free(i), two(i - 2));
            uint32_t any = 0;
#pragma unroll 1
            for (int j = 0; j < S::V_EACH; ++j) {
                const uint32_t key = v_key(j), token = t0.token0 + key;
                float s, b;
                read_planes(S::OFF_VS + (((i & 1) * S::V_EACH + j) * S::UNPACK + u) * 8, v_half, s, b);
                const bool broken = !(s - s == 0.0f && b - b == 0.0f);
                const float most = token_most(broken ? 0.0f : magnitude(s, b), S::V_ROW);
                const int32_t page = page_at(v_page(i, j));
                const bool missing = token < t0.end && !(page >= 0 && (uint32_t)page < a.table.pages);
                const uint32_t of_token = __ballot_sync(kFullMask, broken) >> (lane / S::V_ROW * S::V_ROW);
                if (v_piece == 0) {
                    uint32_t bits = missing ? 0x80u : 0u;
#pragma unroll
                    for (int g = 0; g < S::GV; ++g) bits |= (of_token >> (4 * g) & 1u) << g;
                    meta.v_up[i & 1][key] = rows_power(exponent(most));
                    meta.bad[i & 1][key] = (uint8_t)bits;
                    any |= bits;
                    if (missing) *a.error = kErrKvPage;
                }
            }
            any = __any_sync(kFullMask, any != 0);
#pragma unroll 1
            for (int j = 0; j < S::K_EACH; ++j) {
                const uint32_t key = k_key(j);
                uint32_t r[BITS / 2];
                load_words(r, smem + S::OFF_KC + (j * S::UNPACK + u) * S::PIECE);
                float s, b;
                read_planes(S::OFF_KS + (j * S::UNPACK + u) * 8, k_half, s, b);
                const bool broken = !(s - s == 0.0f && b - b == 0.0f);
                const int e = exponent(token_most(broken ? 0.0f : magnitude(s, b), S::K_ROW));
                const float down = rows_power(-e);
                if (k_piece == 0) meta.k_up[i & 1][key] = rows_power(e) * (a.scale * 1.4426950408889634f);
                store(S::OFF_K, r, s * down, b * down, key, k_piece);
                if (i + 1 < count) ask_k(t1, i + 1, j);
            }
            if (lane == 0) meta.flags[i & 1][uw] = (uint8_t)any;
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(k_full());
                mbar_arrive(told(i));
            }
            if (i + 1 < count) {
#pragma unroll 1
                for (int j = 0; j < S::V_EACH; ++j) ask_v_planes(t1, i + 1, j);
            }
            if (i + 2 < count) {
                for (int j = 0; j < S::K_EACH; ++j) ask_page(t2, k_key(j), k_page(i + 2, j));
                if (!S::SAME)
                    for (int j = 0; j < S::V_EACH; ++j) ask_page(t2, v_key(j), v_page(i + 2, j));
            }
            commit();
            // ---- V_i; the codes of V_(i+1) are requested ----
            landed();
            if (i >= S::V_BUFS) wait(v_free(i), of_v(i - S::V_BUFS));
#pragma unroll 1
            for (int j = 0; j < S::V_EACH; ++j) {
                const uint32_t key = v_key(j);
                uint32_t r[BITS / 2];
                load_words(r, smem + S::OFF_VC + (j * S::UNPACK + u) * S::PIECE);
                float s, b;
                read_planes(S::OFF_VS + (((i & 1) * S::V_EACH + j) * S::UNPACK + u) * 8, v_half, s, b);
                if (!(s - s == 0.0f && b - b == 0.0f)) s = b = 0.0f;
                const float down = __uint_as_float(0x7F000000u - __float_as_uint(meta.v_up[i & 1][key]));      // the reciprocal of a power of two
                store(S::OFF_V + (i % S::V_BUFS) * S::V_BYTES, r, s * down, b * down, key, v_piece);
                if (i + 1 < count) ask_v(t1, i + 1, j);
            }
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(v_full(i));
            commit();
            t0 = t1;
            t1 = t2;
            step();
            t2 = tile_of(next);
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
    } else if (warp == S::WARPS - 1) {
        // ===================== MMA issuer =====================
        constexpr uint32_t idesc_s = (1u << 4) | ((uint32_t)(TILE >> 3) << 17) | ((uint32_t)(MT >> 4) << 24);
        constexpr uint32_t idesc_o = (1u << 4) | (1u << 16) | ((uint32_t)(S::DV >> 3) << 17) | ((uint32_t)(MT >> 4) << 24);      // B: MN-major
        uint32_t segment = 0, segments = 0;
        bool opens = false;                                    // tile i - 1 is its unit's first here: its product starts O anew
        auto logits = [&](uint32_t i) -> bool {
            if (!wait(k_full(), one(i)) || (i >= 2 && !wait(s_free(i), two(i - 2)))) return false;
            tiles_fence_after();
            if (lane == 0) {
                const uint64_t q0 = tiles_desc(base, 16, 1024), k0 = tiles_desc(base + S::OFF_K, 16, 1024);
#pragma unroll
                for (int e = 0; e < D / 16; ++e)
                    tiles_mma_ss(tmem + S::COL_S + (i & 1) * TILE, q0 + (((e / 4) * (MT * 128) + e % 4 * 32) >> 4), k0 + (((e / 4) * (TILE * 128) + e % 4 * 32) >> 4),
                                 idesc_s, e > 0);
                tiles_commit(s_full(i));
                tiles_commit(k_free());
            }
            __syncwarp();
            return true;
        };
        auto values = [&](uint32_t j) -> bool {
            if (!wait(p_full(j), two(j)) || !wait(v_full(j), of_v(j))) return false;
            tiles_fence_after();
            if (lane == 0) {
                const uint64_t v0 = tiles_desc(base + S::OFF_V + (j % S::V_BUFS) * S::V_BYTES, TILE * 128, 1024);
#pragma unroll
                for (int e = 0; e < TILE / 16; ++e)
                    tiles_mma_ts(tmem + S::COL_O, tmem + S::COL_P + (j & 1) * (TILE / 2) + e * 8, v0 + (e * 2048 >> 4), idesc_o, e > 0 || !opens);
                tiles_commit(o_done(j));
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
            const float down = rows_power(-e_q), q_up = rows_power(e_q);
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
            float m = -INFINITY, l = 0.0f;                     // l and O: in units of 2^(m + E)
            int e_o = -126;
            uint32_t poison = 0;                               // groups that are not a number
            const uint32_t begin_i = i, stop_i = i + segment;
            uint32_t token0 = now.token0();
#pragma unroll 1
            for (; i < stop_i; ++i, token0 += TILE) {
                const uint32_t st = i & 1;
                ok = wait(s_full(i), two(i)) && wait(told(i), two(i));
                if (!ok) break;
                tiles_fence_after();
                const uint2 flags = *reinterpret_cast<const uint2*>(meta.flags[st]);
                const bool odd = (flags.x | flags.y) != 0;
                const bool open = !odd && token0 >= low_most && token0 + TILE <= open_end;
                // the tokens of chunk w that the row sees
                auto see = [&](int w) -> uint32_t {
                    const uint32_t t0 = token0 + 32 * w;
                    auto below = [&](uint32_t end) { return end <= t0 ? 0u : end - t0 >= 32 ? 0xFFFFFFFFu : (1u << (end - t0)) - 1u; };      // tokens before `end`
                    uint32_t seen = below(open_end) & ~below(low);
                    const uint32_t drafted = below(now.range.end) & ~below(now.seq.context);
                    if (drafted) {
                        const uint32_t shift = t0 < now.seq.context ? now.seq.context - t0 : 0, j = t0 + shift - now.seq.context;      // row j at bit `shift`
                        if (a.mask) {
                            const unsigned long long* bits = a.mask + (size_t)(now.seq.row0 + node) * a.mask_words;
                            const uint32_t word = j >> 6, off = j & 63u;
                            unsigned long long b = word < a.mask_words ? bits[word] >> off : 0ull;
                            if (off && word + 1 < a.mask_words) b |= bits[word + 1] << (64 - off);
                            seen |= (uint32_t)b << shift & drafted;
                        } else {
                            uint32_t chain = below(now.seq.context + node + 1);
                            if (a.window && node + 1 > a.window) chain &= ~below(now.seq.context + node + 1 - a.window);
                            seen |= chain & drafted;
                        }
                    }
                    if (odd)
                        for (int j = 0; j < 32; ++j)
                            if (meta.bad[st][32 * w + j] & 0x80u) seen &= ~(1u << j);
                    return is ? seen : 0u;
                };
                // the logits of 32 tokens, in base 2 but for the row's power of two
                auto load_logits = [&](int w, float (&x)[32]) {
                    uint32_t raw[32];
                    tiles_ld32(lanes + S::COL_S + st * TILE + w * 32, raw);
                    tiles_wait_ld();
#pragma unroll
                    for (int j = 0; j < 32; j += 4) {
                        const float4 up = *reinterpret_cast<const float4*>(&meta.k_up[st][32 * w + j]);
                        x[j] = __uint_as_float(raw[j]) * up.x;
                        x[j + 1] = __uint_as_float(raw[j + 1]) * up.y;
                        x[j + 2] = __uint_as_float(raw[j + 2]) * up.z;
                        x[j + 3] = __uint_as_float(raw[j + 3]) * up.w;
                    }
                    if (!open) {
                        const uint32_t seen = see(w);
#pragma unroll
                        for (int j = 0; j < 32; ++j) x[j] = seen >> j & 1u ? x[j] : -INFINITY;
                    }
                };
                // ---- maximum ----
                float top = -INFINITY;
#pragma unroll 1
                for (int w = 0; w < TILE / 32; ++w) {
                    float x[32];
                    load_logits(w, x);
#pragma unroll
                    for (int j = 0; j < 32; ++j) top = fmaxf(top, x[j]);
                }
                top *= q_up;
                float alpha = 1.0f;
                if (top > m + 8.0f) {
                    alpha = rows_exp2(m - top);                // m = -inf: zero
                    m = top;
                }
                // ---- probabilities, two to a column ----
                if (i >= 2) {
                    ok = wait(o_done(i), two(i - 2));          // P's buffer has been read
                    if (!ok) break;
                }
                float sum;
                for (int round = 0;; ++round) {
                    const float shift = (m == -INFINITY ? 0.0f : m) + (float)e_o;
                    float heavy = 0.0f;
                    sum = 0.0f;
#pragma unroll 1
                    for (int w = 0; w < TILE / 32; ++w) {
                        float x[32];
                        uint32_t p[16];
                        load_logits(w, x);
#pragma unroll
                        for (int j = 0; j < 32; j += 4) {
                            const float4 up = *reinterpret_cast<const float4*>(&meta.v_up[st][32 * w + j]);
                            const float p0 = rows_exp2(fmaf(x[j], q_up, -shift)), p1 = rows_exp2(fmaf(x[j + 1], q_up, -shift));
                            const float p2 = rows_exp2(fmaf(x[j + 2], q_up, -shift)), p3 = rows_exp2(fmaf(x[j + 3], q_up, -shift));
                            sum += (p0 + p1) + (p2 + p3);
                            const float v0 = p0 * up.x, v1 = p1 * up.y, v2 = p2 * up.z, v3 = p3 * up.w;
                            heavy = fmaxf(fmaxf(heavy, fmaxf(v0, v1)), fmaxf(v2, v3));
                            p[j / 2] = rows_half2(v0, v1);
                            p[j / 2 + 1] = rows_half2(v2, v3);
                        }
                        tiles_st16(lanes + S::COL_P + st * (TILE / 2) + w * 16, p);
                        if (odd) {
                            // a row that gives a token weight whose planes are not finite in a group becomes NaN there
#pragma unroll 1
                            for (int j = 0; j < 32; ++j) {
                                const uint32_t bad = meta.bad[st][32 * w + j] & 0x7Fu;
                                if (bad && (see(w) >> j & 1u)) {
                                    float z = 0.0f;
#pragma unroll
                                    for (int k = 0; k < 32; ++k) z = k == j ? x[k] : z;
                                    if (rows_exp2(fmaf(z, q_up, -shift)) > 0.0f) poison |= bad;
                                }
                            }
                        }
                    }
                    if (!__any_sync(kFullMask, heavy > 16384.0f) || round == 2) break;
                    tiles_wait_st();                           // the next round stores to the same columns
                    // E of the rows that have outgrown it: their largest p' to below 16, by what it is when nothing is divided
                    float most = 0.0f;
                    const float plain = m == -INFINITY ? 0.0f : m;
#pragma unroll 1
                    for (int w = 0; w < TILE / 32; ++w) {
                        float x[32];
                        load_logits(w, x);
#pragma unroll
                        for (int j = 0; j < 32; ++j) most = fmaxf(most, rows_exp2(fmaf(x[j], q_up, -plain)) * meta.v_up[st][32 * w + j]);
                    }
                    if (heavy > 16384.0f) {
                        const int e_new = min(max(e_o, rows_exponent(most) - 3), 119);
                        alpha *= rows_power(e_o - e_new);
                        e_o = e_new;
                    }
                }
                l = fmaf(l, alpha, sum);
                // ---- O, when m or E moved ----
                if (i > begin_i && __any_sync(kFullMask, alpha != 1.0f)) {
                    ok = wait(o_done(i - 1), two(i - 1));
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
                }
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
            if (!wait(o_done(i - 1), two(i - 1))) break;
            tiles_fence_after();
            float* part = a.partial + (size_t)(2 * blockIdx.x + (from_start ? 1 : 0)) * MT * (S::DV + 2);
            if (!whole && is) {
                part[r] = m + (float)e_o;
                part[MT + r] = l;
            }
            const float inv = whole ? (l == 0.0f ? 0.0f : 1.0f / l) : 1.0f;
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
                info.last = shares.of(item + begin_i + now.range.tiles - 1);
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
