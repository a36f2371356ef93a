// Attention over the quantised, paged cache for units of up to 128 rows (trees and chains): tcgen05 with tensor-memory accumulators.
//
// With this many rows the products bound it, 4 * 128 * D FLOP per token and unit, next to the unpacking, which a unit pays once for its 128 rows.
// One persistent block per SM: 8 warps of softmax, two threads to a row; 8 that unpack; two that measure the planes; a loader; one that issues the
// MMAs. For tile i of TILE tokens:
//   loader:  codes and planes by bulk copies, as they lie in the cache; a page's run of tokens is one copy
//   measure: a token's power of two (below), and scale and bias of its groups as fp16
//   unpack:  K_i, V_i in fp16, [64 elements][token][128 bytes] with the 128-byte swizzle (K in two buffers but for heads of 512, V in one: V_(i+1) is
//            unpacked behind K_(i+2), while O takes V_i)
//   MMA:     S_i = Q K_i^T into tensor memory (two buffers), then O += P_(i-1) V_(i-1); K is K-major, V, as it lies, MN-major
//   softmax: S_i -> registers -> mask, 2^(x - m), P_i as fp16 into tensor memory (the A operand of the second product)
// What it measured: 8 trees of 61 rows over 8000 tokens, 16 heads of 256 on 8 kv heads, 8 bits: 102 us, 1.9 TB/s and 329 TFLOP/s; 333 rows over 8000
// cached tokens, the same heads: 111 us, 408 TFLOP/s. A tile of 64 tokens takes about 4000 clocks, of which the tensor cores are busy for 1000. The
// rest is instructions that wait for one another: the warps' roles do not share code, so what a role takes must be short. Bodies are rolled
// and stand once (one for K and V), a wait that is over takes one look, the MMAs are issued without a branch, and the usual tile, which every row sees
// and whose powers of two are 1, leaves out the rest: in this order 139 -> 131 -> 114 -> 101 us. The warps that unpack were 8 that also
// loaded and measured: 127 us with all of the above left out.
// K_i and V_i carry code * scale + bias rounded once to fp16, at most 2^-11 of the value, and P its probabilities likewise: each adds an error of the size
// of the output's own rounding to fp16 (together 4e-4 to 5e-4 of the output's norm against 64 bits, 2e-4 of which fp16 outputs have anyhow; nothing next to
// bf16's 1.7e-3). Exact products of codes, as the kernel for few rows has them, would need an accumulator per group. A token whose planes are
// out of the ordinary is divided by a power of two of its own first; K's comes back with the logits, V's goes into the probabilities,
// p' = 2^(x - m - E) * 2^e, where E is a row's own and follows the largest p' so far, up and, as m is raised, down: tokens that a row does not
// see, or that have lost their weight, have no say, and no cache leaves fp16's range. m is raised only when a logit exceeds it by 8, and what O
// holds is rescaled only when m or E moves. TILE * D is 16384 but for heads of 64; heads of 512, whose product would fill tensor memory
// alone, are two units with half of the values each.
#pragma once

#include "async_copy.cuh"
#include "attention_rows.cuh"

namespace tf {

constexpr uint32_t kErrAttentionWait = 0x7F000053u;           // a bounded wait of attention_tiles_kernel ran out
constexpr uint32_t kLooks = 1u << 22;                         // looks of a bounded wait

template <int D, int BITS>
struct TilesShape {
    static constexpr int MT = 128, TILE = D == 512 ? 32 : D == 256 ? 64 : 128, DV = D < 256 ? D : 256, PARTS = D / DV, G = D / 64, GV = DV / 64;
    static constexpr int SOFT_WARPS = 8, UNPACK_WARPS = 8, MEASURE = SOFT_WARPS + UNPACK_WARPS, LOADER = MEASURE + 2, WARPS = LOADER + 2, THREADS = WARPS * kWarp, UNPACK = UNPACK_WARPS * kWarp;
    static constexpr int ROW_BYTES = D * BITS / 8, PIECE = 2 * BITS;          // bytes of 16 codes
    static constexpr int K_ROW = D / 16, V_ROW = DV / 16;                     // pieces of a token
    static constexpr int K_EACH = TILE * K_ROW / UNPACK, V_EACH = TILE * V_ROW / UNPACK;
    static constexpr int K_BUFS = D == 512 ? 1 : 2;
    static constexpr int Q_BYTES = MT * D * 2, K_BYTES = TILE * D * 2, V_BYTES = TILE * DV * 2;
    static constexpr int OFF_K = Q_BYTES, OFF_V = OFF_K + K_BUFS * K_BYTES;
    static constexpr int CHUNK = TILE / 2 < 32 ? TILE / 2 : 32;                // logits that a softmax thread has in registers at a time, of its half of a tile
    // what the loader has requested: codes and planes as they lie in the cache; and what it made of the planes, of four tiles [token][groups]
    static constexpr int KC_BUFS = TILE * ROW_BYTES > 8192 ? 1 : 2, V_ROW_BYTES = DV * BITS / 8;
    static constexpr int KC_BYTES = TILE * ROW_BYTES, VC_BYTES = TILE * V_ROW_BYTES, PLANE = TILE * G * 2;
    static constexpr int OFF_KC = OFF_V + V_BYTES, OFF_VC = OFF_KC + KC_BUFS * KC_BYTES, OFF_PL = OFF_VC + VC_BYTES, OFF_KW = OFF_PL + 2 * 4 * PLANE,
                         OFF_VW = OFF_KW + 4 * TILE * G * 4, OFF_META = OFF_VW + 4 * TILE * GV * 4;
    static constexpr int META = (28 * 8 + 224 + 8 * TILE * 9 + 127) / 128 * 128 + 2 * MT * 8 + MT * 4, SMEM = OFF_META + META + 1024;
    // tensor memory, in columns
    static constexpr int COL_S = 0, COL_P = 2 * TILE, COL_O = 3 * TILE, COLS = 512;
    static_assert(COL_O + DV <= COLS && SMEM <= 227 * 1024 && K_EACH * UNPACK == TILE * K_ROW && V_EACH * UNPACK == TILE * V_ROW, "sizes");
    // a 16-byte chunk (eight elements) of an operand row: [64 elements][rows][128 bytes], chunks swizzled by the row
    static __host__ __device__ __forceinline__ uint32_t chunk_at(uint32_t rows, uint32_t row, uint32_t chunk) {
        return (chunk >> 3) * (rows * 128) + row * 128 + (((chunk & 7u) ^ (row & 7u)) << 4);
    }
};

// The block's barriers, what the loader tells about a tile whose planes are there, and what the measuring warps tell the softmax (of eight tiles).
template <int TILE>
struct TilesMeta {
    unsigned long long bars[28];
    uint32_t tmem, dead;
    uint32_t flags[8][2];          // K's and V's: 1: powers of two that are not 1; 2: something in `bad`
    float v_most[8];               // the largest of v_up
    alignas(16) uint4 tile[4];     // first token, end of what is seen, the runs that have a page, first value group
    alignas(16) float k_up[8][TILE];          // what a token's logits are multiplied with: its power of two, the scale, log2 e
    alignas(16) float v_up[8][TILE];          // a token's power of two
    uint8_t bad[8][TILE];          // bit g: value planes of group g are not finite; bit 7: the token's page is missing
    float pair[2][128][2];         // between the two softmax threads of a row, by turns
    float q_up[128];               // a row's power of two
};

// Operand descriptors for the 128-byte swizzle: the lower word holds the address and the leading offset, the upper one a stride of 1024 bytes. The MMAs
// are issued by all lanes under a predicate of one: code without a branch, whose addresses the compiler can keep in uniform registers.
__device__ __forceinline__ uint32_t tiles_desc(uint32_t addr, uint32_t leading) { return ((addr & 0x3FFFFu) >> 4) | (leading >> 4) << 16; }
constexpr uint32_t kDescUpper = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ void tiles_mma_ss(bool issues, uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p, q;\n\t.reg .b64 a, b;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\tmov.b64 a, {%1, %6};\n\tmov.b64 b, {%2, %6};\n\t"
                 "@q tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n\t}"
                 ::"r"(d), "r"(a), "r"(b), "r"(idesc), "r"(accumulate), "r"((uint32_t)issues), "r"(kDescUpper) : "memory");
}
__device__ __forceinline__ void tiles_mma_ts(bool issues, uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p, q;\n\t.reg .b64 b;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\tmov.b64 b, {%2, %6};\n\t"
                 "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p;\n\t}"
                 ::"r"(d), "r"(a), "r"(b), "r"(idesc), "r"(accumulate), "r"((uint32_t)issues), "r"(kDescUpper) : "memory");
}
__device__ __forceinline__ void tiles_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void tiles_ld(uint32_t addr, uint32_t (&r)[32]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 "
                 "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
                   "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]),
                   "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
                 : "r"(addr) : "memory");
}
__device__ __forceinline__ void tiles_st(uint32_t addr, const uint32_t (&r)[32]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
                 "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};"
                 ::"r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
                   "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]),
                   "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]) : "memory");
}
__device__ __forceinline__ void tiles_st(uint32_t addr, const uint32_t (&r)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
                 ::"r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
                   "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]) : "memory");
}
__device__ __forceinline__ void tiles_ld(uint32_t addr, uint32_t (&r)[16]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
                   "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void tiles_st(uint32_t addr, const uint32_t (&r)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};"
                 ::"r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]) : "memory");
}
__device__ __forceinline__ void tiles_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tiles_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tiles_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tiles_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// Sixteen codes as code * s + b in fp16, rounded once (code, s and b are fp16 numbers), two 16-byte chunks of eight elements. 4-bit codes of eight elements come in the order
// (0, 4, 1, 5, 2, 6, 3, 7), as one mask yields them: the rows of q are laid out alike, and the product's columns are put back at the end.
template <int BITS>
__device__ __forceinline__ void tiles_unpack(const uint32_t (&w)[BITS / 2], __half2 s, __half2 b, uint4 (&out)[2]) {
    uint32_t h[8];
    auto put = [&](int i, uint32_t bits, float off, __half2 by) {
        const __half2 v = __hfma2(__hadd2(*reinterpret_cast<const __half2*>(&bits), __float2half2_rn(off)), by, b);
        h[i] = *reinterpret_cast<const uint32_t*>(&v);
    };
    if constexpr (BITS == 8) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            put(2 * i, gm_prmt(w[i], 0x64646464u, 0x4140), -1024.0f, s);             // 1024 from the bits
            put(2 * i + 1, gm_prmt(w[i], 0x64646464u, 0x4342), -1024.0f, s);
        }
    } else {
        const __half2 s16 = __hmul2(s, __float2half2_rn(0.0625f));
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint32_t v = w[i] >> 8;
            put(4 * i, (w[i] & 0x000F000Fu) | 0x64006400u, -1024.0f, s);
            put(4 * i + 1, (w[i] & 0x00F000F0u) | 0x64006400u, -1024.0f, s16);
            put(4 * i + 2, (v & 0x000F000Fu) | 0x64006400u, -1024.0f, s);
            put(4 * i + 3, (v & 0x00F000F0u) | 0x64006400u, -1024.0f, s16);
        }
    }
    out[0] = make_uint4(h[0], h[1], h[2], h[3]);
    out[1] = make_uint4(h[4], h[5], h[6], h[7]);
}

__device__ __forceinline__ bool tiles_look(uint32_t bar, uint32_t phase) {
    uint32_t ok;
    asm volatile("{ .reg .pred p; mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2; selp.u32 %0, 1, 0, p; }" : "=r"(ok) : "r"(bar), "r"(phase) : "memory");
    return ok;
}
// Looks until the phase is over; a wait that runs out tells all others, which end at their next 64th look.
static __device__ __noinline__ bool tiles_wait(uint32_t bar, uint32_t phase, volatile uint32_t* dead, uint32_t* error) {
#pragma unroll 1
    for (uint32_t look = 0; look < kLooks; ++look) {
        if (tiles_look(bar, phase)) return true;
        if (look % 64 == 0 && *dead) return false;
    }
    *dead = 1;
    *error = kErrAttentionWait;
    return false;
}

template <int MT, int TILE>
__device__ __noinline__ void tiles_next_unit(const AttnArgs& a, Cursor<MT, TILE>& c) { c.next_unit(a); }

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
    // Barriers of tile i and the phase in which they are done with it, by the number of their buffers. The issuer's order makes one stand for others:
    // a commit counts all MMAs before it, so S_i there (s_full, k_free) means that O holds tile i - 2, and that the softmax had left
    // tile i - 2 (its probabilities were waited for).
    auto k_full = [&](uint32_t i) { return bars + (i % S::K_BUFS) * 8; };
    auto k_free = [&](uint32_t i) { return bars + 16 + (i % S::K_BUFS) * 8; };       // K's buffer: the logits of tile i are there
    auto s_full = [&](uint32_t i) { return bars + 32 + (i & 1) * 8; };      // S_i, and by an arrival of the issuer what it saw: what is told about tile i
    auto p_full = [&](uint32_t i) { return bars + 48 + (i & 1) * 8; };      // P_i; S_i has been read, and what was told
    auto o_done = [&](uint32_t i) { return bars + 64 + (i & 1) * 8; };      // O holds tile i
    const uint32_t q_full = bars + 80, all_done = bars + 88, v_full = bars + 96;
    auto pl_full = [&](uint32_t i) { return bars + 104 + (i & 1) * 8; };                   // planes
    auto kc_full = [&](uint32_t i) { return bars + 120 + (i % S::KC_BUFS) * 8; };          // K's codes
    auto kc_free = [&](uint32_t i) { return bars + 136 + (i % S::KC_BUFS) * 8; };
    auto pl_free = [&](uint32_t i) { return bars + 152 + (i & 1) * 8; };
    const uint32_t vc_full = bars + 168, vc_free = bars + 176;
    auto told = [&](uint32_t i) { return bars + 184 + (i & 3) * 8; };       // what the planes say; four, as nobody waits for those who look at it
    auto one = [](uint32_t i) { return i & 1u; };
    auto two = [](uint32_t i) { return i >> 1 & 1u; };
    auto of_k = [](uint32_t i) { return i / S::K_BUFS & 1u; };
    auto of_kc = [](uint32_t i) { return i / S::KC_BUFS & 1u; };
    // of a whole warp; what a wait that is over already takes is kept short
    auto wait = [&](uint32_t bar, uint32_t phase) -> bool {
        return __all_sync(kFullMask, tiles_look(bar, phase)) || __all_sync(kFullMask, tiles_wait(bar, phase, &meta.dead, a.error));
    };

    if (tid == 0) {
        mbar_init(v_full, S::UNPACK_WARPS);
        for (uint32_t i = 0; i < 2; ++i) {
            mbar_init(bars + i * 8, S::UNPACK_WARPS);
            mbar_init(bars + 16 + i * 8, 1);
            mbar_init(s_full(i), 2);
            mbar_init(p_full(i), S::SOFT_WARPS);
            mbar_init(o_done(i), 1);
            mbar_init(pl_full(i), 1);
            mbar_init(pl_free(i), 2);
            mbar_init(bars + 120 + i * 8, 1);
            mbar_init(told(i), 2);
            mbar_init(told(i + 2), 2);
            mbar_init(bars + 136 + i * 8, S::UNPACK_WARPS);
        }
        mbar_init(vc_full, 1);
        mbar_init(vc_free, S::UNPACK_WARPS);
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

    if (warp >= S::SOFT_WARPS && warp < S::SOFT_WARPS + S::UNPACK_WARPS) {
        // ===================== unpacking: a thread's piece is sixteen elements of one token =====================
        const uint32_t u = tid - S::SOFT_WARPS * kWarp;
        const uint32_t k_piece = u % S::K_ROW, v_piece = u % S::V_ROW, k_key0 = u / S::K_ROW, v_key0 = u / S::V_ROW;
        constexpr int kBoth = S::K_EACH < S::V_EACH ? S::K_EACH : S::V_EACH, kAtOnce = kBoth < 4 ? kBoth : 4;
        // K_0, K_1, V_0, K_2, V_1, ...: one body for both. A wait that runs out is told to all, whose later waits end at once; every warp goes through all tiles.
#pragma unroll 1
        for (uint32_t turn = 0; turn <= 2 * count; ++turn) {
            const bool is_v = turn && turn % 2 == 0;
            const uint32_t n = is_v ? turn / 2 - 1 : (turn + 1) / 2;
            if (n >= count) continue;
            if (is_v) {
                if (n >= 1) wait(o_done(n - 1), two(n - 1));
                wait(vc_full, one(n));
            } else {
                if (n >= S::K_BUFS) wait(k_free(n), of_k(n - S::K_BUFS));
                wait(told(n), n >> 2 & 1u);
                wait(kc_full(n), of_kc(n));
            }
            const uint32_t from = is_v ? S::OFF_VC : S::OFF_KC + (n % S::KC_BUFS) * S::KC_BYTES, to = is_v ? S::OFF_V : S::OFF_K + (n % S::K_BUFS) * S::K_BYTES;
            const uint32_t words = is_v ? S::OFF_VW + (n & 3) * (TILE * S::GV * 4) : S::OFF_KW + (n & 3) * (TILE * S::G * 4);
            const uint32_t row_bytes = S::PARTS > 1 && is_v ? S::V_ROW_BYTES : S::ROW_BYTES, groups = S::PARTS > 1 && is_v ? S::GV : S::G;
            const uint32_t piece = S::PARTS > 1 && is_v ? v_piece : k_piece, keys = S::PARTS > 1 && is_v ? S::UNPACK / S::V_ROW : S::UNPACK / S::K_ROW;
            const bool odd = S::K_ROW >= 8 && (piece / 4 & 1u);
            uint32_t key = S::PARTS > 1 && is_v ? v_key0 : k_key0;
#pragma unroll 1
            for (; key < (uint32_t)TILE; key += kAtOnce * keys) {
                uint32_t r[kAtOnce][BITS / 2], w[kAtOnce];
#pragma unroll
                for (int j = 0; j < kAtOnce; ++j) {
                    const uint8_t* at = smem + from + (key + j * keys) * row_bytes + piece * S::PIECE;
                    w[j] = *reinterpret_cast<const uint32_t*>(smem + words + ((key + j * keys) * groups + piece / 4) * 4);
                    // lanes of odd groups take the second eight first, so that eight lanes meet eight different banks when they store
                    if constexpr (BITS == 8) {
                        const uint4 x = *reinterpret_cast<const uint4*>(at);
                        r[j][0] = odd ? x.z : x.x; r[j][1] = odd ? x.w : x.y; r[j][2] = odd ? x.x : x.z; r[j][3] = odd ? x.y : x.w;
                    } else {
                        const uint2 x = *reinterpret_cast<const uint2*>(at);
                        r[j][0] = odd ? x.y : x.x; r[j][1] = odd ? x.x : x.y;
                    }
                }
#pragma unroll
                for (int j = 0; j < kAtOnce; ++j) {
                    const uint32_t k = key + j * keys, sc = gm_prmt(w[j], 0, 0x1010), bi = gm_prmt(w[j], 0, 0x3232);
                    uint4 h[2];
                    tiles_unpack<BITS>(r[j], *reinterpret_cast<const __half2*>(&sc), *reinterpret_cast<const __half2*>(&bi), h);
                    const uint32_t at = to + k * 128 + (piece / 4) * (TILE * 128), c0 = (piece % 4 * 2 + odd) ^ (k & 7u);
                    *reinterpret_cast<uint4*>(smem + at + c0 * 16) = h[0];
                    *reinterpret_cast<uint4*>(smem + at + (c0 ^ 1u) * 16) = h[1];
                }
            }
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(is_v ? v_full : k_full(n));
                mbar_arrive(is_v ? vc_free : kc_free(n));
            }
        }
    } else if (warp >= S::MEASURE && warp < S::LOADER) {
        // ===================== what the planes say: one warp for K's, one for V's, a token per lane =====================
        // Scale and bias of a token's groups as fp16, by a power of two of the token's, 2^e: e = 0 where all its groups are of ordinary sizes. fp16 holds a bf16 of its normal
        // range exactly, and one below it to 2^-25, which 255 codes (15 of 16 times the step) make 2^-17 of a value: a group whose scale is that small (kExact) is
        // ordinary only if its bias is 2^-4 or more. Elsewhere a key's largest group is brought to [2^7, 2^8). A value's 2^e goes into fp16 probabilities, next to those of
        // tokens with e = 0: were it far below the value's size, long tails of small probabilities would be lost there. So from 2^-1 down it is at least 2^-8, and
        // from 2^-12 down 2^4 times the size, and ordinary values are within [2^-7, 2^7]. No rounding of the planes is above 2^-13 of the token's largest group.
        constexpr float kExact = BITS == 8 ? 7.62939453125e-6f : 1.220703125e-4f;              // 2^-17; 2^-13, since 4-bit codes take a sixteenth of the scale too
        const bool of_v = warp != S::MEASURE;
        const float least = of_v ? 0.0078125f : 0.001953125f, largest = of_v ? 128.0f : 16384.0f;      // of an ordinary group
        const uint32_t run_log2 = lesser(a.table.page_log2, (uint32_t)(31 - __builtin_clz(TILE)));
        auto measure = [&](auto groups, uint32_t n, const uint4& t) {
            constexpr int N = decltype(groups)::value;
            uint32_t any = 0;
            float most_up = 0.0f;
#pragma unroll 1
            for (uint32_t key = lane; key < (uint32_t)TILE; key += kWarp) {
                const bool held = t.x + key < t.y, is = held && (t.z >> (key >> run_log2) & 1u);
                const uint16_t* scales = reinterpret_cast<const uint16_t*>(smem + S::OFF_PL + ((n & 1) * 4 + 2 * of_v) * S::PLANE) + key * S::G + (of_v ? t.w : 0u);
                uint32_t words[N], bits = 0;
                float sc[N], bi[N], most = 0.0f;
                bool plain = true;
#pragma unroll
                for (int g = 0; g < N; ++g) {
                    sc[g] = is ? bf16_bits_to_float(scales[g]) : 0.0f;
                    bi[g] = is ? bf16_bits_to_float(scales[S::PLANE / 2 + g]) : 0.0f;
                }
#pragma unroll
                for (int g = 0; g < N; ++g) {
                    const float size = fmaxf(kCentre * fabsf(sc[g]), fabsf(bi[g]));        // a third of the largest value or more
                    // nor do planes whose values leave fp32 have a place in fp16 (times a probability of zero they would be no number)
                    const bool finite = sc[g] - sc[g] == 0.0f && bi[g] - bi[g] == 0.0f && size <= 3.402823466e38f;
                    plain = plain && finite && size >= (fabsf(sc[g]) >= kExact ? least : 0.0625f) && size <= largest;
                    most = finite ? fmaxf(most, size) : most;
                    if (of_v && !finite) {
                        bits |= 1u << g;
                        sc[g] = bi[g] = 0.0f;
                    }
                }
                const int at = rows_exponent(most), brought = of_v ? min(at + 4, max(at - 7, -8)) : at - 7;
                const int e = plain || !is ? 0 : min(max(brought, -126), 119);                       // both parts of a value below 2^8
                const float down = rows_power(-e), up = rows_power(e);
                any |= e != 0;
#pragma unroll
                for (int g = 0; g < N; ++g) words[g] = rows_half2(sc[g] * down, bi[g] * down);
                uint32_t* to = reinterpret_cast<uint32_t*>(smem + (of_v ? S::OFF_VW : S::OFF_KW)) + ((n & 3) * TILE + key) * N;
#pragma unroll
                for (int g = 0; g < N; g += 4) {
                    if constexpr (N >= 4) *reinterpret_cast<uint4*>(to + g) = make_uint4(words[g], words[g + 1], words[g + 2], words[g + 3]);
                    else if constexpr (N == 2) *reinterpret_cast<uint2*>(to) = make_uint2(words[0], words[1]);
                    else to[0] = words[0];
                }
                if (of_v) {
                    if (held && !is) bits = 0x80u;
                    meta.v_up[n & 7][key] = up;
                    meta.bad[n & 7][key] = (uint8_t)bits;
                    if (bits) any |= 2u;
                    most_up = fmaxf(most_up, up);
                } else {
                    meta.k_up[n & 7][key] = up * (a.scale * 1.4426950408889634f);
                }
            }
            any = __reduce_or_sync(kFullMask, any);
            most_up = __uint_as_float(__reduce_max_sync(kFullMask, __float_as_uint(most_up)));
            if (lane == 0) {
                meta.flags[n & 7][of_v] = any;
                if (of_v) meta.v_most[n & 7] = most_up;
            }
        };
#pragma unroll 1
        for (uint32_t n = 0; n < count; ++n) {
            wait(pl_full(n), two(n));
            const uint4 t = meta.tile[n & 3];
            if (of_v) measure(std::integral_constant<int, S::GV>(), n, t);
            else measure(std::integral_constant<int, S::G>(), n, t);
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(pl_free(n));
                mbar_arrive(told(n));
            }
        }
    } else if (warp == S::LOADER) {
        // ===================== loader: which rows of the cache, their codes and planes by bulk copies =====================
        // Lane r has the tile's r-th run of tokens, which one page holds. Steps of tile n: planes of n + 1, K of n, V of n - 1: the order in which
        // the unpacking takes them, so that no request waits for a buffer that is freed after another one's. By then V_(n-3) has been unpacked, which
        // was behind O's taking V_(n-4): what was told about tile n - 7 is not looked at any more, nor the words of tile n - 3.
        struct Tile { uint32_t token0, end, head; const int32_t* table; };
        const uint32_t page_log2 = a.table.page_log2, run_log2 = lesser(page_log2, (uint32_t)(31 - __builtin_clz(TILE))), first = (uint32_t)lane << run_log2;
        constexpr uint32_t kNone = 0xFFFFFFFFu;                // rows of the cache are below, as the entry point has checked
        auto tile_of = [&](const Cursor<MT, TILE>& c) { return Tile{c.token0(), c.range.end, c.head, a.table.table + (size_t)c.b * a.table.stride}; };
        auto page_of = [&](const Tile& t) -> int32_t { return first < (uint32_t)TILE && t.token0 + first < t.end ? t.table[(t.token0 + first) >> page_log2] : -1; };
        auto row_of = [&](const Tile& t, int32_t page) -> uint32_t {
            return page >= 0 && (uint32_t)page < a.table.pages
                       ? (((uint32_t)page * a.kv_heads + t.head / S::PARTS) << page_log2) + ((t.token0 + first) & ((1u << page_log2) - 1u)) : kNone;
        };
        // tells the barrier what comes: `bytes` for every token of the runs that are there
        auto expect = [&](uint32_t bar, uint32_t runs, uint32_t bytes) {
            if (lane == 0) mbar_arrive_expect_tx(bar, (__popc(runs) << run_log2) * bytes);
            __syncwarp();
        };
        auto ask = [&](uint32_t to, const void* plane, uint32_t row, uint32_t bytes, uint32_t bar) {
            bulk_copy_g2s(base + to + first * bytes, static_cast<const uint8_t*>(plane) + (size_t)row * bytes, bytes << run_log2, bar);
        };
        auto ask_planes = [&](uint32_t n, const Tile& t, uint32_t row) {
            const uint32_t runs = __ballot_sync(kFullMask, row != kNone);
            if (lane == 0) meta.tile[n & 3] = make_uint4(t.token0, t.end, runs, t.head % S::PARTS * S::GV);
            expect(pl_full(n), runs, 4 * S::G * 2);
            if (row != kNone) {
                const uint32_t to = S::OFF_PL + (n & 1) * (4 * S::PLANE);
                ask(to, a.k.scales, row, S::G * 2, pl_full(n));
                ask(to + S::PLANE, a.k.biases, row, S::G * 2, pl_full(n));
                ask(to + 2 * S::PLANE, a.v.scales, row, S::G * 2, pl_full(n));
                ask(to + 3 * S::PLANE, a.v.biases, row, S::G * 2, pl_full(n));
            }
        };
        auto ask_k = [&](uint32_t n, uint32_t row) {
            expect(kc_full(n), __ballot_sync(kFullMask, row != kNone), S::ROW_BYTES);
            if (row != kNone) ask(S::OFF_KC + (n % S::KC_BUFS) * S::KC_BYTES, a.k.codes, row, S::ROW_BYTES, kc_full(n));
        };
        auto ask_v = [&](uint32_t row, uint32_t head) {
            expect(vc_full, __ballot_sync(kFullMask, row != kNone), S::V_ROW_BYTES);
            if constexpr (S::PARTS == 1) {
                if (row != kNone) ask(S::OFF_VC, a.v.codes, row, S::ROW_BYTES, vc_full);
            } else {                                           // half of every token's
#pragma unroll
                for (uint32_t key = lane; key < (uint32_t)TILE; key += kWarp) {
                    const uint32_t r = __shfl_sync(kFullMask, row, key >> run_log2);
                    if (r != kNone)
                        bulk_copy_g2s(base + S::OFF_VC + key * S::V_ROW_BYTES, a.v.codes + (size_t)(r + (key & ((1u << run_log2) - 1u))) * S::ROW_BYTES + head % S::PARTS * S::V_ROW_BYTES,
                                      S::V_ROW_BYTES, vc_full);
                }
            }
        };
        Cursor<MT, TILE> next = now;                           // of the tile whose pages are looked up
        uint32_t left = busy ? (uint32_t)lesser((uint64_t)(now.range.tiles - now.tile), stop - item) : 0, ahead = 0;
        auto step = [&](const Tile& t) -> Tile {               // the tile after t, if there is one; `next` is its cursor
            if (++ahead >= count) return t;
            if (--left == 0) {
                tiles_next_unit<MT, TILE>(a, next);
                left = (uint32_t)lesser((uint64_t)next.range.tiles, (uint64_t)(count - ahead));
                return tile_of(next);
            }
            ++next.tile;
            return Tile{t.token0 + TILE, t.end, t.head, t.table};
        };
        // After a wait that ran out nothing more is requested; what was is waited for before the block leaves.
        bool fine = true;
        uint32_t k_asked = 0, v_asked = 0, p_asked = 0;
        if (count) {
            Tile t0 = tile_of(next), t1 = step(t0);
            uint32_t row0 = row_of(t0, page_of(t0)), row_v = kNone, head_v = 0;
            int32_t page1 = page_of(t1);
            ask_planes(0, t0, row0);
            p_asked = 1;
#pragma unroll 1
            for (uint32_t n = 0; n <= count; ++n) {
                uint32_t row1 = kNone;
                const Tile t2 = step(t1);
                const int32_t page2 = page_of(t2);             // needed a tile later
                if (n + 1 < count) {
                    row1 = row_of(t1, page1);
                    if (n) fine = fine && wait(pl_free(n - 1), two(n - 1));
                    if (fine) {
                        ask_planes(n + 1, t1, row1);
                        p_asked = n + 2;
                    }
                }
                if (n < count) {
                    if (n >= S::KC_BUFS) fine = fine && wait(kc_free(n), of_kc(n - S::KC_BUFS));
                    if (fine) {
                        ask_k(n, row0);
                        k_asked = n + 1;
                    }
                }
                if (n) {
                    if (n >= 2) fine = fine && wait(vc_free, one(n - 2));
                    if (fine) {
                        ask_v(row_v, head_v);
                        v_asked = n;
                    }
                }
                if (!fine) break;
                row_v = row0;
                head_v = t0.head;
                row0 = row1;
                t0 = t1;
                t1 = t2;
                page1 = page2;
            }
        }
        auto drain = [&](uint32_t bar, uint32_t phase) {       // whatever the others have told
            for (uint32_t look = 0; look < kLooks && !tiles_look(bar, phase); ++look) {}
        };
        for (uint32_t n = k_asked > S::KC_BUFS ? k_asked - S::KC_BUFS : 0; n < k_asked; ++n) drain(kc_full(n), of_kc(n));
        if (v_asked) drain(vc_full, one(v_asked - 1));
        for (uint32_t n = p_asked > 2 ? p_asked - 2 : 0; n < p_asked; ++n) drain(pl_full(n), two(n));
    } else if (warp == S::WARPS - 1) {
        // ===================== MMA issuer =====================
        constexpr uint32_t idesc_s = (1u << 4) | ((uint32_t)(TILE >> 3) << 17) | ((uint32_t)(MT >> 4) << 24);
        constexpr uint32_t idesc_o = (1u << 4) | (1u << 16) | ((uint32_t)(S::DV >> 3) << 17) | ((uint32_t)(MT >> 4) << 24);      // B: MN-major
        uint32_t segment = 0, segments = 0;
        bool opens = false;                                    // tile i - 1 is its unit's first here: its product starts O anew
        auto logits = [&](uint32_t i) -> bool {
            if (!wait(k_full(i), of_k(i))) return false;
            tiles_fence_after();
            {
                const uint32_t q0 = tiles_desc(base, 16), k0 = tiles_desc(base + S::OFF_K + (i % S::K_BUFS) * S::K_BYTES, 16);
#pragma unroll
                for (int e = 0; e < D / 16; ++e)
                    tiles_mma_ss(lane == 0, tmem + S::COL_S + (i & 1) * TILE, q0 + (((e / 4) * (MT * 128) + e % 4 * 32) >> 4), k0 + (((e / 4) * (TILE * 128) + e % 4 * 32) >> 4),
                                 idesc_s, e > 0);
            }
            if (lane == 0) {
                tiles_commit(s_full(i));
                tiles_commit(k_free(i));
                mbar_arrive(s_full(i));
            }
            __syncwarp();
            return true;
        };
        auto values = [&](uint32_t j) -> bool {
            if (!wait(v_full, one(j)) || !wait(p_full(j), two(j))) return false;
            tiles_fence_after();
            {
                const uint32_t v0 = tiles_desc(base + S::OFF_V, TILE * 128);
#pragma unroll
                for (int e = 0; e < TILE / 16; ++e)
                    tiles_mma_ts(lane == 0, tmem + S::COL_O, tmem + S::COL_P + (j & 1) * (TILE / 2) + e * 8, v0 + (e * 2048 >> 4), idesc_o, e > 0 || !opens);
            }
            if (lane == 0) tiles_commit(o_done(j));
            __syncwarp();
            return true;
        };
        bool fine = true;
#pragma unroll 1
        for (uint32_t i = 0; i <= count && fine; ++i) {
            // Within a unit the logits of tile i go ahead of the values of tile i - 1; at a unit's end the softmax waits for those values before it
            // lays out the next rows of q.
            const bool new_unit = i < count && segment == 0, behind = new_unit || i == count;
#pragma unroll 1
            for (int half = 0; half < 2 && fine; ++half) {
                if (behind == (half == 0)) {
                    if (i) fine = values(i - 1);
                } else if (i < count) {
                    if (new_unit) {
                        if (i) tiles_next_unit<MT, TILE>(a, now);
                        segment = (uint32_t)lesser((uint64_t)(now.range.tiles - now.tile), (uint64_t)(count - i));
                        fine = wait(q_full, segments++ & 1u);
                    }
                    fine = fine && logits(i);
                }
            }
            opens = new_unit;
            --segment;
        }
        // nothing is in flight when the block leaves
        if (lane == 0) tiles_commit(all_done);
        __syncwarp();
        for (uint32_t look = 0; look < kLooks && !tiles_look(all_done, 0); ++look) {}
    } else {
        // ===================== softmax: two threads per row, warps w and w + 4, with half of a tile each =====================
        const uint32_t quad = warp % 4, side = warp / 4, r = quad * 32 + lane, lanes = tmem + (quad * 32u << 16);
        constexpr int CHUNK = S::CHUNK, HALF = TILE / 2;
        uint32_t turn = 0;
        // both threads' values of a pair, and a barrier of the two warps
        auto swap = [&](float x, float& y) {
            meta.pair[turn][r][side] = x;
            asm volatile("bar.sync %0, 64;" ::"r"(2 + quad) : "memory");
            y = meta.pair[turn][r][side ^ 1];
            turn ^= 1;
        };
        uint32_t i = 0;
        bool ok = true;
        while (i < count) {
            // ---- the unit's rows of q: fp16 in the operand's layout, brought to one range by a power of two ----
            const uint32_t valid = lesser((uint32_t)MT, now.flat_rows(a) - now.flat0), first_tile = now.tile;
            const uint32_t segment = (uint32_t)lesser((uint64_t)(now.range.tiles - first_tile), (uint64_t)(count - i));
            const bool is = r < valid, from_start = first_tile == 0, whole = from_start && segment == now.range.tiles;
            const uint32_t flat = now.flat0 + (is ? r : 0), node = flat / a.group, head = now.head / S::PARTS;
            {
                // lanes side by side along the rows; bf16 rows are brought to one range, their largest element to [1, 2)
                constexpr int ROW_LANES = D / 8 < 32 ? D / 8 : 32, EACH = D / 8 / ROW_LANES, AT_ONCE = S::SOFT_WARPS * kWarp / ROW_LANES;
                const uint32_t row_lane = tid % ROW_LANES;
#pragma unroll 4
                for (uint32_t q = tid / ROW_LANES; q < MT; q += AT_ONCE) {
                    const uint32_t f = now.flat0 + (q < valid ? q : 0);
                    const uint4* src = reinterpret_cast<const uint4*>(a.q + (size_t)(now.seq.row0 + f / a.group) * a.q_stride + (size_t)(head * a.group + f % a.group) * D) + row_lane;
                    uint4 v[EACH];
#pragma unroll
                    for (int e = 0; e < EACH; ++e) v[e] = q < valid ? src[e * ROW_LANES] : make_uint4(0, 0, 0, 0);
                    float up = 1.0f;
                    if constexpr (BF16) {
                        uint32_t most = 0;
#pragma unroll
                        for (int e = 0; e < EACH; ++e)
                            most = __vmaxu2(__vmaxu2(__vmaxu2(most, v[e].x & 0x7FFF7FFFu), __vmaxu2(v[e].y & 0x7FFF7FFFu, v[e].z & 0x7FFF7FFFu)), v[e].w & 0x7FFF7FFFu);
                        most = max(most & 0xFFFFu, most >> 16);
#pragma unroll
                        for (int off = ROW_LANES / 2; off >= 1; off >>= 1) most = max(most, __shfl_xor_sync(kFullMask, most, off));
                        const float top = bf16_bits_to_float((uint16_t)most);
                        const int e_q = top > 0.0f && top <= 3.402823466e38f ? max(rows_exponent(top), -126) : 0;
                        const float down = rows_power(-e_q);
                        up = rows_power(e_q);
#pragma unroll
                        for (int e = 0; e < EACH; ++e) {
                            uint32_t* w = reinterpret_cast<uint32_t*>(&v[e]);
#pragma unroll
                            for (int j = 0; j < 4; ++j) w[j] = rows_half2(__uint_as_float(w[j] << 16) * down, __uint_as_float(w[j] & 0xFFFF0000u) * down);
                        }
                    }
                    if (row_lane == 0) meta.q_up[q] = up;
#pragma unroll
                    for (int e = 0; e < EACH; ++e) {
                        const uint4 h = v[e];
                        const uint4 out = BITS == 8 ? h : make_uint4(gm_prmt(h.x, h.z, 0x5410), gm_prmt(h.x, h.z, 0x7632), gm_prmt(h.y, h.w, 0x5410), gm_prmt(h.y, h.w, 0x7632));
                        *reinterpret_cast<uint4*>(smem + S::chunk_at(MT, q, row_lane + e * ROW_LANES)) = out;
                    }
                }
            }
            fence_proxy_async();
            asm volatile("bar.sync 1, %0;" ::"n"(S::SOFT_WARPS * kWarp) : "memory");           // the rows' powers of two
            if (lane == 0) mbar_arrive(q_full);
            const float q_up = meta.q_up[r];
            uint32_t low = 0;                                  // first token that the row sees
            if (a.window && is) {
                const int64_t pos = a.mask ? max((int64_t)a.positions[now.seq.row0 + node], (int64_t)now.seq.context) : (int64_t)now.seq.context + node;
                low = (uint32_t)max((int64_t)0, lesser(pos - (int64_t)a.window + 1, (int64_t)kMostTokens));
            }
            const uint32_t low_most = __reduce_max_sync(kFullMask, low), open_end = lesser(now.seq.context, now.range.end);
            float m = -INFINITY, l = 0.0f;                     // of the row; l of this thread's tokens, in units of 2^m; O is in units of 2^(m + E)
            int e_o = kLeastPower;                             // E
            bool far = false;                                  // a row's E is beyond the usual tile's reach
            uint32_t poison = 0;                               // groups that are not a number
            const uint32_t begin_i = i, stop_i = i + segment;
            uint32_t token0 = now.token0() + side * HALF;
            // A wait that runs out is told to all, whose later waits end at once; the warps of a pair go through all tiles, since they meet in each.
#pragma unroll 1
            for (; i < stop_i; ++i, token0 += TILE) {
                const uint32_t st = i & 1;
                ok = wait(s_full(i), two(i));
                tiles_fence_after();
                const uint2 flags = *reinterpret_cast<const uint2*>(meta.flags[i & 7]);
                const float v_most = meta.v_most[i & 7];
                const bool odd = flags.y & 2u, open = !odd && token0 >= low_most && token0 + HALF <= open_end;
                // The usual tile: all rows see all tokens, whose powers of two are 1. What other tiles take is kept out of its way.
                const bool usual = open && (flags.x | flags.y) == 0 && a.scale > 0.0f && !far;
                const float by = usual ? q_up * (a.scale * 1.4426950408889634f) : q_up;
                // the tokens from `t0` on that the row sees, a chunk of them
                auto see = [&](int c0) -> uint32_t {
                    const uint32_t t0 = token0 + c0;
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
#pragma unroll 1
                        for (int j = 0; j < CHUNK; ++j)
                            if ((meta.bad[i & 7][side * HALF + c0 + j] & 0x80u) && (seen >> j & 1u)) {
                                seen &= ~(1u << j);
                                if (is) *a.error = kErrKvPage;         // (pages of tokens that no row sees may be missing: those that fell out of every window)
                            }
                    return is ? seen : 0u;
                };
                // the logits of a chunk, in base 2 but for `by`
                auto load_logits = [&](int c0, float (&x)[CHUNK]) {
                    uint32_t raw[CHUNK];
                    tiles_ld(lanes + S::COL_S + st * TILE + side * HALF + c0, raw);
                    tiles_wait_ld();
#pragma unroll
                    for (int j = 0; j < CHUNK; ++j) x[j] = __uint_as_float(raw[j]);
                    if (!usual) {
                        const uint32_t seen = open ? 0xFFFFFFFFu : see(c0);
#pragma unroll
                        for (int j = 0; j < CHUNK; j += 4) {
                            const float4 up = *reinterpret_cast<const float4*>(&meta.k_up[i & 7][side * HALF + c0 + j]);
                            x[j] = seen >> j & 1u ? x[j] * up.x : -INFINITY;
                            x[j + 1] = seen >> (j + 1) & 1u ? x[j + 1] * up.y : -INFINITY;
                            x[j + 2] = seen >> (j + 2) & 1u ? x[j + 2] * up.z : -INFINITY;
                            x[j + 3] = seen >> (j + 3) & 1u ? x[j + 3] * up.w : -INFINITY;
                        }
                    }
                };
                // ---- maximum ----
                float top = -INFINITY, x[CHUNK];               // x: where a half is one chunk, it stays
#pragma unroll 1
                for (int c0 = 0; c0 < HALF; c0 += CHUNK) {
                    load_logits(c0, x);
#pragma unroll
                    for (int j = 0; j < CHUNK; ++j) top = fmaxf(top, x[j]);
                }
                float other;
                const float own = top * by;
                swap(own, other);
                top = fmaxf(own, other);
                // E, the power of what had weight so far, falls by as much as that weight when m is raised (whole powers: at least 8 of every 9).
                float turn_o = 0.0f;                           // O is multiplied with 2^turn_o
                const bool raised = top > m + 8.0f;
                if (raised) {
                    const float fall = m - top;                // m = -inf: nothing was summed
                    const int e_new = max(e_o + (int)ceilf(fmaxf(fall, -1000.0f)), kLeastPower);
                    l *= rows_exp2(fall);
                    turn_o = fall + (float)(e_o - e_new);
                    e_o = e_new;
                    m = top;
                }
                const float base_m = m == -INFINITY ? 0.0f : m;
                // ---- E: a value's power of two times 2^8, the largest probability, must not leave fp16 ----
                if (__any_sync(kFullMask, v_most * rows_power(-e_o) > 64.0f)) {
                    float heavy = usual ? rows_exp2(own - base_m) : 0.0f;
#pragma unroll 1
                    for (int c0 = usual ? HALF : 0; c0 < HALF; c0 += CHUNK) {
                        if (HALF > CHUNK) load_logits(c0, x);
#pragma unroll
                        for (int j = 0; j < CHUNK; ++j) heavy = fmaxf(heavy, rows_exp2(fmaf(x[j], by, -base_m)) * meta.v_up[i & 7][side * HALF + c0 + j]);
                    }
                    swap(heavy, other);
                    heavy = fmaxf(heavy, other);
                    const int e_new = min(rows_exponent(heavy) - 3, 119);                    // the row's largest p' below 16
                    if (e_new > e_o && (heavy * rows_power(-e_o) > 16384.0f || raised || e_o == kLeastPower)) {
                        turn_o += (float)(e_o - e_new);
                        e_o = e_new;
                    }
                    far = __any_sync(kFullMask, e_o > 24);
                }
                // ---- probabilities, two to a column ----
                // The usual tile's come as 2^(x - m - E): all p' below 2^14, E is at most 24, so neither they nor their sum leave fp32's range. Elsewhere E may be
                // anything (values of 2^-126, or zeros, which have no say in it) and is taken apart from them.
                const float shift = usual ? base_m + (float)e_o : base_m;
                float sums[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 1
                for (int c0 = 0; c0 < HALF; c0 += CHUNK) {
                    uint32_t p[CHUNK / 2];
                    if (HALF > CHUNK) load_logits(c0, x);
                    if (odd) {
                        // a row that gives a token weight whose planes are not finite in a group becomes NaN there
#pragma unroll 1
                        for (int j = 0; j < CHUNK; ++j) {
                            const uint32_t bad = meta.bad[i & 7][side * HALF + c0 + j] & 0x7Fu;
                            if (bad) {
                                float z = -INFINITY;
#pragma unroll
                                for (int k = 0; k < CHUNK; ++k) z = k == j ? x[k] : z;
                                if (rows_exp2(fmaf(z, by, -base_m)) > 0.0f) poison |= bad;
                            }
                        }
                    }
#pragma unroll
                    for (int j = 0; j < CHUNK; ++j) {
                        x[j] = rows_exp2(fmaf(x[j], by, -shift));
                        sums[j % 4] += x[j];
                    }
                    if (!usual) {
                        const float down = rows_power(-e_o);
#pragma unroll
                        for (int j = 0; j < CHUNK; j += 4) {
                            const float4 up = *reinterpret_cast<const float4*>(&meta.v_up[i & 7][side * HALF + c0 + j]);
                            x[j] = x[j] * up.x * down; x[j + 1] = x[j + 1] * up.y * down; x[j + 2] = x[j + 2] * up.z * down; x[j + 3] = x[j + 3] * up.w * down;
                        }
                    }
#pragma unroll
                    for (int j = 0; j < CHUNK; j += 2) p[j / 2] = rows_half2(x[j], x[j + 1]);
                    tiles_st(lanes + S::COL_P + st * (TILE / 2) + (side * HALF + c0) / 2, p);
                }
                l = fmaf((sums[0] + sums[1]) + (sums[2] + sums[3]), usual ? rows_power(e_o) : 1.0f, l);
                // ---- O, when m or E moved: half of its columns ----
                if (i > begin_i && __any_sync(kFullMask, turn_o != 0.0f)) {
                    const float alpha = rows_exp2(turn_o);
                    ok = wait(o_done(i - 1), two(i - 1)) && ok;
                    tiles_fence_after();
#pragma unroll 1
                    for (int c = side * (S::DV / 2); c < (int)(side + 1) * (S::DV / 2); c += 32) {
                        uint32_t o[32];
                        tiles_ld(lanes + S::COL_O + c, o);
                        tiles_wait_ld();
#pragma unroll
                        for (int j = 0; j < 32; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * alpha);
                        tiles_st(lanes + S::COL_O + c, o);
                    }
                }
                tiles_wait_st();
                tiles_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(p_full(i));
            }
            // ---- the segment's result ----
            float other;
            swap(l, other);
            l += other;
            swap(__uint_as_float(poison), other);
            poison |= __float_as_uint(other);
            ok = wait(o_done(i - 1), two(i - 1)) && ok;
            tiles_fence_after();
            float* part = a.partial + (size_t)(2 * blockIdx.x + (from_start ? 1 : 0)) * MT * (S::DV + 3);
            if (!whole && is && side == 0) {
                part[r] = m;
                part[MT + r] = l;
                part[2 * MT + r] = (float)e_o;
            }
            const float inv = whole ? (l == 0.0f ? 0.0f : rows_power(e_o) / l) : 1.0f;
            uint16_t* dst = a.out + (size_t)(now.seq.row0 + node) * a.out_stride + (size_t)(head * a.group + flat % a.group) * D + now.head % S::PARTS * S::DV;
            float* pdst = part + 3 * MT + (size_t)r * S::DV;
#pragma unroll 1
            for (int c = side * (S::DV / 2); c < (int)(side + 1) * (S::DV / 2); c += 32) {
                uint32_t o[32];
                tiles_ld(lanes + S::COL_O + c, o);
                tiles_wait_ld();
                const float by = poison >> (c / 64) & 1u ? __int_as_float(0x7FC00000) : inv;
                if (is && ok) {
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
            if (i < count) tiles_next_unit<MT, TILE>(a, now);
        }
    }
    tiles_fence_before();
    __syncthreads();
    if (warp == S::WARPS - 1) {
        tiles_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"((uint32_t)S::COLS) : "memory");
    }
}

// Joins the shares of the unit that block c's share ends in: a warp per row, lanes over the elements. A second launch, which is on its way while the
// first one ends: it adds 3 us to the call.
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
    // A slot: [rows] maxima, sums in units of 2^m, exponents E, then [rows][DV] products in units of 2^(m + E).
    constexpr size_t kSlot = (size_t)MT * (DV + 3);
    auto slot = [&](uint32_t p) { return a.partial + (size_t)(p == 0 ? 2 * c + 1 : 2 * (c + p)) * kSlot; };
    float top = -INFINITY, high = -INFINITY;                   // the largest m and m + E
    for (uint32_t p = lane; p < parts; p += kWarp) {
        const float* s = slot(p);
        top = fmaxf(top, s[r]);
        high = fmaxf(high, s[r] + s[2 * MT + r]);
    }
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) {
        top = fmaxf(top, __shfl_xor_sync(kFullMask, top, off));
        high = fmaxf(high, __shfl_xor_sync(kFullMask, high, off));
    }
    if (top == -INFINITY) top = high = 0.0f;
    float sum = 0.0f, v[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) v[e] = 0.0f;
    for (uint32_t p0 = 0; p0 < parts; p0 += kWarp) {
        float w = 0.0f, l = 0.0f;
        if (p0 + lane < parts) {
            const float* s = slot(p0 + lane);
            w = rows_exp2(s[r] + s[2 * MT + r] - high);
            l = s[MT + r] * rows_exp2(s[r] - top);
        }
        const uint32_t n = min(parts - p0, (uint32_t)kWarp);
#pragma unroll 4
        for (uint32_t j = 0; j < n; ++j) {
            const float wj = __shfl_sync(kFullMask, w, j);
            const float* src = slot(p0 + j) + 3 * MT + (size_t)r * DV + lane * VEC;
            sum += __shfl_sync(kFullMask, l, j);
#pragma unroll
            for (int e = 0; e < VEC; e += 2) {
                const float2 x = *reinterpret_cast<const float2*>(src + e);
                v[e] = fmaf(wj, x.x, v[e]);
                v[e + 1] = fmaf(wj, x.y, v[e + 1]);
            }
        }
    }
    const float inv = sum == 0.0f ? 0.0f : rows_exp2(high - top) / sum;
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
    // Rows of one kv head in a mean sequence: units of eight read and unpack the cache once each, units of 128 once for all, but cost more to enter and leave,
    // so it takes more rows where there are many units; where there are few, many warps share one of eight, and joining their shares costs a few us per row.
    // Measured in us, eight / 128: 8 * 2 units of 4000 tokens with heads of 256, 4 rows: 48 / 36, 1 row: 34 / 36; 8 * 8 of 8000, 16 rows: 127 / 127, 24: 160 / 127;
    // 8 * 32 of 3000 with 4-bit heads of 128, 24 rows: 134 / 124, of 1800 on average, 28 rows: 84 / 110. Heads of 512 are two units each, whose tiles
    // are of 32 tokens: 2 * 32 units of 4000, 32 rows: 176 / 272, 48: 248 / 279. All of these are batches of like sequences. The mean goes by the call's rows,
    // padding included, and by all its sequences: single tokens beside a long prompt chunk all go by the one or the other, right but slower than apart.
    const uint64_t mean = ((uint64_t)a.rows + a.sequences - 1) / a.sequences * a.group, units = (uint64_t)a.sequences * a.kv_heads * (D == 512 ? 4 : 1);
    // In place heads of 512 have units of eight: a unit of 128 rows reads all of a row of q for half of its values, and the other half's unit may do so
    // later. Us beside / in place, 16 heads on 2: 200 trees of 5 rows over 40 tokens 84 / 80, 8 trees of 61 over 8000 532 / 1135, 333 rows over 8000 369 / 901.
    if (mean <= (units <= 32 ? 4 : units <= 128 ? 16 : 32) || (D == 512 && a.out == a.q)) return bf16 ? launch_rows<D, BITS, 8, true>(ctx, st, a, ws) : launch_rows<D, BITS, 8, false>(ctx, st, a, ws);
    return bf16 ? launch_tiles<D, BITS, true>(ctx, st, a, ws) : launch_tiles<D, BITS, false>(ctx, st, a, ws);
}

}  // namespace tf
