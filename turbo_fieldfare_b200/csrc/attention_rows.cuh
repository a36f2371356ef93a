// Attention over the quantised, paged cache for units of at most eight rows: decode steps and small trees.
//
// What bounds it is HBM: a cached token's codes and planes are read once and used for a handful of rows. So everything that is not
// unpacking is kept out of the way. A worker is one warp: it owns its share of the tiles (16 tokens each), its ring of stages, filled by its own
// cp.async, its running maximum, sum and product; no thread block meets at a barrier after the start, and the shares of a unit are joined
// by the worker that is the last to leave one (rows_join), in the workers' order, which is a property of the lengths alone.
//
// Logits, S^T[token][row] = K Q^T (mma.sync m16n8k16, tokens as A, rows as B): an 8-bit code c enters as the fp16 subnormal c * 2^-24 (one PRMT
// per two codes), a 4-bit one as c * 2^-24 or, against a q pre-scaled by 1/16, c * 2^-20 (one AND). Scale and bias come in fp32 per
// group: s (q . c) + b sum(q). An 8x8 transpose of the logits (movmatrix on their halves, exact) gives a lane row g and the tokens
// 2t, 2t + 1, which is the B fragment of the second product,
// O^T[element][row] = V^T P^T, with V's codes as A, again as subnormals: the value scale goes into the probability, p' = p s 2^-E rounded to
// fp16, and what the bias adds is summed in fp32. The rounding of p' shall weigh a code's distance from the centre of the codes, not the code
// itself: sum p' (c - centre) = sum p' c - centre sum p', with sum p' of all groups by one more MMA each into the rows of a common
// accumulator, against sum p (b + centre s). (The tensor cores line a subnormal up as if it were fp16's least normal number: a sum of
// 4-bit codes is good to 2^-16 of sum p |b|, which shows only in outputs that are a small remainder of it.) E is a row's own, after the largest
// p s so far (tokens that it does not see have p = 0 and no say; when m is raised, those before lose theirs), and m a maximum that is raised
// only when a logit exceeds it by 8: one vote per tile, and what was summed is rescaled only when one of them moves.
//
// What it measured, 8-bit heads of 256 on 8 kv heads, two rows each: 64 sequences of up to 4096 tokens 130 us, 4.9 TB/s; 131000 tokens of one sequence, heads of
// 128: 75 us, 3.7 TB/s; 4-bit heads of 512, 200 sequences of up to 8192 tokens, eight rows per kv head: 310 us, 3.6 TB/s, bound by unpacking (2200 clocks a
// tile with two warps to a scheduler). The same with blocks that share tiles behind barriers: 268, 178, 768 us. Units of 16 rows, which would unpack half as
// often, need so many registers that a third of the warps goes: no faster at 28 rows.
#pragma once

#include "attention_launch.cuh"
#include "mma_gemv.cuh"

#include <type_traits>

namespace tf {

constexpr int kRowsTile = 16;                                  // tokens: a tile never straddles two pages
constexpr int kLeastPower = -118;                              // of E: 2^-E times a probability, 2^8 at most, stays in fp32's range where a value scale is zero

template <int D, int BITS, int RB>
struct RowsShape {
    // A head of 512 is shared by two warps, which have half of its elements each (DW) and add their logits.
    static constexpr int DW = D < 256 ? D : 256, SPLIT = D / DW, G = DW / 64, GROUPS = D / 64;
    static constexpr int ROW = DW * BITS / 8, ROW_BYTES = D * BITS / 8, PIECES = ROW / 16, NR = RB / 8;      // of a warp's part, and of the cache's row
    static constexpr int CODES = kRowsTile * ROW, PLANE = kRowsTile * G * 2, STAGE = 2 * CODES + 4 * PLANE;
    static constexpr int WARPS = 4, WORKERS = WARPS / SPLIT, BLOCKS = D >= 256 ? 2 : 3;
    static constexpr int THREADS = WARPS * kWarp;
    static constexpr int SWAP = SPLIT > 1 ? 2 * WARPS * kWarp * NR * 16 : 0;                       // logits of the other warp, by turns in two buffers
    static constexpr int FIT = (227 * 1024 / BLOCKS - 1024 - 256 - SWAP) / (WARPS * STAGE), STAGES = FIT > 8 ? 8 : FIT;
    static constexpr int SMEM = WARPS * STAGES * STAGE + SWAP;
    static_assert(STAGES >= 2 && STAGE % 128 == 0, "a ring needs two stages");
    // 16-byte pieces are moved within their 128-byte lines so that the reads of a quarter or half warp meet every bank once
    static __host__ __device__ __forceinline__ uint32_t k_at(uint32_t row, uint32_t byte) {
        uint32_t at = row * ROW + byte;
        if constexpr (BITS == 8) { if constexpr (ROW >= 128) at ^= (row & 1u) << 6; }
        else if constexpr (ROW >= 128) at ^= (row & 3u) << 5;
        else if constexpr (ROW == 64) at ^= ((row >> 1) & 1u) << 5;
        return at;
    }
    static __host__ __device__ __forceinline__ uint32_t v_at(uint32_t row, uint32_t byte) { return (row * ROW + byte) ^ (((row >> 1) & 3u) << 5); }
};

__device__ __forceinline__ void rows_cp_async(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void rows_cp_async_8(uint32_t dst, const void* src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void rows_mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// The first product of a chain.
__device__ __forceinline__ void rows_mma_first(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                 : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}
__device__ __forceinline__ float rows_exp2(float x) {          // 2^x; results below fp32's normal range are zero
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float rows_max_nan(float a, float b) {      // a NaN stays
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
}
__device__ __forceinline__ uint32_t rows_half2(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t rows_mul2(uint32_t a, uint32_t b) {
    const __half2 r = __hmul2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
}
template <bool BF16>
__device__ __forceinline__ uint32_t rows_pair(float lo, float hi) {
    if constexpr (BF16) {
        const __nv_bfloat162 b = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&b);
    } else {
        return rows_half2(lo, hi);
    }
}
__device__ __forceinline__ int rows_exponent(float v) { return max(-126, min((int)((__float_as_uint(v) >> 23) & 255u) - 127, 126)); }
__device__ __forceinline__ float rows_power(int e) { return __uint_as_float((uint32_t)(max(-126, min(e, 127)) + 127) << 23); }

// bf16 values of one token's G groups.
template <int G>
struct TokenPlane {
    uint32_t w[G / 2 + (G == 1)];
    __device__ __forceinline__ void load(const uint8_t* plane, int token) {
        const uint8_t* p = plane + token * (2 * G);
        if constexpr (G == 1) w[0] = *reinterpret_cast<const uint16_t*>(p);
        else if constexpr (G == 2) w[0] = *reinterpret_cast<const uint32_t*>(p);
        else { const uint2 v = *reinterpret_cast<const uint2*>(p); w[0] = v.x; w[1] = v.y; }
    }
    __device__ __forceinline__ float at(int grp) const { return __uint_as_float(grp % 2 ? w[grp / 2] & 0xFFFF0000u : w[grp / 2] << 16); }
};

// bf16 values of two neighbouring tokens (2i, then 2i + 1) in G groups. G = 1: one word holds both.
template <int G>
struct PlanePair {
    uint32_t w[G];
    __device__ __forceinline__ void load(const uint8_t* plane, int pair) {
        const uint8_t* p = plane + pair * (4 * G);
        if constexpr (G == 1) w[0] = *reinterpret_cast<const uint32_t*>(p);
        else if constexpr (G == 2) { const uint2 v = *reinterpret_cast<const uint2*>(p); w[0] = v.x; w[1] = v.y; }
        else { const uint4 v = *reinterpret_cast<const uint4*>(p); w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w; }
    }
    __device__ __forceinline__ float at(int token, int grp) const {
        const int i = token * G + grp;
        return __uint_as_float(i % 2 ? w[i / 2] & 0xFFFF0000u : w[i / 2] << 16);
    }
    __device__ __forceinline__ void raise_all(__nv_bfloat162& most) const {
#pragma unroll
        for (int i = 0; i < G; ++i) most = __hmax2_nan(most, __habs2(*reinterpret_cast<const __nv_bfloat162*>(&w[i])));
    }
    // The largest magnitudes of either token so far, in both halves of its word (G = 1: both tokens' in the first word); a NaN stays.
    __device__ __forceinline__ void raise(__nv_bfloat162& most0, __nv_bfloat162& most1) const {
        auto word = [&](int i) { return __habs2(*reinterpret_cast<const __nv_bfloat162*>(&w[i])); };
        if constexpr (G == 1) {
            most0 = __hmax2_nan(most0, word(0));
        } else {
            __nv_bfloat162 a = word(0), b = word(G / 2);
            if constexpr (G == 4) { a = __hmax2_nan(a, word(1)); b = __hmax2_nan(b, word(3)); }
            most0 = __hmax2_nan(most0, __hmax2_nan(a, __lowhigh2highlow(a)));
            most1 = __hmax2_nan(most1, __hmax2_nan(b, __lowhigh2highlow(b)));
        }
    }
};

// Zeros in the place of value planes that are not finite; bit key * G + grp: it was so at the lane's token `key` (2t, 2t + 1, 2t + 8, 2t + 9).
template <int G>
__device__ __noinline__ uint32_t rows_sanitise(uint8_t* scales, int plane_bytes, int t) {
    uint16_t *vs = reinterpret_cast<uint16_t*>(scales), *vb = reinterpret_cast<uint16_t*>(scales + plane_bytes);
    uint32_t flags = 0;
    for (int i = 0; i < 4 * G; ++i) {
        const int at = (2 * t + (i / G & 1) + (i / G & 2) * 4) * G + i % G;
        if ((vs[at] & 0x7F80) == 0x7F80 || (vb[at] & 0x7F80) == 0x7F80) flags |= 1u << i;
    }
    __syncwarp();                                              // all lanes have seen them
    for (int i = 0; i < 4 * G; ++i)
        if (flags >> i & 1u) {
            const int at = (2 * t + (i / G & 1) + (i / G & 2) * 4) * G + i % G;
            vs[at] = vb[at] = 0;                               // the lanes of a column write the same
        }
    __syncwarp();
    return flags;
}

// Joins the shares of a unit, sixteen at a time: the worker that is the last to leave its share of a group joins the group, in the order of the
// shares, into the place of its first, and goes on as that group's worker among the groups. Tickets are back at zero when their
// group is joined. Share 0 lies in worker c0's second slot, share i in worker c0 + i's first; a slot is [rows] maxima, [rows] sums and
// [rows][DW] products of each of the SPLIT parts of the head's elements, which are joined apart.
template <int D, int DW, int RB, bool BF16>
__device__ __noinline__ void rows_join(const AttnArgs& a, uint32_t row0, uint32_t head, uint32_t flat0, uint32_t c0, uint32_t i, uint32_t parts, uint32_t valid,
                                       uint32_t half, int lane) {
    // Loops that are short in code: a block runs them once or twice, and what is not in the instruction cache yet costs more than the work.
    constexpr int VEC = DW / 32, SPLIT = D / DW, BATCH = VEC == 8 ? 8 : 16;
    constexpr uint32_t kSlot = RB * (DW + 2);
    using Vec = std::conditional_t<VEC == 2, float2, float4>;
    constexpr int VECS = VEC / (sizeof(Vec) / 4);
    auto place = [&](uint32_t p) { return (p == 0 ? 2 * c0 + 1 : 2 * (c0 + p)) * SPLIT + half; };
    uint32_t span = 1;
#pragma unroll 1
    for (uint32_t* tickets = a.tickets; parts > 1; tickets += a.ticket_stride, span *= kJoin) {
        const uint32_t group = i / kJoin, base = group * kJoin, members = min((uint32_t)kJoin, parts - base);
        uint32_t* ticket = tickets + place(base * span);
        __syncwarp();                                          // this worker's share, or the group that it joined, before its ticket
        uint32_t old = 0;
        if (lane == 0) asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(old) : "l"(ticket) : "memory");
        if (__shfl_sync(kFullMask, old, 0) != members - 1) return;
        __syncwarp();                                          // what the others left, after their tickets
        if (lane == 0) *ticket = 0;
        const bool final = parts <= kJoin, is = (uint32_t)lane < members;
        float* first = a.partial + (size_t)place(base * span) * kSlot;
        const float* mine = a.partial + (size_t)place((base + (is ? lane : 0)) * span) * kSlot;
#pragma unroll 1
        for (uint32_t r = 0; r < valid; ++r) {
            // past L1, which may hold a slot as it was before
            const float mp = is ? __ldcg(mine + r) : -INFINITY, lp = is ? __ldcg(mine + RB + r) : 0.0f;
            float w = 0.0f, v[VEC], top = mp, sum = 0.0f;
#pragma unroll
            for (int e = 0; e < VEC; ++e) v[e] = 0.0f;
#pragma unroll 1
            for (uint32_t p0 = 0; p0 < members; p0 += BATCH) {
                Vec x[BATCH][VECS];
#pragma unroll
                for (int k = 0; k < BATCH; ++k) {
                    const Vec* src = reinterpret_cast<const Vec*>(a.partial + (size_t)place((base + min(p0 + k, members - 1)) * span) * kSlot + 2 * RB + r * DW + lane * VEC);
#pragma unroll
                    for (int e = 0; e < VECS; ++e) x[k][e] = __ldcg(src + e);
                }
                if (p0 == 0) {
#pragma unroll
                    for (int off = kJoin / 2; off >= 1; off >>= 1) top = fmaxf(top, __shfl_xor_sync(kFullMask, top, off));
                    top = __shfl_sync(kFullMask, top, 0);
                    w = is ? rows_exp2(mp - (top == -INFINITY ? 0.0f : top)) : 0.0f;
                    sum = w * lp;
#pragma unroll
                    for (int off = kJoin / 2; off >= 1; off >>= 1) sum += __shfl_xor_sync(kFullMask, sum, off);
                    sum = __shfl_sync(kFullMask, sum, 0);
                }
#pragma unroll
                for (int k = 0; k < BATCH; ++k) {
                    // a slot behind the last one counts for nothing, whatever it holds
                    const float wk = __shfl_sync(kFullMask, w, (p0 + k) & 31);
#pragma unroll
                    for (int e = 0; e < VEC; ++e) v[e] = p0 + k < members ? fmaf(wk, reinterpret_cast<const float*>(x[k])[e], v[e]) : v[e];
                }
            }
            if (final) {
                const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
                const uint32_t flat = flat0 + r;
                uint16_t* dst = a.out + (size_t)(row0 + flat / a.group) * a.out_stride + (size_t)(head * a.group + flat % a.group) * D + half * DW + lane * VEC;
#pragma unroll
                for (int e = 0; e < VEC; e += 2) *reinterpret_cast<uint32_t*>(dst + e) = rows_pair<BF16>(v[e] * inv, v[e + 1] * inv);
            } else {
                if (lane == 0) {
                    first[r] = top;
                    first[RB + r] = sum;
                }
#pragma unroll
                for (int e = 0; e < VEC; e += 2) *reinterpret_cast<float2*>(first + 2 * RB + r * DW + lane * VEC + e) = make_float2(v[e], v[e + 1]);
            }
        }
        parts = (parts + kJoin - 1) / kJoin;
        i = group;
    }
}

// A worker's share, found by a whole warp that goes over the sequences 32 at a time, first for the total, then for the place. False: there are fewer
// tiles than workers. One body for both turns: what a block runs once costs what it takes to fetch its instructions.
template <int MT, int TILE>
__device__ __forceinline__ bool find_share(const AttnArgs& a, uint32_t worker, uint32_t workers_most, int lane, bool report, Cursor<MT, TILE>& now, Shares& shares,
                                           uint64_t& item, uint64_t& stop) {
    shares.total = 0;
    item = stop = 0;
    uint64_t before = 0;
    bool placing = false;
#pragma unroll 1
    for (uint32_t b0 = 0;;) {
        Sequence s = {};
        uint64_t mine = 0;
        if (b0 + lane < a.sequences) {
            s.load(a, b0 + lane, report && !placing);
            mine = sequence_tiles<MT, TILE>(a, s) * a.kv_heads * a.head_parts;
        }
        uint64_t upto = mine;
#pragma unroll 1
        for (int off = 1; off < kWarp; off <<= 1) {
            const uint64_t o = __shfl_up_sync(kFullMask, upto, off);
            if (lane >= off) upto += o;
        }
        const uint64_t all = __shfl_sync(kFullMask, upto, kWarp - 1);
        if (placing && item < before + all) {
            const int owner = __ffs(__ballot_sync(kFullMask, before + upto > item)) - 1;
            const uint64_t left = item - before - __shfl_sync(kFullMask, upto - mine, owner);
            now.b = b0 + owner;
            now.seq.row0 = __shfl_sync(kFullMask, s.row0, owner);
            now.seq.rows = __shfl_sync(kFullMask, s.rows, owner);
            now.seq.context = __shfl_sync(kFullMask, s.context, owner);
            uint32_t place[3];
            place_in_sequence<MT, TILE>(a, now.seq, left, place);
            now.head = place[0]; now.flat0 = place[1]; now.tile = place[2];
            now.range.set(a, now.seq, now.flat0, MT, TILE);
            return true;
        }
        before += all;
        b0 += kWarp;
        if (b0 >= a.sequences) {                               // the second time this is not reached: item is below the total
            shares.set(before, workers_most);
            if (worker >= shares.workers) return false;
            item = shares.begin(worker);
            stop = shares.begin(worker + 1);
            before = 0;
            b0 = 0;
            placing = true;
        }
    }
}

template <int RB>
__device__ __noinline__ void rows_next_unit(const AttnArgs& a, Cursor<RB, kRowsTile>& c) { c.next_unit(a); }

// 8x8 transpose over a warp of fp32 values, exact: lane (g, t) gives elements (g, 2t) and (g, 2t + 1) and gets (2t, g) and (2t + 1, g).
__device__ __forceinline__ void rows_transpose(float& x0, float& x1) {
    uint32_t lo = gm_prmt(__float_as_uint(x0), __float_as_uint(x1), 0x5410), hi = gm_prmt(__float_as_uint(x0), __float_as_uint(x1), 0x7632);
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %0;" : "+r"(lo));
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %0;" : "+r"(hi));
    x0 = __uint_as_float(gm_prmt(lo, hi, 0x5410));
    x1 = __uint_as_float(gm_prmt(lo, hi, 0x7632));
}

template <int D, int BITS, int RB, bool BF16>
__global__ void __launch_bounds__(RowsShape<D, BITS, RB>::THREADS, RowsShape<D, BITS, RB>::BLOCKS)
attention_rows_kernel(const __grid_constant__ AttnArgs a) {
    using S = RowsShape<D, BITS, RB>;
    constexpr int G = S::G, NR = S::NR, W = S::WARPS;
    constexpr float kCentre = BITS == 8 ? 128.0f : 8.0f;
    extern __shared__ __align__(128) uint8_t smem[];
    const int tid = threadIdx.x, warp = tid / kWarp, lane = tid % kWarp, g = lane / 4, t = lane % 4;
    const uint32_t half = warp % S::SPLIT, worker = blockIdx.x * S::WORKERS + warp / S::SPLIT;

    Cursor<RB, kRowsTile> now;
    Shares shares;
    uint64_t item, stop;
    if (!find_share<RB, kRowsTile>(a, worker, gridDim.x * S::WORKERS, lane, blockIdx.x == 0, now, shares, item, stop)) return;

    // ---- this warp's ring: what the next request needs is in registers, the rest of its cursor in memory ----
    uint8_t* ring = smem + warp * (S::STAGES * S::STAGE);
    const uint32_t ring_addr = (uint32_t)__cvta_generic_to_shared(ring);
    float4* swap = reinterpret_cast<float4*>(smem + W * S::STAGES * S::STAGE);       // [2][warps][NR][lanes]
    uint32_t turn = 0;
    Cursor<RB, kRowsTile> next = now;
    uint32_t ahead = (uint32_t)(stop - item);                  // tiles not requested yet
    uint32_t there = 0;                                        // a bit per stage: its tile has a page
    uint32_t next_left, next_token, next_end, next_head;
    const int32_t* next_table;
    int32_t next_page;
    auto look_up = [&] {
        next_page = -1;
        if (next_token < next_end) {                           // (the table is read once per page)
            const int32_t p = next_table[next_token >> a.table.page_log2];
            if (p >= 0 && (uint32_t)p < a.table.pages) next_page = p;
        }
    };
    auto enter_unit = [&] {
        next_left = next.range.tiles - next.tile;
        next_token = next.token0();
        next_end = next.range.end;
        next_head = next.head;
        next_table = a.table.table + (size_t)next.b * a.table.stride;
        look_up();
    };
    const uint32_t k_dst = S::k_at(lane / S::PIECES, lane % S::PIECES * 16), v_dst = S::CODES + S::v_at(lane / S::PIECES, lane % S::PIECES * 16);
    auto request = [&](uint32_t stage) {
        there &= ~(1u << stage);
        if (next_page >= 0) {
            there |= 1u << stage;
            const size_t row = (((size_t)next_page * a.kv_heads + next_head) << a.table.page_log2) + (next_token & ((1u << a.table.page_log2) - 1u));
            const uint32_t base = ring_addr + stage * S::STAGE;
            const size_t from = (row + lane / S::PIECES) * S::ROW_BYTES + half * S::ROW + lane % S::PIECES * 16;
            const uint8_t *kc = a.k.codes + from, *vc = a.v.codes + from;
#pragma unroll
            for (int i = 0; i < kRowsTile * S::PIECES / kWarp; ++i) {
                // rows `first` and on of the tile: their swizzle on top of the lane's own
                const uint32_t first = i * kWarp / S::PIECES, src = first * S::ROW_BYTES, k_more = S::k_at(first, 0) ^ (first * S::ROW), v_more = S::v_at(first, 0) ^ (first * S::ROW);
                rows_cp_async(((base + k_dst) ^ k_more) + i * 512, kc + src);
                rows_cp_async(((base + v_dst) ^ v_more) + i * 512, vc + src);
            }
            if constexpr (S::SPLIT > 1) {
                // planes: eight bytes of a token each
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const uint32_t id = lane + i * kWarp, plane = id / kRowsTile, token = id % kRowsTile;
                    const uint16_t* src = plane == 0 ? a.k.scales : plane == 1 ? a.k.biases : plane == 2 ? a.v.scales : a.v.biases;
                    rows_cp_async_8(base + 2 * S::CODES + id * 8, src + (row + token) * S::GROUPS + half * S::G);
                }
            } else if (8 * G == kWarp || lane < 8 * G) {
                // planes: 2 G pieces each
                const uint32_t plane = lane / (2 * G), c = lane % (2 * G);
                const uint16_t* src = plane == 0 ? a.k.scales : plane == 1 ? a.k.biases : plane == 2 ? a.v.scales : a.v.biases;
                rows_cp_async(base + 2 * S::CODES + lane * 16, src + row * G + c * 8);
            }
        }
        if (--ahead) {
            if (--next_left) {
                next_token += kRowsTile;
                if ((next_token & ((1u << a.table.page_log2) - 1u)) == 0 || next_token >= next_end) look_up();
            } else {
                rows_next_unit(a, next);
                enter_unit();
            }
        }
    };
    enter_unit();
#pragma unroll 1
    for (int i = 0; i < S::STAGES - 1; ++i) {
        if (ahead) request(i);
        asm volatile("cp.async.commit_group;" ::: "memory");
    }

    // ---- where this lane reads: codes of tokens g and g + 8 (K), of tokens 2t, 2t + 1, 2t + 8, 2t + 9 (V) ----
    constexpr int KB = BITS * 8, KV = 128 / KB < G ? 128 / KB : G;           // bytes of a group; groups whose swizzles differ
    uint32_t k_off[KV], v_off[KV];
#pragma unroll
    for (int i = 0; i < KV; ++i) {
        k_off[i] = S::k_at(g, i * KB + t * (BITS * 2));
        v_off[i] = S::CODES + S::v_at(2 * t, i * KB + g * BITS);
    }

    uint32_t stage = 0;
    while (item < stop) {
        // ---- a unit's segment: the rows of q as B fragments, their sums per group, what they see ----
        const uint32_t valid = lesser((uint32_t)RB, now.flat_rows(a) - now.flat0);
        const uint32_t first_tile = now.tile;
        const uint32_t segment = (uint32_t)lesser((uint64_t)(now.range.tiles - first_tile), stop - item);
        const bool from_start = first_tile == 0, whole = from_start && segment == now.range.tiles;
        uint32_t qf[NR][4 * G][2];
        float q_sum[NR][G][2], factor[NR], m[NR], l[NR], b_sum[NR][G];       // q_sum: of rows 2t and 2t + 1; the others: of row g
        int32_t low[NR];                                       // first token that the row sees, from the unit's first tile on
        uint32_t node[NR];
        int32_t low_most = 0;
#pragma unroll
        for (int n = 0; n < NR; ++n) {
            const uint32_t r = g + 8 * n, flat = now.flat0 + r;
            const bool is = r < valid;
            node[n] = is ? flat / a.group : 0;
            const uint16_t* src = a.q + (size_t)(now.seq.row0 + node[n]) * a.q_stride + (size_t)(now.head * a.group + (is ? flat % a.group : 0)) * D + half * S::DW + 16 * t;
            // Sixteen elements of each group: as fp16 they are the fragments of four steps, but for 4-bit codes, whose order within eight elements is
            // (0, 4, 1, 5, 2, 6, 3, 7) and whose odd ones come sixteenfold. The row is brought to one range by a power of two, its largest
            // element to [128, 256), where fp16 rows do not have it (8-bit codes) or as far as fp16 has the power.
            uint32_t raw[G][8];
#pragma unroll
            for (int grp = 0; grp < G; ++grp) {
                const uint4 lo = is ? *reinterpret_cast<const uint4*>(src + grp * 64) : make_uint4(0, 0, 0, 0);
                const uint4 hi = is ? *reinterpret_cast<const uint4*>(src + grp * 64 + 8) : make_uint4(0, 0, 0, 0);
                raw[grp][0] = lo.x; raw[grp][1] = lo.y; raw[grp][2] = lo.z; raw[grp][3] = lo.w;
                raw[grp][4] = hi.x; raw[grp][5] = hi.y; raw[grp][6] = hi.z; raw[grp][7] = hi.w;
            }
            int e = 0;
            if constexpr (BF16 || BITS == 4) {
                uint32_t most = 0;                             // magnitudes order as their bits do
#pragma unroll
                for (int grp = 0; grp < G; ++grp)
#pragma unroll
                    for (int i = 0; i < 8; ++i) most = __vmaxu2(most, raw[grp][i] & 0x7FFF7FFFu);
                most = max(most & 0xFFFFu, most >> 16);
                most = max(most, __shfl_xor_sync(kFullMask, most, 1));
                most = max(most, __shfl_xor_sync(kFullMask, most, 2));
                const float top = BF16 ? bf16_bits_to_float((uint16_t)most) : f16_bits_to_float((uint16_t)most);
                if (top > 0.0f && top <= 3.402823466e38f) e = BF16 ? max(rows_exponent(top) - 7, -126) : min(max(rows_exponent(top) - 7, -15), 15);
                const float down = rows_power(-e);
#pragma unroll
                for (int grp = 0; grp < G; ++grp)
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        if constexpr (BF16) raw[grp][i] = rows_half2(__uint_as_float(raw[grp][i] << 16) * down, __uint_as_float(raw[grp][i] & 0xFFFF0000u) * down);
                        else raw[grp][i] = rows_mul2(raw[grp][i], rows_half2(down, down));
                    }
            }
#pragma unroll
            for (int grp = 0; grp < G; ++grp) {
                float sum[4];
#pragma unroll
                for (int ks = 0; ks < 4; ++ks) {
                    uint32_t lo = raw[grp][2 * ks], hi = raw[grp][2 * ks + 1];
                    if constexpr (BITS == 4) {
                        const uint32_t u = raw[grp][4 * (ks / 2) + ks % 2], v = raw[grp][4 * (ks / 2) + ks % 2 + 2];       // elements (j, j + 1) and (j + 4, j + 5)
                        lo = gm_prmt(u, v, 0x5410);
                        hi = gm_sixteenth(gm_prmt(u, v, 0x7632));
                    }
                    qf[n][grp * 4 + ks][0] = lo;
                    qf[n][grp * 4 + ks][1] = hi;
                    // sums of the rows 2t and 2t + 1 by a product with ones (sixteens)
                    const uint32_t one = 0x3C003C00u, other = BITS == 4 ? 0x4C004C00u : one;
                    if (ks == 0) rows_mma_first(sum, one, one, other, other, lo, hi);
                    else rows_mma(sum, one, one, other, other, lo, hi);
                }
                q_sum[n][grp][0] = sum[0] * 5.9604644775390625e-8f;                  // 2^-24, as the products
                q_sum[n][grp][1] = sum[1] * 5.9604644775390625e-8f;
                b_sum[n][grp] = 0.0f;
            }
            factor[n] = a.scale * 1.4426950408889634f * rows_power(e) * 16777216.0f;      // in this order rows of 2^127 have one too, where the scale is as small
            m[n] = -INFINITY;
            l[n] = 0.0f;
            low[n] = 0;
            if (a.window && is) {
                const int64_t pos = a.mask ? max((int64_t)a.positions[now.seq.row0 + node[n]], (int64_t)now.seq.context) : (int64_t)now.seq.context + node[n];
                const int64_t first = pos - (int64_t)a.window + 1 - (int64_t)now.range.tile0 * kRowsTile;
                low[n] = (int32_t)max((int64_t)0, lesser(first, (int64_t)0x7FFFFFFF));
            }
            low_most = max(low_most, low[n]);
        }
        if (a.window) low_most = (int32_t)__reduce_max_sync(kFullMask, (uint32_t)low_most);
        float o[NR][G][4][4], ones[NR][4];                     // ones: sums of the rounded p', row grp for group grp
        float e_real[NR];                                      // E, the exponent that the row's products p s are divided by, not rounded up, and 2^-E
        float down_v[NR];
#pragma unroll
        for (int n = 0; n < NR; ++n) {
            ones[n][0] = ones[n][1] = ones[n][2] = ones[n][3] = 0.0f;
            e_real[n] = kLeastPower;
            down_v[n] = rows_power(-kLeastPower);
#pragma unroll
            for (int grp = 0; grp < G; ++grp)
#pragma unroll
                for (int j = 0; j < 4; ++j) o[n][grp][j][0] = o[n][grp][j][1] = o[n][grp][j][2] = o[n][grp][j][3] = 0.0f;
        }
        // From the unit's first tile on: tokens before open_end are cached ones; every row sees them from low_most on.
        const int32_t base_token = (int32_t)(now.range.tile0 * kRowsTile), open_end = (int32_t)lesser(now.seq.context, now.range.end) - base_token,
                      end_rel = (int32_t)now.range.end - base_token;
        int32_t rel0 = first_tile * kRowsTile;

#pragma unroll 1
        for (uint32_t left = segment; left; --left, rel0 += kRowsTile) {
            asm volatile("cp.async.wait_group %0;" ::"n"(S::STAGES - 2) : "memory");
            __syncwarp();
            const uint8_t* st = ring + stage * S::STAGE;

            // ---- logits: rows of the accumulator are tokens g and g + 8, columns the rows 2t and 2t + 1 of q ----
            float x[NR][4] = {};
            const uint8_t* planes = st + 2 * S::CODES;
            TokenPlane<G> ks_lo, ks_hi, kb_lo, kb_hi;
            ks_lo.load(planes, g); ks_hi.load(planes, g + 8);
            kb_lo.load(planes + S::PLANE, g); kb_hi.load(planes + S::PLANE, g + 8);
#pragma unroll
            for (int grp = 0; grp < G; ++grp) {
                uint32_t w[2][4];
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    const uint8_t* at = st + k_off[grp % KV] + grp / KV * 128 + n * 8 * S::ROW;
                    if constexpr (BITS == 8) {
                        const uint4 c = *reinterpret_cast<const uint4*>(at);
                        w[n][0] = c.x; w[n][1] = c.y; w[n][2] = c.z; w[n][3] = c.w;
                    } else {
                        const uint2 c = *reinterpret_cast<const uint2*>(at);
                        w[n][0] = c.x; w[n][1] = c.x >> 8; w[n][2] = c.y; w[n][3] = c.y >> 8;
                    }
                }
                float acc[NR][4];
#pragma unroll
                for (int ks = 0; ks < 4; ++ks) {
                    uint32_t a0, a1, a2, a3;
                    if constexpr (BITS == 8) {
                        a0 = gm_prmt(w[0][ks], 0, 0x4140); a1 = gm_prmt(w[1][ks], 0, 0x4140);
                        a2 = gm_prmt(w[0][ks], 0, 0x4342); a3 = gm_prmt(w[1][ks], 0, 0x4342);
                    } else {
                        a0 = w[0][ks] & 0x000F000Fu; a1 = w[1][ks] & 0x000F000Fu;
                        a2 = w[0][ks] & 0x00F000F0u; a3 = w[1][ks] & 0x00F000F0u;
                    }
#pragma unroll
                    for (int n = 0; n < NR; ++n) {
                        if (ks == 0) rows_mma_first(acc[n], a0, a1, a2, a3, qf[n][grp * 4][0], qf[n][grp * 4][1]);
                        else rows_mma(acc[n], a0, a1, a2, a3, qf[n][grp * 4 + ks][0], qf[n][grp * 4 + ks][1]);
                    }
                }
                const float s0 = ks_lo.at(grp), s1 = ks_hi.at(grp), b0 = kb_lo.at(grp), b1 = kb_hi.at(grp);
#pragma unroll
                for (int n = 0; n < NR; ++n) {
                    x[n][0] = fmaf(s0, acc[n][0], fmaf(b0, q_sum[n][grp][0], x[n][0]));
                    x[n][1] = fmaf(s0, acc[n][1], fmaf(b0, q_sum[n][grp][1], x[n][1]));
                    x[n][2] = fmaf(s1, acc[n][2], fmaf(b1, q_sum[n][grp][0], x[n][2]));
                    x[n][3] = fmaf(s1, acc[n][3], fmaf(b1, q_sum[n][grp][1], x[n][3]));
                }
            }
            // from here on a lane has row g (+ 8 n) and the tokens 2t, 2t + 1, 2t + 8, 2t + 9
#pragma unroll
            for (int n = 0; n < NR; ++n) {
                rows_transpose(x[n][0], x[n][1]);
                rows_transpose(x[n][2], x[n][3]);
#pragma unroll
                for (int c = 0; c < 4; ++c) x[n][c] *= factor[n];
            }
            if constexpr (S::SPLIT > 1) {
                float4* mine = swap + ((turn * W + warp) * NR) * kWarp + lane;
                const float4* other = swap + ((turn * W + (warp ^ 1)) * NR) * kWarp + lane;
#pragma unroll
                for (int n = 0; n < NR; ++n) mine[n * kWarp] = make_float4(x[n][0], x[n][1], x[n][2], x[n][3]);
                asm volatile("bar.sync %0, 64;" ::"r"(1 + warp / 2) : "memory");
#pragma unroll
                for (int n = 0; n < NR; ++n) {
                    const float4 y = other[n * kWarp];
                    x[n][0] += y.x; x[n][1] += y.y; x[n][2] += y.z; x[n][3] += y.w;
                }
                turn ^= 1;
            }
            if (!((there >> stage & 1u) && rel0 >= low_most && rel0 + kRowsTile <= open_end)) {
                const bool has_page = there >> stage & 1u;
                if (!has_page && lane == 0 && rel0 < end_rel) *a.error = kErrKvPage;
#pragma unroll
                for (int n = 0; n < NR; ++n) {
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        const int32_t rel = rel0 + 2 * t + (c & 1) + (c & 2) * 4;
                        bool seen = has_page && g + 8 * n < (int)valid && rel < end_rel;
                        if (seen) {
                            if (rel < open_end) {
                                seen = rel >= low[n];
                            } else {
                                const uint32_t j = (uint32_t)(base_token + rel) - now.seq.context;
                                if (a.mask) seen = (a.mask[(size_t)(now.seq.row0 + node[n]) * a.mask_words + (j >> 6)] >> (j & 63u)) & 1ull;
                                else seen = j <= node[n] && (!a.window || node[n] - j < a.window);
                            }
                        }
                        if (!seen) x[n][c] = -INFINITY;
                    }
                }
            }

            // ---- probabilities, at most 2^8 ----
            float p[NR][4], over = -INFINITY;
            auto raise_p = [&](int n) {
                const float base = m[n] == -INFINITY ? 0.0f : m[n];
#pragma unroll
                for (int c = 0; c < 4; ++c) p[n][c] = rows_exp2(x[n][c] - base);
            };
#pragma unroll
            for (int n = 0; n < NR; ++n) {
                over = fmaxf(over, fmaxf(fmaxf(x[n][0], x[n][1]), fmaxf(x[n][2], x[n][3])) - m[n]);
                raise_p(n);
            }

            // ---- does a maximum or a row's exponent move, is a value plane not finite? ----
            const uint8_t *vs_plane = planes + 2 * S::PLANE, *vb_plane = vs_plane + S::PLANE;
            PlanePair<G> vs_lo, vs_hi, vb_lo, vb_hi;
            auto load_value_planes = [&] {
                vs_lo.load(vs_plane, t); vs_hi.load(vs_plane, t + 4);
                vb_lo.load(vb_plane, t); vb_hi.load(vb_plane, t + 4);
            };
            const __nv_bfloat162 none = __float2bfloat162_rn(0.0f), finite = __halves2bfloat162(__ushort_as_bfloat16(0x7F7F), __ushort_as_bfloat16(0x7F7F));
            __nv_bfloat162 most_s[4] = {none, none, none, none}, most_b = none;     // per token; a NaN stays
            load_value_planes();
            vs_lo.raise(most_s[0], most_s[1]); vs_hi.raise(most_s[2], most_s[3]);
            vb_lo.raise_all(most_b); vb_hi.raise_all(most_b);
            bool moves = over > 8.0f || !__hble2(most_b, finite);
#pragma unroll
            for (int n = 0; n < NR; ++n) {
                float most = 0.0f;
#pragma unroll
                for (int key = 0; key < 4; ++key) {
                    const float s = G == 1 ? __uint_as_float((*reinterpret_cast<const uint32_t*>(&most_s[key & 2])) << (key & 1 ? 0 : 16) & 0xFFFF0000u)
                                               : __uint_as_float((*reinterpret_cast<const uint32_t*>(&most_s[key])) & 0xFFFF0000u);
                    most = rows_max_nan(most, p[n][key] * s);
                }
                moves |= !(most * down_v[n] < 16384.0f);
            }
            if (__any_sync(kFullMask, moves)) {
                // E, the power of what had weight so far, falls by as much as that weight when m is raised. It is rounded up from e_real, so that many rises add up.
                float fall[NR];
#pragma unroll
                for (int n = 0; n < NR; ++n) {
                    float top = fmaxf(fmaxf(x[n][0], x[n][1]), fmaxf(x[n][2], x[n][3]));
                    top = fmaxf(top, __shfl_xor_sync(kFullMask, top, 1));
                    top = fmaxf(top, __shfl_xor_sync(kFullMask, top, 2));
                    const float m_new = fmaxf(m[n], top);
                    fall[n] = m_new == -INFINITY ? 0.0f : m[n] - m_new;
                    const float alpha = rows_exp2(fall[n]);    // m = -inf: nothing was summed
                    m[n] = m_new;
                    l[n] *= alpha;
                    raise_p(n);
#pragma unroll
                    for (int grp = 0; grp < G; ++grp) b_sum[n][grp] *= alpha;
                }
                bool bad = !__hble2(most_b, finite);
#pragma unroll
                for (int key = 0; key < 4; ++key) bad |= !__hble2(most_s[key], finite);
                if (__any_sync(kFullMask, bad)) {
                    // Planes that are not finite become zeros in the stage, and a row whose probability there is not zero a NaN in that group.
                    const uint32_t flags = rows_sanitise<G>(ring + stage * S::STAGE + 2 * S::CODES + 2 * S::PLANE, S::PLANE, t);
#pragma unroll
                    for (int key = 0; key < 4; ++key)
#pragma unroll
                        for (int grp = 0; grp < G; ++grp)
#pragma unroll
                            for (int n = 0; n < NR; ++n)
                                if ((flags >> (key * G + grp) & 1u) && p[n][key] > 0.0f) b_sum[n][grp] = __int_as_float(0x7FC00000);
                    load_value_planes();
                }
#pragma unroll
                for (int n = 0; n < NR; ++n) {
                    float most = 0.0f;
#pragma unroll
                    for (int grp = 0; grp < G; ++grp)
#pragma unroll
                        for (int key = 0; key < 4; ++key)
                            most = fmaxf(most, p[n][key] * fabsf(key < 2 ? vs_lo.at(key, grp) : vs_hi.at(key - 2, grp)));      // a NaN of p leaves it as it is
                    most = fmaxf(most, __shfl_xor_sync(kFullMask, most, 1));
                    most = fmaxf(most, __shfl_xor_sync(kFullMask, most, 2));
                    const float e_old = ceilf(e_real[n]);
                    e_real[n] = fminf(fmaxf(fmaxf(e_real[n] + fall[n], (float)kLeastPower), (float)(rows_exponent(most) - 3)), 119.0f);      // p' below 16 now
                    const float e_new = ceilf(e_real[n]);
                    // what was summed of rows g + 8 n: their accumulators lie in the columns of other lanes
                    const float f = rows_exp2(fall[n] + (e_old - e_new));
                    const float f0 = __shfl_sync(kFullMask, f, 8 * t), f1 = __shfl_sync(kFullMask, f, 8 * t + 4);      // rows 2t, 2t + 1
                    ones[n][0] *= f0; ones[n][1] *= f1;
#pragma unroll
                    for (int grp = 0; grp < G; ++grp)
#pragma unroll
                        for (int j = 0; j < 4; ++j) { o[n][grp][j][0] *= f0; o[n][grp][j][1] *= f1; o[n][grp][j][2] *= f0; o[n][grp][j][3] *= f1; }
                    down_v[n] = rows_power(-(int)e_new);
                }
            }
            float pd[NR][4], pc[NR][4];
#pragma unroll
            for (int n = 0; n < NR; ++n)
#pragma unroll
                for (int key = 0; key < 4; ++key) {
                    pd[n][key] = p[n][key] * down_v[n];
                    pc[n][key] = p[n][key] * kCentre;
                    l[n] += p[n][key];
                }

            // ---- values ----
#pragma unroll
            for (int grp = 0; grp < G; ++grp) {
                uint32_t pb[NR][2];
                float s[4], b[4];
#pragma unroll
                for (int key = 0; key < 4; ++key) {
                    s[key] = key < 2 ? vs_lo.at(key, grp) : vs_hi.at(key - 2, grp);
                    b[key] = key < 2 ? vb_lo.at(key, grp) : vb_hi.at(key - 2, grp);
                }
#pragma unroll
                for (int n = 0; n < NR; ++n) {
                    pb[n][0] = rows_half2(pd[n][0] * s[0], pd[n][1] * s[1]);
                    pb[n][1] = rows_half2(pd[n][2] * s[2], pd[n][3] * s[3]);
#pragma unroll
                    for (int key = 0; key < 4; ++key) b_sum[n][grp] = fmaf(p[n][key], b[key], fmaf(pc[n][key], s[key], b_sum[n][grp]));
                    const uint32_t one = g == grp ? 0x3C003C00u : 0u;
                    rows_mma(ones[n], one, 0u, one, 0u, pb[n][0], pb[n][1]);
                }
                // A: rows g and g + 8 of m tile j are elements 8g + j and 8g + 4 + j of the group
                uint32_t av[4][4];
                const uint8_t* at = st + v_off[grp % KV] + grp / KV * 128;
                // token 2t + 1: with rows of less than 128 bytes the swizzle moves it the other way for some lanes
                const uint8_t* at1 = S::ROW >= 128 ? at + S::ROW : st + (v_off[grp % KV] ^ S::ROW) + grp / KV * 128;
                if constexpr (BITS == 8) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {               // tokens 2t, 2t + 1 and 2t + 8, 2t + 9
                        const uint2 wa = *reinterpret_cast<const uint2*>(at + h * 8 * S::ROW), wb = *reinterpret_cast<const uint2*>(at1 + h * 8 * S::ROW);
                        const uint32_t lo0 = gm_prmt(wa.x, wb.x, 0x5140), lo1 = gm_prmt(wa.x, wb.x, 0x7362), hi0 = gm_prmt(wa.y, wb.y, 0x5140), hi1 = gm_prmt(wa.y, wb.y, 0x7362);
                        av[0][2 * h] = gm_prmt(lo0, 0, 0x4140); av[0][2 * h + 1] = gm_prmt(hi0, 0, 0x4140);
                        av[1][2 * h] = gm_prmt(lo0, 0, 0x4342); av[1][2 * h + 1] = gm_prmt(hi0, 0, 0x4342);
                        av[2][2 * h] = gm_prmt(lo1, 0, 0x4140); av[2][2 * h + 1] = gm_prmt(hi1, 0, 0x4140);
                        av[3][2 * h] = gm_prmt(lo1, 0, 0x4342); av[3][2 * h + 1] = gm_prmt(hi1, 0, 0x4342);
                    }
                } else {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const uint32_t wa = *reinterpret_cast<const uint32_t*>(at + h * 8 * S::ROW), wb = *reinterpret_cast<const uint32_t*>(at1 + h * 8 * S::ROW);
                        const uint32_t lo = gm_prmt(wa, wb, 0x5410), hi = gm_prmt(wa, wb, 0x7632);
                        av[0][2 * h] = lo & 0x000F000Fu; av[0][2 * h + 1] = hi & 0x000F000Fu;
                        av[1][2 * h] = lo & 0x00F000F0u; av[1][2 * h + 1] = hi & 0x00F000F0u;      // sixteen times the code
                        av[2][2 * h] = lo >> 8 & 0x000F000Fu; av[2][2 * h + 1] = hi >> 8 & 0x000F000Fu;
                        av[3][2 * h] = lo >> 8 & 0x00F000F0u; av[3][2 * h + 1] = hi >> 8 & 0x00F000F0u;
                    }
                }
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int n = 0; n < NR; ++n) rows_mma(o[n][grp][j], av[j][0], av[j][1], av[j][2], av[j][3], pb[n][0], pb[n][1]);
            }

            __syncwarp();                                      // the stage's values are in registers of all lanes
            if (ahead) request(stage == 0 ? S::STAGES - 1 : stage - 1);
            asm volatile("cp.async.commit_group;" ::: "memory");
            stage = stage + 1 == S::STAGES ? 0 : stage + 1;
        }
        item += segment;

        // ---- the segment's result: out^T = 2^E (2^24 o - centre * ones) + b_sum, over l ----
        float* part = a.partial + (size_t)((2 * worker + (from_start ? 1 : 0)) * S::SPLIT + half) * RB * (S::DW + 2);
#pragma unroll
        for (int n = 0; n < NR; ++n) {
            float sum = l[n];
            sum += __shfl_xor_sync(kFullMask, sum, 1);
            sum += __shfl_xor_sync(kFullMask, sum, 2);
            if (!whole && t == 0 && g + 8 * n < (int)valid) {
                part[g + 8 * n] = m[n];
                part[RB + g + 8 * n] = sum;
            }
            const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
            const float up0 = rows_power((int)ceilf(__shfl_sync(kFullMask, e_real[n], 8 * t))), up1 = rows_power((int)ceilf(__shfl_sync(kFullMask, e_real[n], 8 * t + 4)));
            const float inv0 = __shfl_sync(kFullMask, inv, 8 * t), inv1 = __shfl_sync(kFullMask, inv, 8 * t + 4);
#pragma unroll
            for (int grp = 0; grp < G; ++grp) {
                float b = b_sum[n][grp];
                b += __shfl_xor_sync(kFullMask, b, 1);
                b += __shfl_xor_sync(kFullMask, b, 2);
#pragma unroll
                for (int c = 0; c < 2; ++c) {                  // rows 2t and 2t + 1
                    const int r = 2 * t + c + 8 * n;
                    const float bc = __shfl_sync(kFullMask, b, 8 * t + 4 * c), centred = -kCentre * __shfl_sync(kFullMask, ones[n][c], 4 * grp + t);
                    if (r >= (int)valid) continue;
                    const float up = c ? up1 : up0;
                    float v[8];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float unit = BITS == 4 && j % 2 ? 1048576.0f : 16777216.0f;
                        v[j] = fmaf(up, fmaf(unit, o[n][grp][j][c], centred), bc);
                        v[4 + j] = fmaf(up, fmaf(unit, o[n][grp][j][2 + c], centred), bc);
                    }
                    const int d = grp * 64 + 8 * g;
                    if (whole) {
                        const float i = c ? inv1 : inv0;
                        const uint32_t flat = now.flat0 + r;
                        uint16_t* dst = a.out + (size_t)(now.seq.row0 + flat / a.group) * a.out_stride + (size_t)(now.head * a.group + flat % a.group) * D + half * S::DW + d;
                        *reinterpret_cast<uint4*>(dst) = make_uint4(rows_pair<BF16>(v[0] * i, v[1] * i), rows_pair<BF16>(v[2] * i, v[3] * i),
                                                                    rows_pair<BF16>(v[4] * i, v[5] * i), rows_pair<BF16>(v[6] * i, v[7] * i));
                    } else {
                        float* dst = part + 2 * RB + r * S::DW + d;
                        *reinterpret_cast<float4*>(dst) = make_float4(v[0], v[1], v[2], v[3]);
                        *reinterpret_cast<float4*>(dst + 4) = make_float4(v[4], v[5], v[6], v[7]);
                    }
                }
            }
        }
        if (!whole) {
            const uint64_t unit_item = item - segment - (uint64_t)first_tile;
            const uint32_t c0 = shares.of(unit_item), parts = shares.of(unit_item + now.range.tiles - 1) - c0 + 1;
            rows_join<D, S::DW, RB, BF16>(a, now.seq.row0, now.head, now.flat0, c0, worker - c0, parts, valid, half, lane);
        }
        if (item < stop) rows_next_unit(a, now);
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
}

template <int D, int BITS, int RB, bool BF16>
static tf_status launch_rows(tf_context* ctx, cudaStream_t st, const AttnArgs& a, const tf_attention_workspace* ws) {
    using S = RowsShape<D, BITS, RB>;
    auto kernel = attention_rows_kernel<D, BITS, RB, BF16>;
    static DeviceSmemCache smem_cache;
    static ResidentBlocksCache blocks_cache;
    const tf_status s = ensure_dynamic_smem(ctx, kernel, smem_cache, S::SMEM);
    if (s != TF_OK) return s;
    uint32_t blocks = resident_blocks(ctx, kernel, blocks_cache, S::THREADS, S::SMEM);
    blocks = lesser(blocks, lesser(ws->row_capacity / RB, ws->max_workers) / S::WORKERS);
    TF_REQUIRE(ctx, blocks > 0, TF_ERR_CUDA, "tf_tree_attention: the kernel does not fit on the device");
    kernel<<<blocks, S::THREADS, S::SMEM, st>>>(a);
    return check_launch(ctx, "tf_tree_attention");
}

}  // namespace tf
