// Verification of drafted tokens, and with one row per sequence a sampler (tf_verify_drafts).
//
// With weights w(v) = exp((l(v) - max l) / T) and Z their sum, p = w / Z. A child x drawn from q is kept when u q(x) < p_r(x), where r of its
// siblings were refused: p_{r+1} = max(p_r - q, 0) over its sum. Undivided, n_0 = w and n_{r+1} = max(n_r - S_r q, 0) with S_r the sum of n_r: a refusal
// costs one sum over the vocabulary and leaves one number, and no distribution is ever stored, since n_r(v) follows from w(v), q(v) and the sums so far. (It could be written
// as max(w - c q, 0) with one c, which cancels once little is left; step by step nothing does.) Without q a refused token's weight is left out.
//
// Two launches. The first reads every row that has children once, all in parallel, and leaves its maximum and sum by chunks in 32 bits: HBM bounds it.
// The second has a cluster of thread blocks per sequence. Its first block walks the tree: a test needs a logit, a number of q and Z. Z in 32 bits is off by
// less than 2^-15 of itself (see kBound), which decides nearly all tests; where it does not, the cluster sums the row again in 64 bits. Sums behind a
// refusal, and the row that the next token is drawn from, are 64-bit throughout: the token lies between two of up to 2.6e5 borders of the running sum, and
// an error of 1e-7 in it would make up to one draw in a hundred another token. The draw itself goes from the sums of blocks to those of warps to a warp's pieces.
#include <cooperative_groups.h>

#include <new>
#include <type_traits>

#include "kv_cache.cuh"

struct tf_verify_workspace {
    int device = 0;
    uint64_t stats = 0, bytes = 0;     // room, in chunks of rows
    void* memory = nullptr;
};

namespace tf {
namespace {

namespace cg = cooperative_groups;

constexpr int kStatsThreads = 256, kChunk = 8192;          // elements that a block of the first launch takes at a time
constexpr int kWalkThreads = 512, kWalkWarps = kWalkThreads / kWarp;
constexpr uint32_t kMostNodes = 1024;
constexpr double kLog2E = 1.4426950408889634074;

// The largest logit of some chunks, the sum of their weights relative to that, and where the largest stands first.
struct ChunkStat {
    float most, sum;
    uint32_t at, unused;
};

struct VerifyArgs {
    const void* logits;
    uint64_t stride;
    const int32_t *row_offsets, *tokens, *parents;
    const float *uniforms, *temperatures;
    const void* probs;
    uint64_t probs_sequence, probs_node;
    int32_t *out_tokens, *out_rows, *kept;
    float* logprobs;
    ChunkStat* stats;
    uint32_t* error;
    uint32_t vocab, rows, sequences, draft_stride, probs_nodes, probs_dtype, chunks, parts, per;       // a row's chunks are done in parts of `per`
    float softcap;
};

template <typename T> __device__ __forceinline__ float number(T v);
template <> __device__ __forceinline__ float number(float v) { return v; }
template <> __device__ __forceinline__ float number(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float number(__nv_bfloat16 v) { return __bfloat162float(v); }

__device__ __forceinline__ float verify_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// What counts for nothing is -infinity.
__device__ __forceinline__ float counted(float x) { return fabsf(x) < INFINITY ? x : -INFINITY; }

// A row's elements in pieces of 16 aligned bytes: piece v holds elements [E v - lead, E v - lead + E), where the row begins `lead` elements behind
// a 16-byte boundary. What lies outside the row is not read and counts for nothing.
template <typename T>
struct Row {
    static constexpr int E = 16 / sizeof(T);
    const T* p;
    uint32_t lead, vocab;
    __device__ __forceinline__ Row(const void* base, uint64_t at, uint32_t n) : p(static_cast<const T*>(base) + at), vocab(n) {
        lead = (uint32_t)(reinterpret_cast<uintptr_t>(p) % 16 / sizeof(T));
    }
    __device__ __forceinline__ uint32_t pieces() const { return (uint32_t)(((uint64_t)vocab + lead + E - 1) / E); }
    __device__ __forceinline__ int64_t first(uint32_t piece) const { return (int64_t)piece * E - lead; }
    __device__ __forceinline__ uint4 load(uint32_t piece) const {
        const int64_t at = first(piece);
        if (at >= 0 && at + E <= (int64_t)vocab) return *reinterpret_cast<const uint4*>(p + at);
        constexpr uint32_t nothing = sizeof(T) == 4 ? 0xFF800000u : std::is_same<T, __half>::value ? 0xFC00FC00u : 0xFF80FF80u;
        T v[E];
        uint4 w = make_uint4(nothing, nothing, nothing, nothing);
        memcpy(v, &w, 16);
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (at + e >= 0 && at + e < (int64_t)vocab) v[e] = p[at + e];
        memcpy(&w, v, 16);
        return w;
    }
    static __device__ __forceinline__ void numbers(const uint4& w, float (&x)[E]) {
        T v[E];
        memcpy(v, &w, 16);
#pragma unroll
        for (int e = 0; e < E; ++e) x[e] = number(v[e]);
    }
    // The largest, without NaN
    static __device__ __forceinline__ float most(const uint4& w) {
        if constexpr (sizeof(T) == 4) {
            return fmaxf(fmaxf(__uint_as_float(w.x), __uint_as_float(w.y)), fmaxf(__uint_as_float(w.z), __uint_as_float(w.w)));
        } else {
            using T2 = std::conditional_t<std::is_same<T, __half>::value, __half2, __nv_bfloat162>;
            T2 v[4];
            memcpy(v, &w, 16);
            const T2 all = __hmax2(__hmax2(v[0], v[1]), __hmax2(v[2], v[3]));
            return number(__hmax(all.x, all.y));
        }
    }
};

// softcap * tanh(x / softcap); tanh(u) = 1 - 2 / (exp(2 u) + 1), which needs no care at either end: 2^x is 0 or infinite there.
__device__ __forceinline__ float capped(float x, float cap) {
    return x == -INFINITY ? x : cap * (1.0f - __fdividef(2.0f, verify_exp2(x * (float)(2 * kLog2E) / cap) + 1.0f));
}

struct Heat {
    bool greedy;
    double k;                  // log2(e) / T
    __device__ __forceinline__ Heat(const VerifyArgs& a, uint32_t b) {
        const float t = a.temperatures ? a.temperatures[b] : 1.0f;
        greedy = !(t > 0.0f);
        k = kLog2E / (greedy ? 1.0 : (double)fminf(t, 1e30f));
    }
    // In 32 bits: where k is beyond them, differences of logits are so far apart that only the largest counts
    __device__ __forceinline__ float k32() const { return k < 3e38 ? (float)k : 3e38f; }
};

struct Nodes {                 // a sequence's rows, cut to what the arrays can hold
    uint32_t row0, n;
    __device__ __forceinline__ Nodes(const VerifyArgs& a, uint32_t b, bool report) {
        const int32_t begin = a.row_offsets[b], end = a.row_offsets[b + 1], most = (int32_t)a.rows;
        const int32_t lo = begin < 0 ? 0 : begin > most ? most : begin, hi = end < lo ? lo : end > most ? most : end;
        row0 = (uint32_t)lo;
        n = (uint32_t)(hi - lo);
        if (report && (lo != begin || hi != end || n > a.draft_stride)) *a.error = kErrKvOffsets;
        if (n > a.draft_stride) n = a.draft_stride;
    }
};
// The node that node i > 0 continues, or -1.
__device__ __forceinline__ int32_t parent_of(const VerifyArgs& a, uint32_t b, uint32_t i) {
    if (!a.parents) return (int32_t)i - 1;
    const int32_t p = a.parents[(size_t)b * a.draft_stride + i];
    return p >= 0 && p < (int32_t)i ? p : -1;
}

// ---------------------------------------------------------------------------
// maxima and sums of the rows with children
// ---------------------------------------------------------------------------

// softcap * tanh(x / softcap) where |x| <= softcap, as x P((x / softcap)^2): P is tanh(u) / u by its Chebyshev coefficients in u^2, 1.5e-7 of itself off in 32 bits. On the
// arithmetic units, which have room here: with a reciprocal and a second power of two a logit these take as long as everything else together.
__device__ __forceinline__ float capped_near(float x, float inverse) {
    const float u = x * inverse, z = u * u;
    float p = 0.0010455535957589746f;
    p = fmaf(p, z, -0.006217069923877716f);
    p = fmaf(p, z, 0.020305519923567772f);
    p = fmaf(p, z, -0.05346517637372017f);
    p = fmaf(p, z, 0.13325397670269012f);
    p = fmaf(p, z, -0.33332857489585876f);
    p = fmaf(p, z, 0.9999999403953552f);
    return x * p;
}

// A thread keeps a maximum and a sum of its own over the chunks, so that no block meets at a barrier before the end, and has the next chunk's loads under way
// while it works on one; the first chunk's before it knows whether the row has children.
template <typename T, bool CAP>
__global__ void __launch_bounds__(kStatsThreads, 4) verify_stats_kernel(const __grid_constant__ VerifyArgs a) {
    pdl_launch_dependents();
    using R = Row<T>;
    constexpr int E = R::E, PIECES = kChunk / E / kStatsThreads, WARPS = kStatsThreads / kWarp;
    constexpr uint32_t STEP = kChunk / E;
    __shared__ uint32_t found, best;
    __shared__ float warp_most[WARPS], warp_sum_[WARPS];
    const uint32_t tid = threadIdx.x, warp = tid / kWarp, lane = tid % kWarp;
    const uint32_t row = blockIdx.x / a.parts, part = blockIdx.x % a.parts;
    const R r(a.logits, row * a.stride, a.vocab);
    const uint32_t pieces = r.pieces(), end = min(pieces, (part + 1) * a.per * STEP);
    uint32_t piece = part * a.per * STEP + tid;                // of this thread, the first of its chunk
    uint4 next[PIECES];
    auto request = [&] {
#pragma unroll
        for (int j = 0; j < PIECES; ++j)
            if (piece + j * kStatsThreads < end) next[j] = r.load(piece + j * kStatsThreads);
    };
    request();
    if (tid == 0) found = best = 0xFFFFFFFFu;
    __syncthreads();
    for (uint32_t b = tid; b < a.sequences; b += kStatsThreads) {
        const Nodes of(a, b, false);
        if (row >= of.row0 && row - of.row0 < of.n) atomicMin(&found, b);      // one, unless the offsets contradict themselves
    }
    __syncthreads();
    const uint32_t b = found;
    if (b == 0xFFFFFFFFu) return;
    const Nodes of(a, b, false);
    const uint32_t i = row - of.row0;
    const Heat heat(a, b);
    if (!heat.greedy) {        // a greedy sequence ends with the likeliest token of any of its rows; of others' leaves at most one is looked at
        bool child = false;
        if (!a.parents) child = i + 1 < of.n;
        else for (uint32_t j = i + 1 + tid; j < of.n; j += kStatsThreads) child |= parent_of(a, b, j) == (int32_t)i;
        if (!__syncthreads_or(child)) return;
    }
    const float k = heat.k32(), inverse = CAP ? 1.0f / a.softcap : 0.0f;
    float most = -INFINITY, from = -INFINITY, sum = 0.0f;
    uint32_t where = 0;                                        // the chunk of the first largest
    for (; piece < end; piece += STEP) {
        uint4 w[PIECES];
        uint32_t n = 0;
        float top = -INFINITY;
#pragma unroll
        for (int j = 0; j < PIECES; ++j)
            if (piece + j * kStatsThreads < end) {
                w[j] = next[j];
                top = fmaxf(top, R::most(w[j]));
                n = j + 1;
            }
        const uint32_t here = piece;
        piece += STEP;
        request();
        piece = here;
        if (top == INFINITY) {                                 // does not count
            top = -INFINITY;
#pragma unroll
            for (int j = 0; j < PIECES; ++j) {
                float x[E];
                R::numbers(w[j], x);
#pragma unroll
                for (int e = 0; e < E; ++e)
                    if (j < n) top = fmaxf(top, counted(x[e]));
            }
        }
        if (top > most) {
            const float to = CAP ? capped(top, a.softcap) : top;
            sum *= verify_exp2((from - to) * k);               // nothing so far: 0 times 0
            most = top;
            from = to;
            where = piece;
        }
        if (most == -INFINITY) continue;
        float add = 0.0f;
        bool far = false;
#pragma unroll
        for (int j = 0; j < PIECES; ++j)
            if (j < n) {
                float x[E];
                R::numbers(w[j], x);
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    if constexpr (CAP) {
                        far |= !(fabsf(x[e]) <= a.softcap);
                        x[e] = capped_near(x[e], inverse);
                    }
                    add += verify_exp2((x[e] - from) * k);
                }
            }
        if (far || !(add < INFINITY)) {                        // logits beyond the cap's polynomial, infinities and NaN
            add = 0.0f;
#pragma unroll
            for (int j = 0; j < PIECES; ++j) {
                float x[E];
                R::numbers(w[j], x);
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const float c = counted(x[e]);
                    if (j < n) add += verify_exp2(((CAP ? capped(c, a.softcap) : c) - from) * k);
                }
            }
        }
        sum += add;
    }
    float top = most;
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) top = fmaxf(top, __shfl_xor_sync(kFullMask, top, off));
    if (lane == 0) warp_most[warp] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WARPS; ++w) top = fmaxf(top, warp_most[w]);
    if (most > -INFINITY) {
        sum *= verify_exp2((from - (CAP ? capped(top, a.softcap) : top)) * k);
        if (heat.greedy && most == top) {                      // few threads
            uint32_t at = 0xFFFFFFFFu;
            for (int j = 0; j < PIECES && where + j * kStatsThreads < end && at == 0xFFFFFFFFu; ++j) {
                float x[E];
                R::numbers(r.load(where + j * kStatsThreads), x);
#pragma unroll
                for (int e = E - 1; e >= 0; --e)
                    if (x[e] == top) at = (uint32_t)(r.first(where + j * kStatsThreads) + e);
            }
            atomicMin(&best, at);
        }
    }
    sum = warp_sum(sum);
    if (lane == 0) warp_sum_[warp] = sum;
    __syncthreads();
    if (tid == 0) {
        sum = 0.0f;
        for (int w = 0; w < WARPS; ++w) sum += warp_sum_[w];
        a.stats[(size_t)row * a.parts + part] = {top, sum, best, 0};
    }
}

// ---------------------------------------------------------------------------
// the walk, and the draw
// ---------------------------------------------------------------------------

// How far a row's sum in 32 bits may be from the true one, relative to it: an exponent of up to 126 carries two roundings (2^-16), 2^x itself and the sums of 32, 32 and 8
// add less than 2^-17; capped logits are off by at most softcap 2^-20 each.
__device__ __forceinline__ double sum_bound(float cap, double k) { return 0x1p-15 + (cap > 0.0f ? (double)cap * k * 0x1p-19 : 0.0); }

// 2^(y k / 32) in 64 bits by all lanes of a warp: 2^(j/32) from a table that the lanes hold, times the Taylor sum of 2^r, |r| <= 1/64, to its fifth power
// (2e-15 of it), times a power of two. Exponents from -1000 to 1000; below, and for y = -infinity, 0.
__device__ __forceinline__ double warp_exp2(double y, double k, double table) {
    const double shift = 6755399441055744.0;                                    // 1.5 2^52: the sum's last bits are the rounded number
    const double t = fma(y, k, shift);
    const int j = __double2loint(t);
    const double r = fma(y, k, shift - t);
    constexpr double c = 0.69314718055994530942 / 32;
    double s = c * c * c * c * c / 120;
    s = fma(s, r, c * c * c * c / 24);
    s = fma(s, r, c * c * c / 6);
    s = fma(s, r, c * c / 2);
    s = fma(s, r, c);
    s = s * r;
    const double base = __shfl_sync(kFullMask, table, j & 31);
    const double v = fma(base, s, base);
    return t >= shift - 32000.0 ? __hiloint2double(__double2hiint(v) + ((j >> 5) << 20), __double2loint(v)) : 0.0;
}

template <bool CAP>
__device__ __forceinline__ double logit64(float x, float cap) {
    if constexpr (CAP) return (double)cap * tanh((double)x / (double)cap);
    else return (double)x;
}
// The same by all lanes of a warp, 1e-13 softcap off: cap - 2 cap / (exp(2 x / cap) + 1), the quotient from 23 bits by one of Newton's steps. twice: 64 log2(e) / cap.
template <bool CAP>
__device__ __forceinline__ double warp_logit64(float x, double cap, double twice, double table) {
    if constexpr (!CAP) return (double)x;
    const float edge = 20.0f * (float)cap;                                      // tanh is 1 to the last bit from there on
    const double d = warp_exp2((double)fminf(fmaxf(x, -edge), edge), twice, table) + 1.0;
    float y0;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y0) : "f"((float)d));
    const double y = fma((double)y0, fma(-d, (double)y0, 1.0), (double)y0);
    return x > -INFINITY ? fma(-2.0 * cap, y, cap) : -INFINITY;
}

// What the cluster does next, and with which row.
struct Order {
    int what;                  // 0: nothing more; 1: sums; 2: sums and a draw, which is the last thing
    uint32_t node, at;         // at: where the token goes
    int known, summed, step, drawn, refused;   // its maximum is known; so is Z; the last refusal's sum is not noted yet; q counts; children refused
    float most, u;
    double z, s;               // Z, and the last sum
};

struct Walk {
    uint32_t i, node, at;
    int known, refused, summed, step;
    double z, s, gone;         // gone: weight of the refused tokens, without q
};

// The first block's shared memory: what it knows of the nodes. 48 bytes of each.
struct NodeTable {
    double *z, *weight;        // of a row: its sum in 32 bits; of a token: its weight in its parent's row
    double* gone;              // of the current node's refused children: S before each, or (as int32) the tokens
    float *most, *prob;
    uint32_t* best;
    int32_t *parent, *token, *inner;       // inner: has children; -1 - place of a kept node
    __device__ __forceinline__ NodeTable(uint8_t* memory, uint32_t n) {
        z = reinterpret_cast<double*>(memory);
        weight = z + n;
        gone = weight + n;
        most = reinterpret_cast<float*>(gone + n);
        prob = most + n;
        best = reinterpret_cast<uint32_t*>(prob + n);
        parent = reinterpret_cast<int32_t*>(best + n);
        token = parent + n;
        inner = token + n;
    }
    static constexpr size_t kBytes = 48;
};

__device__ const double kPowers[32] = {               // 2^(j / 32)
    1.0, 1.0218971486541166, 1.0442737824274138, 1.0671404006768237, 1.0905077326652577, 1.1143867425958924,
    1.1387886347566916, 1.1637248587775775, 1.189207115002721, 1.215247359980469, 1.241857812073484, 1.2690509571917332,
    1.2968395546510096, 1.3252366431597413, 1.3542555469368927, 1.383909881963832, 1.4142135623730951, 1.4451808069770467,
    1.4768261459394993, 1.5091644275934228, 1.5422108254079407, 1.5759808451078865, 1.6104903319492543, 1.645755478153965,
    1.681792830507429, 1.718619298122478, 1.7562521603732995, 1.7947090750031072, 1.8340080864093424, 1.8741676341103,
    1.9152065613971474, 1.9571441241754002};

__device__ __forceinline__ float prob_at(const VerifyArgs& a, uint64_t at) {
    float q;
    if (a.probs_dtype == TF_FP32) q = static_cast<const float*>(a.probs)[at];
    else if (a.probs_dtype == TF_FP16) q = __half2float(static_cast<const __half*>(a.probs)[at]);
    else q = __bfloat162float(static_cast<const __nv_bfloat16*>(a.probs)[at]);
    return fmaxf(q, 0.0f);     // NaN too
}
// E of them, of which those outside the row are zero
template <int E>
__device__ __forceinline__ void probs_at(const VerifyArgs& a, uint64_t row, int64_t first, float (&q)[E]) {
    const bool whole = first >= 0 && first + E <= (int64_t)a.vocab;
    if (a.probs_dtype == TF_FP32) {
        const float* p = static_cast<const float*>(a.probs) + (int64_t)row + first;
        if (whole && reinterpret_cast<uintptr_t>(p) % 16 == 0) {
            uint4 w[E / 4];
#pragma unroll
            for (int i = 0; i < E / 4; ++i) w[i] = reinterpret_cast<const uint4*>(p)[i];
#pragma unroll
            for (int e = 0; e < E; ++e) q[e] = fmaxf(__uint_as_float(e % 4 == 0 ? w[e / 4].x : e % 4 == 1 ? w[e / 4].y : e % 4 == 2 ? w[e / 4].z : w[e / 4].w), 0.0f);
            return;
        }
    } else {
        const uint16_t* p = static_cast<const uint16_t*>(a.probs) + (int64_t)row + first;
        if (whole && reinterpret_cast<uintptr_t>(p) % (2 * E) == 0) {
            uint32_t w[E / 2];
            load_words<E / 2>(w, p);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const uint16_t v = (uint16_t)(w[e / 2] >> (16 * (e % 2)));
                q[e] = fmaxf(a.probs_dtype == TF_FP16 ? f16_bits_to_float(v) : bf16_bits_to_float(v), 0.0f);
            }
            return;
        }
    }
#pragma unroll
    for (int e = 0; e < E; ++e) q[e] = first + e >= 0 && first + e < (int64_t)a.vocab ? prob_at(a, row + first + e) : 0.0f;
}

// Inclusive sums over a warp's lanes.
__device__ __forceinline__ double warp_scan(double v, uint32_t lane) {
#pragma unroll
    for (int off = 1; off < kWarp; off <<= 1) {
        const double o = __shfl_up_sync(kFullMask, v, off);
        if (lane >= off) v += o;
    }
    return v;
}

// Among parts in the lanes' order, whose sums `upto` are, the one that the target falls in; rounding may leave it behind the last that has anything, which is then it.
// The target becomes that within the part.
__device__ __forceinline__ uint32_t warp_fall(double part, double upto, double& target) {
    const uint32_t any = __ballot_sync(kFullMask, part > 0.0), over = __ballot_sync(kFullMask, part > 0.0 && upto > target);
    const uint32_t who = over ? __ffs(over) - 1 : any ? 31 - __clz(any) : 0;
    const double before = __shfl_sync(kFullMask, upto - part, who);
    target = over ? target - before : INFINITY;
    return who;
}

// One thread goes from node to node until a sum over the vocabulary is needed, or the walk is over.
template <bool CAP>
__device__ __forceinline__ void walk_on(const VerifyArgs& a, const Nodes& of, const Heat& heat, uint32_t b, const NodeTable& t, Walk& w, Order& order,
                                        int32_t* out_tokens, int32_t* out_rows) {
    const double bound = sum_bound(a.softcap, heat.k);
    const float* uniforms = a.uniforms + (size_t)b * a.draft_stride;
    const int32_t* gone_tokens = reinterpret_cast<const int32_t*>(t.gone);
    order.what = 0;
    if (of.n == 0) return;
    for (; w.i < of.n; ++w.i) {
        const uint32_t i = w.i;
        if (t.parent[i] != (int32_t)w.node || t.token[i] < 0) continue;
        const bool drawn = a.probs && w.node < a.probs_nodes;
        bool keep;
        if (heat.greedy) {
            keep = t.most[w.node] > -INFINITY && (uint32_t)t.token[i] == t.best[w.node];
        } else {
            const double u = (double)fminf(fmaxf(uniforms[i], 0.0f), 0x1.fffffep-1f), weight = t.weight[i];
            bool ask = false;
            double left, right = weight;
            if (drawn) {
                const double q = (double)t.prob[i];
                if (w.step) ask = true;                // the last refusal's sum first
                left = u * q * (w.refused ? w.s : w.z);
                for (int g = 0; g < w.refused && !w.step; ++g) right = fmax(fma(-t.gone[g], q, right), 0.0);
                if (!w.refused && !w.summed) ask = fabs(left - right) < bound * left;
            } else {
                bool before = false;
                for (int g = 0; g < w.refused; ++g) before |= gone_tokens[g] == t.token[i];
                if (before) continue;                  // refused already
                left = u * (w.z - w.gone);
                if (!w.summed) ask = fabs(left - right) < bound * u * w.z;
            }
            if (ask) {
                order = {1, w.node, 0, 1, w.summed, w.step, drawn, w.refused, t.most[w.node], 0.0f, w.z, w.s};
                return;
            }
            keep = left < right;
        }
        if (keep) {
            out_rows[w.at + 1] = (int32_t)i;
            out_tokens[w.at] = t.token[i];
            w.known = t.inner[i];
            t.inner[i] = -1 - (int32_t)w.at;
            w.at += 1;
            w.node = i;
            const double z = w.z;
            w.z = t.z[i];
            t.z[i] = z;                                // now what the kept token's weight is a part of
            w.refused = w.summed = w.step = 0;
            w.gone = 0.0;
        } else if (!heat.greedy) {
            if (drawn) {
                w.step = 1;
            } else {
                reinterpret_cast<int32_t*>(t.gone)[w.refused] = t.token[i];
                w.gone += t.weight[i];
            }
            w.refused += 1;
        }
    }
    if (heat.greedy) {
        out_tokens[w.at] = (int32_t)t.best[w.node];
        if (a.logprobs) a.logprobs[(size_t)b * a.draft_stride + w.at] = w.z > 0.0 ? (float)-log(w.z) : -INFINITY;
        return;
    }
    const float u = fminf(fmaxf(uniforms[0], 0.0f), 0x1.fffffep-1f);
    order = {2, w.node, w.at, w.known, w.summed, w.step, a.probs && w.node < a.probs_nodes, w.refused, t.most[w.node], u, w.z, w.s};
}

template <typename T, bool CAP>
__global__ void __launch_bounds__(kWalkThreads, 1) verify_walk_kernel(const __grid_constant__ VerifyArgs a) {
    using R = Row<T>;
    constexpr int E = R::E;
    extern __shared__ __align__(16) uint8_t dynamic[];
    __shared__ Order orders[2];                    // by turns: one is read while the next is written
    __shared__ Walk walk;
    __shared__ double block_sum[2], warp_part[kWalkWarps];
    __shared__ float block_most[2], warp_most[kWalkWarps];
    __shared__ uint32_t likeliest;
    const cg::cluster_group cluster = cg::this_cluster();
    const uint32_t tid = threadIdx.x, warp = tid / kWarp, lane = tid % kWarp;
    const uint32_t rank = cluster.block_rank(), ranks = cluster.num_blocks(), b = blockIdx.x / ranks;
    const double table = kPowers[lane];
    pdl_wait();
    const Nodes of(a, b, rank == 0 && tid == 0);
    const Heat heat(a, b);
    const NodeTable nodes(dynamic, a.draft_stride);
    int32_t* gone_tokens = reinterpret_cast<int32_t*>(nodes.gone);
    int32_t* out_tokens = a.out_tokens + (size_t)b * a.draft_stride;
    int32_t* out_rows = a.out_rows + (size_t)b * a.draft_stride;
    float* logprobs = a.logprobs ? a.logprobs + (size_t)b * a.draft_stride : nullptr;
    const double k = heat.k * 32.0, cap = a.softcap, twice = CAP ? 64.0 * kLog2E / cap : 0.0;
    constexpr double kLn2 = 0.69314718055994530942;
    // A lone row is drawn from at once by all blocks, whatever there is to know of it.
    const bool alone = of.n == 1 && (a.draft_stride == 1 || !heat.greedy);
    if (tid == 0) {
        walk = {1, 0, 0, 0, 0, 0, 0, 0.0, 0.0, 0.0};
        likeliest = 0xFFFFFFFFu;
    }

    if (rank == 0 && !alone) {
        for (uint32_t i = tid; i < of.n; i += kWalkThreads) {
            const int32_t x = a.tokens[(size_t)b * a.draft_stride + i];
            nodes.parent[i] = i ? parent_of(a, b, i) : -1;
            nodes.token[i] = x >= 0 && (uint32_t)x < a.vocab ? x : -1;
            nodes.inner[i] = 0;
            nodes.most[i] = -INFINITY;
        }
        __syncthreads();
        for (uint32_t i = tid; i < of.n; i += kWalkThreads) {
            const int32_t p = nodes.parent[i], x = nodes.token[i];
            if (p < 0) continue;
            nodes.inner[p] = 1;
            if (x < 0) continue;
            nodes.weight[i] = (double)counted(number(static_cast<const T*>(a.logits)[(of.row0 + (uint64_t)p) * a.stride + x]));     // for now
            nodes.prob[i] = a.probs && (uint32_t)p < a.probs_nodes ? prob_at(a, b * a.probs_sequence + p * a.probs_node + x) : 0.0f;
        }
        __syncthreads();
        for (uint32_t i = warp; i < of.n; i += kWalkWarps) {
            if (!nodes.inner[i] && !heat.greedy) continue;
            const ChunkStat* s = a.stats + (size_t)(of.row0 + i) * a.parts;
            float top = -INFINITY;
            uint32_t at = 0xFFFFFFFFu;
            for (uint32_t c = lane; c < a.parts; c += kWarp) {
                const ChunkStat x = s[c];
                if (x.most > top) { top = x.most; at = x.at; }                 // parts ascend: the first of equals stays
            }
            float all = top;
#pragma unroll
            for (int off = 16; off >= 1; off >>= 1) all = fmaxf(all, __shfl_xor_sync(kFullMask, all, off));
            if (top != all) at = 0xFFFFFFFFu;
            at = __reduce_min_sync(kFullMask, at);
            const float from = CAP ? capped(all, a.softcap) : all, k32 = heat.k32();
            double sum = 0.0;
            for (uint32_t c = lane; c < a.parts; c += kWarp) {
                const ChunkStat x = s[c];
                if (x.most > -INFINITY) sum += (double)(x.sum * verify_exp2(((CAP ? capped(x.most, a.softcap) : x.most) - from) * k32));
            }
#pragma unroll
            for (int off = 16; off >= 1; off >>= 1) sum += __shfl_xor_sync(kFullMask, sum, off);
            if (lane == 0) {
                nodes.most[i] = all;
                nodes.z[i] = sum;
                nodes.best[i] = at == 0xFFFFFFFFu ? 0u : at;
            }
        }
        __syncthreads();
        for (uint32_t i0 = warp * kWarp; i0 < of.n; i0 += kWalkThreads) {
            const uint32_t i = i0 + lane;
            const bool is = i < of.n && nodes.parent[i] >= 0 && nodes.token[i] >= 0;
            const float x = is ? (float)nodes.weight[i] : -INFINITY, top = is ? nodes.most[nodes.parent[i]] : -INFINITY;
            const double l = warp_logit64<CAP>(x, cap, twice, table), from = warp_logit64<CAP>(top, cap, twice, table);
            const double w = warp_exp2(top > -INFINITY ? l - from : -INFINITY, k, table);
            if (is) nodes.weight[i] = w;
        }
        __syncthreads();
        if (tid == 0 && of.n) {
            walk.z = nodes.z[0];
            walk.known = nodes.inner[0];
        }
    }
    __syncthreads();

    for (uint32_t round = 0, turn = 0;; ++round) {
        Order o = {2, 0, 0, 0, 0, 0, 0, 0, 0.0f, 0.0f, 0.0, 0.0};
        if (alone) {
            o.u = fminf(fmaxf(a.uniforms[(size_t)b * a.draft_stride], 0.0f), 0x1.fffffep-1f);
        } else {
            if (rank == 0 && tid == 0) walk_on<CAP>(a, of, heat, b, nodes, walk, orders[round & 1], out_tokens, out_rows);
            __syncwarp();
            cluster.sync();
            o = *cluster.map_shared_rank(&orders[round & 1], 0);
        }
        if (o.what == 0) break;
        if (rank != 0) {
            for (int g = tid; g < o.refused; g += kWalkThreads)
                if (!o.drawn) gone_tokens[g] = *cluster.map_shared_rank(&gone_tokens[g], 0);
                else if (!o.step || g + 1 < o.refused) nodes.gone[g] = *cluster.map_shared_rank(&nodes.gone[g], 0);
            __syncthreads();
        }

        // ---- the pieces: a warp's are neighbours, and a block's warps, so that sums run in the order of the tokens ----
        const R row(a.logits, (of.row0 + (uint64_t)o.node) * a.stride, a.vocab);
        const uint32_t pieces = row.pieces(), steps = (pieces + ranks * kWalkThreads - 1) / (ranks * kWalkThreads);
        const uint64_t q_row = b * a.probs_sequence + o.node * a.probs_node;
        uint32_t begin = rank * kWalkWarps * steps * kWarp, count = kWalkWarps * steps, sub = steps;       // first piece, steps of a warp's width, steps a warp
        // A row without a maximum (a leaf: nothing was refused) is summed by every block relative to its own, one meeting less.
        float top = o.most;
        if (!o.known) {
            top = -INFINITY;
            for (uint32_t i = 0, piece = begin + warp * steps * kWarp + lane; i < steps && piece < pieces; i += 4, piece += 4 * kWarp) {
                uint4 w[4];
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (i + j < steps && piece + j * kWarp < pieces) w[j] = row.load(piece + j * kWarp);
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (i + j < steps && piece + j * kWarp < pieces) {
                        float most = R::most(w[j]);
                        if (most == INFINITY) {            // does not count
                            float x[E];
                            R::numbers(w[j], x);
                            most = -INFINITY;
#pragma unroll
                            for (int e = 0; e < E; ++e) most = fmaxf(most, counted(x[e]));
                        }
                        top = fmaxf(top, most);
                    }
            }
#pragma unroll
            for (int off = 16; off >= 1; off >>= 1) top = fmaxf(top, __shfl_xor_sync(kFullMask, top, off));
            if (lane == 0) warp_most[warp] = top;
            __syncthreads();
            top = lane < kWalkWarps ? warp_most[lane] : -INFINITY;
#pragma unroll
            for (int off = 16; off >= 1; off >>= 1) top = fmaxf(top, __shfl_xor_sync(kFullMask, top, off));
        }
        const double from = top > -INFINITY ? warp_logit64<CAP>(top, cap, twice, table) : 0.0;

        // ---- sums, and the draw from block to warp to step to token, with one body for all of it: what runs once costs what its instructions take to fetch ----
        enum { kAll, kLeft, kAgain, kWithin, kStep };
        int stage = !o.summed ? kAll : o.refused && (o.drawn || o.what == 2) ? kLeft : kAgain;
        double z = o.z, target = 0.0, whole = from;    // whole: the logit that z is relative to
        int refused = 0;
        for (;;) {
            if (stage == kLeft) {
                refused = o.refused;
                if (o.drawn && o.step) {
                    if (tid == 0) nodes.gone[refused - 1] = refused == 1 ? z : o.s;
                    __syncthreads();
                }
            } else if (stage == kAgain) {
                refused = 0;
            }
            // what `refused` children leave of the weights of this warp's steps; in a single step every warp has all of it
            const uint32_t first = stage == kStep ? 0u : min(warp * sub, count), last = stage == kStep ? 1u : min(first + sub, count);
            double w[E], all = 0.0;
            uint32_t piece = begin + first * kWarp + lane;
            uint4 next = make_uint4(0, 0, 0, 0);
            if (first < last && piece < pieces) next = row.load(piece);
            for (uint32_t i = first; i < last; ++i, piece += kWarp) {
                float x[E];
                R::numbers(next, x);
                if (i + 1 < last && piece + kWarp < pieces) next = row.load(piece + kWarp);
                float q[E];
                if (refused && o.drawn) probs_at<E>(a, q_row, piece < pieces ? row.first(piece) : (int64_t)a.vocab, q);
#pragma unroll
                for (int e = 0; e < E; ++e)
                    w[e] = warp_exp2(warp_logit64<CAP>(piece < pieces ? counted(x[e]) : -INFINITY, cap, twice, table) - from, k, table);
                for (int g = 0; g < refused; ++g) {
                    if (o.drawn) {
                        const double s = nodes.gone[g];
#pragma unroll
                        for (int e = 0; e < E; ++e) w[e] = fmax(fma(-s, (double)q[e], w[e]), 0.0);
                    } else {
                        const int64_t e0 = (int64_t)gone_tokens[g] - row.first(piece);
#pragma unroll
                        for (int e = 0; e < E; ++e) w[e] = e0 == e ? 0.0 : w[e];
                    }
                }
#pragma unroll
                for (int e = 0; e < E; ++e) all += w[e];
            }
            if (stage == kStep) {
                const double upto = warp_scan(all, lane);
                if (warp_fall(all, upto, target) == lane && warp == 0) {
                    double at = 0.0;
                    int found = -1, end = 0;
#pragma unroll
                    for (int e = 0; e < E; ++e) {
                        at += w[e];
                        if (w[e] > 0.0) {
                            end = e;
                            if (found < 0 && at > target) found = e;
                        }
                    }
                    found = found < 0 ? end : found;
                    out_tokens[o.at] = (int32_t)(row.first(begin + lane) + found);
                    if (logprobs) {
                        const float x = number(row.p[row.first(begin + lane) + found]);
                        logprobs[o.at] = (float)((logit64<CAP>(x, a.softcap) - whole) * heat.k * kLn2 - log(z));
                    }
                }
                break;
            }
#pragma unroll
            for (int off = 16; off >= 1; off >>= 1) all += __shfl_xor_sync(kFullMask, all, off);
            __syncthreads();                           // the sums before these have been read
            if (lane == 0) warp_part[warp] = all;
            __syncthreads();
            const double part = lane < kWalkWarps ? warp_part[lane] : 0.0, upto = warp_scan(part, lane);
            if (stage != kWithin) {
                // ---- over the cluster ----
                if (tid == kWarp - 1) {
                    block_sum[turn & 1] = upto;
                    block_most[turn & 1] = top;
                }
                __syncwarp();
                cluster.sync();
                double mine = lane < ranks ? *cluster.map_shared_rank(&block_sum[turn & 1], lane) : 0.0, scale = 1.0;
                if (!o.known) {
                    const float its = lane < ranks ? *cluster.map_shared_rank(&block_most[turn & 1], lane) : -INFINITY;
                    float most = its;
#pragma unroll
                    for (int off = 16; off >= 1; off >>= 1) most = fmaxf(most, __shfl_xor_sync(kFullMask, most, off));
                    whole = warp_logit64<CAP>(most, cap, twice, table);
                    scale = warp_exp2(most > -INFINITY ? warp_logit64<CAP>(its, cap, twice, table) - whole : -INFINITY, k, table);
                    mine *= scale;
                    if (heat.greedy) {                 // alone: the likeliest token instead of a draw
                        if (top == most && top > -INFINITY) {
                            for (uint32_t i = 0, p = begin + warp * steps * kWarp + lane; i < steps && p < pieces; ++i, p += kWarp) {
                                float x[E];
                                R::numbers(row.load(p), x);
#pragma unroll
                                for (int e = E - 1; e >= 0; --e)
                                    if (x[e] == top) atomicMin(cluster.map_shared_rank(&likeliest, 0), (uint32_t)(row.first(p) + e));
                            }
                        }
                    }
                }
                ++turn;
                const double run = warp_scan(mine, lane), s = __shfl_sync(kFullMask, run, ranks - 1);
                if (stage == kAll) z = s;
                if (heat.greedy) {
                    cluster.sync();
                    if (rank == 0 && tid == 0) {
                        out_tokens[o.at] = likeliest == 0xFFFFFFFFu ? 0 : (int32_t)likeliest;
                        if (logprobs) logprobs[o.at] = z > 0.0 ? (float)-log(z) : -INFINITY;
                    }
                    break;
                }
                if (stage == kAll && o.refused && (o.drawn || o.what == 2)) {
                    stage = kLeft;
                    continue;
                }
                if (o.what == 1) {
                    if (rank == 0 && tid == 0) {       // the thread that walks
                        walk.z = z;
                        walk.s = s;
                        walk.summed = 1;
                        walk.step = 0;
                    }
                    break;
                }
                if (!(s > 0.0)) {
                    if (stage == kLeft) {              // nothing left: from all of it
                        stage = kAgain;
                        continue;
                    }
                    if (rank == 0 && tid == 0) {
                        out_tokens[o.at] = 0;
                        if (logprobs) logprobs[o.at] = -INFINITY;
                    }
                    break;
                }
                target = (double)o.u * s;
                const uint32_t who = warp_fall(mine, run, target);
                if (who != rank) break;
                target /= __shfl_sync(kFullMask, scale, who);
            }
            const uint32_t its = warp_fall(part, upto, target);
            begin += its * sub * kWarp;
            count = min(sub, count - its * sub);
            sub = (count + kWalkWarps - 1) / kWalkWarps;
            stage = count > 1 ? kWithin : kStep;
        }
        if (o.what == 2) break;
    }
    if (rank == 0) {
        __syncthreads();
        const uint32_t tokens = of.n ? walk.at + 1 : 0;
        for (uint32_t i = tid; i < a.draft_stride; i += kWalkThreads) {
            if (i == 0) out_rows[0] = of.n ? 0 : -1;
            if (logprobs && !alone && i < of.n && nodes.inner[i] < 0)
                logprobs[-1 - nodes.inner[i]] = (float)(heat.greedy ? -log(nodes.z[i]) : log(nodes.weight[i] / nodes.z[i]));
            if (i < tokens) continue;
            out_tokens[i] = -1;
            if (i) out_rows[i] = -1;
            if (logprobs) logprobs[i] = 0.0f;
        }
        if (tid == 0) a.kept[b] = (int32_t)tokens;
    }
    __syncwarp();
    cluster.sync();                                // nobody leaves while its shared memory may be read
}

template <typename T, bool CAP>
tf_status launch_verify(tf_context* ctx, cudaStream_t st, VerifyArgs a) {
    const char* name = "tf_verify_drafts";
    constexpr uint32_t E = Row<T>::E;
    if (a.rows && a.draft_stride > 1) {            // lone rows need none of it
        const bool even = aligned(a.logits, 16) && a.stride % E == 0;          // else a row may begin anywhere in a piece
        a.chunks = (uint32_t)(((uint64_t)a.vocab + (even ? 0 : E - 1) + kChunk - 1) / kChunk);
        // several chunks a block, as long as that leaves every place on the chip a few blocks
        const uint64_t all = (uint64_t)a.rows * a.chunks / ((uint64_t)ctx->sm_count * 16);
        a.per = (uint32_t)(all < 1 ? 1 : all > 4 ? 4 : all);
        a.parts = (a.chunks + a.per - 1) / a.per;
        verify_stats_kernel<T, CAP><<<a.rows * a.parts, kStatsThreads, 0, st>>>(a);
        const tf_status s = check_launch(ctx, name);
        if (s != TF_OK) return s;
    }
    uint32_t ranks = 8;
    while (ranks > 1 && (uint64_t)a.sequences * ranks > (uint64_t)ctx->sm_count) ranks /= 2;
    const size_t smem = a.draft_stride * NodeTable::kBytes;
    static DeviceSmemCache smem_cache;
    const tf_status m = ensure_dynamic_smem(ctx, verify_walk_kernel<T, CAP>, smem_cache, smem);
    if (m != TF_OK) return m;
    TF_CUDA(ctx, launch_pdl_cluster(verify_walk_kernel<T, CAP>, dim3(a.sequences * ranks), dim3(kWalkThreads), smem, st, ranks, a));
    return check_launch(ctx, name);
}

}  // namespace
}  // namespace tf

extern "C" {

tf_status tf_verify_workspace_create(tf_context* ctx, uint32_t max_rows, uint32_t max_vocab, tf_verify_workspace** out) {
    const char* name = "tf_verify_workspace_create";
    TF_REQUIRE(ctx, ctx != nullptr && out != nullptr, TF_ERR_INVALID_ARGUMENT, "%s: NULL argument", name);
    *out = nullptr;
    TF_REQUIRE(ctx, max_rows > 0 && max_vocab > 0, TF_ERR_INVALID_ARGUMENT, "%s: no rows or no vocabulary", name);
    const tf::DeviceScope scope(ctx->device);
    tf_verify_workspace* ws = new (std::nothrow) tf_verify_workspace();
    TF_REQUIRE(ctx, ws != nullptr, TF_ERR_OUT_OF_MEMORY, "%s: out of host memory", name);
    ws->device = ctx->device;
    ws->stats = (uint64_t)max_rows * (((uint64_t)max_vocab + 7 + tf::kChunk - 1) / tf::kChunk);
    ws->bytes = ws->stats * sizeof(tf::ChunkStat);
    const cudaError_t e = cudaMalloc(&ws->memory, ws->bytes);
    if (e != cudaSuccess) {
        cudaGetLastError();
        delete ws;
        return tf::fail(ctx, TF_ERR_OUT_OF_MEMORY, "%s: %s", name, cudaGetErrorString(e));
    }
    *out = ws;
    return TF_OK;
}

void tf_verify_workspace_destroy(tf_verify_workspace* ws) {
    if (!ws) return;
    const tf::DeviceScope scope(ws->device);
    if (ws->memory) cudaFree(ws->memory);
    delete ws;
}

uint64_t tf_verify_workspace_bytes(const tf_verify_workspace* ws) { return ws ? ws->bytes : 0; }

tf_status tf_verify_drafts(tf_context* ctx, void* stream, const void* logits, uint64_t logits_stride, tf_dtype logits_dtype, uint32_t vocab,
                           const int32_t* row_offsets, uint32_t rows, uint32_t sequences, const tf_drafts* drafts, const float* uniforms,
                           const tf_draft_probs* probs, const float* temperatures, float softcap, int32_t* out_tokens, int32_t* out_rows, int32_t* kept,
                           float* logprobs, tf_verify_workspace* ws) {
    const char* name = "tf_verify_drafts";
    TF_REQUIRE(ctx, ctx != nullptr, TF_ERR_INVALID_ARGUMENT, "%s: ctx is NULL", name);
    TF_REQUIRE(ctx, drafts != nullptr && ws != nullptr, TF_ERR_INVALID_ARGUMENT, "%s: drafts or workspace is NULL", name);
    TF_REQUIRE(ctx, ws->device == ctx->device, TF_ERR_INVALID_ARGUMENT, "%s: the workspace belongs to device %d, the context to %d", name, ws->device, ctx->device);
    auto known = [](tf_dtype t) { return t == TF_FP16 || t == TF_BF16 || t == TF_FP32; };
    TF_REQUIRE(ctx, known(logits_dtype), TF_ERR_UNSUPPORTED, "%s: logits are fp16, bf16 or fp32", name);
    TF_REQUIRE(ctx, vocab > 0 && vocab <= 0x7FFFFFFFu, TF_ERR_INVALID_ARGUMENT, "%s: vocab must be from 1 to 2^31 - 1", name);
    TF_REQUIRE(ctx, drafts->stride > 0 && drafts->stride <= tf::kMostNodes, TF_ERR_UNSUPPORTED, "%s: a sequence has from 1 to %u nodes, not %u", name, tf::kMostNodes,
               drafts->stride);
    TF_REQUIRE(ctx, rows <= 0x7FFFFFFFu && sequences <= 0x7FFFFFFFu / 16, TF_ERR_INVALID_ARGUMENT, "%s: too many rows or sequences", name);
    TF_REQUIRE(ctx, softcap >= 0.0f && softcap <= 3.4e38f, TF_ERR_INVALID_ARGUMENT, "%s: softcap must be finite and not negative", name);
    if (sequences == 0) return TF_OK;
    TF_REQUIRE(ctx, (logits || rows == 0) && row_offsets && uniforms && out_tokens && out_rows && kept && drafts->tokens, TF_ERR_INVALID_ARGUMENT, "%s: NULL buffer", name);
    TF_REQUIRE(ctx, rows <= 1 || logits_stride >= vocab, TF_ERR_INVALID_ARGUMENT, "%s: a row stride is smaller than its row", name);
    auto size = [](tf_dtype t) { return t == TF_FP32 ? (size_t)4 : (size_t)2; };
    TF_REQUIRE(ctx, tf::aligned(logits, size(logits_dtype)) && tf::aligned(row_offsets, 4) && tf::aligned(uniforms, 4) && tf::aligned(temperatures, 4) &&
                        tf::aligned(out_tokens, 4) && tf::aligned(out_rows, 4) && tf::aligned(kept, 4) && tf::aligned(logprobs, 4) && tf::aligned(drafts->tokens, 4) &&
                        tf::aligned(drafts->parents, 4), TF_ERR_ALIGNMENT, "%s: arrays must be aligned to their elements", name);
    const uint64_t chunks = ((uint64_t)vocab + 7 + tf::kChunk - 1) / tf::kChunk;
    TF_REQUIRE(ctx, rows * chunks <= ws->stats, TF_ERR_SCRATCH_TOO_SMALL, "%s: the workspace has room for %llu chunks of rows, not %llu", name,
               (unsigned long long)ws->stats, (unsigned long long)(rows * chunks));
    TF_REQUIRE(ctx, rows * chunks <= 0x7FFFFFFFu, TF_ERR_UNSUPPORTED, "%s: too many rows for the vocabulary", name);
    tf::VerifyArgs a = {};
    if (probs && probs->nodes) {
        TF_REQUIRE(ctx, probs->values != nullptr, TF_ERR_INVALID_ARGUMENT, "%s: probs has no values", name);
        TF_REQUIRE(ctx, known(probs->dtype), TF_ERR_UNSUPPORTED, "%s: probabilities are fp16, bf16 or fp32", name);
        TF_REQUIRE(ctx, tf::aligned(probs->values, size(probs->dtype)), TF_ERR_ALIGNMENT, "%s: arrays must be aligned to their elements", name);
        TF_REQUIRE(ctx, probs->nodes == 1 || probs->node_stride >= vocab, TF_ERR_INVALID_ARGUMENT, "%s: a row stride is smaller than its row", name);
        a.probs = probs->values; a.probs_sequence = probs->sequence_stride; a.probs_node = probs->node_stride; a.probs_nodes = probs->nodes;
        a.probs_dtype = probs->dtype;
    }
    a.logits = logits; a.stride = logits_stride; a.row_offsets = row_offsets; a.tokens = drafts->tokens; a.parents = drafts->parents;
    a.uniforms = uniforms; a.temperatures = temperatures;
    a.out_tokens = out_tokens; a.out_rows = out_rows; a.kept = kept; a.logprobs = logprobs;
    a.stats = static_cast<tf::ChunkStat*>(ws->memory);
    a.error = ctx->device_error;
    a.vocab = vocab; a.rows = rows; a.sequences = sequences; a.draft_stride = drafts->stride;
    a.softcap = softcap;
    const tf::DeviceScope scope(ctx->device);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const bool cap = softcap > 0.0f;
    switch (logits_dtype) {
        case TF_FP16: return cap ? tf::launch_verify<__half, true>(ctx, st, a) : tf::launch_verify<__half, false>(ctx, st, a);
        case TF_BF16: return cap ? tf::launch_verify<__nv_bfloat16, true>(ctx, st, a) : tf::launch_verify<__nv_bfloat16, false>(ctx, st, a);
        default: return cap ? tf::launch_verify<float, true>(ctx, st, a) : tf::launch_verify<float, false>(ctx, st, a);
    }
}

}  // extern "C"
