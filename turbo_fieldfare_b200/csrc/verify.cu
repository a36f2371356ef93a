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

#include "kv_cache.cuh"

struct tf_verify_workspace {
    int device = 0;
    uint64_t stats = 0, bytes = 0;     // room, in chunks of rows
    void* memory = nullptr;
};

namespace tf {
namespace {

namespace cg = cooperative_groups;

constexpr int kStatsThreads = 256, kChunk = 8192;          // elements of a row that a block of the first launch takes
constexpr int kWalkThreads = 512, kWalkWarps = kWalkThreads / kWarp;
constexpr uint32_t kMostNodes = 1024;
constexpr double kLog2E = 1.4426950408889634074;

// A chunk's largest logit, the sum of its weights relative to that, and where the largest stands first.
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
    uint32_t vocab, rows, sequences, draft_stride, probs_nodes, probs_dtype, chunks;
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
// a 16-byte boundary. What lies outside the row is -infinity and is not read.
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
    __device__ __forceinline__ void load(uint32_t piece, float (&x)[E]) const {
        const int64_t at = first(piece);
        if (at >= 0 && at + E <= (int64_t)vocab) {
            const uint4 w = *reinterpret_cast<const uint4*>(p + at);
            T v[E];
            memcpy(v, &w, 16);
#pragma unroll
            for (int e = 0; e < E; ++e) x[e] = counted(number(v[e]));
        } else {
#pragma unroll
            for (int e = 0; e < E; ++e) x[e] = at + e >= 0 && at + e < (int64_t)vocab ? counted(number(p[at + e])) : -INFINITY;
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

template <typename T, bool CAP>
__global__ void __launch_bounds__(kStatsThreads) verify_stats_kernel(const __grid_constant__ VerifyArgs a) {
    pdl_launch_dependents();
    constexpr int E = Row<T>::E, PIECES = kChunk / E / kStatsThreads, WARPS = kStatsThreads / kWarp;
    __shared__ uint32_t found, best;
    __shared__ float warp_most[WARPS], warp_sum_[WARPS];
    const uint32_t tid = threadIdx.x, warp = tid / kWarp, lane = tid % kWarp;
    const uint32_t row = blockIdx.x / a.chunks, chunk = blockIdx.x % a.chunks;
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
    const Row<T> r(a.logits, row * a.stride, a.vocab);
    const uint32_t pieces = r.pieces(), piece0 = chunk * (kChunk / E) + tid;
    const float k = heat.k32();
    float x[PIECES][E], most = -INFINITY;
#pragma unroll
    for (int j = 0; j < PIECES; ++j) {
        if (piece0 + j * kStatsThreads < pieces) r.load(piece0 + j * kStatsThreads, x[j]);
        else
#pragma unroll
            for (int e = 0; e < E; ++e) x[j][e] = -INFINITY;
    }
#pragma unroll
    for (int j = 0; j < PIECES; ++j)
#pragma unroll
        for (int e = 0; e < E; ++e) most = fmaxf(most, x[j][e]);
    float top = most;          // of the warp, then of the block
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) top = fmaxf(top, __shfl_xor_sync(kFullMask, top, off));
    if (lane == 0) warp_most[warp] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WARPS; ++w) top = fmaxf(top, warp_most[w]);
    float sum = 0.0f;
    if (top > -INFINITY) {
        const float from = CAP ? capped(top, a.softcap) : top;
#pragma unroll
        for (int j = 0; j < PIECES; ++j)
#pragma unroll
            for (int e = 0; e < E; ++e) sum += verify_exp2(((CAP ? capped(x[j][e], a.softcap) : x[j][e]) - from) * k);
        if (heat.greedy && most == top) {
            uint32_t at = 0xFFFFFFFFu;
#pragma unroll
            for (int j = PIECES - 1; j >= 0; --j)
#pragma unroll
                for (int e = E - 1; e >= 0; --e)
                    if (x[j][e] == top) at = (uint32_t)(r.first(piece0 + j * kStatsThreads) + e);
            atomicMin(&best, at);
        }
    }
    sum = warp_sum(sum);
    if (lane == 0) warp_sum_[warp] = sum;
    __syncthreads();
    if (tid == 0) {
        sum = 0.0f;
        for (int w = 0; w < WARPS; ++w) sum += warp_sum_[w];
        a.stats[(size_t)row * a.chunks + chunk] = {top, sum, best, 0};
    }
}

// ---------------------------------------------------------------------------
// the walk, and the draw
// ---------------------------------------------------------------------------

// How far a row's sum in 32 bits may be from the true one, relative to it: an exponent of up to 126 carries two roundings (2^-16), 2^x itself and the sums of 32, 32 and 8
// add less than 2^-17; capped logits are off by at most softcap 2^-20 each.
__device__ __forceinline__ double sum_bound(float cap, double k) { return 0x1p-15 + (cap > 0.0f ? (double)cap * k * 0x1p-19 : 0.0); }

// 2^x for x <= 0 in 64 bits, by all lanes of a warp: 2^(j/32) from a table that the lanes hold, times the Taylor sum of 2^r, |r| <= 1/64, to its
// fifth power (2e-15 of it), times a power of two. Below 2^-1000: 0.
__device__ __forceinline__ double warp_exp2(double x, double table) {
    const double y = fmax(x, -1000.0), shift = 6755399441055744.0;             // 1.5 2^52: the sum's last bits are the rounded number
    const double t = fma(y, 32.0, shift);
    const int j = __double2loint(t);
    const double r = fma(t - shift, -1.0 / 32, y);
    double s = 0.0013333558146428443;                                           // ln(2)^i / i!, i = 5 ... 1
    s = fma(s, r, 0.009618129107628477);
    s = fma(s, r, 0.05550410866482158);
    s = fma(s, r, 0.24022650695910072);
    s = fma(s, r, 0.6931471805599453);
    s = s * r;
    const double base = __shfl_sync(kFullMask, table, j & 31);
    const double v = fma(base, s, base);
    return x < -1000.0 ? 0.0 : __hiloint2double(__double2hiint(v) + ((j >> 5) << 20), __double2loint(v));
}

template <bool CAP>
__device__ __forceinline__ double logit64(float x, float cap) {
    if constexpr (CAP) return (double)cap * tanh((double)x / (double)cap);
    else return (double)x;
}

// What the cluster does next, and with which row.
struct Order {
    int what;                  // 0: nothing more; 1: sums; 2: sums and a draw
    uint32_t node, at;         // at: where the token goes
    int known, summed, step, drawn, refused;   // its maximum is known; so is Z; the last refusal's sum is not noted yet; q counts; children refused
    float most, u;
    double z, s;               // Z, and the last sum
};

struct Walk {
    uint32_t i, node, at;
    int refused, done, summed, step;
    double z, s, gone;         // gone: weight of the refused tokens, without q
};

__device__ __forceinline__ float prob_at(const VerifyArgs& a, uint64_t at) {
    float q;
    if (a.probs_dtype == TF_FP32) q = static_cast<const float*>(a.probs)[at];
    else if (a.probs_dtype == TF_FP16) q = __half2float(static_cast<const __half*>(a.probs)[at]);
    else q = __bfloat162float(static_cast<const __nv_bfloat16*>(a.probs)[at]);
    return fmaxf(q, 0.0f);     // NaN too
}

template <typename T, bool CAP>
__global__ void __launch_bounds__(kWalkThreads) verify_walk_kernel(const __grid_constant__ VerifyArgs a) {
    constexpr int E = Row<T>::E;
    extern __shared__ __align__(16) uint8_t dynamic[];
    __shared__ Order orders[2];                    // by turns: one is read while the next is written
    __shared__ Walk walk;
    __shared__ double block_sum[2], warp_part[kWalkWarps];
    __shared__ float block_most[2], warp_most[kWalkWarps];
    __shared__ union { double sum[kMostNodes]; int32_t token[kMostNodes]; } gone;      // of the node's refused children: S before each, or the tokens
    const cg::cluster_group cluster = cg::this_cluster();
    const uint32_t tid = threadIdx.x, warp = tid / kWarp, lane = tid % kWarp;
    const uint32_t rank = cluster.block_rank(), ranks = cluster.num_blocks(), b = blockIdx.x / ranks;
    pdl_wait();
    const Nodes of(a, b, rank == 0 && tid == 0);
    const Heat heat(a, b);
    // of the first block: the nodes
    double* z32 = reinterpret_cast<double*>(dynamic);
    float *most = reinterpret_cast<float*>(z32 + a.draft_stride), *logit = most + a.draft_stride, *prob = logit + a.draft_stride;
    uint32_t* best = reinterpret_cast<uint32_t*>(prob + a.draft_stride);
    int32_t *parent = reinterpret_cast<int32_t*>(best + a.draft_stride), *token = parent + a.draft_stride, *inner = token + a.draft_stride;

    if (rank == 0) {
        for (uint32_t i = tid; i < of.n; i += kWalkThreads) {
            parent[i] = i ? parent_of(a, b, i) : -1;
            token[i] = a.tokens[(size_t)b * a.draft_stride + i];
            inner[i] = 0;
        }
        __syncthreads();
        for (uint32_t i = tid; i < of.n; i += kWalkThreads) {
            if (parent[i] < 0) continue;
            inner[parent[i]] = 1;
            if (token[i] < 0 || (uint32_t)token[i] >= a.vocab) continue;
            logit[i] = counted(number(static_cast<const T*>(a.logits)[(of.row0 + (uint64_t)parent[i]) * a.stride + token[i]]));
            prob[i] = a.probs && (uint32_t)parent[i] < a.probs_nodes ? prob_at(a, b * a.probs_sequence + parent[i] * a.probs_node + token[i]) : 0.0f;
        }
        __syncthreads();
        for (uint32_t i = warp; i < of.n; i += kWalkWarps) {
            if (!inner[i] && !heat.greedy) {
                if (lane == 0) most[i] = -INFINITY;
                continue;
            }
            const ChunkStat* s = a.stats + (size_t)(of.row0 + i) * a.chunks;
            float top = -INFINITY;
            uint32_t at = 0xFFFFFFFFu;
            for (uint32_t c = lane; c < a.chunks; c += kWarp) {
                const ChunkStat x = s[c];
                if (x.most > top) { top = x.most; at = x.at; }                 // chunks ascend: the first of equals stays
            }
            float all = top;
#pragma unroll
            for (int off = 16; off >= 1; off >>= 1) all = fmaxf(all, __shfl_xor_sync(kFullMask, all, off));
            if (top != all) at = 0xFFFFFFFFu;
            at = __reduce_min_sync(kFullMask, at);
            const float from = CAP ? capped(all, a.softcap) : all, k = heat.k32();
            double sum = 0.0;
            for (uint32_t c = lane; c < a.chunks; c += kWarp) {
                const ChunkStat x = s[c];
                if (x.most > -INFINITY) sum += (double)(x.sum * verify_exp2(((CAP ? capped(x.most, a.softcap) : x.most) - from) * k));
            }
#pragma unroll
            for (int off = 16; off >= 1; off >>= 1) sum += __shfl_xor_sync(kFullMask, sum, off);
            if (lane == 0) {
                most[i] = all;
                z32[i] = sum;
                best[i] = at == 0xFFFFFFFFu ? 0u : at;
            }
        }
        if (tid == 0) walk = {1, 0, 0, 0, 0, 0, 0, 0.0, 0.0, 0.0};
        __syncthreads();
        if (tid == 0 && of.n) walk.z = z32[0];
    }

    int32_t* out_tokens = a.out_tokens + (size_t)b * a.draft_stride;
    int32_t* out_rows = a.out_rows + (size_t)b * a.draft_stride;
    float* logprobs = a.logprobs ? a.logprobs + (size_t)b * a.draft_stride : nullptr;
    // w of one logit; log(w) stays finite where w is 0
    auto power = [&](float x, float top) { return (logit64<CAP>(x, a.softcap) - logit64<CAP>(top, a.softcap)) * heat.k; };
    constexpr double kLn2 = 0.69314718055994530942;

    // One thread goes from node to node until a sum over the vocabulary is needed; false: the walk is over.
    auto advance = [&](Order& order) {
        Walk& w = walk;
        const double bound = sum_bound(a.softcap, heat.k);
        order.what = 0;
        if (of.n == 0) return;
        for (; w.i < of.n; ++w.i) {
            const uint32_t i = w.i;
            if (parent[i] != (int32_t)w.node || token[i] < 0 || (uint32_t)token[i] >= a.vocab) continue;
            bool keep;
            double weight = 0.0, x2 = 0.0;
            const bool drawn = a.probs && w.node < a.probs_nodes;
            if (most[w.node] > -INFINITY && logit[i] > -INFINITY) {
                x2 = power(logit[i], most[w.node]);
                weight = exp2(x2);
            }
            if (heat.greedy) {
                keep = most[w.node] > -INFINITY && (uint32_t)token[i] == best[w.node];
            } else {
                const double u = (double)fminf(fmaxf(a.uniforms[(size_t)b * a.draft_stride + i], 0.0f), 0x1.fffffep-1f);
                bool ask = false;
                double left, right = weight;
                if (drawn) {
                    const double q = (double)prob[i];
                    if (w.step) ask = true;            // the last refusal's sum first
                    left = u * q * (w.refused ? w.s : w.z);
                    for (int g = 0; g < w.refused && !w.step; ++g) right = fmax(right - gone.sum[g] * q, 0.0);
                    if (!w.refused && !w.summed) ask = fabs(left - right) < bound * left;
                } else {
                    bool before = false;
                    for (int g = 0; g < w.refused; ++g) before |= gone.token[g] == token[i];
                    if (before) continue;              // refused already
                    left = u * (w.z - w.gone);
                    if (!w.summed) ask = fabs(left - right) < bound * u * w.z;
                }
                if (ask) {
                    order = {1, w.node, 0, 1, w.summed, w.step, drawn, w.refused, most[w.node], 0.0f, w.z, w.s};
                    return;
                }
                keep = left < right;
            }
            if (keep) {
                out_rows[w.at + 1] = (int32_t)i;
                out_tokens[w.at] = token[i];
                if (logprobs) logprobs[w.at] = (float)(x2 * kLn2 - log(w.z));
                w.at += 1;
                w.node = i;
                w.refused = w.summed = w.step = 0;
                w.z = z32[i];
                w.gone = 0.0;
            } else if (!heat.greedy) {
                if (drawn) {
                    w.step = 1;
                } else {
                    gone.token[w.refused] = token[i];
                    w.gone += weight;
                }
                w.refused += 1;
            }
        }
        if (w.done) return;
        w.done = 1;
        if (heat.greedy) {
            out_tokens[w.at] = (int32_t)best[w.node];
            if (logprobs) logprobs[w.at] = w.z > 0.0 ? (float)-log(w.z) : -INFINITY;
            return;
        }
        const float u = fminf(fmaxf(a.uniforms[(size_t)b * a.draft_stride], 0.0f), 0x1.fffffep-1f);
        order = {2, w.node, w.at, inner[w.node], w.summed, w.step, a.probs && w.node < a.probs_nodes, w.refused, most[w.node], u, w.z, w.s};
    };

    const double table = exp2((double)lane / 32.0);
    uint32_t turn = 0;
    // Sums and maxima over the cluster, in the order of warps and blocks; the last sums of warps and blocks stay for the draw.
    double block_part = 0.0;                       // lane r: block r's last sum
    auto sum_all = [&](double v) {
#pragma unroll
        for (int off = 16; off >= 1; off >>= 1) v += __shfl_xor_sync(kFullMask, v, off);
        __syncthreads();
        if (lane == 0) warp_part[warp] = v;
        __syncthreads();
        if (tid == 0) {
            double s = 0.0;
            for (int w = 0; w < kWalkWarps; ++w) s += warp_part[w];
            block_sum[turn & 1] = s;
        }
        __syncwarp();
        cluster.sync();
        block_part = lane < ranks ? *cluster.map_shared_rank(&block_sum[turn & 1], lane) : 0.0;
        ++turn;
        double s = 0.0;
        for (uint32_t r = 0; r < ranks; ++r) s += __shfl_sync(kFullMask, block_part, r);
        return s;
    };
    auto most_all = [&](float v) {
#pragma unroll
        for (int off = 16; off >= 1; off >>= 1) v = fmaxf(v, __shfl_xor_sync(kFullMask, v, off));
        __syncthreads();
        if (lane == 0) warp_most[warp] = v;
        __syncthreads();
        if (tid == 0) {
            for (int w = 0; w < kWalkWarps; ++w) v = fmaxf(v, warp_most[w]);
            block_most[turn & 1] = v;
        }
        __syncwarp();
        cluster.sync();
        v = lane < ranks ? *cluster.map_shared_rank(&block_most[turn & 1], lane) : -INFINITY;
        ++turn;
#pragma unroll
        for (int off = 16; off >= 1; off >>= 1) v = fmaxf(v, __shfl_xor_sync(kFullMask, v, off));
        return v;
    };

    for (uint32_t round = 0;; ++round) {
        if (rank == 0 && tid == 0) advance(orders[round & 1]);
        __syncwarp();
        cluster.sync();
        const Order o = *cluster.map_shared_rank(&orders[round & 1], 0);
        if (o.what == 0) break;
        if (rank != 0) {
            for (int g = tid; g < o.refused; g += kWalkThreads)
                if (!o.drawn) gone.token[g] = *cluster.map_shared_rank(&gone.token[g], 0);
                else if (!o.step || g + 1 < o.refused) gone.sum[g] = *cluster.map_shared_rank(&gone.sum[g], 0);
        }
        __syncthreads();

        // ---- this warp's pieces of the row: neighbours, so that sums run in the order of the tokens ----
        const Row<T> row(a.logits, (of.row0 + (uint64_t)o.node) * a.stride, a.vocab);
        const uint32_t pieces = row.pieces(), steps = (pieces + ranks * kWalkThreads - 1) / (ranks * kWalkThreads);
        const uint32_t piece0 = (rank * kWalkWarps + warp) * steps * kWarp + lane;
        const uint64_t q_row = b * a.probs_sequence + o.node * a.probs_node;
        float top = o.most;
        if (!o.known) {
            top = -INFINITY;
            for (uint32_t s = 0; s < steps; ++s) {
                float x[E];
                if (piece0 + s * kWarp >= pieces) break;
                row.load(piece0 + s * kWarp, x);
#pragma unroll
                for (int e = 0; e < E; ++e) top = fmaxf(top, x[e]);
            }
            top = most_all(top);
        }
        const double from = top > -INFINITY ? logit64<CAP>(top, a.softcap) : 0.0;
        // what `refused` children leave of the weights of a piece
        auto left = [&](uint32_t piece, int refused, double (&w)[E]) {
            float x[E];
            if (piece < pieces) row.load(piece, x);
            else
#pragma unroll
                for (int e = 0; e < E; ++e) x[e] = -INFINITY;
            const int64_t first = row.first(piece);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const double v = warp_exp2(x[e] > -INFINITY ? (logit64<CAP>(x[e], a.softcap) - from) * heat.k : 0.0, table);
                w[e] = x[e] > -INFINITY ? v : 0.0;
            }
            if (refused && o.drawn) {
                float q[E];
#pragma unroll
                for (int e = 0; e < E; ++e) q[e] = piece < pieces && first + e >= 0 && first + e < (int64_t)a.vocab ? prob_at(a, q_row + first + e) : 0.0f;
                for (int g = 0; g < refused; ++g) {
                    const double s = gone.sum[g];
#pragma unroll
                    for (int e = 0; e < E; ++e) w[e] = fmax(w[e] - s * (double)q[e], 0.0);
                }
            } else {
                for (int g = 0; g < refused; ++g) {
                    const int64_t e0 = (int64_t)gone.token[g] - first;
#pragma unroll
                    for (int e = 0; e < E; ++e) w[e] = e0 == e ? 0.0 : w[e];
                }
            }
        };
        auto sum_left = [&](int refused) {
            double s = 0.0;
            for (uint32_t i = 0; i < steps; ++i) {
                double w[E];
                left(piece0 + i * kWarp, refused, w);
#pragma unroll
                for (int e = 0; e < E; ++e) s += w[e];
            }
            return sum_all(s);
        };
        double z = o.z, s = 0.0;
        int refused = o.what == 2 || o.drawn ? o.refused : 0;      // a test without q goes by Z alone
        bool parts = false;                        // the last sums are those that are drawn from
        if (!o.summed) {
            s = z = sum_left(0);
            parts = refused == 0;
        }
        if (refused) {
            if (o.step && tid == 0) gone.sum[refused - 1] = refused == 1 ? z : o.s;
            __syncthreads();
            s = sum_left(refused);
            parts = o.what == 1 || s > 0.0;
            if (!parts) refused = 0;               // nothing left: from all of it
        }
        if (o.what == 1) {
            if (rank == 0 && tid == 0) {
                walk.z = z;
                walk.s = s;
                walk.summed = 1;
                walk.step = 0;
            }
            continue;                              // the thread that walks is the one that wrote
        }
        if (!parts) s = sum_left(0);

        // ---- the draw: block, warp, piece, token ----
        const double target = (double)o.u * s;
        if (!(s > 0.0)) {
            if (rank == 0 && tid == 0) {
                out_tokens[o.at] = 0;
                if (logprobs) logprobs[o.at] = -INFINITY;
            }
            continue;
        }
        double before = 0.0;
        uint32_t mine = ranks;                     // the block that the target falls in
        for (uint32_t r = 0; r < ranks; ++r) {
            const double v = __shfl_sync(kFullMask, block_part, r);
            if (before + v > target) { mine = r; break; }
            before += v;
        }
        if (mine != rank) continue;
        uint32_t its = 0;
        double upto = before;
        bool hit = false;
        for (int w = 0; w < kWalkWarps; ++w) {     // rounding may leave it behind the last warp that has anything: then its last token
            if (!(warp_part[w] > 0.0)) continue;
            its = w;
            before = upto;
            upto += warp_part[w];
            if (upto > target) { hit = true; break; }
        }
        if (warp != its) continue;
        double sum = before;
        int64_t token_at = -1, last = -1;
        for (uint32_t i = 0; i < steps; ++i) {
            double w[E], all = 0.0;
            left(piece0 + i * kWarp, refused, w);
#pragma unroll
            for (int e = 0; e < E; ++e) all += w[e];
            double run = all;
#pragma unroll
            for (int off = 1; off < kWarp; off <<= 1) {
                const double v = __shfl_up_sync(kFullMask, run, off);
                if (lane >= off) run += v;
            }
            const uint32_t over = __ballot_sync(kFullMask, all > 0.0 && sum + run > target), any = __ballot_sync(kFullMask, all > 0.0);
            const int who = hit && over ? __ffs(over) - 1 : any ? 31 - __clz(any) : -1;
            if (who >= 0) {
                int64_t found = -1, end = -1;
                double at = sum + run - all;
                const int64_t first = row.first(piece0 + i * kWarp);
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    at += w[e];
                    if (w[e] > 0.0) {
                        end = first + e;
                        if (found < 0 && at > target) found = first + e;
                    }
                }
                found = hit && over ? (found < 0 ? end : found) : -1;
                last = __shfl_sync(kFullMask, end, who);
                token_at = __shfl_sync(kFullMask, found, who);
                if (token_at >= 0) break;
            }
            sum += __shfl_sync(kFullMask, run, kWarp - 1);
        }
        if (token_at < 0) token_at = last;
        if (lane == 0) {
            out_tokens[o.at] = (int32_t)token_at;
            if (logprobs) {
                const float x = counted(number(row.p[token_at]));
                logprobs[o.at] = (float)((logit64<CAP>(x, a.softcap) - from) * heat.k * kLn2 - log(z));
            }
        }
    }
    if (rank == 0) {
        const uint32_t tokens = of.n ? walk.at + 1 : 0;
        for (uint32_t i = tid; i < a.draft_stride; i += kWalkThreads) {
            if (i == 0) out_rows[0] = of.n ? 0 : -1;
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
tf_status launch_verify(tf_context* ctx, cudaStream_t st, const VerifyArgs& a) {
    const char* name = "tf_verify_drafts";
    if (a.rows) {
        verify_stats_kernel<T, CAP><<<a.rows * a.chunks, kStatsThreads, 0, st>>>(a);
        const tf_status s = check_launch(ctx, name);
        if (s != TF_OK) return s;
    }
    constexpr uint32_t kRanks = 8;
    const size_t smem = (size_t)a.draft_stride * 36;
    TF_CUDA(ctx, launch_pdl_cluster(verify_walk_kernel<T, CAP>, dim3(a.sequences * kRanks), dim3(kWalkThreads), smem, st, kRanks, a));
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
    a.vocab = vocab; a.rows = rows; a.sequences = sequences; a.draft_stride = drafts->stride; a.chunks = (uint32_t)chunks;
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
