// Verification of drafted tokens, and with one row per sequence a sampler (tf_verify_drafts).
//
// With weights w(v) = exp((l(v) - max l) / T) and Z their sum, p = w / Z. A child x drawn from q is kept when u q(x) < p_r(x), where r of its
// siblings were refused: p_{r+1} = max(p_r - q, 0) over its sum. Undivided, n_0 = w and n_{r+1} = max(n_r - S_r q, 0) with S_r the sum of n_r: a refusal
// costs one sum over the vocabulary and leaves one number, and no distribution is ever stored, since n_r(v) follows from w(v), q(v) and the sums so far. (It could be written
// as max(w - c q, 0) with one c, which cancels once little is left; step by step nothing does.) Without q a refused token's weight is left out.
//
// Two launches. The first reads every row that has children (of greedy sequences every row) once, all in parallel, and leaves its maximum and sum by parts in 32 bits: HBM bounds it.
// Where there are few logits, or one row a sequence, it leaves those sums of all rows in 64 bits, and the second launch seldom reads a row again.
// The second has a cluster of thread blocks per sequence. Its first block walks the tree: a test needs a logit, a number of q and Z. Z in 32 bits is off by
// less than 2^-15 of itself (see kBound), which decides nearly all tests; where it does not, the cluster sums the row again in 64 bits. Sums behind a
// refusal, and the row that the next token is drawn from, are 64-bit throughout: the token lies between two of up to 2.6e5 borders of the running sum, and
// an error of 1e-7 in it would make up to one draw in a hundred another token. The draw itself goes from the sums of blocks to those of warps to a warp's pieces.
#include <cooperative_groups.h>

#include <atomic>
#include <new>
#include <type_traits>

#include "kv_cache.cuh"

struct tf_verify_workspace {
    int device = 0;
    uint64_t room = 0, stats = 0, bytes = 0;   // chunks of rows that calls may have; sums that there is place for
    void* memory = nullptr;
};

namespace tf {
namespace {

namespace cg = cooperative_groups;

constexpr int kStatsThreads = 256, kChunk = 8192;          // elements that a block of the first launch takes at a time
constexpr int kWalkThreads = 256, kWalkWarps = kWalkThreads / kWarp, kGroups = 8;
constexpr uint32_t kMostNodes = 1024, kMostRanks = 16;       // blocks of a sequence: a cluster beyond eight is to be asked for
constexpr double kLog2E = 1.4426950408889634074;

// The largest logit of some chunks, the sum of their weights relative to that, and where the largest stands first.
struct ChunkStat {
    double sum;
    float most;
    uint32_t at, infinite;     // infinite: there are +infinities, which count for nothing
    uint32_t unused;
};

struct VerifyArgs {
    const void* logits;
    uint64_t stride;
    EarlyTable<int32_t> row_offsets, tokens, parents;          // the first launch reads them plainly: it is an ordinary one
    EarlyTable<float> uniforms, temperatures;
    const void* probs;
    uint64_t probs_sequence, probs_node;
    int32_t *out_tokens, *out_rows, *kept;
    float* logprobs;
    ChunkStat* stats;
    uint32_t* error;
    uint32_t vocab, rows, sequences, draft_stride, probs_nodes, probs_dtype, chunks, parts, per;       // a row's chunks are done in parts of `per`; exact: pieces of a thread
    float softcap;
    bool exact;                // all rows have been summed in 64 bits
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
    const uint4* base;         // of piece 0, where the row begins at a boundary or inside the piece
    uint32_t lead, vocab, whole0, whole;       // pieces [whole0, whole0 + whole) hold elements of the row alone
    __device__ __forceinline__ Row(const void* start, uint64_t at, uint32_t n) : p(static_cast<const T*>(start) + at), vocab(n) {
        lead = (uint32_t)(reinterpret_cast<uintptr_t>(p) % 16 / sizeof(T));
        base = reinterpret_cast<const uint4*>(p - lead);
        whole0 = lead ? 1 : 0;
        const uint32_t end = (uint32_t)(((uint64_t)vocab + lead) / E);
        whole = end > whole0 ? end - whole0 : 0;
    }
    __device__ __forceinline__ uint32_t pieces() const { return (uint32_t)(((uint64_t)vocab + lead + E - 1) / E); }
    __device__ __forceinline__ int64_t first(uint32_t piece) const { return (int64_t)piece * E - lead; }
    // A drawn element, which is one of the row's unless offsets contradict themselves and the sums are of another call
    __device__ __forceinline__ int64_t inside(int64_t at) const { return at < 0 ? 0 : at < (int64_t)vocab ? at : (int64_t)vocab - 1; }
    static __device__ __forceinline__ uint4 nothing() {
        constexpr uint32_t w = sizeof(T) == 4 ? 0xFF800000u : std::is_same<T, __half>::value ? 0xFC00FC00u : 0xFF80FF80u;
        return make_uint4(w, w, w, w);
    }
    // Behind the last piece too
    __device__ __forceinline__ uint4 load(uint32_t piece) const {
        if (piece - whole0 < whole) return base[piece];
        const int64_t at = first(piece);
        T v[E];
        uint4 w = nothing();
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
    // The magnitudes of a piece
    static __device__ __forceinline__ uint4 magnitudes(uint4 w) {
        constexpr uint32_t mask = sizeof(T) == 4 ? 0x7FFFFFFFu : 0x7FFF7FFFu;
        return make_uint4(w.x & mask, w.y & mask, w.z & mask, w.w & mask);
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

// softcap * tanh(x / softcap) where |x| <= softcap, as x + x z R(z), z = (x / softcap)^2: R is (tanh(u) / u - 1) / u^2 by a polynomial in u^2 whose largest error times u^2 is least (by weighted least
// squares, each coefficient rounded to 32 bits before the next ones are found): 5.5e-9 of it off, and one rounding of the result. On the arithmetic units, which have room here: with a reciprocal and a second power of two a logit these take as long as everything else together.
__device__ __forceinline__ float capped_near(float x, float inverse) {
    const float u = x * inverse, z = u * u;
    float r = -0.00036188133526593447f;
    r = fmaf(r, z, 0.002313370117917657f);
    r = fmaf(r, z, -0.00796255562454462f);
    r = fmaf(r, z, 0.021497756242752075f);
    r = fmaf(r, z, -0.053883593529462814f);
    r = fmaf(r, z, 0.1333240419626236f);
    r = fmaf(r, z, -0.33333298563957214f);
    return fmaf(x, r * z, x);
}
// 1 / cap, of caps below 2^-128 the largest number: with an infinity a logit of zero would be NaN.
__device__ __forceinline__ float inverse_of(float cap) { return fminf(1.0f / cap, 3.402823466e38f); }
// The same of any logit; tanh(u) = 1 - 2 / (exp(2 u) + 1), which needs no care at either end: 2^x is 0 or infinite there.
__device__ __forceinline__ float capped(float x, float cap) {
    if (fabsf(x) <= cap) return capped_near(x, inverse_of(cap));
    return x == -INFINITY ? x : cap * (1.0f - __fdividef(2.0f, verify_exp2(x * (float)(2 * kLog2E) / cap) + 1.0f));
}

// A random number, in [0, 1) whatever it is.
__device__ __forceinline__ float uniform(float u) { return fminf(fmaxf(u, 0.0f), 0x1.fffffep-1f); }

// What a launch reads before its wait comes past L1 (see EarlyTable): the second launches say so of what they call there.
constexpr std::true_type kEarly{};
constexpr std::false_type kWaited{};

struct Heat {
    bool greedy;
    double k;                  // log2(e) / T
    template <bool EARLY>
    __device__ __forceinline__ Heat(const VerifyArgs& a, uint32_t b, std::bool_constant<EARLY>) {
        const float t = a.temperatures.p ? a.temperatures.at<EARLY>(b) : 1.0f;
        greedy = !(t > 0.0f);
        k = kLog2E / (greedy ? 1.0 : (double)fminf(t, 1e30f));
    }
    // In 32 bits: where k is beyond them, differences of logits are so far apart that only the largest counts
    __device__ __forceinline__ float k32() const { return k < 3e38 ? (float)k : 3e38f; }
};

struct Nodes {                 // a sequence's rows, cut to what the arrays can hold
    uint32_t row0, n;
    template <bool EARLY>
    __device__ __forceinline__ Nodes(const VerifyArgs& a, uint32_t b, bool report, std::bool_constant<EARLY>) {
        const int32_t begin = a.row_offsets.at<EARLY>(b), end = a.row_offsets.at<EARLY>(b + 1), most = (int32_t)a.rows;
        const int32_t lo = begin < 0 ? 0 : begin > most ? most : begin, hi = end < lo ? lo : end > most ? most : end;
        row0 = (uint32_t)lo;
        n = (uint32_t)(hi - lo);
        if (report && (lo != begin || hi != end || n > a.draft_stride)) *a.error = kErrKvOffsets;
        if (n > a.draft_stride) n = a.draft_stride;
    }
};
// Whose row it is, into `found` (which stays as it is where it is nobody's), by all threads of a block: a block a row must not look through all of many sequences, so from 1024 on it
// first takes a 256th, in which the last one lies that begins no later. Offsets that contradict themselves find one of those that have the row, or none.
__device__ __forceinline__ void owner_of(const VerifyArgs& a, uint32_t row, uint32_t* found) {
    uint32_t lo = 0, n = a.sequences;
    while (n > 1024) {
        const uint32_t part = (n + kStatsThreads - 1) / kStatsThreads, at = threadIdx.x * part;
        const uint32_t before = (uint32_t)__syncthreads_count(at < n && a.row_offsets.at<false>(lo + at) <= (int32_t)row);
        const uint32_t skip = (before ? before - 1 : 0) * part;
        lo += skip;
        n = min(part, n - skip);
    }
    for (uint32_t b = lo + threadIdx.x; b < lo + n; b += kStatsThreads) {
        const Nodes of(a, b, false, kWaited);
        if (row >= of.row0 && row - of.row0 < of.n) atomicMin(found, b);
    }
}
// The node that node i > 0 continues, or -1.
template <bool EARLY>
__device__ __forceinline__ int32_t parent_of(const VerifyArgs& a, uint32_t b, uint32_t i, std::bool_constant<EARLY>) {
    if (!a.parents.p) return (int32_t)i - 1;
    const int32_t p = a.parents.at<EARLY>((size_t)b * a.draft_stride + i);
    return p >= 0 && p < (int32_t)i ? p : -1;
}

// ---------------------------------------------------------------------------
// maxima and sums of the rows with children
// ---------------------------------------------------------------------------

// A thread keeps a maximum and a sum of its own over the chunks, so that no block meets at a barrier before the end, and has the next chunk's loads under way
// while it works on one; the first chunk's before it knows whether the row has children. Chunks with a row's edge are done apart. The powers of two bound it beside HBM: sixteen a clock and SM
// are 4.5e12 a second, what 16-bit logits at the full 6.5 TB/s would ask for is 3.3e12. 200 chains of four, all rows needed: 58 us cold, 5.4 TB/s. In 64 registers the two sets of eight pieces that
// fp32 logits take do not fit: 172 bytes of a thread are spilled (272 capped; 16-bit ones none, up to 16 capped). Capped pieces with a logit wider than the cap, -infinity among them, are done twice.
template <typename T, bool CAP>
__global__ void __launch_bounds__(kStatsThreads, 4) verify_stats_kernel(const __grid_constant__ VerifyArgs a) {
    pdl_launch_dependents();
    using R = Row<T>;
    constexpr int E = R::E, PIECES = kChunk / E / kStatsThreads, WARPS = kStatsThreads / kWarp;
    constexpr uint32_t STEP = kChunk / E;
    __shared__ uint32_t found, best, infinite;
    __shared__ float warp_most[WARPS], warp_sum_[WARPS];
    const uint32_t tid = threadIdx.x, warp = tid / kWarp, lane = tid % kWarp;
    const uint32_t row = blockIdx.x / a.parts, part = blockIdx.x % a.parts;
    const R r(a.logits, row * a.stride, a.vocab);
    const uint32_t pieces = r.pieces(), chunk0 = part * a.per, chunk1 = min(chunk0 + a.per, (pieces + STEP - 1) / STEP);
    // chunks [full0, full1) have nothing but whole pieces
    const uint32_t full0 = max(chunk0, r.whole0 ? 1u : 0u), full1 = max(full0, min(chunk1, (r.whole0 + r.whole) / STEP));
    const uint4* p = r.base + (size_t)full0 * STEP + tid;
    uint4 next[PIECES];
    if (full0 < full1)
#pragma unroll
        for (int j = 0; j < PIECES; ++j) next[j] = p[j * kStatsThreads];
    if (tid == 0) {
        found = best = 0xFFFFFFFFu;
        infinite = 0;
    }
    __syncthreads();
    owner_of(a, row, &found);
    __syncthreads();
    const uint32_t b = found;
    if (b == 0xFFFFFFFFu) return;
    const Nodes of(a, b, false, kWaited);
    const uint32_t i = row - of.row0;
    const Heat heat(a, b, kWaited);
    if (!heat.greedy) {        // a greedy sequence ends with the likeliest token of any of its rows; of others' leaves at most one is looked at
        bool child = false;
        if (!a.parents.p) child = i + 1 < of.n;
        else for (uint32_t j = i + 1 + tid; j < of.n; j += kStatsThreads) child |= parent_of(a, b, j, kWaited) == (int32_t)i;
        if (!__syncthreads_or(child)) return;
    }
    const float k = heat.k32(), inverse = CAP ? inverse_of(a.softcap) : 0.0f;
    float most = -INFINITY, from = -INFINITY, sum = 0.0f;
    uint32_t where = 0;                                        // the chunk of the first largest
    auto take = [&](const uint4 (&w)[PIECES], uint32_t chunk) {
        float top = R::most(w[0]);
#pragma unroll
        for (int j = 1; j < PIECES; ++j) top = fmaxf(top, R::most(w[j]));
        if (top == INFINITY) {                                 // does not count
            infinite = 1;
            top = -INFINITY;
#pragma unroll
            for (int j = 0; j < PIECES; ++j) {
                float x[E];
                R::numbers(w[j], x);
#pragma unroll
                for (int e = 0; e < E; ++e) top = fmaxf(top, counted(x[e]));
            }
        }
        if (top > most) {
            const float to = CAP ? capped(top, a.softcap) : top;
            sum *= verify_exp2((from - to) * k);               // nothing so far: 0 times 0
            most = top;
            from = to;
            where = chunk;
        }
        if (most == -INFINITY) return;
        float add = 0.0f, widest = 0.0f;
#pragma unroll
        for (int j = 0; j < PIECES; ++j) {
            float x[E];
            R::numbers(w[j], x);
            if constexpr (CAP) widest = fmaxf(widest, R::most(R::magnitudes(w[j])));
#pragma unroll
            for (int e = 0; e < E; ++e) {
                if constexpr (CAP) x[e] = capped_near(x[e], inverse);
                add += verify_exp2((x[e] - from) * k);
            }
        }
        if (!(widest <= (CAP ? a.softcap : 0.0f)) || !(add < INFINITY)) {      // logits beyond the cap's polynomial, infinities and NaN
            add = 0.0f;
#pragma unroll
            for (int j = 0; j < PIECES; ++j) {
                float x[E];
                R::numbers(w[j], x);
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const float c = counted(x[e]);
                    add += verify_exp2(((CAP ? capped(c, a.softcap) : c) - from) * k);
                }
            }
        }
        sum += add;
    };
    for (uint32_t chunk = chunk0; chunk < chunk1;) {
        if (chunk == full0 && full0 < full1) {
#pragma unroll 1
            for (; chunk < full1; ++chunk) {
                uint4 w[PIECES];
#pragma unroll
                for (int j = 0; j < PIECES; ++j) w[j] = next[j];
                p += STEP;
                if (chunk + 1 < full1)
#pragma unroll
                    for (int j = 0; j < PIECES; ++j) next[j] = p[j * kStatsThreads];
                take(w, chunk);
            }
        } else {
            uint4 w[PIECES];
#pragma unroll
            for (int j = 0; j < PIECES; ++j) w[j] = r.load(chunk * STEP + tid + j * kStatsThreads);
            take(w, chunk);
            ++chunk;
        }
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
            for (int j = 0; j < PIECES && at == 0xFFFFFFFFu; ++j) {
                const uint32_t piece = where * STEP + tid + j * kStatsThreads;
                float x[E];
                R::numbers(r.load(piece), x);
#pragma unroll
                for (int e = E - 1; e >= 0; --e)
                    if (x[e] == top) at = (uint32_t)(r.first(piece) + e);
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
        a.stats[(size_t)row * a.parts + part] = {(double)sum, top, best, infinite, 0};
    }
}

// ---------------------------------------------------------------------------
// the walk, and the draw
// ---------------------------------------------------------------------------

// How far a row's sum in 32 bits may be from the true one, relative to it: an exponent of up to 126 carries two roundings (2^-16), 2^x itself and the sums of 32, 32 and 8
// add less than 2^-17; capped logits are off by at most softcap 2^-20 each.
__device__ __forceinline__ double sum_bound(float cap, double k) { return 0x1p-15 + (cap > 0.0f ? (double)cap * k * 0x1p-19 : 0.0); }

// 2^((y k + shift - kShift) / 32) in 64 bits by all lanes of a warp, as base times y: 2^(j/32) from a table that the lanes hold, with a power of two that goes into its number (whose upper words
// are lower by what the last bits of j add there), and 2^(r/32), |r| <= 1/2, by its Chebyshev sum to the fourth power (8e-14 of it: a border between tokens moves by no more than that of all). The
// caller's sums multiply: eight operations a logit. shift is kShift, or that less a whole number. Exponents from -1010 to 1010. All N at once, so that none waits for the operations in a row.
constexpr double kShift = 6755399441055744.0;                                   // 1.5 2^52: the sum's last bits are the rounded number
template <int N>
__device__ __forceinline__ void warp_exp2(double (&y)[N], double k, double shift, int2 table, double (&base)[N]) {
    constexpr double c = 0.69314718055994530942 / 32, fifth = c * c * c * c * c / 120;
    constexpr double poly[4] = {c - fifth * 5 / 256, c * c / 2, c * c * c / 6 + fifth * 5 / 16, c * c * c * c / 24};
    int j[N];
    double r[N];
#pragma unroll
    for (int e = 0; e < N; ++e) {
        const double t = fma(y[e], k, shift);
        j[e] = __double2loint(t);
        r[e] = fma(y[e], k, shift - t);
    }
#pragma unroll
    for (int e = 0; e < N; ++e) {
        const int hi = __shfl_sync(kFullMask, table.x, j[e]), lo = __shfl_sync(kFullMask, table.y, j[e]);       // by their last five bits
        base[e] = __hiloint2double(hi + j[e] * 32768, lo);
    }
#pragma unroll
    for (int e = 0; e < N; ++e) y[e] = poly[3];
#pragma unroll
    for (int i = 2; i >= 0; --i)
#pragma unroll
        for (int e = 0; e < N; ++e) y[e] = fma(y[e], r[e], poly[i]);
#pragma unroll
    for (int e = 0; e < N; ++e) y[e] = fma(y[e], r[e], 1.0);
}
template <int N>
__device__ __forceinline__ void warp_exp2(double (&y)[N], double k, int2 table) {
    double base[N];
    warp_exp2(y, k, kShift, table, base);
#pragma unroll
    for (int e = 0; e < N; ++e) y[e] *= base[e];
}
__device__ __forceinline__ double positive(double v) { return __double2hiint(v) < 0 ? 0.0 : v; }

template <bool CAP>
__device__ __forceinline__ double logit64(float x, float cap) {
    if constexpr (CAP) return (double)cap * tanh((double)x / (double)cap);
    else return (double)x;
}
__device__ const double kPowers[32] = {               // 2^(j / 32)
    1.0, 1.0218971486541166, 1.0442737824274138, 1.0671404006768237, 1.0905077326652577, 1.1143867425958924,
    1.1387886347566916, 1.1637248587775775, 1.189207115002721, 1.215247359980469, 1.241857812073484, 1.2690509571917332,
    1.2968395546510096, 1.3252366431597413, 1.3542555469368927, 1.383909881963832, 1.4142135623730951, 1.4451808069770467,
    1.4768261459394993, 1.5091644275934228, 1.5422108254079407, 1.5759808451078865, 1.6104903319492543, 1.645755478153965,
    1.681792830507429, 1.718619298122478, 1.7562521603732995, 1.7947090750031072, 1.8340080864093424, 1.8741676341103,
    1.9152065613971474, 1.9571441241754002};
__device__ __forceinline__ int2 power_table(int lane) { return make_int2(__double2hiint(kPowers[lane]) - lane * 32768, __double2loint(kPowers[lane])); }

// From logits to weights, what a row has in common.
struct Scale {
    double from, k, shift;     // the logit of weight 1, 32 log2(e) / T; kShift - from k
    double cap, twice, inverse;        // softcap, 64 log2(e) / softcap, 1 / softcap
    double lowest;             // -32000 / k: that far below a weight is 2^-1000
    float least;               // logits from here down count as that, where the row needs no care
    int2 table;
    bool careful;              // the row holds infinities, steps of 32 bits that are as large as that, or a cap far above T and its logits
    template <bool CAP>
    __device__ __forceinline__ void set(float softcap, double log2e_by_heat, int lane) {
        table = power_table(lane);
        k = log2e_by_heat * 32.0;
        cap = softcap;
        twice = CAP ? 64.0 * kLog2E / cap : 0.0;
        inverse = CAP ? 1.0 / cap : 0.0;
        lowest = -32000.0 / k;
    }
    // What the weights of a row with such a logit are relative to: one nearby that k makes a whole number.
    __device__ __forceinline__ double unit(double logit) const {
        const double by = logit * k;
        return fabs(by) < 0x1p40 ? rint(by) * (lowest * (-1.0 / 32000.0)) : logit;
    }
    // With the row's largest logit, as it is; infinite: there are some that do not count. By all lanes.
    template <bool CAP>
    __device__ __forceinline__ void relative_to(float top, bool infinite);
};
constexpr double kNothing = 0x1p-900;          // more than a vocabulary of tokens that do not count

// Logits that are no wider than the cap: x P((x / cap)^2), P being tanh(u) / u by its Chebyshev coefficients in u^2 on [0, 1], 2e-14 of it off.
template <int N>
__device__ __forceinline__ void near_capped(const float (&x)[N], double inverse, double (&w)[N]) {
    constexpr double c[13] = {0.9999999999999823, -0.3333333333272711, 0.13333333298786137, -0.05396824620692592, 0.021869397540056224, -0.008862596767873559, 0.0035892253083668387,
                              -0.0014468841456978221, 0.0005707702734400899, -0.0002097698327657338, 6.496419251345914e-05, -1.4302828371933043e-05, 1.5987624655853251e-06};
    double z[N], p[N];
#pragma unroll
    for (int e = 0; e < N; ++e) {
        w[e] = (double)x[e];
        z[e] = w[e] * inverse;
        z[e] *= z[e];
        p[e] = c[12];
    }
#pragma unroll
    for (int i = 11; i >= 0; --i)
#pragma unroll
        for (int e = 0; e < N; ++e) p[e] = fma(p[e], z[e], c[i]);
#pragma unroll
    for (int e = 0; e < N; ++e) w[e] *= p[e];
}

// Weights in 64 bits by all lanes of a warp. Capped logits: cap - 2 cap / (exp(2 x / cap) + 1), the quotient from 23 bits by one of Newton's steps, 1e-13 cap off; a row whose weights
// that would move is a careful one, where logits no wider than the cap go by the series of near_capped.
// They come as products base w, which sums multiply. NEAR: no logit that counts is wider than the cap, the series for all: half of the instructions.
template <bool CAP, int N, bool CARE = true, bool NEAR = false>
__device__ __forceinline__ void warp_weights(const Scale& s, const float (&x)[N], double (&w)[N], double (&base)[N]) {
    if constexpr (!CAP) {
#pragma unroll
        for (int e = 0; e < N; ++e) w[e] = (double)fmaxf(x[e], s.least);       // NaN too
    } else if constexpr (NEAR) {
        near_capped(x, s.inverse, w);
    } else {
        const float edge = 20.0f * (float)s.cap;                                // tanh is 1 to the last bit from there on
        double y[N];
#pragma unroll
        for (int e = 0; e < N; ++e) w[e] = (double)fminf(fmaxf(x[e], -edge), edge);
        warp_exp2(w, s.twice, s.table);
#pragma unroll
        for (int e = 0; e < N; ++e) {
            w[e] += 1.0;
            float y0;
            asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y0) : "f"((float)w[e]));
            y[e] = (double)y0;
        }
#pragma unroll
        for (int e = 0; e < N; ++e) w[e] = fma(-w[e], y[e], 1.0);
#pragma unroll
        for (int e = 0; e < N; ++e) y[e] = fma(y[e], w[e], y[e]);
#pragma unroll
        for (int e = 0; e < N; ++e) w[e] = fma(-2.0 * s.cap, y[e], s.cap);
        if (CARE && s.careful) {
            near_capped(x, s.inverse, y);
#pragma unroll
            for (int e = 0; e < N; ++e) w[e] = fabsf(x[e]) <= (float)s.cap ? y[e] : w[e];
        }
    }
    if constexpr (CAP) {
#pragma unroll
        for (int e = 0; e < N; ++e) w[e] = x[e] > s.least ? w[e] : s.from + s.lowest;
    }
    double shift = s.shift;
    if (CARE && s.careful) {
        shift = kShift;
#pragma unroll
        for (int e = 0; e < N; ++e) {
            w[e] -= s.from;
            w[e] = fabsf(x[e]) < INFINITY && w[e] >= s.lowest ? w[e] : s.lowest;
        }
    }
    warp_exp2(w, s.k, shift, s.table, base);
}
// One logit by all lanes, whatever it is and what the others are.
template <bool CAP>
__device__ __forceinline__ double warp_logit64(const Scale& s, float x) {
    if constexpr (!CAP) return (double)x;
    const float its[1] = {x};
    double near[1];
    near_capped(its, s.inverse, near);
    const bool finite = fabsf(x) < INFINITY, far = finite && fabsf(x) > (float)s.cap;
    if (__any_sync(kFullMask, far)) {              // seldom
        const float edge = 20.0f * (float)s.cap;
        double d[1] = {(double)fminf(fmaxf(x, -edge), edge)};
        warp_exp2(d, s.twice, s.table);
        if (far) near[0] = s.cap - 2.0 * s.cap / (d[0] + 1.0);
    }
    return finite ? near[0] : -INFINITY;
}
__device__ __forceinline__ double warp_weight(const Scale& s, double logit) {
    const double y = logit - s.from;
    const bool is = y * s.k >= -32000.0;               // not for NaN
    double w[1] = {is ? y : 0.0};
    warp_exp2(w, s.k, s.table);
    return is ? w[0] : 0.0;
}
template <bool CAP>
__device__ __forceinline__ void Scale::relative_to(float top, bool infinite) {
    from = top > -INFINITY ? unit(warp_logit64<CAP>(*this, top)) : 0.0;
    shift = kShift - rint(from * k);                   // exact where no care is needed
    const double bottom = from + lowest;
    if (CAP) {
        // the cap's inverse, cap atanh(bottom / cap); 2^-23 of the cap is the widest step of its logits. Beyond 5700 T of cap what the quotients are off by would move weights by more than 6e-10,
        // which counts where the logits are far below the cap: near it, so cold a row has few tokens (33 trees capped at 30 with T = 0.01 take 76 us, carefully 99).
        careful = infinite || cap * 0x1p-22 * k > 320.0 || (cap * k > 0x1p18 && fabs((double)top) * 64.0 < cap);
        least = bottom > -cap && !careful ? (float)(0.5 * cap * log((cap + bottom) / (cap - bottom))) : -INFINITY;
    } else {
        careful = infinite || bottom < -3.4028234e38 || fabs(from) * 0x1p-22 * k > 320.0;
        least = careful ? -3.4028234e38f : (float)bottom;
    }
}

// ---------------------------------------------------------------------------
// all rows in 64 bits
// ---------------------------------------------------------------------------
//
// Where there are few logits, or one row a sequence: the same sums for every row, in 64 bits, by blocks all over the chip. The walk then needs no sum but those behind
// a refusal, and a draw no more than a part's logits again. Eight 64-bit operations a logit (23 capped) at 64 a clock and SM would let 2.2e12 logits a second through (8e11), HBM 3.3e12 of 16 bits;
// 200 rows of 262144 take 76 us with their draws (177 capped), 7e11 (3e11): conversions, the table's shuffles and latencies, not one unit. A block with a capped logit wider than the cap, -infinity among
// them, goes the long way: 208 us where all but 64 logits of a row are masked.
constexpr int kMostPieces = 8;

template <typename T, bool CAP>
__global__ void __launch_bounds__(kStatsThreads, 2) verify_sums_kernel(const __grid_constant__ VerifyArgs a) {
    pdl_launch_dependents();
    using R = Row<T>;
    constexpr int E = R::E, WARPS = kStatsThreads / kWarp;
    __shared__ uint32_t found, best, infinite;
    __shared__ float warp_most[WARPS];
    __shared__ double warp_sum_[WARPS];
    const uint32_t tid = threadIdx.x, warp = tid / kWarp, lane = tid % kWarp;
    const uint32_t row = blockIdx.x / a.parts, part = blockIdx.x % a.parts;
    const R r(a.logits, row * a.stride, a.vocab);
    const uint32_t piece = part * a.per * kStatsThreads + tid;
    uint4 w[kMostPieces];
#pragma unroll
    for (int j = 0; j < kMostPieces; ++j) w[j] = (uint32_t)j < a.per ? r.load(piece + j * kStatsThreads) : R::nothing();
    if (tid == 0) {
        found = best = 0xFFFFFFFFu;
        infinite = 0;
    }
    __syncthreads();
    owner_of(a, row, &found);
    float most = -INFINITY, widest = 0.0f;
#pragma unroll
    for (int j = 0; j < kMostPieces; ++j) {
        float top = R::most(w[j]);
        if (CAP && (uint32_t)j < a.per) widest = fmaxf(widest, R::most(R::magnitudes(w[j])));
        if (top == INFINITY) {
            infinite = 1;
            float x[E];
            R::numbers(w[j], x);
            top = -INFINITY;
#pragma unroll
            for (int e = 0; e < E; ++e) top = fmaxf(top, counted(x[e]));
        }
        most = fmaxf(most, top);
    }
    float top = most;
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) top = fmaxf(top, __shfl_xor_sync(kFullMask, top, off));
    if (lane == 0) warp_most[warp] = top;
    __syncthreads();
    const uint32_t b = found;
    if (b == 0xFFFFFFFFu) return;
    top = lane < WARPS ? warp_most[lane] : -INFINITY;
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) top = fmaxf(top, __shfl_xor_sync(kFullMask, top, off));
    const Heat heat(a, b, kWaited);
    Scale scale;
    scale.set<CAP>(a.softcap, heat.k, lane);
    scale.relative_to<CAP>(top, infinite);
    const bool far = CAP && __any_sync(kFullMask, !(widest <= a.softcap));     // masked ones too: a block with them goes the long way
    double sums[4] = {};
    if (top > -INFINITY) {
#pragma unroll
        for (int j = 0; j < kMostPieces; ++j) {
            if ((uint32_t)j >= a.per) break;
            float x[E];
            R::numbers(w[j], x);
#pragma unroll
            for (int h = 0; h < E; h += 4) {
                float some[4];
                double v[4], base[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) some[e] = x[h + e];
                if (CAP && !far && !scale.careful) warp_weights<CAP, 4, false, CAP>(scale, some, v, base);
                else warp_weights<CAP>(scale, some, v, base);
#pragma unroll
                for (int e = 0; e < 4; ++e) sums[e] = fma(base[e], v[e], sums[e]);
            }
        }
        if (heat.greedy && most == top) {
            uint32_t at = 0xFFFFFFFFu;
#pragma unroll
            for (int j = kMostPieces - 1; j >= 0; --j) {
                float x[E];
                R::numbers(w[j], x);
#pragma unroll
                for (int e = E - 1; e >= 0; --e)
                    if ((uint32_t)j < a.per && x[e] == top) at = (uint32_t)(r.first(piece + j * kStatsThreads) + e);
            }
            atomicMin(&best, at);
        }
    }
    __syncwarp();
    double sum = (sums[0] + sums[1]) + (sums[2] + sums[3]);
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) sum += __shfl_xor_sync(kFullMask, sum, off);
    if (lane == 0) warp_sum_[warp] = sum;
    __syncthreads();
    if (tid == 0) {
        sum = 0.0;
        for (int i = 0; i < WARPS; ++i) sum += warp_sum_[i];
        a.stats[(size_t)row * a.parts + part] = {sum, top, best, infinite, 0};
    }
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

// The first block's shared memory: what it knows of the nodes.
struct NodeTable {
    double *z, *weight;        // of a row: its sum in 32 bits; of a token: its weight in its parent's row
    double* gone;              // of the current node's refused children: S before each, or (as int32) the tokens
    float *most, *prob, *number;           // number: the random one
    uint32_t* best;
    int32_t *parent, *token, *inner;       // inner: has children; -1 - place of a kept node
    __device__ __forceinline__ NodeTable(uint8_t* memory, uint32_t n) {
        z = reinterpret_cast<double*>(memory);
        weight = z + n;
        gone = weight + n;
        most = reinterpret_cast<float*>(gone + n);
        prob = most + n;
        number = prob + n;
        best = reinterpret_cast<uint32_t*>(number + n);
        parent = reinterpret_cast<int32_t*>(best + n);
        token = parent + n;
        inner = token + n;
    }
    static constexpr size_t kBytes = 52;
};

// Before the wait
__device__ __forceinline__ float prob_at(const VerifyArgs& a, uint64_t at) {
    float q;
    if (a.probs_dtype == TF_FP32) q = EarlyTable<float>{static_cast<const float*>(a.probs)}.at<true>(at);
    else if (a.probs_dtype == TF_FP16) q = __half2float(EarlyTable<__half>{static_cast<const __half*>(a.probs)}.at<true>(at));
    else q = __bfloat162float(EarlyTable<__nv_bfloat16>{static_cast<const __nv_bfloat16*>(a.probs)}.at<true>(at));
    return fmaxf(q, 0.0f);     // NaN too
}
// A node's row of probabilities by the pieces of its logits.
template <typename T>
struct ProbRow {
    static constexpr int E = Row<T>::E;
    uint64_t at;
    bool even;                 // a piece's lie at a boundary of as many bytes, up to 16
    __device__ __forceinline__ ProbRow(const VerifyArgs& a, uint64_t row, uint32_t lead) : at(row - lead) {
        const uint32_t size = a.probs_dtype == TF_FP32 ? 4 : 2;
        even = (reinterpret_cast<uintptr_t>(a.probs) + at * size) % (size * E < 16 ? size * E : 16) == 0;
    }
    static constexpr int WORDS = E / 4;        // a piece's as 32-bit numbers; 16-bit ones take half of it
    __device__ __forceinline__ void load(const VerifyArgs& a, const Row<T>& row, uint32_t piece, uint4 (&w)[WORDS]) const {
        const uint64_t from = at + (uint64_t)piece * E;
        const bool whole = even && piece - row.whole0 < row.whole;
        const int64_t first = row.first(piece);
        if (a.probs_dtype == TF_FP32) {
            const float* p = static_cast<const float*>(a.probs) + from;
            if (whole) {
#pragma unroll
                for (int i = 0; i < WORDS; ++i) w[i] = reinterpret_cast<const uint4*>(p)[i];
            } else {
                float v[E];
#pragma unroll
                for (int e = 0; e < E; ++e) v[e] = first + e >= 0 && first + e < (int64_t)row.vocab ? p[e] : 0.0f;
                memcpy(w, v, sizeof(v));
            }
        } else {
            const uint16_t* p = static_cast<const uint16_t*>(a.probs) + from;
            if (whole) {
                if constexpr (E == 8) {
                    w[0] = *reinterpret_cast<const uint4*>(p);
                } else {
                    const uint2 v = *reinterpret_cast<const uint2*>(p);
                    w[0].x = v.x;
                    w[0].y = v.y;
                }
            } else {
                uint16_t v[E];
#pragma unroll
                for (int e = 0; e < E; ++e) v[e] = first + e >= 0 && first + e < (int64_t)row.vocab ? p[e] : (uint16_t)0;
                memcpy(w, v, sizeof(v));
            }
        }
    }
    static __device__ __forceinline__ void numbers(const VerifyArgs& a, const uint4 (&w)[WORDS], float (&q)[E]) {
        if (a.probs_dtype == TF_FP32) {
            memcpy(q, w, sizeof(q));
        } else {
            uint16_t v[E];
            memcpy(v, w, sizeof(v));
#pragma unroll
            for (int e = 0; e < E; ++e) q[e] = a.probs_dtype == TF_FP16 ? f16_bits_to_float(v[e]) : bf16_bits_to_float(v[e]);
        }
#pragma unroll
        for (int e = 0; e < E; ++e) q[e] = fmaxf(q[e], 0.0f);
    }
};

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
    const uint32_t any = __ballot_sync(kFullMask, part > kNothing), over = __ballot_sync(kFullMask, part > kNothing && upto > target);
    const uint32_t who = over ? __ffs(over) - 1 : any ? 31 - __clz(any) : 0;
    const double before = __shfl_sync(kFullMask, upto - part, who);
    target = over ? target - before : INFINITY;
    return who;
}

// One thread goes from node to node until a sum over the vocabulary is needed, or the walk is over. A child's test goes through all refusals of its siblings before it: 63 refused ones without q
// over 2000 logits take 0.18 ms in all, 255 0.47, 1023 3.6.
template <bool CAP>
__device__ __forceinline__ void walk_on(const VerifyArgs& a, const Nodes& of, const Heat& heat, uint32_t b, const NodeTable& t, Walk& walk, Order& order,
                                        int32_t* out_tokens, int32_t* out_rows) {
    Walk w = walk;                                     // in registers: it was most of the walk to fetch it back and forth
    const double bound = sum_bound(a.softcap, heat.k);
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
            const double u = (double)t.number[i], weight = t.weight[i];
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
                walk = w;
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
            w.refused = w.step = 0;
            w.summed = a.exact;
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
    walk = w;
    if (heat.greedy) {
        out_tokens[w.at] = (int32_t)t.best[w.node];
        if (a.logprobs) a.logprobs[(size_t)b * a.draft_stride + w.at] = w.z > 0.0 ? (float)-log(w.z) : -INFINITY;
        return;
    }
    order = {2, w.node, w.at, w.known, w.summed, w.step, a.probs && w.node < a.probs_nodes, w.refused, t.most[w.node], t.number[0], w.z, w.s};
}

// What the refused children of a node leave of its weights: without q the refused tokens are left out, with q each refusal takes its sum times q.
struct Refused {
    int count;
    bool drawn;
    const double* gone;        // in shared memory: sums, or (as int32) tokens
};

// Sums of a lane's pieces, every `per` steps apart in `parts` too (kWalkThreads apart), where that is given.
struct Tally {
    double all = 0.0, part = 0.0;
    double* parts;
    uint32_t per, until;
    __device__ __forceinline__ void add(double v) {
        part += v;
        if (--until == 0) close();
    }
    __device__ __forceinline__ void close() {
        all += part;
        if (parts) {
            *parts = part;
            parts += kWalkThreads;
        }
        part = 0.0;
        until = per;
    }
};

// The weights of one piece, wherever it lies, and their sum.
template <typename T, bool CAP>
__device__ __noinline__ double one_step(const VerifyArgs& a, const Row<T>& row, const ProbRow<T>& probs, const Refused& r, const Scale& s, uint32_t piece, double (&w)[Row<T>::E]) {
    using P = ProbRow<T>;
    constexpr int E = Row<T>::E;
    float x[E], q[E];
    Row<T>::numbers(row.load(piece), x);
    if (r.drawn) {
        uint4 raw[P::WORDS] = {};
        probs.load(a, row, piece, raw);
        P::numbers(a, raw, q);
    }
    double all = 0.0;
#pragma unroll
    for (int h = 0; h < E; h += 4) {
        float some[4];
        double v[4], base[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) some[e] = x[h + e];
        warp_weights<CAP>(s, some, v, base);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] *= base[e];
        for (int g = 0; g < r.count; ++g) {
            if (r.drawn) {
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = positive(fma(-r.gone[g], (double)q[h + e], v[e]));
            } else {
                const int64_t e0 = (int64_t) reinterpret_cast<const int32_t*>(r.gone)[g] - row.first(piece);
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = e0 == h + e ? 0.0 : v[e];
            }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            all += v[e];
            w[h + e] = v[e];
        }
    }
    return all;
}

// Where the time goes: `steps` whole pieces from p on, a warp apart, whose weights need no care. Nothing but this in a function, without a branch on what a call fixes: as a part of the walk, with the
// edges' checks, 64 chains of seven took 138 us; as a function 127, without the checks 114. Eight operations of 64 bits a logit, two more
// a refusal, 23 capped; a step takes 205 clocks a warp with four warps a sub-core, by issue slots and latencies together (without loads, shuffles and most of the series still 150). Q: the type of q, 0 none, else as tf_dtype + 1; EVEN: q's pieces lie at boundaries.
template <typename T, bool CAP, int Q, bool EVEN>
__device__ __noinline__ void many_steps(const uint4* p, const void* q_at, uint32_t steps, int32_t first, const Refused& refused, const Scale& by, Tally& tally) {
    constexpr int E = Row<T>::E, WORDS = Q == 0 ? 1 : Q == TF_FP32 + 1 ? E / 4 : 1;
    using V = std::conditional_t<Q == TF_FP32 + 1, float, std::conditional_t<Q == TF_FP16 + 1, __half, __nv_bfloat16>>;
    const Scale s = by;
    const Refused r = refused;
    Tally t = tally;
    const V* q = static_cast<const V*>(q_at);
    auto load_q = [&](const V* from, uint4 (&w)[WORDS]) {
        if constexpr (Q == 0) {
        } else if constexpr (!EVEN) {
            V v[E];
#pragma unroll
            for (int e = 0; e < E; ++e) v[e] = from[e];
            memcpy(w, v, sizeof(v));
        } else if constexpr (E * sizeof(V) == 8) {
            memcpy(w, static_cast<const uint2*>(static_cast<const void*>(from)), 8);
        } else {
#pragma unroll
            for (int i = 0; i < WORDS; ++i) w[i] = reinterpret_cast<const uint4*>(from)[i];
        }
    };
    // The first eight steps towards L2, a line of 128 bytes a lane: where there are no more, all of HBM's latency is met at once. (In the loop it cost more than it brought.)
    const uint32_t lane = threadIdx.x % kWarp, some = min(steps, 8u);
    if (lane * 128 < some * kWarp * 16) asm volatile("prefetch.global.L2 [%0];" ::"l"(reinterpret_cast<const uint8_t*>(p - lane) + lane * 128));
    if constexpr (Q != 0) {
        constexpr uint32_t kBytes = kWarp * E * sizeof(V);
#pragma unroll
        for (uint32_t at = 0; at < 8 * kBytes; at += kWarp * 128)
            if (at + lane * 128 < some * kBytes) asm volatile("prefetch.global.L2 [%0];" ::"l"(reinterpret_cast<const uint8_t*>(q - lane * E) + at + lane * 128));
    }
    double sums[4] = {};                           // without q: the products' sums so far
    // the next two steps' logits and probabilities are on their way
    uint4 next[2] = {p[0], steps > 1 ? p[kWarp] : p[0]}, next_q[2][WORDS] = {};
    if constexpr (Q != 0) {
        load_q(q, next_q[0]);
        if (steps > 1) load_q(q + E * kWarp, next_q[1]);
    }
#pragma unroll 1
    for (; steps; --steps) {
        float x[E], u[E];
        Row<T>::numbers(next[0], x);
        // wider than the cap: a whole warp's step the long way
        const bool far = CAP && __any_sync(kFullMask, Row<T>::most(Row<T>::magnitudes(next[0])) > (float)s.cap);
        next[0] = next[1];
        p += kWarp;
        if (steps > 2) next[1] = p[kWarp];
        if constexpr (Q != 0) {
            V v[E];
            memcpy(v, next_q[0], sizeof(v));
#pragma unroll
            for (int e = 0; e < E; ++e) u[e] = fmaxf(number(v[e]), 0.0f);
#pragma unroll
            for (int i = 0; i < WORDS; ++i) next_q[0][i] = next_q[1][i];
            q += E * kWarp;
            if (steps > 2) load_q(q + E * kWarp, next_q[1]);
        }
        constexpr int N = CAP ? 4 : E;             // capped, eight at once take more registers than there are
        double w[E], base[E];
#pragma unroll
        for (int h = 0; h < E; h += N) {
            float some[N];
            double v[N], its[N];
#pragma unroll
            for (int e = 0; e < N; ++e) some[e] = x[h + e];
            if (CAP && far) warp_weights<CAP, N, false>(s, some, v, its);
            else warp_weights<CAP, N, false, CAP>(s, some, v, its);
#pragma unroll
            for (int e = 0; e < N; ++e) {
                w[h + e] = v[e];
                base[h + e] = its[e];
            }
        }
        if constexpr (Q != 0) {
#pragma unroll
            for (int e = 0; e < E; ++e) w[e] *= base[e];
#pragma unroll 1
            for (int g = 0; g < r.count; ++g) {
                const double taken = r.gone[g];
#pragma unroll
                for (int e = 0; e < E; ++e) w[e] = positive(fma(-taken, (double)u[e], w[e]));
            }
            if constexpr (E == 8) t.add(((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7])));
            else t.add((w[0] + w[1]) + (w[2] + w[3]));
        } else {
#pragma unroll 1
            for (int g = 0; g < r.count; ++g) {
                const uint32_t at = (uint32_t)(reinterpret_cast<const int32_t*>(r.gone)[g] - first);
                if (at < E)
#pragma unroll
                    for (int e = 0; e < E; ++e) base[e] = at == e ? 0.0 : base[e];
            }
            first += E * kWarp;
#pragma unroll
            for (int e = 0; e < E; ++e) sums[e % 4] = fma(base[e], w[e], sums[e % 4]);
            if (--t.until == 0) {
                t.part += (sums[0] + sums[1]) + (sums[2] + sums[3]);
                sums[0] = sums[1] = sums[2] = sums[3] = 0.0;
                t.close();
            }
        }
    }
    t.part += (sums[0] + sums[1]) + (sums[2] + sums[3]);
    tally = t;
}

// The sum of what is left of the weights of `steps` pieces, a warp apart, from `piece` on, with the sums of every `per` in `parts`: room for one more than there are.
template <typename T, bool CAP>
__device__ __forceinline__ double sum_steps(const VerifyArgs& a, const Row<T>& row, const ProbRow<T>& probs, const Refused& r, const Scale& s, uint32_t piece, uint32_t steps,
                                            double* parts, uint32_t per) {
    constexpr int E = Row<T>::E;
    Tally t;
    t.parts = parts;
    t.per = t.until = per;
    const uint32_t piece0 = piece - threadIdx.x % kWarp, end = row.whole0 + row.whole;
    // steps of whole pieces; a row's first and last ones, and all of a row that needs care, go one by one
    const uint32_t lo = min(piece0 < row.whole0 || s.careful ? (s.careful ? steps : 1u) : 0u, steps), hi = max(lo, min(end > piece0 ? (end - piece0) / kWarp : 0u, steps));
    for (uint32_t i = 0; i < steps;) {
        if (i == lo && hi > lo) {
            const uint32_t at = piece + lo * kWarp;
            const uint4* p = row.base + at;
            const void* q = static_cast<const uint8_t*>(a.probs) + (probs.at + (uint64_t)at * E) * (a.probs_dtype == TF_FP32 ? 4 : 2);
            const int32_t first = (int32_t)row.first(at);
            switch (r.drawn ? (int)a.probs_dtype + 1 : 0) {
                case 0: many_steps<T, CAP, 0, true>(p, q, hi - lo, first, r, s, t); break;
                case TF_FP32 + 1: probs.even ? many_steps<T, CAP, TF_FP32 + 1, true>(p, q, hi - lo, first, r, s, t) : many_steps<T, CAP, TF_FP32 + 1, false>(p, q, hi - lo, first, r, s, t); break;
                case TF_FP16 + 1: probs.even ? many_steps<T, CAP, TF_FP16 + 1, true>(p, q, hi - lo, first, r, s, t) : many_steps<T, CAP, TF_FP16 + 1, false>(p, q, hi - lo, first, r, s, t); break;
                default: probs.even ? many_steps<T, CAP, TF_BF16 + 1, true>(p, q, hi - lo, first, r, s, t) : many_steps<T, CAP, TF_BF16 + 1, false>(p, q, hi - lo, first, r, s, t);
            }
            i = hi;
        } else {
            double w[E];
            t.add(piece0 + i * kWarp < row.pieces() ? one_step<T, CAP>(a, row, probs, r, s, piece + i * kWarp, w) : 0.0);
            ++i;
        }
    }
    t.close();
    return t.all;
}

// The weight of a part of a row whose 64-bit sums these are, relative to s.from; by all lanes.
template <bool CAP>
__device__ __forceinline__ double part_weight(const Scale& s, const ChunkStat* stats, uint32_t c, uint32_t parts) {
    ChunkStat x = {0.0, -INFINITY, 0, 0, 0};
    if (c < parts) x = stats[c];
    return x.sum * warp_weight(s, s.unit(warp_logit64<CAP>(s, x.most)));       // 0 where there is no finite logit
}

// The part that the target falls in, from the sums of the first launch, by all lanes. The target becomes that within the part, and the scale the part's.
template <bool CAP>
__device__ __forceinline__ uint32_t part_of(Scale& scale, const ChunkStat* s, uint32_t parts, double& target) {
    uint32_t last = 0;
    double before = 0.0, of_last = 0.0;
    bool hit = false;
    for (uint32_t c0 = 0; c0 < parts && !hit; c0 += kWarp) {
        const uint32_t lane = threadIdx.x % kWarp;
        const double mine = part_weight<CAP>(scale, s, c0 + lane, parts), run = before + warp_scan(mine, lane);
        const uint32_t any = __ballot_sync(kFullMask, mine > kNothing), over = __ballot_sync(kFullMask, mine > kNothing && run > target);
        hit = over != 0;
        if (any) {                                     // behind the last one that has anything: its last token
            const uint32_t who = hit ? __ffs(over) - 1 : 31 - __clz(any);
            last = c0 + who;
            of_last = __shfl_sync(kFullMask, run - mine, who);
        }
        before = __shfl_sync(kFullMask, run, kWarp - 1);
    }
    const ChunkStat part = s[last];
    const double share = warp_weight(scale, scale.unit(warp_logit64<CAP>(scale, part.most)));
    target = hit ? (target - of_last) / share : INFINITY;
    scale.relative_to<CAP>(part.most, part.infinite);
    return last;
}

// One row a sequence: nothing to walk, and all that a draw needs is there. A block takes the part that the token lies in as the first launch did, all its logits at once, and sums them by steps
// of a warp; the step's warp draws. Latency bounds it: six loads, one after another, and what stands between them. A token of 262144 takes 13.6 us
// in all and 1000 rows of 300 34; by the walk, which goes from part to token in three readings, 15.5 and 93.
template <typename T, bool CAP>
__global__ void __launch_bounds__(kStatsThreads, 2) verify_lone_kernel(const __grid_constant__ VerifyArgs a) {
    using R = Row<T>;
    constexpr int E = R::E, WARPS = kStatsThreads / kWarp;
    static_assert(kMostPieces * WARPS == 2 * kWarp, "two steps a lane");
    constexpr double kLn2 = 0.69314718055994530942;
    __shared__ double step_sum[kMostPieces * WARPS];
    const uint32_t tid = threadIdx.x, warp = tid / kWarp, lane = tid % kWarp, b = blockIdx.x;
    if (a.parts == 0) pdl_wait();
    const Nodes of(a, b, tid == 0, kEarly);
    const Heat heat(a, b, kEarly);
    const double u = (double)uniform(a.uniforms.at<true>(b));
    Scale scale;
    scale.set<CAP>(a.softcap, heat.k, lane);
    if (a.parts) pdl_wait();
    if (tid == 0) {
        a.out_rows[b] = of.n ? 0 : -1;
        a.kept[b] = of.n;
    }
    auto leave = [&](int32_t token, float logprob) {
        a.out_tokens[b] = token;
        if (a.logprobs) a.logprobs[b] = logprob;
    };
    if (of.n == 0) {
        if (tid == 0) leave(-1, 0.0f);
        return;
    }
    const ChunkStat* s = a.stats + (size_t)of.row0 * a.parts;
    float top = -INFINITY;
    for (uint32_t c = lane; c < a.parts; c += kWarp) top = fmaxf(top, s[c].most);
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) top = fmaxf(top, __shfl_xor_sync(kFullMask, top, off));
    const double logit = warp_logit64<CAP>(scale, top);
    scale.from = heat.greedy ? logit : scale.unit(logit);
    double z = 0.0;
    for (uint32_t c0 = 0; c0 < a.parts; c0 += kWarp) z += part_weight<CAP>(scale, s, c0 + lane, a.parts);
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) z += __shfl_xor_sync(kFullMask, z, off);
    if (heat.greedy) {
        uint32_t at = 0xFFFFFFFFu;
        for (uint32_t c = lane; c < a.parts; c += kWarp)
            if (s[c].most == top) at = min(at, s[c].at);
        at = __reduce_min_sync(kFullMask, at);
        if (tid == 0) leave(at == 0xFFFFFFFFu ? 0 : (int32_t)at, z > 0.0 ? (float)-log(z) : -INFINITY);
        return;
    }
    if (!(z > kNothing)) {
        if (tid == 0) leave(0, -INFINITY);
        return;
    }
    const double whole = scale.from;
    double target = u * z;
    const uint32_t part = part_of<CAP>(scale, s, a.parts, target);
    const R row(a.logits, of.row0 * a.stride, a.vocab);
    const uint32_t piece = part * a.per * kStatsThreads + tid;
    uint4 w[kMostPieces];
#pragma unroll
    for (int j = 0; j < kMostPieces; ++j) w[j] = (uint32_t)j < a.per ? row.load(piece + j * kStatsThreads) : R::nothing();
    bool far = false;
#pragma unroll
    for (int j = 0; j < kMostPieces; ++j)
        if (CAP && (uint32_t)j < a.per) far |= !(R::most(R::magnitudes(w[j])) <= a.softcap);
    far = CAP && __any_sync(kFullMask, far);
#pragma unroll
    for (int j = 0; j < kMostPieces; ++j) {
        if ((uint32_t)j >= a.per) {
            if (lane == 0) step_sum[j * WARPS + warp] = 0.0;
            continue;
        }
        double sums[4] = {};
        float x[E];
        R::numbers(w[j], x);
#pragma unroll
        for (int h = 0; h < E; h += 4) {
            float some[4];
            double v[4], base[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) some[e] = x[h + e];
            if (CAP && !far && !scale.careful) warp_weights<CAP, 4, false, CAP>(scale, some, v, base);
            else warp_weights<CAP>(scale, some, v, base);
#pragma unroll
            for (int e = 0; e < 4; ++e) sums[e] = fma(base[e], v[e], sums[e]);
        }
        double sum = (sums[0] + sums[1]) + (sums[2] + sums[3]);
#pragma unroll
        for (int off = 16; off >= 1; off >>= 1) sum += __shfl_xor_sync(kFullMask, sum, off);
        if (lane == 0) step_sum[j * WARPS + warp] = sum;
    }
    __syncthreads();
    const double first = step_sum[2 * lane], second = step_sum[2 * lane + 1], pair = first + second;
    const uint32_t who = warp_fall(pair, warp_scan(pair, lane), target);
    const double one = __shfl_sync(kFullMask, first, who), two = __shfl_sync(kFullMask, second, who);
    uint32_t step = 2 * who;
    if (!(one > kNothing && (one > target || !(two > kNothing)))) {
        step += 1;
        target -= one;
    }
    if (warp != step % WARPS) return;
    const uint32_t mine = piece + step / WARPS * kStatsThreads;
    float x[E];
    R::numbers(row.load(mine), x);
    double v[E], all = 0.0;
#pragma unroll
    for (int h = 0; h < E; h += 4) {
        float some[4];
        double some_v[4], base[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) some[e] = x[h + e];
        if (CAP && !far && !scale.careful) warp_weights<CAP, 4, false, CAP>(scale, some, some_v, base);
        else warp_weights<CAP>(scale, some, some_v, base);
#pragma unroll
        for (int e = 0; e < 4; ++e) all += v[h + e] = some_v[e] * base[e];
    }
    if (warp_fall(all, warp_scan(all, lane), target) != lane) return;
    double at = 0.0;
    int found = -1, end = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        at += v[e];
        if (v[e] > kNothing / 8) {                 // of a lane that has more than kNothing one has
            end = e;
            if (found < 0 && at > target) found = e;
        }
    }
    const int64_t token = row.inside(row.first(mine) + (found < 0 ? end : found));
    leave((int32_t)token, a.logprobs ? (float)((logit64<CAP>(number(row.p[token]), a.softcap) - whole) * heat.k * kLn2 - log(z)) : 0.0f);
}

template <typename T, bool CAP>
__global__ void __launch_bounds__(kWalkThreads, 2) verify_walk_kernel(const __grid_constant__ VerifyArgs a) {
    using R = Row<T>;
    using P = ProbRow<T>;
    constexpr int E = R::E;
    extern __shared__ __align__(16) uint8_t dynamic[];
    __shared__ Order orders[2];                    // by turns: one is read while the next is written
    __shared__ Walk walk;
    __shared__ double block_sum[2], warp_part[kWalkWarps], parts[(kGroups + 1) * kWalkThreads];
    __shared__ float block_most[2], warp_most[kWalkWarps];
    const cg::cluster_group cluster = cg::this_cluster();
    const uint32_t tid = threadIdx.x, warp = tid / kWarp, lane = tid % kWarp;
    const uint32_t rank = cluster.block_rank(), ranks = cluster.num_blocks(), b = blockIdx.x / ranks;
    Scale scale;
    // The first launch starts when what came before it has ended and writes nothing but its sums: all else may be read while it is at work, past L1.
    if (a.parts == 0) pdl_wait();
    const Nodes of(a, b, rank == 0 && tid == 0, kEarly);
    const Heat heat(a, b, kEarly);
    const NodeTable nodes(dynamic, a.draft_stride);
    int32_t* gone_tokens = reinterpret_cast<int32_t*>(nodes.gone);
    int32_t* out_tokens = a.out_tokens + (size_t)b * a.draft_stride;
    int32_t* out_rows = a.out_rows + (size_t)b * a.draft_stride;
    float* logprobs = a.logprobs ? a.logprobs + (size_t)b * a.draft_stride : nullptr;
    scale.set<CAP>(a.softcap, heat.k, lane);
    constexpr double kLn2 = 0.69314718055994530942;
    if (tid == 0) walk = {1, 0, 0, 0, 0, 0, 0, 0.0, 0.0, 0.0};

    if (rank == 0) {
        for (uint32_t i = tid; i < of.n; i += kWalkThreads) nodes.inner[i] = 0;
        __syncthreads();
        for (uint32_t i = tid; i < of.n; i += kWalkThreads) {
            const int32_t x = a.tokens.at<true>((size_t)b * a.draft_stride + i), p = i ? parent_of(a, b, i, kEarly) : -1;
            const bool token = x >= 0 && (uint32_t)x < a.vocab;
            nodes.parent[i] = p;
            nodes.token[i] = token ? x : -1;
            nodes.number[i] = uniform(a.uniforms.at<true>((size_t)b * a.draft_stride + i));
            if (p < 0) continue;
            atomicOr(nodes.inner + p, 1);
            if (!token) continue;
            const EarlyTable<T> logits{static_cast<const T*>(a.logits)};
            nodes.weight[i] = (double)counted(number(logits.template at<true>((of.row0 + (uint64_t)p) * a.stride + x)));     // for now
            nodes.prob[i] = a.probs && (uint32_t)p < a.probs_nodes ? prob_at(a, b * a.probs_sequence + p * a.probs_node + x) : 0.0f;
        }
        if (a.parts) pdl_wait();
        // A leaf's numbers are whatever an earlier call left: nobody looks at them.
        for (uint32_t i = warp; i < of.n; i += kWalkWarps) {
            const ChunkStat* s = a.stats + (size_t)(of.row0 + i) * a.parts;
            float top = -INFINITY;
            uint32_t at = 0xFFFFFFFFu, infinite = 0;
            for (uint32_t c = lane; c < a.parts; c += kWarp) {
                const ChunkStat x = s[c];
                if (x.most > top) { top = x.most; at = x.at; }                 // parts ascend: the first of equals stays
                infinite |= x.infinite;
            }
            float all = top;
#pragma unroll
            for (int off = 16; off >= 1; off >>= 1) all = fmaxf(all, __shfl_xor_sync(kFullMask, all, off));
            if (top != all) at = 0xFFFFFFFFu;
            at = __reduce_min_sync(kFullMask, at);
            const float from = CAP ? capped(all, a.softcap) : all, k32 = heat.k32();
            double sum = 0.0;
            // Relative to the unit of the row, but of a greedy sequence to the largest itself, whose weight is what is asked for
            const double logit = warp_logit64<CAP>(scale, all);
            scale.from = heat.greedy ? logit : scale.unit(logit);
            if (a.exact) {
                for (uint32_t c0 = 0; c0 < a.parts; c0 += kWarp) sum += part_weight<CAP>(scale, s, c0 + lane, a.parts);
            } else {
                for (uint32_t c = lane; c < a.parts; c += kWarp) {
                    const ChunkStat x = s[c];
                    if (x.most > -INFINITY) sum += (double)((float)x.sum * verify_exp2(((CAP ? capped(x.most, a.softcap) : x.most) - from) * k32));
                }
                sum *= warp_weight(scale, logit);
            }
#pragma unroll
            for (int off = 16; off >= 1; off >>= 1) sum += __shfl_xor_sync(kFullMask, sum, off);
            if (lane == 0) {
                nodes.most[i] = all;
                nodes.z[i] = sum;
                nodes.best[i] = at == 0xFFFFFFFFu ? 0u : at;
            }
            infinite = (__any_sync(kFullMask, infinite) ? 2u : 0u) | (a.exact ? 1u : 0u);
            if (infinite && lane == 0) atomicOr(nodes.inner + i, (int)infinite);
        }
        __syncthreads();
        for (uint32_t i0 = warp * kWarp; i0 < of.n; i0 += kWalkThreads) {
            const uint32_t i = i0 + lane;
            const bool is = i < of.n && nodes.parent[i] >= 0 && nodes.token[i] >= 0;
            const float x = is ? (float)nodes.weight[i] : -INFINITY, top = is ? nodes.most[nodes.parent[i]] : -INFINITY;
            const double l = warp_logit64<CAP>(scale, x);
            scale.from = scale.unit(warp_logit64<CAP>(scale, top));
            const double w = warp_weight(scale, l);    // of infinities and NaN: 0
            if (is) nodes.weight[i] = w;
        }
        __syncthreads();
        if (tid == 0 && of.n) {
            walk.z = nodes.z[0];
            walk.known = nodes.inner[0];               // a leaf may have the second bit of another call's row: no matter
            walk.summed = a.exact;
        }
    } else if (a.parts) {
        pdl_wait();                                    // before anything is written
    }
    __syncthreads();

    for (uint32_t round = 0, turn = 0;; ++round) {
        if (rank == 0 && tid == 0) walk_on<CAP>(a, of, heat, b, nodes, walk, orders[round & 1], out_tokens, out_rows);
        __syncwarp();
        cluster.sync();
        const Order o = *cluster.map_shared_rank(&orders[round & 1], 0);
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
        const P probs(a, b * a.probs_sequence + o.node * a.probs_node, row.lead);
        uint32_t begin = rank * kWalkWarps * steps * kWarp;
        const uint32_t per = (steps + kGroups - 1) / kGroups;  // steps whose sum is kept for the draw
        // A row without a maximum (a leaf: nothing was refused) is summed by every block relative to its own, one meeting less.
        float top = o.most;
        bool infinite = o.known & 2;
        if (!(o.known & 1)) {
            top = -INFINITY;
            infinite = false;
            constexpr int LOADS = 8;
            for (uint32_t i = 0, piece = begin + warp * steps * kWarp + lane; i < steps && piece < pieces; i += LOADS, piece += LOADS * kWarp) {
                uint4 w[LOADS];
#pragma unroll
                for (int j = 0; j < LOADS; ++j) w[j] = i + j < steps && piece + j * kWarp < pieces ? row.load(piece + j * kWarp) : R::nothing();
#pragma unroll
                for (int j = 0; j < LOADS; ++j) {
                    float most = R::most(w[j]);
                    if (most == INFINITY) {            // does not count
                        float x[E];
                        R::numbers(w[j], x);
                        infinite = true;
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
            infinite = __syncthreads_or(infinite);
            top = lane < kWalkWarps ? warp_most[lane] : -INFINITY;
#pragma unroll
            for (int off = 16; off >= 1; off >>= 1) top = fmaxf(top, __shfl_xor_sync(kFullMask, top, off));
        }
        scale.relative_to<CAP>(top, infinite);

        // ---- sums, and the draw from block to warp to step to token, with one body for all of it: what runs once costs what its instructions take to fetch ----
        enum { kAll, kLeft, kAgain };
        int stage = !o.summed ? kAll : o.refused && (o.drawn || o.what == 2) ? kLeft : kAgain;
        double z = o.z, target = 0.0, whole = scale.from, part, upto;          // whole: the logit that z is relative to; part, upto: lane w's sum of warp w, and up to it
        int refused = 0;
        // Sums of warps from those of lanes, in every warp.
        auto warps = [&](double mine) {
#pragma unroll
            for (int off = 16; off >= 1; off >>= 1) mine += __shfl_xor_sync(kFullMask, mine, off);
            __syncthreads();                           // the sums before these have been read
            if (lane == 0) warp_part[warp] = mine;
            __syncthreads();
            part = lane < kWalkWarps ? warp_part[lane] : 0.0;
            upto = warp_scan(part, lane);
        };
        bool chosen = false;                           // this block has the token
        uint32_t count = 0;                            // steps that it is among
        const bool direct = a.exact && o.what == 2 && o.refused == 0;
        if (direct) {
            // ---- from the sums of the first launch, by the first block ----
            if (rank != 0) break;
            const ChunkStat* s = a.stats + (size_t)(of.row0 + o.node) * a.parts;
            if (!(z > kNothing)) {
                if (tid == 0) {
                    out_tokens[o.at] = 0;
                    if (logprobs) logprobs[o.at] = -INFINITY;
                }
                break;
            }
            target = (double)o.u * z;
            const uint32_t last = part_of<CAP>(scale, s, a.parts, target);
            chosen = true;
            begin = last * a.per * kStatsThreads;
            count = a.per * (kStatsThreads / kWarp);
        }
        while (!direct) {
            if (stage == kLeft) {
                refused = o.refused;
                if (o.drawn && o.step) {
                    if (tid == 0) nodes.gone[refused - 1] = refused == 1 ? z : o.s;
                    __syncthreads();
                }
            } else if (stage == kAgain) {
                refused = 0;
            }
            const Refused by = {refused, refused && o.drawn, nodes.gone};
            warps(sum_steps<T, CAP>(a, row, probs, by, scale, begin + warp * steps * kWarp + lane, steps, parts + tid, per));
            // ---- over the cluster ----
            if (tid == kWarp - 1) {
                block_sum[turn & 1] = upto;
                block_most[turn & 1] = top;
            }
            __syncwarp();
            cluster.sync();
            double mine = lane < ranks ? *cluster.map_shared_rank(&block_sum[turn & 1], lane) : 0.0, share = 1.0;
            if (!(o.known & 1)) {
                const float its = lane < ranks ? *cluster.map_shared_rank(&block_most[turn & 1], lane) : -INFINITY;
                float most = its;
#pragma unroll
                for (int off = 16; off >= 1; off >>= 1) most = fmaxf(most, __shfl_xor_sync(kFullMask, most, off));
                const double logit = scale.unit(warp_logit64<CAP>(scale, its));
                whole = scale.unit(warp_logit64<CAP>(scale, most));
                Scale to = scale;
                to.from = whole;
                share = warp_weight(to, logit);            // 0 where there is no finite logit
                mine *= share;
            }
            ++turn;
            __syncwarp();
            const double run = warp_scan(mine, lane), s = __shfl_sync(kFullMask, run, ranks - 1);
            if (stage == kAll) z = s;
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
            if (!(s > kNothing)) {
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
            chosen = who == rank;
            target /= __shfl_sync(kFullMask, share, who);
            break;
        }
        if (chosen) {
            // ---- the draw: the warp whose sum the target falls in, its group of steps by the sums that were kept, the step, the lane, the token ----
            uint32_t group;
            if (!direct) {
                const uint32_t its = warp_fall(part, upto, target);
                warps(warp * per < steps ? parts[warp * kWalkThreads + its * kWarp + lane] : 0.0);
                group = warp_fall(part, upto, target);
                count = min(per, steps - group * per);
                begin += (its * steps + group * per) * kWarp;
            }
            const Refused by = {refused, refused && o.drawn, nodes.gone};
            for (;;) {
                const uint32_t sub = (count + kWalkWarps - 1) / kWalkWarps, first = min(warp * sub, count), last = min(first + sub, count);
                double all = 0.0, w[E];
                if (sub > 2) all = sum_steps<T, CAP>(a, row, probs, by, scale, begin + first * kWarp + lane, last - first, nullptr, 1);
                else for (uint32_t i = first; i < last; ++i) all += one_step<T, CAP>(a, row, probs, by, scale, begin + i * kWarp + lane, w);
                warps(all);
                group = warp_fall(part, upto, target);
                begin += group * sub * kWarp;
                count = min(sub, count - group * sub);
                if (sub > 1) continue;
                if (warp == group) {                   // a step of its own
                    const double lanes = warp_scan(all, lane);
                    if (warp_fall(all, lanes, target) == lane) {
                        double at = 0.0;
                        int found = -1, end = 0;
#pragma unroll
                        for (int e = 0; e < E; ++e) {
                            at += w[e];
                            if (w[e] > kNothing / 8) {             // of a lane that has more than kNothing one has
                                end = e;
                                if (found < 0 && at > target) found = e;
                            }
                        }
                        const int64_t token = row.inside(row.first(begin + lane) + (found < 0 ? end : found));
                        out_tokens[o.at] = (int32_t)token;
                        if (logprobs) logprobs[o.at] = (float)((logit64<CAP>(number(row.p[token]), a.softcap) - whole) * heat.k * kLn2 - log(z));
                    }
                }
                break;
            }
        }
        if (o.what == 2) break;
    }
    if (rank == 0) {
        __syncthreads();
        const uint32_t tokens = of.n ? walk.at + 1 : 0;
        for (uint32_t i = tid; i < a.draft_stride; i += kWalkThreads) {
            if (i == 0) out_rows[0] = of.n ? 0 : -1;
            if (logprobs && i < of.n && nodes.inner[i] < 0)
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
tf_status launch_verify(tf_context* ctx, cudaStream_t st, VerifyArgs a, uint64_t room) {
    const char* name = "tf_verify_drafts";
    constexpr uint32_t E = Row<T>::E;
    uint32_t ranks = kMostRanks;
    // All rows in 64 bits (us a call, beside the 32-bit sums): 6 rows of 262144 logits 19, beside 23, 16 rows 36, beside 38, 32 rows 38, beside 39, but 270 rows of 32000 37, beside 35;
    // capped 6 rows 37, beside 43, 16 rows 49, beside 53, 32 rows 61, beside 58.
    a.exact = a.draft_stride == 1 || (uint64_t)a.rows * a.vocab <= (CAP ? 4000000u : 6000000u);
    if (a.rows) {
        const bool even = aligned(a.logits, 16) && a.stride % E == 0;          // else a row may begin anywhere in a piece
        if (a.exact) {
            // Pieces of a thread: as many as leave every place on the chip a block, but no more than 64 parts of a row, which the walk goes through 32 at a time (128 where a logit
            // takes twice as long), and as the workspace needs.
            const uint64_t pieces = ((uint64_t)a.vocab + (even ? 0 : E - 1) + E - 1) / E;
            auto parts = [&](uint32_t per) { return (pieces + (uint64_t)kStatsThreads * per - 1) / ((uint64_t)kStatsThreads * per); };
            a.per = kMostPieces;
            while (a.per > 1 && parts(a.per / 2) == 1) a.per /= 2;             // short rows: 1000 of 300 67 us with eight pieces, 37 with one
            while (a.per > 1 && a.rows * parts(a.per) < (uint64_t)ctx->sm_count * 2 && parts(a.per / 2) <= (CAP ? 128 : 64) && a.rows * parts(a.per / 2) <= room) a.per /= 2;
            a.parts = (uint32_t)parts(a.per);
            verify_sums_kernel<T, CAP><<<(uint32_t)(a.rows * (uint64_t)a.parts), kStatsThreads, 0, st>>>(a);
        } else {
            a.chunks = (uint32_t)(((uint64_t)a.vocab + (even ? 0 : E - 1) + kChunk - 1) / kChunk);
            // Several chunks a block, as long as that leaves every place on the chip two blocks: a block's start and end take as long as a chunk or two (200 chains of four: 102 us
            // with one chunk, 76 with two, 66 with four, 64 with eight).
            const uint64_t all = (uint64_t)a.rows * a.chunks / ((uint64_t)ctx->sm_count * 8);
            a.per = (uint32_t)(all < 1 ? 1 : all > 8 ? 8 : all);
            a.parts = (a.chunks + a.per - 1) / a.per;
            verify_stats_kernel<T, CAP><<<a.rows * a.parts, kStatsThreads, 0, st>>>(a);
        }
        const tf_status s = check_launch(ctx, name);
        if (s != TF_OK) return s;
    }
    if (a.draft_stride == 1) {
        TF_CUDA(ctx, launch_pdl(verify_lone_kernel<T, CAP>, dim3(a.sequences), dim3(kStatsThreads), 0, st, a));
        return check_launch(ctx, name);
    }
    // Blocks of a sequence: 16, 8, 4 or 2 of them take 22, 33, 55, 96 us for a lone row that is not summed yet, 81, 80, 95, 123 for 33 trees of 12, 114, 114, 113, 156 for 64 chains of seven.
    // So as many as are on the chip at once, two an SM, with two steps a warp; beyond that they wait for one another's places.
    while (ranks > 1 && ((uint64_t)a.sequences * ranks > (uint64_t)ctx->sm_count * 2 || (uint64_t)a.vocab < (uint64_t)ranks * kWalkThreads * 2 * E)) ranks /= 2;
    const size_t smem = a.draft_stride * NodeTable::kBytes;
    static DeviceSmemCache smem_cache;
    const tf_status m = ensure_dynamic_smem(ctx, verify_walk_kernel<T, CAP>, smem_cache, smem);
    if (m != TF_OK) return m;
    static std::atomic<uint64_t> wide{0};          // devices whose kernel may run in clusters of sixteen
    const uint64_t bit = 1ull << (ctx->device & 63);
    if (ranks > 8 && !(wide.load(std::memory_order_relaxed) & bit)) {
        TF_CUDA(ctx, cudaFuncSetAttribute(verify_walk_kernel<T, CAP>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
        wide.fetch_or(bit, std::memory_order_relaxed);
    }
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
    ws->room = (uint64_t)max_rows * (((uint64_t)max_vocab + 7 + tf::kChunk - 1) / tf::kChunk);
    ws->stats = ws->room + (uint64_t)ctx->sm_count * 512;      // more where there are few rows, in smaller parts
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
    TF_REQUIRE(ctx, rows * chunks <= ws->room, TF_ERR_SCRATCH_TOO_SMALL, "%s: the workspace has room for %llu chunks of rows, not %llu", name,
               (unsigned long long)ws->room, (unsigned long long)(rows * chunks));
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
    a.logits = logits; a.stride = logits_stride; a.row_offsets = {row_offsets}; a.tokens = {drafts->tokens}; a.parents = {drafts->parents};
    a.uniforms = {uniforms}; a.temperatures = {temperatures};
    a.out_tokens = out_tokens; a.out_rows = out_rows; a.kept = kept; a.logprobs = logprobs;
    a.stats = static_cast<tf::ChunkStat*>(ws->memory);
    a.error = ctx->device_error;
    a.vocab = vocab; a.rows = rows; a.sequences = sequences; a.draft_stride = drafts->stride;
    a.softcap = softcap;
    const tf::DeviceScope scope(ctx->device);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const bool cap = softcap > 0.0f;
    switch (logits_dtype) {
        case TF_FP16: return cap ? tf::launch_verify<__half, true>(ctx, st, a, ws->stats) : tf::launch_verify<__half, false>(ctx, st, a, ws->stats);
        case TF_BF16: return cap ? tf::launch_verify<__nv_bfloat16, true>(ctx, st, a, ws->stats) : tf::launch_verify<__nv_bfloat16, false>(ctx, st, a, ws->stats);
        default: return cap ? tf::launch_verify<float, true>(ctx, st, a, ws->stats) : tf::launch_verify<float, false>(ctx, st, a, ws->stats);
    }
}

}  // extern "C"
