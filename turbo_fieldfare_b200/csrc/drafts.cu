// What stands before and behind the layers of a step with drafted tokens: its rows and pages (tf_kv_plan) and the cache rows of the kept nodes
// (tf_kv_cache_keep).
//
// The plan is two sums over the sequences, pages given back and then (pages needed, rows asked for) of those that fit their table, and what
// follows from them for each sequence and row. Since both sums only rise, the sequences that are served are all before the first one that does
// not fit: a comparison for each, no loop over them. Latency is all that counts: one thread block does the sums.
#include "kv_cache.cuh"

namespace tf {

constexpr uint32_t kErrPlan = 0x7F000054u;         // the arrays of a plan contradict themselves
constexpr int kPlanThreads = 512, kPlanWarps = kPlanThreads / kWarp;
constexpr int kPlanRows = 128;                     // rows of a block of the second launch
constexpr uint32_t kPlanTokens = 0x7FFFFF00u;      // tokens of a sequence: as far as the attention looks

struct PlanArgs {
    int32_t *page_table, *held_pages, *first_pages, *free_pages, *free_count;
    int32_t* context_lengths;
    const int32_t *new_rows, *kept, *draft_tokens, *parents;
    int32_t *row_offsets, *positions, *row_sequences, *row_tokens;
    int64_t* slots;
    unsigned long long* tree_mask;
    uint32_t* error;
    uint32_t table_stride, num_pages, page_log2, sequences, window, draft_stride, mask_words, rows;
    uint32_t drafted;                              // 1: draft_stride limits the rows of a sequence
};

// Sums that stay at the top once they are there: numbers of pages and rows far beyond what fits compare as they should.
__device__ __forceinline__ uint32_t plan_add(uint32_t a, uint32_t b) {
    const uint32_t s = a + b;
    return s < a ? 0xFFFFFFFFu : s;
}

// A page that goes back, is taken or has a row on it: -1, and a report, where there is no such page.
__device__ __forceinline__ int32_t plan_page(const PlanArgs& a, int32_t page) {
    if ((uint32_t)page < a.num_pages) return page;
    *a.error = kErrPlan;
    return -1;
}

// Inclusive sums of two numbers over the block, and the block's totals.
struct PlanScan {
    uint32_t warp_sum[2][kPlanWarps];
};
__device__ __forceinline__ void plan_scan(PlanScan& s, uint32_t (&v)[2], uint32_t (&total)[2]) {
    const int warp = threadIdx.x / kWarp, lane = threadIdx.x % kWarp;
#pragma unroll
    for (int off = 1; off < kWarp; off <<= 1) {
        const uint32_t a = __shfl_up_sync(kFullMask, v[0], off), b = __shfl_up_sync(kFullMask, v[1], off);
        if (lane >= off) { v[0] = plan_add(v[0], a); v[1] = plan_add(v[1], b); }
    }
    __syncthreads();                               // what an earlier scan left there has been read
    if (lane == kWarp - 1) { s.warp_sum[0][warp] = v[0]; s.warp_sum[1][warp] = v[1]; }
    __syncthreads();
    uint32_t a = lane < kPlanWarps ? s.warp_sum[0][lane] : 0, b = lane < kPlanWarps ? s.warp_sum[1][lane] : 0;
#pragma unroll
    for (int off = 1; off < kPlanWarps; off <<= 1) {
        const uint32_t c = __shfl_up_sync(kFullMask, a, off), d = __shfl_up_sync(kFullMask, b, off);
        if (lane >= off) { a = plan_add(a, c); b = plan_add(b, d); }
    }
    total[0] = __shfl_sync(kFullMask, a, kPlanWarps - 1);
    total[1] = __shfl_sync(kFullMask, b, kPlanWarps - 1);
    const uint32_t before_a = __shfl_sync(kFullMask, a, warp ? warp - 1 : 0), before_b = __shfl_sync(kFullMask, b, warp ? warp - 1 : 0);
    if (warp) { v[0] = plan_add(v[0], before_a); v[1] = plan_add(v[1], before_b); }
}

// A sequence as the step finds it: its context, what it gives back ([lo, hi) of its table entries) and what it holds after that.
struct PlanSequence {
    uint32_t context, lo, hi, first, held, wanted;
    bool ends;
    __device__ __forceinline__ void load(const PlanArgs& a, uint32_t b) {
        const int32_t n = a.new_rows[b], h = a.held_pages[b], f = a.first_pages ? a.first_pages[b] : 0;
        held = h < 0 ? 0u : lesser_u32((uint32_t)h, a.table_stride);
        first = f < 0 ? 0u : lesser_u32((uint32_t)f, held);
        ends = n < 0;
        wanted = ends ? 0u : (uint32_t)n;
        lo = first;
        if (ends) {
            hi = held;
            context = first = held = 0;
            return;
        }
        const int32_t c = a.context_lengths[b], k = a.kept ? a.kept[b] : 0;
        context = lesser_u32((c < 0 ? 0u : (uint32_t)c) + (k < 0 ? 0u : (uint32_t)k), 0x7FFFFFFFu);
        hi = lo;
        if (a.window && context + 1 > a.window) {
            const uint32_t out = lesser_u32((context + 1 - a.window) >> a.page_log2, held);
            if (out > lo) hi = out;
        }
        first = hi;
    }
    static __device__ __forceinline__ uint32_t lesser_u32(uint32_t a, uint32_t b) { return a < b ? a : b; }
};

// One row of the step: sequence b, node i, whose tree is `parents`. Page entries and contexts are those that the sums left.
__device__ __forceinline__ void plan_row(const PlanArgs& a, uint32_t row, uint32_t b, uint32_t i, const int32_t* parents) {
    const uint32_t context = (uint32_t)a.context_lengths[b], token = context + i;
    uint32_t depth = i;
    if (a.drafted && (a.parents || a.tree_mask)) {
        // ancestors descend, so the words of the mask are done one by one from the node's own down
        unsigned long long* mask = a.tree_mask ? a.tree_mask + (size_t)row * a.mask_words : nullptr;
        if (mask) {
            if ((i >> 6) >= a.mask_words) *a.error = kErrPlan;
            for (uint32_t w = (i >> 6) + 1; w < a.mask_words; ++w) mask[w] = 0;
        }
        unsigned long long bits = 0;
        uint32_t at = i;
        depth = 0;
        for (;;) {
            bits |= 1ull << (at & 63);
            const int32_t up = parents ? parents[at] : (int32_t)at - 1;
            if (up >= (int32_t)at) *a.error = kErrPlan;
            const bool top = up < 0 || up >= (int32_t)at;
            if (mask && (top || (uint32_t)up >> 6 != at >> 6)) {
                uint32_t w = at >> 6;
                if (w < a.mask_words) mask[w] = bits;
                for (const uint32_t stop = top ? 0u : ((uint32_t)up >> 6) + 1; w > stop;)
                    if (--w < a.mask_words) mask[w] = 0;
                bits = 0;
            }
            if (top) break;
            at = (uint32_t)up;
            ++depth;
        }
    }
    a.positions[row] = (int32_t)(context + depth);
    if (a.row_sequences) a.row_sequences[row] = (int32_t)b;
    if (a.row_tokens) a.row_tokens[row] = a.draft_tokens[(size_t)b * a.draft_stride + i];
    if (a.slots) {
        const int32_t page = plan_page(a, a.page_table[(size_t)b * a.table_stride + (token >> a.page_log2)]);
        a.slots[row] = page < 0 ? -1ll : ((int64_t)page << a.page_log2) + (token & ((1u << a.page_log2) - 1u));
    }
}

// The sequence of a row: offsets[b] <= row < offsets[b + 1].
__device__ __forceinline__ uint32_t plan_sequence(const PlanArgs& a, const int32_t* offsets, uint32_t row) {
    uint32_t lo = 0, hi = a.sequences;
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) / 2;
        if ((uint32_t)offsets[mid] <= row) lo = mid;
        else hi = mid;
    }
    return lo;
}

// Kept in shared memory for the rows, since both are chased: the offsets of so many sequences, and so many nodes' parents.
constexpr uint32_t kPlanHeld = 2047, kPlanTree = 4096;

template <bool ROWS>
__global__ void __launch_bounds__(kPlanThreads) plan_kernel(const __grid_constant__ PlanArgs a) {
    __shared__ PlanScan scan;
    __shared__ uint32_t row_limit, page_limit;
    __shared__ int32_t held_offsets[ROWS ? kPlanHeld + 1 : 1], held_tree[ROWS ? kPlanTree : 1];
    const uint32_t tid = threadIdx.x, lane = tid % kWarp;
    const uint64_t nodes = (uint64_t)a.sequences * a.draft_stride;
    if (ROWS && a.parents && nodes <= kPlanTree)
        for (uint32_t i = tid; i < nodes; i += kPlanThreads) held_tree[i] = a.parents[i];
    if constexpr (!ROWS) pdl_launch_dependents();  // the rows' launch
    if (tid == 0) row_limit = page_limit = 0xFFFFFFFFu;
    const int32_t stack = *a.free_count;
    uint32_t count = stack < 0 ? 0u : PlanSequence::lesser_u32((uint32_t)stack, a.num_pages);
    bool bad = stack < 0 || (uint32_t)stack > a.num_pages;

    // ---- pages that go back ----
    uint32_t back = 0;
    for (uint32_t b0 = 0; b0 < a.sequences; b0 += kPlanThreads) {
        PlanSequence s;
        uint32_t v[2] = {0, 0}, total[2];
        if (b0 + tid < a.sequences) {
            s.load(a, b0 + tid);
            v[0] = s.hi - s.lo;
        }
        plan_scan(scan, v, total);
        back = plan_add(back, total[0]);
    }
    if (back > a.num_pages - count) { bad = true; back = a.num_pages - count; }
    for (uint32_t b0 = 0, before = 0; b0 < a.sequences; b0 += kPlanThreads) {
        const uint32_t b = b0 + tid;
        PlanSequence s;
        uint32_t v[2] = {0, 0}, total[2] = {0, 0}, mine = 0;
        if (b < a.sequences) {
            s.load(a, b);
            v[0] = mine = s.hi - s.lo;
            a.context_lengths[b] = (int32_t)s.context;
            a.held_pages[b] = (int32_t)s.held;
            if (a.first_pages) a.first_pages[b] = (int32_t)s.first;
        }
        if (back) {
            plan_scan(scan, v, total);
            uint32_t todo = __ballot_sync(kFullMask, mine != 0);
            while (todo) {                         // a warp moves the pages of one sequence after the other
                const int who = __ffs(todo) - 1;
                todo &= todo - 1;
                const uint32_t from = plan_add(before, __shfl_sync(kFullMask, v[0] - mine, who)), n = __shfl_sync(kFullMask, mine, who);
                int32_t* entries = a.page_table + (size_t)(b0 + tid - lane + who) * a.table_stride + __shfl_sync(kFullMask, s.lo, who);
                for (uint32_t e = lane; e < n; e += kWarp) {
                    const uint32_t j = plan_add(from, e);
                    if (j < back) a.free_pages[count + back - 1 - j] = plan_page(a, entries[e]);
                    entries[e] = -1;
                }
            }
            before = plan_add(before, total[0]);
        }
    }
    count += back;
    __syncthreads();                               // the stack and the sequences are written

    // ---- rows and pages of the step ----
    uint32_t pages_before = 0, rows_before = 0;
    for (uint32_t b0 = 0; b0 < a.sequences; b0 += kPlanThreads) {
        const uint32_t b = b0 + tid;
        uint32_t v[2] = {0, 0}, total[2], need = 0, wanted = 0, held = 0;
        if (b < a.sequences) {
            const int32_t n = a.new_rows[b];
            const uint64_t end = (uint64_t)(uint32_t)a.context_lengths[b] + (n < 0 ? 0u : (uint32_t)n);
            held = (uint32_t)a.held_pages[b];
            if (n > 0 && end <= kPlanTokens && (end + (1u << a.page_log2) - 1) >> a.page_log2 <= a.table_stride && !(a.drafted && (uint32_t)n > a.draft_stride)) {
                wanted = (uint32_t)n;
                const uint32_t upto = (uint32_t)((end + (1u << a.page_log2) - 1) >> a.page_log2);
                need = upto > held ? upto - held : 0u;
            }
        }
        v[0] = need; v[1] = wanted;
        plan_scan(scan, v, total);
        const uint32_t pages_upto = plan_add(pages_before, v[0]), rows_upto = plan_add(rows_before, v[1]);
        const bool fits = pages_upto <= count && rows_upto <= a.rows;
        const uint32_t pages_from = plan_add(pages_before, v[0] - need), rows_from = plan_add(rows_before, v[1] - wanted);
        if (!fits && pages_from <= count && rows_from <= a.rows && wanted) { page_limit = pages_from; row_limit = rows_from; }   // the first that does not
        __syncthreads();
        if (b < a.sequences) {
            const int32_t offset = (int32_t)PlanSequence::lesser_u32(rows_from, row_limit);
            a.row_offsets[b] = offset;
            if constexpr (ROWS) { if (b <= kPlanHeld) held_offsets[b] = offset; }
            if (fits && need) a.held_pages[b] = (int32_t)(held + need);
        }
        uint32_t todo = __ballot_sync(kFullMask, fits && need);
        while (todo) {
            const int who = __ffs(todo) - 1;
            todo &= todo - 1;
            const uint32_t from = __shfl_sync(kFullMask, pages_from, who), n = __shfl_sync(kFullMask, need, who);
            int32_t* entries = a.page_table + (size_t)(b0 + tid - lane + who) * a.table_stride + __shfl_sync(kFullMask, held, who);
            for (uint32_t e = lane; e < n; e += kWarp) entries[e] = plan_page(a, a.free_pages[count - 1 - (from + e)]);
        }
        pages_before = plan_add(pages_before, total[0]);
        rows_before = plan_add(rows_before, total[1]);
    }
    if (tid == 0) {
        const int32_t all = (int32_t)PlanSequence::lesser_u32(rows_before, row_limit);
        a.row_offsets[a.sequences] = all;
        if constexpr (ROWS) { if (a.sequences <= kPlanHeld) held_offsets[a.sequences] = all; }
        *a.free_count = (int32_t)(count - PlanSequence::lesser_u32(pages_before, page_limit));
        if (bad) *a.error = kErrPlan;
    }
    if constexpr (ROWS) {
        __syncthreads();
        const int32_t *offsets = a.sequences <= kPlanHeld ? held_offsets : a.row_offsets, *trees = a.parents && nodes <= kPlanTree ? held_tree : a.parents;
        const uint32_t all = (uint32_t)offsets[a.sequences];
        for (uint32_t row = tid; row < all; row += kPlanThreads) {
            const uint32_t b = plan_sequence(a, offsets, row);
            plan_row(a, row, b, row - (uint32_t)offsets[b], trees ? trees + (size_t)b * a.draft_stride : nullptr);
        }
    }
}

__global__ void __launch_bounds__(kPlanRows) plan_rows_kernel(const __grid_constant__ PlanArgs a) {
    __shared__ int32_t held_offsets[kPlanHeld + 1], held_tree[kPlanTree];
    const uint32_t tid = threadIdx.x;
    pdl_wait();
    const int32_t* offsets = a.row_offsets;
    if (a.sequences <= kPlanHeld) {
        for (uint32_t i = tid; i <= a.sequences; i += kPlanRows) held_offsets[i] = a.row_offsets[i];
        offsets = held_offsets;
    }
    __syncthreads();
    const uint32_t all = (uint32_t)offsets[a.sequences];
    for (uint32_t row0 = blockIdx.x * kPlanRows; row0 < all; row0 += gridDim.x * kPlanRows) {
        const int32_t* trees = a.parents;
        uint32_t first = 0;
        if (a.parents) {                           // the trees of this block's rows
            first = plan_sequence(a, offsets, row0);
            const uint32_t last = plan_sequence(a, offsets, min(row0 + kPlanRows, all) - 1);
            const uint64_t nodes = (uint64_t)(last - first + 1) * a.draft_stride;
            if (nodes <= kPlanTree) {
                __syncthreads();                   // those of the rows before have been followed
                for (uint32_t i = tid; i < nodes; i += kPlanRows) held_tree[i] = a.parents[(size_t)first * a.draft_stride + i];
                trees = held_tree;
                __syncthreads();
            } else {
                first = 0;
            }
        }
        if (row0 + tid < all) {
            const uint32_t b = plan_sequence(a, offsets, row0 + tid);
            plan_row(a, row0 + tid, b, row0 + tid - (uint32_t)offsets[b], trees ? trees + (size_t)(b - first) * a.draft_stride : nullptr);
        }
    }
}

// ---------------------------------------------------------------------------
// cache rows of the kept nodes
// ---------------------------------------------------------------------------
//
// Token c + node(i) goes to token c + i. Nodes ascend, so node(i) >= i and no token is written that a later move reads; a token that an earlier move reads is written
// after it, since every byte of a (sequence, head) is moved by the same lane of one warp, and a lane loads a batch of moves before it stores it. So the moves are
// done in place without a barrier. Bytes are few (a node is kv_heads * (2 head_dim bits / 8 + ...) of them): one launch for all layers is what counts.

constexpr uint32_t kKeepCaches = 32;               // layers of one launch: their descriptors are its parameters
constexpr int kKeepWarps = 4, kKeepBatch = 4;

struct KeepCache {
    KvPlanes planes[2];
    uint32_t num_pages, kv_heads, row_bytes, groups;
};
struct KeepArgs {
    KeepCache cache[kKeepCaches];
    const int32_t *page_table, *row_offsets, *context_lengths, *kept_rows, *kept;
    uint32_t* error;
    uint32_t table_stride, page_log2, sequences, rows, kept_stride;
};

__global__ void __launch_bounds__(kKeepWarps * kWarp) kv_cache_keep_kernel(const __grid_constant__ KeepArgs a) {
    const KeepCache& c = a.cache[blockIdx.y];
    const uint32_t lane = threadIdx.x % kWarp;
    const uint64_t unit = (uint64_t)blockIdx.x * kKeepWarps + threadIdx.x / kWarp;
    if (unit >= (uint64_t)a.sequences * c.kv_heads) return;
    const uint32_t b = (uint32_t)(unit / c.kv_heads), head = (uint32_t)(unit % c.kv_heads);
    const int32_t k = a.kept[b], begin = a.row_offsets[b], end = a.row_offsets[b + 1], context = a.context_lengths[b];
    const int32_t most = (int32_t)a.rows, lo = begin < 0 ? 0 : begin > most ? most : begin, hi = end < lo ? lo : end > most ? most : end;
    const uint32_t nodes = (uint32_t)(hi - lo);
    if (k <= 0) return;
    const uint32_t moves = (uint32_t)k < a.kept_stride ? (uint32_t)k : a.kept_stride;
    const KvTable table = {a.page_table, a.table_stride, c.num_pages, a.page_log2};
    auto place = [&](int64_t token) -> int64_t {   // row of the planes, or -1
        const int32_t page = context < 0 ? -1 : table.page(b, token);
        if (page < 0) return -1;
        return (((int64_t)page * c.kv_heads + head) << a.page_log2) + (token & ((1 << a.page_log2) - 1));
    };
    int32_t before = -1;
    for (uint32_t i0 = 0; i0 < moves; i0 += kWarp) {
        // ---- where the next 32 moves go ----
        const uint32_t i = i0 + lane;
        const int32_t node = i < moves ? a.kept_rows[(size_t)b * a.kept_stride + i] : 0x7FFFFFFF;
        int32_t last = __shfl_up_sync(kFullMask, node, 1);
        if (lane == 0) last = before;
        const bool wrong = i < moves && (node <= last || (uint32_t)node >= nodes);
        const uint32_t wrongs = __ballot_sync(kFullMask, wrong);
        const uint32_t good = wrongs ? (1u << (__ffs(wrongs) - 1)) - 1u : kFullMask;
        before = __shfl_sync(kFullMask, node, kWarp - 1);
        int64_t src = -1, dst = -1;
        const bool moved = i < moves && (good >> lane & 1u) && node != (int32_t)i;
        if (moved) {
            src = place((int64_t)context + node);
            dst = place((int64_t)context + i);
        }
        uint32_t todo = __ballot_sync(kFullMask, moved && src >= 0 && dst >= 0);
        if (head == 0) {
            if (wrongs && lane == 0) *a.error = kErrKvOffsets;
            if (moved && (src < 0 || dst < 0)) *a.error = kErrKvPage;
        }
        // ---- a batch at a time: loads, then stores; a lane has the same bytes of every token ----
        while (todo) {
            int64_t from[kKeepBatch], to[kKeepBatch];
            int n = 0;
#pragma unroll
            for (int m = 0; m < kKeepBatch; ++m) {
                const int who = todo ? __ffs(todo) - 1 : 0;
                from[m] = __shfl_sync(kFullMask, src, who);
                to[m] = __shfl_sync(kFullMask, dst, who);
                if (todo) { n = m + 1; todo &= todo - 1; }
            }
            const uint32_t pieces = c.row_bytes / 16;
            for (uint32_t p = lane; p < 2 * pieces; p += kWarp) {
                uint8_t* plane = c.planes[p >= pieces].codes + (p >= pieces ? p - pieces : p) * 16;
                uint4 w[kKeepBatch];
#pragma unroll
                for (int m = 0; m < kKeepBatch; ++m)
                    if (m < n) w[m] = *reinterpret_cast<const uint4*>(plane + from[m] * c.row_bytes);
#pragma unroll
                for (int m = 0; m < kKeepBatch; ++m)
                    if (m < n) *reinterpret_cast<uint4*>(plane + to[m] * c.row_bytes) = w[m];
            }
            if (lane < 4 * c.groups) {             // scales and biases: at most eight groups of four planes
                const uint32_t which = lane / c.groups, g = lane % c.groups;
                const KvPlanes& of = c.planes[which >> 1];
                uint16_t* plane = (which & 1 ? of.biases : of.scales) + g;
                uint16_t w[kKeepBatch];
#pragma unroll
                for (int m = 0; m < kKeepBatch; ++m)
                    if (m < n) w[m] = plane[from[m] * c.groups];
#pragma unroll
                for (int m = 0; m < kKeepBatch; ++m)
                    if (m < n) plane[to[m] * c.groups] = w[m];
            }
        }
        if (wrongs) return;
    }
}

}  // namespace tf

extern "C" {

tf_status tf_kv_plan(tf_context* ctx, void* stream, const tf_kv_pages* pages, int32_t* context_lengths, const int32_t* new_rows, const int32_t* kept,
                     uint32_t window, const tf_drafts* drafts, const tf_kv_rows* rows) {
    const char* name = "tf_kv_plan";
    TF_REQUIRE(ctx, ctx != nullptr, TF_ERR_INVALID_ARGUMENT, "%s: ctx is NULL", name);
    TF_REQUIRE(ctx, pages != nullptr && rows != nullptr, TF_ERR_INVALID_ARGUMENT, "%s: pages or rows is NULL", name);
    TF_REQUIRE(ctx, rows->row_offsets != nullptr, TF_ERR_INVALID_ARGUMENT, "%s: row_offsets is NULL", name);
    TF_REQUIRE(ctx, tf::aligned(rows->row_offsets, 4), TF_ERR_ALIGNMENT, "%s: row_offsets must be 4-byte aligned", name);
    TF_REQUIRE(ctx, pages->sequences < 0x7FFFFFFFu && rows->rows <= 0x7FFFFFFFu, TF_ERR_INVALID_ARGUMENT, "%s: rows and sequences must be below 2^31", name);
    if (pages->sequences) {
        TF_REQUIRE(ctx, pages->page_table && pages->held_pages && pages->free_pages && pages->free_count && context_lengths && new_rows, TF_ERR_INVALID_ARGUMENT,
                   "%s: NULL array", name);
        TF_REQUIRE(ctx, rows->positions || rows->rows == 0, TF_ERR_INVALID_ARGUMENT, "%s: positions is NULL", name);
        TF_REQUIRE(ctx, pages->page_size >= 16 && pages->page_size <= 65536 && (pages->page_size & (pages->page_size - 1)) == 0, TF_ERR_UNSUPPORTED,
                   "%s: page_size %u is not a power of two from 16 to 65536", name, pages->page_size);
        TF_REQUIRE(ctx, pages->page_table_stride > 0, TF_ERR_INVALID_ARGUMENT, "%s: page_table_stride is 0", name);
        TF_REQUIRE(ctx, pages->num_pages > 0 && pages->num_pages <= 0x7FFFFFFFu && pages->page_table_stride <= 0x7FFFFFFFu, TF_ERR_INVALID_ARGUMENT,
                   "%s: num_pages must be from 1 to 2^31 - 1, page_table_stride below 2^31", name);
        TF_REQUIRE(ctx, window == 0 || pages->first_pages, TF_ERR_INVALID_ARGUMENT, "%s: a window needs first_pages", name);
        TF_REQUIRE(ctx, window <= 0x7FFFFFFFu, TF_ERR_INVALID_ARGUMENT, "%s: window must be below 2^31", name);
        TF_REQUIRE(ctx, drafts == nullptr || drafts->stride > 0, TF_ERR_INVALID_ARGUMENT, "%s: the drafts' stride is 0", name);
        TF_REQUIRE(ctx, rows->tokens == nullptr || (drafts && drafts->tokens), TF_ERR_INVALID_ARGUMENT, "%s: tokens of rows need drafts with tokens", name);
        TF_REQUIRE(ctx, rows->tree_mask == nullptr || (drafts && rows->mask_words > 0), TF_ERR_INVALID_ARGUMENT, "%s: a tree mask needs drafts and mask_words", name);
        TF_REQUIRE(ctx, tf::aligned(pages->page_table, 4) && tf::aligned(pages->held_pages, 4) && tf::aligned(pages->first_pages, 4) && tf::aligned(pages->free_pages, 4) &&
                            tf::aligned(pages->free_count, 4) && tf::aligned(context_lengths, 4) && tf::aligned(new_rows, 4) && tf::aligned(kept, 4) &&
                            tf::aligned(rows->positions, 4) && tf::aligned(rows->sequences, 4) && tf::aligned(rows->tokens, 4) &&
                            tf::aligned(rows->slots, 8) && tf::aligned(rows->tree_mask, 8) &&
                            (!drafts || (tf::aligned(drafts->tokens, 4) && tf::aligned(drafts->parents, 4))),
                   TF_ERR_ALIGNMENT, "%s: arrays must be aligned to their elements", name);
    }
    const tf::DeviceScope scope(ctx->device);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (pages->sequences == 0) {                   // no rows: the one offset says so
        TF_CUDA(ctx, cudaMemsetAsync(rows->row_offsets, 0, sizeof(int32_t), st));
        return TF_OK;
    }
    tf::PlanArgs a = {};
    a.page_table = pages->page_table; a.held_pages = pages->held_pages; a.first_pages = pages->first_pages; a.free_pages = pages->free_pages;
    a.free_count = pages->free_count;
    a.context_lengths = context_lengths; a.new_rows = new_rows; a.kept = kept;
    if (drafts) { a.drafted = 1; a.draft_tokens = drafts->tokens; a.parents = drafts->parents; a.draft_stride = drafts->stride; }
    a.row_offsets = rows->row_offsets; a.positions = rows->positions; a.row_sequences = rows->sequences; a.row_tokens = rows->tokens; a.slots = rows->slots;
    a.tree_mask = reinterpret_cast<unsigned long long*>(rows->tree_mask); a.mask_words = rows->mask_words;
    a.error = ctx->device_error;
    a.table_stride = pages->page_table_stride; a.num_pages = pages->num_pages; a.page_log2 = tf::log2_of(pages->page_size);
    a.sequences = pages->sequences; a.window = window; a.rows = rows->rows;
    // Few rows: by the block of the sums, one launch (us a call, one launch / two; trees of so many nodes each: 4 x 64 4.5 / 6.4, 64 x 16 6.3 / 6.7, 64 x 32 10.1 / 6.9,
    // 64 x 128 31 / 6.9; chains 4 x 64 3.7 / 5.2, 1 x 1024 3.8 / 5.1, 64 x 32 5.1 / 5.1, 64 x 128 10.6 / 5.1).
    if (rows->rows <= 1024) {
        tf::plan_kernel<true><<<1, tf::kPlanThreads, 0, st>>>(a);
        return tf::check_launch(ctx, name);
    }
    tf::plan_kernel<false><<<1, tf::kPlanThreads, 0, st>>>(a);
    tf_status s = tf::check_launch(ctx, name);
    if (s != TF_OK) return s;
    const uint32_t blocks = (uint32_t)(((uint64_t)rows->rows + tf::kPlanRows - 1) / tf::kPlanRows), most = (uint32_t)ctx->sm_count * 8;
    TF_CUDA(ctx, tf::launch_pdl(tf::plan_rows_kernel, dim3(blocks < most ? blocks : most), dim3(tf::kPlanRows), 0, st, a));
    return tf::check_launch(ctx, name);
}

tf_status tf_kv_cache_keep(tf_context* ctx, void* stream, const tf_kv_cache* caches, uint32_t cache_count, const tf_kv_batch* batch,
                           const int32_t* kept_rows, uint32_t kept_stride, const int32_t* kept) {
    const char* name = "tf_kv_cache_keep";
    TF_REQUIRE(ctx, ctx != nullptr, TF_ERR_INVALID_ARGUMENT, "%s: ctx is NULL", name);
    TF_REQUIRE(ctx, caches != nullptr || cache_count == 0, TF_ERR_INVALID_ARGUMENT, "%s: caches is NULL", name);
    tf_status s = tf::check_kv_batch(ctx, name, batch);
    for (uint32_t i = 0; i < cache_count && s == TF_OK; ++i) {
        s = tf::check_kv_cache(ctx, name, caches + i);
        if (s != TF_OK) break;
        TF_REQUIRE(ctx, caches[i].page_size == caches[0].page_size, TF_ERR_DIMENSION_MISMATCH, "%s: cache %u has pages of %u tokens, the first of %u", name, i,
                   caches[i].page_size, caches[0].page_size);
        for (uint32_t j = 0; j < i; ++j)           // two warps would move the same bytes
            TF_REQUIRE(ctx, caches[j].k_codes != caches[i].k_codes && caches[j].v_codes != caches[i].v_codes, TF_ERR_INVALID_ARGUMENT, "%s: caches %u and %u are the same", name, j, i);
        TF_REQUIRE(ctx, ((uint64_t)batch->sequences * caches[i].kv_heads + tf::kKeepWarps - 1) / tf::kKeepWarps <= 0x7FFFFFFFu, TF_ERR_UNSUPPORTED,
                   "%s: too many sequences for the number of heads", name);
    }
    if (s != TF_OK) return s;
    if (cache_count == 0 || batch->rows == 0 || batch->sequences == 0 || kept_stride == 0) return TF_OK;
    TF_REQUIRE(ctx, kept_rows && kept, TF_ERR_INVALID_ARGUMENT, "%s: NULL array", name);
    TF_REQUIRE(ctx, tf::aligned(kept_rows, 4) && tf::aligned(kept, 4), TF_ERR_ALIGNMENT, "%s: arrays must be aligned to their elements", name);
    const tf::DeviceScope scope(ctx->device);
    for (uint32_t i0 = 0; i0 < cache_count; i0 += tf::kKeepCaches) {
        const uint32_t n = cache_count - i0 < tf::kKeepCaches ? cache_count - i0 : tf::kKeepCaches;
        tf::KeepArgs a = {};
        uint32_t heads = 0;
        for (uint32_t i = 0; i < n; ++i) {
            const tf_kv_cache& c = caches[i0 + i];
            a.cache[i].planes[0] = {static_cast<uint8_t*>(c.k_codes), static_cast<uint16_t*>(c.k_scales), static_cast<uint16_t*>(c.k_biases)};
            a.cache[i].planes[1] = {static_cast<uint8_t*>(c.v_codes), static_cast<uint16_t*>(c.v_scales), static_cast<uint16_t*>(c.v_biases)};
            a.cache[i].num_pages = c.num_pages; a.cache[i].kv_heads = c.kv_heads; a.cache[i].row_bytes = c.head_dim * c.bits / 8; a.cache[i].groups = c.head_dim / 64;
            if (c.kv_heads > heads) heads = c.kv_heads;
        }
        a.page_table = batch->page_table; a.row_offsets = batch->row_offsets; a.context_lengths = batch->context_lengths;
        a.kept_rows = kept_rows; a.kept = kept; a.error = ctx->device_error;
        a.table_stride = batch->page_table_stride; a.page_log2 = tf::log2_of(caches[0].page_size);
        a.sequences = batch->sequences; a.rows = batch->rows; a.kept_stride = kept_stride;
        const uint64_t units = (uint64_t)batch->sequences * heads;
        tf::kv_cache_keep_kernel<<<dim3((uint32_t)((units + tf::kKeepWarps - 1) / tf::kKeepWarps), n), tf::kKeepWarps * tf::kWarp, 0, static_cast<cudaStream_t>(stream)>>>(a);
        s = tf::check_launch(ctx, name);
        if (s != TF_OK) return s;
    }
    return TF_OK;
}

}  // extern "C"
