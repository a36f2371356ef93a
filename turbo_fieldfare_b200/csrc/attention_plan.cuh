// Which tiles of which rows a worker of the attention takes: lengths, units and shares. Host and device code alike, so that the CPU tests walk
// every worker of a call.
#pragma once

#include "kv_cache.cuh"

namespace tf {

// What a block of the kernel for many rows leaves for the unit that its share ends in: where the other shares are and which rows they hold.
struct ShareInfo {
    uint32_t active, last;
    uint32_t row0, flat0, valid, head;    // first row of the sequence; first (token, head) row of the unit and how many; kv head
};

struct AttnArgs {
    const uint16_t* q;
    uint16_t* out;
    KvPlanes k, v;
    KvTable table;
    const int32_t *row_offsets, *context_lengths, *positions;
    const unsigned long long* mask;
    float* partial;
    ShareInfo* info;
    uint32_t* tickets;        // [levels][ticket_stride], zero between calls
    uint32_t ticket_stride;
    uint32_t* error;
    uint32_t q_stride, out_stride, sequences, rows, kv_heads, group, mask_words, window;
    uint32_t head_parts;      // units per kv head whose values are parts of the head's
    float scale;
};

constexpr int kJoin = 16;             // shares that are joined at a time

template <typename T>
__host__ __device__ __forceinline__ T lesser(T a, T b) { return a < b ? a : b; }

// Tokens are 32-bit numbers: from here on none is looked at (a cache of more would be 2^37 bytes at the least).
constexpr uint32_t kMostTokens = 0x7FFFFF00u;

// The lengths of a sequence, cut to what the arrays and the table can hold.
struct Sequence {
    uint32_t row0, rows;      // its rows of the call
    uint32_t context;         // cached tokens before them
    __host__ __device__ __forceinline__ void load(const AttnArgs& a, uint32_t b, bool report) {
        const int32_t begin = a.row_offsets[b], end = a.row_offsets[b + 1], c = a.context_lengths[b];
        const int32_t most = (int32_t)a.rows, lo = begin < 0 ? 0 : begin > most ? most : begin, hi = end < lo ? lo : end > most ? most : end;
        row0 = (uint32_t)lo;
        rows = (uint32_t)(hi - lo);
        context = c < 0 ? 0u : (uint32_t)c;
        if (report) {
            if (lo != begin || hi != end) *a.error = kErrKvOffsets;
            if (rows && (c < 0 || (uint64_t)context + rows > (uint64_t)a.table.stride << a.table.page_log2)) *a.error = kErrKvPage;
        }
    }
};

// The tokens that the rows [flat0, flat0 + mt) of a sequence's kv head may see, in tiles.
struct UnitRange {
    uint32_t end;             // tokens from here on are seen by no row
    uint32_t tile0, tiles;    // at least one tile, so that rows which see nothing are still written
    __host__ __device__ __forceinline__ void set(const AttnArgs& a, const Sequence& s, uint32_t flat0, uint32_t mt, uint32_t tile) {
        uint32_t first = 0, drafted = s.rows;
        if ((uint64_t)s.rows * a.group > mt) {                 // (a lone unit needs no division)
            first = flat0 / a.group;
            if (!a.mask) drafted = lesser((flat0 + mt - 1) / a.group + 1, s.rows);
        }
        if (a.mask && (drafted >> 6) >= a.mask_words) drafted = a.mask_words * 64;
        end = s.context + drafted;                             // both below 2^31
        const uint32_t held = (a.table.stride - 1) >> (31 - a.table.page_log2) ? kMostTokens : lesser(a.table.stride << a.table.page_log2, kMostTokens);
        end = lesser(end, held);
        uint32_t low = 0;
        if (a.window) {
            const uint32_t from = s.context + (a.mask ? 0u : first) + 1;
            low = from > a.window ? lesser(from - a.window, end) : 0u;
        }
        tile0 = low / tile;
        const uint32_t stop = (end + tile - 1) / tile;
        tiles = stop > tile0 ? stop - tile0 : 1u;
    }
};

// A place in the row of all tiles: sequence, kv head, unit of rows, tile.
template <int MT, int TILE>
struct Cursor {
    Sequence seq;
    UnitRange range;
    uint32_t b, head, flat0, tile;       // tile counts from range.tile0
    __host__ __device__ __forceinline__ uint32_t token0() const { return (range.tile0 + tile) * TILE; }
    __host__ __device__ __forceinline__ uint32_t flat_rows(const AttnArgs& a) const { return seq.rows * a.group; }
    // to the first tile of the next unit
    __host__ __device__ __forceinline__ void next_unit(const AttnArgs& a) {
        tile = 0;
        if (flat0 + MT < flat_rows(a)) {
            flat0 += MT;
        } else if (flat0 = 0; ++head == a.kv_heads * a.head_parts) {
            head = 0;
            do { if (++b >= a.sequences) return; seq.load(a, b, false); } while (seq.rows == 0);
        }
        range.set(a, seq, flat0, MT, TILE);
    }
};

// Tiles of a sequence's rows for one kv head, over all its units.
template <int MT, int TILE>
__host__ __device__ __forceinline__ uint64_t sequence_tiles(const AttnArgs& a, const Sequence& s) {
    uint64_t n = 0;
    const uint32_t flat_rows = s.rows * a.group;               // below 2^31
    for (uint32_t f = 0; f < flat_rows; f += MT) {
        UnitRange r;
        r.set(a, s, f, MT, TILE);
        n += r.tiles;
    }
    return n;
}

// `total` tiles in shares that differ by one at the most: the first `more` workers have one more than `each`. No more workers than tiles.
struct Shares {
    uint64_t total;
    uint32_t workers, more;
    uint64_t each;
    __host__ __device__ __forceinline__ void set(uint64_t tiles, uint32_t most) {
        total = tiles;
        workers = (uint32_t)lesser((uint64_t)most, tiles);
        each = workers ? divide(tiles, workers) : 0;
        more = (uint32_t)(tiles - each * workers);
    }
    __host__ __device__ __forceinline__ uint64_t begin(uint32_t c) const { return each * c + lesser(c, more); }
    __host__ __device__ __forceinline__ uint32_t of(uint64_t tile) const {
        const uint64_t longer = (each + 1) * more;
        return (uint32_t)(tile < longer ? divide(tile, each + 1) : more + divide(tile - longer, each));
    }
    // A 32-bit division where the numbers are (a 64-bit one takes four times as long); the other is kept out of line.
    static __host__ __device__ __forceinline__ uint64_t divide(uint64_t a, uint64_t b) {
        return ((a | b) >> 32) == 0 ? (uint64_t)((uint32_t)a / (uint32_t)b) : divide_wide(a, b);
    }
    static __host__ __device__ __noinline__ uint64_t divide_wide(uint64_t a, uint64_t b) { return a / b; }
};

// The place `left` tiles into a sequence's tiles, of which there are more: kv head, first row of the unit, tile of the unit.
template <int MT, int TILE>
__host__ __device__ __forceinline__ void place_in_sequence(const AttnArgs& a, const Sequence& s, uint64_t left, uint32_t (&place)[3]) {
    const uint64_t n = sequence_tiles<MT, TILE>(a, s);
    place[0] = 0;
    if (left >= n) {
        place[0] = (uint32_t)Shares::divide(left, n);
        left -= n * place[0];
    }
    for (uint32_t f = 0;; f += MT) {
        UnitRange r;
        r.set(a, s, f, MT, TILE);
        if (left < r.tiles) {
            place[1] = f;
            place[2] = (uint32_t)left;
            return;
        }
        left -= r.tiles;
    }
}

}  // namespace tf
