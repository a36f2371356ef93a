"""Attention operators without a GPU: the shares of every block, the addresses in shared memory, pages that are not there, refusals."""
import shutil
import subprocess
from pathlib import Path

import pytest
import torch

ROOT = Path(__file__).resolve().parent.parent
SRC = r'''
#include <cstdio>
#include <cstdlib>
#include <map>
#include <random>
#include <set>
#include <tuple>
#include <vector>
#include "attention_tiles.cuh"
using namespace tf;
#define CHECK(c) do { if (!(c)) { std::printf("line %d: %s\n", __LINE__, #c); std::exit(1); } } while (0)

static std::mt19937_64 rng(7);
static int64_t pick(int64_t lo, int64_t hi) { return lo + (int64_t)(rng() % (uint64_t)(hi - lo + 1)); }

// Every block of a call walks its share as the kernel does: units are covered tile by tile exactly once, and the blocks that share a unit are those
// that the join will read. Tokens are looked up in the table on the way; what comes back is inside of the planes.
template <int MT, int TILE>
static void walk(const AttnArgs& a, uint32_t grid) {
    uint64_t total = 0;
    std::vector<uint64_t> before(a.sequences + 1, 0);
    for (uint32_t b = 0; b < a.sequences; ++b) {
        Sequence s;
        s.load(a, b, true);
        CHECK(s.row0 + (uint64_t)s.rows <= a.rows && s.context >= 0);
        total += sequence_tiles<MT, TILE>(a, s) * a.kv_heads * a.head_parts;
        before[b + 1] = total;
    }
    Shares shares;
    shares.set(total, grid);
    const uint32_t blocks = shares.workers;
    CHECK(shares.begin(0) == 0 && shares.begin(blocks) == total);
    using Unit = std::tuple<uint32_t, uint32_t, uint32_t>;
    std::map<Unit, std::vector<std::pair<uint32_t, uint32_t>>> seen;       // unit -> (block, tiles) in order
    std::map<Unit, uint32_t> tiles;
    std::map<Unit, uint32_t> first_block, said;
    for (uint32_t c = 0; c < blocks; ++c) {
        uint64_t item = shares.begin(c);
        const uint64_t stop = shares.begin(c + 1);
        CHECK(item < stop && shares.of(item) == c && shares.of(stop - 1) == c);
        uint32_t b = 0;
        while (before[b + 1] <= item) ++b;
        uint32_t place[3];
        Cursor<MT, TILE> now;
        now.b = b;
        now.seq.load(a, b, false);
        place_in_sequence<MT, TILE>(a, now.seq, item - before[b], place);
        now.head = place[0]; now.flat0 = place[1]; now.tile = place[2];
        now.range.set(a, now.seq, now.flat0, MT, TILE);
        std::set<int> slots;
        while (item < stop) {
            const Unit u{now.b, now.head, now.flat0};
            const bool from_start = now.tile == 0;
            const uint32_t segment = (uint32_t)lesser((uint64_t)(now.range.tiles - now.tile), stop - item);
            const bool to_end = now.tile + segment == now.range.tiles;
            CHECK(now.flat0 < now.flat_rows(a) && segment > 0);
            CHECK((int64_t)now.range.end <= (int64_t)a.table.stride << a.table.page_log2);
            for (uint32_t k = 0; k < segment; ++k) {
                const int64_t token0 = (int64_t)(now.range.tile0 + now.tile + k) * TILE;
                for (int i = 0; i < TILE / 16; ++i)
                    if (token0 + 16 * i < (int64_t)now.range.end) CHECK(a.table.page(now.b, token0 + 16 * i) < (int32_t)a.table.pages);
            }
            seen[u].push_back({c, segment});
            tiles[u] = now.range.tiles;
            if (!(from_start && to_end)) CHECK(slots.insert(from_start ? 1 : 0).second);     // a partial slot is written once
            item += segment;
            if (from_start) {
                first_block[u] = c;
                said[u] = shares.of(item - segment + now.range.tiles - 1);
            }
            now.tile += segment - 1;
            if (item < stop) { CHECK(to_end); now.next_unit(a); CHECK(now.b < a.sequences); }
        }
    }
    uint64_t units = 0;
    for (uint32_t b = 0; b < a.sequences; ++b) {
        Sequence s;
        s.load(a, b, false);
        units += ((uint64_t)s.rows * a.group + MT - 1) / MT * a.kv_heads * a.head_parts;
    }
    CHECK(seen.size() == units);
    for (auto& [u, parts] : seen) {
        uint64_t n = 0;
        uint32_t expect = first_block.at(u);
        for (auto& [block, count] : parts) { CHECK(block == expect++); n += count; }
        CHECK(n == tiles[u] && said.at(u) == parts.back().first);
    }
}

static void divisions() {
    for (int i = 0; i < 100000; ++i) {
        const uint64_t a = rng() >> pick(0, 63), b = (rng() >> pick(0, 63)) | 1;
        CHECK(Shares::divide(a, b) == a / b);
    }
}

static void all_shares() {
    for (int round = 0; round < 400; ++round) {
        const uint32_t n = (uint32_t)pick(1, 40);
        const bool bad = round % 4 == 3;
        std::vector<int32_t> offsets(n + 1), contexts(n), table;
        offsets[0] = bad ? (int32_t)pick(-5, 5) : 0;
        for (uint32_t b = 0; b < n; ++b) {
            offsets[b + 1] = offsets[b] + (int32_t)(pick(0, 3) ? pick(0, round % 3 ? 5 : 90) : 0) - (bad ? (int32_t)pick(0, 9) : 0);
            contexts[b] = (int32_t)(pick(0, 2) ? pick(0, 4000) : pick(0, 70));
            if (bad && pick(0, 5) == 0) contexts[b] = pick(0, 1) ? 0x7FFFFFFF : -(int32_t)pick(1, 1 << 30);
        }
        uint32_t error = 0;
        AttnArgs a = {};
        a.error = &error;
        a.rows = (uint32_t)(bad ? pick(1, 60) : offsets[n] > 0 ? offsets[n] : 1);
        a.table.page_log2 = (uint32_t)pick(4, 8);
        a.table.pages = (uint32_t)pick(1, 500);
        a.table.stride = (uint32_t)((4200 >> a.table.page_log2) + (bad ? -(int)pick(0, 10) : 5));
        table.resize((size_t)n * a.table.stride);
        for (auto& p : table) p = bad && pick(0, 3) == 0 ? (int32_t)rng() : (int32_t)pick(0, a.table.pages - 1);
        a.table.table = table.data();
        a.row_offsets = offsets.data(); a.context_lengths = contexts.data();
        a.head_parts = (uint32_t)pick(1, 2);
        a.sequences = n; a.kv_heads = (uint32_t)pick(1, 8); a.group = (uint32_t)pick(1, 9);
        a.window = pick(0, 1) ? 0 : (uint32_t)pick(1, 300);
        static const unsigned long long word = 0;
        if (pick(0, 1)) { a.mask = &word; a.mask_words = (uint32_t)pick(1, 2); }
        const uint32_t grid = (uint32_t)(pick(0, 1) ? 296 : pick(1, 500));
        walk<8, 16>(a, grid);
        walk<16, 16>(a, 3 * grid);
        walk<128, 32>(a, grid);
        walk<128, 64>(a, grid);
        walk<128, 128>(a, grid);
        CHECK(bad || error == 0);
    }
}

// What lands in shared memory: every 16-byte piece of a tile at a place of its own, inside of the codes.
template <int D, int BITS>
static void tile_places() {
    using S = TilesShape<D, BITS>;
    for (uint32_t rows : {(uint32_t)S::MT, (uint32_t)S::TILE}) {
        std::set<uint32_t> at;
        for (uint32_t r = 0; r < rows; ++r)
            for (uint32_t c = 0; c < D / 8; ++c) {
                const uint32_t x = S::chunk_at(rows, r, c);
                CHECK(x % 16 == 0 && x + 16 <= rows * D * 2 && at.insert(x).second);
            }
    }
    // every piece of a tile belongs to one thread's turn
    CHECK(S::UNPACK % S::K_ROW == 0 && S::UNPACK % S::V_ROW == 0 && S::K_EACH * S::UNPACK == S::TILE * S::K_ROW && sizeof(TilesMeta<S::TILE>) <= S::META);
    CHECK(S::OFF_K % 1024 == 0 && S::OFF_V % 1024 == 0 && S::OFF_META % 16 == 0 && S::OFF_KC % 16 == 0 && S::OFF_VC % 16 == 0 && S::OFF_PL % 16 == 0 && S::OFF_KW % 16 == 0 && S::OFF_VW % 16 == 0 && S::K_BYTES % 1024 == 0 && S::V_BYTES % 1024 == 0 && S::SMEM <= 227 * 1024);
}
template <int D, int BITS, int RB>
static void rows_places() {
    using S = RowsShape<D, BITS, RB>;
    std::set<uint32_t> k, v;
    for (uint32_t r = 0; r < kRowsTile; ++r)
        for (uint32_t p = 0; p < S::PIECES; ++p) {
            const uint32_t x = S::k_at(r, p * 16), y = S::v_at(r, p * 16);
            CHECK(x % 16 == 0 && y % 16 == 0 && x + 16 <= S::CODES && y + 16 <= S::CODES);
            CHECK(k.insert(x).second && v.insert(y).second);
            for (uint32_t byte = 0; byte < 16; byte += 2) CHECK(S::k_at(r, p * 16 + byte) == x + byte && S::v_at(r, p * 16 + byte) == y + byte);
        }
    CHECK(kRowsTile * S::PIECES % kWarp == 0 && S::SWAP % 16 == 0);
    CHECK(S::STAGES >= 2 && S::STAGES <= 31 && S::BLOCKS * (S::SMEM + 1024 + 256) <= 227 * 1024);
}
template <int D, int BITS>
static void places() { tile_places<D, BITS>(); rows_places<D, BITS, 8>(); }

// Refusals: none of them reaches the device.
static tf_context context;
static void refused(tf_status got, tf_status want, const char* words) {
    if (got != want || std::string(tf_last_error(&context)).find(words) == std::string::npos) {
        std::printf("got %d (%s), expected %d with \"%s\"\n", got, tf_last_error(&context), want, words);
        std::exit(1);
    }
}
alignas(16) static uint8_t mem[4096];
static void refusals() {
    int32_t* ints = reinterpret_cast<int32_t*>(mem);
    const tf_kv_cache cache = {mem, mem, mem, mem, mem, mem, 4, 16, 2, 64, 8};
    const tf_kv_batch batch = {ints, ints, ints, ints, 3, 1, 2};
    tf_attention_workspace ws;
    ws.head_dim = 64;
    auto attend = [&](tf_kv_cache c, tf_kv_batch b, uint32_t q_stride = 256, uint32_t heads = 4, uint32_t words = 0, uint32_t window = 0, float scale = 1.0f,
                      int dtype = TF_FP16, const void* q = mem, tf_attention_workspace* w = nullptr, const uint64_t* mask = nullptr) {
        return tf_tree_attention(&context, nullptr, q, q_stride, mem, 256, &c, &b, mask, words, window, scale, heads, (tf_dtype)dtype, w ? w : &ws);
    };
    const uint64_t* mask = reinterpret_cast<const uint64_t*>(mem);
    tf_kv_cache c = cache; tf_kv_batch b = batch;
    refused(tf_tree_attention(&context, nullptr, mem, 256, mem, 256, nullptr, &batch, nullptr, 0, 0, 1.0f, 4, TF_FP16, &ws), TF_ERR_INVALID_ARGUMENT, "cache is NULL");
    refused(tf_tree_attention(&context, nullptr, mem, 256, mem, 256, &cache, nullptr, nullptr, 0, 0, 1.0f, 4, TF_FP16, &ws), TF_ERR_INVALID_ARGUMENT, "batch is NULL");
    refused(tf_tree_attention(&context, nullptr, nullptr, 256, mem, 256, &cache, &batch, nullptr, 0, 0, 1.0f, 4, TF_FP16, &ws), TF_ERR_INVALID_ARGUMENT, "NULL buffer");
    refused(tf_tree_attention(&context, nullptr, mem, 256, mem, 256, &cache, &batch, nullptr, 0, 0, 1.0f, 4, TF_FP16, nullptr), TF_ERR_INVALID_ARGUMENT, "workspace");
    c.bits = 5; refused(attend(c, batch), TF_ERR_UNSUPPORTED, "4 or 8 bits"); c = cache;
    c.head_dim = 96; refused(attend(c, batch), TF_ERR_UNSUPPORTED, "head_dim 96"); c = cache;
    for (uint32_t p : {0u, 8u, 24u, 131072u}) { c.page_size = p; refused(attend(c, batch), TF_ERR_UNSUPPORTED, "page_size"); } c = cache;
    c.num_pages = 0; refused(attend(c, batch), TF_ERR_INVALID_ARGUMENT, "num_pages"); c = cache;
    c.kv_heads = 0; refused(attend(c, batch), TF_ERR_INVALID_ARGUMENT, "kv_heads"); c = cache;
    c.v_biases = nullptr; refused(attend(c, batch), TF_ERR_INVALID_ARGUMENT, "NULL cache plane"); c = cache;
    c.k_codes = mem + 8; refused(attend(c, batch), TF_ERR_ALIGNMENT, "planes"); c = cache;
    c.head_dim = 128; refused(attend(c, batch), TF_ERR_DIMENSION_MISMATCH, "heads of 64"); c = cache;
    b.page_table = nullptr; refused(attend(cache, b), TF_ERR_INVALID_ARGUMENT, "NULL array"); b = batch;
    b.page_table_stride = 0; refused(attend(cache, b), TF_ERR_INVALID_ARGUMENT, "page_table_stride"); b = batch;
    b.rows = 0x80000000u; refused(attend(cache, b), TF_ERR_INVALID_ARGUMENT, "below 2^31"); b = batch;
    b.context_lengths = reinterpret_cast<int32_t*>(mem + 2); refused(attend(cache, b), TF_ERR_ALIGNMENT, "batch arrays"); b = batch;
    refused(attend(cache, batch, 248), TF_ERR_INVALID_ARGUMENT, "stride");
    refused(attend(cache, batch, 260), TF_ERR_ALIGNMENT, "multiples of 8");
    refused(attend(cache, batch, 256, 3), TF_ERR_INVALID_ARGUMENT, "share");
    refused(attend(cache, batch, 256, 0), TF_ERR_INVALID_ARGUMENT, "share");
    refused(attend(cache, batch, 256, 4, 0, 0, 1.0f, TF_FP16, mem, nullptr, mask), TF_ERR_INVALID_ARGUMENT, "mask_words");
    refused(attend(cache, batch, 256, 4, 1, 0, 1.0f, TF_FP16, mem, nullptr, reinterpret_cast<const uint64_t*>(mem + 4)), TF_ERR_ALIGNMENT, "tree_mask");
    b.positions = nullptr;
    refused(attend(cache, b, 256, 4, 1, 9, 1.0f, TF_FP16, mem, nullptr, mask), TF_ERR_INVALID_ARGUMENT, "positions"); b = batch;
    refused(attend(cache, batch, 256, 4, 0, 0x80000000u), TF_ERR_INVALID_ARGUMENT, "window");
    refused(attend(cache, batch, 256, 4, 0, 0, INFINITY), TF_ERR_INVALID_ARGUMENT, "finite");
    refused(attend(cache, batch, 256, 4, 0, 0, 1.0f, 2), TF_ERR_UNSUPPORTED, "fp16 or bf16");
    refused(attend(cache, batch, 256, 4, 0, 0, 1.0f, TF_FP16, mem + 2), TF_ERR_ALIGNMENT, "16-byte");
    tf_attention_workspace other = ws;
    other.device = 1;
    refused(attend(cache, batch, 256, 4, 0, 0, 1.0f, TF_FP16, mem, &other), TF_ERR_INVALID_ARGUMENT, "device");
    b.rows = 0x7FFFFFFFu; refused(attend(cache, b), TF_ERR_UNSUPPORTED, "2^31"); b = batch;

    refused(tf_kv_cache_read(&context, nullptr, &cache, &batch, nullptr, 0, nullptr, 0, TF_FP16), TF_ERR_INVALID_ARGUMENT, "NULL buffer");
    refused(tf_kv_cache_read(&context, nullptr, &cache, &batch, mem, 120, nullptr, 0, TF_FP16), TF_ERR_INVALID_ARGUMENT, "stride");
    refused(tf_kv_cache_read(&context, nullptr, &cache, &batch, mem, 132, nullptr, 0, TF_FP16), TF_ERR_ALIGNMENT, "multiples of 8");
    refused(tf_kv_cache_read(&context, nullptr, &cache, &batch, mem, 128, mem + 2, 128, TF_FP16), TF_ERR_ALIGNMENT, "16-byte");
    refused(tf_kv_cache_read(&context, nullptr, &cache, &batch, mem, 128, mem, 128, (tf_dtype)7), TF_ERR_UNSUPPORTED, "fp16 or bf16");

    struct E { const void* q = mem; const void* k = mem + 512; const void* v = mem + 1024; uint32_t qs = 256, ks = 128, vs = 128; const void* w = nullptr; const float* f = nullptr;
               uint32_t pairs = 0; float eps = 1e-6f; void* qo = mem + 2048; void* ko = nullptr; uint32_t kos = 0; void* vo = nullptr; uint32_t vos = 0; uint32_t heads = 4, kv = 2, dim = 64; int dtype = TF_FP16; };
    auto write = [&](E e, const tf_kv_cache* cc, tf_kv_batch bb) {
        return tf_qkv_epilogue(&context, nullptr, e.q, e.qs, e.k, e.ks, e.v, e.vs, e.w, e.w, 0, e.f, e.pairs, e.eps, e.qo, 256, e.ko, e.kos, e.vo, e.vos, &bb, cc, e.heads, e.kv, e.dim,
                               (tf_dtype)e.dtype);
    };
    const float* freq = reinterpret_cast<const float*>(mem);
    E e;
    e.q = nullptr; refused(write(e, &cache, batch), TF_ERR_INVALID_ARGUMENT, "NULL buffer"); e = E();
    refused(write(e, nullptr, batch), TF_ERR_INVALID_ARGUMENT, "k_out and v_out"); e = E();
    e.dtype = 3; refused(write(e, &cache, batch), TF_ERR_UNSUPPORTED, "fp16 or bf16"); e = E();
    e.dim = 80; refused(write(e, &cache, batch), TF_ERR_UNSUPPORTED, "head_dim 80"); e = E();
    e.heads = 0; refused(write(e, &cache, batch), TF_ERR_INVALID_ARGUMENT, "head counts"); e = E();
    e.kv = 1; refused(write(e, &cache, batch), TF_ERR_DIMENSION_MISMATCH, "the cache has 2 heads"); e = E();
    e.ks = 120; refused(write(e, &cache, batch), TF_ERR_INVALID_ARGUMENT, "stride"); e = E();
    e.vs = 130; refused(write(e, &cache, batch), TF_ERR_ALIGNMENT, "multiples of 8"); e = E();
    e.w = mem + 2; refused(write(e, &cache, batch), TF_ERR_ALIGNMENT, "16-byte"); e = E();
    e.pairs = 3; e.f = freq; refused(write(e, &cache, batch), TF_ERR_UNSUPPORTED, "rotated_pairs 3"); e = E();
    e.pairs = 34; e.f = freq; refused(write(e, &cache, batch), TF_ERR_UNSUPPORTED, "rotated_pairs 34"); e = E();
    e.pairs = 32; refused(write(e, &cache, batch), TF_ERR_INVALID_ARGUMENT, "frequencies"); e = E();
    b.positions = nullptr; e.pairs = 32; e.f = freq; refused(write(e, &cache, b), TF_ERR_INVALID_ARGUMENT, "positions"); e = E(); b = batch;
    e.v = e.k; e.ko = const_cast<void*>(e.k); e.kos = 128; refused(write(e, &cache, batch), TF_ERR_INVALID_ARGUMENT, "both k and v"); e = E();
    e.eps = -1.0f; refused(write(e, &cache, batch), TF_ERR_INVALID_ARGUMENT, "eps"); e = E();
    e.eps = NAN; refused(write(e, &cache, batch), TF_ERR_INVALID_ARGUMENT, "eps"); e = E();
    b.row_offsets = nullptr; refused(write(e, &cache, b), TF_ERR_INVALID_ARGUMENT, "NULL array"); b = batch;

    tf_attention_workspace* made = &ws;
    refused(tf_attention_workspace_create(&context, 100, &made), TF_ERR_UNSUPPORTED, "head_dim 100");
    CHECK(made == nullptr);
    refused(tf_attention_workspace_create(&context, 64, nullptr), TF_ERR_INVALID_ARGUMENT, "NULL");
    CHECK(tf_tree_attention(nullptr, nullptr, mem, 256, mem, 256, &cache, &batch, nullptr, 0, 0, 1.0f, 4, TF_FP16, &ws) == TF_ERR_INVALID_ARGUMENT);
    CHECK(tf_qkv_epilogue(nullptr, nullptr, mem, 256, mem, 128, mem, 128, nullptr, nullptr, 0, nullptr, 0, 0.0f, mem, 256, nullptr, 0, nullptr, 0, &batch, &cache, 4, 2, 64, TF_FP16) ==
          TF_ERR_INVALID_ARGUMENT);
    CHECK(tf_kv_cache_read(nullptr, nullptr, &cache, &batch, mem, 128, nullptr, 0, TF_FP16) == TF_ERR_INVALID_ARGUMENT);
    tf_attention_workspace_destroy(nullptr);
    CHECK(tf_attention_workspace_bytes(nullptr) == 0);
}

int main() {
    divisions();
    all_shares();
    places<64, 4>(); places<64, 8>(); places<128, 4>(); places<128, 8>(); places<256, 4>(); places<256, 8>(); places<512, 4>(); places<512, 8>();
    refusals();
    std::printf("all fine\n");
    return 0;
}
'''


def test_shares_addresses_and_refusals(tmp_path):
    from turbo_fieldfare_b200 import build as tf_build
    lib = tf_build.build(verbose=False)
    src = tmp_path / "attention_host.cu"
    src.write_text(SRC)
    exe = tmp_path / "attention_host"
    cmd = [tf_build.nvcc_path(), *tf_build.ARCH_FLAGS, "-std=c++17", "-O1", "--expt-relaxed-constexpr", "-I", str(ROOT / "include"), "-I", str(tf_build.CSRC), str(src),
           "-o", str(exe), "-L", str(lib.parent), "-ltfcuda", "-Xlinker", f"-rpath={lib.parent}"]
    built = subprocess.run(cmd, capture_output=True, text=True)
    assert built.returncode == 0, built.stdout + built.stderr
    run = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and "all fine" in run.stdout, run.stdout + run.stderr


def _planes(pages=3, heads=2, page=16, dim=64, bits=8):
    codes = lambda: torch.zeros(pages, heads, page, dim * bits // 8, dtype=torch.uint8)  # noqa: E731
    half = lambda: torch.zeros(pages, heads, page, dim // 64, dtype=torch.bfloat16)  # noqa: E731
    return [codes(), half(), half(), codes(), half(), half()]


def test_cache_of_planes():
    from turbo_fieldfare_b200.attention import KVCache
    for dim, bits in ((64, 8), (128, 4), (512, 8)):
        c = KVCache(*_planes(dim=dim, bits=bits))
        assert (c.num_pages, c.kv_heads, c.page_size, c.head_dim, c.bits) == (3, 2, 16, dim, bits)
        assert c.nbytes == 2 * 3 * 2 * 16 * (dim * bits // 8 + 4 * (dim // 64))
        assert KVCache.allocate(3, 16, 2, dim, bits, device="cpu").nbytes == c.nbytes
    for i, change in ((0, lambda t: t[:, :, :, :60]), (0, lambda t: t.float()), (1, lambda t: t[:, :1].contiguous()), (3, lambda t: t[..., :32].contiguous()),
                      (4, lambda t: t.half()), (5, lambda t: t.transpose(0, 1)), (2, lambda t: t[0])):
        p = _planes()
        p[i] = change(p[i])
        with pytest.raises(ValueError):
            KVCache(*p)


def test_batch_of_arrays():
    from turbo_fieldfare_b200.attention import KVBatch
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    table = torch.zeros(2, 5, dtype=torch.int32)
    assert KVBatch(i32(0, 2, 3), i32(4, 5), table).rows == 3
    assert KVBatch(i32(0, 2, 3), i32(4, 5), table, i32(4, 5, 5, 0)).rows == 4
    assert KVBatch(i32(0, 2, 3), i32(4, 5), table, rows=9).rows == 9
    for args, more in (((i32(0, 2), i32(4, 5), table), {}), ((i32(0, 2, 3).long(), i32(4, 5), table), {}), ((i32(0, 2, 3), i32(4, 5), table[:1]), {}),
                       ((i32(0, 2, 3), i32(4, 5), table[:, :3]), {}), ((i32(0, 2, 3), i32(4, 5), table, i32(1)), {"rows": 3}), ((i32(0, 2, 3), i32(4, 5), table), {"rows": -1})):
        with pytest.raises(ValueError):
            KVBatch(*args, **more)


def test_tensors_elsewhere_are_refused():
    """Host tensors never reach the library, whose pointers are device pointers."""
    from turbo_fieldfare_b200 import attention as at
    context = type("Context", (), {"device": 0})()
    cache = at.KVCache(*_planes())
    batch = at.KVBatch(torch.zeros(2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32), torch.zeros(1, 3, dtype=torch.int32), rows=1)
    x = torch.zeros(1, 128, dtype=torch.float16)
    with pytest.raises(ValueError, match="cuda:0"):
        at.TreeAttention(context).encode(x, x, cache, batch, None, scale=1.0)
    with pytest.raises(ValueError, match="cuda:0"):
        at.KVCacheRead(context).encode(cache, batch, x)
    with pytest.raises(ValueError, match="cuda:0"):
        at.FusedQKVEpilogue(context).encode(x, x, x, x, batch, cache, head_dim=64)


def test_rows_of_tensors():
    from turbo_fieldfare_b200.attention import _row_stride
    cpu = torch.device("cpu")
    x = torch.zeros(4, 96, dtype=torch.float16)
    assert _row_stride("x", x, cpu, torch.float16, 4, 96) == 96
    assert _row_stride("x", x[:, :64], cpu, torch.float16, 3, 64) == 96
    assert _row_stride("x", x[:1, :64], cpu, torch.float16, 1, 64) >= 64
    for t, rows, cols in ((x, 5, 96), (x, 4, 95), (x.t(), 4, 4), (x.float(), 4, 96), (x[0], 1, 96), (x[:, ::2], 4, 48)):
        with pytest.raises(ValueError):
            _row_stride("x", t, cpu, torch.float16, rows, cols)


MIRROR = r'''
#include <cstdio>
#include "turbofieldfare.hpp"
namespace tf = turbofieldfare;
int main() {
    try {
        tf::Context ctx(0);
        alignas(16) static char mem[64];
        const tf_kv_cache cache = {mem, mem, mem, mem, mem, mem, 1, 16, 1, 64, 5};
        const tf_kv_batch batch = {};
        tf::AttentionWorkspace workspace(ctx, 64);
        int refused = 0;
        auto expect = [&](auto call) { try { call(); } catch (const tf::Error&) { ++refused; } };
        expect([&] { tf::TreeAttention(ctx).encode(nullptr, {mem, 64}, {mem, 64}, cache, batch, workspace, 1, 1.0f); });
        expect([&] { tf::KVCacheRead(ctx).encode(nullptr, cache, batch, {mem, 64}, {}); });
        expect([&] { tf::FusedQKVEpilogue(ctx).encode(nullptr, {mem, 64}, {mem, 64}, {mem, 64}, {mem, 64}, batch, &cache, 1, 1, 64); });
        expect([&] { tf::AttentionWorkspace bad(ctx, 96); });
        std::printf("refused %d\n", refused);
        return refused == 4 ? 0 : 1;
    } catch (const tf::Error& e) {
        std::printf("status %d\n", e.status);
        return e.status == TF_ERR_NO_DEVICE ? 0 : 2;
    }
}
'''


def test_cpp_mirror_of_the_attention_calls(tmp_path):
    """The classes of include/turbofieldfare.hpp compile, link, and hand on what the library refuses (no work on a device)."""
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("no g++")
    from turbo_fieldfare_b200 import build as tf_build
    lib = tf_build.build(verbose=False)
    src, exe = tmp_path / "mirror.cpp", tmp_path / "mirror"
    src.write_text(MIRROR)
    subprocess.run([gxx, "-std=c++17", "-O1", "-Wall", "-Werror", "-I", str(ROOT / "include"), "-I", "/usr/local/cuda/include", str(src), "-o", str(exe),
                    "-L", str(lib.parent), "-ltfcuda", f"-Wl,-rpath,{lib.parent}"], check=True, capture_output=True, text=True)
    run = subprocess.run([str(exe)], capture_output=True, text=True)
    assert run.returncode == 0, run.stdout + run.stderr
