"""Calls of a step with drafted tokens that are refused, or do nothing, before anything reaches a device."""
import subprocess
from pathlib import Path

import numpy as np
import pytest
import torch

import drafts_reference as ref

ROOT = Path(__file__).resolve().parent.parent
I32 = dict(dtype=torch.int32)


class _Library:
    """Stands for the library: keeps the calls that reach it."""

    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        return lambda *a: self.calls.append(name) or 0


def _context():
    lib = _Library()
    return type("Context", (), {"device": -1, "lib": lib, "handle": None, "check": lambda self, status: None})()


def _plan(**more):
    from turbo_fieldfare_b200 import drafts as dr
    a = dict(sequences=3, context=torch.zeros(3, **I32), wanted=torch.zeros(3, **I32), rows=dr.KVRows.allocate(3, 8, mask_words=1, tokens=True, device="cpu"))
    a.update({k: v for k, v in more.items() if k in a})
    call = {k: v for k, v in more.items() if k not in a}
    call.setdefault("tokens", torch.zeros(3, 4, **I32))
    ctx = _context()
    dr.KVPlan(ctx).encode(dr.KVPages.allocate(3, 4, 9, 16, device="cpu"), a["context"], a["wanted"], a["rows"], stream=0, **call)
    return ctx.lib.calls


def test_a_plan_reaches_the_library():
    assert _plan() == ["tf_kv_plan"] and _plan(parents=torch.zeros(3, 4, **I32), kept=torch.zeros(3, **I32), window=7) == ["tf_kv_plan"]


@pytest.mark.parametrize("more,words", [
    (dict(context=torch.zeros(4, **I32)), "context_lengths"), (dict(wanted=torch.zeros(3)), "new_rows"), (dict(kept=torch.zeros(3, dtype=torch.int64)), "kept"),
    (dict(window=-1), "window"), (dict(window=1 << 31), "window"), (dict(tokens=torch.zeros(2, 4, **I32)), "tokens"), (dict(parents=torch.zeros(3, 5, **I32)), "parents"),
    (dict(tokens=torch.zeros(3, 8, **I32)[:, ::2]), "contiguous"), (dict(tokens=None, nodes=0), "nodes"), (dict(wanted=torch.zeros(6, **I32)[::2]), "contiguous")])
def test_plans_of_other_shapes_are_refused(more, words):
    with pytest.raises(ValueError, match=words):
        _plan(**more)


def test_descriptors_of_other_shapes_are_refused():
    from turbo_fieldfare_b200 import drafts as dr
    z = lambda *s, **k: torch.zeros(*s, **(k or I32))  # noqa: E731
    with pytest.raises(ValueError, match="held_pages"):
        dr.KVPages(z(2, 3), z(3), z(9), z(1), 16)
    with pytest.raises(ValueError, match="free_count"):
        dr.KVPages(z(2, 3), z(2), z(9), z(2), 16)
    with pytest.raises(ValueError, match="slots"):
        dr.KVRows(z(3), z(5), slots=z(5))
    with pytest.raises(ValueError, match="tokens has"):
        dr.KVRows(z(3), z(5), tokens=z(4))
    with pytest.raises(ValueError, match="tree_mask"):
        dr.KVRows(z(3), z(5), tree_mask=z(5, 0, dtype=torch.int64))
    ctx = _context()
    with pytest.raises(ValueError, match="row offsets"):
        dr.KVPlan(ctx).encode(dr.KVPages.allocate(2, 3, 9, 16, device="cpu"), z(2), z(2), dr.KVRows.allocate(3, 5, device="cpu"), stream=0)


def _verify(**more):
    from turbo_fieldfare_b200 import drafts as dr
    a = dict(logits=torch.zeros(5, 7), row_offsets=torch.zeros(3, **I32), tokens=torch.zeros(2, 4, **I32), uniforms=torch.zeros(2, 4), out_tokens=torch.zeros(2, 4, **I32),
             out_rows=torch.zeros(2, 4, **I32), kept=torch.zeros(2, **I32))
    a.update({k: v for k, v in more.items() if k in a})
    ctx = _context()
    dr.DraftVerification(ctx).encode(*a.values(), type("Workspace", (), {"handle": None})(), stream=0, **{k: v for k, v in more.items() if k not in a})
    return ctx.lib.calls


def test_a_verification_reaches_the_library():
    assert _verify() == ["tf_verify_drafts"]
    assert _verify(draft_probs=torch.zeros(2, 3, 7).half(), temperatures=torch.ones(2), logprobs=torch.zeros(2, 4), parents=torch.zeros(2, 4, **I32)) == ["tf_verify_drafts"]


@pytest.mark.parametrize("more,words", [
    (dict(logits=torch.zeros(5, 7, dtype=torch.float64)), "logits"), (dict(logits=torch.zeros(7)), "logits"), (dict(logits=torch.zeros(7, 5).T), "next to one another"),
    (dict(logits=torch.zeros(5, 0)), "one at the least"), (dict(row_offsets=torch.zeros(0, **I32)), "empty"), (dict(tokens=None), "tokens"), (dict(tokens=torch.zeros(3, 4, **I32)), "tokens"),
    (dict(uniforms=torch.zeros(2, 3)), "uniforms"), (dict(uniforms=torch.zeros(2, 4).double()), "uniforms"), (dict(out_rows=torch.zeros(2, 5, **I32)), "out_rows"),
    (dict(kept=torch.zeros(3, **I32)), "kept"), (dict(temperatures=torch.ones(3)), "temperatures"), (dict(logprobs=torch.zeros(2, 3)), "logprobs"),
    (dict(draft_probs=torch.zeros(2, 3, 8)), "draft_probs"), (dict(draft_probs=torch.zeros(2, 7, 3).transpose(1, 2)), "next to one another"),
    (dict(draft_probs=torch.zeros(2, 3, 7).int()), "draft_probs")])
def test_verifications_of_other_shapes_are_refused(more, words):
    with pytest.raises(ValueError, match=words):
        _verify(**more)


def test_kept_rows_of_other_shapes_are_refused():
    from turbo_fieldfare_b200 import attention as at
    from turbo_fieldfare_b200 import drafts as dr
    cache = at.KVCache.allocate(3, 16, 2, 64, 8, device="cpu")
    batch = at.KVBatch(torch.tensor([0, 2], **I32), torch.zeros(1, **I32), torch.zeros(1, 3, **I32), rows=2)
    ctx = _context()
    keep = dr.KVCacheKeep(ctx)
    keep.encode([cache], batch, torch.zeros(1, 4, **I32), torch.zeros(1, **I32), stream=0)
    keep.encode(cache, batch, torch.zeros(1, 4, **I32), torch.zeros(1, **I32), stream=0)
    assert ctx.lib.calls == ["tf_kv_cache_keep"] * 2
    for rows, kept, words in ((torch.zeros(2, 4, **I32), torch.zeros(1, **I32), "kept_rows"), (torch.zeros(4, **I32), torch.zeros(1, **I32), "kept_rows"),
                              (torch.zeros(1, 4), torch.zeros(1, **I32), "kept_rows"), (torch.zeros(1, 4, **I32), torch.zeros(2, **I32), "kept")):
        with pytest.raises(ValueError, match=words):
            keep.encode(cache, batch, rows, kept, stream=0)


# ---------------------------------------------------------------------------
# the plain statement itself
# ---------------------------------------------------------------------------

def test_the_plain_verification_keeps_the_targets_distribution():
    """Over all random numbers a chain of one draft leaves the first token with the target's probabilities: by counting a grid of numbers for every drafted token."""
    g = torch.Generator().manual_seed(0)
    p, q = (torch.softmax(torch.randn(5, generator=g) * 1.5, 0).double() for _ in range(2))
    got = np.zeros(5)
    grid = (np.arange(60) + 0.5) / 60
    for x in range(5):
        for u in grid:
            for v in grid:
                tokens, _, kept, _ = ref.verify(torch.stack((p.log(), p.log())), [0, 2], [[0, x]], [[v, u]], probs=q.view(1, 1, 5), nodes=2)
                got[tokens[0, 0]] += float(q[x]) / 3600
    assert np.abs(got - p.numpy()).max() < 5 / 60                  # a border of the grid is off by a step at the most


SRC = r'''
#include <cstdio>
#include <cstdlib>
#include <string>
#include "kv_cache.cuh"
static tf_context context;
alignas(16) static uint8_t mem[8192];
static void answers(int line, tf_status got, tf_status want, const char* words = "") {
    if (got == want && std::string(want == TF_OK ? "" : tf_last_error(&context)).find(words) != std::string::npos) return;
    std::printf("line %d: got %d (%s), expected %d with \"%s\"\n", line, got, tf_last_error(&context), want, words);
    std::exit(1);
}
#define ANSWERS(...) answers(__LINE__, __VA_ARGS__)
template <typename T, typename F> static T with(T v, F f) { f(v); return v; }
int main() {
    int32_t* ints = reinterpret_cast<int32_t*>(mem);
    float* floats = reinterpret_cast<float*>(mem);
    const tf_drafts drafts = {ints, ints, 4};
    // ---- plans ----
    const tf_kv_pages pages = {ints, ints, ints, ints, ints, 4, 9, 16, 2};
    const tf_kv_rows rows = {ints, ints, ints, reinterpret_cast<int64_t*>(mem), ints, reinterpret_cast<uint64_t*>(mem), 1, 8};
    auto plan = [&](const tf_kv_pages& p, const tf_kv_rows& r, const tf_drafts* d = nullptr, uint32_t window = 0, int32_t* lengths = nullptr) {
        return tf_kv_plan(&context, nullptr, &p, lengths ? lengths : ints, ints, nullptr, window, d, &r);
    };
    ANSWERS(tf_kv_plan(&context, nullptr, nullptr, ints, ints, nullptr, 0, nullptr, &rows), TF_ERR_INVALID_ARGUMENT, "NULL");
    ANSWERS(tf_kv_plan(&context, nullptr, &pages, nullptr, ints, nullptr, 0, &drafts, &rows), TF_ERR_INVALID_ARGUMENT, "NULL array");
    ANSWERS(plan(pages, rows), TF_ERR_INVALID_ARGUMENT, "tokens of rows need drafts");
    ANSWERS(plan(pages, with(rows, [](tf_kv_rows& r) { r.tokens = nullptr; })), TF_ERR_INVALID_ARGUMENT, "tree mask needs drafts");
    ANSWERS(plan(pages, with(rows, [](tf_kv_rows& r) { r.mask_words = 0; }), &drafts), TF_ERR_INVALID_ARGUMENT, "mask_words");
    ANSWERS(plan(pages, with(rows, [](tf_kv_rows& r) { r.positions = nullptr; }), &drafts), TF_ERR_INVALID_ARGUMENT, "positions");
    ANSWERS(plan(pages, with(rows, [](tf_kv_rows& r) { r.row_offsets = nullptr; }), &drafts), TF_ERR_INVALID_ARGUMENT, "row_offsets");
    ANSWERS(plan(pages, with(rows, [](tf_kv_rows& r) { r.slots = reinterpret_cast<int64_t*>(mem + 4); }), &drafts), TF_ERR_ALIGNMENT, "aligned");
    for (uint32_t size : {0u, 8u, 24u, 131072u})
        ANSWERS(plan(with(pages, [&](tf_kv_pages& p) { p.page_size = size; }), rows, &drafts), TF_ERR_UNSUPPORTED, "page_size");
    ANSWERS(plan(with(pages, [](tf_kv_pages& p) { p.page_table_stride = 0; }), rows, &drafts), TF_ERR_INVALID_ARGUMENT, "page_table_stride");
    ANSWERS(plan(with(pages, [](tf_kv_pages& p) { p.num_pages = 0; }), rows, &drafts), TF_ERR_INVALID_ARGUMENT, "num_pages");
    ANSWERS(plan(with(pages, [](tf_kv_pages& p) { p.first_pages = nullptr; }), rows, &drafts, 9), TF_ERR_INVALID_ARGUMENT, "first_pages");
    ANSWERS(plan(pages, rows, &drafts, 0x80000000u), TF_ERR_INVALID_ARGUMENT, "window");
    const tf_drafts none = {ints, ints, 0};
    ANSWERS(plan(pages, rows, &none), TF_ERR_INVALID_ARGUMENT, "stride is 0");
    // ---- verifications ----
    tf_verify_workspace* ws = nullptr;
    ANSWERS(tf_verify_workspace_create(&context, 0, 5, &ws), TF_ERR_INVALID_ARGUMENT, "no rows");
    ANSWERS(tf_verify_workspace_create(&context, 5, 5, nullptr), TF_ERR_INVALID_ARGUMENT, "NULL");
    // a workspace as the library lays it out: device, room, sums, bytes, memory
    struct { int device; uint64_t room, stats, bytes; void* memory; } space = {0, 4, 4, 64, mem}, other = {1, 4, 4, 64, mem};
    ws = reinterpret_cast<tf_verify_workspace*>(&space);
    struct Call {
        const void* logits = mem; uint64_t stride = 64; tf_dtype type = TF_FP16; uint32_t vocab = 64, rows = 4, sequences = 2; const int32_t* offsets; const tf_drafts* drafts;
        const float* uniforms; const tf_draft_probs* probs = nullptr; float cap = 0.0f; int32_t* out; tf_verify_workspace* ws;
    } base;
    base.offsets = ints; base.drafts = &drafts; base.uniforms = floats; base.out = ints; base.ws = ws;
    auto verify = [&](const Call& c) {
        return tf_verify_drafts(&context, nullptr, c.logits, c.stride, c.type, c.vocab, c.offsets, c.rows, c.sequences, c.drafts, c.uniforms, c.probs, nullptr, c.cap, c.out, ints, ints,
                                nullptr, c.ws);
    };
    ANSWERS(verify(with(base, [](Call& c) { c.sequences = 0; })), TF_OK);
    ANSWERS(verify(with(base, [](Call& c) { c.ws = nullptr; })), TF_ERR_INVALID_ARGUMENT, "workspace");
    ANSWERS(verify(with(base, [&](Call& c) { c.ws = reinterpret_cast<tf_verify_workspace*>(&other); })), TF_ERR_INVALID_ARGUMENT, "belongs to device 1");
    ANSWERS(verify(with(base, [](Call& c) { c.drafts = nullptr; })), TF_ERR_INVALID_ARGUMENT, "drafts");
    ANSWERS(verify(with(base, [](Call& c) { c.type = (tf_dtype)3; })), TF_ERR_UNSUPPORTED, "logits are");
    ANSWERS(verify(with(base, [](Call& c) { c.vocab = 0; })), TF_ERR_INVALID_ARGUMENT, "vocab");
    ANSWERS(verify(with(base, [](Call& c) { c.vocab = 0x80000000u; })), TF_ERR_INVALID_ARGUMENT, "vocab");
    ANSWERS(verify(with(base, [](Call& c) { c.stride = 63; })), TF_ERR_INVALID_ARGUMENT, "stride");
    ANSWERS(verify(with(base, [](Call& c) { c.rows = 5; })), TF_ERR_SCRATCH_TOO_SMALL, "room");
    ANSWERS(verify(with(base, [](Call& c) { c.uniforms = nullptr; })), TF_ERR_INVALID_ARGUMENT, "NULL buffer");
    ANSWERS(verify(with(base, [](Call& c) { c.logits = mem + 1; })), TF_ERR_ALIGNMENT, "aligned");
    ANSWERS(verify(with(base, [](Call& c) { c.logits = mem + 2; c.type = TF_FP32; })), TF_ERR_ALIGNMENT, "aligned");
    for (float cap : {-1.0f, (float)(1.0 / 0.0 * 1.0), (float)(0.0 / 0.0)})
        ANSWERS(verify(with(base, [&](Call& c) { c.cap = cap; })), TF_ERR_INVALID_ARGUMENT, "softcap");
    const tf_drafts zero = {ints, ints, 0}, many = {ints, ints, 1025}, untold = {nullptr, ints, 4};
    ANSWERS(verify(with(base, [&](Call& c) { c.drafts = &zero; })), TF_ERR_UNSUPPORTED, "nodes");
    ANSWERS(verify(with(base, [&](Call& c) { c.drafts = &many; })), TF_ERR_UNSUPPORTED, "nodes");
    ANSWERS(verify(with(base, [&](Call& c) { c.drafts = &untold; })), TF_ERR_INVALID_ARGUMENT, "NULL buffer");
    const tf_draft_probs empty = {nullptr, 64, 64, 3, TF_FP32}, close = {mem, 64, 63, 3, TF_FP32}, odd = {mem + 2, 64, 64, 3, TF_FP32}, strange = {mem, 64, 64, 3, (tf_dtype)7};
    ANSWERS(verify(with(base, [&](Call& c) { c.probs = &empty; })), TF_ERR_INVALID_ARGUMENT, "no values");
    ANSWERS(verify(with(base, [&](Call& c) { c.probs = &close; })), TF_ERR_INVALID_ARGUMENT, "stride");
    ANSWERS(verify(with(base, [&](Call& c) { c.probs = &odd; })), TF_ERR_ALIGNMENT, "aligned");
    ANSWERS(verify(with(base, [&](Call& c) { c.probs = &strange; })), TF_ERR_UNSUPPORTED, "probabilities are");
    // ---- kept rows ----
    uint8_t* m = mem;
    tf_kv_cache caches[2] = {{m, m, m, m, m, m, 4, 16, 2, 64, 8}, {m + 64, m, m, m + 64, m, m, 4, 32, 2, 64, 8}};
    const tf_kv_batch batch = {ints, ints, ints, ints, 3, 1, 2}, idle = {nullptr, nullptr, nullptr, nullptr, 0, 1, 0};
    auto keep = [&](uint32_t n, const tf_kv_batch& b, const int32_t* nodes, uint32_t stride = 4) { return tf_kv_cache_keep(&context, nullptr, caches, n, &b, nodes, stride, ints); };
    ANSWERS(keep(0, batch, ints), TF_OK);
    ANSWERS(keep(1, idle, nullptr), TF_OK);
    ANSWERS(keep(1, batch, ints, 0), TF_OK);
    ANSWERS(keep(1, batch, nullptr), TF_ERR_INVALID_ARGUMENT, "NULL array");
    ANSWERS(keep(2, batch, ints), TF_ERR_DIMENSION_MISMATCH, "pages of 32");
    caches[1] = caches[0];
    ANSWERS(keep(2, batch, ints), TF_ERR_INVALID_ARGUMENT, "the same");
    caches[0].bits = 5;
    ANSWERS(keep(1, batch, ints), TF_ERR_UNSUPPORTED, "bits");
    ANSWERS(tf_kv_cache_keep(&context, nullptr, nullptr, 1, &batch, ints, 4, ints), TF_ERR_INVALID_ARGUMENT, "caches");
    // rows of 32 bits are for these calls alone
    ANSWERS(tf_rmsnorm(&context, nullptr, mem, 0, nullptr, 0, mem, 0, 1, 64, 64, 1e-6f, TF_FP32), TF_ERR_UNSUPPORTED, "fp16 or bf16");
    std::printf("all fine\n");
    return 0;
}
'''


def test_calls_of_the_library_without_a_device(tmp_path):
    from turbo_fieldfare_b200 import build as tf_build
    lib = tf_build.build(verbose=False)
    src, exe = tmp_path / "calls.cu", tmp_path / "calls"
    src.write_text(SRC)
    built = subprocess.run([tf_build.nvcc_path(), *tf_build.ARCH_FLAGS, "-std=c++17", "-O1", "--expt-relaxed-constexpr", "-I", str(ROOT / "include"), "-I", str(tf_build.CSRC),
                            str(src), "-o", str(exe), "-L", str(lib.parent), "-ltfcuda", "-Xlinker", f"-rpath={lib.parent}"], capture_output=True, text=True)
    assert built.returncode == 0, built.stdout + built.stderr
    run = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert run.returncode == 0 and "all fine" in run.stdout, run.stdout + run.stderr


CALLER = r"""
#include "turbofieldfare.hpp"
namespace tf = turbofieldfare;
void step(const tf::Context& c, void* stream, tf_kv_pages pages, tf_kv_rows rows, tf_kv_batch batch, tf_kv_cache cache, tf_drafts drafts, int32_t* numbers, float* uniforms,
          const void* logits, const tf::VerificationWorkspace& workspace) {
    tf::KVPlan(c).encode(stream, pages, numbers, numbers, rows, numbers, 0, &drafts);
    tf::DraftVerification(c).encode(stream, {logits, 1000, TF_FP32, 1000}, rows.row_offsets, rows.rows, pages.sequences, drafts, uniforms, {numbers, numbers, numbers}, workspace);
    tf::KVCacheKeep(c).encode(stream, &cache, 1, batch, numbers, drafts.stride, numbers);
}
int main() {
    try {
        tf::Context c(0);
        tf::VerificationWorkspace w(c, 0, 1000);
        return 2;                                  // no rows: refused
    } catch (const tf::Error& e) {
        return e.status == TF_ERR_NO_DEVICE || e.status == TF_ERR_INVALID_ARGUMENT ? 0 : 3;
    }
}
"""


def test_the_cpp_classes_compile_and_raise(tmp_path):
    from turbo_fieldfare_b200 import build as tf_build
    lib = tf_build.build(verbose=False)
    src, exe = tmp_path / "caller.cpp", tmp_path / "caller"
    src.write_text(CALLER)
    built = subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", "-I", str(ROOT / "include"), str(src), "-o", str(exe), "-L", str(lib.parent), "-ltfcuda",
                            f"-Wl,-rpath,{lib.parent}"], capture_output=True, text=True)
    assert built.returncode == 0, built.stderr
    assert subprocess.run([str(exe)], timeout=120).returncode == 0
