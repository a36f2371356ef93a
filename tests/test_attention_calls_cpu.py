"""Calls of the attention classes that are refused, or do nothing, before anything reaches a device."""
import subprocess
from pathlib import Path

import pytest
import torch

ROOT = Path(__file__).resolve().parent.parent


class _Library:
    """Stands for the library where no call may reach it."""

    def __getattr__(self, name):
        raise AssertionError(f"{name} was called")


def _context():
    return type("Context", (), {"device": -1, "lib": _Library(), "handle": None})()         # the device of host tensors


def _cache(dim=64):
    from turbo_fieldfare_b200.attention import KVCache
    return KVCache.allocate(3, 16, 2, dim, 8, device="cpu")


def _batch(rows):
    from turbo_fieldfare_b200.attention import KVBatch
    i32 = dict(dtype=torch.int32)
    return KVBatch(torch.tensor([0, rows], **i32), torch.zeros(1, **i32), torch.zeros(1, 3, **i32), torch.zeros(rows, **i32))


def _attend(rows=2, **more):
    from turbo_fieldfare_b200 import attention as at
    q = torch.zeros(rows, 4 * 64, dtype=torch.float16)
    workspace = type("Workspace", (), {"handle": None})()
    at.TreeAttention(_context()).encode(q, torch.zeros_like(q), _cache(), _batch(rows), workspace, scale=1.0, **more)


def test_a_mask_without_words_is_refused():
    with pytest.raises(ValueError, match="no words"):
        _attend(tree_mask=torch.zeros(2, 0, dtype=torch.int64))


@pytest.mark.parametrize("window", [-1, 1 << 31, 1 << 32, (1 << 32) + 5])
def test_windows_beyond_31_bits_are_refused(window):
    with pytest.raises(ValueError, match="window"):
        _attend(window=window)


def test_strides_beyond_32_bits_are_refused():
    from turbo_fieldfare_b200.attention import _row_stride
    far = torch.empty_strided((2, 64), ((1 << 32) + 64, 1), dtype=torch.float16, device="meta")
    with pytest.raises(ValueError, match="apart"):
        _row_stride("x", far, far.device, torch.float16, 2, 64)
    assert _row_stride("x", far[:1], far.device, torch.float16, 1, 64) == 64       # a lone row has no next one


SRC = r'''
#include <cstdio>
#include <cstdlib>
#include <string>
#include "attention_launch.cuh"
static tf_context context;
alignas(16) static uint8_t mem[4096];
static void answers(int line, tf_status got, tf_status want, const char* words = "") {
    if (got == want && std::string(want == TF_OK ? "" : tf_last_error(&context)).find(words) != std::string::npos) return;
    std::printf("line %d: got %d (%s), expected %d with \"%s\"\n", line, got, tf_last_error(&context), want, words);
    std::exit(1);
}
#define ANSWERS(...) answers(__LINE__, __VA_ARGS__)
int main() {
    int32_t* ints = reinterpret_cast<int32_t*>(mem);
    const tf_kv_cache cache = {mem, mem, mem, mem, mem, mem, 4, 16, 2, 64, 8};
    tf_attention_workspace ws;
    ws.head_dim = 64;
    const tf_kv_batch empty = {nullptr, nullptr, nullptr, nullptr, 0, 1, 0}, batch = {ints, ints, ints, ints, 3, 1, 2};
    const uint64_t* mask = reinterpret_cast<const uint64_t*>(mem);
    const float* turns = reinterpret_cast<const float*>(mem);
    // calls without rows do nothing, with or without buffers
    ANSWERS(tf_tree_attention(&context, nullptr, nullptr, 256, nullptr, 256, &cache, &empty, nullptr, 0, 0, 1.0f, 4, TF_FP16, &ws), TF_OK);
    ANSWERS(tf_tree_attention(&context, nullptr, mem, 256, mem, 256, &cache, &empty, mask, 1, 9, 1.0f, 4, TF_FP16, &ws), TF_OK);
    ANSWERS(tf_kv_cache_read(&context, nullptr, &cache, &empty, nullptr, 0, nullptr, 0, TF_FP16), TF_OK);
    for (const tf_kv_cache* c : {&cache, (const tf_kv_cache*)nullptr})
        ANSWERS(tf_qkv_epilogue(&context, nullptr, nullptr, 256, nullptr, 128, nullptr, 128, nullptr, nullptr, 0, turns, 32, 0.0f, nullptr, 256, nullptr, 0, nullptr, 0, &empty, c, 4, 2, 64,
                                TF_FP16), TF_OK);
    ANSWERS(tf_tree_attention(&context, nullptr, nullptr, 256, nullptr, 256, &cache, nullptr, nullptr, 0, 0, 1.0f, 4, TF_FP16, &ws), TF_ERR_INVALID_ARGUMENT, "NULL");
    ANSWERS(tf_kv_cache_read(&context, nullptr, &cache, &batch, nullptr, 0, nullptr, 0, TF_FP16), TF_ERR_INVALID_ARGUMENT, "NULL buffer");
    // outputs over their inputs have the inputs' stride
    ANSWERS(tf_tree_attention(&context, nullptr, mem, 256, mem, 264, &cache, &batch, nullptr, 0, 0, 1.0f, 4, TF_FP16, &ws), TF_ERR_INVALID_ARGUMENT, "same stride");
    for (int which = 0; which < 3; ++which)
        ANSWERS(tf_qkv_epilogue(&context, nullptr, mem, 256, mem + 512, 128, mem + 1024, 128, nullptr, nullptr, 0, nullptr, 0, 0.0f, which == 0 ? mem : mem + 1536, which == 0 ? 264 : 256,
                                which == 1 ? mem + 512 : nullptr, 136, which == 2 ? mem + 1024 : nullptr, 136, &batch, &cache, 4, 2, 64, TF_FP16),
                TF_ERR_INVALID_ARGUMENT, "same stride");
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
