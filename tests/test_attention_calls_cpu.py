"""Calls of the attention classes that are refused, or do nothing, before anything reaches a device."""
import pytest
import torch


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
