"""Page numbers that no cache has, in tables and on the stack of a plan: they are reported and stand as -1 wherever the plan puts them."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
I32 = dict(dtype=torch.int32, device=DEV)


def dev(a):
    return torch.tensor(np.ascontiguousarray(a), **I32)


def reported(ctx):
    from turbo_fieldfare_b200.kernels import TFError
    with pytest.raises(TFError, match="7F000054|7f000054"):
        ctx.device_status()
    assert ctx.device_status() == 0


def planned(ctx, table, held, stack, count, wanted, context, *, rows=64, first=None, window=0, pages=6):
    """One plan over pages of 16 tokens; what it leaves, and the rows."""
    from turbo_fieldfare_b200 import drafts as dr
    n = len(held)
    p = dr.KVPages(dev(table), dev(held), dev(stack), dev([count]), 16, None if first is None else dev(first))
    assert p.num_pages == pages
    into = dr.KVRows(torch.zeros(n + 1, **I32), torch.zeros(rows, **I32), slots=torch.full((rows,), -7, dtype=torch.int64, device=DEV))
    dr.KVPlan(ctx).encode(p, dev(context), dev(wanted), into, window=window)
    torch.cuda.synchronize()
    return p, into


@pytest.mark.parametrize("bad", [-1, -9, 6, 2**31 - 1, -2**31])
@pytest.mark.parametrize("rows", [64, 3000])
def test_pages_that_go_back(tf_ctx, bad, rows):
    """A sequence ends, pages fall out of a window."""
    p, _ = planned(tf_ctx, [[4, bad, 2], [-1, -1, -1]], [3, 0], [0, 1, 7, 7, 7, 7], 2, [-1, 0], [40, 0], rows=rows)
    reported(tf_ctx)
    assert p.free_count.tolist() == [5] and p.free_pages.tolist() == [0, 1, 2, -1, 4, 7]
    assert p.page_table.tolist() == [[-1, -1, -1]] * 2
    p, _ = planned(tf_ctx, [[4, bad, 2]], [3], [0, 1, 7, 7, 7, 7], 2, [0], [40], rows=rows, first=[0], window=9)
    reported(tf_ctx)
    assert p.free_count.tolist() == [4] and p.free_pages.tolist() == [0, 1, -1, 4, 7, 7] and p.page_table.tolist() == [[-1, -1, 2]] and p.first_pages.tolist() == [2]


@pytest.mark.parametrize("bad", [-1, 6, 2**31 - 1, -2**31])
@pytest.mark.parametrize("rows", [64, 3000])
def test_pages_that_are_taken(tf_ctx, bad, rows):
    p, into = planned(tf_ctx, [[-1, -1, -1], [-1, -1, -1]], [0, 0], [5, 3, bad, 1, 7, 7], 4, [20, 17], [0, 0], rows=rows)
    reported(tf_ctx)
    assert p.free_count.tolist() == [0] and p.held_pages.tolist() == [2, 2]
    assert p.page_table.tolist() == [[1, -1, -1], [3, 5, -1]]
    want = list(range(16, 32)) + [-1] * 4 + list(range(48, 64)) + [80]
    assert into.slots.tolist() == want + [-7] * (rows - 37)


@pytest.mark.parametrize("bad", [-1, 6, 2**31 - 1, -2**31])
@pytest.mark.parametrize("rows", [64, 3000])
def test_pages_that_a_row_lies_on(tf_ctx, bad, rows):
    """Held, neither given back nor taken: the rows' slots are -1."""
    p, into = planned(tf_ctx, [[4, bad, -1]], [2], [0, 1, 7, 7, 7, 7], 2, [20], [14], rows=rows)
    reported(tf_ctx)
    assert p.page_table.tolist() == [[4, bad, 1]] and into.slots[:20].tolist() == [78, 79] + [-1] * 16 + [16, 17]


def test_pages_of_other_arrays_are_left_alone(tf_ctx):
    """Entries outside what a sequence holds, and the stack above its count, may hold anything."""
    p, into = planned(tf_ctx, [[99, 3, -8], [-5, 77, 77]], [2, 0], [5, 2, 99, -1, 99, 99], 2, [3, 0], [30, 0], first=[1, 0], window=20)
    assert tf_ctx.device_status() == 0
    assert p.page_table.tolist() == [[99, 3, 2], [-5, 77, 77]] and into.slots[:3].tolist() == [62, 63, 32]
