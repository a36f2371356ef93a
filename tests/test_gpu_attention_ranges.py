"""Attention operators at the ends of their ranges, through both attention kernels: values, keys and queries far from one, planes that are zero,
outputs over inputs, batches of unlike sequences."""
import numpy as np
import pytest
import torch

import attention_reference as ref
from attention_reference import Case, F64, half_step
from test_gpu_attention import BF16, DEV, F16, _close, _definition, _ops, _q, _run, _tree, _words, workspaces  # noqa: F401

pytestmark = pytest.mark.gpu


def _by(case, heads, many):
    """Sends the case to the kernel for many rows or to the one for few: sequences without rows lower the mean that the choice goes by."""
    def takes_many(crowd):
        sequences, rows = len(case.rows) + crowd, sum(case.rows)
        mean, units = -(-rows // sequences) * (heads // case.kv), sequences * case.kv * (4 if case.dim == 512 else 1)
        return mean > (4 if units <= 32 else 16 if units <= 128 else 32)
    case.crowd = 0 if many else next(c for c in range(0, 5000, 10) if not takes_many(c))
    assert takes_many(case.crowd) == many
    return case


def _all_visible(case, window=0):
    return [ref.visible(n, c, window) for n, c in zip(case.rows, case.contexts)]


SHAPES = [([40, 24], [300, 700]), ([5] * 200, [60] * 200)]        # units shared by workers; units that a worker has whole
KINDS = [(64, 8, F16), (128, 4, BF16), (256, 8, BF16), (512, 4, F16), (512, 8, BF16)]


# ---- outputs over inputs ----

@pytest.mark.parametrize("many", [True, False])
@pytest.mark.parametrize("dim,bits", [(64, 8), (128, 4), (256, 8), (512, 8), (512, 4)])
@pytest.mark.parametrize("rows,contexts", [([5] * 200, [40] * 200), ([48] * 40, [20] * 40), ([90], [1500])])
def test_attention_in_place(tf_ctx, workspaces, many, dim, bits, rows, contexts):
    case = _by(Case(60 + dim, rows, contexts, 2, dim, bits, 32, DEV), 16, many).upload()
    q = _q(case, 16, F16)
    beside = _run(tf_ctx, workspaces, case, q, F16)
    over = q.to(DEV)
    _ops(tf_ctx)[2].encode(over, over, case.cache, case.batch(), workspaces(dim), scale=dim ** -0.5)
    assert tf_ctx.device_status() == 0
    want, tol = ref.attention(case, q, _all_visible(case), dim ** -0.5, half_step(F16))
    _close(over, want, tol)
    _close(beside, want, tol)
    if not (many and dim == 512):                               # those have units of eight rows in place
        assert torch.equal(over, beside)
