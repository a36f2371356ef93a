"""Attention operators through the C ABI against plain 64-bit statements: cache write with head norms and rotation, cache read, tree attention."""
import numpy as np
import pytest
import torch

import attention_reference as ref
from attention_reference import Case, F64, half_step

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F16, BF16 = torch.float16, torch.bfloat16


@pytest.fixture(params=[0, 70], autouse=True)
def crowd(request, monkeypatch):
    """Each test also with sequences that have no rows: few rows in a mean sequence go by units of eight, many by units of 128."""
    monkeypatch.setattr(Case, "crowd", request.param)


def _ops(ctx):
    from turbo_fieldfare_b200 import attention as at
    return at.FusedQKVEpilogue(ctx), at.KVCacheRead(ctx), at.TreeAttention(ctx)


@pytest.fixture(scope="module")
def workspaces(tf_ctx):
    from turbo_fieldfare_b200 import attention as at
    made = {}

    def get(dim):
        if dim not in made:
            made[dim] = at.AttentionWorkspace(tf_ctx, dim)
        return made[dim]
    return get


def _q(case, heads, dtype, scale=1.5):
    n = case.offsets[-1]
    return (torch.randn(n, heads * case.dim, generator=case.gen) * scale).to(dtype)


def _words(masks, words=1):
    out = np.zeros((len(masks), words), dtype=np.uint64)
    for r, seen in enumerate(masks):
        for j in seen:
            out[r, j // 64] |= np.uint64(1) << np.uint64(j % 64)
    return torch.from_numpy(out.view(np.int64)).to(DEV)


def _tree(rows, rng):
    """Ancestor sets and depths: token i hangs under a random earlier one."""
    seen, depth = [], []
    for i in range(rows):
        p = int(rng.integers(0, i)) if i else -1
        seen.append((seen[p] if i else set()) | {i})
        depth.append(depth[p] + 1 if i else 0)
    return seen, depth


def _run(ctx, workspaces, case, q, dtype, window=0, masks=None, positions=None, words=1, scale=None, rows=None, out=None):
    out = torch.full((q.shape[0], q.shape[1]), 7.0, dtype=dtype, device=DEV) if out is None else out
    scale = case.dim ** -0.5 if scale is None else scale
    _ops(ctx)[2].encode(q.to(DEV), out, case.cache, case.batch(positions, rows=rows), workspaces(case.dim), scale=scale, window=window,
                        tree_mask=None if masks is None else _words(masks, words))
    assert ctx.device_status() == 0
    return out


def _close(got, want, tol):
    got = got.cpu().to(F64)
    assert torch.isfinite(got).all()
    off = (got - want).abs()
    assert (off <= tol).all(), f"worst {(off / tol).max().item():.3f} of the tolerance at {(off / tol).argmax().item()}"


# ---- attention ----

@pytest.mark.parametrize("dim,bits", [(64, 8), (64, 4), (128, 8), (128, 4), (256, 8), (256, 4), (512, 8), (512, 4)])
@pytest.mark.parametrize("rows,contexts,heads,kv,dtype", [
    ([1], [0], 2, 2, F16),                                        # the row sees itself alone
    ([1, 1, 1], [5, 200, 63], 4, 2, BF16),
    ([3, 0, 2, 1], [64, 10, 0, 129], 6, 1, F16),                  # a sequence without rows, one without context
    ([17, 40], [70, 33], 8, 2, BF16),                             # units of 64 rows
])
def test_chain(tf_ctx, workspaces, dim, bits, rows, contexts, heads, kv, dtype):
    case = Case(dim + bits, rows, contexts, kv, dim, bits, 32, DEV).upload()
    q = _q(case, heads, dtype)
    got = _run(tf_ctx, workspaces, case, q, dtype)
    see = [ref.visible(n, c) for n, c in zip(rows, contexts)]
    _close(got, *ref.attention(case, q, see, dim ** -0.5, half_step(dtype)))


@pytest.mark.parametrize("page", [16, 64, 256])
@pytest.mark.parametrize("heads,kv", [(5, 1), (12, 4), (16, 2)])
@pytest.mark.parametrize("rows,contexts", [([1, 1], [700, 15]), ([9, 30, 1], [300, 64, 1000])])
def test_pages_and_groups(tf_ctx, workspaces, page, heads, kv, rows, contexts):
    case = Case(page + heads, rows, contexts, kv, 128, 8, page, DEV).upload()
    q = _q(case, heads, F16)
    got = _run(tf_ctx, workspaces, case, q, F16)
    _close(got, *ref.attention(case, q, [ref.visible(n, c) for n, c in zip(rows, contexts)], 128 ** -0.5, half_step(F16)))


@pytest.mark.parametrize("window", [1, 7, 64, 100, 5000])
@pytest.mark.parametrize("rows,contexts", [([1, 1, 1], [0, 99, 640]), ([20, 3], [130, 400])])
def test_window_of_a_chain(tf_ctx, workspaces, window, rows, contexts):
    case = Case(window, rows, contexts, 2, 64, 8, 16, DEV).upload()
    q = _q(case, 6, BF16)
    got = _run(tf_ctx, workspaces, case, q, BF16, window=window)
    _close(got, *ref.attention(case, q, [ref.visible(n, c, window) for n, c in zip(rows, contexts)], 64 ** -0.5, half_step(BF16)))


@pytest.mark.parametrize("bits,dim", [(8, 256), (4, 128)])
@pytest.mark.parametrize("window", [0, 50])
@pytest.mark.parametrize("rows", [[1, 2, 7], [61, 64, 13]])
def test_tree(tf_ctx, workspaces, bits, dim, window, rows):
    contexts = [100, 0, 333]
    case = Case(dim + len(rows), rows, contexts, 2, dim, bits, 64, DEV).upload()
    rng = np.random.default_rng(5)
    trees = [_tree(n, rng) for n in rows]
    positions = [c + d for c, (_, depth) in zip(contexts, trees) for d in depth]
    q = _q(case, 4, F16)
    masks = [s for seen, _ in trees for s in seen]
    got = _run(tf_ctx, workspaces, case, q, F16, window=window, masks=masks, positions=positions)
    see = [ref.visible(n, c, window, seen, [c + d for d in depth]) for n, c, (seen, depth) in zip(rows, contexts, trees)]
    _close(got, *ref.attention(case, q, see, dim ** -0.5, half_step(F16)))


def test_tree_of_more_rows_than_a_mask_word(tf_ctx, workspaces):
    rows, contexts = [150, 70], [40, 0]
    case = Case(3, rows, contexts, 1, 64, 8, 16, DEV).upload()
    rng = np.random.default_rng(6)
    trees = [_tree(n, rng) for n in rows]
    q = _q(case, 3, F16)
    masks = [s for seen, _ in trees for s in seen]
    got = _run(tf_ctx, workspaces, case, q, F16, masks=masks, words=3)
    see = [ref.visible(n, c, 0, seen) for n, c, (seen, _) in zip(rows, contexts, trees)]
    _close(got, *ref.attention(case, q, see, 64 ** -0.5, half_step(F16)))
    # with one word nobody sees rows from 64 on
    cut = [{j for j in s if j < 64} for s in masks]
    got = _run(tf_ctx, workspaces, case, q, F16, masks=cut)
    see = [ref.visible(n, c, 0, cut[o:o + n]) for n, c, o in zip(rows, contexts, case.offsets)]
    _close(got, *ref.attention(case, q, see, 64 ** -0.5, half_step(F16)))


@pytest.mark.parametrize("rows", [[3, 2], [20, 30]])
def test_rows_that_see_nothing_are_zero_and_masked_values_reach_nobody(tf_ctx, workspaces, rows):
    contexts = [0, 30]
    case = Case(8, rows, contexts, 2, 128, 8, 16, DEV)
    # the last row of each sequence: infinite and NaN planes, seen by itself alone
    for b in range(2):
        t = rows[b] + contexts[b] - 1
        for i, bad in ((1, float("inf")), (2, float("nan")), (4, float("nan")), (5, -float("inf"))):
            case.planes[i][int(case.table[b, t // 16]), :, t % 16, 0] = bad
    case.upload()
    masks = [{j for j in range(i + 1)} for n in rows for i in range(n)]
    masks[1] = set()                                            # sequence 0 has no context: this row sees nothing
    q = _q(case, 4, F16)
    got = _run(tf_ctx, workspaces, case, q, F16, masks=masks)
    last = [case.offsets[1] - 1, case.offsets[2] - 1]
    see = [ref.visible(n, c, 0, masks[o:o + n]) for n, c, o in zip(rows, contexts, case.offsets)]
    clean = [r for r in range(case.offsets[-1]) if r not in last]
    # the expected values of the others, without the last token
    for b in range(2):
        t = rows[b] + contexts[b] - 1
        for i in (1, 2, 4, 5):
            case.planes[i][int(case.table[b, t // 16]), :, t % 16, 0] = 0.0
    want, tol = ref.attention(case, q, see, 128 ** -0.5, half_step(F16))
    _close(got[clean], want[clean], tol[clean])
    assert (got[1] == 0).all()
    assert torch.isnan(got[last]).all()                         # a logit that is not a number
    # values alone: only the group that is broken
    for b in range(2):
        t = rows[b] + contexts[b] - 1
        case.planes[4][int(case.table[b, t // 16]), :, t % 16, 0] = float("nan")
    case.upload()
    got = _run(tf_ctx, workspaces, case, q, F16, masks=masks)
    heads = got[last].unflatten(1, (4, 128))
    assert torch.isnan(heads[..., :64]).all() and torch.isfinite(heads[..., 64:]).all()
    _close(got[clean], want[clean], tol[clean])


@pytest.mark.parametrize("dim,bits", [(64, 8), (128, 4), (256, 8), (512, 4)])
@pytest.mark.parametrize("rows", [7, 40])
def test_a_token_that_is_not_finite_at_any_place_of_a_tile(tf_ctx, workspaces, dim, bits, rows):
    """A drafted token that no row sees, at every place of a tile of 16, with planes that are not finite, one at a time."""
    for place in range(16):
        context = 32 + place                                    # row 0 stands at `place` of its tile
        case = Case(50 + place, [rows], [context], 1, dim, bits, 16, DEV)
        for i, bad in ((1, float("nan")), (2, float("inf")), (4, float("inf")), (5, float("nan"))):
            plane = case.planes[i][int(case.table[0, context // 16]), :, context % 16]
            old = plane.clone()
            plane[:, -1] = bad
            case.upload()
            plane.copy_(old)
            masks = [{j for j in range(1, r + 1)} for r in range(rows)]
            q = _q(case, 2, F16)
            got = _run(tf_ctx, workspaces, case, q, F16, masks=masks)
            _close(got, *ref.attention(case, q, [ref.visible(rows, context, 0, masks)], dim ** -0.5, half_step(F16)))


@pytest.mark.parametrize("rows", [[4], [40]])
def test_large_values_reach_only_the_rows_that_see_them(tf_ctx, workspaces, rows):
    """A drafted token with values 10^5 times the others', seen by itself alone: the other rows keep their precision. The same for
    what stands in a page behind the sequence's last token."""
    case = Case(18, rows, [20], 1, 128, 8, 16, DEV)
    t = 20 + 1
    for i in (4, 5):
        case.planes[i][int(case.table[0, t // 16]), :, t % 16] *= 1e5
    last = 20 + rows[0]
    case.planes[4][int(case.table[0, last // 16]), :, last % 16:] = 3e38
    case.planes[5][int(case.table[0, last // 16]), :, last % 16:] = -3e38
    case.upload()
    masks = [{j for j in range(i + 1) if j != 1} for i in range(rows[0])]
    masks[1] = {0, 1}
    q = _q(case, 2, BF16)
    got = _run(tf_ctx, workspaces, case, q, BF16, masks=masks)
    see = [ref.visible(rows[0], 20, 0, masks)]
    want, tol = ref.attention(case, q, see, 128 ** -0.5, half_step(BF16))
    others = [r for r in range(rows[0]) if r != 1]
    _close(got[[1]], want[[1]], tol[[1]])
    # the tolerance's share for probabilities below fp16's least step goes by the largest value that is seen
    kept = Case.of_cache(case.cache, case.table, rows, [20])
    for i in (4, 5):
        kept.planes[i][int(case.table[0, t // 16]), :, t % 16] = 0.0
    want, tol = ref.attention(kept, q, see, 128 ** -0.5, half_step(BF16))
    _close(got[others], want[others], tol[others])


@pytest.mark.parametrize("value_scale", [1e-6, 1e4, 1e30])
def test_values_outside_of_fp16(tf_ctx, workspaces, value_scale):
    case = Case(9, [2, 1], [90, 300], 2, 64, 8, 16, DEV, value_scale=value_scale).upload()
    q = _q(case, 2, BF16)
    got = _run(tf_ctx, workspaces, case, q, BF16)
    want, tol = ref.attention(case, q, [ref.visible(2, 90), ref.visible(1, 300)], 64 ** -0.5, half_step(BF16))
    _close(got, want, tol - 1e-7 + 1e-7 * value_scale)


@pytest.mark.parametrize("q_scale", [1e-20, 3e-5, 1e20])
def test_queries_outside_of_fp16(tf_ctx, workspaces, q_scale):
    case = Case(10, [2, 1], [90, 300], 2, 64, 4, 16, DEV).upload()
    q = _q(case, 2, BF16, scale=q_scale)
    got = _run(tf_ctx, workspaces, case, q, BF16, scale=0.2 / q_scale)
    _close(got, *ref.attention(case, q, [ref.visible(2, 90), ref.visible(1, 300)], 0.2 / q_scale, half_step(BF16)))


@pytest.mark.parametrize("scale", [-0.09, 0.0])
@pytest.mark.parametrize("rows,contexts,dim,bits", [([1, 3], [300, 20], 128, 8), ([45, 2], [150, 700], 256, 4)])
def test_scales_that_are_not_positive(tf_ctx, workspaces, scale, rows, contexts, dim, bits):
    case = Case(14, rows, contexts, 2, dim, bits, 32, DEV).upload()
    q = _q(case, 4, F16)
    got = _run(tf_ctx, workspaces, case, q, F16, scale=scale, window=200)
    _close(got, *ref.attention(case, q, [ref.visible(n, c, 200) for n, c in zip(rows, contexts)], scale, half_step(F16)))


def test_peaked_logits(tf_ctx, workspaces):
    """Logits of hundreds: nearly all the weight on one token, and maxima that grow from tile to tile."""
    case = Case(11, [1, 5], [900, 500], 2, 256, 8, 64, DEV).upload()
    q = _q(case, 4, F16, scale=20.0)
    got = _run(tf_ctx, workspaces, case, q, F16)
    _close(got, *ref.attention(case, q, [ref.visible(1, 900), ref.visible(5, 500)], 256 ** -0.5, half_step(F16)))


def test_padded_batch_strides_and_in_place(tf_ctx, workspaces):
    case = Case(12, [1, 4, 1], [50, 20, 90], 2, 128, 8, 32, DEV).upload()
    q = _q(case, 6, F16)
    wide = torch.full((11, 6 * 128 + 24), 3.0, dtype=F16, device=DEV)
    wide[:6, :6 * 128] = q.to(DEV)
    view = wide[:, :6 * 128]
    want, tol = ref.attention(case, q, [ref.visible(n, c) for n, c in zip(case.rows, case.contexts)], 128 ** -0.5, half_step(F16))
    out = torch.full((11, 6 * 128), 7.0, dtype=F16, device=DEV)
    op = _ops(tf_ctx)[2]
    op.encode(view, out, case.cache, case.batch(rows=11), workspaces(128), scale=128 ** -0.5)
    assert tf_ctx.device_status() == 0
    _close(out[:6], want, tol)
    assert (out[6:] == 7).all()
    op.encode(view, view, case.cache, case.batch(rows=11), workspaces(128), scale=128 ** -0.5)
    assert torch.equal(view[:6], out[:6]) and (wide[6:] == 3).all() and (wide[:, 6 * 128:] == 3).all()


@pytest.mark.parametrize("rows,contexts", [([1], [30000]), ([40], [9000]), ([1] * 70, [257] * 70)])
def test_repeats_and_graphs_give_the_same_bits(tf_ctx, workspaces, rows, contexts):
    case = Case(13, rows, contexts, 2, 128, 8, 64, DEV).upload()
    q = _q(case, 8, F16).to(DEV)
    first = _run(tf_ctx, workspaces, case, q, F16)
    assert torch.equal(first, _run(tf_ctx, workspaces, case, q, F16))
    want, tol = ref.attention(case, q.cpu(), [ref.visible(n, c) for n, c in zip(rows, contexts)], 128 ** -0.5, half_step(F16))
    _close(first, want, tol)
    out, batch, op = torch.zeros_like(first), case.batch(), _ops(tf_ctx)[2]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        op.encode(q, out, case.cache, batch, workspaces(128), scale=128 ** -0.5, stream=torch.cuda.current_stream())
    # the lengths are read when the graph runs
    batch.context_lengths.fill_(17)
    graph.replay()
    torch.cuda.synchronize()
    short = out.clone()
    batch.context_lengths[:len(contexts)].copy_(torch.tensor(contexts, dtype=torch.int32))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, first) and not torch.equal(short, first)


def test_two_streams_with_a_workspace_each(tf_ctx, workspaces):
    from turbo_fieldfare_b200 import attention as at
    cases = [Case(20 + i, [1] * 3, [4000, 70, 900], 2, 128, 8, 64, DEV).upload() for i in range(2)]
    qs = [_q(c, 4, F16).to(DEV) for c in cases]
    alone = [_run(tf_ctx, workspaces, c, q, F16) for c, q in zip(cases, qs)]
    spaces, streams = [at.AttentionWorkspace(tf_ctx, 128) for _ in range(2)], [torch.cuda.Stream() for _ in range(2)]
    outs, batches, op = [torch.zeros_like(a) for a in alone], [c.batch() for c in cases], _ops(tf_ctx)[2]
    torch.cuda.synchronize()
    for _ in range(20):
        for i in range(2):
            op.encode(qs[i], outs[i], cases[i].cache, batches[i], spaces[i], scale=128 ** -0.5, stream=streams[i])
    torch.cuda.synchronize()
    assert all(torch.equal(o, a) for o, a in zip(outs, alone))


def test_pages_that_are_missing_are_left_out(tf_ctx, workspaces):
    from turbo_fieldfare_b200.kernels import TFError
    case = Case(14, [1, 2], [100, 40], 1, 64, 8, 16, DEV)
    see = [ref.visible(1, 100), ref.visible(2, 40)]
    full = case.table.clone()
    q = torch.randn(3, 2 * 64, generator=case.gen).to(F16)
    case.table[0, 2], case.table[0, 4] = -5, case.planes[0].shape[0]       # below and above the planes
    case.upload()
    out = torch.zeros(3, 2 * 64, dtype=F16, device=DEV)
    _ops(tf_ctx)[2].encode(q.to(DEV), out, case.cache, case.batch(), workspaces(64), scale=0.125)
    with pytest.raises(TFError, match="7f000051"):
        tf_ctx.device_status()
    assert tf_ctx.device_status() == 0
    case.table = full
    see[0][:, 32:48] = False
    see[0][:, 64:80] = False
    want, tol = ref.attention(case, q, see, 0.125, half_step(F16))
    _close(out, want, tol)
    # contexts beyond the table: the table's tokens are used
    _ops(tf_ctx)[2].encode(q.to(DEV), out, case.cache, case.batch(contexts=[2 ** 31 - 1, -3]), workspaces(64), scale=0.125)
    with pytest.raises(TFError, match="7f000051"):
        tf_ctx.device_status()
    assert torch.isfinite(out[1:]).all()


def test_offsets_that_descend_or_pass_the_rows(tf_ctx, workspaces):
    from turbo_fieldfare_b200 import attention as at
    from turbo_fieldfare_b200.kernels import TFError
    case = Case(15, [2, 2, 2], [30, 20, 10], 1, 64, 8, 16, DEV).upload()
    q = _q(case, 1, F16)
    i32 = dict(dtype=torch.int32, device=DEV)
    for offsets in ([0, 2, 1, 9], [-4, 2, 4, 6], [0, 100, 100, 100]):
        batch = at.KVBatch(torch.tensor(offsets, **i32), torch.tensor(case.contexts, **i32), case.table.to(DEV), rows=6)
        out = torch.full((8, 64), 5.0, dtype=F16, device=DEV)
        _ops(tf_ctx)[2].encode(q.to(DEV), out[:6], case.cache, batch, workspaces(64), scale=0.125)
        with pytest.raises(TFError):
            tf_ctx.device_status()
        assert (out[6:] == 5).all()


def test_planes_of_more_than_four_gigabytes(tf_ctx, workspaces):
    """Pages behind 2^32 bytes of codes and 2^31 elements of them."""
    small = Case(16, [1, 3], [200, 50], 8, 256, 8, 64, DEV)
    first = (1 << 32) // (8 * 64 * 256) + 5
    from turbo_fieldfare_b200 import attention as at
    big = []
    for p in small.planes:
        t = torch.empty(first + p.shape[0], *p.shape[1:], dtype=p.dtype, device=DEV)
        t[first:] = p.to(DEV)
        big.append(t)
    small.upload()
    small.cache = at.KVCache(*big)
    q = _q(small, 16, F16)
    i32 = dict(dtype=torch.int32, device=DEV)
    table = torch.where(small.table >= 0, small.table + first, small.table)
    batch = at.KVBatch(torch.tensor(small.offsets, **i32), torch.tensor(small.contexts, **i32), table.to(DEV), rows=4)
    out = torch.zeros(4, 16 * 256, dtype=F16, device=DEV)
    op = _ops(tf_ctx)
    op[2].encode(q.to(DEV), out, small.cache, batch, workspaces(256), scale=1 / 16)
    k = torch.zeros(4, 8 * 256, dtype=F16, device=DEV)
    op[1].encode(small.cache, batch, k)
    assert tf_ctx.device_status() == 0
    _close(out, *ref.attention(small, q, [ref.visible(1, 200), ref.visible(3, 50)], 1 / 16, half_step(F16)))
    for b, n in enumerate(small.rows):
        c, s, o = small.stored(b, 0)
        assert torch.equal(k[small.offsets[b]:small.offsets[b + 1]].cpu(), (c * s + o)[-n:].reshape(n, -1).float().to(F16))


# ---- cache write ----

def _definition(x, weight, eps, norm, freqs, position):
    """Norm and rotation of one tensor of heads [rows, heads, dim] in 64 bits."""
    y = x.to(F64)
    if norm:
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + eps)
        if weight is not None:
            y = y * weight.to(F64)
    size = y.abs()
    if freqs is not None and len(freqs):
        r = len(freqs)
        angle = position.to(F64)[:, None, None] * freqs.to(F64)
        a, b = y[..., :r].clone(), y[..., r:2 * r].clone()
        size[..., :r] = a.abs() + b.abs()
        size[..., r:2 * r] = size[..., :r]
        y[..., :r], y[..., r:2 * r] = a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin()
    return y, size


def _check_stored(case, rows_of, y, size, first):
    """Planes and codes of the rows against the definition: planes within a half step of bf16 (and fp32's error of the values), codes those of the
    stored planes but for values within fp32's error of a tie."""
    planes = [p.cpu() for p in case.cache.planes[first:first + 3]]
    for r, (b, token) in enumerate(rows_of):
        page, slot = int(case.table[b, token // case.page]), token % case.page
        code, s, o = (p[page, :, slot] for p in planes)
        code, s, o = ref.unpack(code, case.bits), s.to(F64), o.to(F64)
        g, err = y[r].unflatten(-1, (-1, 64)), 2.0 ** -19 * size[r].unflatten(-1, (-1, 64)).amax(-1)
        low, high = g.amin(-1), g.amax(-1)
        top = 2 ** case.bits - 1
        step = torch.where(high == low, torch.ones_like(low), (high - low) / top)
        assert ((s - step).abs() <= 2.0 ** -8 * step + 2 * err / top).all()
        assert ((o - low).abs() <= 2.0 ** -8 * low.abs() + err).all()
        exact = ((g - o[..., None]) / s[..., None] + 0.5).clamp(0.25, top + 0.75)
        c = code.unflatten(-1, (-1, 64))
        slack = (2 * err / s + 1e-4)[..., None]
        near = (exact - exact.round()).abs() <= slack
        assert ((c == exact.floor()) | (near & ((c - exact.floor()).abs() <= 1))).all()


@pytest.mark.parametrize("dim,pairs", [(64, 32), (64, 6), (128, 64), (128, 0), (256, 128), (256, 32), (512, 64), (512, 256)])
@pytest.mark.parametrize("bits,dtype,rows,contexts", [(8, F16, [1], [0]), (4, BF16, [3, 1, 0, 5], [70, 900000, 3, 12]), (8, BF16, [90, 70], [1, 33]),
                                                       (8, F16, [900, 0, 701, 33], [5, 2, 40, 64]), (4, BF16, [7] * 90, list(range(90)))])
def test_epilogue_writes_the_cache(tf_ctx, dim, pairs, bits, dtype, rows, contexts):
    heads, kv = 6, 2
    case = Case(dim + pairs, rows, [min(c, 100) for c in contexts], kv, dim, bits, 16, DEV).upload()
    n = case.offsets[-1]
    qkv = (torch.randn(n, (heads + 2 * kv) * dim, generator=case.gen) * torch.rand(n, 1, generator=case.gen) * 3).to(dtype)
    wq, wk = (1 + 0.2 * torch.randn(2, dim, generator=case.gen)).bfloat16()
    freqs = (1e6 ** (-torch.arange(pairs, dtype=F64) / max(pairs, 1))).float()
    position = torch.tensor([c + i for c, r in zip(contexts, rows) for i in range(r)], dtype=torch.int32)
    before = [p.clone() for p in case.cache.planes]
    packed = qkv.to(DEV)
    q_out = torch.zeros(n, heads * dim, dtype=dtype, device=DEV)
    k_out, v_out = torch.zeros(n, kv * dim, dtype=dtype, device=DEV), torch.zeros(n, kv * dim, dtype=dtype, device=DEV)
    hq, hk = heads * dim, kv * dim
    _ops(tf_ctx)[0].encode(packed[:, :hq], packed[:, hq:hq + hk], packed[:, hq + hk:], q_out, case.batch(position), case.cache, head_dim=dim,
                           q_weight=wq.to(DEV), k_weight=wk.to(DEV), norm_v=True, frequencies=freqs.to(DEV) if pairs else None, k_out=k_out, v_out=v_out)
    assert tf_ctx.device_status() == 0
    x = qkv.unflatten(-1, (-1, dim))
    parts = [(x[:, :heads], wq, freqs), (x[:, heads:heads + kv], wk, freqs), (x[:, heads + kv:], None, None)]
    rows_of = [(b, case.contexts[b] + i) for b, r in enumerate(rows) for i in range(r)]
    for i, ((part, w, f), out) in enumerate(zip(parts, (q_out, k_out, v_out))):
        y, size = _definition(part, w, 1e-6, True, f, position)
        _close(out, y.flatten(1), (half_step(dtype) * y.abs() + 2.0 ** -19 * size + 1e-7).flatten(1))
        if i:
            _check_stored(case, rows_of, y, size, 3 * (i - 1))
    # nothing else in the cache was written
    touched = torch.zeros(case.cache.num_pages, case.page, dtype=torch.bool)
    for b, token in rows_of:
        touched[int(case.table[b, token // case.page]), token % case.page] = True
    keep = ~touched.to(DEV)
    for old, new in zip(before, case.cache.planes):
        old, new = old.transpose(1, 2)[keep], new.transpose(1, 2)[keep]
        assert torch.equal(old.view(torch.uint8), new.view(torch.uint8))


def test_epilogue_without_cache_norms_weights_or_rotation(tf_ctx):
    from turbo_fieldfare_b200 import attention as at
    gen = torch.Generator().manual_seed(4)
    n, dim, heads, kv = 5, 128, 4, 2
    qkv = torch.randn(n, (heads + 2 * kv) * dim, generator=gen).to(F16)
    dev = qkv.to(DEV)
    q, k, v = dev[:, :512], dev[:, 512:768], dev[:, 768:]
    i32 = dict(dtype=torch.int32, device=DEV)
    batch = at.KVBatch(torch.zeros(1, **i32), torch.zeros(0, **i32), torch.zeros(0, 1, **i32), rows=n)
    k_out, v_out = torch.zeros(n, 256, dtype=F16, device=DEV), torch.zeros(n, 256, dtype=F16, device=DEV)
    _ops(tf_ctx)[0].encode(q, k, v, q, batch, head_dim=dim, k_out=k_out, v_out=v_out)           # q in place
    assert tf_ctx.device_status() == 0
    for part, out, norm in ((qkv[:, :512], q, True), (qkv[:, 512:768], k_out, True), (qkv[:, 768:], v_out, False)):
        y, size = _definition(part.unflatten(-1, (-1, dim)), None, 1e-6, norm, None, None)
        _close(out, y.flatten(1), (half_step(F16) * y.abs() + 2.0 ** -19 * size + 1e-7).flatten(1))
    assert torch.equal(v_out.cpu(), qkv[:, 768:])


def test_epilogue_padded_rows_equal_groups_and_values_that_are_not_finite(tf_ctx):
    case = Case(30, [2, 1], [20, 3], 2, 64, 8, 16, DEV).upload()
    n, rows = 3, 6
    x = torch.randn(rows, 4 * 64, generator=case.gen).to(BF16)
    x[0, 128:192] = 2.5                       # a group of equal values: scale 1, bias the value
    x[1, 192 + 5] = float("inf")
    x[2, 130] = float("nan")
    dev = x.to(DEV)
    q_out = torch.full((rows, 128), 9.0, dtype=BF16, device=DEV)
    k = dev[:, 128:]
    before = [p.clone() for p in case.cache.planes]
    op, read, _ = _ops(tf_ctx)
    op.encode(dev[:, :128], k, k, q_out, case.batch(rows=rows), case.cache, head_dim=64)          # v: the same rows as k, without norm
    k_out, v_out = (torch.full((rows, 128), 9.0, dtype=BF16, device=DEV) for _ in range(2))
    read.encode(case.cache, case.batch(rows=rows), k_out, v_out)
    assert tf_ctx.device_status() == 0
    assert (q_out[n:] == 9).all() and (k_out[n:] == 9).all() and (v_out[n:] == 9).all()
    assert (v_out[0, :64] == 2.5).all()
    assert torch.isnan(v_out[1, 64:]).all() and torch.isfinite(v_out[1, :64]).all()
    assert torch.isnan(v_out[2, :64]).all() and torch.isfinite(v_out[2, 64:]).all()
    assert torch.isnan(k_out[2, :64]).all() and torch.isfinite(k_out[2, 64:]).all()
    changed = sum(int((a.view(torch.uint8) != b.view(torch.uint8)).flatten(3).any(-1).any(1).sum()) > 0 for a, b in zip(before, case.cache.planes))
    assert changed == 6


@pytest.mark.parametrize("rows", [1, 2, 37, 1600])
@pytest.mark.parametrize("dim,heads,kv", [(64, 19, 11), (128, 1, 1), (256, 9, 3), (512, 17, 9)])
def test_epilogue_in_place(tf_ctx, rows, dim, heads, kv):
    """Numbers of heads that fill no block, every output over its own input: the same bits as beside it."""
    gen = torch.Generator().manual_seed(rows)
    case = Case(31, [rows], [3], kv, dim, 8, 16, DEV).upload()
    q, k, v = (torch.randn(rows, n * dim, generator=gen).to(F16).to(DEV) for n in (heads, kv, kv))
    w = (1 + 0.2 * torch.randn(dim, generator=gen)).bfloat16().to(DEV)
    freqs = (1e4 ** (-torch.arange(dim // 4, dtype=F64) / (dim // 4))).float().to(DEV)
    batch, op = case.batch(torch.arange(3, 3 + rows)), _ops(tf_ctx)[0]
    beside = [torch.zeros_like(t) for t in (q, k, v)]
    op.encode(q, k, v, beside[0], batch, case.cache, head_dim=dim, q_weight=w, k_weight=w, norm_v=True, frequencies=freqs, k_out=beside[1], v_out=beside[2])
    planes = [p.clone() for p in case.cache.planes]
    raw = q.cpu()
    op.encode(q, k, v, q, batch, case.cache, head_dim=dim, q_weight=w, k_weight=w, norm_v=True, frequencies=freqs, k_out=k, v_out=v)
    assert tf_ctx.device_status() == 0
    for a, b in zip((q, k, v), beside):
        assert torch.equal(a, b)
    for a, b in zip(case.cache.planes, planes):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    y, size = _definition(raw.unflatten(-1, (-1, dim)), w.cpu(), 1e-6, True, freqs.cpu(), torch.arange(3, 3 + rows))
    _close(q, y.flatten(1), (half_step(F16) * y.abs() + 2.0 ** -19 * size + 1e-7).flatten(1))


def test_epilogue_far_positions(tf_ctx):
    """Angles of positions of hundreds of millions, where 32 bits have lost the turn."""
    from turbo_fieldfare_b200 import attention as at
    gen = torch.Generator().manual_seed(5)
    position = torch.tensor([0, 1, 2 ** 24 + 1, 987654321, 2 ** 31 - 1, -17], dtype=torch.int32)
    n = len(position)
    x = torch.randn(n, 3 * 64, generator=gen).to(F16)
    freqs = torch.tensor([1.0, 0.7, 0.3, 1e-3] * 8).float()
    dev = x.to(DEV)
    i32 = dict(dtype=torch.int32, device=DEV)
    batch = at.KVBatch(torch.zeros(1, **i32), torch.zeros(0, **i32), torch.zeros(0, 1, **i32), position.to(DEV))
    out = [torch.zeros(n, 64, dtype=F16, device=DEV) for _ in range(3)]
    _ops(tf_ctx)[0].encode(dev[:, :64], dev[:, 64:128], dev[:, 128:], out[0], batch, head_dim=64, frequencies=freqs.to(DEV), k_out=out[1], v_out=out[2])
    for i in range(2):
        y, size = _definition(x[:, 64 * i:64 * i + 64].unflatten(-1, (1, 64)), None, 1e-6, True, freqs, position)
        # 2^31 turns lose 2^-53 * 2^31 of a turn: 1e-6 of the size
        _close(out[i], y.flatten(1), (half_step(F16) * y.abs() + (2.0 ** -19 + 2e-6) * size + 1e-7).flatten(1))


def test_rows_without_a_page_leave_the_cache_alone(tf_ctx):
    from turbo_fieldfare_b200.kernels import TFError
    case = Case(31, [3, 2], [30, 5], 1, 64, 8, 16, DEV).upload()
    case.table[0, 2] = 10 ** 6                                  # tokens 32 and on: beyond the planes
    x = torch.randn(5, 3 * 64, generator=case.gen).to(F16).to(DEV)
    before = [p.clone() for p in case.cache.planes]
    q_out = torch.zeros(5, 64, dtype=F16, device=DEV)
    op, read, _ = _ops(tf_ctx)
    op.encode(x[:, :64], x[:, 64:128], x[:, 128:], q_out, case.batch(contexts=[30, -1]), case.cache, head_dim=64)
    with pytest.raises(TFError, match="7f000051"):
        tf_ctx.device_status()
    assert (q_out.abs().sum(1) > 0).all()
    for i, (old, new) in enumerate(zip(before, case.cache.planes)):
        rows = (old.view(torch.uint8) != new.view(torch.uint8)).flatten(3).any(-1).any(1)      # [pages, slots]
        allowed = torch.zeros_like(rows)
        for token in (30, 31):
            allowed[int(case.table[0, token // 16]), token % 16] = True
        assert not (rows & ~allowed).any()
    out = torch.full((5, 64), 9.0, dtype=F16, device=DEV)
    read.encode(case.cache, case.batch(contexts=[30, -1]), out)
    with pytest.raises(TFError, match="7f000051"):
        tf_ctx.device_status()
    assert (out[2:] == 9).all() and torch.isfinite(out[:2]).all()


# ---- cache read ----

@pytest.mark.parametrize("dim,bits,page", [(64, 4, 16), (64, 8, 32), (128, 4, 64), (256, 8, 16), (512, 4, 128), (512, 8, 16)])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_read(tf_ctx, dim, bits, page, dtype):
    lens = [1, 0, 77, 130]
    case = Case(dim + page, lens, [0] * 4, 3, dim, bits, page, DEV).upload()
    n = case.offsets[-1]
    wide = torch.full((n + 2, 3 * dim + 8), 9.0, dtype=dtype, device=DEV)
    v = torch.full((n + 2, 3 * dim), 9.0, dtype=dtype, device=DEV)
    _ops(tf_ctx)[1].encode(case.cache, case.batch(rows=n + 2), wide[:, :3 * dim], v)
    assert tf_ctx.device_status() == 0
    for out, first in ((wide[:, :3 * dim], 0), (v, 3)):
        want = torch.cat([(c * s + o).flatten(1) for c, s, o in (case.stored(b, first) for b in range(4))])
        assert torch.equal(out[:n].cpu(), want.float().to(dtype))       # code * scale + bias is one fp32 rounding, exact in 64 bits
        assert (out[n:] == 9).all()
    assert (wide[:, 3 * dim:] == 9).all()


def test_empty_calls_do_nothing(tf_ctx, workspaces):
    case = Case(40, [1], [5], 1, 64, 8, 16, DEV).upload()
    from turbo_fieldfare_b200 import attention as at
    i32 = dict(dtype=torch.int32, device=DEV)
    nobody = at.KVBatch(torch.zeros(1, **i32), torch.zeros(0, **i32), torch.zeros(0, 3, **i32), rows=0)
    no_rows = at.KVBatch(torch.zeros(3, **i32), torch.full((2,), 4, **i32), torch.zeros(2, 3, **i32), rows=0)
    padded = at.KVBatch(torch.zeros(3, **i32), torch.full((2,), 4, **i32), torch.zeros(2, 3, **i32), rows=4)
    op, read, attend = _ops(tf_ctx)
    for batch in (nobody, no_rows, padded):
        x = torch.full((4, 64), 5.0, dtype=F16, device=DEV)
        out = x.clone()
        attend.encode(x, out, case.cache, batch, workspaces(64), scale=0.1)
        read.encode(case.cache, batch, out, out.clone())
        op.encode(x, x, x, out, batch, case.cache, head_dim=64)
        assert tf_ctx.device_status() == 0
        assert (out == 5).all()


# ---- the layer that uses them ----

def test_attention_section_of_a_layer(tf_ctx, oracle, workspaces):
    """Projection, norms with rotation and cache write, tree attention, output projection and the norms in front of the experts, step by step:
    two prompt chunks, a tree of drafted tokens and a single token, against the attention in 64 bits over what the cache then holds."""
    from helpers import config0_matrix, to_dev
    from turbo_fieldfare_b200 import attention as at
    from turbo_fieldfare_b200.kernels import FusedPostAttentionSetup, MPPPrefillInt4QMM
    d, heads, kv, dim, page = 256, 4, 2, 64, 16
    rng = np.random.default_rng(77)
    w_qkv, w_o = config0_matrix(oracle, (heads + 2 * kv) * dim, d, rng), config0_matrix(oracle, d, heads * dim, rng)
    dq, do = [to_dev(w_qkv.packed), to_dev(w_qkv.scales), to_dev(w_qkv.biases)], [to_dev(w_o.packed), to_dev(w_o.scales), to_dev(w_o.biases)]
    qmm, setup = MPPPrefillInt4QMM(tf_ctx), FusedPostAttentionSetup(tf_ctx)
    op, _, attend = _ops(tf_ctx)
    cache = at.KVCache.allocate(40, page, kv, dim, 8, device=DEV)
    table = torch.randperm(40, generator=torch.Generator().manual_seed(1))[:24].reshape(2, 12).int().to(DEV)
    weight = torch.ones(dim, dtype=BF16, device=DEV)
    freqs = (1e4 ** (-torch.arange(32, dtype=F64) / 32)).float().to(DEV)
    ones = torch.ones(d, dtype=BF16, device=DEV)
    i32 = dict(dtype=torch.int32, device=DEV)
    lengths = [0, 0]
    for rows, tree in (([37, 5], False), ([20, 64], False), ([9, 6], True), ([1, 1], False)):
        n = sum(rows)
        x = (torch.randn(n, d, generator=torch.Generator().manual_seed(n)) * 0.5).to(F16).to(DEV)
        qkv = torch.zeros(n, (heads + 2 * kv) * dim, dtype=F16, device=DEV)
        qmm.encode(*dq, x, qkv, n, (heads + 2 * kv) * dim, d)
        trees = [_tree(r, rng) for r in rows]
        position = [c + (depth[i] if tree else i) for c, r, (_, depth) in zip(lengths, rows, trees) for i in range(r)]
        batch = at.KVBatch(torch.tensor([0, rows[0], n], **i32), torch.tensor(lengths, **i32), table, torch.tensor(position, **i32))
        q_out, attn = (torch.zeros(n, heads * dim, dtype=F16, device=DEV) for _ in range(2))
        hq, hk = heads * dim, kv * dim
        op.encode(qkv[:, :hq], qkv[:, hq:hq + hk], qkv[:, hq + hk:], q_out, batch, cache, head_dim=dim, q_weight=weight, k_weight=weight, norm_v=True, frequencies=freqs)
        masks = [s for seen, _ in trees for s in seen] if tree else None
        attend.encode(q_out, attn, cache, batch, workspaces(dim), scale=dim ** -0.5, tree_mask=_words(masks) if tree else None)
        projected, hidden = torch.zeros(n, d, dtype=F16, device=DEV), x.clone()
        qmm.encode(*do, attn, projected, n, d, heads * dim)
        outs = [torch.zeros(n, d, dtype=F16, device=DEV) for _ in range(3)]
        setup.encode(hidden, projected, *outs, ones, ones, ones, d, rows=n)
        assert tf_ctx.device_status() == 0
        # the attention against the cache's own values
        case = Case.of_cache(cache, table, rows, lengths)
        see = [ref.visible(r, c, 0, seen if tree else None) for r, c, (seen, _) in zip(rows, lengths, trees)]
        _close(attn, *ref.attention(case, q_out.cpu(), see, dim ** -0.5, half_step(F16)))
        assert all(torch.isfinite(o).all() for o in outs)
        if not tree:
            lengths = [c + r for c, r in zip(lengths, rows)]
