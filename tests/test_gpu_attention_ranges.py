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


# ---- values ----

@pytest.mark.parametrize("many", [True, False])
@pytest.mark.parametrize("dim,bits,dtype", KINDS)
@pytest.mark.parametrize("rows,contexts", SHAPES)
@pytest.mark.parametrize("zeros", [64, 128, 300, 10 ** 6])
def test_tokens_whose_value_planes_are_zero(tf_ctx, workspaces, many, dim, bits, dtype, rows, contexts, zeros):
    """The first tokens of every sequence, or all of them, have value planes of zeros, as an empty cache has them."""
    case = Case(70 + dim + zeros, rows, contexts, 2, dim, bits, 32, DEV)
    for b, (n, c) in enumerate(zip(rows, contexts)):
        t = torch.arange(min(zeros, n + c))
        for i in (4, 5):
            case.planes[i][case.table[b, t // 32].long(), :, t % 32] = 0.0
    _by(case, 16, many).upload()
    q = _q(case, 16, dtype)
    got = _run(tf_ctx, workspaces, case, q, dtype)
    _close(got, *ref.attention(case, q, _all_visible(case), dim ** -0.5, half_step(dtype)))


@pytest.mark.parametrize("many", [True, False])
@pytest.mark.parametrize("dim,bits", [(64, 8), (128, 4), (256, 8), (512, 4)])
@pytest.mark.parametrize("rows,contexts", SHAPES)
@pytest.mark.parametrize("value_scale", [1e-37, 1e-35, 1e-20, 1e-6, 1e4, 1e30])
def test_values_of_any_size(tf_ctx, workspaces, many, dim, bits, rows, contexts, value_scale):
    case = _by(Case(80 + dim, rows, contexts, 2, dim, bits, 16, DEV, value_scale=value_scale), 16, many).upload()
    q = _q(case, 16, BF16)
    got = _run(tf_ctx, workspaces, case, q, BF16)
    # The statement for values of size one, times the power of two that they are apart (planes times a power are exact, the sums linear in them; the
    # tolerance's absolute share of 1e-7 goes by the values' size then, and 64 bits do not lose small ones beside it), and half of bf16's least step.
    power = round(-np.log2(value_scale))
    for i in (4, 5):
        case.planes[i] = torch.ldexp(case.planes[i].float(), torch.tensor(power)).bfloat16()
    want, tol = ref.attention(case, q, _all_visible(case), dim ** -0.5, half_step(BF16))
    _close(got, want * 2.0 ** -power, tol * 2.0 ** -power + 2.0 ** -134)


@pytest.mark.parametrize("many", [True, False])
@pytest.mark.parametrize("dim,bits", [(64, 8), (128, 4), (256, 8), (512, 4)])
@pytest.mark.parametrize("power", [30, 60])
@pytest.mark.parametrize("steps", [1, 9])
@pytest.mark.parametrize("rows,contexts", SHAPES)
def test_large_values_without_weight_take_no_precision(tf_ctx, workspaces, many, dim, bits, power, steps, rows, contexts):
    """The first tokens have values 2^30 or 2^60 times the others' and logits 200 lower, in one step or in several on the way to the others':
    their part of the output is below 2^-200, and the others keep their precision."""
    case = Case(90 + dim, rows, contexts, 2, dim, bits, 32, DEV)
    heavy = min(contexts) // 2 // steps * steps
    for b, c in enumerate(contexts):
        t = torch.arange(heavy)
        where = case.table[b, t // 32].long(), slice(None), t % 32
        # q is 4 on average: a key of -x moves the logit by 4 x sqrt(dim); the last of the heavy tokens still lie 200 below the others
        lower = (200 + 30.0 * (steps - 1 - t // (heavy // steps))) / (4 * dim ** 0.5)
        k = -lower[:, None, None] + 0.02 * torch.randn(heavy, 2, dim, generator=case.gen)
        for plane, new in zip(case.planes[:3], ref.quantised(k, bits)):
            plane[where] = new
        for i in (4, 5):
            case.planes[i][where] *= 2.0 ** power
    _by(case, 16, many).upload()
    q = (torch.randn(case.offsets[-1], 16 * dim, generator=case.gen) * 0.3 + 4).to(BF16)
    got = _run(tf_ctx, workspaces, case, q, BF16)
    for b in range(len(rows)):
        t = torch.arange(heavy)
        for i in (4, 5):
            case.planes[i][case.table[b, t // 32].long(), :, t % 32] = 0.0
    _close(got, *ref.attention(case, q, _all_visible(case), dim ** -0.5, half_step(BF16)))


@pytest.mark.parametrize("many", [True, False])
@pytest.mark.parametrize("dim,bits", [(64, 8), (128, 4), (256, 8), (512, 4)])
@pytest.mark.parametrize("size,tail", [(0.0021, 0.0014), (0.0002, 0.0003), (0.0085, 0.006), (0.07, 0.045), (0.55, 0.4), (90.0, 150.0), (150.0, 90.0), (17000.0, 12000.0)])
def test_long_tails_beside_a_token_of_another_size(tf_ctx, workspaces, many, dim, bits, size, tail):
    """One token has half of the weight, thousands share the other half, and a power of two that the values are divided by lies between their sizes:
    each of the thousands' parts is far below the one's, their sum is not."""
    rows, contexts = [40, 40], [4000, 3000]
    case = Case(150 + dim, rows, contexts, 2, dim, bits, 64, DEV)
    for b, (n, c) in enumerate(zip(rows, contexts)):
        t = torch.arange(n + c)
        where = case.table[b, t // 64].long(), slice(None), t % 64
        # q is 1 on average: the first key moves the logit by log(c)
        k = 0.02 * torch.randn(n + c, 2, dim, generator=case.gen)
        k[0] += np.log(c) / dim ** 0.5
        # a group's least and largest values, and so its size, are those asked for
        v = torch.rand(n + c, 2, dim // 64, 64, generator=case.gen) * 1.5 - 0.25
        v[..., 0], v[..., 1] = -1.0, 1.25
        v = v.flatten(-2) * tail
        v[0] *= size / tail
        for plane, new in zip(case.planes, (*ref.quantised(k, bits), *ref.quantised(v, bits))):
            plane[where] = new
    _by(case, 16, many).upload()
    q = (torch.randn(case.offsets[-1], 16 * dim, generator=case.gen) * 0.1 + 1).to(BF16)
    got = _run(tf_ctx, workspaces, case, q, BF16)
    power = round(-np.log2(tail))                                # the tolerance's absolute share goes by the values' size
    for i in (4, 5):
        case.planes[i] = torch.ldexp(case.planes[i].float(), torch.tensor(power)).bfloat16()
    want, tol = ref.attention(case, q, _all_visible(case), dim ** -0.5, half_step(BF16))
    _close(got, want * 2.0 ** -power, tol * 2.0 ** -power)


@pytest.mark.parametrize("many", [True, False])
@pytest.mark.parametrize("dim,bits", [(64, 8), (64, 4), (128, 4), (256, 8), (512, 4)])
@pytest.mark.parametrize("which", ["keys", "values"])
def test_narrow_groups_around_a_small_offset(tf_ctx, workspaces, many, dim, bits, which):
    """Biases just above 2^-9 and scales far below fp16's normal numbers, halfway between two of its subnormal ones."""
    rows, contexts = [40, 24], [300, 700]
    case = Case(100 + dim, rows, contexts, 2, dim, bits, 32, DEV)
    first, top = 3 * (which == "values"), 2 ** bits - 1
    owned = ~torch.isnan(case.planes[1])
    unit = 2.0 ** -24 if bits == 8 else 2.0 ** -20
    steps = torch.randint(0, 2 if which == "keys" else 1, case.planes[1].shape, generator=case.gen) + 1.5      # keys: a common shift would move no output
    case.planes[first + 1] = torch.where(owned, (steps * unit).bfloat16(), case.planes[first + 1])
    case.planes[first + 2][owned] = 2.0 ** -9 * 1.0078125
    codes = torch.randint(top - top // 8, top + 1, (*case.planes[0].shape[:3], dim), generator=case.gen).to(torch.uint8)
    case.planes[first] = codes if bits == 8 else codes[..., 0::2] | codes[..., 1::2] << 4
    _by(case, 16, many).upload()
    # as keys: a query of large elements of one sign, so that the logits' part from the scales counts
    q = _q(case, 16, F16, scale=300.0) + 2000 if which == "keys" else _q(case, 16, F16)
    got = _run(tf_ctx, workspaces, case, q, F16)
    see = _all_visible(case)
    want, tol = ref.attention(case, q, see, dim ** -0.5, half_step(F16))
    if which == "keys" and many:
        # There a key is rounded to fp16 once, by 2^-11 of it at most, and here the elements of a token, whose codes are nearly alike, with one sign: logits move by
        # up to d = 2^-11 sum |q k| scale, probabilities by p (d_j - mean of d) <= 2 d p, outputs by 2 d sum p |v|. (The bound for signs of their own is in `tol`.)
        moved = []
        for b, n in enumerate(rows):
            k, v = (c * s + o for c, s, o in (case.stored(b, 0), case.stored(b, 3)))
            qb = q[case.offsets[b]:case.offsets[b + 1]].to(F64).reshape(n, case.kv, -1, dim)
            x = torch.einsum("nhgd,jhd->hgnj", qb, k) * dim ** -0.5
            size = (torch.einsum("nhgd,jhd->hgnj", qb.abs(), k.abs()) * dim ** -0.5).masked_fill(~see[b], 0.0).amax(-1).permute(2, 0, 1)[..., None]
            p = x.masked_fill(~see[b], -float("inf")).softmax(-1)
            moved.append((2 * 2.0 ** -11 * size * torch.einsum("hgnj,jhd->nhgd", p, v.abs())).reshape(n, -1))
        tol = tol + torch.cat(moved)
    _close(got, want, tol)


# ---- queries ----

@pytest.mark.parametrize("many", [True, False])
@pytest.mark.parametrize("dim,bits", [(64, 4), (128, 8), (256, 8), (512, 4)])
@pytest.mark.parametrize("q_scale", [1e-36, 1e-20, 3e-5, 1e20, 1e36])
def test_queries_of_any_size(tf_ctx, workspaces, many, dim, bits, q_scale):
    rows, contexts = [40, 24], [300, 700]
    case = _by(Case(110 + dim, rows, contexts, 2, dim, bits, 16, DEV), 16, many).upload()
    q = _q(case, 16, BF16, scale=q_scale)
    got = _run(tf_ctx, workspaces, case, q, BF16, scale=0.1 / q_scale)
    _close(got, *ref.attention(case, q, _all_visible(case), 0.1 / q_scale, half_step(BF16)))


# ---- heads of 512, unlike sequences ----

@pytest.mark.parametrize("many", [True, False])
@pytest.mark.parametrize("dim,bits,dtype", [(512, 8, F16), (512, 4, BF16), (64, 8, BF16)])
@pytest.mark.parametrize("window", [0, 50])
def test_trees_of_many_rows(tf_ctx, workspaces, many, dim, bits, dtype, window):
    rows, contexts = [61, 1, 64, 130], [100, 0, 333, 40]
    case = _by(Case(120, rows, contexts, 2, dim, bits, 64, DEV), 16, many).upload()
    rng = np.random.default_rng(8)
    trees = [_tree(n, rng) for n in rows]
    masks, depths = [s for seen, _ in trees for s in seen], [depth for _, depth in trees]
    positions = [c + d for c, depth in zip(contexts, depths) for d in depth]
    q = _q(case, 16, dtype)
    got = _run(tf_ctx, workspaces, case, q, dtype, window=window, masks=masks, positions=positions, words=3)
    see = [ref.visible(n, c, window, seen, [c + d for d in depth]) for n, c, (seen, depth) in zip(rows, contexts, trees)]
    _close(got, *ref.attention(case, q, see, dim ** -0.5, half_step(dtype)))


@pytest.mark.parametrize("singles,chunk", [(64, 300), (20, 300), (3, 1000)])
@pytest.mark.parametrize("dim,bits", [(128, 8), (512, 4)])
@pytest.mark.parametrize("window", [0, 100])
def test_single_tokens_beside_a_prompt_chunk(tf_ctx, workspaces, singles, chunk, dim, bits, window):
    rows, contexts = [1] * singles + [chunk] + [1], [17 * i for i in range(singles)] + [500, 900]
    case = Case(130, rows, contexts, 2, dim, bits, 32, DEV).upload()
    q = _q(case, 4, F16)
    got = _run(tf_ctx, workspaces, case, q, F16, window=window)
    _close(got, *ref.attention(case, q, _all_visible(case, window), dim ** -0.5, half_step(F16)))


@pytest.mark.parametrize("many", [True, False])
@pytest.mark.parametrize("dim,bits", [(64, 8), (128, 4), (256, 8), (512, 8), (512, 4)])
@pytest.mark.parametrize("planes", [(1,), (2,), (4,), (5,), (4, 5), (1, 2, 4, 5)])
def test_planes_of_the_largest_numbers_reach_only_the_rows_that_see_them(tf_ctx, workspaces, many, dim, bits, planes):
    """Tokens before the window in a tile with tokens inside, and drafted tokens that no row sees, with planes of 3e38, whose values leave fp32."""
    rows, contexts, window = [40, 24], [930, 407], 100
    case = Case(170 + dim, rows, contexts, 2, dim, bits, 16, DEV)
    masks = [{j for j in range(i + 1) if j != 3} for n in rows for i in range(n)]
    for b, (n, c) in enumerate(zip(rows, contexts)):
        t = torch.tensor([*range(c - window), c + 3])
        for i in planes:
            case.planes[i][case.table[b, t // 16].long(), :, t % 16, 0] = 3e38 if i % 3 == 1 else -3e38
    _by(case, 16, many).upload()
    q = _q(case, 16, F16)
    positions = [c + i for n, c in zip(rows, contexts) for i in range(n)]
    got = _run(tf_ctx, workspaces, case, q, F16, window=window, masks=masks, positions=positions)
    for b, (n, c) in enumerate(zip(rows, contexts)):
        t = torch.tensor([*range(c - window), c + 3])
        for i in planes:
            case.planes[i][case.table[b, t // 16].long(), :, t % 16, 0] = 0.0
    see = [ref.visible(n, c, window, masks[o:o + n], positions[o:o + n]) for n, c, o in zip(rows, contexts, case.offsets)]
    _close(got, *ref.attention(case, q, see, dim ** -0.5, half_step(F16)))


# ---- pages ----

@pytest.mark.parametrize("many", [True, False])
@pytest.mark.parametrize("dim,bits", [(64, 8), (128, 4), (256, 8), (512, 4)])
@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("gone", [-1, 10 ** 6])
def test_pages_that_fell_out_of_every_window(tf_ctx, workspaces, many, dim, bits, tree, gone):
    """The table names no page at tokens that no row sees: nothing is wrong with such a call."""
    rows, contexts, window = [40, 24], [930, 407], 100
    case = Case(160 + dim, rows, contexts, 2, dim, bits, 16, DEV)
    full = case.table.clone()
    for b, c in enumerate(contexts):
        case.table[b, :(c - window + 1) // 16] = gone
    _by(case, 16, many).upload()
    rng = np.random.default_rng(9)
    trees = [_tree(n, rng) for n in rows]
    masks, positions = [s for seen, _ in trees for s in seen], [c + d for c, (_, depth) in zip(contexts, trees) for d in depth]
    q = _q(case, 16, F16)
    got = _run(tf_ctx, workspaces, case, q, F16, window=window, masks=masks if tree else None, positions=positions if tree else None)
    case.table = full
    see = [ref.visible(n, c, window, *((seen, [c + d for d in depth]) if tree else ())) for n, c, (seen, depth) in zip(rows, contexts, trees)]
    _close(got, *ref.attention(case, q, see, dim ** -0.5, half_step(F16)))


# ---- cache write ----

@pytest.mark.parametrize("rows", [3, 900])                       # a warp per head; a warp per eight heads
@pytest.mark.parametrize("dim,bits", [(64, 8), (128, 4), (256, 8), (512, 4)])
@pytest.mark.parametrize("size", [1e-38, 3e-37, 1e-36, 1e-30, 1e30, 3e37])
def test_epilogue_of_values_of_any_size(tf_ctx, rows, dim, bits, size):
    """v without a norm: scales down to the least one, 2^-126. Codes are those of the stored planes but next to a tie."""
    case = Case(140 + dim, [rows], [5], 2, dim, bits, 16, DEV).upload()
    x = torch.randn(rows, 4 * dim, generator=case.gen)
    x[:, 2 * dim:] *= size
    x[0, 2 * dim:2 * dim + 64] = size                            # equal values: scale 1
    x = x.to(BF16)
    dev, v_out = x.to(DEV), torch.zeros(rows, 2 * dim, dtype=BF16, device=DEV)
    _ops(tf_ctx)[0].encode(dev[:, :dim], dev[:, :2 * dim], dev[:, 2 * dim:], torch.zeros(rows, dim, dtype=BF16, device=DEV), case.batch(), case.cache, head_dim=dim, v_out=v_out)
    assert tf_ctx.device_status() == 0
    assert torch.equal(v_out.cpu(), x[:, 2 * dim:])
    token = 5 + torch.arange(rows)
    code, s, o = (p.cpu()[case.table[0, token // 16].long(), :, token % 16] for p in case.cache.planes[3:])
    top, g = 2 ** bits - 1, x[:, 2 * dim:].to(F64).reshape(rows, 2, -1, 64)
    low, high = g.amin(-1), g.amax(-1)
    step = torch.where(high == low, torch.ones_like(low), (high - low) / top)
    s, o = s.to(F64), o.to(F64)
    # half a step of bf16 from the quotient that fp32 has, which is off by 2^-23 at the most
    assert ((s - step.clamp(min=2.0 ** -126)).abs() <= (2.0 ** -8 + 2.0 ** -22) * step).all() and torch.equal(o, low)
    exact = ((g - o[..., None]) / s[..., None] + 0.5).clamp(0.25, top + 0.75)
    c = ref.unpack(code, bits).unflatten(-1, (-1, 64))
    near = (exact - exact.round()).abs() <= 1e-4
    assert ((c == exact.floor()) | (near & ((c - exact.floor()).abs() <= 1))).all()


@pytest.mark.parametrize("rows", [4, 900])
@pytest.mark.parametrize("dim,turning", [(64, 8), (256, 32), (512, 64), (128, 1)])
def test_pairs_half_a_head_apart_of_which_the_first_turn(tf_ctx, rows, dim, turning):
    """Frequencies of half a head with zeros behind those that turn: element j is paired with j + dim / 2, the rest stays as it is."""
    gen = torch.Generator().manual_seed(dim)
    x, position = torch.randn(rows, 3 * dim, generator=gen).to(F16), torch.arange(rows, dtype=torch.int32) * 37
    freqs = torch.zeros(dim // 2)
    freqs[:turning] = 1e4 ** (-torch.arange(turning) / turning)
    from turbo_fieldfare_b200 import attention as at
    i32 = dict(dtype=torch.int32, device=DEV)
    batch = at.KVBatch(torch.zeros(1, **i32), torch.zeros(0, **i32), torch.zeros(0, 1, **i32), position.to(DEV))
    dev, out = x.to(DEV), [torch.zeros(rows, dim, dtype=F16, device=DEV) for _ in range(3)]
    _ops(tf_ctx)[0].encode(dev[:, :dim], dev[:, dim:2 * dim], dev[:, 2 * dim:], out[0], batch, head_dim=dim, frequencies=freqs.to(DEV), k_out=out[1], v_out=out[2])
    for i in range(2):
        y = x[:, dim * i:dim * i + dim].to(F64)
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + 1e-6)
        size, angle = y.abs(), position.to(F64)[:, None] * freqs[:turning].to(F64)
        a, b = y[:, :turning].clone(), y[:, dim // 2:dim // 2 + turning].clone()
        y[:, :turning], y[:, dim // 2:dim // 2 + turning] = a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin()
        size[:, :turning] = size[:, dim // 2:dim // 2 + turning] = a.abs() + b.abs()
        _close(out[i], y, half_step(F16) * y.abs() + 2.0 ** -19 * size + 1e-7)
    assert torch.equal(out[2].cpu(), x[:, 2 * dim:])


# ---- calls ----

def test_batches_without_rows(tf_ctx):
    from turbo_fieldfare_b200 import attention as at
    cache = at.KVCache.allocate(3, 16, 2, 64, 8, device=DEV)
    i32 = dict(dtype=torch.int32, device=DEV)
    batch = at.KVBatch(torch.zeros(2, **i32), torch.full((1,), 4, **i32), torch.zeros(1, 3, **i32), torch.zeros(0, **i32))
    q, k = (torch.empty(0, n * 64, dtype=torch.float16, device=DEV) for n in (4, 2))
    at.FusedQKVEpilogue(tf_ctx).encode(q, k, k, torch.empty_like(q), batch, cache, head_dim=64, frequencies=torch.ones(32, device=DEV))
    at.FusedQKVEpilogue(tf_ctx).encode(q, k, k, q, batch, head_dim=64, k_out=torch.empty_like(k), v_out=torch.empty_like(k))
    at.KVCacheRead(tf_ctx).encode(cache, batch, torch.empty_like(k))
    for mask in (None, torch.zeros(0, 1, dtype=torch.int64, device=DEV)):
        at.TreeAttention(tf_ctx).encode(q, torch.empty_like(q), cache, batch, at.AttentionWorkspace(tf_ctx, 64), scale=1.0, window=5, tree_mask=mask)
    assert tf_ctx.device_status() == 0
