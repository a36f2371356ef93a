"""Verifications with so many logits that the first launch sums them in 32 bits, against the plain statement in 64; logarithms of those that it sums in 64."""
import math

import numpy as np
import pytest
import torch

import drafts_reference as ref
from test_gpu_drafts import DEV, I32, TYPES, Draft, dev

pytestmark = pytest.mark.gpu

# Rows times logits up to here are summed in 64 bits by the first launch, of capped logits up to two thirds of it.
SUMMED_IN_64_BITS = 6_000_000


def wide(seed, counts, nodes, vocab, **more):
    d = Draft(seed, counts, nodes, vocab, **more)
    assert nodes > 1 and d.logits.shape[0] * vocab > SUMMED_IN_64_BITS
    return d


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("probs", [None, torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tree", [False, True])
def test_drafts_of_every_type(tf_ctx, dtype, probs, tree):
    """Rows of 21 parts that begin off every boundary, sequences of sixteen blocks."""
    d = wide(3 + tree, [9, 0, 7, 1, 9, 8], 9, 170003, dtype=dtype, probs=probs, tree=tree)
    d.compare(tf_ctx)
    d.compare(tf_ctx, cap=30.0, temperatures=[1.0, 0.7, 0.0, 1.3, 0.5, 2.0])
    assert tf_ctx.device_status() == 0


@pytest.mark.parametrize("counts,nodes,vocab,dtype,probs", [
    ([3, 2], 3, 1100003, torch.float16, torch.float16),            # steps of a warp in groups of several
    ([5, 4, 3, 5] * 10, 5, 40961, torch.bfloat16, torch.float32),  # four blocks a sequence
    ([4] * 150, 4, 40009, torch.float16, None),                    # several chunks a part, several parts a row, a block a sequence
    ([3, 1, 2, 0] * 90, 3, 12007, torch.float32, torch.bfloat16)])  # more sequences than blocks that are on the chip at once
def test_sizes(tf_ctx, counts, nodes, vocab, dtype, probs):
    d = wide(vocab, counts, nodes, vocab, dtype=dtype, probs=probs)
    n = len(counts)
    d.compare(tf_ctx, temperatures=([0.9, 0.0, 1.3] * n)[:n])
    d.compare(tf_ctx, cap=20.0)
    assert tf_ctx.device_status() == 0


@pytest.mark.parametrize("probs", [None, torch.float32])
@pytest.mark.parametrize("cap", [0.0, 30.0])
@pytest.mark.parametrize("dtype", TYPES)
def test_tests_at_their_border(tf_ctx, probs, cap, dtype):
    """Random numbers within what sums in 32 bits are off by: the row is summed again, and every one falls on its side."""
    n, vocab = 240, 13001
    d = wide(11, [2] * n, 2, vocab, dtype=dtype, probs=probs)
    near = 0
    for b in range(n):
        x = int(d.tokens[b, 1])
        w, _ = ref.softmax64(d.logits[d.offsets[b]], float(np.float32(0.9)), cap)
        border = float(w[x] / w.sum()) / (float(d.probs[b, 0, x]) if probs is not None else 1.0)
        u = np.float32(border)
        u = [u, np.nextafter(u, np.float32(0)), np.nextafter(u, np.float32(2)), np.float32(border * (1 + 3e-6)), np.float32(border * (1 - 3e-6)),
             np.float32(border * (1 + 2.0 ** -15)), np.float32(border * (1 - 2.0 ** -15))][b % 7]
        if 0 < u < 1:
            d.uniforms[b, 1] = float(u)
            near += 1
    assert near > n / 4
    d.compare(tf_ctx, temperatures=[0.9] * n, cap=cap)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cap", [0.0, 12.0])
def test_logits_that_count_for_nothing(tf_ctx, dtype, cap):
    """Infinities, NaN and the type's lowest value; rows with one finite logit and with none; logits far beyond the cap."""
    vocab = 160001
    for probs in (None, torch.float32):
        d = wide(21, [4] * 9, 4, vocab, dtype=dtype, probs=probs)
        d.logits[:, ::3] = -math.inf
        d.logits[1::2, 1::7] = math.inf
        d.logits[2::3, 2::11] = math.nan
        d.logits[::4, 5] = torch.finfo(dtype).min
        d.logits[8:12] = -math.inf                                 # a sequence without any
        d.logits[8:12, 17] = math.nan
        d.logits[16:20] = torch.finfo(dtype).min                   # all the same, far down
        d.logits[20:24] = -math.inf
        d.logits[20:24, 4] = 0.25                                  # one token alone
        d.tokens[5, 1:] = 4
        d.logits[28:32, vocab // 2:] = math.nan                    # blocks and parts with nothing in them
        d.logits[32:36, 7] = 3000.0
        for heat in (None, [0.0] * 9, [0.6] * 9):
            out = d.compare(tf_ctx, temperatures=heat, cap=cap)
        assert out[0][2, 0] == 0 and out[3][2, 0] == -math.inf
    assert tf_ctx.device_status() == 0


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cap", [0.0, 30.0])
def test_rows_cut_by_the_caller(tf_ctx, dtype, cap):
    """All but the 64 likeliest logits of a row are -infinity, as a caller cuts a distribution."""
    for probs in (None, torch.float32):
        d = wide(22, [5, 3, 5, 1, 4, 5], 5, 250007, dtype=dtype, probs=probs)
        least = d.logits.topk(64, -1).values[:, -1:]
        d.logits.masked_fill_(d.logits < least, -math.inf)
        for heat in (None, [0.7, 1.4, 0.0, 1.0, 3.0, 0.1]):
            d.compare(tf_ctx, temperatures=heat, cap=cap)


@pytest.mark.parametrize("nodes", [1, 4])
def test_calls_without_rows(tf_ctx, nodes):
    from turbo_fieldfare_b200 import drafts as dr
    d = Draft(1, [0, 0, 0], nodes, 100, padded=0)
    d.workspace = dr.VerificationWorkspace(tf_ctx, 1, 100)
    for heat in (None, [0.0, 1.0, 0.5]):
        out = d.compare(tf_ctx, temperatures=heat)
        assert out[2].tolist() == [0, 0, 0]
    assert tf_ctx.device_status() == 0


def test_temperatures_at_the_ends(tf_ctx):
    for dtype in TYPES:
        d = wide(8, [3] * 8, 3, 240007, dtype=dtype, probs=torch.float32)
        d.compare(tf_ctx, temperatures=[0.0, -2.0, 1e-6, 1e-30, 0.05, 50.0, 1e6, 1e-3])
        d.compare(tf_ctx, temperatures=[math.inf, 1e35, 1e30, math.inf, 1e-45, 1e-38, math.inf, -math.inf])


@pytest.mark.parametrize("cap", [1e-45, 1e-39, 2e-38, 1e-3, 300.0, 4000.0, 1e5, 1e9, 1e20, 3e38])
@pytest.mark.parametrize("counts,vocab", [([3] * 8, 240007), ([3, 2], 3001), ([1] * 8, 30011)])      # sums in 32 bits, in 64, lone rows
def test_caps_at_the_ends(tf_ctx, cap, counts, vocab):
    """From so low that all logits count alike (and that the cap's inverse is no number of 32 bits) to so high that it changes nothing; some logits are wider than any cap."""
    for dtype, far in ((torch.float16, -6e4), (torch.float32, -3.4e38)):
        d = Draft(9, counts, max(counts), vocab, dtype=dtype, tree=max(counts) > 1)
        d.logits[:, ::5] = 0.0
        d.logits[:, 1::97] = far
        d.uniforms[1, 1:] = 0.0
        for heat in (None, [0.0, 1.0, 0.8, 2.0] * 2):
            d.compare(tf_ctx, cap=cap, temperatures=None if heat is None else heat[:len(counts)])


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_at_any_distance_and_place(tf_ctx, dtype):
    """Strides and starts that are off every boundary, for logits and for the drafter's probabilities."""
    vocab = 400009
    d = wide(51, [4, 2, 4, 3], 4, vocab, dtype=dtype, probs=dtype)
    rows = d.logits.shape[0]
    for lead, gap in ((0, 0), (1, 2), (7, 1)):
        room = torch.full((rows * (vocab + gap) + lead + 9,), math.nan, dtype=dtype, device=DEV)
        x = room[lead:lead + rows * (vocab + gap)].view(rows, vocab + gap)[:, :vocab]
        x.copy_(d.logits)
        q = torch.full((4 * (3 * (vocab + gap) + 11) + lead,), math.nan, dtype=dtype, device=DEV)[lead:].as_strided((4, 3, vocab), (3 * (vocab + gap) + 11, vocab + gap, 1))
        q.copy_(d.probs)
        d.compare(tf_ctx, logits=x, probs=q)


def test_drafted_tokens_out_of_place(tf_ctx):
    """Children refused one after the other, the same token twice, probabilities that are zero, below zero, NaN, or the target's own."""
    for probs in (None, torch.float32):
        d = wide(31, [6] * 12, 6, 90001, dtype=torch.float32, probs=probs, tree=True)
        d.tokens[0, 2] = -1
        d.tokens[1, 1] = 90001
        d.tokens[2, 1:] = d.tokens[2, 1]
        d.parents[2:8] = [-1, 0, 0, 0, 0, 0]
        d.tokens[3, 1:] = [int(i) for i in torch.topk(d.logits[18], 5, largest=False).indices]
        d.parents[9, 3] = 5
        d.uniforms[4:8, 1:] = 0.999
        if probs is not None:
            d.probs[5, 0, ::2] = 0
            d.probs[6, 0, 1::3] = -0.5
            d.probs[6, 0, 2::5] = math.nan
            d.probs[7, 0] = torch.softmax(d.logits[42].float(), 0)
            d.probs[8, 0] = 0
        d.compare(tf_ctx)


def test_offsets_beyond_32_bits(tf_ctx):
    """Rows of logits and of probabilities more than 2^32 elements apart."""
    vocab, far = 3000017, (1 << 32) + 24
    d = Draft(9, [2], 2, vocab, probs=torch.float16, padded=0)
    assert 2 * vocab > SUMMED_IN_64_BITS
    x = torch.empty(far + vocab, dtype=torch.float16, device=DEV).as_strided((2, vocab), (far, 1))
    x.copy_(d.logits)
    q = torch.empty(far + vocab, dtype=torch.float16, device=DEV).as_strided((1, 2, vocab), (7, far, 1))
    q[:, :1].copy_(d.probs)
    q[:, 1:] = 0
    for u in (0.0, 0.9999):
        d.uniforms[0, 1] = u                                       # kept, refused
        d.compare(tf_ctx, logits=x, probs=q)


def test_equal_calls_give_equal_bits(tf_ctx):
    for cap in (0.0, 30.0):
        d = wide(81, [9] * 20, 9, 40011, probs=torch.float32, tree=True)
        first = d.run(tf_ctx, cap=cap)
        for _ in range(3):
            assert all(torch.equal(x, y) for x, y in zip(first, d.run(tf_ctx, cap=cap)))


def test_two_graphs_replayed_with_new_inputs(tf_ctx):
    """Each with a workspace and a stream of its own; a kernel of the graph writes the inputs just before the verification, others in every replay."""
    from turbo_fieldfare_b200 import drafts as dr
    made = []
    for seed in (1, 2):
        turns = []
        for turn in range(3):
            d = wide(10 * seed + turn, [5] * 30, 5, 45011, probs=torch.float32, tree=True)
            heat = [0.8 + 0.1 * turn, 0.0, 1.0] * 10
            turns.append(([d.logits.to(DEV), dev(d.offsets), dev(d.tokens), d.uniforms.to(DEV), dev(d.parents), d.probs.to(DEV), dev(heat, torch.float32)],
                          d.run(tf_ctx, temperatures=heat)))
        source, held = [torch.empty_like(t) for t in turns[0][0]], [torch.empty_like(t) for t in turns[0][0]]
        out = [torch.zeros_like(t) for t in turns[0][1]]
        ws = dr.VerificationWorkspace(tf_ctx, *source[0].shape)
        stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            for a, b in zip(held, source):
                torch.add(b, 0, out=a)
            dr.DraftVerification(tf_ctx).encode(*held[:4], *out[:3], ws, parents=held[4], draft_probs=held[5], temperatures=held[6], logprobs=out[3])
        made.append((graph, stream, turns, source, out, held, ws))
    for turn in (0, 1, 2, 0, 2):
        for _, _, turns, source, _, _, _ in made:
            for a, b in zip(source, turns[turn][0]):
                a.copy_(b)
        torch.cuda.synchronize()
        for graph, stream, *_ in made:
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for _, _, turns, _, out, _, _ in made:
            assert all(torch.equal(x, y) for x, y in zip(turns[turn][1], out))
    assert tf_ctx.device_status() == 0


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("nodes", [1, 6])
@pytest.mark.parametrize("cap", [0.0, 30.0, 1e9])
def test_logarithms_of_sums_in_64_bits(tf_ctx, dtype, nodes, cap):
    """Where all rows are summed in 64 bits a logarithm is off by its rounding to 32 bits alone: 2^-24 of it, and less than 1e-10 of what 64 bits leave
    (powers of two 8e-14 of a weight; capped logits, none wider than the cap, 2e-14 of themselves, over the lowest temperature)."""
    counts = [nodes, max(1, nodes // 2), nodes, 1]
    for probs in (None, torch.float32):
        for vocab in (5003, 200003):
            d = Draft(vocab + nodes, counts, nodes, vocab, dtype=dtype, probs=probs, tree=nodes > 1)
            assert nodes == 1 or d.logits.shape[0] * vocab <= SUMMED_IN_64_BITS * 2 // 3
            for heat in (None, [0.0] * 4, [0.6, 1.0, 1.7, 0.9]):
                got = d.compare(tf_ctx, cap=cap, temperatures=heat)[3].double().cpu().numpy()
                want = ref.verify(d.logits, d.offsets, d.tokens, d.uniforms, parents=d.parents, probs=d.probs, nodes=nodes, cap=cap,
                                  temperatures=None if heat is None else np.asarray(heat, dtype=np.float32))[3]
                assert np.all(np.abs(got - want) <= np.abs(want) * 2.0 ** -24 + 1e-10), np.abs(got - want).max()
