"""A step with drafted tokens through the C ABI: plans, verification and kept cache rows against plain statements, and a run of them together."""
import math

import numpy as np
import pytest
import torch

import drafts_reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
I32 = dict(dtype=torch.int32, device=DEV)


def dev(a, dtype=torch.int32):
    return torch.tensor(np.ascontiguousarray(a), dtype=dtype, device=DEV)


# ---------------------------------------------------------------------------
# plans
# ---------------------------------------------------------------------------

class Pages:
    """The same pages on the device and in the plain statement."""

    def __init__(self, sequences, table_pages, num_pages, page, windowed, rng):
        from turbo_fieldfare_b200 import drafts as dr
        order = rng.permutation(num_pages)
        self.state = {"table": np.full((sequences, table_pages), -1, dtype=np.int64), "held": np.zeros(sequences, dtype=np.int64), "first": np.zeros(sequences, dtype=np.int64),
                      "stack": order.tolist(), "context": np.zeros(sequences, dtype=np.int64), "page": page}
        self.pages = dr.KVPages(torch.full((sequences, table_pages), -1, **I32), torch.zeros(sequences, **I32), dev(order), dev([num_pages]), page,
                                torch.zeros(sequences, **I32) if windowed else None)
        self.context = torch.zeros(sequences, **I32)

    def step(self, ctx, new_rows, *, rows, kept=None, window=0, parents=None, tokens=None, nodes=None, words=0):
        """One plan on both sides, compared in everything; returns the offsets."""
        from turbo_fieldfare_b200 import drafts as dr
        n = len(new_rows)
        mark = -77
        into = dr.KVRows(torch.zeros(n + 1, **I32), torch.full((rows,), mark, **I32), sequences=torch.full((rows,), mark, **I32),
                         slots=torch.full((rows,), mark, dtype=torch.int64, device=DEV), tokens=torch.full((rows,), mark, **I32) if tokens is not None else None,
                         tree_mask=torch.full((rows, words), mark, dtype=torch.int64, device=DEV) if words else None)
        dr.KVPlan(ctx).encode(self.pages, self.context, dev(new_rows), into, kept=None if kept is None else dev(kept), window=window,
                              tokens=None if tokens is None else dev(tokens), parents=None if parents is None else dev(parents), nodes=nodes)
        stride = nodes if tokens is None and parents is None else (tokens if tokens is not None else parents).shape[1]
        offsets, got = ref.plan(self.state, new_rows, kept=kept, window=window, rows=rows, stride=stride, parents=parents, tokens=tokens, words=words)
        torch.cuda.synchronize()
        s, p = self.state, self.pages
        assert into.row_offsets.tolist() == offsets
        pad = [mark] * (rows - len(got))
        assert into.positions.tolist() == [r["position"] for r in got] + pad
        assert into.sequences.tolist() == [r["sequence"] for r in got] + pad
        assert into.slots.tolist() == [r["slot"] for r in got] + pad
        if tokens is not None:
            assert into.tokens.tolist() == [r["token"] for r in got] + pad
        if words:
            assert into.tree_mask.tolist() == [[ref.signed(w) for w in r["mask"]] for r in got] + [[mark] * words] * (rows - len(got))
        assert np.array_equal(p.page_table.cpu().numpy(), s["table"])
        assert np.array_equal(p.held_pages.cpu().numpy(), s["held"]) and np.array_equal(self.context.cpu().numpy(), s["context"])
        if p.first_pages is not None:
            assert np.array_equal(p.first_pages.cpu().numpy(), s["first"])
        left = int(p.free_count[0])
        assert left == len(s["stack"]) and p.free_pages[:left].tolist() == s["stack"]
        return offsets


@pytest.mark.parametrize("sequences,page,window,rows", [(1, 64, 0, 40), (3, 16, 0, 64), (7, 16, 40, 200), (61, 32, 100, 1500), (600, 16, 33, 9000), (5000, 16, 0, 12000)])
def test_steps_of_a_plan(tf_ctx, sequences, page, window, rows):
    """Prompts, decode steps, ends and beginnings in turn; pages and rows run short now and then."""
    rng = np.random.default_rng(sequences + page)
    per = rows // sequences + 2
    pages = Pages(sequences, 2 * per // page + 6, max(6, sequences * (2 * per // page + 3) * 2 // 3), page, window > 0, rng)
    served = np.zeros(sequences, dtype=np.int64)
    for step in range(7):
        wanted = rng.integers(0, per + 1, sequences) if step % 3 == 0 else rng.integers(0, 3, sequences)
        wanted[rng.random(sequences) < 0.1] = -1
        kept = np.where(wanted < 0, 5, rng.integers(0, served + 1)) if step else None
        offsets = pages.step(tf_ctx, wanted, rows=rows, kept=kept, window=window)
        served = np.diff(offsets)
    assert tf_ctx.device_status() == 0


@pytest.mark.parametrize("sequences,nodes,words,rows,chain", [(1, 1, 1, 1, False), (1, 13, 1, 13, False), (9, 64, 1, 700, False), (9, 65, 2, 700, False), (40, 130, 3, 6000, False),
                                                              (5, 200, 4, 1000, True), (3, 40, 2, 100, True)])
def test_trees_of_a_plan(tf_ctx, sequences, nodes, words, rows, chain):
    rng = np.random.default_rng(nodes)
    parents = np.array([[-1] + [int(rng.integers(max(-1, i - 9), i)) for i in range(1, nodes)] for _ in range(sequences)])
    tokens = rng.integers(0, 1 << 18, (sequences, nodes))
    pages = Pages(sequences, nodes // 16 + 3, sequences * (nodes // 16 + 3), 16, False, rng)
    for step in range(3):
        wanted = rng.integers(0, nodes + 1, sequences)
        wanted[0] = nodes
        pages.step(tf_ctx, wanted, rows=rows, kept=np.minimum(wanted, 2) if step else None, parents=None if chain else parents, tokens=tokens, words=words)
    assert tf_ctx.device_status() == 0


def test_plans_pass_over_what_cannot_fit(tf_ctx):
    """More tokens than the table, more rows than the tree has nodes: passed over; those behind are served. A mask without a tree, and chains said by `nodes`."""
    rng = np.random.default_rng(0)
    pages = Pages(4, 3, 20, 16, False, rng)
    assert pages.step(tf_ctx, [48, 49, 3, 0], rows=80) == [0, 48, 48, 51, 51]
    assert pages.step(tf_ctx, [0, 9, 8, 1], rows=80, nodes=8, words=1) == [0, 0, 0, 8, 9]
    assert pages.step(tf_ctx, [-1, -1, -1, -1], rows=80) == [0] * 5
    assert pages.step(tf_ctx, [0, 0, 0, 0], rows=0) == [0] * 5
    assert tf_ctx.device_status() == 0


def test_plans_of_contradicting_arrays_are_reported(tf_ctx):
    from turbo_fieldfare_b200 import drafts as dr
    from turbo_fieldfare_b200.kernels import TFError
    guard = 99

    def tried(free_count, held, parents=None, words=0, wanted=3):
        held_pages = dev([held, 0])
        room = torch.full((40,), guard, **I32)
        pages = dr.KVPages(room[8:16].view(2, 4), held_pages, dev(np.arange(6)), dev([free_count]), 16)
        rows = dr.KVRows(torch.zeros(3, **I32), torch.zeros(8, **I32), slots=torch.zeros(8, dtype=torch.int64, device=DEV),
                         tree_mask=torch.zeros(8, words, dtype=torch.int64, device=DEV) if words else None)
        dr.KVPlan(tf_ctx).encode(pages, torch.zeros(2, **I32), dev([wanted, -1]), rows, parents=None if parents is None else dev(parents))
        with pytest.raises(TFError, match="7F000054|7f000054"):
            tf_ctx.device_status()
        assert room[:8].tolist() == [guard] * 8 and room[16:].tolist() == [guard] * 24
        return rows

    tried(7, 0)                                                    # a stack of more pages than there are
    tried(-1, 0)
    rows = tried(6, 0, parents=[[-1, 1, 0], [-1, -1, -1]], words=1)    # node 1 hangs under itself: it counts as a first one
    assert rows.tree_mask[:3, 0].tolist() == [1, 2, 5] and rows.positions[:3].tolist() == [0, 0, 1]
    assert tf_ctx.device_status() == 0


def test_nodes_behind_the_mask_are_reported(tf_ctx):
    from turbo_fieldfare_b200 import drafts as dr
    from turbo_fieldfare_b200.kernels import TFError
    pages = dr.KVPages.allocate(1, 8, 8, 16)
    rows = dr.KVRows.allocate(1, 70, mask_words=1)
    dr.KVPlan(tf_ctx).encode(pages, torch.zeros(1, **I32), dev([66]), rows, nodes=66)
    with pytest.raises(TFError, match="7F000054|7f000054"):
        tf_ctx.device_status()
    assert rows.tree_mask[:66, 0].tolist() == [ref.signed((1 << min(i + 1, 64)) - 1) for i in range(66)] and rows.tree_mask[66:].eq(0).all()


# ---------------------------------------------------------------------------
# verification
# ---------------------------------------------------------------------------

def likely_logits(gen, rows, vocab):
    x = torch.randn(rows, vocab, generator=gen) * 2
    top = torch.randint(0, vocab, (rows, 6), generator=gen)
    return x.scatter(1, top, math.log(vocab) + 3 - 1.5 * torch.arange(6) + torch.randn(rows, 6, generator=gen))


class Draft:
    """Logits, a tree of tokens and random numbers for some sequences, on the CPU."""

    def __init__(self, seed, counts, nodes, vocab, *, dtype=torch.float16, probs=None, tree=False, padded=3):
        g = self.gen = torch.Generator().manual_seed(seed)
        rng = np.random.default_rng(seed)
        self.nodes, self.vocab, self.counts = nodes, vocab, counts
        self.offsets = np.concatenate([[0], np.cumsum(counts)]).tolist()
        self.logits = likely_logits(g, self.offsets[-1] + padded, vocab).to(dtype)
        n = len(counts)
        self.parents = np.array([[-1] + [int(rng.integers(max(0, i - 4), i)) for i in range(1, nodes)] for _ in range(n)]) if tree else None
        self.tokens = rng.integers(0, vocab, (n, nodes))
        self.uniforms = torch.rand(n, nodes, generator=g)
        self.probs = None
        if probs is not None and nodes > 1:
            self.probs = torch.zeros(n, nodes - 1, vocab, dtype=probs)
        for b in range(n):
            for i in range(1, min(counts[b], nodes)):
                p = int(self.parents[b, i]) if tree else i - 1
                guess = self.logits[self.offsets[b] + p].float()
                guess = torch.softmax(torch.where(guess.isfinite(), guess, torch.full_like(guess, -30.0)) + 0.5 * torch.randn(vocab, generator=g), 0)
                if self.probs is not None:
                    if not bool(self.probs[b, p].any()):
                        self.probs[b, p] = guess.to(probs)
                    guess = self.probs[b, p].float()
                    self.tokens[b, i] = int(torch.multinomial(guess, 1, generator=g))
                else:
                    self.tokens[b, i] = int(torch.topk(guess, min(3, vocab)).indices[i % min(3, vocab)])

    def run(self, ctx, *, temperatures=None, cap=0.0, logits=None, probs=None, stream=None, logprobs=True):
        from turbo_fieldfare_b200 import drafts as dr
        n = len(self.counts)
        x = self.logits.to(DEV) if logits is None else logits
        if not hasattr(self, "workspace"):
            self.workspace = dr.VerificationWorkspace(ctx, x.shape[0], self.vocab)
        out = [torch.full((n, self.nodes), 7, **I32), torch.full((n, self.nodes), 7, **I32), torch.full((n,), 7, **I32), torch.full((n, self.nodes), 7.0, device=DEV) if logprobs else None]
        q = probs if probs is not None else None if self.probs is None else self.probs.to(DEV)
        dr.DraftVerification(ctx).encode(x, dev(self.offsets), dev(self.tokens), self.uniforms.to(DEV), *out[:3], self.workspace,
                                         parents=None if self.parents is None else dev(self.parents), draft_probs=q,
                                         temperatures=None if temperatures is None else dev(temperatures, torch.float32), softcap=cap, logprobs=out[3], stream=stream)
        return out

    def compare(self, ctx, *, temperatures=None, cap=0.0, **more):
        out = self.run(ctx, temperatures=temperatures, cap=cap, **more)
        # the kernel's temperatures are the fp32 ones
        heat = None if temperatures is None else np.asarray(temperatures, dtype=np.float32)
        want = ref.verify(self.logits, self.offsets, self.tokens, self.uniforms, parents=self.parents, probs=self.probs, temperatures=heat, cap=cap, nodes=self.nodes)
        assert out[2].tolist() == want[2].tolist()
        assert np.array_equal(out[1].cpu().numpy(), want[1])
        assert np.array_equal(out[0].cpu().numpy(), want[0])
        if out[3] is not None:
            # log w - log Z: Z in 32 bits is off by 2^-15 of itself at the most where a node was not summed again (capped logits: by cap 2^-19 / T more),
            # and the result is rounded to fp32
            got, t = out[3].double().cpu().numpy(), np.ones(len(self.counts)) if heat is None else np.where(heat > 0, heat, 1.0).astype(np.float64)
            bound = 2.0 ** -15 + cap * 2.0 ** -19 / t[:, None] * 1.4427 + np.abs(np.where(np.isfinite(want[3]), want[3], 0)) * 2.0 ** -23
            same = np.isinf(got) & (got == want[3])
            assert np.all(same | (np.abs(got - want[3]) <= bound)), np.abs(got - want[3]).max()
        return out


TYPES = [torch.float16, torch.bfloat16, torch.float32]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("probs", [None, torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tree", [False, True])
def test_drafts_of_every_type(tf_ctx, dtype, probs, tree):
    counts = [5, 0, 9, 1, 9, 7, 2, 9, 8, 3]
    d = Draft(3 + tree, counts, 9, 1013, dtype=dtype, probs=probs, tree=tree)
    for cap, heat in ((0.0, None), (30.0, [1.0, 0.7, 0.0, 1.3, 0.5, 1.0, 2.0, -1.0, 1.0, 0.9])):
        d.compare(tf_ctx, cap=cap, temperatures=heat)
    assert tf_ctx.device_status() == 0


@pytest.mark.parametrize("vocab", [1, 2, 7, 8, 9, 300, 8191, 8192, 8193, 32000, 100003, 262144])
@pytest.mark.parametrize("dtype", TYPES)
def test_vocabularies(tf_ctx, vocab, dtype):
    counts = [3, 4, 1] if vocab > 9000 else [3, 4, 1, 2, 4, 4, 4, 1, 3, 4]
    d = Draft(vocab, counts, 4, vocab, dtype=dtype, probs=torch.float32)
    d.compare(tf_ctx, temperatures=[0.8] * len(counts))
    d.compare(tf_ctx, temperatures=[0.0] * len(counts))
    d = Draft(vocab + 1, counts, 4, vocab, dtype=dtype, tree=True)
    d.compare(tf_ctx, cap=20.0)


def test_a_single_token_is_drawn_by_its_number(tf_ctx):
    """All of [0, 1) in steps, one sequence each over the same logits: every token's turn comes, in order."""
    n, vocab = 900, 53
    d = Draft(1, [1] * n, 1, vocab, dtype=torch.float32, padded=0)
    d.logits[:] = d.logits[0]
    d.logits[:, ::5] = -math.inf
    d.uniforms[:, 0] = (torch.arange(n) + 0.5) / n
    out = d.compare(tf_ctx, temperatures=[1.7] * n)
    drawn = out[0][:, 0].cpu()
    assert bool((drawn[1:] >= drawn[:-1]).all()) and not bool((drawn % 5 == 0).any()) and len(set(drawn.tolist())) > 30


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cap", [0.0, 12.0])
def test_lone_rows(tf_ctx, dtype, cap):
    """The sampler: greedy and drawn rows side by side, sequences without a row, infinities, ties of the likeliest token in parts that different blocks have."""
    for vocab in (1, 37, 5000, 70001, 262144):
        counts = [1, 1, 0, 1, 1, 1, 0, 1]
        d = Draft(vocab, counts, 1, vocab, dtype=dtype)
        heat = [0.0, 0.9, 0.0, 0.0, 3.0, math.nan, 1.0, 1.0]
        d.logits[1, ::3] = -math.inf
        d.logits[2, :] = 1.5                                       # all the same
        d.logits[3, vocab // 2:] = math.nan
        d.logits[5, vocab // 3] = d.logits[5, vocab - 1] = math.inf
        d.logits[4, [vocab // 5, vocab - 1]] = 40.0
        d.compare(tf_ctx, temperatures=heat, cap=cap)
        d.compare(tf_ctx, cap=cap)
    assert tf_ctx.device_status() == 0


def test_more_sequences_than_blocks_of_the_chip(tf_ctx):
    counts = ([3, 1, 2, 0] * 90)[:350]
    for probs in (None, torch.float32):
        d = Draft(7, counts, 3, 3001, probs=probs)
        d.compare(tf_ctx, temperatures=([1.0, 0.0, 0.8] * 120)[:350])


@pytest.mark.parametrize("vocab,counts,tree", [(40, [2, 0, 1, 3, 0, 0] * 900, False), (1100, [2] * 3000, False), (300, [0] * 1500 + [4] + [0] * 1500 + [3], True)])
def test_rows_find_their_sequence_among_many(tf_ctx, vocab, counts, tree):
    d = Draft(8, counts, 4, vocab, tree=tree)
    d.compare(tf_ctx, temperatures=([0.9, 0.0, 1.3] * len(counts))[:len(counts)])
    assert tf_ctx.device_status() == 0


def test_offsets_beyond_32_bits(tf_ctx):
    """Rows of logits and of probabilities more than 2^32 elements apart."""
    d = Draft(9, [2], 2, 1500, probs=torch.float16, padded=0)
    far = (1 << 32) + 24
    room = torch.empty(far + 1500, dtype=torch.float16, device=DEV)
    x = room.as_strided((2, 1500), (far, 1))
    x.copy_(d.logits)
    q = torch.empty(far + 1500, dtype=torch.float16, device=DEV).as_strided((1, 2, 1500), (7, far, 1))
    q[:, :1].copy_(d.probs)
    q[:, 1:] = 0
    d.compare(tf_ctx, logits=x, probs=q)
    d.uniforms[:] = 0.9999
    d.compare(tf_ctx, logits=x, probs=q)


@pytest.mark.parametrize("probs", [None, torch.float32])
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_tests_at_their_border(tf_ctx, probs, dtype):
    """Random numbers next to the border: what 32 bits cannot tell apart is told apart."""
    n, vocab = 240, 700
    d = Draft(11, [2] * n, 2, vocab, dtype=dtype, probs=probs)
    heat = [0.9] * n
    near = 0
    for b in range(n):
        x = int(d.tokens[b, 1])
        w, _ = ref.softmax64(d.logits[d.offsets[b]], float(np.float32(0.9)), 0.0)
        border = float(w[x] / w.sum()) / (float(d.probs[b, 0, x]) if probs is not None else 1.0)
        u = np.float32(border)
        u = [u, np.nextafter(u, np.float32(0)), np.nextafter(u, np.float32(2)), np.float32(border * (1 + 3e-6)), np.float32(border * (1 - 3e-6))][b % 5]
        if 0 < u < 1:
            d.uniforms[b, 1] = float(u)
            near += 1
    assert near > n / 4
    d.compare(tf_ctx, temperatures=heat)


def test_random_numbers_at_the_ends(tf_ctx):
    counts = [4] * 12
    for seed, probs in ((5, None), (6, torch.float32)):
        d = Draft(seed, counts, 4, 500, probs=probs)
        d.uniforms[:4] = 0.0
        d.uniforms[4:8] = 1 - 2.0 ** -24
        d.uniforms[8:] = 1.0                                       # beyond the end: as the last number before it
        d.compare(tf_ctx)


def test_logits_that_count_for_nothing(tf_ctx):
    """Infinities, NaN and the type's lowest value; rows with one finite logit and with none."""
    for dtype in TYPES:
        for probs in (None, torch.float32):
            d = Draft(21, [4] * 9, 4, 300, dtype=dtype, probs=probs)
            d.logits[:, ::3] = -math.inf
            d.logits[1::2, 1::7] = math.inf
            d.logits[2::3, 2::11] = math.nan
            d.logits[::4, 5] = torch.finfo(dtype).min
            d.logits[8:12] = -math.inf                             # a sequence without any
            d.logits[8:12, 17] = math.nan
            d.logits[16:20] = torch.finfo(dtype).min               # all the same, far down
            d.logits[20:24] = -math.inf
            d.logits[20:24, 4] = 0.25                              # one token alone
            d.tokens[5, 1:] = 4
            for heat in (None, [0.0] * 9, [0.6] * 9):
                out = d.compare(tf_ctx, temperatures=heat)
            assert out[0][2, 0] == 0 and out[3][2, 0] == -math.inf


def test_temperatures_at_the_ends(tf_ctx):
    for dtype in TYPES:
        d = Draft(8, [3] * 8, 3, 400, dtype=dtype, probs=torch.float32)
        # greedy: zero, below zero and NaN; so cold that only the likeliest counts; so hot that all count alike
        d.compare(tf_ctx, temperatures=[0.0, -2.0, 1e-6, 1e-30, 0.05, 50.0, 1e6, 1e-3])
        out = d.run(tf_ctx, temperatures=[math.nan] * 8)
        again = d.run(tf_ctx, temperatures=[0.0] * 8)
        assert all(torch.equal(x, y) for x, y in zip(out, again))


def test_drafted_tokens_out_of_place(tf_ctx):
    """Tokens outside the vocabulary are passed over; the same token twice; probabilities that are zero, below zero, NaN, or the target's own."""
    for probs in (None, torch.float32):
        d = Draft(31, [6] * 12, 6, 200, dtype=torch.float32, probs=probs, tree=True)
        d.tokens[0, 2] = -1
        d.tokens[1, 1] = 200
        d.tokens[2, 1:] = d.tokens[2, 1]
        d.parents[2:8] = [-1, 0, 0, 0, 0, 0]                       # children of one node, refused one after the other
        d.tokens[3, 1:] = [int(i) for i in torch.topk(d.logits[18], 5, largest=False).indices]
        d.parents[9, 3] = 5                                        # hangs under a node behind it: under none
        d.uniforms[4:8, 1:] = 0.999
        if probs is not None:
            d.probs[5, 0, ::2] = 0
            d.probs[6, 0, 1::3] = -0.5
            d.probs[6, 0, 2::5] = math.nan
            d.probs[7, 0] = torch.softmax(d.logits[42].float(), 0)
            d.probs[8, 0] = 0
        d.compare(tf_ctx)


def test_nodes_without_a_row_of_the_drafter(tf_ctx):
    d = Draft(41, [7] * 10, 7, 600, probs=torch.float16, tree=True)
    d.probs = d.probs[:, :2].contiguous()
    d.compare(tf_ctx)
    d.probs = d.probs[:, :0]
    assert d.run(tf_ctx, probs=torch.zeros(10, 0, 600, device=DEV))[2].tolist() == ref.verify(
        d.logits, d.offsets, d.tokens, d.uniforms, parents=d.parents, nodes=7)[2].tolist()


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_at_any_distance_and_place(tf_ctx, dtype):
    """Strides and starts that are off every boundary, for logits and for the drafter's probabilities."""
    d = Draft(51, [4, 2, 4, 3], 4, 777, dtype=dtype, probs=dtype)
    rows = d.logits.shape[0]
    for lead, gap in ((0, 0), (1, 2), (3, 5), (7, 1)):
        room = torch.full((rows * (777 + gap) + lead + 9,), math.nan, dtype=dtype, device=DEV)
        x = room[lead:lead + rows * (777 + gap)].view(rows, 777 + gap)[:, :777]
        x.copy_(d.logits)
        q = torch.full((4 * (3 * (777 + gap) + 11) + lead,), math.nan, dtype=dtype, device=DEV)[lead:].as_strided((4, 3, 777), (3 * (777 + gap) + 11, 777 + gap, 1))
        q.copy_(d.probs)
        d.compare(tf_ctx, logits=x, probs=q)


def test_many_nodes_and_many_children(tf_ctx):
    counts = [1024, 300, 1024]
    for probs in (None, torch.bfloat16):
        d = Draft(61, counts, 1024, 40, probs=probs, tree=True, padded=0)
        d.parents[0] = [-1] + [0] * 1023                           # all children of the first node, most of them refused
        d.uniforms[0, 1:] = 0.97
        d.compare(tf_ctx)


def test_offsets_that_contradict_themselves_are_reported(tf_ctx):
    from turbo_fieldfare_b200.kernels import TFError
    d = Draft(71, [3, 3, 3], 3, 100, padded=0)
    for offsets in ([0, 4, 5, 9], [0, 3, 6, 90], [-5, 3, 6, 9]):   # more rows than nodes; behind the rows; before them
        d.offsets = offsets
        d.run(tf_ctx)
        with pytest.raises(TFError, match="7F000052|7f000052"):
            tf_ctx.device_status()
    assert tf_ctx.device_status() == 0


@pytest.mark.parametrize("nodes", [1, 3])
@pytest.mark.parametrize("sequences", [40, 2500])
def test_offsets_out_of_order_draw_tokens_of_the_row(tf_ctx, sequences, nodes):
    from turbo_fieldfare_b200.kernels import TFError
    vocab = 4001
    d = Draft(12, [1] * sequences, nodes, vocab)
    d.offsets = np.random.default_rng(3).integers(-3, sequences + 3, sequences + 1).tolist()
    out = d.run(tf_ctx)
    with pytest.raises(TFError, match="7F000052|7f000052"):
        tf_ctx.device_status()
    assert bool(((out[0] >= -1) & (out[0] < vocab)).all()) and bool(((out[2] >= 0) & (out[2] <= nodes)).all())


def test_equal_calls_give_equal_bits(tf_ctx):
    d = Draft(81, [9] * 20, 9, 30011, probs=torch.float32, tree=True)
    first = d.run(tf_ctx)
    for _ in range(3):
        assert all(torch.equal(x, y) for x, y in zip(first, d.run(tf_ctx)))


def test_other_streams_and_graphs(tf_ctx):
    """Two captured graphs with a workspace each replayed side by side, on streams of their own."""
    from turbo_fieldfare_b200 import drafts as dr
    made = []
    for seed in (1, 2):
        d = Draft(seed, [5] * 30, 5, 20011, probs=torch.float32)
        want = d.run(tf_ctx)
        held = [d.logits.to(DEV), dev(d.offsets), dev(d.tokens), d.uniforms.to(DEV), d.probs.to(DEV)]
        out = [torch.zeros_like(t) for t in want]
        ws = dr.VerificationWorkspace(tf_ctx, *d.logits.shape)
        stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            dr.DraftVerification(tf_ctx).encode(*held[:4], *out[:3], ws, draft_probs=held[4], logprobs=out[3])
        made.append((graph, stream, want, out, held, ws))
    for _ in range(5):
        for _, _, _, out, _, _ in made:
            for t in out:
                t.zero_()
        torch.cuda.synchronize()
        for graph, stream, *_ in made:
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for _, _, want, out, _, _ in made:
            assert all(torch.equal(x, y) for x, y in zip(want, out))
    assert tf_ctx.device_status() == 0


# ---------------------------------------------------------------------------
# kept cache rows
# ---------------------------------------------------------------------------

def _cache(pages, page, kv, dim, bits, gen):
    from turbo_fieldfare_b200.attention import KVCache
    planes = []
    for _ in range(2):
        planes.append(torch.randint(0, 256, (pages, kv, page, dim * bits // 8), generator=gen, dtype=torch.uint8).to(DEV))
        for _ in range(2):
            planes.append(torch.randn(pages, kv, page, dim // 64, generator=gen).bfloat16().to(DEV))
    return KVCache(*planes)


@pytest.mark.parametrize("dim,bits", [(64, 4), (64, 8), (128, 8), (256, 4), (512, 8), (512, 4)])
@pytest.mark.parametrize("sequences,nodes,layers", [(1, 5, 1), (9, 70, 3), (3, 20, 35)])
def test_kept_rows_move_in_place(tf_ctx, dim, bits, sequences, nodes, layers):
    """Every byte of every plane is as the plain statement leaves it: paths that overlap what they are moved to, whole chains, nothing kept."""
    from turbo_fieldfare_b200 import attention as at
    from turbo_fieldfare_b200 import drafts as dr
    rng, gen = np.random.default_rng(dim + nodes), torch.Generator().manual_seed(dim)
    page = 16
    context = rng.integers(0, 40, sequences)
    counts = rng.integers(1, nodes + 1, sequences)
    counts[0] = nodes
    per = int((context + counts).max()) // page + 1
    order = rng.permutation(sequences * per + 2)[:sequences * per].reshape(sequences, per)
    path, kept = np.full((sequences, nodes), -1), np.zeros(sequences, dtype=np.int64)
    for b in range(sequences):
        kept[b] = [counts[b], 0, 1][b % 7] if b % 7 < 3 and b else rng.integers(1, counts[b] + 1)
        path[b, :kept[b]] = np.sort(np.concatenate([[0], rng.choice(np.arange(1, counts[b]), max(0, kept[b] - 1), replace=False)]))[:kept[b]]
    caches = [_cache(sequences * per + 2, page, 1 + i % 3, dim, bits, gen) for i in range(layers)]
    want = []
    for c in caches:
        planes = [t.clone() for t in c.planes]
        for b in range(sequences):
            for i in range(kept[b]):
                s, t = int(context[b] + path[b, i]), int(context[b] + i)
                for p in planes:
                    p[order[b, t // page], :, t % page] = p[order[b, s // page], :, s % page].clone()
        want.append(planes)
    batch = at.KVBatch(dev(np.concatenate([[0], np.cumsum(counts)])), dev(context), dev(order), rows=int(counts.sum()) + 2)
    dr.KVCacheKeep(tf_ctx).encode(caches, batch, dev(path), dev(kept))
    assert tf_ctx.device_status() == 0
    for c, planes in zip(caches, want):
        assert all(torch.equal(x, y) for x, y in zip(c.planes, planes))


def test_kept_rows_out_of_place_are_reported(tf_ctx):
    from turbo_fieldfare_b200 import attention as at
    from turbo_fieldfare_b200 import drafts as dr
    from turbo_fieldfare_b200.kernels import TFError
    for path, table, code in (([0, 3, 3, 4], [[0, 1]], "52"), ([0, 2, 9, 4], [[0, 1]], "52"), ([0, -2, 3, 4], [[0, 1]], "52"), ([0, 2, 3, 4], [[0, 7]], "51"), ([0, 2, 3, 4], [[0, -1]], "51")):
        cache = _cache(2, 16, 2, 64, 8, torch.Generator().manual_seed(1))
        before = [t.clone() for t in cache.planes]
        batch = at.KVBatch(dev([0, 5]), dev([13]), dev(table), rows=5)
        dr.KVCacheKeep(tf_ctx).encode(cache, batch, dev([path]), dev([4]))
        with pytest.raises(TFError, match=f"7F0000{code}|7f0000{code}"):
            tf_ctx.device_status()
        # tokens 13 ... 15 lie on page 0; what moved, moved whole
        good = 1 if path[1] == 2 and table[0][1] == 1 else 0
        for x, y in zip(cache.planes, before):
            assert torch.equal(x[0, :, :13], y[0, :, :13]) and torch.equal(x[1], y[1])
            if good:
                assert torch.equal(x[0, :, 14], y[0, :, 15])
    assert tf_ctx.device_status() == 0


# ---------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------

def test_steps_together_in_one_graph(tf_ctx):
    """Plan, cache write, attention, logits, verification and kept rows as one captured step over two layers, replayed with growing contexts. What the cache then holds
    is what the kept tokens, written one behind the other, leave there, and a greedy sequence's tokens are the target's likeliest."""
    from turbo_fieldfare_b200 import attention as at
    from turbo_fieldfare_b200 import drafts as dr
    from turbo_fieldfare_b200.kernels import MPPPrefillInt4QMM
    heads, kv, dim, vocab, n, nodes, page, layers, hidden = 4, 2, 64, 256, 6, 9, 16, 2, 256
    g = torch.Generator().manual_seed(5)
    rows = n * nodes
    embed = torch.randn(vocab, (heads + 2 * kv) * dim, generator=g).half().to(DEV)
    weights, scales, biases = torch.zeros(vocab, hidden // 2, dtype=torch.uint8, device=DEV), *(torch.zeros(vocab, hidden // 64, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    tf_ctx.check(tf_ctx.lib.tf_fill_affine_synthetic(tf_ctx.handle, torch.cuda.current_stream().cuda_stream, weights.data_ptr(), scales.data_ptr(), biases.data_ptr(), vocab, hidden, 4, 9))
    scales *= 8
    biases *= 8
    freqs = torch.linspace(1.0, 0.01, 32, device=DEV)
    pages = dr.KVPages.allocate(n, 12, n * 12, page)
    caches = [at.KVCache.allocate(n * 12, page, kv, dim, 8) for _ in range(layers)]
    into = dr.KVRows.allocate(n, rows, mask_words=1, tokens=True)
    context, wanted, kept = torch.zeros(n, **I32), torch.full((n,), nodes, **I32), torch.zeros(n, **I32)
    tokens, parents = torch.zeros(n, nodes, **I32), torch.zeros(n, nodes, **I32)
    uniforms, heat = torch.zeros(n, nodes, device=DEV), dev([0.0, 1.0, 0.8, 0.0, 1.2, 1.0], torch.float32)
    out_tokens, out_rows, logprobs = torch.zeros(n, nodes, **I32), torch.zeros(n, nodes, **I32), torch.zeros(n, nodes, device=DEV)
    q, attn, logits = torch.zeros(rows, heads * dim, dtype=torch.float16, device=DEV), torch.zeros(rows, heads * dim, dtype=torch.float16, device=DEV), torch.zeros(rows, vocab, dtype=torch.float16, device=DEV)
    x = torch.zeros(rows, (heads + 2 * kv) * dim, dtype=torch.float16, device=DEV)
    ws, vs = at.AttentionWorkspace(tf_ctx, dim), dr.VerificationWorkspace(tf_ctx, rows, vocab)
    batch = at.KVBatch(into.row_offsets, context, pages.page_table, into.positions)
    split = [heads * dim, kv * dim, kv * dim]

    def step():
        dr.KVPlan(tf_ctx).encode(pages, context, wanted, into, kept=kept, tokens=tokens, parents=parents)
        for layer in range(layers):
            torch.index_select(embed, 0, into.tokens, out=x)
            x.add_(float(layer))
            at.FusedQKVEpilogue(tf_ctx).encode(*x.split(split, 1), q, batch, caches[layer], head_dim=dim, norm_v=True, frequencies=freqs)
            at.TreeAttention(tf_ctx).encode(q, attn, caches[layer], batch, ws, scale=0.3, tree_mask=into.tree_mask)
        MPPPrefillInt4QMM(tf_ctx).encode(weights, scales, biases, attn, logits, rows, vocab, hidden)
        dr.DraftVerification(tf_ctx).encode(logits, into.row_offsets, tokens, uniforms, out_tokens, out_rows, kept, vs, parents=parents, temperatures=heat, logprobs=logprobs)
        dr.KVCacheKeep(tf_ctx).encode(caches, batch, out_rows, kept)

    def drafted(rng, newest):
        """New trees under the newest tokens; two chains among them."""
        t = rng.integers(0, vocab, (n, nodes))
        t[:, 0] = newest
        p = np.array([[-1] + [int(rng.integers(max(0, i - 3), i)) for i in range(1, nodes)] for _ in range(n)])
        p[:2] = np.arange(-1, nodes - 1)
        tokens.copy_(dev(t)), parents.copy_(dev(p))
        uniforms.copy_(torch.rand(n, nodes, generator=g).to(DEV))
        return t, p

    rng = np.random.default_rng(3)
    newest = rng.integers(0, vocab, n)
    history = [[] for _ in range(n)]
    drafted(rng, newest)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):                                # before capture: attributes and lazy loads
        step()
    torch.cuda.synchronize()
    for t in (context, kept, pages.held_pages):
        t.zero_()
    pages.free_count.fill_(n * 12)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        step()
    accepted = 0
    for turn in range(8):
        t, p = drafted(rng, newest)
        if turn % 2:                                               # the target's own choices, so that drafts are kept: the last step's logits say what they would be
            with torch.cuda.stream(stream):
                graph.replay()
            torch.cuda.synchronize()
            kept.zero_()                                           # the same step again, with better tokens
            context_now = context.tolist()
            offs = into.row_offsets.tolist()
            for b in range(n):
                t[b, 1] = int(logits[offs[b]].argmax())
                p[b, 1] = 0
            tokens.copy_(dev(t)), parents.copy_(dev(p))
            assert context.tolist() == context_now
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert tf_ctx.device_status() == 0
        offs = into.row_offsets.tolist()
        assert offs == [nodes * i for i in range(n + 1)]
        want = ref.verify(logits.cpu(), offs, t, uniforms.cpu(), parents=p, temperatures=heat.cpu().numpy(), nodes=nodes)
        assert np.array_equal(out_tokens.cpu().numpy(), want[0]) and np.array_equal(out_rows.cpu().numpy(), want[1]) and kept.tolist() == want[2].tolist()
        for b in range(n):
            history[b] += [int(newest[b])] + [int(v) for v in want[0][b, :want[2][b] - 1]]
            newest[b] = want[0][b, want[2][b] - 1]
        accepted += int(want[2].sum()) - n
    assert accepted > 8
    # the same tokens written one behind the other into caches of their own
    lens = [len(h) for h in history]
    assert [int(c) + int(k) for c, k in zip(context, kept)] == lens
    total = sum(lens)
    flat = dev(np.concatenate(history), torch.int64)
    plain = at.KVBatch(dev(np.concatenate([[0], np.cumsum(lens)])), torch.zeros(n, **I32), dev(np.arange(n * 12).reshape(n, 12)), dev(np.concatenate([np.arange(m) for m in lens])), rows=total)
    mine = at.KVBatch(dev(np.concatenate([[0], np.cumsum(lens)])), torch.zeros(n, **I32), pages.page_table, rows=total)
    for layer in range(layers):
        other = at.KVCache.allocate(n * 12, page, kv, dim, 8)
        y = embed[flat] + float(layer)
        at.FusedQKVEpilogue(tf_ctx).encode(*y.split(split, 1), torch.empty(total, heads * dim, dtype=torch.float16, device=DEV), plain, other, head_dim=dim, norm_v=True, frequencies=freqs)
        got = [torch.zeros(total, kv * dim, dtype=torch.float16, device=DEV) for _ in range(4)]
        at.KVCacheRead(tf_ctx).encode(other, plain, got[0], got[1])
        at.KVCacheRead(tf_ctx).encode(caches[layer], mine, got[2], got[3])
        assert torch.equal(got[0], got[2]) and torch.equal(got[1], got[3])
    assert tf_ctx.device_status() == 0
