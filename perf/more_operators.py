"""What a batched step with drafted tokens needs around its layers, as cases with inputs, one pass, a plain form and a definition.

  plan     from request lengths: pages given back and taken, block tables, row offsets, positions, slots, tokens and tree masks of the step's rows
  verify   the drafted tokens of every sequence against the target's logits, with given random numbers: which are accepted, the next token,
           and the logarithms of their probabilities. With one row per sequence it is the sampler of a single token
  keep     the cache rows of the accepted nodes of every tree moved next to their context, in the caches of several layers; the kept
           rows are then read back, which is how the pass shows what it moved

The vocabulary of 262144, head counts, head sizes and the window of 1024 are those of the model that this framework's expert blocks belong to, beside
common and odd ones. A pass leaves what it finds the second time as the first time left it: a plan that is made again takes no more pages, and the
accepted nodes of a tree stand behind the place that they are moved to.
"""
import math

import numpy as np
import torch

own = False
_kept = {}


def listed():
    return [
        # a single chat user with a small tree: the smallest call, latency only
        {"name": "plan_1", "kind": "plan", "seqs": 1, "rows": 13, "ctx": 700, "page": 64, "window": 0, "tree": True},
        # a busy server's decode batch in the layers with a window: some requests end, some begin, pages fall out of the window
        {"name": "plan_200", "kind": "plan", "seqs": 200, "rows": 1, "ctx": 8192, "page": 64, "window": 1024, "tree": False},
        # trees of drafted tokens of a batch
        {"name": "plan_tree_61", "kind": "plan", "seqs": 64, "rows": 61, "ctx": 5000, "page": 32, "window": 0, "tree": True},
        # prompts that begin together, small pages
        {"name": "plan_prompts", "kind": "plan", "seqs": 9, "rows": 4096, "ctx": 0, "page": 16, "window": 0, "tree": False},
        # one token of one user: sampled from the capped logits of the benchmark's vocabulary, nothing drafted
        {"name": "sample_1", "kind": "verify", "seqs": 1, "rows": 1, "vocab": 262144, "type": "f16", "draft": "none", "tree": False, "temperature": 1.0, "cap": 30.0},
        # one user with a chain of five drafted tokens and the drafter's probabilities
        {"name": "verify_1x6", "kind": "verify", "seqs": 1, "rows": 6, "vocab": 262144, "type": "f16", "draft": "f32", "tree": False, "temperature": 0.8, "cap": 0.0},
        # the benchmark's batch with chains of seven drafted tokens
        {"name": "verify_64x8", "kind": "verify", "seqs": 64, "rows": 8, "vocab": 262144, "type": "f16", "draft": "f32", "tree": False, "temperature": 1.0, "cap": 0.0},
        # trees drafted without probabilities (the drafter's likeliest tokens), an odd vocabulary, greedy requests among the others
        {"name": "verify_tree_33x13", "kind": "verify", "seqs": 33, "rows": 13, "vocab": 100003, "type": "bf16", "draft": "none", "tree": True, "temperature": 0.7, "cap": 30.0},
        # trees drawn from a drafter with a small vocabulary, logits in 32 bits
        {"name": "verify_tree_16x25", "kind": "verify", "seqs": 16, "rows": 25, "vocab": 32000, "type": "f32", "draft": "bf16", "tree": True, "temperature": 1.0, "cap": 0.0},
        # a busy server's greedy batch with short chains
        {"name": "greedy_200x4", "kind": "verify", "seqs": 200, "rows": 4, "vocab": 262144, "type": "f16", "draft": "none", "tree": False, "temperature": 0.0, "cap": 0.0},
        # the accepted path of one user's tree, one layer
        {"name": "keep_1", "kind": "keep", "seqs": 1, "rows": 13, "ctx": 700, "kv": 8, "dim": 256, "bits": 8, "page": 64, "layers": 1},
        # wide trees of a batch, layers with two heads of 512
        {"name": "keep_64", "kind": "keep", "seqs": 64, "rows": 61, "ctx": 900, "kv": 2, "dim": 512, "bits": 4, "page": 64, "layers": 5},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    kind = rng.choice(["plan", "verify", "verify", "verify", "verify", "keep"])
    if kind == "plan":
        c = {"kind": kind, "seqs": _log_int(rng, 1, 300), "page": rng.choice([16, 32, 64, 64, 128]), "window": rng.choice([0, 0, 1024, 100]), "tree": rng.random() < 0.5}
        c.update(rows=_log_int(rng, 1, 64) if c["tree"] else _log_int(rng, 1, max(1, min(5000, 40000 // c["seqs"]))), ctx=rng.choice([0, _log_int(rng, 1, 20000)]))
        return c
    if kind == "keep":
        kv, dim = rng.choice([(8, 256), (2, 512), (8, 128), (4, 128), (8, 64), (1, 64)])
        return {"kind": kind, "seqs": _log_int(rng, 1, 60), "rows": _log_int(rng, 3, 64), "ctx": _log_int(rng, 1, 900), "kv": kv, "dim": dim, "bits": rng.choice([8, 4]),
                "page": rng.choice([16, 32, 64, 128]), "layers": rng.choice([1, 2, 3, 5])}
    c = {"kind": kind, "vocab": rng.choice([262144, _log_int(rng, 300, 262144), _log_int(rng, 20000, 262144)]), "type": rng.choice(["f16", "bf16", "f32"]),
         "draft": rng.choice(["none", "f32", "f32", "bf16"]), "temperature": rng.choice([0.0, 1.0, 1.0, 0.7, 1.3]), "cap": rng.choice([0.0, 0.0, 30.0])}
    tree = rng.random() < 0.4
    c.update(tree=tree, seqs=_log_int(rng, 1, 40 if tree else 100))
    c["rows"] = _log_int(rng, 2, 32) if tree else _log_int(rng, 1, 12)
    c["rows"] = max(1, min(c["rows"], 100_000_000 // (c["seqs"] * c["vocab"])))
    return c


# --- what a case fixes, whatever the seed: lengths and the shape of the trees ---

def _lengths(case):
    """(rows, context) of every sequence: ragged, the first one with the full numbers."""
    n, ctx = case["seqs"], case.get("ctx", 0)
    r = np.random.RandomState(1 + n * 7919 + ctx)
    rows = np.full(n, case["rows"], dtype=np.int64)
    lens = np.full(n, ctx, dtype=np.int64)
    if n > 1:
        lens[1:] = np.ceil(ctx * r.uniform(0.1, 1.0, n - 1)).astype(np.int64)
        if case["rows"] > 1:
            rows[1:] = r.randint(max(1, case["rows"] // 2), case["rows"] + 1, n - 1)
    return rows, lens


def _parents(case):
    """[seqs, rows]: token i hangs under one of the few before it, the first under none; -1 behind a sequence's own."""
    rows, _ = _lengths(case)
    r = np.random.RandomState(case["rows"] + 31 * case["seqs"])
    out = np.full((case["seqs"], case["rows"]), -1, dtype=np.int64)
    for b, n in enumerate(rows):
        for i in range(1, n):
            out[b, i] = r.randint(max(0, i - 6), i) if case["tree"] else i - 1
    return out


def _deepest(case):
    p, most = _parents(case), 0
    for b in range(p.shape[0]):
        depth = np.zeros(p.shape[1], dtype=np.int64)
        for i in range(1, p.shape[1]):
            depth[i] = depth[p[b, i]] + 1 if p[b, i] >= 0 else 0
        most = max(most, int(depth.max()))
    return most


def _requests(case):
    """Rows asked for in a plan: every 16th sequence ends, every 16th begins."""
    rows, lens = _lengths(case)
    b = np.arange(case["seqs"])
    rows = np.where(b % 16 == 7, -1, rows)
    return rows, np.where(b % 16 == 11, 0, lens)


def _path(case):
    """[seqs, rows] of accepted nodes and how many: the root, then nodes that stand behind the last place of the path."""
    rows, _ = _lengths(case)
    r = np.random.RandomState(5 + case["rows"] * case["seqs"])
    path, kept = np.full((case["seqs"], case["rows"]), -1, dtype=np.int64), np.zeros(case["seqs"], dtype=np.int64)
    for b, n in enumerate(rows):
        a = int(r.randint(0, min(8, max(1, n // 2)))) if b else min(7, (n - 1) // 2)
        path[b, 0], kept[b] = 0, a + 1
        path[b, 1:a + 1] = np.sort(r.choice(np.arange(a + 1, n), a, replace=False))
    return path, kept


def _size(name):
    return {"f16": 2, "bf16": 2, "f32": 4, "none": 0}[name]


def work(case):
    rows, lens = _lengths(case)
    n = int(rows.sum())
    if case["kind"] == "plan":
        asked, ctx = _requests(case)
        n = int(np.maximum(asked, 0).sum())
        pages = int(((ctx + np.maximum(asked, 0) + case["page"] - 1) // case["page"] - (ctx + case["page"] - 1) // case["page"]).sum())
        # rows: position, slot, sequence and token, a mask word and the parent of a tree's; sequences: lengths, offsets, pages held; pages taken
        return {"bytes": n * (4 + 8 + 4 + (20 if case["tree"] else 0)) + case["seqs"] * 28 + pages * 8, "flops": 0}
    if case["kind"] == "keep":
        _, kept = _path(case)
        token = 2 * case["kv"] * (case["dim"] * case["bits"] // 8 + case["dim"] // 64 * 4)
        # accepted nodes read and written, the kept rows read back as 16-bit ones
        return {"bytes": case["layers"] * (int((kept - 1).sum()) * 2 * token + int(kept.sum()) * (token + 4 * case["kv"] * case["dim"])), "flops": 0}
    inner = n
    if case["temperature"] > 0:                     # a leaf's logits are needed where the path ends there; a drafter's row where it was refused
        p = _parents(case)
        inner = sum(len(set(p[b][p[b] >= 0].tolist())) for b in range(case["seqs"])) + case["seqs"]
    size = inner * _size(case["type"]) + (case["seqs"] * _size(case["draft"]) if case["rows"] > 1 and case["temperature"] > 0 else 0)
    return {"bytes": size * case["vocab"], "flops": 4 * inner * case["vocab"]}


# --- inputs ---

_TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def _dev(a, t=torch.int32):
    return torch.tensor(np.ascontiguousarray(a), dtype=t, device="cuda")


def _prepare_plan(case, gen, s):
    asked, lens = _requests(case)
    n, page = case["seqs"], case["page"]
    held = -(-lens // page)
    first = np.minimum(held, np.maximum(0, lens - 4 - case["window"] + 1) // page) if case["window"] else np.zeros_like(held)
    wanted = -(-(lens + np.maximum(asked, 0)) // page)
    pages = int(np.maximum(held, wanted).sum()) + 5
    order = torch.randperm(pages, generator=gen, device="cuda").cpu().numpy()
    table = np.full((n, int(np.maximum(held, wanted).max()) + 1), -1, dtype=np.int64)
    at = 0
    for b in range(n):
        table[b, first[b]:held[b]] = order[at:at + held[b] - first[b]]
        at += held[b] - first[b]
    rows = int(np.maximum(asked, 0).sum()) + 3                    # a padded batch
    s.update(page_table=_dev(table), held_pages=_dev(held), first_pages=_dev(first) if case["window"] else None, free_pages=_dev(np.concatenate([order[at:], np.zeros(at, dtype=np.int64)])),
             free_count=_dev([pages - at]), context_lengths=_dev(lens), new_rows=_dev(asked), parents=None, tokens=None)
    zeros = lambda *shape, t=torch.int32: torch.zeros(*shape, dtype=t, device="cuda")  # noqa: E731
    s.update(row_offsets=zeros(n + 1), positions=zeros(rows), sequences=zeros(rows), slots=zeros(rows, t=torch.int64), row_tokens=None, tree_mask=None)
    if case["tree"]:
        s["parents"] = _dev(_parents(case))
        s["tokens"] = torch.randint(0, 262144, (n, case["rows"]), generator=gen, device="cuda", dtype=torch.int32)
        s["row_tokens"], s["tree_mask"] = zeros(rows), zeros(rows, 1, t=torch.int64)
        s["deepest"] = _deepest(case)


def _prepare_verify(case, gen, s):
    rows, _ = _lengths(case)
    n, most, vocab = case["seqs"], case["rows"], case["vocab"]
    total = int(rows.sum())
    offsets = np.concatenate([[0], np.cumsum(rows)])
    logits = torch.empty(total, vocab, dtype=_TYPES[case["type"]], device="cuda")
    parents = _parents(case)
    drawn = case["draft"] != "none" and most > 1
    drafter = torch.zeros(n, most - 1, vocab, dtype=_TYPES[case["draft"]], device="cuda") if drawn else None
    tokens = torch.full((n, most), -1, dtype=torch.int32, device="cuda")
    temperature = case["temperature"] if case["temperature"] > 0 else 1.0
    for b in range(n):
        # a wide tail and a few likely tokens; a drafter that is right most of the time
        m, lo = int(rows[b]), int(offsets[b])
        x = torch.randn(m, vocab, generator=gen, device="cuda") * 2
        likely = torch.randint(0, vocab, (m, 8), generator=gen, device="cuda")
        x.scatter_(1, likely, math.log(vocab) + 3 - 1.5 * torch.arange(8, device="cuda") + torch.randn(m, 8, generator=gen, device="cuda"))
        logits[lo:lo + m] = x.to(logits.dtype)
        tokens[b, 0] = int(b) % vocab
        if m == 1:
            continue
        guess = x[:most - 1] / temperature + 0.5 * torch.randn(min(m, most - 1), vocab, generator=gen, device="cuda")
        q = torch.softmax(guess, -1)
        if drawn:
            drafter[b, :q.shape[0]] = q.to(drafter.dtype)
            q = drafter[b, :q.shape[0]].float()
        inner = torch.tensor(parents[b, 1:m], device="cuda")
        if drawn:
            tokens[b, 1:m] = torch.multinomial(q[inner], 1, generator=gen).squeeze(1).int()
        else:
            rank = np.array([int((parents[b, 1:i] == parents[b, i]).sum()) for i in range(1, m)])      # the drafter's likeliest tokens, each once
            best = torch.topk(q, min(vocab, most)).indices
            tokens[b, 1:m] = best[inner, torch.tensor(rank, device="cuda")].int()
    heat = torch.full((n,), case["temperature"], dtype=torch.float32, device="cuda")
    if case["tree"] and not drawn:
        heat[4::5] = 0                               # greedy requests among the others
    s.update(logits=logits, tokens=tokens, parents=_dev(parents) if case["tree"] else None, drafter=drafter, row_offsets=_dev(offsets), temperatures=heat,
             uniforms=torch.rand(n, most, generator=gen, device="cuda"))
    s.update(out_tokens=torch.zeros_like(tokens), out_rows=torch.zeros_like(tokens), kept=torch.zeros(n, dtype=torch.int32, device="cuda"),
             logprobs=torch.zeros(n, most, device="cuda"))


def _prepare_keep(case, gen, s):
    rows, lens = _lengths(case)
    path, kept = _path(case)
    page, kv, dim = case["page"], case["kv"], case["dim"]
    per_seq = -(-(rows + lens) // page)
    pages = int(per_seq.sum()) + 3
    table = np.zeros((case["seqs"], int(per_seq.max())), dtype=np.int64)
    order = torch.randperm(pages, generator=gen, device="cuda").cpu().numpy()
    at = 0
    for b, n in enumerate(per_seq):
        table[b, :n] = order[at:at + n]
        at += n
    shape = (pages, kv, page)
    s["layers"] = []
    for _ in range(case["layers"]):
        planes = []
        for _ in range(2):
            planes.append(torch.randint(0, 256, (*shape, dim * case["bits"] // 8), generator=gen, device="cuda", dtype=torch.uint8))
            planes.append((torch.rand(*shape, dim // 64, generator=gen, device="cuda") * 0.02 + 0.005).bfloat16())
            planes.append(torch.randn(*shape, dim // 64, generator=gen, device="cuda").bfloat16())
        s["layers"].append(planes)
    n = int(kept.sum())
    s.update(page_table=_dev(table), context_lengths=_dev(lens), row_offsets=_dev(np.concatenate([[0], np.cumsum(rows)])), path=_dev(path), kept=_dev(kept),
             kept_offsets=_dev(np.concatenate([[0], np.cumsum(kept)])), rows=int(rows.sum()), kept_rows=n)
    s["read"] = [tuple(torch.zeros(n, kv * dim, dtype=torch.float16, device="cuda") for _ in range(2)) for _ in range(case["layers"])]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": case}
    {"plan": _prepare_plan, "verify": _prepare_verify, "keep": _prepare_keep}[case["kind"]](case, gen, s)
    return s


# --- one pass ---

def run(state):
    kind = state["case"]["kind"]
    if kind == "plan":
        (_own_plan if own else _plain_plan)(state)
        names = ["row_offsets", "positions", "sequences", "slots", "page_table", "held_pages", "free_pages", "free_count", "context_lengths"]
        names += ["first_pages"] if state["case"]["window"] else []
        return {k: state[k] for k in names + (["row_tokens", "tree_mask"] if state["case"]["tree"] else [])}
    if kind == "verify":
        (_own_verify if own else _plain_verify)(state)
        return {k: state[k] for k in ("out_tokens", "out_rows", "kept", "logprobs")}
    (_own_keep if own else _plain_keep)(state)
    return state["read"]


def _context():
    from turbo_fieldfare_b200.kernels import TurboContext
    device = torch.cuda.current_device()
    if device not in _kept:                           # one context per device, kept for the program's life as a server keeps it
        _kept[device] = TurboContext(device)
    return _kept[device]


def _own_plan(s):
    from turbo_fieldfare_b200 import drafts as dr
    c, ctx = s["case"], _context()
    if "pages" not in s:                              # descriptors of the caller's buffers, laid out once
        s["pages"] = dr.KVPages(s["page_table"], s["held_pages"], s["free_pages"], s["free_count"], c["page"], first_pages=s["first_pages"])
        s["into"] = dr.KVRows(s["row_offsets"], s["positions"], slots=s["slots"], sequences=s["sequences"], tokens=s["row_tokens"], tree_mask=s["tree_mask"])
    dr.KVPlan(ctx).encode(s["pages"], s["context_lengths"], s["new_rows"], s["into"], window=c["window"], tokens=s["tokens"], parents=s["parents"])


def _own_verify(s):
    from turbo_fieldfare_b200 import drafts as dr
    ctx = _context()
    size = (torch.cuda.current_device(), s["logits"].shape)
    if size not in _kept:                             # the workspace of a server's batch, kept as the context is
        _kept[size] = dr.VerificationWorkspace(ctx, *s["logits"].shape)
    dr.DraftVerification(ctx).encode(s["logits"], s["row_offsets"], s["tokens"], s["uniforms"], s["out_tokens"], s["out_rows"], s["kept"], _kept[size],
                                     parents=s["parents"], draft_probs=s["drafter"], temperatures=s["temperatures"], softcap=s["case"]["cap"], logprobs=s["logprobs"])


def _own_keep(s):
    from turbo_fieldfare_b200 import attention as at
    from turbo_fieldfare_b200 import drafts as dr
    ctx = _context()
    if "caches" not in s:
        s["caches"] = [at.KVCache(*planes) for planes in s["layers"]]
        s["batch"] = at.KVBatch(s["row_offsets"], s["context_lengths"], s["page_table"], rows=s["rows"])
        s["kept_batch"] = at.KVBatch(s["kept_offsets"], s["context_lengths"], s["page_table"], rows=s["kept_rows"])
    dr.KVCacheKeep(ctx).encode(s["caches"], s["batch"], s["path"], s["kept"])
    read = at.KVCacheRead(ctx)
    for cache, (k, v) in zip(s["caches"], s["read"]):
        read.encode(cache, s["kept_batch"], k, v)


def _plain_plan(s):
    c, page = s["case"], s["case"]["page"]
    table, held, count = s["page_table"].long(), s["held_pages"].long(), s["free_count"].long()
    first = s["first_pages"].long() if c["window"] else torch.zeros_like(held)
    free = torch.cat((s["free_pages"].long(), s["free_pages"].new_zeros(1).long()))            # a place more, for what is not wanted
    spare = free.shape[0] - 1
    ends, n = s["new_rows"] < 0, s["new_rows"].long().clamp(min=0)
    ctx = torch.where(ends, 0, s["context_lengths"].long())
    e = torch.arange(table.shape[1], device="cuda")
    # given back: all of a sequence that ends, what no row of the step sees of the others
    fallen = torch.minimum(held, (ctx - c["window"] + 1).clamp(min=0) // page) if c["window"] else torch.zeros_like(held)
    upto = torch.where(ends, held, torch.maximum(first, fallen))
    back = (e >= first[:, None]) & (e < upto[:, None])
    rank = back.flatten().long().cumsum(0).view_as(back) - 1
    released = back.sum()
    free[torch.where(back, count + released - 1 - rank, spare)] = torch.where(back, table, 0)
    table = torch.where(back, -1, table)
    count = count + released
    first, held = torch.where(ends, 0, upto), torch.where(ends, 0, held)
    # taken, in the order of the sequences
    fits = ctx + n <= table.shape[1] * page
    need = torch.where(fits & (n > 0), (-(-(ctx + n) // page) - held).clamp(min=0), 0)
    asked = torch.where(fits, n, 0)
    granted = fits & (need.cumsum(0) <= count) & (asked.cumsum(0) <= s["positions"].shape[0])
    need, n = torch.where(granted, need, 0), torch.where(granted, asked, 0)
    taken = (e >= held[:, None]) & (e < (held + need)[:, None])
    rank = taken.flatten().long().cumsum(0).view_as(taken) - 1
    table = torch.where(taken, free[torch.where(taken, count - 1 - rank, spare)], table)
    count, held = count - taken.sum(), held + need
    s["page_table"].copy_(table), s["held_pages"].copy_(held), s["free_pages"].copy_(free[:-1]), s["free_count"].copy_(count), s["context_lengths"].copy_(ctx)
    if c["window"]:
        s["first_pages"].copy_(first)
    # the rows
    offsets = torch.cat((n.new_zeros(1), n.cumsum(0)))
    s["row_offsets"].copy_(offsets)
    r = torch.arange(s["positions"].shape[0], device="cuda")
    there = r < offsets[-1]
    b = torch.searchsorted(offsets[1:], r, right=True).clamp(max=c["seqs"] - 1)
    i = torch.where(there, r - offsets[b], 0)
    token = ctx[b] + i
    depth = i
    if c["tree"]:
        at, depth = i, torch.zeros_like(i)
        mask = torch.zeros_like(i)
        parents = s["parents"].long()
        for _ in range(s["deepest"] + 1):
            mask = torch.where(at >= 0, mask | (1 << at.clamp(min=0)), mask)
            at = torch.where(at >= 0, parents[b, at.clamp(min=0)], -1)
            depth = depth + (at >= 0)
        s["tree_mask"][:, 0] = torch.where(there, mask, s["tree_mask"][:, 0])
        s["row_tokens"].copy_(torch.where(there, s["tokens"][b, i], s["row_tokens"]))
    s["positions"].copy_(torch.where(there, ctx[b] + depth, s["positions"]))
    s["sequences"].copy_(torch.where(there, b, s["sequences"]))
    s["slots"].copy_(torch.where(there, table[b, (token // page).clamp(max=table.shape[1] - 1)] * page + token % page, s["slots"]))


def _plain_verify(s):
    c, vocab = s["case"], s["case"]["vocab"]
    offsets = s["row_offsets"].long()
    n, every = offsets[1:] - offsets[:-1], torch.arange(c["seqs"], device="cuda")
    greedy = s["temperatures"] <= 0
    heat = torch.where(greedy, 1.0, s["temperatures"]).double()[:, None]
    last = s["logits"].shape[0] - 1

    def weights(node):
        """Weights of the target's distribution behind each sequence's node, and its likeliest token."""
        x = s["logits"][(offsets[:-1] + node).clamp(max=last)].double()          # sums over a vocabulary, borders between its tokens: 64 bits
        if c["cap"]:
            x = c["cap"] * torch.tanh(x / c["cap"])
        x = x.masked_fill(~x.isfinite(), -math.inf)
        top = x.amax(-1, keepdim=True)
        top = torch.where(top == -math.inf, 0.0, top)
        best = torch.where(x == top, torch.arange(vocab, device="cuda"), vocab).amin(-1)
        return ((x - top) / heat).exp(), torch.where(best == vocab, 0, best)

    node, path_at = torch.zeros_like(n), torch.zeros_like(n)
    out_rows, out_tokens = torch.full_like(s["out_rows"], -1).long(), torch.full_like(s["out_tokens"], -1).long()
    out_rows[:, 0] = torch.where(n > 0, 0, -1)
    logprobs = torch.zeros_like(s["logprobs"]).double()
    taken = torch.zeros(c["seqs"], 1, dtype=torch.float64, device="cuda")        # how much of the drafter's row was taken off
    w, best = weights(node)
    gone = torch.zeros_like(w, dtype=torch.bool)

    def rest():
        if s["drafter"] is None:
            return torch.where(gone, 0.0, w)
        q = s["drafter"][every, node.clamp(max=c["rows"] - 2)].double()
        return torch.where(taken > 0, (w - taken * q).clamp(min=0), w)

    for i in range(1, c["rows"]):
        x = s["tokens"][:, i].long()
        at = x.clamp(0, vocab - 1)
        parent = s["parents"][:, i].long() if c["tree"] else i - 1
        asked = (i < n) & (parent == node) & (x >= 0) & (x < vocab)
        r = rest()
        total, chance = r.sum(-1), r[every, at]
        u = s["uniforms"][:, i].double()
        if s["drafter"] is not None:
            u = u * s["drafter"][every, node.clamp(max=c["rows"] - 2), at].double()
        good = asked & torch.where(greedy, x == best, u * total < chance)
        bad = asked & ~good & ~greedy
        if s["drafter"] is None:
            gone[every, at] |= bad
        else:
            taken = torch.where(bad[:, None], taken + total[:, None], taken)
        out_tokens[every, path_at] = torch.where(good, x, out_tokens[every, path_at])
        logprobs[every, path_at] = torch.where(good, (w[every, at] / w.sum(-1)).log(), logprobs[every, path_at])
        path_at = path_at + good
        out_rows[every, path_at] = torch.where(good, i, out_rows[every, path_at])
        node = torch.where(good, i, node)
        taken, gone = torch.where(good[:, None], 0.0, taken), gone & ~good[:, None]
        w, best = weights(node)
    r = rest()
    r = torch.where(r.sum(-1, keepdim=True) > 0, r, w)
    upto = r.cumsum(-1)
    ids = torch.arange(vocab, device="cuda")
    drawn = torch.where(upto > s["uniforms"][:, :1].double() * r.sum(-1, keepdim=True), ids, vocab).amin(-1)
    drawn = torch.where(drawn == vocab, torch.where(r > 0, ids, 0).amax(-1), drawn)
    token = torch.where(greedy, best, drawn)
    out_tokens[every, path_at] = torch.where(n > 0, token, -1)
    logprobs[every, path_at] = torch.where(n > 0, (w[every, token] / w.sum(-1)).log(), 0.0)
    s["logprobs"].copy_(logprobs)
    s["out_tokens"].copy_(out_tokens), s["out_rows"].copy_(out_rows), s["kept"].copy_(torch.where(n > 0, path_at + 1, 0))


def _values(codes, scales, biases, bits):
    if bits == 4:
        codes = torch.stack((codes & 15, codes >> 4), -1).flatten(-2)
    g = codes.float().unflatten(-1, (-1, 64))
    return (g * scales.float().unsqueeze(-1) + biases.float().unsqueeze(-1)).flatten(-2)


def _plain_keep(s):
    c, page = s["case"], s["case"]["page"]
    r = torch.arange(s["kept_rows"], device="cuda")
    b = torch.searchsorted(s["kept_offsets"], r.int(), right=True) - 1
    i = r - s["kept_offsets"][b]
    ctx = s["context_lengths"][b]
    of = lambda token: (s["page_table"][b, token // page].long(), slice(None), token % page)  # noqa: E731
    source, target = of(ctx + s["path"][b, i]), of(ctx + i)
    for planes, (k, v) in zip(s["layers"], s["read"]):
        for plane in planes:
            plane[target] = plane[source]
        k.copy_(_values(planes[0][target], planes[1][target], planes[2][target], c["bits"]).flatten(1))
        v.copy_(_values(planes[3][target], planes[4][target], planes[5][target], c["bits"]).flatten(1))


# --- the definition in 64 bits ---

def exact(case, seed):
    s = prepare(case, seed)
    return {"plan": _exact_plan, "verify": _exact_verify, "keep": _exact_keep}[case["kind"]](case, s)


def _exact_plan(case, s):
    page, n = case["page"], case["seqs"]
    got = {k: (v.cpu().numpy().copy() if v is not None else None) for k, v in s.items() if k != "case" and (v is None or torch.is_tensor(v))}
    table, held, ctx = got["page_table"], got["held_pages"], got["context_lengths"]
    first = got["first_pages"] if case["window"] else np.zeros_like(held)
    stack = got["free_pages"][:int(got["free_count"][0])].tolist()
    back = []
    for b in range(n):
        if got["new_rows"][b] < 0:
            lo, hi = first[b], held[b]
            first[b] = held[b] = ctx[b] = 0
        else:
            lo, hi = first[b], min(held[b], max(0, ctx[b] - case["window"] + 1) // page) if case["window"] else first[b]
            first[b] = max(lo, hi)
        for e in range(lo, hi):
            back.append(int(table[b, e]))
            table[b, e] = -1
    stack += back[::-1]
    free, total, waiting = got["free_pages"], 0, False
    free[:len(stack)] = stack
    for b in range(n):
        m = max(0, int(got["new_rows"][b]))
        got["row_offsets"][b] = total
        last = int(ctx[b]) + m
        if m == 0 or last > table.shape[1] * page:
            continue
        need = max(0, -(-last // page) - int(held[b]))
        waiting = waiting or need > len(stack) or total + m > len(got["positions"])
        if waiting:
            continue
        for _ in range(need):
            table[b, held[b]] = stack.pop()
            held[b] += 1
        for i in range(m):
            r, token = total + i, int(ctx[b]) + i
            got["sequences"][r], got["positions"][r], got["slots"][r] = b, token, int(table[b, token // page]) * page + token % page
            if case["tree"]:
                p = int(got["parents"][b, i])
                up = 0 if p < 0 else int(got["tree_mask"][total + p, 0])
                got["tree_mask"][r, 0] = np.array(up | 1 << i, dtype=np.uint64).astype(np.int64)
                got["positions"][r] = ctx[b] if p < 0 else got["positions"][total + p] + 1
                got["row_tokens"][r] = got["tokens"][b, i]
        total += m
    got["row_offsets"][n] = total
    got["free_count"][0] = len(stack)
    return {k: torch.tensor(got[k], device="cuda") for k in ["row_offsets", "positions", "sequences", "slots", "page_table", "held_pages", "free_pages", "free_count", "context_lengths"] +
            (["first_pages"] if case["window"] else []) + (["row_tokens", "tree_mask"] if case["tree"] else [])}


def _exact_verify(case, s):
    offsets, vocab = s["row_offsets"].tolist(), case["vocab"]
    tokens, u, heat = s["tokens"].tolist(), s["uniforms"].double().tolist(), s["temperatures"].double().tolist()
    parents = _parents(case).tolist()
    out_tokens, out_rows, kept = (np.full((case["seqs"], case["rows"]), -1), np.full((case["seqs"], case["rows"]), -1), np.zeros(case["seqs"]))
    logprobs = np.zeros((case["seqs"], case["rows"]))
    for b in range(case["seqs"]):
        n = offsets[b + 1] - offsets[b]
        if n == 0:
            continue

        def target(node):
            x = s["logits"][offsets[b] + node].double()
            if case["cap"]:
                x = torch.tanh(x / case["cap"]) * case["cap"]
            if heat[b] <= 0:
                return (x == x.max()).double(), torch.log_softmax(x, 0)
            return torch.softmax(x / heat[b], 0), torch.log_softmax(x / heat[b], 0)

        node, accepted, (p, log) = 0, [], target(0)
        q = s["drafter"][b, 0].double() if s["drafter"] is not None else None
        for i in range(1, n):
            if parents[b][i] != node:
                continue
            x = tokens[b][i]
            if heat[b] <= 0:
                good = int(p.argmax()) == x if int((p > 0).sum()) == 1 else int(torch.nonzero(p)[0]) == x
            else:
                good = u[b][i] * (float(q[x]) if q is not None else 1.0) < float(p[x])
            if good:
                logprobs[b, len(accepted)] = float(log[x])
                node, (p, log) = i, target(i)
                q = s["drafter"][b, i].double() if s["drafter"] is not None and i < case["rows"] - 1 else None
                accepted.append(i)
            elif heat[b] > 0:
                before = p
                if q is not None:
                    p = (p - q).clamp(min=0)
                else:
                    p = p.clone()
                    p[x] = 0
                p = p / p.sum() if float(p.sum()) > 0 else before
        if heat[b] <= 0:
            token = int(torch.nonzero(p)[0])
        else:
            upto = p.cumsum(0)
            token = min(int(torch.searchsorted(upto, torch.tensor([u[b][0] * float(upto[-1])], dtype=torch.float64, device="cuda"), right=True)), int(torch.nonzero(p)[-1]))
        kept[b] = len(accepted) + 1
        logprobs[b, len(accepted)] = float(log[token])
        out_rows[b, :len(accepted) + 1] = [0] + accepted
        out_tokens[b, :len(accepted) + 1] = [tokens[b][i] for i in accepted] + [token]
    return {"out_tokens": _dev(out_tokens), "out_rows": _dev(out_rows), "kept": _dev(kept), "logprobs": _dev(logprobs, torch.float64)}


def _exact_keep(case, s):
    path, kept = _path(case)
    table, ctx, page = s["page_table"].cpu().numpy(), s["context_lengths"].cpu().numpy(), case["page"]
    where = [(table[b, t // page], t % page) for b in range(case["seqs"]) for t in ctx[b] + path[b, :int(kept[b])]]
    pages, at = (torch.tensor([int(w[i]) for w in where], device="cuda") for i in (0, 1))
    outs = []
    for planes in s["layers"]:
        pair = []
        for i in (0, 3):
            codes, scales, biases = (p[pages, :, at] for p in planes[i:i + 3])
            if case["bits"] == 4:
                codes = torch.stack((codes % 16, codes // 16), -1).flatten(-2)
            wide = lambda p: p.double().repeat_interleave(64, -1)  # noqa: E731
            pair.append((codes.double() * wide(scales) + wide(biases)).flatten(1))
        outs.append(tuple(pair))
    return outs
