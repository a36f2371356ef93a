"""The attention operators of a decoded or prefilled layer over a quantised, paged cache, as cases with inputs, one pass,
a plain form and a 64-bit definition.

  append   what follows the QKV projection of a layer: per-head norms of q, k and v, rotation of q and k, k and v quantised into
           the cache; the stored rows are then read back, which is how the pass shows what it stored
  read     the cache's rows of some sequences back as 16-bit rows
  attend   attention of the newest tokens of every sequence (one token, a tree of drafted ones, a chunk of a prompt) over the
           cache, which holds them already

Head counts, head sizes and the window of 1024 are those of the layers that this framework's expert blocks belong to (16 query
heads of 256 over 8, or of 512 over 2), beside common ones (32 heads of 128 over 8, 64-wide heads). Lengths run from one token to long contexts.
"""
import math

import numpy as np
import torch

own = False
_kept = {}


def listed():
    return [
        # a single chat user: the smallest call, latency only
        {"name": "append_1", "kind": "append", "seqs": 1, "rows": 1, "ctx": 700, "heads": 16, "kv": 8, "dim": 256, "bits": 8, "page": 64, "type": "f16", "rot": 128},
        # trees of drafted tokens of a batch, full-attention layers with partly rotated heads, 4-bit cache
        {"name": "append_tree", "kind": "append", "seqs": 37, "rows": 13, "ctx": 9000, "heads": 16, "kv": 2, "dim": 512, "bits": 4, "page": 64, "type": "bf16", "rot": 64},
        # the benchmark's prompt block
        {"name": "append_4096", "kind": "append", "seqs": 1, "rows": 4096, "ctx": 0, "heads": 16, "kv": 8, "dim": 256, "bits": 8, "page": 64, "type": "f16", "rot": 128},
        # a short prefix of a few sequences, handed to another attention
        {"name": "read_short", "kind": "read", "seqs": 3, "ctx": 777, "kv": 8, "dim": 128, "bits": 4, "page": 16, "type": "f16"},
        # a long context read back whole
        {"name": "read_65536", "kind": "read", "seqs": 1, "ctx": 65536, "kv": 8, "dim": 256, "bits": 8, "page": 64, "type": "bf16"},
        # one token of one user in a layer with a window
        {"name": "decode_1", "kind": "attend", "seqs": 1, "rows": 1, "ctx": 2500, "heads": 16, "kv": 8, "dim": 256, "bits": 8, "page": 64, "type": "f16", "window": 1024, "tree": False},
        # the benchmark's batched decode, ragged contexts
        {"name": "decode_64", "kind": "attend", "seqs": 64, "rows": 1, "ctx": 4096, "heads": 16, "kv": 8, "dim": 256, "bits": 8, "page": 64, "type": "f16", "window": 0, "tree": False},
        # a busy server's decode batch in a full-attention layer, 4-bit cache
        {"name": "decode_200", "kind": "attend", "seqs": 200, "rows": 1, "ctx": 8192, "heads": 16, "kv": 2, "dim": 512, "bits": 4, "page": 64, "type": "f16", "window": 0, "tree": False},
        # one user with a long document
        {"name": "decode_long", "kind": "attend", "seqs": 1, "rows": 1, "ctx": 131000, "heads": 32, "kv": 8, "dim": 128, "bits": 8, "page": 64, "type": "bf16", "window": 0, "tree": False},
        # small trees of drafted tokens, small pages
        {"name": "tree_32x7", "kind": "attend", "seqs": 32, "rows": 7, "ctx": 3000, "heads": 32, "kv": 8, "dim": 128, "bits": 4, "page": 16, "type": "bf16", "window": 0, "tree": True},
        # wide trees of drafted tokens
        {"name": "tree_8x61", "kind": "attend", "seqs": 8, "rows": 61, "ctx": 8000, "heads": 16, "kv": 8, "dim": 256, "bits": 8, "page": 64, "type": "f16", "window": 0, "tree": True},
        # a chunk of a long prompt
        {"name": "chunk_333", "kind": "attend", "seqs": 1, "rows": 333, "ctx": 8000, "heads": 16, "kv": 8, "dim": 256, "bits": 8, "page": 64, "type": "f16", "window": 0, "tree": False},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "append", "read", "attend", "attend", "attend", "attend"])
    heads, kv, dim = rng.choice([(16, 8, 256), (16, 8, 256), (16, 2, 512), (32, 8, 128), (24, 4, 128), (8, 8, 64), (7, 1, 64)])
    c = {"kind": kind, "heads": heads, "kv": kv, "dim": dim, "bits": rng.choice([8, 8, 4]), "page": rng.choice([16, 32, 64, 64, 128]), "type": rng.choice(["f16", "bf16"])}
    if kind == "append":
        c.update(seqs=_log_int(rng, 1, 100), rot=rng.choice([dim // 2, dim // 8]))
        c.update(rows=_log_int(rng, 1, max(1, 4000 // c["seqs"])), ctx=_log_int(rng, 1, 20000))
    elif kind == "read":
        c.update(seqs=_log_int(rng, 1, 60))
        c.update(ctx=_log_int(rng, 1, max(1, 60000 * 2048 // (kv * dim) // c["seqs"])))
        del c["heads"]
    else:
        shape = rng.choice(["one", "one", "tree", "tree", "chunk"])
        tokens = int(1.2e9 / (kv * dim))
        if shape == "chunk":
            c.update(seqs=_log_int(rng, 1, 4), rows=_log_int(rng, 8, 300), ctx=_log_int(rng, 1, 6000))
        else:
            c.update(seqs=_log_int(rng, 1, 120), rows=1 if shape == "one" else _log_int(rng, 2, 64))
            c.update(ctx=_log_int(rng, 1, max(1, min(100000, tokens // c["seqs"] // (1 if shape == "one" else 4)))))
            if shape == "tree":
                c["seqs"] = min(c["seqs"], 40)
        c.update(window=rng.choice([0, 0, 0, 1024, 100]), tree=shape == "tree")
    return c


# --- what a case fixes, whatever the seed: lengths and the shape of the trees ---

def _lengths(case):
    """(rows, context) of every sequence: ragged, the first one with the full numbers, some contexts short."""
    r = np.random.RandomState(1 + case["seqs"] * 7919 + case["ctx"])
    n, ctx = case["seqs"], case["ctx"]
    rows = np.full(n, case.get("rows", 0), dtype=np.int64)
    lens = np.full(n, ctx, dtype=np.int64)
    if n > 1:
        lens[1:] = np.ceil(ctx * r.uniform(0.1, 1.0, n - 1)).astype(np.int64)
        if case.get("rows", 0) > 1:
            rows[1:] = r.randint(max(1, case["rows"] // 2), case["rows"] + 1, n - 1)
    return rows, lens


def _tree(case):
    """Ancestor table of the drafted tokens and their depths, per sequence: token i hangs under a random earlier one."""
    rows, _ = _lengths(case)
    r = np.random.RandomState(case["rows"] + 31 * case["seqs"])
    out = []
    for n in rows:
        seen, depth = np.zeros((n, n), dtype=bool), np.zeros(n, dtype=np.int64)
        for i in range(n):
            if i:
                p = r.randint(max(0, i - 8), i)
                seen[i] = seen[p]
                depth[i] = depth[p] + 1
            seen[i, i] = True
        out.append((seen, depth))
    return out


def _visible(case):
    """Per sequence (cached tokens that any row sees, (row, token) pairs)."""
    rows, lens = _lengths(case)
    trees = _tree(case) if case["tree"] else None
    got = []
    for b, (n, ctx) in enumerate(zip(rows.tolist(), lens.tolist())):
        depth = trees[b][1] if trees else np.arange(n)
        w = case["window"]
        low = np.maximum(0, ctx + depth - w + 1) if w else np.zeros(n, dtype=np.int64)
        drafted = trees[b][0].sum(1) if trees else (np.minimum(np.arange(n) + 1, w) if w else np.arange(n) + 1)
        got.append((ctx - min(ctx, int(low.min())) + n, int(np.maximum(0, ctx - low).sum() + drafted.sum())))
    return got


def _token_bytes(case):
    return 2 * case["kv"] * (case["dim"] * case["bits"] // 8 + case["dim"] // 64 * 4)


def work(case):
    rows, lens = _lengths(case)
    row = case["dim"] * 2
    if case["kind"] == "append":
        n = int(rows.sum())
        stored = n * _token_bytes(case)
        # q, k and v rows in, q rows out, the cache's rows written, and the same rows read back as 16-bit ones
        return {"bytes": n * row * (2 * case["heads"] + 2 * case["kv"]) + 2 * stored + n * 2 * case["kv"] * row, "flops": n * row * 6 * (case["heads"] + 2 * case["kv"])}
    if case["kind"] == "read":
        n = int(lens.sum())
        return {"bytes": n * (_token_bytes(case) + 2 * case["kv"] * row), "flops": n * case["kv"] * row * 2}
    seen = _visible(case)
    n = int(rows.sum())
    return {"bytes": sum(t for t, _ in seen) * _token_bytes(case) + 2 * n * case["heads"] * row, "flops": 4 * case["dim"] * case["heads"] * sum(p for _, p in seen)}


# --- inputs ---

def _type(case):
    return torch.float16 if case["type"] == "f16" else torch.bfloat16


def _quantised(x, bits):
    """(codes as bytes, scales, biases) of rows in groups of 64: w = code * scale + bias, both planes bfloat16."""
    g = x.unflatten(-1, (-1, 64))
    low, high = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    top = 2 ** bits - 1
    scale = torch.where(high == low, torch.ones_like(low), (high - low) / top).bfloat16()
    bias = low.bfloat16()
    s, o = scale.to(x.dtype), bias.to(x.dtype)
    code = torch.clamp(torch.floor((g - o) / s + 0.5), 0, top).to(torch.uint8).flatten(-2)
    if bits == 4:
        code = code[..., 0::2] | (code[..., 1::2] << 4)
    return code, scale.squeeze(-1), bias.squeeze(-1)


def _values(codes, scales, biases, bits, dtype=torch.float32):
    """The values that quantised rows stand for."""
    if bits == 4:
        codes = torch.stack((codes & 15, codes >> 4), -1).flatten(-2)
    g = codes.to(dtype).unflatten(-1, (-1, 64))
    return (g * scales.to(dtype).unsqueeze(-1) + biases.to(dtype).unsqueeze(-1)).flatten(-2)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *shape: torch.randn(*shape, generator=gen, device="cuda")  # noqa: E731
    dev = lambda a, t=torch.int32: torch.tensor(np.ascontiguousarray(a), dtype=t, device="cuda")  # noqa: E731
    dt, kv, dim, bits, page = _type(case), case["kv"], case["dim"], case["bits"], case["page"]
    rows, lens = _lengths(case)
    per_seq = -(-(rows + lens) // page)
    pages = int(per_seq.sum()) + 3
    table = np.zeros((case["seqs"], int(per_seq.max())), dtype=np.int32)
    order = torch.randperm(pages, generator=gen, device="cuda").cpu().numpy()
    at = 0
    for b, n in enumerate(per_seq):
        table[b, :n] = order[at:at + n]
        at += n
    shape = (pages, kv, page)
    if case["kind"] == "append":
        half = lambda: torch.zeros(*shape, dim // 64, dtype=torch.bfloat16, device="cuda")  # noqa: E731
        code = lambda: torch.zeros(*shape, dim * bits // 8, dtype=torch.uint8, device="cuda")  # noqa: E731
        planes = [code(), half(), half(), code(), half(), half()]
    else:
        # normed keys and values; a few channels of a key are larger than the others
        gain = 1 + 2 * (torch.arange(dim, device="cuda") % 61 == 0)
        planes = [*_quantised(rand(*shape, dim) * gain, bits), *_quantised(rand(*shape, dim), bits)]
    read = case["kind"] == "read"
    held = lens if read else rows        # a read takes the whole prefix, the others the rows behind the context
    first = np.zeros_like(lens) if read else lens
    s = {"case": case, "planes": planes, "page_table": dev(table), "context_lengths": dev(first),
         "row_offsets": dev(np.concatenate([[0], np.cumsum(held)])), "rows": int(held.sum()), "most_rows": int(held.max()), "pages_seen": table.shape[1]}
    n = s["rows"]
    if read:
        s["k_out"], s["v_out"] = torch.zeros(n, kv * dim, dtype=dt, device="cuda"), torch.zeros(n, kv * dim, dtype=dt, device="cuda")
        return s
    heads = case["heads"]
    if case["kind"] == "append":
        # one row of the projection holds q, k and v side by side
        s["qkv"] = (rand(n, (heads + 2 * kv) * dim) * (0.5 + torch.rand(n, 1, generator=gen, device="cuda"))).to(dt)
        s["q_weight"], s["k_weight"] = ((1 + 0.1 * rand(dim)).bfloat16() for _ in range(2))
        s["frequencies"] = (1e6 ** (-torch.arange(case["rot"], device="cuda", dtype=torch.float64) / case["rot"])).float()
        s["positions"] = dev(np.concatenate([c + np.arange(m) for c, m in zip(lens, rows)]))
        s["q_out"] = torch.zeros(n, heads * dim, dtype=dt, device="cuda")
        s["k_out"], s["v_out"] = torch.zeros(n, kv * dim, dtype=dt, device="cuda"), torch.zeros(n, kv * dim, dtype=dt, device="cuda")
        return s
    s["q"] = (2 * rand(n, heads * dim)).to(dt)
    s["out"] = torch.zeros(n, heads * dim, dtype=dt, device="cuda")
    s["positions"], s["tree_mask"] = None, None
    if case["tree"]:
        trees = _tree(case)
        words = np.zeros((n, 1), dtype=np.uint64)
        words[:, 0] = [sum(1 << int(j) for j in np.flatnonzero(row)) for seen, _ in trees for row in seen]
        s["tree_mask"] = dev(words.view(np.int64), torch.int64)
        s["positions"] = dev(np.concatenate([c + d for c, (_, d) in zip(lens, trees)]))
    return s


# --- one pass ---

def run(state):
    return _own_run(state) if own else _plain_run(state)


def _own_run(s):
    from turbo_fieldfare_b200 import attention as at
    from turbo_fieldfare_b200.kernels import TurboContext
    c, device = s["case"], torch.cuda.current_device()
    if device not in _kept:                       # one context per device, kept for the program's life as a server keeps it
        _kept[device] = TurboContext(device)
    ctx = _kept[device]
    if "cache" not in s:                          # descriptors of the caller's buffers, laid out once per sequence batch
        s["cache"] = at.KVCache(*s["planes"])
        s["batch"] = at.KVBatch(s["row_offsets"], s["context_lengths"], s["page_table"], s.get("positions"))
    if c["kind"] == "read":
        at.KVCacheRead(ctx).encode(s["cache"], s["batch"], s["k_out"], s["v_out"])
        return s["k_out"], s["v_out"]
    if c["kind"] == "append":
        hq, hk = c["heads"] * c["dim"], c["kv"] * c["dim"]
        q, k, v = s["qkv"][:, :hq], s["qkv"][:, hq:hq + hk], s["qkv"][:, hq + hk:]
        at.FusedQKVEpilogue(ctx).encode(q, k, v, s["q_out"], s["batch"], s["cache"], head_dim=c["dim"], q_weight=s["q_weight"],
                                        k_weight=s["k_weight"], norm_v=True, frequencies=s["frequencies"], eps=1e-6)
        at.KVCacheRead(ctx).encode(s["cache"], s["batch"], s["k_out"], s["v_out"])
        return s["q_out"], s["k_out"], s["v_out"]
    if (device, c["dim"]) not in _kept:           # the workspace of a head size, kept as the context is
        _kept[device, c["dim"]] = at.AttentionWorkspace(ctx, c["dim"])
    at.TreeAttention(ctx).encode(s["q"], s["out"], s["cache"], s["batch"], _kept[device, c["dim"]], scale=c["dim"] ** -0.5,
                                 window=c["window"], tree_mask=s["tree_mask"])
    return s["out"]


def _rows_of(s):
    """(sequence, token) of every row."""
    r = torch.arange(s["rows"], device="cuda")
    seq = torch.searchsorted(s["row_offsets"], r.int(), right=True) - 1
    return seq, r - s["row_offsets"][seq] + s["context_lengths"][seq]


def _plain_run(s):
    c = s["case"]
    dt, kv, dim, bits, page = _type(c), c["kv"], c["dim"], c["bits"], c["page"]
    seq, token = _rows_of(s)
    if c["kind"] != "attend":
        where = s["page_table"][seq, token // page].long(), slice(None), token % page
    if c["kind"] == "append":
        hq, hk = c["heads"] * dim, kv * dim
        x = s["qkv"].float()
        q, k, v = (t.unflatten(-1, (-1, dim)) for t in (x[:, :hq], x[:, hq:hq + hk], x[:, hq + hk:]))
        normed = lambda t: t * torch.rsqrt(t.square().mean(-1, keepdim=True) + 1e-6)  # noqa: E731
        q, k, v = normed(q) * s["q_weight"].float(), normed(k) * s["k_weight"].float(), normed(v)
        angle = s["positions"].double()[:, None, None] * s["frequencies"].double()     # far positions need 64 bits
        cos, sin, half = angle.cos().float(), angle.sin().float(), c["rot"]

        def rotated(t):
            a, b = t[..., :half], t[..., half:2 * half]
            return torch.cat((a * cos - b * sin, b * cos + a * sin, t[..., 2 * half:]), -1)

        s["q_out"].copy_(rotated(q).flatten(1))
        for plane, new in zip(s["planes"], (*_quantised(rotated(k), bits), *_quantised(v, bits))):
            plane[where] = new
    if c["kind"] != "attend":
        p = s["planes"]
        s["k_out"].copy_(_values(p[0][where], p[1][where], p[2][where], bits).flatten(1))
        s["v_out"].copy_(_values(p[3][where], p[4][where], p[5][where], bits).flatten(1))
        return (s["q_out"], s["k_out"], s["v_out"]) if c["kind"] == "append" else (s["k_out"], s["v_out"])
    most, group = s["most_rows"], c["heads"] // kv
    table = s["page_table"][:, :s["pages_seen"]].long()
    k, v = (_values(*(p[table].transpose(1, 2).flatten(2, 3) for p in s["planes"][i:i + 3]), bits) for i in (0, 3))   # [seqs, kv, tokens, dim]
    at = s["row_offsets"][:-1, None] + torch.arange(most, device="cuda")                # [seqs, most], beyond a sequence's own: clamped
    there = at < s["row_offsets"][1:, None]
    at = at.clamp(max=s["rows"] - 1)
    q = s["q"].float()[at].unflatten(-1, (kv, group, dim)).permute(0, 2, 1, 3, 4).flatten(2, 3)                      # [seqs, kv, most * group, dim]
    ctx = s["context_lengths"][:, None, None]
    j = torch.arange(k.shape[2], device="cuda")[None, None]
    i = torch.arange(most, device="cuda")[None, :, None]
    if c["tree"]:
        bit = (s["tree_mask"][at][..., 0, None] >> (j - ctx).clamp(0, 63)) & 1
        drafted, position = (bit == 1) & (j - ctx < 64), s["positions"][at][..., None]
    else:
        drafted, position = j - ctx <= i, ctx + i
        if c["window"]:
            drafted = drafted & (position - j < c["window"])
    cached = position - j < c["window"] if c["window"] else torch.ones_like(drafted)
    seen = torch.where(j < ctx, cached, drafted) & there[..., None]                     # [seqs, most, tokens]
    logits = (q @ k.transpose(2, 3) * dim ** -0.5).unflatten(2, (most, group)).masked_fill(~seen[:, None, :, None], -math.inf)
    e = (logits - logits.amax(-1, keepdim=True).clamp(min=-1e30)).exp()
    p = (e / e.sum(-1, keepdim=True).clamp(min=1e-30)).flatten(2, 3)
    o = (p @ v).unflatten(2, (most, group)).permute(0, 2, 1, 3, 4).flatten(2)           # [seqs, most, heads * dim]
    s["out"].copy_(o[there])
    return s["out"]


# --- the definition in 64 bits ---

def exact(case, seed):
    s = prepare(case, seed)
    kv, dim, bits, page = case["kv"], case["dim"], case["bits"], case["page"]
    offsets, firsts, table = s["row_offsets"].tolist(), s["context_lengths"].tolist(), s["page_table"].long()
    f64 = torch.float64

    def stored(b, lo, hi, first_plane):
        t = torch.arange(lo, hi, device="cuda")
        codes, scales, biases = (p[table[b, t // page], :, t % page] for p in s["planes"][first_plane:first_plane + 3])
        if bits == 4:
            both = torch.empty(*codes.shape[:-1], dim, dtype=f64, device="cuda")
            both[..., 0::2], both[..., 1::2] = (codes % 16).to(f64), (codes // 16).to(f64)
        else:
            both = codes.to(f64)
        wide = lambda plane: plane.to(f64).repeat_interleave(64, -1)  # noqa: E731
        return both * wide(scales) + wide(biases)                    # [tokens, kv, dim]

    if case["kind"] == "read":
        return tuple(torch.cat([stored(b, 0, offsets[b + 1] - offsets[b], i).flatten(1) for b in range(case["seqs"])]) for i in (0, 3))
    if case["kind"] == "append":
        n, heads, half = s["rows"], case["heads"], case["rot"]
        x = s["qkv"].to(f64).view(n, heads + 2 * kv, dim)
        x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / dim + 1e-6)
        x[:, :heads] *= s["q_weight"].to(f64)
        x[:, heads:heads + kv] *= s["k_weight"].to(f64)
        turn = torch.polar(torch.ones(n, half, dtype=f64, device="cuda"), torch.outer(s["positions"].to(f64), s["frequencies"].to(f64)))
        z = torch.complex(x[:, :heads + kv, :half].contiguous(), x[:, :heads + kv, half:2 * half].contiguous()) * turn[:, None]
        x[:, :heads + kv, :half], x[:, :heads + kv, half:2 * half] = z.real, z.imag
        g = x[:, heads:].reshape(n, 2 * kv, dim // 64, 64)
        low, high = g.min(-1, keepdim=True).values, g.max(-1, keepdim=True).values
        step = ((high - low) / (2 ** bits - 1)).bfloat16().to(f64)
        step[high == low] = 1
        low = low.bfloat16().to(f64)
        held = ((g - low) / step + 0.5).floor().clamp(0, 2 ** bits - 1) * step + low
        held = held.reshape(n, 2 * kv, dim)
        return x[:, :heads].flatten(1), held[:, :kv].flatten(1), held[:, kv:].flatten(1)
    trees = _tree(case) if case["tree"] else None
    outs = []
    for b in range(case["seqs"]):
        n, ctx = offsets[b + 1] - offsets[b], firsts[b]
        k, v = stored(b, 0, ctx + n, 0).transpose(0, 1), stored(b, 0, ctx + n, 3).transpose(0, 1)
        q = s["q"][offsets[b]:offsets[b + 1]].to(f64).view(n, kv, -1, dim).permute(1, 2, 0, 3)       # [kv, group, n, dim]
        depth = trees[b][1] if trees else np.arange(n)
        seen = np.ones((n, ctx + n), dtype=bool)
        seen[:, ctx:] = trees[b][0] if trees else np.tril(np.ones((n, n), dtype=bool))
        if case["window"]:
            inside = (ctx + depth)[:, None] - np.arange(ctx + n)[None] < case["window"]
            if trees:
                inside[:, ctx:] = True                               # among drafted tokens the mask says it all
            seen &= inside
        bias = torch.zeros(n, ctx + n, dtype=f64, device="cuda").masked_fill_(~torch.tensor(seen, device="cuda"), -math.inf)
        p = torch.softmax(q @ k[:, None].transpose(2, 3) / math.sqrt(dim) + bias, -1)
        outs.append((p @ v[:, None]).permute(2, 0, 1, 3).reshape(n, -1))
    return torch.cat(outs)
