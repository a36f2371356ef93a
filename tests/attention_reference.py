"""Plain 64-bit statements of the attention operators for their tests (test infrastructure only)."""
import torch

F64 = torch.float64


def unpack(codes, bits):
    if bits == 4:
        codes = torch.stack((codes & 15, codes >> 4), -1).flatten(-2)
    return codes.to(F64)


def quantised(x, bits):
    """Codes and planes of rows in groups of 64 (the affine format of the weights)."""
    g = x.to(torch.float32).unflatten(-1, (-1, 64))
    low, high = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    top = 2 ** bits - 1
    scale = torch.where(high == low, torch.ones_like(low), (high - low) / top).bfloat16()
    bias = low.bfloat16()
    code = torch.clamp(torch.floor((g - bias.float()) / scale.float() + 0.5), 0, top).to(torch.uint8).flatten(-2)
    if bits == 4:
        code = code[..., 0::2] | (code[..., 1::2] << 4)
    return code, scale.squeeze(-1), bias.squeeze(-1)


class Case:
    """A batch over a paged cache: pages in random order, everything that no sequence owns filled with NaN planes and codes of ones."""

    def __init__(self, seed, rows, contexts, kv_heads, dim, bits, page_size, device, extra_pages=2, value_scale=1.0):
        gen = torch.Generator().manual_seed(seed)
        self.rows, self.contexts, self.kv, self.dim, self.bits, self.page = list(rows), list(contexts), kv_heads, dim, bits, page_size
        need = [max(1, -(-(r + c) // page_size)) for r, c in zip(rows, contexts)]
        pages = sum(need) + extra_pages
        order = torch.randperm(pages, generator=gen).tolist()
        table = torch.full((len(need), max(need)), -1, dtype=torch.int32)
        at = 0
        for b, n in enumerate(need):
            table[b, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
            at += n
        shape = (pages, kv_heads, page_size)
        self.planes = []
        for _ in range(2):
            self.planes += [torch.full((*shape, dim * bits // 8), 255, dtype=torch.uint8), torch.full((*shape, dim // 64), float("nan"), dtype=torch.bfloat16),
                            torch.full((*shape, dim // 64), float("nan"), dtype=torch.bfloat16)]
        for b, (r, c) in enumerate(zip(rows, contexts)):
            t = torch.arange(r + c)
            where = table[b, t // page_size].long(), slice(None), t % page_size
            for i, mul in ((0, 1.0), (3, value_scale)):
                x = torch.randn(r + c, kv_heads, dim, generator=gen) * mul + 0.3 * mul
                for plane, new in zip(self.planes[i:i + 3], quantised(x, bits)):
                    plane[where] = new
        self.table = table
        self.gen, self.device = gen, device

    @classmethod
    def of_cache(cls, cache, table, rows, contexts):
        """The rows behind some contexts of a cache that the library has written."""
        case = cls.__new__(cls)
        case.rows, case.contexts, case.kv, case.dim, case.bits, case.page = list(rows), list(contexts), cache.kv_heads, cache.head_dim, cache.bits, cache.page_size
        case.planes, case.table = [p.cpu() for p in cache.planes], table.cpu()
        case.offsets = [0]
        for r in rows:
            case.offsets.append(case.offsets[-1] + r)
        return case

    def upload(self):
        from turbo_fieldfare_b200 import attention as at
        dev = lambda t: t.to(self.device)  # noqa: E731
        self.cache = at.KVCache(*[dev(p) for p in self.planes])
        offsets = [0]
        for r in self.rows:
            offsets.append(offsets[-1] + r)
        self.offsets = offsets
        return self

    crowd = 0          # sequences without rows behind the others: a mean sequence has few rows then, which another kernel takes

    def batch(self, positions=None, rows=None, contexts=None):
        from turbo_fieldfare_b200 import attention as at
        i32 = dict(dtype=torch.int32, device=self.device)
        contexts = list(self.contexts if contexts is None else contexts) + [0] * self.crowd
        table = torch.cat([self.table, torch.full((self.crowd, self.table.shape[1]), -1, dtype=torch.int32)])
        return at.KVBatch(torch.tensor(self.offsets + self.offsets[-1:] * self.crowd, **i32), torch.tensor(contexts, **i32), table.to(self.device),
                          None if positions is None else torch.as_tensor(positions, **i32), rows=self.offsets[-1] if rows is None else rows)

    def stored(self, b, first):
        """(codes, scales, biases) in 64 bits of sequence b's tokens, planes `first` on: [tokens, kv, dim]."""
        t = torch.arange(self.rows[b] + self.contexts[b])
        codes, scales, biases = (p[self.table[b, t // self.page].long(), :, t % self.page] for p in self.planes[first:first + 3])
        wide = lambda p: p.to(F64).repeat_interleave(64, -1)  # noqa: E731
        return unpack(codes, self.bits), wide(scales), wide(biases)


def visible(rows, context, window=0, masks=None, positions=None):
    """[rows, context + rows] truth table of one sequence; masks: list of sets of seen rows."""
    see = torch.zeros(rows, context + rows, dtype=torch.bool)
    for i in range(rows):
        p = context + i if masks is None else max(int(positions[i]), context) if positions is not None else context
        see[i, :context] = True if not window else p - torch.arange(context) < window
        if masks is None:
            see[i, context:context + i + 1] = True if not window else i - torch.arange(i + 1) < window
        else:
            for j in masks[i]:
                see[i, context + j] = True
    return see


def attention(case, q, see, scale, out_half_step):
    """(expected, tolerance) of [rows, heads * dim] 16-bit rows q (CPU), see: a truth table per sequence.

    Tolerance, element by element, from the roundings that the kernels name (half steps 2^-11 of fp16): probabilities twice (product and sum),
    values once and what a bias, centred, adds once, the output; logits in fp32: products of a group in 4 steps, groups, factor, together under
    2^-17 of sum |q||k|; probabilities below fp16's least step count as zero (2^-25 each, against a sum of at least one). With many rows a key is
    rounded to fp16 too and nothing is centred: each element moves the logit by up to 2^-12 |q_d k_d| scale, with a sign of its own, together
    about 2^-12 sqrt(sum (q_d k_d)^2) scale, which is 2^-12 for logits of size one: the share of the centred bias and of a second rounding of the
    probabilities, which that kernel does not have, holds it."""
    want, tol = [], []
    centre = 128.0 if case.bits == 8 else 8.0
    for b, n in enumerate(case.rows):
        o0 = case.offsets[b]
        if n == 0:
            continue
        kc, ks, ko = case.stored(b, 0)
        vc, vs, vo = case.stored(b, 3)
        qb = q[o0:o0 + n].to(F64).reshape(n, case.kv, -1, case.dim)
        t = torch.einsum
        logits = t("nhgd,jhd->hgnj", qb, kc * ks + ko) * scale
        spread = t("nhgd,jhd->hgnj", qb.abs(), kc * ks.abs() + ko.abs()) * abs(scale)
        s = see[b][None, None]
        logits = logits.masked_fill(~s, -float("inf"))
        top = logits.amax(-1, keepdim=True)
        top = torch.where(torch.isinf(top), torch.zeros_like(top), top)
        e = (logits - top).exp()
        p = e / e.sum(-1, keepdim=True).clamp(min=1e-300)
        v = vc * vs + vo
        out = t("hgnj,jhd->nhgd", p, v)
        a = t("hgnj,jhd->nhgd", p, v.abs())
        centred = t("hgnj,jhd->nhgd", p, (vo + centre * vs).abs())
        worst = spread.masked_fill(~s, 0.0).amax(-1).permute(2, 0, 1)[..., None]
        seen = see[b].sum(-1).to(F64)[:, None, None, None]
        most = v.abs().amax() if v.numel() else torch.zeros((), dtype=F64)
        want.append(out.reshape(n, -1))
        tol.append((a * (3 * 2.0 ** -11 + 2 * worst * 2.0 ** -17 + 2.0 ** -18) + centred * 2.0 ** -11 + seen * 2.0 ** -25 * most
                    + out_half_step * out.abs() + 1e-7).reshape(n, -1))
    return torch.cat(want), torch.cat(tol)


def half_step(dtype):
    return torch.finfo(dtype).eps / 2
