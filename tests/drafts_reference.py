"""Plain statements of a step with drafted tokens: its plan, the verification in 64 bits, what is kept of the cache."""
import math

import numpy as np
import torch


def ancestors(parents, i):
    """Node i and what it hangs under, from itself up; a parent that is not before its node is none."""
    out = [i]
    while True:
        p = int(parents[out[-1]]) if parents is not None else out[-1] - 1
        if p < 0 or p >= out[-1]:
            return out
        out.append(p)


def plan(state, new_rows, *, kept=None, window=0, rows, stride=None, parents=None, tokens=None, words=0):
    """One plan over `state` (dict of numpy arrays table, held, first, stack (list), context, page), in place; what the rows get."""
    table, held, first, context, page = state["table"], state["held"], state["first"], state["context"], state["page"]
    back = []
    for b, n in enumerate(new_rows):
        lo = int(first[b])
        if n < 0:
            hi = int(held[b])
            held[b] = first[b] = context[b] = 0
        else:
            context[b] += max(0, int(kept[b])) if kept is not None else 0
            out = max(0, int(context[b]) + 1 - window) // page if window else 0
            hi = max(lo, min(out, int(held[b])))
            first[b] = hi
        back += [int(p) for p in table[b, lo:hi]]
        table[b, lo:hi] = -1
    state["stack"] += back[::-1]
    offsets, got, waiting, needed = [0], [], False, 0
    for b, n in enumerate(new_rows):
        end = int(context[b]) + max(0, int(n))
        take = 0
        if n > 0 and -(-end // page) <= table.shape[1] and (stride is None or n <= stride):
            need = max(0, -(-end // page) - int(held[b]))
            waiting = waiting or need > len(state["stack"]) or len(got) + n > rows
            if not waiting:
                take = int(n)
                for _ in range(need):
                    table[b, held[b]] = state["stack"].pop()
                    held[b] += 1
        for i in range(take):
            token = int(context[b]) + i
            row = {"sequence": b, "slot": int(table[b, token // page]) * page + token % page, "position": token, "mask": [0] * words, "token": None}
            if stride is not None:
                up = ancestors(None if parents is None else parents[b], i) if parents is not None or words else None
                if up is not None:
                    row["position"] = int(context[b]) + len(up) - 1
                    for j in up:
                        if j // 64 < words:
                            row["mask"][j // 64] |= 1 << (j % 64)
                row["token"] = None if tokens is None else int(tokens[b][i])
            got.append(row)
        offsets.append(len(got))
    return offsets, got


def signed(word):
    return word - (1 << 64) if word >> 63 else word


def softmax64(x, temperature, cap):
    """Weights of the finite logits relative to the largest (64 bits), and the lowest index of the largest."""
    x = x.double()
    good = x.isfinite()                                            # of the logits as they are: a cap would make infinities finite
    if cap:
        x = cap * torch.tanh(x / cap)
    if not bool(good.any()):
        return torch.zeros_like(x), 0
    x = torch.where(good, x, torch.full_like(x, -math.inf))
    return torch.exp((x - x.max()) / temperature), int(torch.nonzero(x == x.max())[0])


def verify(logits, offsets, tokens, uniforms, *, parents=None, probs=None, temperatures=None, cap=0.0, nodes):
    """(tokens, rows, kept, logprobs) of every sequence, on CPU tensors."""
    n = len(offsets) - 1
    out_tokens, out_rows = np.full((n, nodes), -1, dtype=np.int64), np.full((n, nodes), -1, dtype=np.int64)
    kept, logprobs = np.zeros(n, dtype=np.int64), np.zeros((n, nodes))
    vocab = logits.shape[1]
    for b in range(n):
        count = min(offsets[b + 1] - offsets[b], nodes)
        if count <= 0:
            continue
        t = 1.0 if temperatures is None else float(temperatures[b])
        greedy = not t > 0
        uniform = np.clip(np.asarray(uniforms[b], dtype=np.float64), 0, 1 - 2.0 ** -24)

        def target(node):
            # likeliest by the logits as they are: a cap keeps their order but may round two of them together
            raw = logits[offsets[b] + node]
            best = softmax64(raw, 1.0, 0.0)[1]
            return softmax64(raw, 1.0 if greedy else t, cap)[0], best

        node, at = 0, 0
        w, best = target(0)
        left, q = w.clone(), None
        out_rows[b, 0] = 0

        def drafter(node):
            if probs is None or node >= probs.shape[1]:
                return None
            return torch.nan_to_num(probs[b, node].double(), nan=0.0, posinf=math.inf).clamp(min=0)

        q = drafter(0)
        refused = set()
        for i in range(1, count):
            p = int(parents[b][i]) if parents is not None else i - 1
            x = int(tokens[b][i])
            if p != node or not 0 <= x < vocab or x in refused:
                continue
            if greedy:
                good = x == best and float(w.sum()) > 0
            else:
                chance = uniform[i] * (float(q[x]) if q is not None else 1.0) * float(left.sum())
                good = chance < float(left[x])
            if good:
                out_tokens[b, at], out_rows[b, at + 1] = x, i
                logprobs[b, at] = math.log(float(w[x]) / float(w.sum()))
                at, node = at + 1, i
                w, best = target(i)
                left, q, refused = w.clone(), drafter(i), set()
            elif not greedy:
                if q is not None:
                    # p_{r+1} = max(p_r - q, 0) over its sum, with p_r = left / sum
                    s = float(left.sum())
                    left = (left - s * q).clamp(min=0) if s > 0 else left
                else:
                    left[x] = 0
                    refused.add(x)
        if not float(left.sum()) > 0:
            left = w
        if greedy or not float(w.sum()) > 0:
            token = best if float(w.sum()) > 0 else 0
        else:
            upto = left.cumsum(0)
            over = torch.nonzero(upto > uniform[0] * float(upto[-1]))
            token = int(over[0]) if len(over) else int(torch.nonzero(left > 0)[-1])
        out_tokens[b, at] = token
        logprobs[b, at] = math.log(float(w[token]) / float(w.sum())) if float(w.sum()) > 0 else -math.inf
        kept[b] = at + 1
    return out_tokens, out_rows, kept, logprobs
