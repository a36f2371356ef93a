"""What a batched step with drafted tokens needs around its layers.

Host-side mirror of ``tf_kv_plan``, ``tf_verify_drafts`` and ``tf_kv_cache_keep``. A step over the paged cache of :mod:`.attention`:

    plan.encode(pages, context_lengths, new_rows, rows, kept=kept, tokens=tokens, parents=parents)      # rows and pages of the step
    ...                                                        # per layer: FusedQKVEpilogue and TreeAttention over KVBatch(rows ...)
    verify.encode(logits, rows.row_offsets, tokens, uniforms, out_tokens, out_rows, kept, workspace, parents=parents)
    keep.encode(caches, batch, out_rows, kept)                 # the kept nodes behind their context, in all layers at once

The reference decodes one sequence and does this on the CPU (Runtime/Generation/RawCompletion.swift:81-246). Lengths, pages and what was kept stay on the
device, every call only enqueues work on the given or the current stream of the context's device, and a captured step serves growing contexts.
Tensors of another type, device or shape than a call takes raise ``ValueError``; what the library refuses raises
:class:`~turbo_fieldfare_b200.kernels.TFError`.
"""
from __future__ import annotations

import ctypes as C

import torch

from ._capi import DraftProbs, Drafts, KVCacheDesc, KVPagesDesc, KVRowsDesc, TF_BF16, TF_FP16, TF_FP32
from .attention import KVBatch, KVCache, _check, _same_device, _stream_of
from .kernels import TurboContext, _ptr

_VALUE = {torch.float16: TF_FP16, torch.bfloat16: TF_BF16, torch.float32: TF_FP32}
_I32 = (torch.int32,)


def _is(t, dtype, index: int, shape) -> bool:
    """The common case in one go: what follows where it is not costs a microsecond a tensor."""
    try:
        return t.dtype is dtype and t.get_device() == index and t.shape == shape and t.is_contiguous()
    except AttributeError:
        return False


def _need(name: str, t, dtype, like, shape) -> int:
    """Address of a contiguous tensor of a type and shape on the device of `like`."""
    if not _is(t, dtype, like.get_device(), shape):
        _check(name, t, like.device, (dtype,), len(shape))
        if tuple(t.shape) != tuple(shape):
            raise ValueError(f"{name} must be {list(shape)}, got {list(t.shape)}")
    return t.data_ptr()


def _ints(name: str, t, device, dims: int, shape=None):
    _check(name, t, device, _I32, dims)
    if shape is not None and tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} must be {list(shape)}, got {list(t.shape)}")


def _number(name: str, value) -> None:
    """ctypes would cut a larger number to 32 bits."""
    if not 0 < value < 1 << 31:
        raise ValueError(f"{name} must be from 1 to 2^31 - 1, got {value}")


class KVPages:
    """``tf_kv_pages``: ``page_table`` int32 [sequences, pages of the longest], ``held_pages`` and ``first_pages`` int32 [sequences], ``free_pages`` int32 [pages], a
    stack of which the first ``free_count`` [1] are nobody's (it is as long as the cache has pages, also where these are only some of them). ``first_pages`` is needed with a window."""

    def __init__(self, page_table, held_pages, free_pages, free_count, page_size: int, first_pages=None):
        self.device = page_table.device
        _check("page_table", page_table, self.device, _I32, 2)
        self.sequences, stride = page_table.shape
        _ints("held_pages", held_pages, self.device, 1, (self.sequences,))
        _check("free_pages", free_pages, self.device, _I32, 1)
        _ints("free_count", free_count, self.device, 1, (1,))
        if first_pages is not None:
            _ints("first_pages", first_pages, self.device, 1, (self.sequences,))
        _number("page_size", page_size)
        self.page_table, self.held_pages, self.free_pages, self.free_count, self.first_pages = page_table, held_pages, free_pages, free_count, first_pages
        self.page_size, self.num_pages = page_size, free_pages.shape[0]
        self._c = KVPagesDesc(_ptr(page_table), _ptr(held_pages), _ptr(first_pages), _ptr(free_pages), _ptr(free_count), stride, self.num_pages, page_size, self.sequences)
        self._ref, self._index = C.byref(self._c), page_table.get_device()

    @classmethod
    def allocate(cls, sequences: int, table_pages: int, num_pages: int, page_size: int, windowed: bool = False, device="cuda") -> "KVPages":
        """Nobody holds a page; page 0 is taken first."""
        i32 = dict(dtype=torch.int32, device=device)
        return cls(torch.full((sequences, table_pages), -1, **i32), torch.zeros(sequences, **i32), torch.arange(num_pages - 1, -1, -1, **i32),
                   torch.full((1,), num_pages, **i32), page_size, torch.zeros(sequences, **i32) if windowed else None)


class KVRows:
    """``tf_kv_rows``: what a plan writes. ``row_offsets`` int32 [sequences + 1], ``positions`` int32 [rows], and where they are wanted ``sequences`` and ``tokens`` int32 [rows],
    ``slots`` int64 [rows], ``tree_mask`` int64 [rows, words]."""

    def __init__(self, row_offsets, positions, *, sequences=None, slots=None, tokens=None, tree_mask=None):
        self.device = row_offsets.device
        _check("row_offsets", row_offsets, self.device, _I32, 1)
        _check("positions", positions, self.device, _I32, 1)
        self.rows = positions.shape[0]
        for name, t, dtype in (("sequences", sequences, torch.int32), ("tokens", tokens, torch.int32), ("slots", slots, torch.int64)):
            if t is not None:
                _check(name, t, self.device, (dtype,), 1)
                if t.shape[0] != self.rows:
                    raise ValueError(f"{name} has {t.shape[0]} rows, positions {self.rows}")
        words = 0
        if tree_mask is not None:
            _check("tree_mask", tree_mask, self.device, (torch.int64,), 2)
            words = tree_mask.shape[1]
            if tree_mask.shape[0] != self.rows or words == 0:
                raise ValueError(f"tree_mask must be [{self.rows}, words], got {list(tree_mask.shape)}")
        self.row_offsets, self.positions, self.sequences, self.slots, self.tokens, self.tree_mask = row_offsets, positions, sequences, slots, tokens, tree_mask
        self.sequence_count = row_offsets.shape[0] - 1
        self._c = KVRowsDesc(_ptr(row_offsets), _ptr(positions), _ptr(sequences), _ptr(slots), _ptr(tokens), _ptr(tree_mask), words, self.rows)
        self._ref, self._index = C.byref(self._c), row_offsets.get_device()

    @classmethod
    def allocate(cls, sequences: int, rows: int, mask_words: int = 0, tokens: bool = False, device="cuda") -> "KVRows":
        i32 = dict(dtype=torch.int32, device=device)
        return cls(torch.zeros(sequences + 1, **i32), torch.zeros(rows, **i32), tokens=torch.zeros(rows, **i32) if tokens else None,
                   tree_mask=torch.zeros(rows, mask_words, dtype=torch.int64, device=device) if mask_words else None)


def _drafts(like, sequences: int, tokens, parents, stride: int | None = None) -> Drafts | None:
    """``tf_drafts`` over tensors of [sequences, stride]."""
    if stride is None:
        first = tokens if tokens is not None else parents
        if first is None:
            return None
        if not isinstance(first, torch.Tensor) or first.dim() != 2:
            _check("tokens" if tokens is not None else "parents", first, like.device, _I32, 2)
        stride = first.shape[1]
    shape = (sequences, stride)
    return Drafts(None if tokens is None else _need("tokens", tokens, torch.int32, like, shape),
                  None if parents is None else _need("parents", parents, torch.int32, like, shape), stride)


class KVPlan:
    """Rows and pages of the next step from its request lengths."""

    def __init__(self, context: TurboContext):
        self.context = context

    def encode(self, pages: KVPages, context_lengths, new_rows, rows: KVRows, *, kept=None, window: int = 0, tokens=None, parents=None, nodes: int | None = None,
               stream=None) -> None:
        """``context_lengths`` int32 [sequences], updated in place by ``kept`` int32 [sequences]; ``new_rows`` int32 [sequences]: rows wanted, -1 for a sequence that has
        ended. ``tokens`` and ``parents`` int32 [sequences, nodes]: the drafted nodes, without parents chains (``nodes`` says how many at most where neither is given
        and ``rows`` has a mask)."""
        ctx, n = self.context, pages.sequences
        if pages._index != ctx.device or rows._index != ctx.device:
            _same_device(ctx, pages, rows)
        like, one, i32 = pages.page_table, (n,), torch.int32
        context_lengths, new_rows = _need("context_lengths", context_lengths, i32, like, one), _need("new_rows", new_rows, i32, like, one)
        if kept is not None:
            kept = _need("kept", kept, i32, like, one)
        if rows.sequence_count != n:
            raise ValueError(f"{n} sequences, but {rows.sequence_count + 1} row offsets")
        if not 0 <= window < 1 << 31:                          # ctypes would cut it to 32 bits
            raise ValueError("window must be from 0 to 2^31 - 1")
        if nodes is not None and not 0 < nodes < 1 << 31:
            raise ValueError("nodes must be from 1 to 2^31 - 1")
        drafts = _drafts(like, n, tokens, parents, nodes)
        ctx.check(ctx.lib.tf_kv_plan(ctx.handle, _stream_of(ctx, stream), pages._ref, context_lengths, new_rows, kept, window,
                                     None if drafts is None else C.byref(drafts), rows._ref))


class VerificationWorkspace:
    """``tf_verify_workspace``: scratch of :class:`DraftVerification` for ``rows`` rows of ``vocab`` logits; serves one call at a time."""

    def __init__(self, context: TurboContext, rows: int, vocab: int):
        self.context = context
        _number("rows", rows)
        _number("vocab", vocab)
        handle = C.c_void_p()
        context.check(context.lib.tf_verify_workspace_create(context.handle, rows, vocab, C.byref(handle)))
        self.handle = handle

    @property
    def nbytes(self) -> int:
        return int(self.context.lib.tf_verify_workspace_bytes(self.handle))

    def close(self) -> None:
        if getattr(self, "handle", None):
            self.context.lib.tf_verify_workspace_destroy(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class DraftVerification:
    """Which drafted tokens are kept and what comes next; with one node per sequence the sampler of a token."""

    def __init__(self, context: TurboContext):
        self.context = context

    def encode(self, logits, row_offsets, tokens, uniforms, out_tokens, out_rows, kept, workspace: VerificationWorkspace, *, parents=None, draft_probs=None,
               temperatures=None, softcap: float = 0.0, logprobs=None, stream=None) -> None:
        """``logits`` [rows, vocab] (fp16, bf16 or fp32; rows may be further apart): row ``row_offsets[b] + i`` is what the target says behind node i of sequence b. ``tokens`` and
        ``parents`` int32 [sequences, nodes], ``uniforms`` fp32 [sequences, nodes] in [0, 1): a node's test, the first one the draw of the next token. ``draft_probs``
        [sequences, nodes that have a row, vocab]: what a node's children were drawn from. ``temperatures`` fp32 [sequences]. Out: ``out_tokens`` and ``out_rows`` int32 and
        ``logprobs`` fp32 [sequences, nodes], ``kept`` int32 [sequences]."""
        ctx = self.context
        if not isinstance(logits, torch.Tensor) or logits.dim() != 2 or logits.dtype not in _VALUE:
            raise ValueError("logits must be [rows, vocab] of float16, bfloat16 or float32")
        rows, vocab = logits.shape
        if logits.get_device() != ctx.device:
            raise ValueError(f"logits are on {logits.device}, the context on cuda:{ctx.device}")
        stride, step = logits.stride()
        if vocab == 0 or vocab > 1 and step != 1:
            raise ValueError("the logits of a row must be next to one another, one at the least")
        if not _is(row_offsets, torch.int32, ctx.device, (out_tokens.shape[0] + 1,) if isinstance(out_tokens, torch.Tensor) and out_tokens.dim() else ()):
            _check("row_offsets", row_offsets, logits.device, _I32, 1)
        n = row_offsets.shape[0] - 1
        if n < 0:
            raise ValueError("row_offsets is empty")
        if tokens is None:
            raise ValueError("tokens are needed")
        drafts = _drafts(logits, n, tokens, parents)
        shape, one, i32, f32 = (n, drafts.stride), (n,), torch.int32, torch.float32
        uniforms = _need("uniforms", uniforms, f32, logits, shape)
        out_tokens, out_rows, kept = _need("out_tokens", out_tokens, i32, logits, shape), _need("out_rows", out_rows, i32, logits, shape), _need("kept", kept, i32, logits, one)
        if temperatures is not None:
            temperatures = _need("temperatures", temperatures, f32, logits, one)
        if logprobs is not None:
            logprobs = _need("logprobs", logprobs, f32, logits, shape)
        probs = None
        if draft_probs is not None:
            if not isinstance(draft_probs, torch.Tensor) or draft_probs.dim() != 3 or draft_probs.dtype not in _VALUE or draft_probs.get_device() != ctx.device:
                _check("draft_probs", draft_probs, logits.device, tuple(_VALUE), 3, contiguous=False)
            have, count, width = draft_probs.shape
            if have != n or width != vocab:
                raise ValueError(f"draft_probs must be [{n}, nodes, {vocab}], got {list(draft_probs.shape)}")
            sequence_stride, node_stride, step = draft_probs.stride()
            if vocab > 1 and step != 1:
                raise ValueError("the probabilities of a node must be next to one another")
            if n and count:
                probs = C.byref(DraftProbs(draft_probs.data_ptr(), sequence_stride, node_stride, count, _VALUE[draft_probs.dtype]))
        ctx.check(ctx.lib.tf_verify_drafts(
            ctx.handle, _stream_of(ctx, stream), logits.data_ptr(), stride if rows > 1 else vocab, _VALUE[logits.dtype], vocab, row_offsets.data_ptr(), rows, n,
            C.byref(drafts), uniforms, probs, temperatures, softcap, out_tokens, out_rows, kept, logprobs, workspace.handle))


class KVCacheKeep:
    """The cache rows of the kept nodes behind their context."""

    def __init__(self, context: TurboContext):
        self.context = context

    def encode(self, caches, batch: KVBatch, kept_rows, kept, *, stream=None) -> None:
        """``caches``: the layers' caches that share the batch's page table; ``kept_rows`` int32 [sequences, nodes] and ``kept`` int32 [sequences] as
        :class:`DraftVerification` writes them, before the next plan raises the context lengths."""
        ctx = self.context
        if isinstance(caches, KVCache):
            caches = (caches,)
        if batch._index != ctx.device or any(c._index != ctx.device for c in caches):
            _same_device(ctx, batch, *caches)
        if not isinstance(kept_rows, torch.Tensor) or kept_rows.dim() != 2:
            _check("kept_rows", kept_rows, batch.device, _I32, 2)
        have, stride = kept_rows.shape
        if have != batch.sequences:
            raise ValueError(f"kept_rows has {have} sequences, the batch {batch.sequences}")
        like = batch.row_offsets
        kept_rows, kept = _need("kept_rows", kept_rows, torch.int32, like, (have, stride)), _need("kept", kept, torch.int32, like, (have,))
        descriptors = caches[0]._ref if len(caches) == 1 else (KVCacheDesc * len(caches))(*[c._c for c in caches])
        ctx.check(ctx.lib.tf_kv_cache_keep(ctx.handle, _stream_of(ctx, stream), descriptors, len(caches), batch._ref, kept_rows, stride, kept))
