"""Attention of a layer over a quantised, paged key/value cache.

Host-side mirror of ``tf_qkv_epilogue``, ``tf_kv_cache_read`` and ``tf_tree_attention``: what the reference spreads over
``fused_qkv_epilogue`` (Metal/Fusions/fused.metal:86), the rotary kernels (Metal/Primitives/rope.metal:52,75), its cache
(Runtime/KVCache/KVCacheManager.swift:26-50) and ``Attention`` (Metal/Attention/attention.metal:135,227,343). A layer calls them between its
QKV projection and its output projection:

    epilogue.encode(q, k, v, q_out, batch, cache, head_dim=256, q_weight=..., k_weight=..., norm_v=True, frequencies=...)
    attention.encode(q_out, attn, cache, batch, workspace, scale=1.0)

Lengths stay on the device, every call only enqueues work on the given or the current stream of the context's device, and each can be
captured in a CUDA graph. Tensors of another type, device or shape than a call takes raise ``ValueError``; what the
library refuses raises :class:`~turbo_fieldfare_b200.kernels.TFError`.
"""
from __future__ import annotations

import ctypes as C

import torch

from ._capi import KVBatchDesc, KVCacheDesc, TF_BF16, TF_FP16
from .kernels import TurboContext, _ptr, _raw_current_stream, _stream

_ACT = {torch.float16: TF_FP16, torch.bfloat16: TF_BF16}
_MOST = (1 << 32) - 1                                          # of a stride


def _stream_of(context: TurboContext, stream) -> int:
    """The stream's handle; without one the current stream of the context's device, whichever device is current."""
    if stream is None:
        if _raw_current_stream is not None:
            return _raw_current_stream(context.device)
        return torch.cuda.current_stream(context.device).cuda_stream
    return _stream(stream)


def _check(name: str, t, device, dtypes, dims: int, contiguous: bool = True):
    if not isinstance(t, torch.Tensor) or t.dtype not in dtypes or t.dim() != dims:
        got = f"{tuple(t.shape)} {t.dtype}" if isinstance(t, torch.Tensor) else type(t).__name__
        raise ValueError(f"{name} must be a tensor of {dims} dimension(s) and type {' or '.join(str(d) for d in dtypes)}, got {got}")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, not on {device}")
    if contiguous and not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


def _row_stride(name: str, t, device, dtype, rows: int, cols: int) -> int:
    """Stride of a two-dimensional tensor of rows; columns are next to one another."""
    try:                                                       # the common case first: what follows costs microseconds a call
        if t.dtype is dtype and t.get_device() == device.index:
            have, width = t.shape
            stride, step = t.stride()
            if have >= rows and width == cols and step == 1:
                if have == 1:
                    return cols                                # a lone row has no next one
                if stride <= _MOST:
                    return stride
    except (AttributeError, ValueError):
        pass
    _check(name, t, device, (dtype,), 2, contiguous=False)
    if t.shape[0] < rows or t.shape[1] != cols:
        raise ValueError(f"{name} must be [>= {rows}, {cols}], got {tuple(t.shape)}")
    if cols > 1 and t.stride(1) != 1:
        raise ValueError(f"{name}: the columns of a row must be next to one another")
    stride = t.stride(0) if t.shape[0] > 1 else cols
    if stride > _MOST:                                         # ctypes would cut it to 32 bits
        raise ValueError(f"{name}: rows that are {stride} elements apart are further than 2^32 - 1")
    return stride


def _vector(name: str, t, device, dtype) -> int:
    """Length of a contiguous one-dimensional tensor."""
    if not (isinstance(t, torch.Tensor) and t.dtype is dtype and t.dim() == 1 and t.get_device() == device.index and t.is_contiguous()):
        _check(name, t, device, (dtype,), 1)
    return t.shape[0]


class KVCache:
    """``tf_kv_cache`` over the caller's planes: codes ``uint8 [pages, kv_heads, page_size, head_dim * bits / 8]``, scales and biases
    ``bfloat16 [pages, kv_heads, page_size, head_dim / 64]``, for keys and for values."""

    def __init__(self, k_codes, k_scales, k_biases, v_codes, v_scales, v_biases):
        self.planes = (k_codes, k_scales, k_biases, v_codes, v_scales, v_biases)
        self.device = k_codes.device
        for name, t in zip(("k_codes", "k_scales", "k_biases", "v_codes", "v_scales", "v_biases"), self.planes):
            _check(name, t, self.device, (torch.uint8,) if name.endswith("codes") else (torch.bfloat16,), 4)
        pages, heads, page_size, groups = k_scales.shape
        self.num_pages, self.kv_heads, self.page_size, self.head_dim = pages, heads, page_size, 64 * groups
        width = k_codes.shape[3]
        self.bits = 8 * width // max(self.head_dim, 1)
        if self.bits * self.head_dim != 8 * width or self.bits not in (4, 8):
            raise ValueError(f"codes of {width} bytes a row do not fit {groups} groups of 64 codes of 4 or 8 bits")
        for t in self.planes:
            if t.shape[:3] != k_scales.shape[:3] or t.shape[3] not in ((width,) if t.dtype == torch.uint8 else (groups,)):
                raise ValueError(f"cache planes disagree: {[tuple(p.shape) for p in self.planes]}")
        self._c = KVCacheDesc(*[_ptr(t) for t in self.planes], pages, page_size, heads, self.head_dim, self.bits)
        self._ref, self._index = C.byref(self._c), k_codes.get_device()

    @classmethod
    def allocate(cls, num_pages: int, page_size: int, kv_heads: int, head_dim: int, bits: int, device="cuda") -> "KVCache":
        """An empty cache (all values zero)."""
        shape = (num_pages, kv_heads, page_size)
        planes = []
        for _ in range(2):
            planes += [torch.zeros(*shape, head_dim * bits // 8, dtype=torch.uint8, device=device),
                       torch.zeros(*shape, head_dim // 64, dtype=torch.bfloat16, device=device),
                       torch.zeros(*shape, head_dim // 64, dtype=torch.bfloat16, device=device)]
        return cls(*planes)

    @property
    def nbytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in self.planes)


class KVBatch:
    """``tf_kv_batch``: which sequence and token every row of a call is. ``row_offsets`` int32 [sequences + 1], ``context_lengths``
    int32 [sequences], ``page_table`` int32 [sequences, pages of the longest], ``positions`` int32 [rows]. ``rows``: rows of the
    calls' tensors (default: those of ``positions``; without any the number is read back from ``row_offsets``, once)."""

    def __init__(self, row_offsets, context_lengths, page_table, positions=None, rows: int | None = None):
        self.device = row_offsets.device
        _check("row_offsets", row_offsets, self.device, (torch.int32,), 1)
        _check("context_lengths", context_lengths, self.device, (torch.int32,), 1)
        _check("page_table", page_table, self.device, (torch.int32,), 2)
        self.sequences = context_lengths.shape[0]
        if row_offsets.shape[0] != self.sequences + 1 or page_table.shape[0] != self.sequences:
            raise ValueError(f"{self.sequences} context lengths, but {row_offsets.shape[0]} row offsets and a table of {tuple(page_table.shape)}")
        if positions is not None:
            _check("positions", positions, self.device, (torch.int32,), 1)
        if rows is None:
            rows = positions.shape[0] if positions is not None else int(row_offsets[-1])
        if rows < 0 or (positions is not None and positions.shape[0] < rows):
            raise ValueError(f"{rows} rows need as many positions")
        self.row_offsets, self.context_lengths, self.page_table, self.positions, self.rows = row_offsets, context_lengths, page_table, positions, rows
        self._c = KVBatchDesc(_ptr(row_offsets), _ptr(context_lengths), _ptr(page_table), _ptr(positions), page_table.shape[1], self.sequences, rows)
        self._ref, self._index = C.byref(self._c), row_offsets.get_device()


class AttentionWorkspace:
    """``tf_attention_workspace``: scratch of :class:`TreeAttention` for one head size; serves one call at a time."""

    def __init__(self, context: TurboContext, head_dim: int):
        self.context, self.head_dim = context, head_dim
        handle = C.c_void_p()
        context.check(context.lib.tf_attention_workspace_create(context.handle, head_dim, C.byref(handle)))
        self.handle = handle

    @property
    def nbytes(self) -> int:
        return int(self.context.lib.tf_attention_workspace_bytes(self.handle))

    def close(self) -> None:
        if getattr(self, "handle", None):
            self.context.lib.tf_attention_workspace_destroy(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


def _same_device(context: TurboContext, *parts):
    for p in parts:
        if p is not None and p._index != context.device:
            raise ValueError(f"{type(p).__name__} is on {p.device}, the context on cuda:{context.device}")


class FusedQKVEpilogue:
    """``fused_qkv_epilogue`` (Metal/Fusions/fused.metal:86): head norms, rotation, cache write."""

    def __init__(self, context: TurboContext):
        self.context = context

    def encode(self, q, k, v, q_out, batch: KVBatch, cache: KVCache | None = None, *, head_dim: int, q_weight=None, k_weight=None,
               norm_v: bool = False, frequencies=None, k_out=None, v_out=None, eps: float = 1e-6, stream=None) -> None:
        """``q`` [rows, q_heads * head_dim], ``k`` and ``v`` [rows, kv_heads * head_dim] (fp16 or bf16; views of one packed
        row may be given); ``frequencies`` fp32: half as many as rotated elements."""
        ctx = self.context
        _same_device(ctx, batch, cache)
        device, dtype, rows = batch.device, q.dtype, batch.rows
        if dtype not in _ACT:
            raise ValueError(f"rows are float16 or bfloat16, not {dtype}")
        q_cols, kv_cols = q.shape[-1], k.shape[-1]
        if q.dim() != 2 or k.dim() != 2 or head_dim <= 0 or q_cols % head_dim or kv_cols % head_dim:
            raise ValueError(f"q {tuple(q.shape)} and k {tuple(k.shape)} are not rows of heads of {head_dim}")
        q_stride, q_out_stride = _row_stride("q", q, device, dtype, rows, q_cols), _row_stride("q_out", q_out, device, dtype, rows, q_cols)
        k_stride, v_stride = _row_stride("k", k, device, dtype, rows, kv_cols), _row_stride("v", v, device, dtype, rows, kv_cols)
        k_out_stride = 0 if k_out is None else _row_stride("k_out", k_out, device, dtype, rows, kv_cols)
        v_out_stride = 0 if v_out is None else _row_stride("v_out", v_out, device, dtype, rows, kv_cols)
        for n, w in (("q_weight", q_weight), ("k_weight", k_weight)):
            if w is not None and _vector(n, w, device, torch.bfloat16) != head_dim:
                raise ValueError(f"{n} has {w.shape[0]} elements, not {head_dim}")
        pairs = 0 if frequencies is None else _vector("frequencies", frequencies, device, torch.float32)
        ctx.check(ctx.lib.tf_qkv_epilogue(
            ctx.handle, _stream_of(ctx, stream), q.data_ptr(), q_stride, k.data_ptr(), k_stride, v.data_ptr(), v_stride, _ptr(q_weight), _ptr(k_weight),
            1 if norm_v else 0, _ptr(frequencies), pairs, eps, q_out.data_ptr(), q_out_stride,
            _ptr(k_out), k_out_stride, _ptr(v_out), v_out_stride, batch._ref, None if cache is None else cache._ref,
            q_cols // head_dim, kv_cols // head_dim, head_dim, _ACT[dtype]))


class KVCacheRead:
    """Cached rows back as fp16 or bf16 rows."""

    def __init__(self, context: TurboContext):
        self.context = context

    def encode(self, cache: KVCache, batch: KVBatch, k_out=None, v_out=None, *, stream=None) -> None:
        """``k_out`` and ``v_out``: [rows, kv_heads * head_dim]; either may be left out."""
        ctx = self.context
        _same_device(ctx, batch, cache)
        out = k_out if k_out is not None else v_out
        if out is None or out.dtype not in _ACT:
            raise ValueError("a read needs k_out or v_out, of float16 or bfloat16")
        cols = cache.kv_heads * cache.head_dim
        k_stride = 0 if k_out is None else _row_stride("k_out", k_out, batch.device, out.dtype, batch.rows, cols)
        v_stride = 0 if v_out is None else _row_stride("v_out", v_out, batch.device, out.dtype, batch.rows, cols)
        ctx.check(ctx.lib.tf_kv_cache_read(ctx.handle, _stream_of(ctx, stream), cache._ref, batch._ref, _ptr(k_out), k_stride, _ptr(v_out), v_stride,
                                           _ACT[out.dtype]))


class TreeAttention:
    """Attention of one token, a chain or a tree of drafted tokens per sequence over the cache."""

    def __init__(self, context: TurboContext):
        self.context = context

    def encode(self, q, out, cache: KVCache, batch: KVBatch, workspace: AttentionWorkspace, *, scale: float, window: int = 0, tree_mask=None,
               stream=None) -> None:
        """``q`` and ``out`` [rows, q_heads * head_dim]. ``tree_mask`` int64 [rows, words]: bit j of a row's words is set where it sees row j of
        its sequence (its ancestors and itself); without one the rows of a sequence are a chain. ``window``: a row sees
        cached tokens fewer than this many positions back (0: all)."""
        ctx = self.context
        _same_device(ctx, batch, cache)
        if q.dtype not in _ACT:
            raise ValueError(f"rows are float16 or bfloat16, not {q.dtype}")
        if q.dim() != 2 or q.shape[1] % cache.head_dim:
            raise ValueError(f"q {tuple(q.shape)} is not rows of heads of {cache.head_dim}")
        cols = q.shape[1]
        q_stride, out_stride = _row_stride("q", q, batch.device, q.dtype, batch.rows, cols), _row_stride("out", out, batch.device, q.dtype, batch.rows, cols)
        words = 0
        if tree_mask is not None:
            _check("tree_mask", tree_mask, batch.device, (torch.int64,), 2)
            words = tree_mask.shape[1]
            if words == 0:
                raise ValueError("tree_mask has no words")     # its pointer would be NULL, which is a chain
            if tree_mask.shape[0] < batch.rows:
                raise ValueError(f"tree_mask has {tree_mask.shape[0]} rows, the batch {batch.rows}")
        if not 0 <= window < 1 << 31:                          # ctypes would cut it to 32 bits
            raise ValueError("window must be from 0 to 2^31 - 1")
        ctx.check(ctx.lib.tf_tree_attention(ctx.handle, _stream_of(ctx, stream), q.data_ptr(), q_stride, out.data_ptr(), out_stride, cache._ref,
                                            batch._ref, _ptr(tree_mask), words, window, scale, cols // cache.head_dim, _ACT[q.dtype],
                                            workspace.handle))
