"""Attention with a sliding window in which the stream's first tokens stay visible.

A query at position p sees the ``window`` latest tokens up to its own and the
first ``sinks`` tokens of the sequence (in a stream of posed views, those of the
view that fixes the coordinate frame), so time and cache stay bounded however
long the stream gets.  ``window_attention`` is the training and prefill form,
``window_attention_step`` takes one token of each of several streams over a
:class:`WindowCache`.
"""

from __future__ import annotations

import ctypes
import math

import torch

from ..kernels.rasterize import _native as nat

_Strides = {n: ctypes.c_int64 * n for n in (6, 9, 12)}
_byref = ctypes.byref


def _scale(scale: float | None, dim: int) -> float:
    if scale is None:
        return 1.0 / math.sqrt(dim)
    scale = float(scale)
    if not 0.0 < scale < math.inf:
        raise ValueError(f"scale must be positive and finite, got {scale}")
    return scale


def _check_types(q: torch.Tensor, others: dict[str, torch.Tensor], what: str) -> None:
    if q.dtype not in nat.TYPES:
        raise TypeError(f"{what} expects float32, float16 or bfloat16, got {q.dtype}")
    for name, t in others.items():
        if t.dtype != q.dtype:
            raise TypeError(f"{name} is {t.dtype}, expected {q.dtype}")


def _check_sizes(window: int, sinks: int, heads: int, kv_heads: int) -> None:
    if window < 1 or sinks < 0:
        raise ValueError(f"window must be positive and sinks non-negative, got {window} and {sinks}")
    if kv_heads < 1 or heads < 1 or heads % kv_heads:
        raise ValueError(f"{heads} heads cannot share {kv_heads} key heads")


def _check_lengths(lengths: torch.Tensor | None, batch: int) -> None:
    if lengths is not None:
        if lengths.dtype != torch.int32:
            raise TypeError(f"lengths is {lengths.dtype}, expected torch.int32")
        if lengths.shape != (batch,):
            raise ValueError(f"lengths {tuple(lengths.shape)} does not fit a batch of {batch}")


def _strides(t: torch.Tensor) -> tuple[int, int, int]:
    """Strides of the first three dimensions, 0 for one of a single element,
    whose stride no address depends on and can be anything."""
    (a, b, c, _), (i, j, k, _) = t.stride(), t.shape
    return a if i > 1 else 0, b if j > 1 else 0, c if k > 1 else 0


def _on_16_bytes(t: torch.Tensor, strides: tuple[int, int, int]) -> bool:
    """Rows start on 16-byte boundaries, neighbouring elements side by side."""
    a, b, c = strides
    return t.stride(3) == 1 and not ((a | b | c) * t.element_size() | t.data_ptr()) & 15


def _aligned(t: torch.Tensor) -> tuple[torch.Tensor, tuple[int, int, int]]:
    """A tensor and its strides: rows on 16-byte boundaries and tokens less than
    2^24 elements apart, a copy where the strides do not give that."""
    strides = _strides(t)
    if strides[1] >= 1 << 24 or not _on_16_bytes(t, strides):
        t = t.contiguous()
        if t.data_ptr() % 16:
            t = t.clone()
        strides = _strides(t)
    return t, strides


def _problem(q, k, v, window, sinks, scale, lengths) -> nat.GsAttention:
    _check_types(q, {"k": k, "v": v}, "window_attention")
    if q.dim() != 4 or k.dim() != 4 or k.shape != v.shape:
        raise ValueError("window_attention expects q [batch, queries, heads, dim] and k, v [batch, "
                         f"keys, kv_heads, dim], got {tuple(q.shape)}, {tuple(k.shape)} and "
                         f"{tuple(v.shape)}")
    b, tq, h, d = q.shape
    if k.shape[0] != b or k.shape[3] != d:
        raise ValueError(f"k {tuple(k.shape)} does not fit q {tuple(q.shape)}")
    _check_sizes(window, sinks, h, k.shape[2])
    _check_lengths(lengths, b)
    return nat.GsAttention(b, tq, k.shape[1], window, sinks, h, k.shape[2], d, nat.TYPES[q.dtype],
                           _scale(scale, d))


def window_attention_forward(
    q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, window: int, sinks: int = 0,
    scale: float | None = None, lengths: torch.Tensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Forward kernel: returns ``(out, lse)`` with ``lse`` the logarithm of each
    softmax's sum, float32 [batch, heads, queries], which
    :func:`window_attention_backward` needs."""
    problem = _problem(q, k, v, window, sinks, scale, lengths)
    device = nat.require_gpu(q, k, v) if lengths is None else nat.require_gpu(q, k, v, lengths)
    (q, sq), (k, sk), (v, sv) = _aligned(q), _aligned(k), _aligned(v)
    lengths = None if lengths is None else lengths.contiguous()
    b, tq, h, _ = q.shape
    out = torch.empty(q.shape, dtype=q.dtype, device=device)
    lse = torch.empty((b, h, tq), dtype=torch.float32, device=device)
    strides = _Strides[9](*sq, *sk, *sv)
    nat.check(
        nat.library().gs_window_attention_fwd(
            _byref(problem), q.data_ptr(), k.data_ptr(), v.data_ptr(), strides, nat.ptr(lengths),
            out.data_ptr(), lse.data_ptr(), nat.stream(device),
        ),
        "window_attention",
    )
    return out, lse


def window_attention_backward(
    q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, out: torch.Tensor, lse: torch.Tensor,
    grad_out: torch.Tensor, window: int, sinks: int = 0, scale: float | None = None,
    lengths: torch.Tensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Backward kernels: gradients of q, k and v for the upstream gradient
    ``grad_out``, from the forward's ``out`` and ``lse``."""
    problem = _problem(q, k, v, window, sinks, scale, lengths)
    device = nat.require_gpu(q, k, v, out, lse, grad_out)
    if lengths is not None:
        nat.require_gpu(q, lengths)
        lengths = lengths.contiguous()
    if grad_out.shape != q.shape or grad_out.dtype != q.dtype:
        raise ValueError(f"grad_out {tuple(grad_out.shape)} {grad_out.dtype} does not fit q")
    if out.shape != q.shape or out.dtype != q.dtype:
        raise ValueError(f"out {tuple(out.shape)} {out.dtype} does not fit q")
    if lse.shape != (q.shape[0], q.shape[2], q.shape[1]) or lse.dtype != torch.float32:
        raise ValueError(f"lse {tuple(lse.shape)} {lse.dtype} does not fit q")
    (q, sq), (k, sk), (v, sv), (grad_out, sg) = _aligned(q), _aligned(k), _aligned(v), _aligned(grad_out)
    out, lse = nat.prepare(out, out.dtype), lse.contiguous()
    dq = torch.empty(q.shape, dtype=q.dtype, device=device)
    dk = torch.empty(k.shape, dtype=q.dtype, device=device)
    dv = torch.empty(k.shape, dtype=q.dtype, device=device)
    lib = nat.library()
    ws_bytes = lib.gs_window_attention_bwd_workspace_bytes(_byref(problem))
    ws = nat.workspace(ws_bytes, device)
    strides = _Strides[12](*sq, *sk, *sv, *sg)
    nat.check(
        lib.gs_window_attention_bwd(
            _byref(problem), q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(),
            lse.data_ptr(), grad_out.data_ptr(), strides, nat.ptr(lengths), dq.data_ptr(),
            dk.data_ptr(), dv.data_ptr(), ws.data_ptr(), ws_bytes, nat.stream(device),
        ),
        "window_attention backward",
    )
    return dq, dk, dv


class _WindowAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, window, sinks, scale, lengths):
        out, lse = window_attention_forward(q, k, v, window, sinks, scale, lengths)
        ctx.save_for_backward(q, k, v, out, lse, lengths)
        ctx.rule = (window, sinks, scale)
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_out):
        q, k, v, out, lse, lengths = ctx.saved_tensors
        return (*window_attention_backward(q, k, v, out, lse, grad_out, *ctx.rule, lengths),
                None, None, None, None)


def window_attention(
    q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, window: int, sinks: int = 0,
    scale: float | None = None, lengths: torch.Tensor | None = None,
) -> torch.Tensor:
    """Attention of q [batch, queries, heads, dim] over k and v [batch, keys,
    kv_heads, dim] (any strides; float32, float16 or bfloat16; dim a multiple of
    8 up to 128; heads a multiple of kv_heads, which they share in order).

    The queries are the last of the keys' positions: query i stands at p = keys
    - queries + i and sees key j when j <= p, and j > p - ``window`` or j <
    ``sinks``, and j < ``lengths[batch]`` (int32; None: all keys exist).  A query
    that sees no key gives zeros.  ``scale`` is 1 / sqrt(dim) unless given.
    Differentiable in q, k and v."""
    return _WindowAttention.apply(q, k, v, int(window), int(sinks), scale, lengths)


def window_attention_step(
    q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor,
    v_cache: torch.Tensor, positions: torch.Tensor, window: int, sinks: int = 0,
    scale: float | None = None,
) -> torch.Tensor:
    """One token of each of ``batch`` streams: q [batch, heads, dim], k and v
    [batch, kv_heads, dim], ``positions`` int32 [batch] on the GPU.  Writes k and
    v into the caches [batch, sinks + window, kv_heads, dim] (slot p, from
    ``sinks`` on ``sinks + (p - sinks) % window``) and attends over the slots that
    are filled.  A stream at a negative position is left alone and gives zeros.
    Not differentiable; no host synchronisation, so a step can be captured in a
    graph."""
    _check_types(q, {"k": k, "v": v, "k_cache": k_cache, "v_cache": v_cache}, "window_attention_step")
    if q.dim() != 3 or k.dim() != 3 or k.shape != v.shape or k.shape[::2] != q.shape[::2]:
        raise ValueError("window_attention_step expects q [batch, heads, dim] and k, v [batch, "
                         f"kv_heads, dim], got {tuple(q.shape)}, {tuple(k.shape)} and {tuple(v.shape)}")
    b, h, d = q.shape
    hk = k.shape[1]
    window, sinks = int(window), int(sinks)
    _check_sizes(window, sinks, h, hk)
    if k_cache.shape != (b, sinks + window, hk, d) or v_cache.shape != k_cache.shape:
        raise ValueError(f"caches {tuple(k_cache.shape)} and {tuple(v_cache.shape)} are not "
                         f"[{b}, {sinks} + {window}, {hk}, {d}]")
    if positions.dtype != torch.int32:
        raise TypeError(f"positions is {positions.dtype}, expected torch.int32")
    if positions.shape != (b,):
        raise ValueError(f"positions {tuple(positions.shape)} does not fit a batch of {b}")
    for name, t in (("k_cache", k_cache), ("v_cache", v_cache)):
        if 0 in t.stride() and any(n > 1 and s == 0 for n, s in zip(t.shape, t.stride())):
            raise ValueError(f"{name} is expanded: its streams or slots share memory that the step writes")
    device = nat.require_gpu(q, k, v, k_cache, v_cache, positions)
    sk, sv = _strides(k_cache), _strides(v_cache)
    for name, t, s in (("k_cache", k_cache, sk), ("v_cache", v_cache, sv)):
        # Written in place, so no aligned copy can stand in for them.
        if not _on_16_bytes(t, s):
            raise ValueError(f"{name} must have its rows on 16-byte boundaries")
    problem = nat.GsAttention(b, 1, 0, window, sinks, h, hk, d, nat.TYPES[q.dtype], _scale(scale, d))
    q, k, v = nat.prepare(q, q.dtype), nat.prepare(k, q.dtype), nat.prepare(v, q.dtype)
    positions = positions.contiguous()
    out = torch.empty((b, h, d), dtype=q.dtype, device=device)
    lib = nat.library()
    ws_bytes = lib.gs_window_attention_step_workspace_bytes(_byref(problem))
    ws = nat.workspace(ws_bytes, device)
    strides = _Strides[6](*sk, *sv)
    nat.check(
        lib.gs_window_attention_step(
            _byref(problem), q.data_ptr(), k.data_ptr(), v.data_ptr(), k_cache.data_ptr(),
            v_cache.data_ptr(), strides, positions.data_ptr(), out.data_ptr(), ws.data_ptr(),
            ws_bytes, nat.stream(device),
        ),
        "window_attention_step",
    )
    return out


class WindowCache:
    """Keys and values of ``batch`` running streams for
    :func:`window_attention_step`: the first ``sinks`` tokens and a ring of the
    last ``window`` ones, and each stream's next position (negative: the stream
    is not in use)."""

    def __init__(self, batch: int, kv_heads: int, dim: int, window: int, sinks: int = 0,
                 dtype: torch.dtype = torch.bfloat16, device: torch.device | str = "cuda"):
        _check_sizes(int(window), int(sinks), kv_heads, kv_heads)
        self.window, self.sinks = int(window), int(sinks)
        shape = (batch, self.sinks + self.window, kv_heads, dim)
        self.k = torch.zeros(shape, dtype=dtype, device=device)
        self.v = torch.zeros(shape, dtype=dtype, device=device)
        self.positions = torch.zeros(batch, dtype=torch.int32, device=device)

    @torch.no_grad()
    def fill(self, k: torch.Tensor, v: torch.Tensor, lengths: torch.Tensor | None = None) -> None:
        """Starts every stream over with the tokens k, v [batch, tokens,
        kv_heads, dim] of a prefill; only those that stay visible are kept.  Of
        sequences that end early only the first ``lengths[batch]`` (int32; None:
        all) are taken, and each stream goes on behind its own."""
        if k.shape != v.shape or k.dim() != 4 or k.shape[::2] != self.k.shape[::2] or k.shape[3] != self.k.shape[3]:
            raise ValueError(f"k {tuple(k.shape)} and v {tuple(v.shape)} do not fit the cache "
                             f"{tuple(self.k.shape)}")
        _check_lengths(lengths, k.shape[0])
        tokens = k.shape[1]
        if lengths is not None:
            lengths = lengths.clamp(0, tokens)
            # The token of each slot: a first token's slot its own, the ring's slot s
            # the last one of s, s + window, ..
            slot = torch.arange(self.sinks + self.window, device=self.k.device)
            behind = lengths[:, None] - 1 - slot
            ring = slot + behind.div(self.window, rounding_mode="floor") * self.window
            stream, at = (behind >= 0).nonzero(as_tuple=True)
            token = torch.where(slot < self.sinks, slot, ring)[stream, at]
            for cache, t in ((self.k, k), (self.v, v)):
                cache[stream, at] = t[stream, token].to(cache.dtype)
            self.positions.copy_(lengths)
            return
        first = min(self.sinks, tokens)
        ring = torch.arange(max(first, tokens - self.window), tokens, device=self.k.device)
        slots = self.sinks + (ring - self.sinks) % self.window
        for cache, t in ((self.k, k), (self.v, v)):
            cache[:, :first] = t[:, :first]
            cache[:, slots] = t[:, ring].to(cache.dtype)
        self.positions.fill_(tokens)

    def step(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
             scale: float | None = None) -> torch.Tensor:
        """Attention of each stream's next token, which joins the cache.  A stream
        at a negative position stays there: zeros, and nothing joins."""
        out = window_attention_step(q, k, v, self.k, self.v, self.positions, self.window, self.sinks,
                                    scale)
        self.positions.add_(self.positions >= 0)
        return out
