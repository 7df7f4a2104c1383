"""The window cache held in 4 bits, and the attention that reads it.

A row of a key or value is cut into blocks of 32 elements; each block has one
power of two, ``2^(floor(log2 max|x|) - 2)``, held as the exponent + 127 in a byte,
and each element a 4-bit code: a sign and one of 0, 0.5, 1, 1.5, 2, 3, 4, 6 times the
power, the nearest (ties to the even code, 6 beyond 6).  That is the microscaling
format MXFP4, 4.25 bits an element: a cache of a given size serves 3.8 times as
many streams as in 16 bits, and a step reads 3.8 times less.  Codes stand for
values of the type that they were made from exactly (float16 does not hold all that
blocks made from bfloat16 or float32 can), and the attention over them is rounded to
the type once, at its end.  A block with an infinity or a NaN is NaN.

Caches are four contiguous uint8 tensors: codes [batch, kv_heads, sinks + window,
dim / 2], the even element in a byte's low half, and exponents [batch, kv_heads,
sinks + window, dim / 32], for keys and for values.
"""

from __future__ import annotations

import torch

from ..kernels.rasterize import _native as nat
from .attention import _aligned, _byref, _check_lengths, _check_sizes, _check_types, _scale, _Strides

BLOCK = 32


def _check_cache(tensors: dict[str, torch.Tensor], batch: int, kv_heads: int, dim: int,
                 window: int, sinks: int) -> None:
    if dim % BLOCK or not 0 < dim <= 128:
        raise NotImplementedError(f"rows of {dim} in 4 bits (a multiple of {BLOCK} up to 128)")
    for name, t in tensors.items():
        shape = (batch, kv_heads, sinks + window, dim // (BLOCK if name.endswith("exponents") else 2))
        if t.dtype != torch.uint8:
            raise TypeError(f"{name} is {t.dtype}, expected torch.uint8")
        if t.shape != shape:
            raise ValueError(f"{name} {tuple(t.shape)} is not {list(shape)}")
        # Written in place, so no copy can stand in for them.
        if not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous")
        if name.endswith("codes") and t.data_ptr() % 16:
            raise ValueError(f"{name} must start on a 16-byte boundary")


def window_attention_step_quant(
    q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, k_codes: torch.Tensor,
    k_exponents: torch.Tensor, v_codes: torch.Tensor, v_exponents: torch.Tensor,
    positions: torch.Tensor, window: int, sinks: int = 0, scale: float | None = None,
) -> torch.Tensor:
    """:func:`window_attention_step` over caches in 4 bits: q [batch, heads, dim], k
    and v [batch, kv_heads, dim], dim a multiple of 32 up to 128, ``positions`` int32
    [batch] on the GPU.  Writes k and v into the caches' slots and attends over the
    slots that are filled; the new token too is seen as the cache holds it.  A stream
    at a negative position is left alone and gives zeros.  Not differentiable; no
    host synchronisation, so a step can be captured in a graph."""
    _check_types(q, {"k": k, "v": v}, "window_attention_step_quant")
    if q.dim() != 3 or k.dim() != 3 or k.shape != v.shape or k.shape[::2] != q.shape[::2]:
        raise ValueError("window_attention_step_quant expects q [batch, heads, dim] and k, v [batch, "
                         f"kv_heads, dim], got {tuple(q.shape)}, {tuple(k.shape)} and {tuple(v.shape)}")
    b, h, d = q.shape
    hk = k.shape[1]
    window, sinks = int(window), int(sinks)
    _check_sizes(window, sinks, h, hk)
    _check_cache({"k_codes": k_codes, "k_exponents": k_exponents, "v_codes": v_codes,
                  "v_exponents": v_exponents}, b, hk, d, window, sinks)
    if positions.dtype != torch.int32:
        raise TypeError(f"positions is {positions.dtype}, expected torch.int32")
    if positions.shape != (b,):
        raise ValueError(f"positions {tuple(positions.shape)} does not fit a batch of {b}")
    problem = nat.GsAttention(b, 1, 0, window, sinks, h, hk, d, nat.TYPES[q.dtype], _scale(scale, d))
    device = nat.require_gpu(q, k, v, k_codes, k_exponents, v_codes, v_exponents, positions)
    q, k, v = nat.prepare(q, q.dtype), nat.prepare(k, q.dtype), nat.prepare(v, q.dtype)
    positions = positions.contiguous()
    out = torch.empty((b, h, d), dtype=q.dtype, device=device)
    lib = nat.library()
    ws_bytes = lib.gs_window_attention_step_quant_workspace_bytes(_byref(problem))
    ws = nat.workspace(ws_bytes, device)
    with nat.on(device):
        nat.check(
            lib.gs_window_attention_step_quant(
                _byref(problem), q.data_ptr(), k.data_ptr(), v.data_ptr(), k_codes.data_ptr(),
                k_exponents.data_ptr(), v_codes.data_ptr(), v_exponents.data_ptr(),
                positions.data_ptr(), out.data_ptr(), ws.data_ptr(), ws_bytes, nat.stream(device),
            ),
            "window_attention_step_quant",
        )
    return out


@torch.no_grad()
def window_cache_fill_quant(
    k: torch.Tensor, v: torch.Tensor, k_codes: torch.Tensor, k_exponents: torch.Tensor,
    v_codes: torch.Tensor, v_exponents: torch.Tensor, window: int, sinks: int = 0,
    lengths: torch.Tensor | None = None,
) -> None:
    """Encodes the tokens k and v [batch, tokens, kv_heads, dim] of a prefill that
    stay visible into caches in 4 bits: each slot takes the last of its tokens.  Of
    sequences that end early only the first ``lengths[batch]`` (int32 on the GPU;
    None: all) are taken; a slot without a token is left as it was."""
    _check_types(k, {"v": v}, "window_cache_fill_quant")
    if k.dim() != 4 or k.shape != v.shape:
        raise ValueError("window_cache_fill_quant expects k and v [batch, tokens, kv_heads, dim], got "
                         f"{tuple(k.shape)} and {tuple(v.shape)}")
    b, tokens, hk, d = k.shape
    window, sinks = int(window), int(sinks)
    _check_sizes(window, sinks, hk, hk)
    _check_cache({"k_codes": k_codes, "k_exponents": k_exponents, "v_codes": v_codes,
                  "v_exponents": v_exponents}, b, hk, d, window, sinks)
    _check_lengths(lengths, b)
    device = nat.require_gpu(k, v, k_codes, k_exponents, v_codes, v_exponents)
    if lengths is not None:
        nat.require_gpu(k, lengths)
        lengths = lengths.contiguous()
    (k, sk), (v, sv) = _aligned(k), _aligned(v)
    problem = nat.GsAttention(b, 0, tokens, window, sinks, hk, hk, d, nat.TYPES[k.dtype], 1.0)
    strides = _Strides[6](*sk, *sv)
    with nat.on(device):
        nat.check(
            nat.library().gs_window_cache_fill_quant(
                _byref(problem), k.data_ptr(), v.data_ptr(), strides, nat.ptr(lengths),
                k_codes.data_ptr(), k_exponents.data_ptr(), v_codes.data_ptr(),
                v_exponents.data_ptr(), nat.stream(device),
            ),
            "window_cache_fill_quant",
        )


class QuantWindowCache:
    """A :class:`WindowCache` in 4 bits: keys and values of ``batch`` running streams
    for :func:`window_attention_step_quant`, and each stream's next position
    (negative: the stream is not in use)."""

    def __init__(self, batch: int, kv_heads: int, dim: int, window: int, sinks: int = 0,
                 device: torch.device | str = "cuda"):
        self.window, self.sinks = int(window), int(sinks)
        _check_sizes(self.window, self.sinks, kv_heads, kv_heads)
        if dim % BLOCK or not 0 < dim <= 128:
            raise NotImplementedError(f"rows of {dim} in 4 bits (a multiple of {BLOCK} up to 128)")
        self.k_codes, self.v_codes = (
            torch.zeros((batch, kv_heads, self.sinks + self.window, dim // 2), dtype=torch.uint8,
                        device=device) for _ in range(2))
        self.k_exponents, self.v_exponents = (
            torch.zeros((batch, kv_heads, self.sinks + self.window, dim // BLOCK), dtype=torch.uint8,
                        device=device) for _ in range(2))
        self.positions = torch.zeros(batch, dtype=torch.int32, device=device)

    def _tensors(self):
        return self.k_codes, self.k_exponents, self.v_codes, self.v_exponents

    @torch.no_grad()
    def fill(self, k: torch.Tensor, v: torch.Tensor, lengths: torch.Tensor | None = None) -> None:
        """Starts every stream over with the tokens k, v [batch, tokens, kv_heads,
        dim] of a prefill; only those that stay visible are kept.  Of sequences that
        end early only the first ``lengths[batch]`` (int32; None: all) are taken, and
        each stream goes on behind its own."""
        window_cache_fill_quant(k, v, *self._tensors(), self.window, self.sinks, lengths)
        if lengths is None:
            self.positions.fill_(k.shape[1])
        else:
            self.positions.copy_(lengths.clamp(0, k.shape[1]))

    @torch.no_grad()
    def step(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
             scale: float | None = None) -> torch.Tensor:
        """Attention of each stream's next token, which joins the cache.  A stream at
        a negative position stays there: zeros, and nothing joins."""
        out = window_attention_step_quant(q, k, v, *self._tensors(), self.positions, self.window,
                                          self.sinks, scale)
        self.positions.add_(self.positions >= 0)
        return out
