"""The 2-norm of many gradients together, and clipping them to a limit.

``clip_grad_norm(parameters, max_norm)`` does what
``torch.nn.utils.clip_grad_norm_`` does: with ``norm`` the 2-norm of all
gradients taken as one vector, each is multiplied by ``min(1, max_norm / (norm +
1e-6))``.  The gradients are read once for the norm, and read and written once
more only where the factor is not one; nothing waits for the host.  The sum is
float64, so float32 gradients whose squares overflow count too, and a step gives
the same bits on every run.
"""

from __future__ import annotations

import ctypes
from collections.abc import Iterable

import torch

from ..kernels.rasterize import _native as nat


def check_max_norm(max_norm: float) -> float:
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError(f"max_norm must be non-negative, got {max_norm}")
    return max_norm


def _check(t: torch.Tensor) -> None:
    if t.layout != torch.strided:
        raise TypeError(f"gradients must be dense, got {t.layout}")
    if t.dtype not in nat.TYPES:
        raise TypeError(f"gradients must be float32, float16 or bfloat16, got {t.dtype}")


def _flat(t: torch.Tensor) -> torch.Tensor:
    """The tensor's elements one behind the other in some order: itself where it
    has no gaps and repeats nothing, whatever the order of its dimensions."""
    if t.is_contiguous() or torch.ops.aten.is_non_overlapping_and_dense(t):
        return t
    return t.contiguous()


def norm_of(tensors: list[torch.Tensor], max_norm: float, scale: bool = False,
            ) -> tuple[torch.Tensor, torch.Tensor]:
    """``(norm, factor)`` of dense tensors on one GPU, which are multiplied by the
    factor with ``scale``: float32, no dimensions."""
    device = nat.require_gpu(*tensors)
    entries = []
    for t in tensors:
        entries += (t.data_ptr(), t.numel(), nat.TYPES[t.dtype])
    both = torch.empty(2, dtype=torch.float32, device=device)
    norm, factor = both[0], both[1]
    lib = nat.library()
    ws_bytes = lib.gs_grad_norm_workspace_bytes(len(tensors))
    ws = nat.workspace(ws_bytes, device)
    array = (ctypes.c_int64 * len(entries))(*entries)
    with nat.on(device):
        nat.check(
            lib.gs_grad_norm(ctypes.cast(array, ctypes.c_void_p), len(tensors), max_norm, int(scale),
                             norm.data_ptr(), factor.data_ptr(), ws.data_ptr(), ws_bytes,
                             nat.stream(device)),
            "grad_norm",
        )
    return norm, factor


def _list(tensors: torch.Tensor | Iterable[torch.Tensor]) -> list[torch.Tensor]:
    return [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)


@torch.no_grad()
def grad_norm(tensors: torch.Tensor | Iterable[torch.Tensor]) -> torch.Tensor:
    """The 2-norm of all elements of one or many tensors (float32, float16 and
    bfloat16 side by side, on one GPU): a float32 tensor without dimensions, zero
    for none.  Not differentiable; no host synchronisation."""
    tensors = _list(tensors)
    for t in tensors:
        _check(t)
    if not tensors:
        return torch.zeros(())
    return norm_of([_flat(t) for t in tensors], 0.0)[0]


@torch.no_grad()
def clip_grad_norm(parameters: torch.Tensor | Iterable[torch.Tensor], max_norm: float) -> torch.Tensor:
    """Multiplies the gradients of ``parameters`` in place by ``min(1, max_norm /
    (norm + 1e-6))`` and returns ``norm``, their 2-norm before, as
    :func:`grad_norm` does.  Parameters without a gradient are passed over, a
    gradient that is met twice counts once; expanded gradients, and two whose
    stretches of memory overlap, are refused.  A norm of NaN makes every gradient NaN, an infinite
    one makes them zero where they are finite."""
    max_norm = check_max_norm(max_norm)
    grads, flat, spans, seen = [], [], [], set()
    for p in _list(parameters):
        g = p.grad
        if g is None:
            continue
        _check(g)
        start, count = g.data_ptr(), g.numel()
        mark = (start, g.shape, g.stride(), g.dtype)
        if not count or mark in seen:
            continue
        seen.add(mark)
        f = _flat(g)
        if f is not g:
            if any(n > 1 and s == 0 for n, s in zip(g.shape, g.stride())):
                raise ValueError("a gradient is expanded: its elements share memory that clipping writes")
            count = 1 + sum((n - 1) * s for n, s in zip(g.shape, g.stride()))
        grads.append(g)
        flat.append(f)
        spans.append((start, start + count * g.element_size()))
    if not grads:
        return torch.zeros(())
    end = 0
    for lo, hi in sorted(spans):
        if lo < end:
            raise ValueError("two gradients' stretches of memory overlap")
        end = hi
    norm, _ = norm_of(flat, max_norm, scale=True)
    for g, f in zip(grads, flat):
        if f is not g:
            g.copy_(f)
    torch.autograd.graph.increment_version(grads)
    return norm
