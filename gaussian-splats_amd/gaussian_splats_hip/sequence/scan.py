"""Gated linear recurrence over a token sequence.

``gated_scan(x, gate)`` mixes the tokens of ``x`` [batch, tokens, channels] in
time linear in their number, per channel:

    a_t = sigmoid(gate_t),   h_t = a_t h_{t-1} + (1 - a_t) x_t,

the recurrence by which front-to-back compositing accumulates colour.  h is
float32 whatever the types; a state carries it from one call to the next, and
``gated_scan_step`` takes one token of a running stream.  A gate of -inf forgets
what came before, one of +inf keeps it whole.

Long scans wait for one another's chunks on the GPU.  A wait that hits its limit
(none should) leaves NaN in what needs its state and a bit in the GPU's word of
failed checks, which the next rasterizer call that synchronises raises.
"""

from __future__ import annotations

import ctypes

import torch

from ..kernels.rasterize import _native as nat

_Strides4 = ctypes.c_int64 * 4
_Strides6 = ctypes.c_int64 * 6


def _check(x: torch.Tensor, gate: torch.Tensor, state: torch.Tensor | None, dims: int, what: str) -> None:
    if x.dtype not in nat.TYPES:
        raise TypeError(f"{what} expects float32, float16 or bfloat16, got {x.dtype}")
    if gate.dtype != x.dtype:
        raise TypeError(f"gate is {gate.dtype}, expected {x.dtype}")
    if x.dim() != dims or gate.shape != x.shape:
        raise ValueError(f"{what} expects x and gate of {dims} equal dimensions, got "
                         f"{tuple(x.shape)} and {tuple(gate.shape)}")
    if state is not None:
        if state.dtype != torch.float32:
            raise TypeError(f"state is {state.dtype}, expected torch.float32")
        if state.shape != (x.shape[0], x.shape[-1]):
            raise ValueError(f"state {tuple(state.shape)} does not fit x {tuple(x.shape)}")


def _inner(t: torch.Tensor) -> torch.Tensor:
    """Neighbouring channels lie side by side."""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def gated_scan_forward(
    x: torch.Tensor, gate: torch.Tensor, state: torch.Tensor | None = None
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Forward kernels: returns ``(y, last, starts)``, with ``starts`` the
    float32 states before each chunk of tokens, which
    :func:`gated_scan_backward` runs the chunks from."""
    _check(x, gate, state, 3, "gated_scan")
    device = nat.require_gpu(x, gate) if state is None else nat.require_gpu(x, gate, state)
    x, gate = _inner(x), _inner(gate)
    state = None if state is None else state.contiguous()
    b, t, c = x.shape
    lib = nat.library()
    y = torch.empty((b, t, c), dtype=x.dtype, device=device)
    starts = torch.empty((b, lib.gs_gated_scan_chunks(t), c), dtype=torch.float32, device=device)
    if t == 0:
        last = torch.zeros((b, c), device=device) if state is None else state.clone()
        return y, last, starts
    last = torch.empty((b, c), dtype=torch.float32, device=device)
    ws = nat.workspace(lib.gs_gated_scan_workspace_bytes(b, t, c, 0), device)
    strides = _Strides4(x.stride(0), x.stride(1), gate.stride(0), gate.stride(1))
    nat.check(
        lib.gs_gated_scan_fwd(
            x.data_ptr(), gate.data_ptr(), nat.ptr(state), b, t, c, strides, nat.TYPES[x.dtype],
            y.data_ptr(), last.data_ptr(), starts.data_ptr(), ws.data_ptr(), ws.numel(),
            nat.stream(device),
        ),
        "gated_scan",
    )
    return y, last, starts


def gated_scan_backward(
    x: torch.Tensor, gate: torch.Tensor, starts: torch.Tensor, grad_y: torch.Tensor | None,
    grad_last: torch.Tensor | None, need_state: bool = True,
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor | None]:
    """Backward kernels: gradients of x, gate and state; a gradient that is
    None counts as zeros."""
    _check(x, gate, None, 3, "gated_scan backward")
    b, t, c = x.shape
    lib = nat.library()
    if starts.dtype != torch.float32:
        raise TypeError(f"starts is {starts.dtype}, expected torch.float32")
    if starts.shape != (b, lib.gs_gated_scan_chunks(t), c) or not starts.is_contiguous():
        raise ValueError(f"starts {tuple(starts.shape)} are not those of x {tuple(x.shape)}")
    if grad_y is not None and (grad_y.shape != x.shape or grad_y.dtype != x.dtype):
        raise ValueError(f"grad_y {tuple(grad_y.shape)} {grad_y.dtype} does not fit x")
    if grad_last is not None and (grad_last.shape != (b, c) or grad_last.dtype != torch.float32):
        raise ValueError(f"grad_last {tuple(grad_last.shape)} {grad_last.dtype} does not fit x")
    device = nat.require_gpu(x, gate, starts, *(g for g in (grad_y, grad_last) if g is not None))
    x, gate = _inner(x), _inner(gate)
    grad_y = None if grad_y is None else _inner(grad_y)
    grad_last = None if grad_last is None else grad_last.contiguous()
    grad_x = torch.empty((b, t, c), dtype=x.dtype, device=device)
    grad_gate = torch.empty((b, t, c), dtype=x.dtype, device=device)
    if t == 0:
        if not need_state:
            return grad_x, grad_gate, None
        return grad_x, grad_gate, (torch.zeros((b, c), device=device) if grad_last is None
                                   else grad_last.clone())
    grad_state = torch.empty((b, c), dtype=torch.float32, device=device) if need_state else None
    ws = nat.workspace(lib.gs_gated_scan_workspace_bytes(b, t, c, 1), device)
    dy = x if grad_y is None else grad_y
    strides = _Strides6(x.stride(0), x.stride(1), gate.stride(0), gate.stride(1), dy.stride(0),
                        dy.stride(1))
    nat.check(
        lib.gs_gated_scan_bwd(
            x.data_ptr(), gate.data_ptr(), starts.data_ptr(), nat.ptr(grad_y), nat.ptr(grad_last),
            b, t, c, strides, nat.TYPES[x.dtype], grad_x.data_ptr(), grad_gate.data_ptr(),
            nat.ptr(grad_state), ws.data_ptr(), ws.numel(), nat.stream(device),
        ),
        "gated_scan backward",
    )
    return grad_x, grad_gate, grad_state


class _GatedScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gate, state):
        ctx.set_materialize_grads(False)
        y, last, starts = gated_scan_forward(x, gate, state)
        ctx.save_for_backward(x, gate, starts)
        return y, last

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_y, grad_last):
        x, gate, starts = ctx.saved_tensors
        return gated_scan_backward(x, gate, starts, grad_y, grad_last, ctx.needs_input_grad[2])


def gated_scan(
    x: torch.Tensor, gate: torch.Tensor, state: torch.Tensor | None = None
) -> tuple[torch.Tensor, torch.Tensor]:
    """``(y, last)``: the recurrence over the tokens of ``x`` and ``gate``
    [batch, tokens, channels] (float32, float16 or bfloat16) from ``state``
    (float32 [batch, channels], None for zeros), y in x's type, and the state
    after the last token in float32; differentiable in x, gate and state."""
    return _GatedScan.apply(x, gate, state)


def gated_scan_step(
    x: torch.Tensor, gate: torch.Tensor, state: torch.Tensor, state_out: torch.Tensor | None = None
) -> tuple[torch.Tensor, torch.Tensor]:
    """One token of each of ``batch`` streams: ``x`` and ``gate`` [batch,
    channels], ``state`` float32 [batch, channels].  Returns ``(y, state)``
    with the state after the token, written to ``state_out`` where given
    (``state`` itself to step in place).  Not differentiable."""
    _check(x, gate, state, 2, "gated_scan_step")
    device = nat.require_gpu(x, gate, state)
    x, gate, state = x.contiguous(), gate.contiguous(), state.contiguous()
    if state_out is None:
        state_out = torch.empty(state.shape, dtype=torch.float32, device=device)
    else:
        nat.require_gpu(x, state_out)
        if (state_out.shape != state.shape or state_out.dtype != torch.float32
                or not state_out.is_contiguous()):
            raise ValueError("state_out must be a contiguous float32 tensor of state's shape")
    y = torch.empty(x.shape, dtype=x.dtype, device=device)
    nat.check(
        nat.library().gs_gated_scan_step(
            x.data_ptr(), gate.data_ptr(), state.data_ptr(), x.shape[0], x.shape[1],
            nat.TYPES[x.dtype], y.data_ptr(), state_out.data_ptr(), nat.stream(device),
        ),
        "gated_scan_step",
    )
    return y, state_out
