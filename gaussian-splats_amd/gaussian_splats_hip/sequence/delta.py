"""The gated delta rule over a token sequence.

Beside ``gated_scan``'s vector, a state that is a matrix S [key_dim, dim] for each
head: an associative memory, from which a token's key reads what is held under it
and into which it writes the difference to the token's value,

    a = sigmoid(gate), b = sigmoid(beta),
    u_t = b_t (v_t - a_t S_{t-1}^T k_t),   S_t = a_t S_{t-1} + k_t u_t^T,
    o_t = scale S_t^T q_t.

Time is linear in the number of tokens and a running stream's memory constant.
``delta_scan`` is the training and prefill form, in chunks of 64 tokens whose
products run on the matrix cores; ``delta_scan_step`` takes one token of each of
several streams.  The recurrence, and the states that go in and come out, are float32;
what bfloat16 calls keep of them for the products of outputs and gradients is bfloat16,
as those products take it.  Keys should not be longer than one
(``torch.nn.functional.normalize``): what a longer one writes can grow from token to
token.
"""

from __future__ import annotations

import ctypes

import torch

from ..kernels.rasterize import _native as nat
from .attention import _aligned, _byref, _check_lengths, _scale, _strides

_Strides = {n: ctypes.c_int64 * (3 * n) for n in (5, 6)}


def _problem(q, k, v, gate, beta, state, scale, tokens: int) -> nat.GsDelta:
    """``tokens``: 1 where the tensors have a token dimension."""
    what = "delta_scan" if tokens else "delta_scan_step"
    if q.dtype not in nat.TYPES:
        raise TypeError(f"{what} expects float32, float16 or bfloat16, got {q.dtype}")
    for name, t in (("k", k), ("v", v), ("gate", gate), ("beta", beta)):
        if t.dtype != q.dtype:
            raise TypeError(f"{name} is {t.dtype}, expected {q.dtype}")
    dims, lead = 3 + tokens, "batch, tokens, " if tokens else "batch, "
    if q.dim() != dims or v.dim() != dims or k.shape != q.shape or v.shape[:-2] != q.shape[:-2]:
        raise ValueError(f"{what} expects q and k [{lead}key_heads, key_dim] and v [{lead}heads, dim], got "
                         f"{tuple(q.shape)}, {tuple(k.shape)} and {tuple(v.shape)}")
    for name, t in (("gate", gate), ("beta", beta)):
        if t.shape != v.shape[:-1]:
            raise ValueError(f"{name} {tuple(t.shape)} does not fit v {tuple(v.shape)}")
    b, hk, d = q.shape[0], q.shape[-2], q.shape[-1]
    h, dv = v.shape[-2], v.shape[-1]
    if hk < 1 or h < 1 or h % hk:
        raise ValueError(f"{h} heads cannot share {hk} key heads")
    if state is not None:
        if state.dtype != torch.float32:
            raise TypeError(f"state or its gradient is {state.dtype}, expected torch.float32")
        if state.shape != (b, h, d, dv):
            raise ValueError(f"state or its gradient {tuple(state.shape)} is not {[b, h, d, dv]}")
    return nat.GsDelta(b, q.shape[1] if tokens else 1, h, hk, d, dv, nat.TYPES[q.dtype], _scale(scale, max(d, 1)))


def _inputs(q, k, v, gate, beta, *more):
    """Tensors as the kernels read them, and their strides in a row."""
    pairs = [_aligned(t) for t in (q, k, v)]
    pairs += [(t, _strides(t.unsqueeze(-1))) for t in (gate, beta)]
    pairs += [_aligned(t) for t in more]
    return [t for t, _ in pairs], _Strides[len(pairs)](*(s for _, three in pairs for s in three))


def delta_scan_forward(
    q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, gate: torch.Tensor, beta: torch.Tensor,
    state: torch.Tensor | None = None, scale: float | None = None,
    lengths: torch.Tensor | None = None, backward: bool = True,
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Forward kernels: returns ``(out, last, kept)``, with ``kept`` the states
    before the chunks, the chunks' updates and, with ``backward``, their solved
    triangles, which :func:`delta_scan_backward` reads."""
    problem = _problem(q, k, v, gate, beta, state, scale, 1)
    _check_lengths(lengths, q.shape[0])
    given = [t for t in (state, lengths) if t is not None]
    device = nat.require_gpu(q, k, v, gate, beta, *given)
    lib = nat.library()
    out = torch.empty(v.shape, dtype=v.dtype, device=device)
    shape = (q.shape[0], v.shape[2], q.shape[3], v.shape[3])
    kept_bytes = lib.gs_delta_scan_kept_bytes(_byref(problem), int(backward))
    kept = torch.empty(kept_bytes // 4, dtype=torch.float32, device=device)
    if q.shape[1] == 0:
        last = torch.zeros(shape, device=device) if state is None else state.clone()
        return out, last, kept
    last = torch.empty(shape, dtype=torch.float32, device=device)
    state = None if state is None else state.contiguous()
    lengths = None if lengths is None else lengths.contiguous()
    (q, k, v, gate, beta), strides = _inputs(q, k, v, gate, beta)
    ws = nat.workspace(lib.gs_delta_scan_workspace_bytes(_byref(problem)), device)
    with nat.on(device):
        nat.check(
            lib.gs_delta_scan_fwd(
                _byref(problem), q.data_ptr(), k.data_ptr(), v.data_ptr(), gate.data_ptr(), beta.data_ptr(),
                strides, nat.ptr(lengths), nat.ptr(state), int(backward), out.data_ptr(), last.data_ptr(),
                kept.data_ptr(), ws.data_ptr(), ws.numel(), nat.stream(device),
            ),
            "delta_scan",
        )
    return out, last, kept


def delta_scan_backward(
    q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, gate: torch.Tensor, beta: torch.Tensor,
    kept: torch.Tensor, grad_out: torch.Tensor | None, grad_last: torch.Tensor | None,
    scale: float | None = None, lengths: torch.Tensor | None = None, need_state: bool = True,
) -> tuple[torch.Tensor, ...]:
    """Backward kernels: gradients of q, k, v, gate, beta and state, from the
    forward's ``kept``; a gradient that is None counts as zeros."""
    problem = _problem(q, k, v, gate, beta, grad_last, scale, 1)
    _check_lengths(lengths, q.shape[0])
    lib = nat.library()
    if kept.dtype != torch.float32 or not kept.is_contiguous():
        raise TypeError(f"kept is {kept.dtype}, expected a contiguous torch.float32 tensor")
    if kept.numel() * 4 != lib.gs_delta_scan_kept_bytes(_byref(problem), 1):
        raise ValueError(f"kept {tuple(kept.shape)} is not that of a forward with backward of q {tuple(q.shape)}")
    if grad_out is not None and (grad_out.shape != v.shape or grad_out.dtype != v.dtype):
        raise ValueError(f"grad_out {tuple(grad_out.shape)} {grad_out.dtype} does not fit v")
    given = [t for t in (grad_out, grad_last, lengths) if t is not None]
    device = nat.require_gpu(q, k, v, gate, beta, kept, *given)
    grads = [torch.empty(t.shape, dtype=t.dtype, device=device) for t in (q, k, v, gate, beta)]
    shape = (q.shape[0], v.shape[2], q.shape[3], v.shape[3])
    if q.shape[1] == 0:
        if not need_state:
            return (*grads, None)
        return (*grads, torch.zeros(shape, device=device) if grad_last is None else grad_last.clone())
    grad_state = torch.empty(shape, dtype=torch.float32, device=device) if need_state else None
    grad_last = None if grad_last is None else grad_last.contiguous()
    lengths = None if lengths is None else lengths.contiguous()
    more = () if grad_out is None else (grad_out,)
    (q, k, v, gate, beta, *more), strides = _inputs(q, k, v, gate, beta, *more)
    ws = nat.workspace(lib.gs_delta_scan_bwd_workspace_bytes(_byref(problem)), device)
    with nat.on(device):
        nat.check(
            lib.gs_delta_scan_bwd(
                _byref(problem), q.data_ptr(), k.data_ptr(), v.data_ptr(), gate.data_ptr(), beta.data_ptr(),
                more[0].data_ptr() if more else None, strides, nat.ptr(lengths),
                nat.ptr(grad_last), kept.data_ptr(), *(g.data_ptr() for g in grads), nat.ptr(grad_state),
                ws.data_ptr(), ws.numel(), nat.stream(device),
            ),
            "delta_scan backward",
        )
    return (*grads, grad_state)


class _DeltaScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, gate, beta, state, scale, lengths, backward):
        ctx.set_materialize_grads(False)
        out, last, kept = delta_scan_forward(q, k, v, gate, beta, state, scale, lengths, backward)
        if backward:
            ctx.save_for_backward(q, k, v, gate, beta, kept, lengths)
            ctx.scale = scale
        return out, last

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_out, grad_last):
        q, k, v, gate, beta, kept, lengths = ctx.saved_tensors
        return (*delta_scan_backward(q, k, v, gate, beta, kept, grad_out, grad_last, ctx.scale, lengths,
                                     ctx.needs_input_grad[5]), None, None, None)


def delta_scan(
    q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, gate: torch.Tensor, beta: torch.Tensor,
    state: torch.Tensor | None = None, scale: float | None = None, lengths: torch.Tensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """``(out, last)`` of the gated delta rule: q and k [batch, tokens, key_heads,
    key_dim], v [batch, tokens, heads, dim], gate and beta [batch, tokens, heads], of
    one type (float32, float16 or bfloat16) and any strides; heads a multiple of
    key_heads, which they share in order; key_dim and dim multiples of 8 up to 128.
    ``state`` float32 [batch, heads, key_dim, dim] is the one before the first token
    (None: zeros), ``last`` the one behind the last.  ``scale`` is 1 / sqrt(key_dim)
    unless given.  Of sequences that end early only the first ``lengths[batch]``
    (int32 on the GPU; None: all) are taken: what lies behind is not read, changes no
    state and gives zeros.

    A gate of -inf forgets what came before, one of +inf keeps it whole; a beta of -inf
    writes nothing, one of +inf with b = 1.  From a gate or beta that is NaN on, or a k or
    v that is not finite, its head gives NaN.  Differentiable in q, k, v, gate, beta and
    state."""
    # needs_input_grad does not know of no_grad, under which nothing is kept for a backward.
    backward = torch.is_grad_enabled() and any(
        t is not None and t.requires_grad for t in (q, k, v, gate, beta, state))
    return _DeltaScan.apply(q, k, v, gate, beta, state, scale, lengths, backward)


def delta_scan_step(
    q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, gate: torch.Tensor, beta: torch.Tensor,
    state: torch.Tensor, scale: float | None = None, state_out: torch.Tensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """One token of each of ``batch`` streams: q and k [batch, key_heads, key_dim], v
    [batch, heads, dim], gate and beta [batch, heads], ``state`` float32 [batch, heads,
    key_dim, dim].  Returns ``(out, state)`` with the state after the token, written
    to ``state_out`` where given (``state`` itself to step in place).  Inputs that are
    not finite go where the formula takes them: a v into its own column of the state,
    for which :func:`delta_scan` gives up the head.  Not differentiable; no host
    synchronisation, so a step can be captured in a graph."""
    if state is None:
        raise TypeError("delta_scan_step needs a state")
    problem = _problem(q, k, v, gate, beta, state, scale, 0)
    device = nat.require_gpu(q, k, v, gate, beta, state)
    if state_out is None:
        state_out = torch.empty(state.shape, dtype=torch.float32, device=device)
    else:
        nat.require_gpu(q, state_out)
        if (state_out.shape != state.shape or state_out.dtype != torch.float32
                or not state_out.is_contiguous() or state_out.data_ptr() % 16):
            raise ValueError("state_out must be a contiguous float32 tensor of state's shape on a "
                             "16-byte boundary")
        apart, size = state_out.data_ptr() - state.data_ptr(), state_out.numel() * 4
        if state.is_contiguous() and apart and abs(apart) < size:
            raise ValueError("state_out overlaps state without being it")
    q, k, v, gate, beta = (nat.prepare(t, t.dtype) for t in (q, k, v, gate, beta))
    state = nat.prepare(state)
    out = torch.empty(v.shape, dtype=v.dtype, device=device)
    with nat.on(device):
        nat.check(
            nat.library().gs_delta_scan_step(
                _byref(problem), q.data_ptr(), k.data_ptr(), v.data_ptr(), gate.data_ptr(), beta.data_ptr(),
                state.data_ptr(), out.data_ptr(), state_out.data_ptr(), nat.stream(device),
            ),
            "delta_scan_step",
        )
    return out, state_out
