"""Root-mean-square norm with the residual's addition.

``add_rms_norm(x, residual, weight)`` opens a block of a sequence model: it adds
a branch's output ``x`` to the residual stream and norms the sum,

    s = x + residual,   y = s / sqrt(mean(s^2) + eps) * weight,

and returns ``(y, s)``: y for the next branch, s for the stream.  The sums are
float32 whatever the types; y is rounded once to x's type, s once to the
residual's.  The stream may be float32 beside 16-bit branches.
``add_rms_norm_quant`` is its serving form: y as int8 or e4m3 codes with a scale
per row.
"""

from __future__ import annotations

import torch

from ..kernels.rasterize import _native as nat

_CODES = {"int8": (nat.TYPE_I8, torch.int8), "e4m3": (nat.TYPE_E4M3, torch.float8_e4m3fn)}


def _check_rows(shape: torch.Size, dtype: torch.dtype, weight: torch.Tensor) -> None:
    if dtype not in nat.TYPES:
        raise TypeError(f"add_rms_norm expects float32, float16 or bfloat16, got {dtype}")
    if len(shape) == 0 or shape[-1] == 0:
        raise ValueError(f"add_rms_norm norms the last dimension, got shape {tuple(shape)}")
    if weight.shape != shape[-1:]:
        raise ValueError(f"weight {tuple(weight.shape)} does not fit rows of {shape[-1]}")
    if weight.dtype != dtype and weight.dtype != torch.float32:
        raise TypeError(f"weight is {weight.dtype}, expected {dtype} or torch.float32")


def _check(x: torch.Tensor, residual: torch.Tensor | None, weight: torch.Tensor, eps: float) -> None:
    _check_rows(x.shape, x.dtype, weight)
    if residual is not None:
        if residual.shape != x.shape:
            raise ValueError(f"x {tuple(x.shape)} and residual {tuple(residual.shape)} differ")
        if residual.dtype != x.dtype and residual.dtype != torch.float32:
            raise TypeError(f"residual is {residual.dtype}, expected {x.dtype} or torch.float32")
    if not eps >= 0.0:
        raise ValueError(f"eps must be non-negative, got {eps}")


def _rows(t: torch.Tensor) -> torch.Tensor:
    """[rows, width] with neighbouring elements in a row; a view where the
    strides allow one."""
    t = t.reshape(-1, t.shape[-1])
    return t if t.stride(1) == 1 or t.shape[1] == 1 else t.contiguous()


def add_rms_norm_forward(
    x: torch.Tensor, residual: torch.Tensor | None, weight: torch.Tensor, eps: float = 1e-6
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Forward kernel: returns ``(y, sum, inverse_rms)``; without a residual
    ``sum`` is ``x`` itself."""
    _check(x, residual, weight, eps)
    device = nat.require_gpu(x, weight) if residual is None else nat.require_gpu(x, residual, weight)
    x2 = _rows(x)
    r2 = None if residual is None else _rows(residual)
    weight = weight.contiguous()
    rows, width = x2.shape
    kept = x.dtype if residual is None else residual.dtype
    y = torch.empty(x.shape, dtype=x.dtype, device=device)
    total = x if residual is None else torch.empty(x.shape, dtype=kept, device=device)
    inverse = torch.empty(rows, dtype=torch.float32, device=device)
    nat.check(
        nat.library().gs_add_rms_norm_fwd(
            x2.data_ptr(), None if r2 is None else r2.data_ptr(), weight.data_ptr(), rows, width,
            x2.stride(0), 0 if r2 is None else r2.stride(0), nat.TYPES[x.dtype], nat.TYPES[kept],
            nat.TYPES[weight.dtype], eps, y.data_ptr(),
            None if residual is None else total.data_ptr(), inverse.data_ptr(), nat.stream(device),
        ),
        "add_rms_norm",
    )
    return y, total, inverse


def add_rms_norm_backward(
    total: torch.Tensor, weight: torch.Tensor, inverse: torch.Tensor,
    grad_y: torch.Tensor | None, grad_sum: torch.Tensor | None, dtype: torch.dtype,
    need_x: bool = True, need_residual: bool = True, need_weight: bool = True,
) -> tuple[torch.Tensor | None, torch.Tensor | None, torch.Tensor | None]:
    """Backward kernels: gradients of x (of type ``dtype``), residual and
    weight.  The first two are one tensor where their types agree."""
    _check_rows(total.shape, dtype, weight)
    if total.dtype != dtype and total.dtype != torch.float32:
        raise TypeError(f"total is {total.dtype}, expected {dtype} or torch.float32")
    if inverse.dtype != torch.float32:
        raise TypeError(f"inverse is {inverse.dtype}, expected torch.float32")
    if inverse.numel() * total.shape[-1] != total.numel():
        raise ValueError(f"inverse {tuple(inverse.shape)} is not that of the rows of {tuple(total.shape)}")
    for g, kind in ((grad_y, dtype), (grad_sum, total.dtype)):
        if g is not None and (g.shape != total.shape or g.dtype != kind):
            raise ValueError(f"gradient {tuple(g.shape)} {g.dtype} does not fit "
                             f"{tuple(total.shape)} {kind}")
    given = [g for g in (grad_y, grad_sum) if g is not None]
    device = nat.require_gpu(total, weight, inverse, *given)
    s2 = _rows(total)
    weight, inverse = weight.contiguous(), inverse.contiguous()
    rows, width = s2.shape
    grads = [None if g is None else g.contiguous() for g in (grad_y, grad_sum)]
    same = dtype == total.dtype
    grad_x = grad_residual = grad_weight = ws = None
    if need_x or (need_residual and same):
        grad_x = torch.empty(total.shape, dtype=dtype, device=device)
    if need_residual:
        grad_residual = grad_x if same else torch.empty(total.shape, dtype=total.dtype, device=device)
    lib = nat.library()
    ws_bytes = 0
    if need_weight:
        grad_weight = torch.empty(width, dtype=weight.dtype, device=device)
        ws_bytes = lib.gs_add_rms_norm_bwd_workspace_bytes(rows, width)
        ws = nat.workspace(ws_bytes, device)
    nat.check(
        lib.gs_add_rms_norm_bwd(
            s2.data_ptr(), weight.data_ptr(), inverse.data_ptr(), nat.ptr(grads[0]),
            nat.ptr(grads[1]), rows, width, s2.stride(0), nat.TYPES[dtype], nat.TYPES[total.dtype],
            nat.TYPES[weight.dtype], nat.ptr(grad_x), None if same else nat.ptr(grad_residual),
            nat.ptr(grad_weight), nat.ptr(ws), ws_bytes, nat.stream(device),
        ),
        "add_rms_norm backward",
    )
    return (grad_x if need_x else None), grad_residual, grad_weight


class _AddRmsNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, eps):
        ctx.set_materialize_grads(False)
        y, total, inverse = add_rms_norm_forward(x, residual, weight, eps)
        if residual is None:
            total = x.view_as(x)
        ctx.dtype = x.dtype
        ctx.save_for_backward(total, weight, inverse)
        return y, total

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_y, grad_sum):
        total, weight, inverse = ctx.saved_tensors
        need = ctx.needs_input_grad
        return (*add_rms_norm_backward(total, weight, inverse, grad_y, grad_sum, ctx.dtype, *need[:3]),
                None)


def add_rms_norm(
    x: torch.Tensor, residual: torch.Tensor | None, weight: torch.Tensor, eps: float = 1e-6
) -> tuple[torch.Tensor, torch.Tensor]:
    """``(y, s)`` of the norm over the last dimension of ``s = x + residual``
    (``residual`` None: s is x); differentiable in x, residual and weight.
    ``x`` is float32, float16 or bfloat16; residual and weight have its type or
    float32."""
    return _AddRmsNorm.apply(x, residual, weight, eps)


def add_rms_norm_quant(
    x: torch.Tensor, residual: torch.Tensor | None, weight: torch.Tensor, eps: float = 1e-6,
    format: str = "int8",
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """``(codes, scales, s)``: the norm's output in 8 bits for serving, one
    float32 scale per row; ``format`` is "int8" (scale max|y| / 127) or "e4m3"
    (max|y| / 448, torch.float8_e4m3fn).  A row of zeros has scale 0, a row that
    holds a NaN a NaN scale.  Not differentiable."""
    if format not in _CODES:
        raise ValueError(f"format must be one of {sorted(_CODES)}, got {format!r}")
    _check(x, residual, weight, eps)
    device = nat.require_gpu(x, weight) if residual is None else nat.require_gpu(x, residual, weight)
    code, dtype = _CODES[format]
    x2 = _rows(x)
    r2 = None if residual is None else _rows(residual)
    weight = weight.contiguous()
    rows, width = x2.shape
    kept = x.dtype if residual is None else residual.dtype
    codes = torch.empty(x.shape, dtype=dtype, device=device)
    scales = torch.empty(x.shape[:-1], dtype=torch.float32, device=device)
    total = x if residual is None else torch.empty(x.shape, dtype=kept, device=device)
    nat.check(
        nat.library().gs_add_rms_norm_quant(
            x2.data_ptr(), None if r2 is None else r2.data_ptr(), weight.data_ptr(), rows, width,
            x2.stride(0), 0 if r2 is None else r2.stride(0), nat.TYPES[x.dtype], nat.TYPES[kept],
            nat.TYPES[weight.dtype], eps, code, codes.data_ptr(), scales.data_ptr(),
            None if residual is None else total.data_ptr(), nat.stream(device),
        ),
        "add_rms_norm_quant",
    )
    return codes, scales, total
