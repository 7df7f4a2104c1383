"""add_rms_norm on the GPU against its definition in float64.

Bounds.  In float32 a row's sum of squares passes through chains of at most
45 additions (32 in a thread, 6 in the wave, 4 over the waves), the factor
1 / sqrt(.) halves its relative error and adds a few roundings, so y is within
40 u32 relative before its one rounding to the type u.  Rows beyond 8192 add
width / 256 terms in a thread.  The backward reads the sum rounded to its type
(unit v): with unit = s r, t = grad_y w, m = mean|t unit|, grad_s is within
r (|unit| m (4 v + 90 u32) + 4 u32 |t|) + u32 |grad_sum| of its own before the
rounding, and grad_w within the sum over the rows of |grad_y unit| (2 v + (rows + 60) u32).
"""

from __future__ import annotations

import pytest
import torch

from gaussian_splats_hip.sequence import add_rms_norm, add_rms_norm_backward, add_rms_norm_quant
from oracle import sequence as orc
from sequence_helpers import TINY, TYPES, U32, UNIT, assert_within, normal

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")
EPS = 1e-6


def _chain(width):
    return 45 + (width // 256 if width > 8192 else 0)


def _y_bound(y, dtype, width):
    return y.abs() * (UNIT[dtype] + _chain(width) * U32) + TINY[dtype]


def _check(x, residual, weight, dy, dsum, eps=EPS):
    """Forward and backward of device copies against the definition."""
    width = x.shape[-1]
    d = [None if t is None else t.detach().to(DEV).requires_grad_(True) for t in (x, residual, weight)]
    y, s = add_rms_norm(*d, eps)
    leaves = [t for t in d if t is not None]
    grads = torch.autograd.grad((y, s), leaves, (dy.to(DEV), dsum.to(DEV)))
    want_y, want_s = orc.add_rms_norm(x, residual, weight, eps)
    kept = x.dtype if residual is None else residual.dtype
    assert y.dtype == x.dtype and s.dtype == kept
    assert_within(y, want_y, _y_bound(want_y, x.dtype, width), "y")
    assert_within(s, want_s, want_s.abs() * (UNIT[kept] + 2 * U32) + TINY[kept], "sum")
    ds, dw = orc.add_rms_norm_grads(x, residual, weight, eps, dy, dsum)
    r = 1 / torch.sqrt((want_s * want_s).mean(-1, keepdim=True) + eps)
    unit, t = (want_s * r).abs(), (dy.double() * weight.double()).abs()
    v = 0.0 if residual is None else UNIT[kept]
    n = 2 * _chain(width) * U32
    own = r * (unit * (t * unit).mean(-1, keepdim=True) * (4 * v + n) + 4 * U32 * t)
    own = own + U32 * (dsum.double().abs() + ds.abs())
    assert_within(grads[0], ds, own + ds.abs() * UNIT[x.dtype] + TINY[x.dtype], "grad x")
    if residual is not None:
        assert_within(grads[1], ds, own + ds.abs() * UNIT[kept] + TINY[kept], "grad residual")
    rows = x.numel() // width
    sums = (dy.double().abs() * unit).reshape(-1, width).sum(0)
    bound = sums * (2 * v + (rows + _chain(width) + 15) * U32) + dw.abs() * UNIT[weight.dtype]
    assert_within(grads[-1], dw, bound + TINY[weight.dtype], "grad weight")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(1, 1), (3, 7), (5, 64), (2, 3, 768), (6, 1000), (4, 1024),
                                   (3, 1032), (2, 2049), (3, 8192), (2, 8200), (1030, 24)])
def test_matches_definition(shape, dtype):
    print(f"[norm] {shape} {dtype}", flush=True)
    x, dy = normal(shape, dtype, 1), normal(shape, dtype, 2)
    w = normal(shape[-1:], dtype, 3, 0.2, 1.0)
    _check(x, normal(shape, dtype, 4, 2.0), w, dy, normal(shape, dtype, 5))
    _check(x, None, w.float(), dy, normal(shape, dtype, 6))
    if dtype != torch.float32:
        _check(x, normal(shape, torch.float32, 7, 2.0), w, dy, normal(shape, torch.float32, 8))


def test_strides_and_alignment():
    """Rows apart, a residual that is one row repeated, an offset of one element."""
    wide = normal((9, 200), torch.bfloat16, 1).to(DEV)
    w = normal((96,), torch.bfloat16, 2, 0.1, 1.0).to(DEV)
    for x in (wide[:, 40:136], wide[:, 1:97], wide[::2, 8:104], wide.T[:96].T):
        one = normal((96,), torch.bfloat16, 3).to(DEV).requires_grad_(True)
        res = one.expand(x.shape)
        y, s = add_rms_norm(x, res, w, EPS)
        want, want_s = orc.add_rms_norm(x.cpu(), res.detach().cpu(), w.cpu(), EPS)
        assert_within(y, want, _y_bound(want, torch.bfloat16, 96), "y")
        (grad,) = torch.autograd.grad((y, s), one, (torch.ones_like(y), torch.ones_like(s)))
        ds, _ = orc.add_rms_norm_grads(x.cpu(), res.detach().cpu(), w.cpu(), EPS,
                                       torch.ones(x.shape), torch.ones(x.shape))
        # Each row's gradient is rounded to bfloat16, then their sum is.
        u = UNIT[torch.bfloat16]
        assert_within(grad, ds.sum(0), 4 * u * ds.abs().sum(0) + 4 * u * x.shape[0], "repeated row")


def test_gradient_by_differences():
    """The kernels' gradient against differences of the definition."""
    x, w, dy = (normal(s, torch.float32, i) for i, s in ((1, (2, 40)), (2, (40,)), (3, (2, 40))))
    d = [t.to(DEV).requires_grad_(True) for t in (x, w)]
    y, _ = add_rms_norm(d[0], None, d[1], EPS)
    gx, gw = torch.autograd.grad(y, d, dy.to(DEV))
    h = 1e-5
    for t, g in ((x, gx), (w, gw)):
        for i in range(0, t.numel(), 7):
            step = torch.zeros(t.numel(), dtype=torch.float64)
            step[i] = h
            step = step.view(t.shape)
            f = [float((orc.add_rms_norm(x.double() + (e * step if t is x else 0), None,
                                         w.double() + (e * step if t is w else 0), EPS)[0]
                        * dy.double()).sum()) for e in (1, -1)]
            # Truncation h^2 times third derivatives of order 10; float32 rounding of the gradient.
            assert abs((f[0] - f[1]) / (2 * h) - float(g.view(-1)[i])) <= 1e-5


@pytest.mark.parametrize("dtype", TYPES)
def test_missing_gradients(dtype):
    """Only one of the outputs used, and leaves that need no gradient."""
    x, res = normal((5, 72), dtype, 1).to(DEV), normal((5, 72), dtype, 2).to(DEV)
    w = normal((72,), dtype, 3).to(DEV)
    zero = torch.zeros(5, 72)
    for dy, dsum in ((normal((5, 72), dtype, 4), None), (None, normal((5, 72), dtype, 5))):
        from gaussian_splats_hip.sequence import add_rms_norm_forward

        _, total, inverse = add_rms_norm_forward(x, res, w, EPS)
        gx, gr, gw = add_rms_norm_backward(total, w, inverse, None if dy is None else dy.to(DEV),
                                           None if dsum is None else dsum.to(DEV), dtype)
        ds, dw = orc.add_rms_norm_grads(total.cpu(), None, w.cpu(), EPS, zero if dy is None else dy,
                                        zero if dsum is None else dsum)
        u = UNIT[dtype]
        # The norm of the sum that was rounded: within a few of its roundings.
        assert_within(gx, ds, 4 * u * (1 + ds.abs().max()), "grad x")
        assert torch.equal(gx, gr)
        assert_within(gw, dw, 4 * u * (1 + dw.abs().max()), "grad weight")
        assert add_rms_norm_backward(total, w, inverse, None, None, dtype, False, False, True)[:2] == (None, None)


@pytest.mark.parametrize("format,top", [("int8", 127.0), ("e4m3", 448.0)])
@pytest.mark.parametrize("shape", [(1, 8), (3, 100), (4, 1024), (5, 1504), (2, 5000), (2, 9001)])
def test_quant(shape, format, top):
    """Codes within half a step of y / scale (e4m3: half the spacing at the
    value), and the scale that of the largest value."""
    x, res = normal(shape, torch.bfloat16, 1), normal(shape, torch.float32, 2)
    w = normal(shape[-1:], torch.bfloat16, 3, 0.2, 1.0)
    codes, scales, s = add_rms_norm_quant(x.to(DEV), res.to(DEV), w.to(DEV), EPS, format)
    y, want_s = orc.add_rms_norm(x, res, w, EPS)
    n = (_chain(shape[-1]) + 4) * U32
    assert codes.dtype == (torch.int8 if format == "int8" else torch.float8_e4m3fn)
    assert_within(s, want_s, want_s.abs() * 3 * U32, "sum")
    scale = y.abs().amax(-1) / top
    assert_within(scales, scale, scale * n, "scale")
    z = y / scale[..., None]
    spacing = (torch.ones_like(z) if format == "int8"
               else torch.exp2(torch.floor(torch.log2(z.abs().clamp_min(2.0**-6))) - 3))
    # At a binade's lower edge float32 may land in the coarser side's neighbour.
    assert_within(codes.float(), z, spacing * 0.5 + z.abs() * 2 * n, "codes")
    assert float(codes.float().abs().max()) == top


def test_quant_zero_and_nan_rows():
    x = normal((4, 256), torch.bfloat16, 1)
    x[1] = 0
    x[2, 5] = float("nan")
    w = torch.ones(256)
    for format in ("int8", "e4m3"):
        codes, scales, _ = add_rms_norm_quant(x.to(DEV), None, w.to(DEV), EPS, format)
        assert float(scales[1]) == 0 and not codes[1].float().any()
        assert torch.isnan(scales[2]) and torch.isfinite(scales[[0, 1, 3]]).all()


def test_infinite_and_nan_values_stay_in_their_row():
    x = normal((6, 768), torch.float32, 1)
    x[2, 7], x[4, 9] = float("inf"), float("nan")
    y, _ = add_rms_norm(x.to(DEV), None, torch.ones(768, device=DEV), EPS)
    want, _ = orc.add_rms_norm(x, None, torch.ones(768), EPS)
    assert_within(y[[0, 1, 3, 5]], want[[0, 1, 3, 5]], _y_bound(want[[0, 1, 3, 5]], torch.float32, 768), "y")
    assert torch.isnan(y[2, 7]) and torch.isnan(y[4]).all()


def test_same_bits_again_and_on_another_stream():
    x, dy = normal((2000, 512), torch.bfloat16, 1).to(DEV), normal((2000, 512), torch.bfloat16, 2).to(DEV)
    w = normal((512,), torch.float32, 3).to(DEV)

    def once():
        a, b = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
        y, s = add_rms_norm(a, None, b, EPS)
        return (y, *torch.autograd.grad((y, s), (a, b), (dy, dy)))

    first = once()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = once()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for a, b in zip(first, second):
        assert torch.equal(a, b)


def test_empty():
    x = torch.zeros(0, 64, device=DEV, requires_grad=True)
    w = torch.ones(64, device=DEV, requires_grad=True)
    y, s = add_rms_norm(x, None, w, EPS)
    gx, gw = torch.autograd.grad((y, s), (x, w), (y.detach(), s.detach()))
    assert y.shape == gx.shape == (0, 64) and not gw.any()
