"""The gradient norm, clipping and FusedAdam's limit on the GPU against float64.

Bounds.  Squares and sums are float64, so the norm is off by its rounding to
float32 alone (U32, and n 2^-53 from the sum).  The factor is rounded to float32,
its product with a value once more, the result to the type: UNIT + 2 U32 relative.
Adam's moments take two and three float32 operations of the scaled gradient, the
update four more; each adds U32 of the largest operand.
"""

from __future__ import annotations

import pytest
import torch

from gaussian_splats_hip.training import FusedAdam, clip_grad_norm, grad_norm
from sequence_helpers import TINY, TYPES, U32, UNIT, assert_within, normal

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")
NORM = U32 * (1 + 2.0**-10)


def _norm64(tensors):
    return float(sum(t.detach().cpu().double().square().sum() for t in tensors)) ** 0.5


def _parameters(grads):
    out = []
    for g in grads:
        p = torch.nn.Parameter(torch.zeros(g.shape, dtype=g.dtype, device=DEV))
        p.grad = g.to(DEV)
        out.append(p)
    return out


SIZES = [1, 0, 7, 4096, 4095, 8192, 8193, 100_003, 12_288, 33]


@pytest.mark.parametrize("count", [1, 3, 10, 128, 129, 300])
@pytest.mark.parametrize("limit", [0.5, 1e9])
def test_norm_and_clip(count, limit):
    print(f"[clip] {count} {limit}", flush=True)
    grads = [normal((SIZES[i % len(SIZES)],), TYPES[i % 3], i, 0.1 * (1 + i % 5)) for i in range(count)]
    want = _norm64(grads)
    params = _parameters(grads)
    assert_within(grad_norm([p.grad for p in params]), torch.tensor(want), want * NORM, "norm")
    got = clip_grad_norm(params, limit)
    assert got.dtype == torch.float32 and got.shape == () and got.device == DEV
    assert_within(got, torch.tensor(want), want * NORM, "norm")
    factor = min(1.0, limit / (want + 1e-6))
    for p, g in zip(params, grads):
        if factor == 1.0:
            assert torch.equal(p.grad.cpu(), g)
        else:
            exact = g.double() * factor
            assert_within(p.grad, exact, exact.abs() * (UNIT[g.dtype] + 2 * NORM) + TINY[g.dtype], "gradient")


@pytest.mark.parametrize("dtype", TYPES)
def test_addresses_off_16_bytes(dtype):
    """Views that start anywhere; what lies beside them stays."""
    base = normal((3 * 20_000,), dtype, 1).to(DEV)
    before = base.clone()
    views = [base[1:9000], base[20_003:38_200], base[40_000:40_001]]
    params = [torch.nn.Parameter(torch.zeros_like(v)) for v in views]
    for p, v in zip(params, views):
        p.grad = v
    want = _norm64(views)
    got = clip_grad_norm(params, 1.0)
    assert_within(got, torch.tensor(want), want * NORM, "norm")
    touched = torch.zeros(base.shape, dtype=torch.bool, device=DEV)
    for lo, hi in ((1, 9000), (20_003, 38_200), (40_000, 40_001)):
        touched[lo:hi] = True
    assert torch.equal(base[~touched], before[~touched])
    exact = before.double()[touched] / (want + 1e-6)
    assert_within(base[touched], exact, exact.abs() * (UNIT[dtype] + 2 * NORM) + TINY[dtype], "gradient")


def test_sizes_whose_squares_float32_does_not_hold():
    big, small = torch.full((1000,), 1e30), torch.full((50_000,), 1e-30)
    assert_within(grad_norm(big.to(DEV)), torch.tensor(_norm64([big])), _norm64([big]) * NORM, "norm")
    assert_within(grad_norm(small.to(DEV)), torch.tensor(_norm64([small])), _norm64([small]) * NORM, "norm")
    (p,) = _parameters([big])
    clip_grad_norm([p], 1.0)
    exact = big.double() / _norm64([big])
    assert_within(p.grad, exact, exact * 4 * NORM, "gradient")


def test_not_finite():
    """As torch.nn.utils.clip_grad_norm_ has it."""
    for value in (float("inf"), -float("inf"), float("nan")):
        grads = [normal((5000,), torch.float32, 1), normal((70,), torch.bfloat16, 2)]
        grads[0][4321] = value
        params = _parameters(grads)
        norm = clip_grad_norm(params, 1.0)
        others = [torch.nn.Parameter(torch.zeros_like(g)) for g in grads]
        for p, g in zip(others, grads):
            p.grad = g.clone()
        want = torch.nn.utils.clip_grad_norm_(others, 1.0)
        assert torch.equal(norm.cpu().isnan(), want.isnan()) and torch.equal(norm.cpu().isinf(), want.isinf())
        for p, o in zip(params, others):
            torch.testing.assert_close(p.grad.cpu(), o.grad, equal_nan=True, rtol=0, atol=0)


def test_limits_at_the_ends():
    g = normal((1000,), torch.float32, 3)
    (p,) = _parameters([g])
    clip_grad_norm(p, float("inf"))
    assert torch.equal(p.grad.cpu(), g)
    clip_grad_norm(p, 0.0)
    assert torch.equal(p.grad.cpu(), torch.zeros(1000))
    assert float(clip_grad_norm(p, 1.0)) == 0.0  # a norm of zero divides nothing


def test_layouts():
    """Dimensions in another order are flat memory; gaps take a copy; a gradient met
    twice counts once."""
    a = normal((6, 50, 7), torch.float32, 1).to(DEV)
    b = normal((40, 90), torch.bfloat16, 2).to(DEV)
    rest = b[:, 50:].clone()
    params = [torch.nn.Parameter(torch.zeros(7, 6, 50, device=DEV)),
              torch.nn.Parameter(torch.zeros(40, 50, dtype=torch.bfloat16, device=DEV))]
    params[0].grad, params[1].grad = a.permute(2, 0, 1), b[:, :50]
    grads = [p.grad.cpu() for p in params]
    versions = [p.grad._version for p in params]
    want = _norm64(grads)
    assert_within(grad_norm([p.grad for p in params]), torch.tensor(want), want * NORM, "norm")
    got = clip_grad_norm([*params, params[0]], 1.0)
    assert_within(got, torch.tensor(want), want * NORM, "norm")
    for p, g, v in zip(params, grads, versions):
        exact = g.double() / (want + 1e-6)
        assert_within(p.grad, exact, exact.abs() * (UNIT[g.dtype] + 2 * NORM), "gradient")
        assert p.grad._version > v
    assert torch.equal(b[:, 50:], rest)


def test_overlaps_are_refused():
    base = torch.ones(100, device=DEV)
    params = [torch.nn.Parameter(torch.zeros(60, device=DEV)) for _ in range(2)]
    params[0].grad, params[1].grad = base[:60], base[40:]
    with pytest.raises(ValueError, match="overlap"):
        clip_grad_norm(params, 1.0)
    params[1].grad = torch.ones(1, device=DEV).expand(60)
    with pytest.raises(ValueError, match="expanded"):
        clip_grad_norm(params, 1.0)
    assert torch.equal(base, torch.ones(100, device=DEV))
    assert_within(grad_norm(params[1].grad), torch.tensor(60.0**0.5), 8 * NORM, "norm")


def test_streams_and_graphs():
    """A captured clip scales whatever the gradients hold at the replay."""
    grads = [normal((9000,), torch.float32, 1), normal((333,), torch.float16, 2)]
    params = _parameters(grads)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        clip_grad_norm(params, 1.0)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = clip_grad_norm(params, 1.0)
    for turn in range(3):
        fresh = [normal(g.shape, g.dtype, 10 + turn, 1.0 + turn) for g in grads]
        for p, g in zip(params, fresh):
            p.grad.copy_(g)
        graph.replay()
        torch.cuda.synchronize()
        eager = _parameters(fresh)
        assert torch.equal(norm, clip_grad_norm(eager, 1.0))
        for p, e in zip(params, eager):
            assert torch.equal(p.grad, e.grad)


@pytest.mark.parametrize("weight_decay", [0.0, 0.1])
@pytest.mark.parametrize("limit", [0.5, 1e9])
def test_adam_with_a_limit(limit, weight_decay):
    shapes = [(1000, 3), (17,), (40, 9, 3), (3,), (1,), (5, 5), (9,), (70_000,), (2, 2), (11,)]
    start = [normal(s, torch.float32, i) for i, s in enumerate(shapes)]
    params = [torch.nn.Parameter(t.to(DEV)) for t in start]
    rates = (1e-2, 3e-3)
    opt = FusedAdam([{"params": params[:4], "lr": rates[0]},
                     {"params": params[4:], "lr": rates[1], "betas": (0.8, 0.99)}],
                    eps=1e-8, weight_decay=weight_decay, max_norm=limit)
    state = [[t.double(), torch.zeros_like(t).double(), torch.zeros_like(t).double()] for t in start]
    slip = [torch.zeros_like(t).double() for t in start]
    for step in range(1, 4):
        grads = [normal(s, torch.float32, 100 * step + i) for i, s in enumerate(shapes)]
        for p, g in zip(params, grads):
            p.grad = g.to(DEV)
        opt.step()
        want = _norm64(grads)
        assert_within(opt.grad_norm, torch.tensor(want), want * NORM, "norm")
        for i, (p, g) in enumerate(zip(params, grads)):
            assert torch.equal(p.grad.cpu(), g)  # left as it was
            b1, b2 = (0.9, 0.999) if i < 4 else (0.8, 0.99)
            x, m, v = state[i]
            scaled = g.double() * min(1.0, limit / (want + 1e-6))
            h = scaled + weight_decay * x
            m = b1 * m + (1 - b1) * h
            v = b2 * v + (1 - b2) * h * h
            denominator = (v / (1 - b2**step)).sqrt() + 1e-8
            update = (rates[0] if i < 4 else rates[1]) / (1 - b1**step) * m / denominator
            # h is off by U32 of both of its operands, however much of them cancels: fl(a +
            # b) with a, b of relative error U32 has |error| <= 2 U32 (|a| + |b|).  The
            # moments and the update pass that on divided by the denominator.
            operands = scaled.abs() + weight_decay * x.abs()
            size = update.abs() + (rates[0] if i < 4 else rates[1]) * operands / denominator
            slip[i] = slip[i] + U32 * (x.abs() + 40 * step * size)
            state[i] = [x - update, m, v]
            # A parameter's own error joins the next gradient with the weight decay.
            assert_within(p, state[i][0], slip[i] * (1 + weight_decay), f"parameter {i}, step {step}")
    empty = FusedAdam([torch.nn.Parameter(torch.zeros(3, device=DEV))], max_norm=1.0)
    empty.step()
    assert empty.grad_norm is None


def test_adam_within_the_limit_keeps_its_bits():
    start, g = normal((12_345,), torch.float32, 1), normal((12_345,), torch.float32, 2)
    out = []
    for limit in (None, 1e6):
        p = torch.nn.Parameter(start.to(DEV))
        opt = FusedAdam([p], lr=1e-2, max_norm=limit)
        for _ in range(3):
            p.grad = g.to(DEV)
            opt.step()
        out.append(p.detach())
    assert torch.equal(*out)


def test_adam_counts_a_shared_gradient_once():
    """One gradient of two parameters counts once, in any layout; two gradients that
    begin at one place and have different shapes are two."""
    held = normal((6, 20), torch.float32, 1).to(DEV)
    for first, second, count in ((held, held, 1), (held.t(), held.t(), 1), (held[:3], held, None)):
        params = [torch.nn.Parameter(torch.zeros(g.shape, device=DEV)) for g in (first, second)]
        for p, g in zip(params, (first, second)):
            p.grad = g
        opt = FusedAdam(params, max_norm=1.0)
        opt.step()
        want = _norm64([first.cpu()] if count else [first.cpu(), second.cpu()])
        assert_within(opt.grad_norm, torch.tensor(want), want * NORM, "norm")


def test_adam_norm_is_the_last_steps():
    """Steps with a gradient, without one and with one again."""
    p = torch.nn.Parameter(torch.zeros(50, device=DEV))
    opt = FusedAdam([p], max_norm=1.0)
    for seed in (1, None, 2):
        p.grad = None if seed is None else normal((50,), torch.float32, seed).to(DEV)
        before = p.detach().clone()
        opt.step()
        if seed is None:
            assert opt.grad_norm is None and torch.equal(p.detach(), before)
        else:
            want = _norm64([p.grad])
            assert_within(opt.grad_norm, torch.tensor(want), want * NORM, "norm")
