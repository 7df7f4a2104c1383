"""gated_scan on the GPU against its definition in float64.

Bounds.  A step's arithmetic has a relative error of at most 10 u32 (exp,
reciprocal, two products and a sum; a's own error included), and h is a convex
combination of what it has seen, so after n steps the error is at most
10 u32 m max|h|, where m = min(n, 1 / (1 - max a)) steps are remembered; cutting
the sequence adds one map a run and a chunk, at most doubling it.  y is then
rounded once.  The carried gradient has the same memory: with g the largest sum of
remembered gradients, its error is at most 20 u32 m g.
"""

from __future__ import annotations

import pytest
import torch

from gaussian_splats_hip.sequence import gated_scan, gated_scan_backward, gated_scan_forward, gated_scan_step
from oracle import sequence as orc
from sequence_helpers import TINY, TYPES, U32, UNIT, assert_within, normal

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")


def _memory(gate, tokens):
    return min(tokens, float(1 / torch.sigmoid(-gate.double()).min().clamp_min(1e-9)))


def _check(x, gate, state, dy, dlast):
    dtype = x.dtype
    d = [None if t is None else t.detach().to(DEV).requires_grad_(True) for t in (x, gate, state)]
    y, last = gated_scan(*d)
    grads = torch.autograd.grad((y, last), [t for t in d if t is not None],
                                (dy.to(DEV), dlast.to(DEV)))
    want, want_last = orc.gated_scan(x, gate, state)
    assert y.dtype == dtype and last.dtype == torch.float32
    m = _memory(gate, x.shape[1])
    top = max(float(x.abs().max()), 0.0 if state is None else float(state.abs().max()))
    own = 20 * U32 * m * top
    assert_within(y, want, want.abs() * UNIT[dtype] + own + TINY[dtype], "y")
    assert_within(last, want_last, want_last.abs() * U32 + own, "last")
    gx, gg, gs = orc.gated_scan_grads(x, gate, state, dy, dlast)
    # The largest carried gradient, by the same recurrence over magnitudes.
    mx, _, ms = orc.gated_scan_grads(x, gate, state, dy.abs(), dlast.abs())
    g = float((mx / torch.sigmoid(-gate.double())).max())
    slip = 20 * U32 * m * g
    keep = torch.sigmoid(-gate.double())
    assert_within(grads[0], gx, gx.abs() * UNIT[dtype] + keep * slip + 20 * U32 * mx + TINY[dtype], "grad x")
    slope = keep * (1 - keep)
    bound = slope * (2 * top * slip + g * 2 * own + 40 * U32 * g * top)
    assert_within(grads[1], gg, gg.abs() * UNIT[dtype] + bound + TINY[dtype], "grad gate")
    if state is not None:
        assert_within(grads[2], gs, gs.abs() * U32 + slip, "grad state")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(1, 1, 1), (2, 2, 3), (1, 15, 64), (3, 17, 130), (1, 31, 127),
                                   (2, 33, 128), (1, 255, 66), (1, 256, 70), (2, 257, 129),
                                   (1, 511, 8), (1, 1300, 40), (2, 3333, 6)])
def test_matches_definition(shape, dtype):
    print(f"[scan] {shape} {dtype}", flush=True)
    b, t, c = shape
    x, gate = normal(shape, dtype, 1), normal(shape, dtype, 2, 2.0, 3.0)
    dy, dlast = normal(shape, dtype, 3), normal((b, c), torch.float32, 4)
    _check(x, gate, normal((b, c), torch.float32, 5), dy, dlast)
    _check(x, gate, None, dy, dlast)


def test_long_memory():
    """Gates near one for thousands of tokens; a chunk's product underflows in others."""
    x = normal((1, 5000, 4), torch.float32, 1)
    gate = torch.tensor([14.0, 9.0, 0.0, -9.0]).expand(1, 5000, 4).contiguous()
    _check(x, gate, normal((1, 4), torch.float32, 2), normal((1, 5000, 4), torch.float32, 3),
           normal((1, 4), torch.float32, 4))


@pytest.mark.parametrize("dtype", TYPES)
def test_gates_at_infinity(dtype):
    """-inf forgets (h = x, no gradient through the state), +inf keeps h whole."""
    shape = (1, 600, 10)
    x, gate = normal(shape, dtype, 1), normal(shape, dtype, 2, 2.0, 3.0)
    gate[0, 300] = -float("inf")
    gate[0, 301:420] = float("inf")
    d = [t.to(DEV).requires_grad_(True) for t in (x, gate)]
    y, last = gated_scan(*d)
    assert torch.equal(y[0, 300:420].cpu(), x[0, 300].expand(120, 10))
    _check(x, gate, None, normal(shape, dtype, 3), normal((1, 10), torch.float32, 4))


@pytest.mark.parametrize("dtype", TYPES)
def test_gates_of_any_size(dtype):
    """Gates far beyond what an exponential holds, and where it is about to
    overflow: forgetting keeps x, remembering keeps h, a NaN stays in its channel."""
    sizes = [-6e4, -120.0, -104.0, -90.0, -89.0, -88.5, -88.0, -87.5, -87.0, -80.0, -70.0, -69.0, -40.0,
             -10.0, 0.0, 10.0, 40.0, 70.0, 80.0, 87.0, 88.0, 89.0, 104.0, 120.0, 6e4]
    gate = torch.tensor(sizes).to(dtype).expand(1, 9, -1).contiguous()
    x, state = normal(gate.shape, dtype, 1), normal((1, len(sizes)), torch.float32, 2)
    _check(x, gate, state, normal(gate.shape, dtype, 3), normal((1, len(sizes)), torch.float32, 4))
    row, _ = gated_scan_step(x[:, 0].to(DEV), gate[:, 0].to(DEV), state.to(DEV))
    want, _ = orc.gated_scan(x[:, :1], gate[:, :1], state)
    assert_within(row, want[:, 0], want[:, 0].abs() * UNIT[dtype] + 40 * U32 * 4, "step")
    gate[0, 4, 3] = float("nan")
    y, _ = gated_scan(x.to(DEV), gate.to(DEV), state.to(DEV))
    bad = torch.isnan(y[0].cpu())
    assert bad[4:, 3].all() and int(bad.sum()) == 5


def test_offsets_beyond_32_bits():
    """Sequences whose tensors lie more than 2^31 elements apart."""
    apart, shape = (1 << 31) + 64, (2, 40, 16)
    far = [torch.empty(apart + 640, dtype=torch.bfloat16, device=DEV).as_strided(shape, (apart, 16, 1))
           for _ in range(3)]
    near = [normal(shape, torch.bfloat16, i).to(DEV) for i in range(3)]
    for a, b in zip(far, near):
        a.copy_(b)
    out = [gated_scan_forward(*t[:2]) for t in (far, near)]
    grads = [gated_scan_backward(t[0], t[1], o[2], t[2], None) for t, o in zip((far, near), out)]
    for a, b in zip((*out[0], *grads[0]), (*out[1], *grads[1])):
        assert torch.equal(a, b)


def test_strides_and_alignment():
    base = normal((3, 700, 300), torch.bfloat16, 1).to(DEV)
    for x in (base[:, :, 40:140], base[:, :, 1:100], base[:, ::2, 10:110], base[:, :, :7],
              base.transpose(0, 1), base[:1].expand(4, -1, -1)[:, :, 2:50],
              base.transpose(1, 2)[:, :, ::7]):
        gate = (x * 2 + 3)
        want, want_last = orc.gated_scan(x.cpu(), gate.cpu())
        y, last = gated_scan(x, gate)
        m = _memory(gate.cpu(), x.shape[1])
        top = float(x.abs().max())
        assert_within(y, want, want.abs() * UNIT[torch.bfloat16] + 20 * U32 * m * top, "y")
        dy = torch.ones_like(want).to(torch.bfloat16).to(DEV)
        again = gated_scan_forward(x.contiguous(), gate.contiguous())
        a = gated_scan_backward(x, gate, again[2], dy.transpose(0, 1).contiguous().transpose(0, 1), None)
        b = gated_scan_backward(x.contiguous(), gate.contiguous(), again[2], dy, None)
        # Vector and scalar lanes do the same arithmetic.
        assert torch.equal(y, again[0])
        for p, q in zip(a, b):
            assert torch.equal(p, q)


def test_gradient_by_differences():
    shape = (1, 37, 3)
    x, gate, dy = (normal(shape, torch.float32, i) for i in (1, 2, 3))
    state = normal((1, 3), torch.float32, 4)
    d = [t.to(DEV).requires_grad_(True) for t in (x, gate, state)]
    grads = torch.autograd.grad(gated_scan(*d)[0], d, dy.to(DEV))
    h = 1e-5
    for k, t in enumerate((x, gate, state)):
        for i in range(0, t.numel(), 11):
            step = torch.zeros(t.numel(), dtype=torch.float64)
            step[i] = h
            f = []
            for e in (1, -1):
                args = [u.double() + (e * step.view(t.shape) if u is t else 0) for u in (x, gate, state)]
                f.append(float((orc.gated_scan(*args)[0] * dy.double()).sum()))
            assert abs((f[0] - f[1]) / (2 * h) - float(grads[k].view(-1)[i])) <= 1e-5


def test_missing_gradients():
    shape = (2, 300, 20)
    x, gate = normal(shape, torch.bfloat16, 1).to(DEV), normal(shape, torch.bfloat16, 2).to(DEV)
    _, _, starts = gated_scan_forward(x, gate)
    dy, dlast = normal(shape, torch.bfloat16, 3).to(DEV), normal((2, 20), torch.float32, 4).to(DEV)
    for a, b in ((None, dlast), (dy, None), (None, None)):
        got = gated_scan_backward(x, gate, starts, a, b)
        full = gated_scan_backward(x, gate, starts, torch.zeros_like(x) if a is None else a,
                                   torch.zeros_like(dlast) if b is None else b)
        for p, q in zip(got, full):
            assert torch.equal(p, q)
    assert gated_scan_backward(x, gate, starts, dy, None, need_state=False)[2] is None


@pytest.mark.parametrize("dtype", TYPES)
def test_step_continues_the_scan(dtype):
    """Steps from the scan's last state equal a longer scan's rows."""
    shape = (3, 300, 34)
    x, gate = normal(shape, dtype, 1).to(DEV), normal(shape, dtype, 2, 2.0, 3.0).to(DEV)
    y, last = gated_scan(x, gate)
    _, state = gated_scan(x[:, :296], gate[:, :296])
    own = 20 * U32 * float(x.abs().max()) * 8
    for t in range(296, 300):
        want, _ = orc.gated_scan(x[:, t:t + 1].cpu(), gate[:, t:t + 1].cpu(), state.cpu())
        row, state = gated_scan_step(x[:, t], gate[:, t], state, state_out=state)
        assert_within(row, want[:, 0], want[:, 0].abs() * UNIT[dtype] + own, "step")
    assert_within(state, last, last.abs() * 8 * U32 + own, "state")


def test_same_bits_again_and_on_another_stream():
    shape = (2, 4000, 200)
    x, gate = normal(shape, torch.bfloat16, 1).to(DEV), normal(shape, torch.bfloat16, 2, 2.0, 3.0).to(DEV)

    def once():
        a, b = x.clone().requires_grad_(True), gate.clone().requires_grad_(True)
        y, last = gated_scan(a, b)
        return (y, last, *torch.autograd.grad((y, last), (a, b), (x, last.detach())))

    first = once()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = once()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for a, b in zip(first, second):
        assert torch.equal(a, b)


def test_scan_in_a_graph():
    """Replays of a captured scan and its backward on new inputs, with eager work
    between them, equal eager calls."""
    shape = (2, 700, 130)
    x, gate, dy = (normal(shape, torch.bfloat16, i).to(DEV) for i in range(3))

    def both():
        y, last, starts = gated_scan_forward(x, gate)
        return y, last, *gated_scan_backward(x, gate, starts, dy, last)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = both()
    for t in range(4):
        for i, v in enumerate((x, gate, dy)):
            v.copy_(normal(shape, torch.bfloat16, 10 * t + i))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, both()):
            assert torch.equal(a, b), t


def test_empty():
    state = torch.ones(2, 5, device=DEV, requires_grad=True)
    x = torch.zeros(2, 0, 5, device=DEV, requires_grad=True)
    y, last = gated_scan(x, x.detach(), state)
    (g,) = torch.autograd.grad(last, state, torch.ones_like(last))
    assert y.shape == x.shape and torch.equal(last, state) and torch.equal(g, torch.ones_like(g))
    y, last = gated_scan(torch.zeros(0, 4, 5, device=DEV), torch.zeros(0, 4, 5, device=DEV))
    assert y.shape == (0, 4, 5) and last.shape == (0, 5)


def test_waits_end_by_themselves():
    """Long scans leave no bit of a failed wait behind."""
    from gaussian_splats_hip.kernels.rasterize import _native as nat

    nat.device_errors(DEV)
    shape = (2, 40000, 512)
    x, gate = (normal(shape, torch.bfloat16, i, s, m).to(DEV) for i, s, m in ((1, 1.0, 0.0), (2, 2.0, 3.0)))
    y, last, starts = gated_scan_forward(x, gate)
    grads = gated_scan_backward(x, gate, starts, x, last)
    for t in (y, last, *grads):
        assert torch.isfinite(t).all()
    assert nat.device_errors(DEV) == 0
