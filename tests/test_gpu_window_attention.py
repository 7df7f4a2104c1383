"""window_attention on the GPU against its definition in float64.

Bounds, with u the type's unit, U that of float32, n the keys a query sees and d
the head dimension.  A score is a sum of d products in float32, its exponent
takes two more roundings of a number of at most s = scale |q| |k|, so a
probability is within e = (2 d + 16) U (1 + s) relative before its rounding to
the type.  Then
  out:  (2 u + 2 e + 2 n U) sum P |v|  and its own rounding;
  dv:   (2 u + 2 e + 2 N U) sum P |g|, N the queries that see the key;
  dS:   P times [(2 u + 2 e) |dP - delta| + 2 d U sum |g| |v| + sum |g| |out's bound|],
which dq and dk sum with |k| and |q|.  A 16-bit factor below the type's normal
range loses up to half its smallest subnormal.
"""

from __future__ import annotations

import math

import pytest
import torch

from gaussian_splats_hip.sequence import (
    WindowCache,
    window_attention,
    window_attention_backward,
    window_attention_forward,
    window_attention_step,
)
from oracle import sequence as orc
from sequence_helpers import TINY, TYPES, U32, UNIT, assert_within, normal

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")


def _dense(q, k, v, window, sinks, scale, lengths, grad):
    """Values and bounds of (out, dq, dk, dv) by dense matrices in float64."""
    dtype = q.dtype
    b, tq, h, d = q.shape
    tk, hk = k.shape[1], k.shape[2]
    scale = 1 / math.sqrt(d) if scale is None else scale
    u, tiny = UNIT[dtype], TINY[dtype]
    q, k, v, grad = (t.double() for t in (q, k, v, grad))
    values = [torch.zeros_like(t) for t in (q, q, k, v)]
    bounds = [torch.zeros_like(t) for t in (q, q, k, v)]
    for i in range(b):
        seen = orc.window_mask(tq, tk, window, sinks, None if lengths is None else int(lengths[i]))
        for n in range(h):
            m = n * hk // h
            qq, kk, vv, g = q[i, :, n], k[i, :, m], v[i, :, m], grad[i, :, n]
            s = (qq @ kk.T * scale).masked_fill(~seen, -1e300)
            p = torch.softmax(s, -1) * seen
            size = scale * float(qq.norm(dim=-1).max()) * float(kk.norm(dim=-1).max())
            e = (2 * d + 16) * U32 * (1 + size)
            rel = 2 * u + 2 * e + 2 * seen.sum(-1, keepdim=True).clamp_min(16) * U32
            out = p @ vv
            ob = rel * (p @ vv.abs()) + tiny * (seen.double() @ vv.abs()) + u * out.abs() + tiny
            values[0][i, :, n], bounds[0][i, :, n] = out, ob
            diff = g @ vv.T - (g * out).sum(-1, keepdim=True)
            ds = p * diff
            slip = p * ((2 * u + 2 * e) * diff.abs() + 2 * d * U32 * (g.abs() @ vv.abs().T)
                        + (g.abs() * ob).sum(-1, keepdim=True)) + tiny * seen.double()
            count = max(tq, tk) * U32
            values[1][i, :, n] = scale * ds @ kk
            bounds[1][i, :, n] = scale * ((slip + 2 * count * ds.abs()) @ kk.abs())
            values[2][i, :, m] += scale * ds.T @ qq
            bounds[2][i, :, m] += scale * ((slip + 2 * count * ds.abs()).T @ qq.abs())
            values[3][i, :, m] += p.T @ g
            bounds[3][i, :, m] += ((2 * u + 2 * e + 2 * count) * p + tiny * seen.double()).T @ g.abs()
    for x, y in zip(values[1:], bounds[1:]):
        y += u * x.abs() + tiny
    return values, bounds


def _check(q, k, v, window, sinks, scale=None, lengths=None, seed=9):
    grad = normal(q.shape, q.dtype, seed)
    values, bounds = _dense(q, k, v, window, sinks, scale, lengths, grad)
    d = [t.to(DEV).requires_grad_(True) for t in (q, k, v)]
    out = window_attention(*d, window, sinks, scale, None if lengths is None else lengths.to(DEV))
    got = (out, *torch.autograd.grad(out, d, grad.to(DEV)))
    for name, x, y, z in zip(("out", "dq", "dk", "dv"), got, values, bounds):
        assert x.dtype == q.dtype
        assert_within(x, y, z, name)
    return got


def _inputs(b, tq, tk, h, hk, d, dtype, seed=0):
    return (normal((b, tq, h, d), dtype, seed + 1), normal((b, tk, hk, d), dtype, seed + 2),
            normal((b, tk, hk, d), dtype, seed + 3))


SHAPES = [
    # b, tq, tk, h, hk, d, window, sinks
    (1, 1, 1, 1, 1, 8, 1, 0),
    (2, 5, 5, 2, 1, 16, 2, 1),
    (1, 31, 33, 3, 1, 32, 7, 0),
    (1, 64, 64, 2, 2, 64, 64, 0),
    (2, 65, 65, 4, 2, 64, 20, 3),
    (1, 127, 300, 2, 1, 40, 33, 5),
    (1, 200, 200, 4, 1, 128, 1000, 0),
    (1, 257, 257, 2, 2, 72, 64, 65),
    (2, 300, 300, 3, 3, 80, 1, 2),
    (1, 400, 400, 6, 2, 128, 130, 140),
    (1, 900, 900, 2, 1, 64, 40, 4),
    (1, 1, 500, 8, 2, 64, 100, 4),
    (1, 40, 20, 2, 1, 32, 6, 2),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_matches_definition(shape, dtype):
    print(f"[attention] {shape} {dtype}", flush=True)
    b, tq, tk, h, hk, d, window, sinks = shape
    _check(*_inputs(b, tq, tk, h, hk, d, dtype), window, sinks)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("sinks", [0, 3, 70])
def test_lengths_and_empty_rows(dtype, sinks):
    """Sequences that end early, one that is empty; without sinks their late
    queries see nothing: zeros, and no gradient."""
    q, k, v = _inputs(4, 260, 260, 2, 1, 64, dtype)
    lengths = torch.tensor([260, 150, 1, 0], dtype=torch.int32)
    out, dq, dk, dv = _check(q, k, v, 50, sinks, lengths=lengths)
    assert not out[3].any() and not dq[3].any()
    assert not dk[1, 150:].any() and not dv[1, 150:].any()
    if sinks == 0:
        assert not out[1, 199:].any() and out[1, 198].any() and not dq[1, 199:].any()


@pytest.mark.parametrize("dtype", TYPES)
def test_unseen_values_do_not_leak(dtype):
    """Infinities and NaN beyond a sequence's length, after a query and before
    its window change nothing of it, nor of the gradients of what it sees."""
    q, k, v = _inputs(1, 200, 200, 2, 1, 64, dtype)
    window, sinks, lengths = 30, 2, torch.tensor([180], dtype=torch.int32)
    grad = normal(q.shape, dtype, 9)
    clean = window_attention_forward(q.to(DEV), k.to(DEV), v.to(DEV), window, sinks, None, lengths.to(DEV))

    def run(q, k, v, grad):
        q, k, v, grad = (t.to(DEV) for t in (q, k, v, grad))
        out, lse = window_attention_forward(q, k, v, window, sinks, None, lengths.to(DEV))
        return [out.cpu(), *(t.cpu() for t in window_attention_backward(
            q, k, v, out, lse, grad, window, sinks, None, lengths.to(DEV)))]

    base = run(q, k, v, grad)
    assert torch.equal(base[0], clean[0].cpu())
    # Beyond the length.
    k2, v2 = k.clone(), v.clone()
    k2[:, 180:], v2[:, 180:] = float("nan"), float("inf")
    for a, b in zip(base, run(q, k2, v2, grad)):
        assert torch.equal(a, b)
    # Key 100: seen by queries 100 .. 129 only.
    for bad in (float("nan"), float("inf"), -float("inf")):
        k2, v2 = k.clone(), v.clone()
        k2[:, 100], v2[:, 100, :, 5] = bad, bad
        got = run(q, k2, v2, grad)
        others = [i for i in range(200) if not 100 <= i < 130]
        assert torch.equal(got[0][:, others], base[0][:, others])
        assert torch.equal(got[1][:, others], base[1][:, others])
        assert not torch.isfinite(got[0][:, 100:130]).all(-1).any()
        # Keys that none of those queries sees.
        apart = [i for i in range(2, 200) if i <= 70 or i >= 130]
        for n in (2, 3):
            assert torch.equal(got[n][:, apart], base[n][:, apart])
        # Query 100 and its gradient: seen by keys 71 .. 100 and the first two.
        for which in (0, 3):
            args = [t.clone() for t in (q, k, v, grad)]
            args[which][:, 100] = bad
            got = run(*args)
            rows = [i for i in range(200) if i != 100]
            keys = [i for i in range(2, 200) if not 71 <= i <= 100]
            assert torch.equal(got[0][:, rows], base[0][:, rows])
            assert torch.equal(got[1][:, rows], base[1][:, rows])
            for n in (2, 3):
                assert torch.equal(got[n][:, keys], base[n][:, keys])


@pytest.mark.parametrize("dtype", TYPES)
def test_large_scores(dtype):
    """Scores of hundreds: the running maximum keeps every exponential in range."""
    q, k, v = _inputs(1, 150, 150, 2, 1, 64, dtype)
    _check(q, (k * 8).to(dtype), v, 70, 1, scale=1.0)
    _check((q * -6).to(dtype), k, v, 70, 1, scale=0.5)


@pytest.mark.parametrize("size", [1e-4, 1e-2, 1e3])
def test_float16_gradients_of_any_size(size):
    """Gradients far below and above one: relative to their size the result is as
    exact as for gradients near one."""
    q, k, v = _inputs(1, 300, 300, 2, 1, 64, torch.float16)
    grad = normal(q.shape, torch.float32, 9)
    d = [t.to(DEV).requires_grad_(True) for t in (q, k, v)]
    out = window_attention(*d, 200, 2)
    got = torch.autograd.grad(out, d, (grad * size).half().to(DEV))
    values, bounds = _dense(q, k, v, 200, 2, None, None, (grad * size).half())
    # grad_out's own subnormals are in both; outputs may add half of one.
    unit, unit_bounds = _dense(q, k, v, 200, 2, None, None, grad.half())
    for name, x, y, b in zip(("dq", "dk", "dv"), got, values[1:], unit_bounds[1:]):
        assert_within(x, y, b * size + 2 * TINY[torch.float16], name)


def test_strides():
    """[batch, heads, tokens, dim] tensors, one block of a fused projection, an
    offset that no 16-byte access allows."""
    b, t, h, d = 2, 130, 2, 64
    fused = normal((b, t, 3, h, d), torch.bfloat16, 1).to(DEV)
    heads_first = normal((3, b, h, t, d), torch.bfloat16, 2).to(DEV)
    shifted = normal((3, b, t, h, d + 1), torch.bfloat16, 3).to(DEV)
    for q, k, v in (fused.unbind(2), heads_first.transpose(2, 3).unbind(0), shifted[..., 1:].unbind(0)):
        leaves = [x.detach().requires_grad_(True) for x in (q, k, v)]
        out = window_attention(*leaves, 40, 2)
        grad = normal(out.shape[:1] + (h, t, d), torch.bfloat16, 4).to(DEV).transpose(1, 2)
        got = (out, *torch.autograd.grad(out, leaves, grad))
        plain = [x.detach().contiguous().requires_grad_(True) for x in (q, k, v)]
        out = window_attention(*plain, 40, 2)
        for x, y in zip(got, (out, *torch.autograd.grad(out, plain, grad.contiguous()))):
            assert torch.equal(x, y)


def test_shared_keys_and_broadcast():
    """Keys expanded over the batch: autograd sums their gradient."""
    q, k, v = _inputs(3, 90, 90, 2, 1, 32, torch.float32)
    one = k[:1].to(DEV).requires_grad_(True)
    out = window_attention(q.to(DEV), one.expand(3, -1, -1, -1), v.to(DEV), 30, 1)
    grad = normal(out.shape, torch.float32, 9)
    (got,) = torch.autograd.grad(out, one, grad.to(DEV))
    values, bounds = _dense(q, k[:1].expand(3, -1, -1, -1), v, 30, 1, None, None, grad)
    assert_within(got, values[2].sum(0, keepdim=True), bounds[2].sum(0, keepdim=True) * 2, "dk")


def test_gradient_by_differences():
    q, k, v = _inputs(1, 23, 23, 2, 1, 8, torch.float32)
    grad = normal(q.shape, torch.float32, 9)
    d = [t.to(DEV).requires_grad_(True) for t in (q, k, v)]
    got = torch.autograd.grad(window_attention(*d, 6, 2), d, grad.to(DEV))
    h = 1e-5
    for n, t in enumerate((q, k, v)):
        for i in range(0, t.numel(), 37):
            step = torch.zeros(t.numel(), dtype=torch.float64)
            step[i] = h
            f = []
            for e in (1, -1):
                args = [x.double() + (e * step.view(t.shape) if x is t else 0) for x in (q, k, v)]
                f.append(float((orc.window_attention(*args, 6, 2) * grad.double()).sum()))
            assert abs((f[0] - f[1]) / (2 * h) - float(got[n].view(-1)[i])) <= 1e-5


def test_lse():
    q, k, v = _inputs(1, 100, 60, 2, 1, 64, torch.float32)
    _, lse = window_attention_forward(q.to(DEV), k.to(DEV), v.to(DEV), 20, 1)
    s = torch.einsum("bihd,bjd->bhij", q.double(), k[:, :, 0].double()) / 8
    want = s.masked_fill(~orc.window_mask(100, 60, 20, 1), -math.inf).logsumexp(-1)
    got = lse.cpu().double()
    assert torch.equal(torch.isinf(got), torch.isinf(want)) and torch.isinf(want[:, :, :40]).all()
    assert_within(lse[:, :, 40:], want[:, :, 40:], 200 * U32 * (1 + want[:, :, 40:].abs()), "lse")


def test_same_bits_again_and_on_another_stream():
    q, k, v = (t.to(DEV) for t in _inputs(1, 1500, 1500, 4, 2, 64, torch.bfloat16))

    def once():
        d = [t.clone().requires_grad_(True) for t in (q, k, v)]
        out = window_attention(*d, 200, 4)
        return (out, *torch.autograd.grad(out, d, q))

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
    q, k, v = (t.to(DEV).requires_grad_(True) for t in _inputs(2, 3, 0, 2, 1, 16, torch.float32))
    out = window_attention(q, k, v, 4, 1)
    dq, dk, _ = torch.autograd.grad(out, (q, k, v), torch.ones_like(out))
    assert out.shape == q.shape and not out.any() and not dq.any() and dk.shape == k.shape
    q, k, v = (t.to(DEV).requires_grad_(True) for t in _inputs(2, 0, 3, 2, 1, 16, torch.float32))
    out = window_attention(q, k, v, 4, 1)
    _, dk, dv = torch.autograd.grad(out, (q, k, v), out.detach())
    assert out.shape == q.shape and not dk.any() and not dv.any()


def test_offsets_beyond_32_bits():
    """Sequences and cache rows that lie more than 2^31 elements apart."""
    apart = (1 << 31) + 64

    def spread(t):
        flat = torch.empty(apart + t[0].numel(), dtype=t.dtype, device=DEV)
        far = flat.as_strided(t.shape, (apart, *t.stride()[1:]))
        far.copy_(t)
        return far

    near = [t.to(DEV) for t in _inputs(2, 70, 70, 2, 1, 64, torch.bfloat16)]
    far = [spread(t) for t in near]
    out = [window_attention_forward(*t, 30, 2) for t in (near, far)]
    grads = [window_attention_backward(*t, *o, near[0], 30, 2) for t, o in zip((near, far), out)]
    for a, b in zip((*out[0], *grads[0]), (*out[1], *grads[1])):
        assert torch.equal(a, b)
    # A window's tokens far apart: copied together first.
    wide = spread(near[1][:, :2].transpose(0, 1).contiguous()).transpose(0, 1)
    assert torch.equal(window_attention_forward(near[0][:, :2], wide, near[2][:, :2], 30)[0],
                       window_attention_forward(near[0][:, :2], near[1][:, :2], near[2][:, :2], 30)[0])
    del far, wide
    cache = [t.clone() for t in near[1:]]
    far = [spread(t) for t in near[1:]]
    q, kv = near[0][:, 0].contiguous(), near[1][:, 1].contiguous()
    at = torch.tensor([69, 200], dtype=torch.int32, device=DEV)
    a = window_attention_step(q, kv, kv, *cache, at, 66, 4)
    b = window_attention_step(q, kv, kv, *far, at, 66, 4)
    assert torch.equal(a, b) and all(torch.equal(x, y) for x, y in zip(cache, far))


def _step_bound(q, k_cache, v_cache, want, positions, dtype):
    d = q.shape[-1]
    size = float(q.double().norm(dim=-1).max() * k_cache.double().norm(dim=-1).max()) / math.sqrt(d)
    e = (2 * d + 16) * U32 * (1 + size)
    rel = 3 * UNIT[dtype] + 2 * e + 2 * k_cache.shape[1] * U32
    return rel * float(v_cache.double().abs().max()) + TINY[dtype] * (1 + k_cache.shape[1])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(1, 1, 1, 8, 1, 0), (3, 4, 2, 64, 5, 2), (2, 7, 1, 40, 100, 0),
                                   (5, 8, 8, 128, 33, 4), (2, 40, 1, 64, 300, 3),
                                   (4, 6, 2, 80, 2000, 16), (1, 2, 1, 32, 64, 100)])
def test_step_matches_definition(shape, dtype):
    """Streams at their first token, among the first tokens, with the ring
    partly filled, just full and wrapped around; slots not filled yet hold NaN."""
    print(f"[step] {shape} {dtype}", flush=True)
    b, h, hk, d, window, sinks = shape
    n = window + sinks
    places = [0, sinks, n - 1, n, n + window // 2 + 1, max(0, sinks - 1), n // 2]
    for turn in range(2):
        positions = torch.tensor([places[(i + 3 * turn) % len(places)] for i in range(b)], dtype=torch.int32)
        q, k, v = normal((b, h, d), dtype, 1), normal((b, hk, d), dtype, 2), normal((b, hk, d), dtype, 3)
        kc, vc = normal((b, n, hk, d), dtype, 4), normal((b, n, hk, d), dtype, 5)
        want, kw, vw = orc.window_attention_step(q, k, v, kc, vc, positions, window, sinks)
        bound = _step_bound(q, kw, vw, want, positions, dtype)
        for i, p in enumerate(positions.tolist()):
            kc[i, p + 1:], vc[i, p + 1:] = float("nan"), float("inf")
            kw[i, p + 1:], vw[i, p + 1:] = kc[i, p + 1:], vc[i, p + 1:]
        kd, vd = kc.to(DEV), vc.to(DEV)
        out = window_attention_step(q.to(DEV), k.to(DEV), v.to(DEV), kd, vd, positions.to(DEV), window, sinks)
        assert_within(out, want, bound, "out")
        for got, kept in ((kd, kw), (vd, vw)):
            assert torch.equal(got.cpu().nan_to_num(7.0), kept.nan_to_num(7.0))


def test_step_leaves_inactive_streams_alone():
    positions = torch.tensor([-1, 3], dtype=torch.int32, device=DEV)
    q, k = torch.ones(2, 2, 32, device=DEV), torch.ones(2, 1, 32, device=DEV)
    kc, vc = torch.zeros(2, 9, 1, 32, device=DEV), torch.zeros(2, 9, 1, 32, device=DEV)
    out = window_attention_step(q, k, k, kc, vc, positions, 8, 1)
    assert not out[0].any() and out[1].any() and not kc[0].any()
    assert torch.equal(kc[1].any(-1)[:, 0].nonzero().cpu(), torch.tensor([[3]]))


@pytest.mark.parametrize("prefill", [1, 3, 30, 31, 100, 131])
def test_stream_equals_attention(prefill):
    """A prefill kept in a cache and steps after it give the rows of attention
    over the whole sequence."""
    tokens, window, sinks, dtype = prefill + 12, 28, 3, torch.bfloat16
    q, k, v = _inputs(2, tokens, tokens, 4, 2, 64, dtype)
    values, bounds = _dense(q, k, v, window, sinks, None, None, torch.zeros_like(q))
    cache = WindowCache(2, 2, 64, window, sinks, dtype, DEV)
    cache.fill(k[:, :prefill].to(DEV), v[:, :prefill].to(DEV))
    for t in range(prefill, tokens):
        out = cache.step(q[:, t].to(DEV), k[:, t].to(DEV), v[:, t].to(DEV))
        assert_within(out, values[0][:, t], bounds[0][:, t], f"token {t}")


def test_step_in_a_graph():
    """Replays with new inputs and positions in the captured buffers, with eager
    work between them, equal eager steps."""
    b, h, hk, d, window, sinks = 2, 4, 2, 64, 600, 2
    q, k, v = (normal((b, n, d), torch.bfloat16, i).to(DEV) for i, n in ((1, h), (2, hk), (3, hk)))
    cache, twin = (WindowCache(b, hk, d, window, sinks, torch.bfloat16, DEV) for _ in range(2))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        cache.step(q, k, v)
    torch.cuda.current_stream().wait_stream(side)
    cache.positions.zero_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = cache.step(q, k, v)
    cache.positions.zero_()
    for t in range(6):
        for i, x in enumerate((q, k, v)):
            x.copy_(normal(x.shape, torch.bfloat16, 10 * t + i))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, twin.step(q, k, v)), t
        assert torch.equal(cache.k, twin.k) and torch.equal(cache.positions, twin.positions)


@pytest.mark.parametrize("dtype", TYPES)
def test_no_queries(dtype):
    """Keys without a query get zeros, whatever the workspace held before."""
    q, k, v = (t.to(DEV) for t in _inputs(2, 0, 70, 2, 1, 64, dtype))
    out, lse = window_attention_forward(q, k, v, 4, 1)
    torch.cuda.empty_cache()
    old = [torch.full((1 << 17,), -1.0, device=DEV) for _ in range(4)]
    del old  # small allocations are cut from these
    _, dk, dv = window_attention_backward(q, k, v, out, lse, out, 4, 1)
    for t in (dk, dv):
        assert torch.isfinite(t).all() and not t.any()


@pytest.mark.parametrize("values,size", [(100.0, 1.0), (1000.0, 1.0), (3000.0, 0.1), (300.0, 1e-3), (1e-3, 1e-3)])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("window", [1, 200])
def test_float16_values_of_any_size(window, dim, values, size):
    """Large and small values beside gradients of one sign.  dS carries a power of
    two that brings B = 2 max|g| max|v| over the rows to 2^13 .. 2^15, so that it
    loses up to max(1, B / 2^13) half subnormals."""
    q, k, v = _inputs(1, 300, 300, 2, 1, dim, torch.float16)
    v = (v.float() * values).half()
    grad = (normal(q.shape, torch.float32, 9).abs() * size).half()
    d = [t.to(DEV).requires_grad_(True) for t in (q, k, v)]
    got = torch.autograd.grad(window_attention(*d, window, 2), d, grad.to(DEV))
    want, bounds = _dense(q, k, v, window, 2, None, None, grad)
    top = 2 * float(grad.double().norm(dim=-1).max() * v.double().norm(dim=-1).max())
    lost = TINY[torch.float16] * max(1.0, top / 2**13) / math.sqrt(dim)
    for name, x, y, b, t in zip(("dq", "dk", "dv"), got, want[1:], bounds[1:], (k, q, None)):
        more = 0 if t is None else 300 * lost * float(t.double().abs().max()) * (1 if name == "dq" else 2)
        assert_within(x, y, b + more, name)


def test_float16_opposite_values():
    """Two equal keys with values of +256 and -256 and gradients of one: dS is
    16384, dk 16384 q / sqrt(128) and dq zero."""
    q = normal((1, 2, 1, 128), torch.float16, 1)
    k = normal((1, 1, 1, 128), torch.float16, 2).expand(1, 2, 1, 128).contiguous()
    v = torch.full((1, 2, 1, 128), 256.0).half()
    v[:, 1] = -256.0
    grad = torch.zeros(q.shape).half()
    grad[:, 1] = 1.0
    d = [t.to(DEV).requires_grad_(True) for t in (q, k, v)]
    dq, dk, dv = torch.autograd.grad(window_attention(*d, 2), d, grad.to(DEV))
    want = 16384 / math.sqrt(128) * q[0, 1, 0].double()
    u = UNIT[torch.float16]
    assert_within(dk[0, 0, 0], want, 4 * u * want.abs(), "dk")
    assert_within(dk[0, 1, 0], -want, 4 * u * want.abs(), "dk")
    assert_within(dv[0, :, 0], torch.full((2, 128), 0.5), 2 * u, "dv")
    # Two terms that cancel, each within the bound on dS.
    assert_within(dq[0, 1, 0], torch.zeros(128), 8 * u * 16384 / math.sqrt(128) * k[0, 0, 0].double().abs(), "dq")


def test_float16_sequences_apart():
    """One sequence's large values and gradients take no bits of another's small
    ones."""
    q, k, v = _inputs(2, 300, 300, 2, 1, 64, torch.float16)
    grad = normal(q.shape, torch.float16, 9)

    def run(q, k, v, grad):
        q, k, v, grad = (t.to(DEV) for t in (q, k, v, grad))
        return window_attention_backward(q, k, v, *window_attention_forward(q, k, v, 200, 2), grad, 200, 2)

    alone = run(q[:1], k[:1], v[:1], grad[:1])
    v[1], grad[1] = v[1] * 4000, grad[1] * 4000
    for a, b in zip(alone, run(q, k, v, grad)):
        assert torch.equal(a[0], b[0])


def test_float16_long_uniform_window():
    """Equal scores over a window of 1.6 million keys: probabilities of ten
    subnormals of float16.  dv_j = sum_i g_i / n_i, within (2 u + 2 e + 2 N U) of
    sum P |g|, N the 64 queries, and its own rounding."""
    keys, queries = 1597830, 64
    q = torch.zeros(1, queries, 1, 8).half()
    k, v = normal((1, keys, 1, 8), torch.float16, 2), normal((1, keys, 1, 8), torch.float16, 3)
    grad = normal(q.shape, torch.float16, 9, 500.0)
    d = [t.to(DEV).requires_grad_(True) for t in (q, k, v)]
    (dv,) = torch.autograd.grad(window_attention(*d, keys), d[2:], grad.to(DEV))
    p = 1 / (keys - queries + 1 + torch.arange(queries, dtype=torch.float64))[:, None]
    g = grad[0, :, 0].double()
    want, size = (p * g).sum(0), (p * g.abs()).sum(0)
    u = UNIT[torch.float16]
    # The sums over the keys that lse holds are of equal terms; n U with n the keys
    # bounds their chains, which are cut over lanes, waves and tiles of 32.
    bound = (2 * u + 2 * (32 + keys / 256) * U32 + 2 * queries * U32) * size + u * want.abs() + TINY[torch.float16]
    seen = dv[0, :keys - queries + 1, 0].cpu().double()
    assert_within(seen, want.expand_as(seen), bound.expand_as(seen), "dv")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("batch", [1, 40])
def test_nan_scores_give_nan(dtype, batch):
    """A query of NaN, and one that sees NaN keys alone, give NaN and a NaN lse,
    few workgroups (one sequence) or many; every other query stays as it is."""
    q, k, v = _inputs(batch, 300, 300, 4, 2, 64, dtype)
    clean = window_attention_forward(q.to(DEV), k.to(DEV), v.to(DEV), 8)
    q[0, 100], k[0, 200:208] = float("nan"), float("nan")
    out, lse = window_attention_forward(q.to(DEV), k.to(DEV), v.to(DEV), 8)
    assert torch.isnan(out[0, 100]).all() and torch.isnan(lse[0, :, 100]).all()
    assert torch.isnan(out[0, 200:215]).all() and torch.isnan(lse[0, :, 200:215]).all()
    rows = [i for i in range(300) if i != 100 and not 200 <= i < 215]
    assert torch.equal(out[0, rows], clean[0][0, rows]) and torch.equal(out[1:], clean[0][1:])
    assert torch.equal(lse[0][:, rows], clean[1][0][:, rows]) and torch.equal(lse[1:], clean[1][1:])


def test_one_token_of_a_wide_row():
    """Dimensions of one element, whose stride no address depends on: one token of
    a fused projection of odd width, a cache of one stream."""
    fused = normal((1, 1, 3 * 64 + 1), torch.bfloat16, 1).to(DEV)
    q, k, v = fused[:, :, None, :192].split(64, -1)
    assert q.stride(1) % 8 and q.is_contiguous()
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    out = window_attention(*leaves, 4, 1)
    assert torch.equal(out, v)
    _, _, dv = torch.autograd.grad(out, leaves, q)
    assert torch.equal(dv, q)
    far = [t.as_strided(t.shape, (t.stride(0), 1 << 25, 64, 1)) for t in leaves]
    assert torch.equal(window_attention(*far, 4, 1), v)
    caches = [torch.zeros(9 * 64 + 1, dtype=torch.bfloat16, device=DEV).as_strided((1, 9, 1, 64), (577, 64, 64, 1))
              for _ in range(2)]
    at = torch.zeros(1, dtype=torch.int32, device=DEV)
    assert torch.equal(window_attention_step(q[0], k[0], v[0], *caches, at, 8, 1), v[0])
    assert torch.equal(caches[0][:, 0], k[0]) and torch.equal(caches[1][:, 0], v[0])


def test_cache_leaves_inactive_streams_alone():
    """A stream at a negative position stays there, step after step."""
    cache = WindowCache(3, 1, 32, 8, 1, torch.float32, DEV)
    cache.positions.copy_(torch.tensor([-1, 3, -5]))
    q, k = torch.ones(3, 2, 32, device=DEV), torch.ones(3, 1, 32, device=DEV)
    for t in range(2):
        out = cache.step(q, k, k)
        assert not out[0].any() and out[1].any() and not out[2].any()
        assert cache.positions.tolist() == [-1, 4 + t, -5]
    assert not cache.k[0].any() and not cache.k[2].any()


@pytest.mark.parametrize("tokens", [5, 31, 100, 131])
def test_stream_continues_sequences_of_different_lengths(tokens):
    """A prefill whose sequences end early, kept with their lengths, and steps
    after it give the rows of attention over each whole sequence."""
    window, sinks, dtype, steps = 28, 3, torch.bfloat16, 9
    lengths = torch.tensor([tokens, tokens // 2, 2, 0], dtype=torch.int32)
    q, k, v = _inputs(4, tokens + steps, tokens + steps, 4, 2, 64, dtype)
    cache = WindowCache(4, 2, 64, window, sinks, dtype, DEV)
    pk, pv = k[:, :tokens].clone(), v[:, :tokens].clone()
    for i, n in enumerate(lengths.tolist()):
        pk[i, n:], pv[i, n:] = float("nan"), float("nan")  # padding
    cache.fill(pk.to(DEV), pv.to(DEV), lengths.to(DEV))
    assert torch.equal(cache.positions.cpu(), lengths)
    for t in range(steps):
        at = lengths.long() + t
        each = torch.arange(4)
        out = cache.step(*(x[each, at].to(DEV) for x in (q, k, v)))
        for i, p in enumerate(at.tolist()):
            values, bounds = _dense(q[i:i + 1, :p + 1], k[i:i + 1, :p + 1], v[i:i + 1, :p + 1], window, sinks,
                                    None, None, torch.zeros_like(q[i:i + 1, :p + 1]))
            assert_within(out[i], values[0][0, p], bounds[0][0, p], f"sequence {i}, token {p}")


def test_fill_refuses():
    cache = WindowCache(2, 1, 32, 8, 1, torch.float32, DEV)
    k = torch.ones(2, 4, 1, 32, device=DEV)
    with pytest.raises(TypeError, match="lengths is"):
        cache.fill(k, k, torch.zeros(2, dtype=torch.int64, device=DEV))
    with pytest.raises(ValueError, match="batch of 2"):
        cache.fill(k, k, torch.zeros(3, dtype=torch.int32, device=DEV))
    with pytest.raises(ValueError, match="do not fit"):
        cache.fill(k[:, :, :, :16], k[:, :, :, :16])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_weights_add_up_to_one(dtype):
    """Values that are the same for every key come back as they are, although
    seven of eight probabilities round down by four tenths of a spacing: the sum
    takes the rounded ones."""
    b, h, d, n = 4, 16, 64, 600
    spacing = UNIT[dtype]  # of the type from 0.5 to 1
    scale = -math.log(0.5 + 0.4 * spacing)
    q, k = torch.zeros(b, n, h, d).to(dtype), torch.zeros(b, n, h, d).to(dtype)
    q[..., 0], k[..., 0] = 1, -1
    k[:, ::8] = 0
    value = 2 - 2 * spacing  # the largest below 2
    v = torch.full((b, n, h, d), value).to(dtype)
    assert float(v[0, 0, 0, 0]) == value
    q, k, v = q.to(DEV), k.to(DEV), v.to(DEV)
    for batch in (1, b):  # few workgroups and many
        out, _ = window_attention_forward(q[:batch], k[:batch], v[:batch], n, 0, scale)
        assert bool((out == value).all())
    at = torch.full((b,), n - 1, dtype=torch.int32, device=DEV)
    out = window_attention_step(q[:, -1], k[:, -1], v[:, -1], k.clone(), v.clone(), at, n, 0, scale)
    assert bool((out == value).all())


def test_float16_unseen_values_take_no_bits():
    """Large values that no query sees (before every window, behind the length),
    and gradients of queries that see nothing, leave the gradients' bits."""
    q, k, v = _inputs(2, 300, 600, 4, 2, 64, torch.float16)
    grad = normal(q.shape, torch.float16, 9)
    lengths = torch.tensor([600, 320], dtype=torch.int32)

    def run(v, grad):
        args = [t.to(DEV) for t in (q, k, v)]
        out, lse = window_attention_forward(*args, 50, 3, None, lengths.to(DEV))
        return window_attention_backward(*args, out, lse, grad.to(DEV), 50, 3, None, lengths.to(DEV))

    def bare(v, grad):
        args = [t.to(DEV) for t in (q[1:], k[1:], v[1:])]
        n = lengths[1:].to(DEV)
        out, lse = window_attention_forward(*args, 50, 0, None, n)
        return window_attention_backward(*args, out, lse, grad[1:].to(DEV), 50, 0, None, n)

    base, alone = run(v, grad), bare(v, grad)
    loud, louder = v.clone(), grad.clone()
    loud[:, 3:251] = 60000
    loud[1, 320:] = -60000
    louder[1, 69:] = 60000  # positions from 369 on, which see no key without first ones
    for x, y in zip(base, run(loud, grad)):
        assert torch.equal(x, y)
    for x, y in zip(alone, bare(loud, louder)):
        assert torch.equal(x, y)
