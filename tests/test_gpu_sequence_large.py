"""The sequence operators' kernels of large calls, against the definitions in
float64: what the tests of small shapes do not launch.  Attention takes 128
queries a workgroup (whose four waves share tiles of keys) from 256 workgroups
on, 160 for heads above 64; a scan's 256 workgroups take several chunks each
where there are more; the norm's backward walks rows from 2049 or 513 on.

The references run on the GPU in float64.  Attention's bounds are those of small
calls: with u the type's unit, U that of float32, n the keys a query sees, N the
queries that see a key, d the head dimension and s = scale |q| |k| the largest
score, a probability is within e = (2 d + 16) U (1 + s) relative before its
rounding to the type, and
  out:  (2 u + 2 e + 2 n U) sum P |v|  and its own rounding;
  dv:   (2 u + 2 e + 2 N U) sum P |g|;
  dS:   P times [(2 u + 2 e) |dP - delta| + 2 d U sum |g| |v| + sum |g| |out's bound|],
which dq and dk sum with |k| and |q|, N or n terms with 2 U each.  A 16-bit factor
below the type's normal range loses up to half its smallest subnormal.
"""

from __future__ import annotations

import math

import pytest
import torch

from gaussian_splats_hip.sequence import (
    add_rms_norm,
    add_rms_norm_backward,
    add_rms_norm_quant,
    gated_scan,
    gated_scan_backward,
    gated_scan_forward,
    gated_scan_step,
    window_attention,
    window_attention_backward,
    window_attention_forward,
)
from oracle import sequence as orc
from sequence_helpers import TINY, TYPES, U32, UNIT, assert_within, normal

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")


def _workgroups(b, tq, h, d):
    """Workgroups of 128 queries, and how many the kernels of large calls start at."""
    return -(-tq // 128) * h * b, 256 if d <= 64 else 160


def _heads(t, n):
    """[B, T, H, D] -> float64 [B * n, T, D], shared heads repeated."""
    b, tokens, h, d = t.shape
    t = t.double().repeat_interleave(n // h, 2)
    return t.transpose(1, 2).reshape(b * n, tokens, d).contiguous()


def _reference(q, k, v, window, sinks, lengths, grad):
    """Values and bounds of (out, dq, dk, dv), all heads at once."""
    dtype, (b, tq, h, d) = q.dtype, q.shape
    tk, hk = k.shape[1], k.shape[2]
    u, tiny, scale = UNIT[dtype], TINY[dtype], 1 / math.sqrt(d)
    qq, kk, vv, g = (_heads(t, h) for t in (q, k, v, grad))
    seen = torch.stack([orc.window_mask(tq, tk, window, sinks, None if lengths is None else int(n))
                        for n in (lengths if lengths is not None else [0] * b)]).to(DEV)
    seen = seen[:, None].expand(b, h, tq, tk).reshape(b * h, tq, tk)
    turned = lambda t: t.transpose(1, 2).contiguous()  # noqa: E731
    s = (torch.bmm(qq, turned(kk)) * scale).masked_fill(~seen, -1e300)
    p = torch.softmax(s, -1) * seen
    size = scale * float(qq.norm(dim=-1).max()) * float(kk.norm(dim=-1).max())
    e = (2 * d + 16) * U32 * (1 + size)
    rel = 2 * u + 2 * e + 2 * seen.sum(-1, keepdim=True).clamp_min(16) * U32
    out = torch.bmm(p, vv)
    ob = rel * torch.bmm(p, vv.abs()) + tiny * torch.bmm(seen.double(), vv.abs()) + u * out.abs() + tiny
    diff = torch.bmm(g, turned(vv)) - (g * out).sum(-1, keepdim=True)
    ds = p * diff
    slip = p * ((2 * u + 2 * e) * diff.abs() + 2 * d * U32 * torch.bmm(g.abs(), turned(vv.abs()))
                + (g.abs() * ob).sum(-1, keepdim=True)) + tiny * seen.double()
    slip = slip + 2 * max(tq, tk) * U32 * ds.abs()
    dq, dqb = scale * torch.bmm(ds, kk), scale * torch.bmm(slip, kk.abs())
    dk, dkb = scale * torch.bmm(turned(ds), qq), scale * torch.bmm(turned(slip), qq.abs())
    dv = torch.bmm(turned(p), g)
    dvb = torch.bmm(turned((2 * u + 2 * e + 2 * max(tq, tk) * U32) * p + tiny * seen.double()), g.abs())

    def back(t, n):  # [B * H, T, D] -> [B, T, n, D], the heads of a key head summed
        return t.view(b, n, h // n, -1, d).sum(2).transpose(1, 2)

    values = [back(out, h), back(dq, h), back(dk, hk), back(dv, hk)]
    bounds = [back(ob, h), *(back(t, n) + u * back(x, n).abs() + tiny
                             for t, x, n in ((dqb, dq, h), (dkb, dk, hk), (dvb, dv, hk)))]
    return values, bounds


def _inputs(b, tq, tk, h, hk, d, dtype):
    return [normal(s, dtype, i).to(DEV) for i, s in enumerate(
        ((b, tq, h, d), (b, tk, hk, d), (b, tk, hk, d), (b, tq, h, d)), 1)]


def _check(q, k, v, grad, window, sinks, lengths=None):
    values, bounds = _reference(q, k, v, window, sinks, lengths, grad)
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    out = window_attention(*leaves, window, sinks, None, None if lengths is None else lengths.to(DEV))
    got = (out, *torch.autograd.grad(out, leaves, grad))
    for name, x, y, z in zip(("out", "dq", "dk", "dv"), got, values, bounds):
        assert_within(x, y, z, name)
    return got


SHAPES = [
    # b, tq, tk, h, hk, d, window, sinks
    (8, 300, 300, 16, 4, 64, 40, 3),      # masks in every tile
    (8, 257, 257, 16, 16, 40, 257, 0),    # plain causal, the last workgroup nearly empty
    (2, 700, 700, 24, 8, 64, 400, 70),    # runs of full tiles between masked ones
    (6, 300, 420, 16, 2, 128, 130, 66),   # queries behind earlier keys
    (4, 420, 300, 12, 4, 72, 100, 5),     # queries before the first key
    (3, 1300, 1300, 12, 12, 64, 700, 4),  # key walks that are not cut
    (2, 650, 650, 16, 4, 128, 500, 0),
    (1, 3000, 3000, 12, 4, 80, 1500, 300),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_attention_matches_definition(shape, dtype):
    print(f"[large attention] {shape} {dtype}", flush=True)
    b, tq, tk, h, hk, d, window, sinks = shape
    count, start = _workgroups(b, tq, h, d)
    assert count >= start
    _check(*_inputs(b, tq, tk, h, hk, d, dtype), window, sinks)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [64, 96])
@pytest.mark.parametrize("sinks", [0, 67])
def test_attention_lengths(sinks, dim, dtype):
    """Sequences that end early, inside a tile and before the first one."""
    b, t, h, hk = 8, 330, 16, 4
    count, start = _workgroups(b, t, h, dim)
    assert count >= start
    lengths = torch.tensor([330, 329, 200, 129, 128, 64, 1, 0], dtype=torch.int32)
    out, dq, dk, dv = _check(*_inputs(b, t, t, h, hk, dim, dtype), 90, sinks, lengths)
    assert not out[7].any() and not dq[7].any()
    for i, n in enumerate(lengths.tolist()):
        assert not dk[i, n:].any() and not dv[i, n:].any()
        if sinks == 0:
            assert not out[i, n + 89:].any() and not dq[i, n + 89:].any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [64, 128])
def test_attention_unseen_values_do_not_leak(dim, dtype):
    """Infinities and NaN where a query does not see: the other rows keep their
    bits, forward and backward."""
    b, t, h, hk, window, sinks = 6, 600, 16, 4, 150, 3
    count, start = _workgroups(b, t, h, dim)
    assert count >= start
    q, k, v, grad = _inputs(b, t, t, h, hk, dim, dtype)
    lengths = torch.full((b,), 580, dtype=torch.int32, device=DEV)

    def run(q, k, v, grad):
        out, lse = window_attention_forward(q, k, v, window, sinks, None, lengths)
        return (out, *window_attention_backward(q, k, v, out, lse, grad, window, sinks, None, lengths))

    base = run(q, k, v, grad)
    k2, v2 = k.clone(), v.clone()
    k2[:, 580:], v2[:, 580:] = float("nan"), float("inf")
    for x, y in zip(base, run(q, k2, v2, grad)):
        assert torch.equal(x, y)
    for bad in (float("nan"), float("inf"), -float("inf")):
        # Key 300: seen by queries 300 .. 449 only.
        k2, v2 = k.clone(), v.clone()
        k2[:, 300], v2[:, 300, :, 5] = bad, bad
        got = run(q, k2, v2, grad)
        others = [i for i in range(t) if not 300 <= i < 450]
        assert torch.equal(got[0][:, others], base[0][:, others])
        assert torch.equal(got[1][:, others], base[1][:, others])
        assert not torch.isfinite(got[0][:, 300:450]).all(-1).any()
        apart = [i for i in range(sinks, t) if i <= 150 or i >= 450]
        for n in (2, 3):
            assert torch.equal(got[n][:, apart], base[n][:, apart])
        # Query 300 and its gradient: seen by keys 151 .. 300 and the first ones.
        for which in (0, 3):
            args = [x.clone() for x in (q, k, v, grad)]
            args[which][:, 300] = bad
            got = run(*args)
            rows = [i for i in range(t) if i != 300]
            keys = [i for i in range(sinks, t) if not 151 <= i <= 300]
            assert torch.equal(got[0][:, rows], base[0][:, rows])
            assert torch.equal(got[1][:, rows], base[1][:, rows])
            for n in (2, 3):
                assert torch.equal(got[n][:, keys], base[n][:, keys])


def test_attention_strides_and_streams():
    """Transposed and fused tensors give the bits of contiguous ones, again and on
    another stream."""
    b, t, h, d = 4, 400, 24, 64
    count, start = _workgroups(b, t, h, d)
    assert count >= start
    heads_first = normal((4, b, h, t, d), torch.bfloat16, 2).to(DEV)
    wide = normal((4, b, t, h, d + 8), torch.bfloat16, 3).to(DEV)

    def run(q, k, v, grad):
        out, lse = window_attention_forward(q, k, v, 130, 2)
        return (out, lse, *window_attention_backward(q, k, v, out, lse, grad, 130, 2))

    for tensors in (heads_first.transpose(2, 3).unbind(0), wide[..., 8:].unbind(0)):
        plain = run(*(x.contiguous() for x in tensors))
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            again = run(*tensors)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        for x, y, z in zip(run(*tensors), plain, again):
            assert torch.equal(x, y) and torch.equal(x, z)


@pytest.mark.parametrize("dtype", TYPES)
def test_scan_of_more_chunks_than_workgroups(dtype):
    """528 chunks and more of 240 tokens, 1056 of 120 backward: every workgroup
    takes several.  Bounds: a step errs by at most 10 U, m = 1 / (1 - max a) steps
    are remembered, cutting the sequence doubles it at most; 20 U m times the
    largest |x|, and for gradients the largest carried one."""
    shape = (16, 2500, 300)
    b, t, c = shape
    lanes = 64 if dtype == torch.float32 else 128
    assert b * -(-t // 240) * -(-c // lanes) > 512
    x, dy = normal(shape, dtype, 1).to(DEV), normal(shape, dtype, 3).to(DEV)
    # Memories of up to a hundred tokens.
    gate = normal(shape, dtype, 2, 2.0, 2.0).clamp(max=4.6).to(DEV)
    state, dlast = (normal((b, c), torch.float32, i).to(DEV) for i in (4, 5))
    leaves = [z.detach().requires_grad_(True) for z in (x, gate, state)]
    y, last = gated_scan(*leaves)
    got = torch.autograd.grad((y, last), leaves, (dy, dlast))
    want, want_last = orc.gated_scan(x, gate, state)
    u, tiny = UNIT[dtype], TINY[dtype]
    keep = torch.sigmoid(-gate.double())
    m, top = float((1 / keep).max()), max(float(x.abs().max()), float(state.abs().max()))
    own = 20 * U32 * m * top
    assert_within(y, want, want.abs() * u + own + tiny, "y")
    assert_within(last, want_last, want_last.abs() * U32 + own, "last")
    gx, gg, gs = orc.gated_scan_grads(x, gate, state, dy, dlast)
    mx, _, _ = orc.gated_scan_grads(x, gate, state, dy.abs(), dlast.abs())
    g = float((mx / keep).max())
    slip = 20 * U32 * m * g
    assert_within(got[0], gx, gx.abs() * u + keep * slip + 20 * U32 * mx + tiny, "grad x")
    bound = keep * (1 - keep) * (2 * top * slip + g * 2 * own + 40 * U32 * g * top)
    assert_within(got[1], gg, gg.abs() * u + bound + tiny, "grad gate")
    assert_within(got[2], gs, gs.abs() * U32 + slip, "grad state")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens", [119, 120, 121, 239, 240, 241, 359, 360, 361, 479, 480, 481])
def test_scan_at_the_chunks_edges(tokens, dtype):
    """Forward chunks have 240 tokens and keep a state every 120; backward chunks
    have 120."""
    b, c = 2, 70
    x, dy = normal((b, tokens, c), dtype, 1).to(DEV), normal((b, tokens, c), dtype, 3).to(DEV)
    gate = normal((b, tokens, c), dtype, 2, 2.0, 2.0).clamp(max=4.6).to(DEV)
    state = normal((b, c), torch.float32, 4).to(DEV)
    leaves = [z.detach().requires_grad_(True) for z in (x, gate, state)]
    y, last = gated_scan(*leaves)
    got = torch.autograd.grad(y, leaves, dy)
    want, want_last = orc.gated_scan(x, gate, state)
    u, tiny = UNIT[dtype], TINY[dtype]
    keep = torch.sigmoid(-gate.double())
    m, top = float((1 / keep).max()), max(float(x.abs().max()), float(state.abs().max()))
    own = 20 * U32 * m * top
    assert_within(y, want, want.abs() * u + own + tiny, "y")
    assert_within(last, want_last, want_last.abs() * U32 + own, "last")
    none = torch.zeros_like(state)
    gx, gg, gs = orc.gated_scan_grads(x, gate, state, dy, none)
    mx, _, _ = orc.gated_scan_grads(x, gate, state, dy.abs(), none)
    g = float((mx / keep).max())
    slip = 20 * U32 * m * g
    assert_within(got[0], gx, gx.abs() * u + keep * slip + 20 * U32 * mx + tiny, "grad x")
    bound = keep * (1 - keep) * (2 * top * slip + g * 2 * own + 40 * U32 * g * top)
    assert_within(got[1], gg, gg.abs() * u + bound + tiny, "grad gate")
    assert_within(got[2], gs, gs.abs() * U32 + slip, "grad state")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,width", [(5000, 40), (5001, 768), (4100, 1023), (1500, 2056), (1100, 5000),
                                        (1030, 1032), (700, 8200)])
def test_norm_backward_over_several_rows_a_workgroup(rows, width, dtype):
    """512 workgroups of four rows (up to 1024 elements) or one walk the rest.
    Bounds, with n = 2 (45 + width / 256) U for the chains of a row's sums, v the
    unit of the sum's rounding, unit = s r, t = grad_y w:
    r (|unit| mean|t unit| (4 v + n) + 4 U |t|) + U (|grad_sum| + |grad_s|) before a
    gradient's rounding, sum |grad_y unit| (2 v + (rows + 60 + width / 256) U) for
    the weight's."""
    x, res = normal((rows, width), dtype, 1).to(DEV), normal((rows, width), dtype, 2, 2.0).to(DEV)
    w = normal((width,), dtype, 3, 0.2, 1.0).to(DEV)
    dy, dsum = normal((rows, width), dtype, 4).to(DEV), normal((rows, width), dtype, 5).to(DEV)
    leaves = [z.detach().requires_grad_(True) for z in (x, res, w)]
    y, s = add_rms_norm(*leaves, 1e-6)
    got = torch.autograd.grad((y, s), leaves, (dy, dsum))
    want_y, want_s = orc.add_rms_norm(x, res, w, 1e-6)
    u, tiny, chain = UNIT[dtype], TINY[dtype], 45 + width // 256
    assert_within(y, want_y, want_y.abs() * (u + chain * U32) + tiny, "y")
    ds, dw = orc.add_rms_norm_grads(x, res, w, 1e-6, dy, dsum)
    r = 1 / torch.sqrt((want_s * want_s).mean(-1, keepdim=True) + 1e-6)
    unit, t = (want_s * r).abs(), (dy.double() * w.double()).abs()
    own = r * (unit * (t * unit).mean(-1, keepdim=True) * (4 * u + 2 * chain * U32) + 4 * U32 * t)
    own = own + U32 * (dsum.double().abs() + ds.abs())
    for name, z in zip(("grad x", "grad residual"), got):
        assert_within(z, ds, own + ds.abs() * u + tiny, name)
    bound = (dy.double().abs() * unit).sum(0) * (2 * u + (rows + chain + 15) * U32) + dw.abs() * u
    assert_within(got[2], dw, bound + tiny, "grad weight")


def test_norm_of_more_threads_than_one_dimension_holds():
    """2^26 rows and more, a wave each: 2^32 threads."""
    rows = (1 << 26) + 5
    x = normal((4096, 8), torch.bfloat16, 1).to(DEV).repeat(rows // 4096 + 1, 1)[:rows]
    w = normal((8,), torch.bfloat16, 2, 0.2, 1.0).to(DEV)
    y, _ = add_rms_norm(x, None, w)
    codes, scales, _ = add_rms_norm_quant(x, None, w)
    want = add_rms_norm(x[:4096], None, w)[0]
    few, few_scales, _ = add_rms_norm_quant(x[:4096], None, w)
    assert torch.equal(y[:rows - 5].view(-1, 4096, 8), want.expand(rows // 4096, -1, -1))
    assert torch.equal(codes[:rows - 5].view(-1, 4096, 8), few.expand(rows // 4096, -1, -1))
    assert torch.equal(y[rows - 5:], want[:5]) and torch.equal(codes[rows - 5:], few[:5])
    assert torch.equal(scales[:rows - 5].view(-1, 4096), few_scales.expand(rows // 4096, -1))


def test_weight_gradient_of_a_very_long_row():
    """2^28 elements: 2^32 threads add the weight's gradient up."""
    width = (1 << 28) + 70
    x = normal((1, 4096), torch.bfloat16, 1).to(DEV).repeat(1, width // 4096 + 1)[:, :width].contiguous()
    w, inverse = torch.ones(width, dtype=torch.bfloat16, device=DEV), torch.ones(1, device=DEV)
    _, _, dw = add_rms_norm_backward(x, w, inverse, x, None, torch.bfloat16, False, False)
    assert torch.equal(dw, (x[0].float() * x[0].float()).to(torch.bfloat16))


def test_scan_of_more_threads_than_one_dimension_holds():
    """One token of 65535 sequences of 16400 channels: 8.4 million workgroups.  One
    step of a running stream of 2^32 channels in all."""
    b, c = 65535, 16400
    x = normal((1, 1, c), torch.bfloat16, 1).to(DEV).expand(b, 1, c)
    gate = normal((1, 1, c), torch.bfloat16, 2).to(DEV).expand(b, 1, c)
    y, last, starts = gated_scan_forward(x, gate)
    few = gated_scan_forward(x[:2], gate[:2])
    assert torch.equal(y, few[0][:1].expand(b, -1, -1)) and torch.equal(last, few[1][:1].expand(b, -1))
    del y, last
    dx, dg, _ = gated_scan_backward(x, gate, starts, x, None, need_state=False)
    one = gated_scan_backward(x[:2], gate[:2], few[2], x[:2], None)
    assert torch.equal(dx, one[0][:1].expand(b, -1, -1)) and torch.equal(dg, one[1][:1].expand(b, -1, -1))
    del dx, dg, starts
    b, c = 1 << 15, (1 << 17) + 8
    x = normal((1, c), torch.float32, 1).to(DEV).repeat(b, 1)
    state = x.clone()
    y, _ = gated_scan_step(x, x, state, state_out=state)
    few, _ = gated_scan_step(x[:1], x[:1], x[:1])
    assert torch.equal(y, few.expand(b, -1)) and torch.equal(state, few.expand(b, -1))


def test_attention_backward_of_many_rows():
    """2^28 rows: delta takes 2^32 threads."""
    b, t, h = (1 << 10) + 1, 1 << 14, 16
    q, k, v, grad = (x.expand(b, -1, -1, -1) for x in _inputs(1, t, t, h, 1, 8, torch.float16))
    few = [x[:2] for x in (q, k, v, grad)]
    out, lse = window_attention_forward(q, k, v, 3, 1)
    got = window_attention_backward(q, k, v, out, lse, grad, 3, 1)
    out2, lse2 = window_attention_forward(*few[:3], 3, 1)
    want = window_attention_backward(*few[:3], out2, lse2, few[3], 3, 1)
    assert torch.equal(out, out2[:1].expand(b, -1, -1, -1)) and torch.equal(lse, lse2[:1].expand(b, -1, -1))
    assert torch.equal(got[0], want[0][:1].expand(b, -1, -1, -1))
    # Keys' walks are cut otherwise in the small call: sums in another order.
    for x, y in zip(got[1:], want[1:]):
        assert torch.equal(x, x[:1].expand(b, -1, -1, -1))
        u = UNIT[torch.float16]
        assert bool(((x[0] - y[0]).float().abs() <= 2 * u * y[0].float().abs() + 64 * u * y.float().abs().mean()).all())
