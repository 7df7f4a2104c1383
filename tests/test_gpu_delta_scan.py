"""delta_scan on the GPU against its definition, token after token, in float64.

Bounds.  Keys are no longer than one, so a chunk's map of the state does not
lengthen anything, and what is wrong in a state stays at most as large; what each
chunk adds is bounded from its own numbers.  With n = 128 + 8, U float32's unit and u
bfloat16's, a product of factors that states depend on is within
  E = n U + 3 u^2   (16-bit types: two bfloat16 parts a factor, u^2 each, their
                     second parts' product left out),  n U for float32,
and one of an output within O = n U + 2 u in bfloat16 (a part a factor), E in the other
types and for dR.  A decay is within (3 + |log2 D|) U.  T = (I + A)^-1 is within |T| dA |T| and
substitution's 70 U |T| (I + |A|) |T|.  From these _bounds() adds up the formulas of the
chunk, with scalar products of errors by Cauchy-Schwarz; every result is then rounded
to its type.
"""

from __future__ import annotations

import math

import pytest
import torch

from gaussian_splats_hip.sequence import (
    delta_scan,
    delta_scan_backward,
    delta_scan_forward,
    delta_scan_step,
)
from oracle import sequence as orc
from sequence_helpers import TINY, TYPES, U32, UNIT, assert_within, normal

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")
C = 64
NAMES = ("out", "last", "q", "k", "v", "gate", "beta", "state")


def _errors(dtype):
    n, u = 136 * U32, UNIT[torch.bfloat16]
    chain = n if dtype == torch.float32 else n + 3 * u * u
    return chain, n + 2 * u if dtype == torch.bfloat16 else chain


def _head(q, k, v, a, b, state, scale, do, dlast, dtype):
    """Bounds of one head's results before their last rounding, all inputs float64
    and zero (a: one) behind the sequence."""
    e_chain, e_out = _errors(dtype)
    tokens = q.shape[0]
    pad = -tokens % C
    q, k, v, do = (torch.cat([t, t.new_zeros(pad, t.shape[1])]) for t in (q, k, v, do))
    a, b = torch.cat([a, a.new_ones(pad)]), torch.cat([b, b.new_zeros(pad)])
    out, chunks, err_s, s = [], [], 0.0, state
    eye = torch.eye(C, dtype=torch.float64)
    for c in range(0, tokens + pad, C):
        x = {"q": q[c:c + C], "k": k[c:c + C], "v": v[c:c + C], "do": do[c:c + C], "b": b[c:c + C], "s": s,
             "err_s": err_s}
        g = a[c:c + C].log2().clamp_min(-300).cumsum(0)
        gap = (g[:, None] - g[None]).tril()
        x["d"] = torch.exp2(gap).tril()
        x["slip"] = (3 + gap.abs()) * U32
        x["up"], x["down"] = torch.exp2(g), torch.exp2(g[-1] - g)
        bk = x["b"][:, None] * x["up"][:, None] * x["k"]
        system = (x["b"][:, None] * x["d"] * (x["k"] @ x["k"].T)).tril(-1)
        t = torch.linalg.inv(eye + system)
        at = t.abs()
        err_t = at @ ((e_chain + x["slip"]) * system.abs() + 70 * U32 * (eye + system.abs())) @ at
        x["t"], x["err_t"], x["w"] = t, err_t, t @ bk
        bv = x["b"][:, None] * x["v"]
        f = t @ bv
        err_w = err_t @ bk.abs() + e_chain * (at @ bk.abs() + x["w"].abs())
        x["err_w"] = err_w
        err_u = err_t @ bv.abs() + e_chain * (at @ bv.abs() + f.abs() + x["w"].abs() @ s.abs()) + err_w @ s.abs()
        x["u"] = f - x["w"] @ s
        x["row_u"] = err_u.norm(dim=1) + x["w"].norm(dim=1) * err_s
        x["p"] = scale * x["d"] * (x["q"] @ x["k"].T)
        reach = scale * x["up"][:, None] * x["q"]
        out.append(reach.norm(dim=1, keepdim=True) * err_s + x["p"].abs() @ x["row_u"][:, None]
                   + (e_out + x["slip"].amax()) * (reach.abs() @ s.abs() + x["p"].abs() @ x["u"].abs()))
        x["reach"] = reach
        down = x["down"][:, None] * x["k"]
        last = torch.exp2(g[-1]) * s + down.T @ x["u"]
        err_s = float(err_s + torch.linalg.matrix_norm(down, 2) * err_u.norm()
                      + (e_chain + 4 * U32) * (s.norm() + (down.abs().T @ x["u"].abs()).norm()))
        s = x["after"] = last
        x["err_after"] = err_s
        chunks.append(x)
    result = {"out": torch.cat(out)[:tokens], "last": err_s}
    ds, err_ds = dlast, 0.0
    rows = {n: [] for n in ("q", "k", "v", "gate", "beta")}
    for x in reversed(chunks):
        up, down, b, d, u, s, do = (x[n] for n in ("up", "down", "b", "d", "u", "s", "do"))
        p, slip = x["p"], x["slip"]
        top = float(slip.amax())
        free = p.T @ do
        kd = down[:, None] * (x["k"] @ ds)
        du = free + kd
        err_du = ((2 * e_chain + top) * (p.abs().T @ do.abs())
                  + (e_chain + top) * (free.abs() + down[:, None] * (x["k"].abs() @ ds.abs())))
        row_du = err_du.norm(dim=1) + down * x["k"].norm(dim=1) * err_ds
        at = x["t"].abs()
        dr = x["t"].T @ du
        row_r = (x["err_t"].T @ du.abs() + e_chain * (at.T @ du.abs())).norm(dim=1) + at.T @ row_du
        n_mat, m_mat = scale * d * (do @ u.T), (d * (dr @ u.T)).tril(-1)
        err_n = scale * d * (do.norm(dim=1)[:, None] * x["row_u"] + (e_out + slip) * (do.abs() @ u.abs().T))
        err_n = err_n + e_out * n_mat.abs()
        err_m = d * (row_r[:, None] * u.norm(dim=1) + dr.norm(dim=1)[:, None] * x["row_u"]
                     + (e_out + slip) * (dr.abs() @ u.abs().T)).tril(-1)
        err_m = err_m + e_out * m_mat.abs()
        aq, ak = x["q"].abs(), x["k"].abs()
        size_s, size_ds = (float(torch.linalg.matrix_norm(t, 2)) for t in (s, ds))
        dq_mag = scale * up[:, None] * (do.abs() @ s.abs().T) + n_mat.abs() @ ak
        dq = (scale * up * do.norm(dim=1) * x["err_s"])[:, None] + (e_out + top) * dq_mag + err_n @ ak
        z_mag = up[:, None] * (dr.abs() @ s.abs().T) + m_mat.abs() @ ak
        z = (up * (dr.norm(dim=1) * x["err_s"] + row_r * size_s))[:, None] + (e_out + top) * z_mag + err_m @ ak
        bm = b[:, None] * m_mat.abs()
        y_mag = down[:, None] * (u.abs() @ ds.abs().T) + n_mat.abs().T @ aq + bm.T @ ak
        y = ((down * (x["row_u"] * size_ds + u.norm(dim=1) * err_ds))[:, None] + (e_out + top) * y_mag
             + err_n.T @ aq + (b[:, None] * err_m).T @ ak)
        few = 136 * U32
        rows["q"].append(dq)
        rows["k"].append(b[:, None] * z + y)
        rows["v"].append((b * row_r)[:, None].expand_as(du))
        # b db = u . dR, which the formula's other side equals.
        rows["beta"].append(row_r * u.norm(dim=1) + dr.norm(dim=1) * x["row_u"] + e_out * (dr * u).abs().sum(1))
        # What crosses a token: pairs, reads of the state before, writes into dS', and the
        # state itself; the sums in float32 of all of it.
        pair = n_mat.abs() * (aq @ ak.T) + bm * (ak @ ak.T)
        err_pair = (err_n + few * n_mat.abs()) * (aq @ ak.T) + (b[:, None] * err_m + few * bm) * (ak @ ak.T)
        read_q = scale * up[:, None] * (do.abs() @ s.abs().T) * aq
        read_k = (b * up)[:, None] * (dr.abs() @ s.abs().T) * ak
        err_r = ((scale * up * do.norm(dim=1) * x["err_s"])[:, None] * aq
                 + (b * up * (dr.norm(dim=1) * x["err_s"] + row_r * size_s))[:, None] * ak
                 + (e_out + top) * (read_q + read_k)).sum(1)
        write = down[:, None] * (u.abs() @ ds.abs().T) * ak
        err_w = ((down * (x["row_u"] * size_ds + u.norm(dim=1) * err_ds))[:, None] * ak
                 + (e_out + top) * write).sum(1)
        inner = float(up[-1]) * (x["err_s"] * float(ds.norm()) + float(s.norm()) * err_ds)
        own = few * float((s.abs() * ds.abs()).sum() + pair.sum() + (read_q + read_k + write).sum())
        over = torch.arange(C)
        after, before = over[:, None] >= over[None], over[:, None] < over[None]  # [i, t], [j, t]
        cross = ((err_pair @ before.double()) * after).sum(0)
        rows["gate"].append(cross + err_r @ after.double() + err_w @ before.double() + inner + own)
        reach = x["reach"]
        new = torch.exp2(torch.log2(up[-1])) * ds + reach.T @ do - x["w"].T @ du
        err_ds = float(err_ds + torch.linalg.matrix_norm(x["w"], 2) * err_du.norm()
                       + (x["err_w"].T @ du.abs()).norm()
                       + (2 * e_chain + top) * (ds.norm() + (reach.abs().T @ do.abs()).norm()
                                                + (x["w"].abs().T @ du.abs()).norm()))
        ds = new
    for name, parts in rows.items():
        result[name] = torch.cat(parts[::-1])[:tokens]
    result["state"] = err_ds
    return result


def _bounds(values, q, k, v, gate, beta, state, scale, lengths, do, dlast):
    """Bounds of all results, shaped like the values."""
    dtype = q.dtype
    h, hk = v.shape[2], q.shape[2]
    tokens = q.shape[1]
    bounds = [torch.zeros(t.shape, dtype=torch.float64) for t in values]
    scale = 1 / math.sqrt(q.shape[3]) if scale is None else scale
    a, b = torch.sigmoid(gate.double()), torch.sigmoid(beta.double())
    for i in range(q.shape[0]):
        there = torch.arange(tokens) < (tokens if lengths is None else int(lengths[i]))
        row = there[:, None].double()
        kept = lambda t: t[i].double().where(row > 0, torch.zeros(()).double())  # noqa: E731
        for n in range(h):
            m = n * hk // h
            one = _head(kept(q[:, :, m]), kept(k[:, :, m]), kept(v[:, :, n]),
                        torch.where(there, a[i, :, n], 1.0), torch.where(there, b[i, :, n], 0.0),
                        torch.zeros(q.shape[3], v.shape[3], dtype=torch.float64) if state is None
                        else state[i, n].double(), scale, kept(do[:, :, n]), dlast[i, n].double(), dtype)
            bounds[0][i, :, n] = one["out"] * row
            bounds[1][i, n] = one["last"]
            bounds[2][i, :, m] += one["q"] * row
            bounds[3][i, :, m] += one["k"] * row
            bounds[4][i, :, n] = one["v"] * row
            # 1 - sigmoid(x) is sigmoid(-x), which float64 does not get from the difference.
            bounds[5][i, :, n] = one["gate"] * torch.sigmoid(-gate[i, :, n].double()) * row[:, 0]
            bounds[6][i, :, n] = one["beta"] * torch.sigmoid(-beta[i, :, n].double()) * row[:, 0]
            bounds[5][i, ~there, n] = bounds[6][i, ~there, n] = 0.0
            bounds[7][i, n] = one["state"]
    for j, (value, bound) in enumerate(zip(values, bounds)):
        kind = torch.float32 if j in (1, 7) else dtype
        # Gates and decays below float32's smallest normal number, 2^-126, may be zero;
        # here they multiply sums of less than 64.
        bound += 2.0**-120
        bound += (UNIT[kind] + 16 * U32) * value.abs() + TINY[kind]
    return bounds


def _inputs(b, t, h, hk, d, dv, dtype, seed=0, shift=3.0):
    unit = lambda s: torch.nn.functional.normalize(normal((b, t, hk, d), torch.float32, s), dim=-1)  # noqa: E731
    # A little below one, so that rounding makes no key longer than one.
    q, k = ((unit(seed + s) * (1 - UNIT[dtype])).to(dtype) for s in (1, 2))
    return (q, k, normal((b, t, h, dv), dtype, seed + 3), normal((b, t, h), dtype, seed + 4, 2.0, shift),
            normal((b, t, h), dtype, seed + 5))


def _check(inputs, state=None, scale=None, lengths=None, seed=50):
    q, k, v, gate, beta = inputs
    b, t, h, dv = v.shape
    d = q.shape[3]
    do, dlast = normal(v.shape, v.dtype, seed), normal((b, h, d, dv), torch.float32, seed + 1)
    values = orc.delta_scan(q, k, v, gate, beta, state, scale, lengths, (do, dlast))
    bounds = _bounds(values, q, k, v, gate, beta, state, scale, lengths, do, dlast)
    on = [x.detach().to(DEV).requires_grad_(True) for x in inputs]
    s = None if state is None else state.to(DEV).requires_grad_(True)
    at = None if lengths is None else lengths.to(DEV)
    got = delta_scan(*on, s, scale, at)
    assert got[0].dtype == v.dtype and got[1].dtype == torch.float32
    leaves = on if s is None else [*on, s]
    grads = torch.autograd.grad(got, leaves, (do.to(DEV), dlast.to(DEV)))
    for name, x, value, bound in zip(NAMES, (*got, *grads), values, bounds):
        assert x.dtype == (torch.float32 if name in ("last", "state") else v.dtype)
        assert_within(x, value, bound, name)
    return got, grads


SHAPES = [(1, 1, 1, 1, 8, 8), (2, 2, 2, 1, 16, 24), (1, 63, 2, 2, 64, 64), (1, 64, 3, 1, 40, 72),
          (2, 65, 2, 1, 64, 128), (1, 129, 2, 2, 128, 64), (1, 200, 2, 1, 128, 128), (1, 330, 1, 1, 72, 8),
          (3, 17, 6, 2, 8, 104), (1, 500, 2, 2, 64, 64)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_matches_definition(shape, dtype):
    print(f"[delta] {shape} {dtype}", flush=True)
    b, _, h, _, d, dv = shape
    _check(_inputs(*shape, dtype), normal((b, h, d, dv), torch.float32, 9))
    _check(_inputs(*shape, dtype, 20), scale=0.7)


@pytest.mark.parametrize("dtype", TYPES)
def test_errors_as_a_whole(dtype):
    """The bounds take every rounding at its worst.  Roundings that know nothing of one
    another leave a sum the relative error (2-norm) of a term, at most their unit over
    sqrt(3) each: results in 16 bits, with three of them (six and a difference for the
    gates), stay within 2 (4) units, states within 2^-16, of some dozen parts' roundings
    of 2^-18 and less; float32, sums of about a hundred terms, within 2^-18."""
    inputs = _inputs(2, 700, 2, 1, 64, 64, dtype)
    state = normal((2, 2, 64, 64), torch.float32, 9)
    do, dlast = normal(inputs[2].shape, dtype, 50, 0.1), normal(state.shape, torch.float32, 51, 0.1)
    values = orc.delta_scan(*inputs, state, grads=(do, dlast))
    on = [t.to(DEV).requires_grad_(True) for t in (*inputs, state)]
    got = delta_scan(*on)
    grads = torch.autograd.grad(got, on, (do.to(DEV), dlast.to(DEV)))
    for name, x, value in zip(NAMES, (*got, *grads), values):
        off = float((x.detach().cpu().double() - value).norm() / value.norm())
        if dtype == torch.float32:
            most = 2.0**-18
        elif name in ("last", "state"):
            most = 2.0**-16
        else:
            most = (4 if name == "gate" else 2) * UNIT[dtype]
        print(f"[delta] {dtype} {name} {off:.2e} of {most:.2e}", flush=True)
        assert off <= most, (name, off, most)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(1, 8300, 2, 1, 64, 64), (1, 8192, 1, 1, 40, 72), (1, 8501, 1, 1, 128, 104)])
def test_long_sequences(shape, dtype):
    """Sequences of so many chunks that the chain is cut into segments: as exact as a
    whole as shorter ones, with a few units more for the segments' maps, and the same
    values as in two calls that hand the state on."""
    b, t, h, hk, d, dv = shape
    print(f"[delta] long {shape} {dtype}", flush=True)
    inputs = _inputs(*shape, dtype, shift=5.0)
    state = normal((b, h, d, dv), torch.float32, 9)
    do, dlast = normal(inputs[2].shape, dtype, 50, 0.1), normal(state.shape, torch.float32, 51, 0.1)
    values = orc.delta_scan(*inputs, state, grads=(do, dlast))
    on = [x.to(DEV).requires_grad_(True) for x in (*inputs, state)]
    got = delta_scan(*on)
    grads = torch.autograd.grad(got, on, (do.to(DEV), dlast.to(DEV)))
    for name, x, value in zip(NAMES, (*got, *grads), values):
        off = float((x.detach().cpu().double() - value).norm() / value.norm())
        if dtype == torch.float32:
            most = 2.0**-17
        elif name in ("last", "state"):
            most = 2.0**-15
        else:
            most = (4 if name == "gate" else 2) * UNIT[dtype]
        print(f"[delta] long {dtype} {name} {off:.2e} of {most:.2e}", flush=True)
        assert off <= most, (name, off, most)
    with torch.no_grad():
        first, middle = delta_scan(*(x[:, :4096] for x in on[:5]), on[5])
        rest, last = delta_scan(*(x[:, 4096:] for x in on[:5]), middle)
    for a, c in ((torch.cat([first, rest], 1), got[0]), (last, got[1])):
        unit = UNIT[a.dtype] if a.dtype == dtype else U32
        chain = 2.0**-20 if dtype == torch.float32 else 2.0**-15
        assert float((a.double() - c.double()).norm() / c.double().norm()) <= 2 * unit + chain


@pytest.mark.parametrize("dtype", TYPES)
def test_lengths(dtype):
    """Sequences that end early, at once and beyond: what lies behind is not read."""
    inputs = _inputs(5, 150, 2, 1, 32, 40, dtype)
    lengths = torch.tensor([150, 0, 64, 97, 1], dtype=torch.int32)
    for t in inputs:
        for i, n in enumerate(lengths.tolist()):
            t[i, n:] = float("nan")
    state = normal((5, 2, 32, 40), torch.float32, 9)
    (out, last), grads = _check(inputs, state, lengths=lengths)
    assert torch.equal(last[1].cpu(), state[1])
    far = torch.tensor([200, -3, 64, 97, 1], dtype=torch.int32, device=DEV)
    again, end = delta_scan(*(t.to(DEV) for t in inputs), state.to(DEV), lengths=far)
    assert torch.equal(again, out) and torch.equal(end, last)


@pytest.mark.parametrize("dtype", TYPES)
def test_gates_of_any_size(dtype):
    """Gates that forget at once, at infinity and where an exponential ends; b of zero
    and of one."""
    q, k, v, gate, beta = _inputs(1, 170, 2, 2, 32, 32, dtype)
    sizes = [-float("inf"), -6e4, -200.0, -104.0, -89.0, -40.0, -10.0, 0.0, 12.0, 40.0, 89.0, 6e4, float("inf")]
    for i, s in enumerate(sizes):
        gate[0, 5 + 12 * i, 0] = s
        beta[0, 9 + 12 * i, 1] = s
    gate[0, 70:90, 1] = float("inf")
    gate[0, 120:126, 1] = -float("inf")
    _check((q, k, v, gate, beta), normal((1, 2, 32, 32), torch.float32, 9))


@pytest.mark.parametrize("dtype", TYPES)
def test_equal_keys(dtype):
    """The same key for every token: a triangle without a small entry, b near one."""
    q, k, v, gate, beta = _inputs(1, 140, 1, 1, 64, 32, dtype)
    k = k[:, :1].expand_as(k).contiguous()
    beta = beta + 4.0
    gate = gate + 6.0
    _check((q, k, v, gate, beta), normal((1, 1, 64, 32), torch.float32, 9))


def test_no_gradient_of_out_or_last():
    inputs = [t.to(DEV).requires_grad_(True) for t in _inputs(1, 100, 2, 1, 32, 32, torch.float32)]
    state = normal((1, 2, 32, 32), torch.float32, 9).to(DEV).requires_grad_(True)
    out, last = delta_scan(*inputs, state)
    do, dlast = torch.randn_like(out), torch.randn_like(last)
    both = torch.autograd.grad((out, last), [*inputs, state], (do, dlast), retain_graph=True)
    one = torch.autograd.grad(out, [*inputs, state], do, retain_graph=True)
    other = torch.autograd.grad(last, [*inputs, state], dlast)
    for a, b, c in zip(both, one, other):
        torch.testing.assert_close(a, b + c, rtol=1e-4, atol=1e-5)


def test_gradient_by_differences():
    g = torch.Generator().manual_seed(3)
    inputs = [t.to(DEV) for t in _inputs(1, 130, 2, 1, 16, 24, torch.float32)]
    inputs.append(normal((1, 2, 16, 24), torch.float32, 9).to(DEV))
    weights = [torch.randn((1, 130, 2, 24), generator=g).to(DEV), torch.randn((1, 2, 16, 24), generator=g).to(DEV)]
    leaves = [t.clone().requires_grad_(True) for t in inputs]
    grads = torch.autograd.grad(delta_scan(*leaves), leaves, weights)
    for i, t in enumerate(inputs):
        step = torch.randn(t.shape, generator=g).to(DEV)
        step *= 1e-2 / step.abs().max()

        def value(s):
            moved = [x + s * step if j == i else x for j, x in enumerate(inputs)]
            return sum(float((a.double() * w.double()).sum()) for a, w in zip(delta_scan(*moved), weights))

        slope = (8 * (value(1) - value(-1)) - (value(2) - value(-2))) / 12
        want = float((grads[i].double() * step.double()).sum())
        size = float((grads[i].double().norm() * step.double().norm()))
        # The fourth-order formula leaves a step's fifth power, the values float32's
        # rounding of some thousand terms of size one.
        assert abs(slope - want) <= 1e-3 * size + 1e-3, (i, slope, want)


def test_strides_and_broadcasts():
    """Views of one projection, heads before tokens, gates across the batch."""
    b, t, h, hk, d, dv = 2, 90, 4, 2, 32, 40
    whole = normal((b, t, 2 * hk * d + h * dv + 2 * h), torch.bfloat16, 1).to(DEV) * 0.1
    q, k, v, gate, beta = whole.split([hk * d, hk * d, h * dv, h, h], -1)
    q, k = q.view(b, t, hk, d), k.view(b, t, hk, d)
    v = v.view(b, t, h, dv).transpose(1, 2).contiguous().transpose(1, 2)
    gate = gate[:1].expand(b, t, h)
    state = normal((1, h, d, dv), torch.float32, 2).to(DEV).expand(b, h, d, dv)
    want = delta_scan(*(x.contiguous() for x in (q, k, v, gate, beta)), state.contiguous())
    got = delta_scan(q, k, v, gate, beta, state)
    for a, c in zip(got, want):
        assert torch.equal(a, c)
    leaf = gate[:1].detach().clone().requires_grad_(True)
    out, _ = delta_scan(q, k, v, leaf.expand(b, t, h), beta, state)
    full = gate.detach().contiguous().requires_grad_(True)
    ref, _ = delta_scan(q, k, v, full, beta, state)
    do = torch.randn_like(out)
    (one,), (both,) = torch.autograd.grad(out, leaf, do), torch.autograd.grad(ref, full, do)
    torch.testing.assert_close(one, both.sum(0, keepdim=True), rtol=2**-7, atol=1e-6)


@pytest.mark.parametrize("dtype", TYPES)
def test_not_finite(dtype):
    """From a token that is not finite on, its head is NaN; tokens before it, other heads
    and other sequences keep their bits.  A query is a matter of its own row."""
    inputs = [t.to(DEV) for t in _inputs(2, 200, 2, 2, 32, 32, dtype)]
    want, last = delta_scan(*inputs)
    for which, place in ((1, (0, 100, 1, 3)), (2, (0, 100, 1, 3)), (3, (0, 100, 1)), (4, (0, 100, 1))):
        for value in (float("nan"), float("inf")):
            if which > 2 and value != value:
                pass
            elif which > 2:
                continue  # infinite gates are numbers
            bad = [t.clone() for t in inputs]
            bad[which][place] = value
            out, end = delta_scan(*bad)
            assert out[0, 100:, 1].isnan().all() and end[0, 1].isnan().all()
            keep = torch.ones_like(want, dtype=torch.bool)
            keep[0, 100:, 1] = False
            assert torch.equal(out[keep], want[keep])
            assert torch.equal(end[1], last[1]) and torch.equal(end[0, 0], last[0, 0])
    bad = [t.clone() for t in inputs]
    bad[0][0, 100, 1, 3] = float("nan")
    out, end = delta_scan(*bad)
    assert out[0, 100, 1].isnan().all() and int(out.isnan().sum()) == 32 and torch.equal(end, last)


def test_empty():
    inputs = [t.to(DEV).requires_grad_(True) for t in _inputs(2, 0, 2, 1, 16, 8, torch.bfloat16)]
    state = normal((2, 2, 16, 8), torch.float32, 1).to(DEV).requires_grad_(True)
    out, last = delta_scan(*inputs, state)
    assert out.shape == (2, 0, 2, 8) and torch.equal(last, state)
    (grad,) = torch.autograd.grad(last, state, torch.ones_like(last))
    assert torch.equal(grad, torch.ones_like(grad))
    out, last = delta_scan(*(t[:0] for t in _inputs(2, 9, 2, 1, 16, 8, torch.bfloat16) for t in [t.to(DEV)]))
    assert out.shape == (0, 9, 2, 8) and last.shape == (0, 2, 16, 8)
    assert not delta_scan(*inputs)[1].any()


def test_parts_equal_the_whole():
    """A sequence cut anywhere, its state handed on, and taken token by token."""
    inputs = [t.to(DEV) for t in _inputs(2, 200, 4, 2, 64, 32, torch.float32)]
    out, last = delta_scan(*inputs)
    for cut in (1, 64, 100, 199):
        first, state = delta_scan(*(t[:, :cut] for t in inputs))
        rest, end = delta_scan(*(t[:, cut:] for t in inputs), state)
        # Two float32 sums of two hundred numbers of about one.
        torch.testing.assert_close(torch.cat([first, rest], 1), out, rtol=1e-4, atol=2e-5)
        torch.testing.assert_close(end, last, rtol=1e-4, atol=2e-5)
    state = torch.zeros(2, 4, 64, 32, device=DEV)
    for t in range(200):
        row, same = delta_scan_step(*(x[:, t] for x in inputs), state, state_out=state)
        assert same is state
        torch.testing.assert_close(row, out[:, t], rtol=1e-4, atol=2e-5)
    torch.testing.assert_close(state, last, rtol=1e-4, atol=2e-5)


def test_same_bits_again_and_on_another_stream():
    inputs = [t.to(DEV).requires_grad_(True) for t in _inputs(1, 300, 4, 2, 64, 64, torch.bfloat16)]
    do = normal((1, 300, 4, 64), torch.bfloat16, 9).to(DEV)
    first = delta_scan(*inputs)
    grads = torch.autograd.grad(first[0], inputs, do)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = delta_scan(*inputs)
        again = torch.autograd.grad(second[0], inputs, do)
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip((*first, *grads), (*second, *again)):
        assert torch.equal(a, b)


def test_in_a_graph():
    """Forward and backward kernels, captured: replays follow the buffers' contents."""
    inputs = [t.to(DEV) for t in _inputs(1, 150, 4, 2, 64, 64, torch.bfloat16)]
    do = normal((1, 150, 4, 64), torch.bfloat16, 9).to(DEV)

    def run():
        out, last, kept = delta_scan_forward(*inputs)
        return out, last, *delta_scan_backward(*inputs, kept, do, None)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = run()
    for turn in range(3):
        for x, fresh in zip(inputs, _inputs(1, 150, 4, 2, 64, 64, torch.bfloat16, 100 * turn)):
            x.copy_(fresh)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(captured, run()):
            assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(1, 1, 1, 8, 8), (3, 6, 2, 40, 24), (2, 4, 4, 64, 64), (2, 3, 1, 128, 128),
                                   (1, 2, 1, 72, 104), (33, 2, 2, 32, 40)])
def test_step_matches_definition(shape, dtype):
    b, h, hk, d, dv = shape
    inputs = [t[:, 0] for t in _inputs(b, 1, h, hk, d, dv, dtype)]
    state = normal((b, h, d, dv), torch.float32, 9)
    want, end = orc.delta_scan(*(t[:, None] for t in inputs), state)
    on = [t.to(DEV) for t in inputs]
    out, new = delta_scan_step(*on, state.to(DEV))
    # Sums of d products in float32, a few operations more.
    q, k, v = (t.double() for t in inputs[:3])
    of = torch.arange(h) * hk // h
    found = (k[:, of, :, None].abs() * state.double().abs()).sum(2) + v.abs()
    own = (2 * d + 16) * U32
    bound = own * (state.double().abs() + k[:, of, :, None].abs() * found[:, :, None])
    assert_within(new, end, bound + U32 * end.abs(), "state")
    reads = (q[:, of, :, None].abs() * (state.double().abs() + k[:, of, :, None].abs() * found[:, :, None])).sum(2)
    assert_within(out, want[:, 0], own * reads + UNIT[dtype] * want[:, 0].abs() + TINY[dtype], "out")
    again = state.to(DEV)
    twice, same = delta_scan_step(*on, again, state_out=again)
    assert same is again and torch.equal(twice, out) and torch.equal(again, new)


def test_step_strides_and_overlaps():
    inputs = [t[:, 0].to(DEV) for t in _inputs(2, 1, 4, 2, 32, 32, torch.bfloat16)]
    state = normal((2, 4, 32, 32), torch.float32, 9).to(DEV)
    want = delta_scan_step(*inputs, state)
    turned = [torch.stack([t, t], -1)[..., 0] for t in inputs]
    got = delta_scan_step(*turned, state.transpose(0, 1).contiguous().transpose(0, 1))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    room = torch.zeros(2 * 4 * 32 * 32 + 64, device=DEV)
    with pytest.raises(ValueError, match="overlaps"):
        delta_scan_step(*inputs, room[:-64].view(2, 4, 32, 32), state_out=room[64:].view(2, 4, 32, 32))


def test_offsets_beyond_32_bits():
    """Sequences whose tensors lie more than 2^31 elements apart."""
    apart = (1 << 31) + 64
    near = [t.to(DEV) for t in _inputs(2, 70, 1, 1, 16, 16, torch.bfloat16)]
    far = []
    for t in near:
        inner = t.stride()[1:]
        far.append(torch.empty(apart + t[0].numel() + 64, dtype=torch.bfloat16, device=DEV)
                   .as_strided(t.shape, (apart, *inner)))
        far[-1].copy_(t)
    do = normal((2, 70, 1, 16), torch.bfloat16, 9).to(DEV)
    results = []
    for inputs in (far, near):
        out, last, kept = delta_scan_forward(*inputs)
        results.append((out, last, *delta_scan_backward(*inputs, kept, do, None)))
    for a, b in zip(*results):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", TYPES)
def test_step_not_finite(dtype):
    """A step takes what is not finite where the formula does: a value into its column of
    the state, a key, gate or beta into its head; all else keeps its bits."""
    inputs = [t[:, 0].to(DEV) for t in _inputs(2, 1, 4, 2, 32, 40, dtype)]
    state = normal((2, 4, 32, 40), torch.float32, 9).to(DEV)
    want, new = delta_scan_step(*inputs, state)
    for which, place in ((1, (0, 1, 3)), (2, (0, 2, 5)), (3, (0, 2)), (4, (0, 2))):
        bad = [t.clone() for t in inputs]
        bad[which][place] = float("nan")
        out, end = delta_scan_step(*bad, state)
        keep = torch.ones_like(want, dtype=torch.bool)
        if which == 2:
            keep[0, 2, 5] = False
        else:
            keep[0, 2:4 if which == 1 else 3] = False  # the key's two heads
        assert out[~keep].isnan().all() and torch.equal(out[keep], want[keep])
        there = keep[:, :, None].expand_as(end)
        assert end[~there].isnan().all() and torch.equal(end[there], new[there])
