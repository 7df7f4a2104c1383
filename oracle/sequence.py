"""Sequence operators in float64, from their definitions: the restatement that
the HIP kernels are tested against."""

from __future__ import annotations

import math

import torch


def add_rms_norm(x, residual, weight, eps):
    """(y, s): s = x + residual, y = s / sqrt(mean(s^2) + eps) * weight."""
    s = x.double() if residual is None else x.double() + residual.double()
    return s / torch.sqrt((s * s).mean(-1, keepdim=True) + eps) * weight.double(), s


def add_rms_norm_grads(x, residual, weight, eps, grad_y, grad_s):
    """Gradients of s (those of x and the residual) and of weight."""
    _, s = add_rms_norm(x, residual, weight, eps)
    r = 1 / torch.sqrt((s * s).mean(-1, keepdim=True) + eps)
    unit, t = s * r, grad_y.double() * weight.double()
    ds = r * (t - unit * (t * unit).mean(-1, keepdim=True)) + grad_s.double()
    dw = (grad_y.double() * unit).reshape(-1, s.shape[-1]).sum(0)
    return ds, dw


def gated_scan(x, gate, state=None):
    """(y, last) of h_t = a h + (1 - a) x, a = sigmoid(gate), token after token."""
    x, a = x.double(), torch.sigmoid(gate.double())
    keep = torch.sigmoid(-gate.double())
    h = torch.zeros_like(x[:, 0]) if state is None else state.double()
    y = torch.empty_like(x)
    for t in range(x.shape[1]):
        h = a[:, t] * h + keep[:, t] * x[:, t]
        y[:, t] = h
    return y, h


def gated_scan_grads(x, gate, state, grad_y, grad_last):
    """Gradients of x, gate and state."""
    y, _ = gated_scan(x, gate, state)
    x, a, keep = x.double(), torch.sigmoid(gate.double()), torch.sigmoid(-gate.double())
    start = torch.zeros_like(x[:, 0]) if state is None else state.double()
    dx, dg = torch.empty_like(x), torch.empty_like(x)
    r = grad_last.double()
    for t in range(x.shape[1] - 1, -1, -1):
        g = grad_y[:, t].double() + r
        dx[:, t] = keep[:, t] * g
        dg[:, t] = g * ((y[:, t - 1] if t else start) - x[:, t]) * a[:, t] * keep[:, t]
        r = a[:, t] * g
    return dx, dg, r


def window_mask(tq, tk, window, sinks, length=None):
    """[tq, tk], true where query i at position tk - tq + i sees key j: not
    after it, within the window or among the first tokens, and not beyond the
    sequence's length."""
    p = torch.arange(tk - tq, tk)[:, None]
    j = torch.arange(tk)[None]
    seen = (j <= p) & ((j > p - window) | (j < sinks))
    return seen if length is None else seen & (j < length)


def window_attention(q, k, v, window, sinks, scale=None, lengths=None, grad=None):
    """Output [B, Tq, H, D]; with ``grad`` also the gradients of q, k and v.
    A query that sees no key gives zeros; what a query does not see (NaN
    included) does not reach it."""
    b, tq, h, d = q.shape
    tk, hk = k.shape[1], k.shape[2]
    scale = 1 / math.sqrt(d) if scale is None else scale
    q, k, v = q.double(), k.double(), v.double()
    out, dq, dk, dv = (torch.zeros_like(t) for t in (q, q, k, v))
    for i in range(b):
        seen = window_mask(tq, tk, window, sinks, None if lengths is None else int(lengths[i]))
        for n in range(h):
            m = n * hk // h
            for r in range(tq):
                at = seen[r].nonzero()[:, 0]
                if at.numel() == 0:
                    continue
                kk, vv = k[i, at, m], v[i, at, m]
                p = torch.softmax(kk @ q[i, r, n] * scale, 0)
                out[i, r, n] = p @ vv
                if grad is None:
                    continue
                g = grad[i, r, n].double()
                ds = p * (vv @ g - g @ out[i, r, n]) * scale
                dq[i, r, n] = ds @ kk
                dk[i, at, m] += ds[:, None] * q[i, r, n]
                dv[i, at, m] += p[:, None] * g
    return out if grad is None else (out, dq, dk, dv)


def cache_slot(position, window, sinks):
    return position if position < sinks else sinks + (position - sinks) % window


def window_attention_step(q, k, v, k_cache, v_cache, positions, window, sinks, scale=None):
    """(out, k_cache, v_cache) of one token of each stream; the caches are
    changed copies."""
    k_cache, v_cache = k_cache.clone(), v_cache.clone()
    b, h, d = q.shape
    hk = k.shape[1]
    scale = 1 / math.sqrt(d) if scale is None else scale
    out = torch.zeros(q.shape, dtype=torch.float64)
    for i in range(b):
        p = int(positions[i])
        slot = cache_slot(p, window, sinks)
        k_cache[i, slot], v_cache[i, slot] = k[i], v[i]
        n = min(p + 1, sinks + window)
        for m in range(h):
            kk = k_cache[i, :n, m * hk // h].double()
            w = torch.softmax(kk @ q[i, m].double() * scale, 0)
            out[i, m] = w @ v_cache[i, :n, m * hk // h].double()
    return out, k_cache, v_cache


#: What the 4-bit codes 0 .. 7 stand for; 8 .. 15 are their negatives.
MXFP4_VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def mxfp4_encode(x):
    """(codes [.., n / 2], exponents [.., n / 32]) of rows, uint8: the power of two
    of a block of 32 is floor(log2 max|x|) - 2, not below -127, held + 127; elements
    go to the nearest value, of two as near the one of the even code.  A block that
    is not finite has the exponent 255 and codes of zero."""
    x = x.double().unflatten(-1, (-1, 32))
    top = x.abs().amax(-1)
    fine = torch.isfinite(x).all(-1)
    power = torch.where(top > 0, torch.floor(torch.log2(torch.where(top > 0, top, 1.0))) - 2, -127.0)
    power = torch.where(fine, power, 0.0).clamp(-127, 127)
    y = (x.abs() / torch.exp2(power)[..., None])[..., None]
    even = (0, 2, 4, 6, 1, 3, 5, 7)
    levels = torch.tensor([MXFP4_VALUES[c] for c in even], dtype=torch.float64)
    codes = torch.tensor(even)[(y - levels).abs().nan_to_num(0.0).argmin(-1)] + 8 * torch.signbit(x)
    codes = torch.where(fine[..., None], codes, 0).flatten(-2).to(torch.uint8)
    exponents = torch.where(fine, power + 127, 255.0).to(torch.uint8)
    return codes[..., ::2] | codes[..., 1::2] << 4, exponents


def mxfp4_decode(codes, exponents):
    """What codes and exponents stand for, in float64."""
    values = torch.tensor(MXFP4_VALUES + tuple(-v for v in MXFP4_VALUES), dtype=torch.float64)
    x = values[torch.stack([codes & 15, codes >> 4], -1).flatten(-2).long()].unflatten(-1, (-1, 32))
    power = torch.exp2(exponents.double() - 127)
    return (x * torch.where(exponents == 255, float("nan"), power)[..., None]).flatten(-2)


def window_cache_fill(x, length, window, sinks, capacity):
    """The token that each slot of a cache takes of a sequence's first ``length``
    tokens; -1: none."""
    token = torch.full((capacity,), -1)
    for t in range(min(length, x.shape[0])):
        token[cache_slot(t, window, sinks)] = t
    return token


def delta_scan(q, k, v, gate, beta, state=None, scale=None, lengths=None, grads=None):
    """(out, last) of the gated delta rule, token after token; with ``grads``, those
    of out and last, also the gradients of q, k, v, gate, beta and state."""
    h, hk, d = v.shape[2], q.shape[2], q.shape[3]
    tokens = q.shape[1]
    scale = 1 / math.sqrt(d) if scale is None else scale
    of = torch.arange(h) * hk // h
    q, k, v, gate, beta = (t.double() for t in (q, k, v, gate, beta))
    qq, kk = q[:, :, of], k[:, :, of]
    a, b = torch.sigmoid(gate), torch.sigmoid(beta)
    there = torch.ones(a.shape[:2], dtype=torch.bool)
    if lengths is not None:
        there = torch.arange(tokens) < lengths.cpu()[:, None]
    hide = ~there[..., None]
    a, b = a.masked_fill(hide, 1.0), b.masked_fill(hide, 0.0)
    qq, kk, v = (t.masked_fill(hide[..., None], 0.0) for t in (qq, kk, v))
    s = torch.zeros(v.shape[0], h, d, v.shape[3], dtype=torch.float64) if state is None else state.double()
    states, out, u = [s], torch.empty_like(v), torch.empty_like(v)
    for t in range(tokens):
        kept = a[:, t, :, None, None] * s
        u[:, t] = b[:, t, :, None] * (v[:, t] - (kk[:, t, :, :, None] * kept).sum(2))
        s = kept + kk[:, t, :, :, None] * u[:, t, :, None]
        out[:, t] = scale * (qq[:, t, :, :, None] * s).sum(2)
        states.append(s)
    if grads is None:
        return out, s
    do = grads[0].double().masked_fill(hide[..., None], 0.0)
    ds = grads[1].double()
    dq, dk, dv = torch.empty_like(qq), torch.empty_like(kk), torch.empty_like(v)
    da, db = torch.empty_like(a), torch.empty_like(b)
    for t in range(tokens - 1, -1, -1):
        before, kt = states[t], kk[:, t, :, :, None]
        ds = ds + scale * qq[:, t, :, :, None] * do[:, t, :, None]
        dq[:, t] = scale * (states[t + 1] * do[:, t, :, None]).sum(-1)
        du = (kt * ds).sum(2)
        found = a[:, t, :, None] * (kt * before).sum(2)
        db[:, t] = (du * (v[:, t] - found)).sum(-1)
        dv[:, t] = b[:, t, :, None] * du
        # found, and through it a S and k, has the gradient -dv.
        dk[:, t] = (ds * u[:, t, :, None]).sum(-1) - a[:, t, :, None] * (before * dv[:, t, :, None]).sum(-1)
        through = ds - kt * dv[:, t, :, None]
        da[:, t] = (before * through).sum((-1, -2))
        ds = a[:, t, :, None, None] * through
    shared = [t.masked_fill(hide[..., None], 0.0).unflatten(2, (hk, h // hk)).sum(3) for t in (dq, dk)]
    dgate = (da * a * torch.sigmoid(-gate)).masked_fill(hide, 0.0)
    dbeta = (db * b * torch.sigmoid(-beta)).masked_fill(hide, 0.0)
    return (out, s, *shared, dv.masked_fill(hide[..., None], 0.0), dgate, dbeta, ds)
