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
