"""The float64 restatement of the sequence operators: its gradients against
autograd of the definitions and against differences, its masks by hand."""

from __future__ import annotations

import torch

from oracle import sequence as orc
from sequence_helpers import normal


def _leaves(*ts):
    return [t.double().requires_grad_(True) for t in ts]


def test_norm_gradients():
    x, r, w = _leaves(normal((3, 9), torch.float64, 1), normal((3, 9), torch.float64, 2),
                      normal((9,), torch.float64, 3))
    dy, ds = normal((3, 9), torch.float64, 4), normal((3, 9), torch.float64, 5)
    y, s = orc.add_rms_norm(x, r, w, 1e-6)
    got = torch.autograd.grad((y, s), (x, r, w), (dy, ds))
    want = orc.add_rms_norm_grads(x.detach(), r.detach(), w.detach(), 1e-6, dy, ds)
    for a, b in zip(got, (want[0], want[0], want[1])):
        torch.testing.assert_close(a, b, rtol=1e-12, atol=1e-12)


def test_scan_gradients():
    x, g, s = _leaves(normal((2, 11, 3), torch.float64, 1), normal((2, 11, 3), torch.float64, 2),
                      normal((2, 3), torch.float64, 3))
    assert torch.autograd.gradcheck(lambda a, b: _scan(a, b, s.detach()), (x, g))
    dy, dl = normal((2, 11, 3), torch.float64, 4), normal((2, 3), torch.float64, 5)
    got = torch.autograd.grad(_scan(x, g, s), (x, g, s), (dy, dl))
    for a, b in zip(got, orc.gated_scan_grads(x.detach(), g.detach(), s.detach(), dy, dl)):
        torch.testing.assert_close(a, b, rtol=1e-12, atol=1e-12)


def _scan(x, gate, state):
    """The recurrence without in-place writes, for autograd."""
    h, rows = state, []
    for t in range(x.shape[1]):
        a = torch.sigmoid(gate[:, t])
        h = a * h + (1 - a) * x[:, t]
        rows.append(h)
    return torch.stack(rows, 1), h


def test_scan_is_compositing():
    """Back to front, a step with 1 - a = alpha lays colour x over h."""
    alpha, colour = torch.rand(1, 6, 1).double(), torch.rand(1, 6, 1).double()
    _, last = orc.gated_scan(colour, torch.log((1 - alpha) / alpha))
    t, c = 1.0, 0.0
    for i in range(5, -1, -1):  # the last token is in front
        c, t = c + t * alpha[0, i, 0] * colour[0, i, 0], t * (1 - alpha[0, i, 0])
    torch.testing.assert_close(last[0, 0], c)


def test_window_mask_by_hand():
    got = orc.window_mask(4, 6, 2, 1)
    want = torch.tensor([[1, 1, 1, 0, 0, 0], [1, 0, 1, 1, 0, 0], [1, 0, 0, 1, 1, 0], [1, 0, 0, 0, 1, 1]])
    assert torch.equal(got, want.bool())
    # More queries than keys: the first ones lie before every key.
    assert not orc.window_mask(5, 3, 2, 1)[:2].any()
    assert not orc.window_mask(4, 4, 1, 0, length=2)[2:].any()


def test_attention_gradients():
    q, k, v = _leaves(normal((2, 7, 4, 3), torch.float64, 1), normal((2, 9, 2, 3), torch.float64, 2),
                      normal((2, 9, 2, 3), torch.float64, 3))
    grad, lengths = normal((2, 7, 4, 3), torch.float64, 4), [9, 2]
    masks = torch.stack([orc.window_mask(7, 9, 3, 1, n) for n in lengths])[:, None]
    kk, vv = (t.repeat_interleave(2, 2).transpose(1, 2) for t in (k, v))
    s = (q.transpose(1, 2) @ kk.transpose(-1, -2) / 3**0.5).masked_fill(~masks, -1e300)
    out = (torch.softmax(s, -1) * masks @ vv).transpose(1, 2)
    got = (out, *torch.autograd.grad(out, (q, k, v), grad))
    want = orc.window_attention(q.detach(), k.detach(), v.detach(), 3, 1, lengths=lengths, grad=grad)
    for a, b in zip(got, want):
        torch.testing.assert_close(a.detach(), b, rtol=1e-12, atol=1e-12)


def test_step_is_a_row_of_attention():
    window, sinks, tokens = 3, 2, 12
    q, k, v = (normal((1, tokens, 2, 4), torch.float64, i) for i in (1, 2, 3))
    want = orc.window_attention(q, k, v, window, sinks)
    kc, vc = torch.zeros(1, window + sinks, 2, 4).double(), torch.zeros(1, window + sinks, 2, 4).double()
    for t in range(tokens):
        out, kc, vc = orc.window_attention_step(q[:, t], k[:, t], v[:, t], kc, vc, [t], window, sinks)
        torch.testing.assert_close(out, want[:, t], rtol=1e-12, atol=1e-12)
