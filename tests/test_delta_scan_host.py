"""The gated delta rule without a GPU: its oracle against autograd and differences, and
what the entry points turn away on the host."""

from __future__ import annotations

import ctypes

import pytest
import torch

from gaussian_splats_hip import sequence
from gaussian_splats_hip.kernels.rasterize import _native as nat
from oracle import sequence as orc

FAKE = ctypes.c_void_p(256)


def _rule(q, k, v, gate, beta, s, scale):
    """The definition once more, for autograd: heads one after the other."""
    group = v.shape[2] // q.shape[2]
    outs, lasts = [], []
    for h in range(v.shape[2]):
        state, rows = s[:, h], []
        for t in range(q.shape[1]):
            key, query = k[:, t, h // group], q[:, t, h // group]
            state = torch.sigmoid(gate[:, t, h])[:, None, None] * state
            found = torch.einsum("bd,bdn->bn", key, state)
            u = torch.sigmoid(beta[:, t, h])[:, None] * (v[:, t, h] - found)
            state = state + torch.einsum("bd,bn->bdn", key, u)
            rows.append(scale * torch.einsum("bd,bdn->bn", query, state))
        outs.append(torch.stack(rows, 1))
        lasts.append(state)
    return torch.stack(outs, 2), torch.stack(lasts, 1)


def test_oracle_against_autograd():
    g = torch.Generator().manual_seed(1)
    shapes = [(2, 9, 2, 5), (2, 9, 2, 5), (2, 9, 4, 3), (2, 9, 4), (2, 9, 4), (2, 4, 5, 3)]
    leaves = [torch.randn(s, generator=g, dtype=torch.float64).requires_grad_(True) for s in shapes]
    do, dlast = (torch.randn(s, generator=g, dtype=torch.float64) for s in ((2, 9, 4, 3), (2, 4, 5, 3)))
    out, last = _rule(*leaves, 0.3)
    grads = torch.autograd.grad((out, last), leaves, (do, dlast))
    got = orc.delta_scan(*(t.detach() for t in leaves), 0.3, None, (do, dlast))
    for a, b in zip(got, (out, last, *grads)):
        torch.testing.assert_close(a, b.detach(), rtol=1e-12, atol=1e-12)


def test_oracle_lengths():
    """A sequence that ends early is the shorter one, with zeros behind it."""
    g = torch.Generator().manual_seed(2)
    t = [torch.randn(s, generator=g, dtype=torch.float64) for s in
         ((2, 8, 1, 4), (2, 8, 1, 4), (2, 8, 2, 3), (2, 8, 2), (2, 8, 2), (2, 2, 4, 3))]
    do, dlast = torch.randn(2, 8, 2, 3, generator=g).double(), torch.randn(2, 2, 4, 3, generator=g).double()
    whole = orc.delta_scan(*t, None, torch.tensor([8, 5], dtype=torch.int32), (do, dlast))
    short = orc.delta_scan(*(x[1:, :5] for x in t[:5]), t[5][1:], grads=(do[1:, :5], dlast[1:]))
    for i, (a, b) in enumerate(zip(whole, short)):
        if i in (1, 7):
            torch.testing.assert_close(a[1:], b)
        else:
            torch.testing.assert_close(a[1:, :5], b)
            assert not a[1:, 5:].any()


def _tensors(b=2, t=5, h=4, hk=2, d=16, dv=24, dtype=torch.float32):
    return [torch.zeros(b, t, hk, d, dtype=dtype), torch.zeros(b, t, hk, d, dtype=dtype),
            torch.zeros(b, t, h, dv, dtype=dtype), torch.zeros(b, t, h, dtype=dtype),
            torch.zeros(b, t, h, dtype=dtype)]


def test_refusals():
    scan = sequence.delta_scan
    ok = _tensors()
    with pytest.raises(ValueError, match="ROCm GPU"):
        scan(*ok)
    with pytest.raises(TypeError, match="float64"):
        scan(*_tensors(dtype=torch.float64))
    for i, name in ((1, "k"), (2, "v"), (3, "gate"), (4, "beta")):
        bad = list(ok)
        bad[i] = ok[i].half()
        with pytest.raises(TypeError, match=f"{name} is torch.float16"):
            scan(*bad)
    with pytest.raises(ValueError, match="expects q and k"):
        scan(ok[0], ok[1][:, :4], *ok[2:])
    with pytest.raises(ValueError, match="expects q and k"):
        scan(ok[0], ok[1], ok[2][:1], *ok[3:])
    with pytest.raises(ValueError, match="expects q and k"):
        scan(*(t[0] for t in ok))
    with pytest.raises(ValueError, match="gate"):
        scan(*ok[:3], ok[3][:, :, :3], ok[4])
    with pytest.raises(ValueError, match="beta"):
        scan(*ok[:4], ok[4][..., None])
    with pytest.raises(ValueError, match="cannot share"):
        scan(*_tensors(h=3))
    with pytest.raises(TypeError, match="state"):
        scan(*ok, torch.zeros(2, 4, 16, 24).half())
    with pytest.raises(ValueError, match="state"):
        scan(*ok, torch.zeros(2, 4, 24, 16))
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        with pytest.raises(ValueError, match="scale"):
            scan(*ok, scale=scale)
    with pytest.raises(TypeError, match="lengths is"):
        scan(*ok, lengths=torch.zeros(2, dtype=torch.int64))
    with pytest.raises(ValueError, match="batch of 2"):
        scan(*ok, lengths=torch.zeros(3, dtype=torch.int32))
    step = [t[:, 0] for t in ok]
    state = torch.zeros(2, 4, 16, 24)
    with pytest.raises(ValueError, match="ROCm GPU"):
        sequence.delta_scan_step(*step, state)
    with pytest.raises(TypeError, match="needs a state"):
        sequence.delta_scan_step(*step, None)
    with pytest.raises(ValueError, match="state"):
        sequence.delta_scan_step(*step, state[:, :3])
    with pytest.raises(ValueError, match="expects q and k"):
        sequence.delta_scan_step(*ok, state)
    with pytest.raises(ValueError, match="not that of a forward"):
        sequence.delta_scan_backward(*ok, torch.zeros(7), None, None)
    with pytest.raises(TypeError, match="kept is"):
        sequence.delta_scan_backward(*ok, torch.zeros(7).half(), None, None)


def test_c_abi_checks():
    lib = nat.library()
    strides = (ctypes.c_int64 * 18)(*[64] * 18)

    def problem(b=1, t=70, h=2, hk=1, d=64, dv=64, kind=2, scale=0.1):
        return ctypes.byref(nat.GsDelta(b, t, h, hk, d, dv, kind, scale))

    def forward(p, q=FAKE, s=strides, kept=FAKE, bytes_=1 << 30, gate=FAKE):
        return lib.gs_delta_scan_fwd(p, q, FAKE, FAKE, gate, FAKE, s, None, None, 1, FAKE, FAKE, kept, FAKE,
                                     bytes_, None)

    assert forward(None) == nat.GS_ERR_INVALID_ARGUMENT
    for d in (4, 12, 136):
        assert forward(problem(d=d)) == nat.GS_ERR_UNSUPPORTED
        assert forward(problem(dv=d)) == nat.GS_ERR_UNSUPPORTED
    assert forward(problem(h=3, hk=2)) == nat.GS_ERR_INVALID_ARGUMENT
    assert forward(problem(b=-1)) == nat.GS_ERR_INVALID_ARGUMENT
    assert forward(problem(kind=3)) == nat.GS_ERR_INVALID_ARGUMENT
    assert forward(problem(scale=0.0)) == nat.GS_ERR_INVALID_ARGUMENT
    assert forward(problem(t=1 << 30)) == nat.GS_ERR_OVERFLOW
    assert forward(problem(b=1 << 20, t=1 << 29, h=64, hk=64)) == nat.GS_ERR_OVERFLOW
    assert forward(problem(), q=None) == nat.GS_ERR_INVALID_ARGUMENT
    assert forward(problem(), q=ctypes.c_void_p(264)) == nat.GS_ERR_INVALID_ARGUMENT
    assert forward(problem(), gate=None) == nat.GS_ERR_INVALID_ARGUMENT
    assert forward(problem(), kept=None) == nat.GS_ERR_INVALID_ARGUMENT
    assert forward(problem(), s=(ctypes.c_int64 * 18)(*[63] * 18)) == nat.GS_ERR_INVALID_ARGUMENT
    need = lib.gs_delta_scan_workspace_bytes(problem())
    assert need > 0 and forward(problem(), bytes_=need - 1) == nat.GS_ERR_WORKSPACE
    assert forward(problem(t=0), q=None) == nat.GS_OK
    assert lib.gs_delta_scan_kept_bytes(problem(), 1) > lib.gs_delta_scan_kept_bytes(problem(), 0) > 0

    def backward(p, bytes_=1 << 30, dq=FAKE, grad=None):
        return lib.gs_delta_scan_bwd(p, FAKE, FAKE, FAKE, FAKE, FAKE, grad, strides, None, None, FAKE, dq, FAKE,
                                     FAKE, FAKE, FAKE, None, FAKE, bytes_, None)

    need = lib.gs_delta_scan_bwd_workspace_bytes(problem())
    assert need > 0 and backward(problem(), need - 1) == nat.GS_ERR_WORKSPACE
    assert backward(problem(), dq=None) == nat.GS_ERR_INVALID_ARGUMENT
    assert backward(problem(), dq=ctypes.c_void_p(264)) == nat.GS_ERR_INVALID_ARGUMENT
    assert backward(problem(), grad=ctypes.c_void_p(264)) == nat.GS_ERR_INVALID_ARGUMENT
    assert lib.gs_delta_scan_step(problem(), FAKE, FAKE, FAKE, FAKE, FAKE, None, FAKE, FAKE,
                                  None) == nat.GS_ERR_INVALID_ARGUMENT
    assert lib.gs_delta_scan_step(problem(), FAKE, FAKE, FAKE, FAKE, FAKE, ctypes.c_void_p(264), FAKE, FAKE,
                                  None) == nat.GS_ERR_INVALID_ARGUMENT
    assert lib.gs_delta_scan_step(problem(b=0), None, None, None, None, None, None, None, None, None) == nat.GS_OK


def test_only_a_backward_keeps_triangles(monkeypatch):
    """What the forward keeps goes by whether a gradient can come: not under no_grad or
    inference_mode, even of inputs that require one."""
    from gaussian_splats_hip.sequence import delta

    asked = []

    def forward(q, k, v, gate, beta, state, scale, lengths, backward):
        asked.append(backward)
        return torch.zeros_like(v), torch.zeros(1, 2, 8, 8), torch.zeros(0)

    monkeypatch.setattr(delta, "delta_scan_forward", forward)
    inputs = [torch.zeros(1, 3, 1, 8), torch.zeros(1, 3, 1, 8), torch.zeros(1, 3, 2, 8), torch.zeros(1, 3, 2),
              torch.zeros(1, 3, 2), torch.zeros(1, 2, 8, 8)]
    sequence.delta_scan(*inputs)
    for i in range(6):
        leaves = [t.clone().requires_grad_(j == i) for j, t in enumerate(inputs)]
        out, last = sequence.delta_scan(*leaves)
        assert out.requires_grad and last.requires_grad
        with torch.no_grad():
            out, last = sequence.delta_scan(*leaves)
        assert not out.requires_grad and not last.requires_grad
        with torch.inference_mode():
            sequence.delta_scan(*leaves)
    assert asked == [False] + [True, False, False] * 6
