"""Refusals of the gradient norm, the clipping and FusedAdam's limit: the Python
entry points and the C ABI turn arguments away on the host."""

from __future__ import annotations

import copy
import ctypes
import pickle

import pytest
import torch

from gaussian_splats_hip.kernels.rasterize import _native as nat
from gaussian_splats_hip.training import FusedAdam, clip_grad_norm, grad_norm

FAKE = ctypes.c_void_p(256)


def _with_grad(grad, shape=None):
    p = torch.nn.Parameter(torch.zeros(shape or grad.shape, dtype=grad.dtype))
    p.grad = grad
    return p


def test_refusals():
    with pytest.raises(ValueError, match="ROCm GPU"):
        grad_norm([torch.zeros(3)])
    with pytest.raises(ValueError, match="ROCm GPU"):
        clip_grad_norm([_with_grad(torch.zeros(3))], 1.0)
    with pytest.raises(TypeError, match="float64"):
        grad_norm(torch.zeros(3, dtype=torch.float64))
    with pytest.raises(TypeError, match="dense"):
        grad_norm([torch.zeros(3, 3).to_sparse()])
    for bad in (-1.0, float("nan")):
        with pytest.raises(ValueError, match="max_norm"):
            clip_grad_norm([], bad)
        with pytest.raises(ValueError, match="max_norm"):
            FusedAdam([torch.nn.Parameter(torch.zeros(3))], max_norm=bad)


def test_nothing_to_do():
    assert float(grad_norm([])) == 0.0
    assert float(clip_grad_norm([], 1.0)) == 0.0
    assert float(clip_grad_norm([torch.nn.Parameter(torch.zeros(3))], 1.0)) == 0.0


def test_limit_survives_copies():
    opt = FusedAdam([torch.nn.Parameter(torch.zeros(3))], max_norm=2.0)
    assert opt.max_norm == 2.0 and opt.grad_norm is None
    assert copy.deepcopy(opt).max_norm == 2.0
    assert pickle.loads(pickle.dumps(opt)).max_norm == 2.0
    assert FusedAdam([torch.nn.Parameter(torch.zeros(3))]).max_norm is None


def test_c_abi_checks():
    lib = nat.library()

    def call(entries, count=None, limit=1.0, norm=FAKE, ws=FAKE, ws_bytes=1 << 20):
        flat = [int(x) for e in entries for x in e]
        array = ctypes.cast((ctypes.c_int64 * max(len(flat), 1))(*flat), ctypes.c_void_p)
        return lib.gs_grad_norm(array, len(entries) if count is None else count, limit, 0, norm, None,
                                ws, ws_bytes, None)

    assert call([], count=-1) == nat.GS_ERR_INVALID_ARGUMENT
    assert call([(0, 5, 0)]) == nat.GS_ERR_INVALID_ARGUMENT and b"null" in lib.gs_last_error()
    assert call([(256, -1, 0)]) == nat.GS_ERR_INVALID_ARGUMENT
    assert call([(256, 5, 3)]) == nat.GS_ERR_INVALID_ARGUMENT and b"type" in lib.gs_last_error()
    assert call([(256, 5, 0)], norm=None) == nat.GS_ERR_INVALID_ARGUMENT
    assert call([(256, 5, 0)], limit=-1.0) == nat.GS_ERR_INVALID_ARGUMENT
    assert call([(256, 5, 0)], limit=float("nan")) == nat.GS_ERR_INVALID_ARGUMENT
    need = lib.gs_grad_norm_workspace_bytes(1)
    assert call([(256, 5, 0)], ws_bytes=need - 1) == nat.GS_ERR_WORKSPACE
    assert call([(256, 5, 0)], ws=None) == nat.GS_ERR_WORKSPACE
    assert lib.gs_grad_norm_workspace_bytes(129) == 2 * need
    assert lib.gs_adam_step_scaled(None, 0, 0.9, 0.999, 1e-8, 0.0, None, None) == nat.GS_ERR_INVALID_ARGUMENT


def test_no_norm_of_an_earlier_step():
    """A step without gradients, or one that is refused, leaves no older step's norm."""
    p = torch.nn.Parameter(torch.zeros(3))
    opt = FusedAdam([p], max_norm=1.0)
    opt.grad_norm = torch.tensor(5.0)
    opt.step()
    assert opt.grad_norm is None
    opt.grad_norm = torch.tensor(5.0)
    p.grad = torch.ones(3)
    with pytest.raises(TypeError, match="ROCm GPU"):
        opt.step()
    assert opt.grad_norm is None
