"""The 4-bit cache without a GPU: the oracle's encoding, and what the entry points
turn away on the host."""

from __future__ import annotations

import ctypes

import pytest
import torch

from gaussian_splats_hip import sequence
from gaussian_splats_hip.kernels.rasterize import _native as nat
from oracle import sequence as orc

FAKE = ctypes.c_void_p(256)


def test_oracle_encoding():
    """Values that codes hold come back; others go to the nearest, ties to the even
    code, beyond six to six."""
    values = torch.tensor(orc.MXFP4_VALUES + (5.5,) * 24, dtype=torch.float64)
    codes, exponents = orc.mxfp4_encode(values * 2.0**-7)
    assert exponents.tolist() == [127 - 7]
    assert torch.equal(orc.mxfp4_decode(codes, exponents)[:8], values[:8] * 2.0**-7)
    assert torch.equal(orc.mxfp4_decode(codes, exponents)[8:], torch.full((24,), 6.0 * 2.0**-7).double())
    ties = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.9] + [0.0] * 24)
    codes, exponents = orc.mxfp4_encode(ties)
    assert orc.mxfp4_decode(codes, exponents)[:8].tolist() == [0.0, 1.0, 1.0, 2.0, 2.0, 4.0, 4.0, 6.0]
    x = torch.randn(50, 64, generator=torch.Generator().manual_seed(1)).double()
    back = orc.mxfp4_decode(*orc.mxfp4_encode(x))
    # A step of two powers at most below six, two from there to eight.
    power = torch.exp2(torch.floor(torch.log2(x.abs().unflatten(-1, (2, 32)).amax(-1))) - 2)
    assert ((x - back).abs().unflatten(-1, (2, 32)) <= 2 * power[..., None]).all()
    assert not orc.mxfp4_decode(*orc.mxfp4_encode(torch.zeros(32))).any()
    x[0, 40] = float("inf")
    back = orc.mxfp4_decode(*orc.mxfp4_encode(x))
    assert back[0, 32:].isnan().all() and back[0, :32].isfinite().all() and back[1:].isfinite().all()


def _caches(b=2, hk=2, n=9, d=64):
    codes = [torch.zeros(b, hk, n, d // 2, dtype=torch.uint8) for _ in range(2)]
    exponents = [torch.zeros(b, hk, n, d // 32, dtype=torch.uint8) for _ in range(2)]
    return [codes[0], exponents[0], codes[1], exponents[1]]


def test_step_refuses():
    q, k, at = torch.zeros(2, 4, 64), torch.zeros(2, 2, 64), torch.zeros(2, dtype=torch.int32)
    step = sequence.window_attention_step_quant

    def swapped(i, t):
        c = _caches()
        c[i] = t
        return c

    with pytest.raises(ValueError, match="ROCm GPU"):
        step(q, k, k, *_caches(), at, 8, 1)
    with pytest.raises(ValueError, match="k_codes"):
        step(q, k, k, *_caches(), at, 9, 1)
    with pytest.raises(TypeError, match="v_codes is torch.int8"):
        step(q, k, k, *swapped(2, torch.zeros(2, 2, 9, 32, dtype=torch.int8)), at, 8, 1)
    with pytest.raises(ValueError, match="k_exponents"):
        step(q, k, k, *swapped(1, torch.zeros(2, 2, 9, 1, dtype=torch.uint8)), at, 8, 1)
    with pytest.raises(ValueError, match="contiguous"):
        step(q, k, k, *swapped(0, torch.zeros(2, 9, 2, 32, dtype=torch.uint8).transpose(1, 2)), at, 8, 1)
    with pytest.raises(ValueError, match="contiguous"):
        step(q, k, k, *swapped(0, torch.zeros(1, 2, 9, 32, dtype=torch.uint8).expand(2, -1, -1, -1)), at, 8, 1)
    with pytest.raises(ValueError, match="16-byte"):
        step(q, k, k, *swapped(0, torch.zeros(2 * 2 * 9 * 32 + 16, dtype=torch.uint8)[1:-15].view(2, 2, 9, 32)),
             at, 8, 1)
    with pytest.raises(TypeError, match="positions is"):
        step(q, k, k, *_caches(), at.long(), 8, 1)
    with pytest.raises(ValueError, match="batch of 2"):
        step(q, k, k, *_caches(), at[:1], 8, 1)
    with pytest.raises(TypeError, match="k is"):
        step(q, k.half(), k.half(), *_caches(), at, 8, 1)
    with pytest.raises(ValueError, match="cannot share"):
        step(q[:, :3], k, k, *_caches(), at, 8, 1)
    with pytest.raises(ValueError, match="window must be positive"):
        step(q, k, k, *_caches(), at, 0, 9)
    with pytest.raises(ValueError, match="scale"):
        step(q, k, k, *_caches(), at, 8, 1, scale=0.0)
    for d in (8, 40, 160):
        with pytest.raises(NotImplementedError, match="4 bits"):
            step(torch.zeros(2, 4, d), torch.zeros(2, 2, d), torch.zeros(2, 2, d), *_caches(), at, 8, 1)


def test_fill_refuses():
    k = torch.zeros(2, 5, 2, 64)
    fill = sequence.window_cache_fill_quant
    with pytest.raises(ValueError, match="ROCm GPU"):
        fill(k, k, *_caches(), 8, 1)
    with pytest.raises(ValueError, match="expects k and v"):
        fill(k, k[:, :4], *_caches(), 8, 1)
    with pytest.raises(ValueError, match="k_codes"):
        fill(k[:1], k[:1], *_caches(), 8, 1)
    with pytest.raises(TypeError, match="lengths is"):
        fill(k, k, *_caches(), 8, 1, torch.zeros(2, dtype=torch.int64))
    with pytest.raises(ValueError, match="batch of 2"):
        fill(k, k, *_caches(), 8, 1, torch.zeros(3, dtype=torch.int32))
    with pytest.raises(TypeError, match="float64"):
        fill(k.double(), k.double(), *_caches(), 8, 1)
    with pytest.raises(NotImplementedError, match="4 bits"):
        sequence.QuantWindowCache(1, 1, 48, 8, device="cpu")
    with pytest.raises(ValueError, match="window must be positive"):
        sequence.QuantWindowCache(1, 1, 64, 0, device="cpu")


def test_c_abi_checks():
    lib = nat.library()

    def problem(b=1, keys=4, window=8, sinks=1, h=2, hk=1, d=64, kind=2):
        return ctypes.byref(nat.GsAttention(b, 1, keys, window, sinks, h, hk, d, kind, 0.1))

    def step(p, codes=FAKE, ws_bytes=1 << 30, q=FAKE):
        return lib.gs_window_attention_step_quant(p, q, FAKE, FAKE, codes, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE,
                                                  ws_bytes, None)

    assert step(None) == nat.GS_ERR_INVALID_ARGUMENT
    assert step(problem(d=40)) == nat.GS_ERR_UNSUPPORTED and b"4 bits" in lib.gs_last_error()
    assert step(problem(window=1 << 30)) == nat.GS_ERR_OVERFLOW
    assert step(problem(), codes=None) == nat.GS_ERR_INVALID_ARGUMENT
    assert step(problem(), codes=ctypes.c_void_p(264)) == nat.GS_ERR_INVALID_ARGUMENT
    assert step(problem(), q=ctypes.c_void_p(264)) == nat.GS_ERR_INVALID_ARGUMENT
    assert step(problem(b=0), codes=None) == nat.GS_OK
    big = problem(window=100_000)
    need = lib.gs_window_attention_step_quant_workspace_bytes(big)
    assert need > 0 and step(big, ws_bytes=need - 1) == nat.GS_ERR_WORKSPACE

    strides = (ctypes.c_int64 * 6)(*[64] * 6)

    def fill(p, k=FAKE, codes=FAKE, s=strides):
        return lib.gs_window_cache_fill_quant(p, k, FAKE, s, None, codes, FAKE, FAKE, FAKE, None)

    assert fill(problem(d=40)) == nat.GS_ERR_UNSUPPORTED
    assert fill(problem(), codes=None) == nat.GS_ERR_INVALID_ARGUMENT
    assert fill(problem(), k=None) == nat.GS_ERR_INVALID_ARGUMENT
    assert fill(problem(), s=(ctypes.c_int64 * 6)(*[63] * 6)) == nat.GS_ERR_INVALID_ARGUMENT
    assert fill(problem(keys=0), k=None) == nat.GS_OK
