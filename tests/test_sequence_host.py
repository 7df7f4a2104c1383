"""Refusals of the sequence operators: the Python entry points and the C ABI
turn arguments away on the host, before any launch."""

from __future__ import annotations

import ctypes

import pytest
import torch

from gaussian_splats_hip import sequence
from gaussian_splats_hip.kernels.rasterize import _native as nat

FAKE = ctypes.c_void_p(256)
NULL = ctypes.c_void_p(0)


def test_cpu_tensors_are_rejected():
    x, w = torch.zeros(2, 8), torch.ones(8)
    q = torch.zeros(1, 4, 2, 8)
    for call in (lambda: sequence.add_rms_norm(x, x, w),
                 lambda: sequence.add_rms_norm_quant(x, None, w),
                 lambda: sequence.gated_scan(x[None], x[None]),
                 lambda: sequence.gated_scan_step(x, x, x),
                 lambda: sequence.window_attention(q, q, q, 2),
                 lambda: sequence.window_attention_step(
                     q[:, 0], q[:, 0], q[:, 0], q, q, torch.zeros(1, dtype=torch.int32), 4)):
        with pytest.raises(ValueError, match="ROCm GPU"):
            call()


def test_norm_refuses():
    x, w = torch.zeros(2, 8), torch.ones(8)
    with pytest.raises(TypeError, match="float64"):
        sequence.add_rms_norm(x.double(), None, w)
    with pytest.raises(TypeError, match="weight is torch.float16"):
        sequence.add_rms_norm(x, None, w.half())
    with pytest.raises(TypeError, match="residual is torch.float16"):
        sequence.add_rms_norm(x.bfloat16(), x.half(), w)
    with pytest.raises(ValueError, match="does not fit rows"):
        sequence.add_rms_norm(x, None, torch.ones(7))
    with pytest.raises(ValueError, match="differ"):
        sequence.add_rms_norm(x, x[:1], w)
    with pytest.raises(ValueError, match="eps"):
        sequence.add_rms_norm(x, None, w, float("nan"))
    with pytest.raises(ValueError, match="last dimension"):
        sequence.add_rms_norm(torch.zeros(3, 0), None, torch.ones(0))
    with pytest.raises(ValueError, match="format"):
        sequence.add_rms_norm_quant(x, None, w, format="int4")


def test_scan_refuses():
    x = torch.zeros(2, 5, 8)
    with pytest.raises(TypeError, match="gate is"):
        sequence.gated_scan(x, x.half())
    with pytest.raises(TypeError, match="int32"):
        sequence.gated_scan(x.int(), x.int())
    with pytest.raises(ValueError, match="equal dimensions"):
        sequence.gated_scan(x, x[:, :4])
    with pytest.raises(ValueError, match="equal dimensions"):
        sequence.gated_scan(x[0], x[0])
    with pytest.raises(TypeError, match="state is"):
        sequence.gated_scan(x, x, torch.zeros(2, 8).half())
    with pytest.raises(ValueError, match="does not fit"):
        sequence.gated_scan(x, x, torch.zeros(2, 7))


def test_attention_refuses():
    q, k = torch.zeros(2, 5, 4, 16), torch.zeros(2, 7, 2, 16)
    with pytest.raises(TypeError, match="k is"):
        sequence.window_attention(q, k.half(), k.half(), 3)
    with pytest.raises(TypeError, match="float64"):
        sequence.window_attention(q.double(), k.double(), k.double(), 3)
    with pytest.raises(ValueError, match="expects q"):
        sequence.window_attention(q, k, k[:, :6], 3)
    with pytest.raises(ValueError, match="does not fit q"):
        sequence.window_attention(q, k[:1], k[:1], 3)
    with pytest.raises(ValueError, match="cannot share"):
        sequence.window_attention(q[:, :, :3], k, k, 3)
    for window, sinks in ((0, 1), (-1, 0), (3, -1)):
        with pytest.raises(ValueError, match="window must be positive"):
            sequence.window_attention(q, k, k, window, sinks)
    for scale in (0.0, -1.0, float("inf"), float("nan")):
        with pytest.raises(ValueError, match="scale"):
            sequence.window_attention(q, k, k, 3, scale=scale)
    with pytest.raises(TypeError, match="lengths is"):
        sequence.window_attention(q, k, k, 3, lengths=torch.zeros(2, dtype=torch.int64))
    with pytest.raises(ValueError, match="batch of 2"):
        sequence.window_attention(q, k, k, 3, lengths=torch.zeros(3, dtype=torch.int32))


def test_step_refuses():
    q, k = torch.zeros(2, 4, 16), torch.zeros(2, 2, 16)
    cache, at = torch.zeros(2, 9, 2, 16), torch.zeros(2, dtype=torch.int32)
    step = sequence.window_attention_step
    with pytest.raises(ValueError, match="caches"):
        step(q, k, k, cache, cache, at, 9, 1)
    with pytest.raises(ValueError, match="caches"):
        step(q, k, k, cache, cache[:, :8], at, 8, 1)
    with pytest.raises(TypeError, match="positions is"):
        step(q, k, k, cache, cache, at.long(), 8, 1)
    with pytest.raises(ValueError, match="batch of 2"):
        step(q, k, k, cache, cache, at[:1], 8, 1)
    with pytest.raises(TypeError, match="k_cache is"):
        step(q, k, k, cache.half(), cache, at, 8, 1)
    with pytest.raises(ValueError, match="expects q"):
        step(q, k[:, :, :8], k[:, :, :8], cache, cache, at, 8, 1)


def test_norm_c_abi_checks():
    lib = nat.library()
    args = [FAKE, FAKE, FAKE, 4, 8, 8, 8, 2, 2, 2, 1e-6]

    def fwd(**change):
        a = list(args)
        for i, v in change.items():
            a[int(i[1:])] = v
        return lib.gs_add_rms_norm_fwd(*a, FAKE, FAKE, FAKE, NULL)

    assert fwd(_3=-1) == nat.GS_ERR_INVALID_ARGUMENT
    assert fwd(_4=0) == nat.GS_ERR_INVALID_ARGUMENT
    assert fwd(_3=1 << 31) == nat.GS_ERR_OVERFLOW
    assert fwd(_7=5) == nat.GS_ERR_INVALID_ARGUMENT
    assert fwd(_8=1) == nat.GS_ERR_UNSUPPORTED and b"residual" in lib.gs_last_error()
    assert fwd(_9=1) == nat.GS_ERR_UNSUPPORTED and b"weight" in lib.gs_last_error()
    assert fwd(_0=None) == nat.GS_ERR_INVALID_ARGUMENT
    assert fwd(_3=0, _0=None) == nat.GS_OK
    assert lib.gs_add_rms_norm_quant(*args, 2, FAKE, FAKE, FAKE, NULL) == nat.GS_ERR_INVALID_ARGUMENT
    ws = lib.gs_add_rms_norm_bwd_workspace_bytes(1000, 64)
    assert ws >= 64 * 4
    assert lib.gs_add_rms_norm_bwd_workspace_bytes(-1, 64) == 0
    assert lib.gs_add_rms_norm_bwd(FAKE, FAKE, FAKE, FAKE, FAKE, 1000, 64, 64, 2, 2, 2, FAKE, NULL, FAKE,
                                   FAKE, ws - 1, NULL) == nat.GS_ERR_WORKSPACE


def test_scan_c_abi_checks():
    lib = nat.library()
    strides = (ctypes.c_int64 * 6)(*[8] * 6)
    assert lib.gs_gated_scan_chunks(0) == 0 and lib.gs_gated_scan_chunks(1) == 1
    assert lib.gs_gated_scan_workspace_bytes(1, 1, 8, 0) == 0  # a single chunk needs none
    ws = lib.gs_gated_scan_workspace_bytes(2, 1000, 8, 1)
    assert ws > lib.gs_gated_scan_workspace_bytes(2, 1000, 8, 0) > 0

    def fwd(b=2, t=1000, c=8, kind=0, x=FAKE, bytes_=ws):
        return lib.gs_gated_scan_fwd(x, FAKE, NULL, b, t, c, strides, kind, FAKE, FAKE, FAKE, FAKE, bytes_, NULL)

    assert fwd(b=-1) == nat.GS_ERR_INVALID_ARGUMENT
    assert fwd(kind=3) == nat.GS_ERR_INVALID_ARGUMENT
    assert fwd(x=None) == nat.GS_ERR_INVALID_ARGUMENT
    assert fwd(bytes_=8) == nat.GS_ERR_WORKSPACE
    assert fwd(b=1 << 16) == nat.GS_ERR_OVERFLOW
    assert fwd(t=0) == nat.GS_OK and fwd(b=0) == nat.GS_OK
    assert lib.gs_gated_scan_bwd(FAKE, FAKE, NULL, FAKE, FAKE, 2, 1000, 8, strides, 0, FAKE, FAKE, FAKE, FAKE,
                                 ws, NULL) == nat.GS_ERR_INVALID_ARGUMENT
    assert lib.gs_gated_scan_step(FAKE, FAKE, FAKE, 2, -1, 0, FAKE, FAKE, NULL) == nat.GS_ERR_INVALID_ARGUMENT
    assert lib.gs_gated_scan_step(NULL, FAKE, FAKE, 2, 4, 0, FAKE, FAKE, NULL) == nat.GS_ERR_INVALID_ARGUMENT


def _attention(**change):
    fields = dict(batch=2, queries=64, keys=64, window=16, sinks=2, heads=4, kv_heads=2, head_dim=64,
                  type=2, scale=0.125)
    fields.update(change)
    return nat.GsAttention(*fields.values())


def test_attention_c_abi_checks():
    lib = nat.library()
    strides = (ctypes.c_int64 * 12)(*[64] * 12)

    def fwd(q=FAKE, strides=strides, **change):
        return lib.gs_window_attention_fwd(ctypes.byref(_attention(**change)), q, FAKE, FAKE, strides, NULL,
                                           FAKE, FAKE, NULL)

    for bad in (dict(heads=3), dict(window=0), dict(sinks=-1), dict(scale=0.0), dict(type=4),
                dict(batch=-1), dict(kv_heads=0), dict(head_dim=0)):
        assert fwd(**bad) == nat.GS_ERR_INVALID_ARGUMENT, bad
    for dim in (4, 36, 136):
        assert fwd(head_dim=dim) == nat.GS_ERR_UNSUPPORTED and b"head_dim" in lib.gs_last_error()
    assert fwd(keys=1 << 30) == nat.GS_ERR_OVERFLOW
    assert fwd(q=None) == nat.GS_ERR_INVALID_ARGUMENT
    assert fwd(q=ctypes.c_void_p(8)) == nat.GS_ERR_INVALID_ARGUMENT
    odd = (ctypes.c_int64 * 12)(*[65] * 12)
    assert fwd(strides=odd) == nat.GS_ERR_INVALID_ARGUMENT and b"16-byte" in lib.gs_last_error()
    far = (ctypes.c_int64 * 12)(*[1 << 24] * 12)
    assert fwd(strides=far) == nat.GS_ERR_OVERFLOW and b"far apart" in lib.gs_last_error()
    assert fwd(batch=0) == nat.GS_OK and fwd(queries=0) == nat.GS_OK
    d = _attention()
    ws = lib.gs_window_attention_bwd_workspace_bytes(ctypes.byref(d))
    assert ws >= 2 * 4 * 64 * 4
    assert lib.gs_window_attention_bwd_workspace_bytes(ctypes.byref(_attention(heads=3))) == 0
    assert lib.gs_window_attention_bwd(ctypes.byref(d), FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, strides, NULL,
                                       FAKE, FAKE, FAKE, FAKE, ws - 1, NULL) == nat.GS_ERR_WORKSPACE
    d = _attention(window=1 << 12)
    ws = lib.gs_window_attention_step_workspace_bytes(ctypes.byref(d))
    assert ws > 0
    assert lib.gs_window_attention_step(ctypes.byref(d), FAKE, FAKE, FAKE, FAKE, FAKE, strides, FAKE, FAKE,
                                        FAKE, ws - 1, NULL) == nat.GS_ERR_WORKSPACE
    assert lib.gs_window_attention_step(ctypes.byref(d), FAKE, FAKE, FAKE, FAKE, FAKE, strides, NULL, FAKE,
                                        FAKE, ws, NULL) == nat.GS_ERR_INVALID_ARGUMENT


def test_predictor_refuses_widths_without_heads():
    from gaussian_splats_hip.sequence.predictor import SplatPredictor

    with pytest.raises(ValueError, match="multiple of 8"):
        SplatPredictor(width=100, heads=4)


def test_first_tokens_workspace_is_bounded():
    """Parts of the first tokens' walks: a few megabytes for long sequences."""
    lib = nat.library()
    d = _attention(batch=1, queries=40000, keys=40000, window=5000, sinks=16, heads=12, kv_heads=4)
    delta = 12 * 40000 * 4
    parts = lib.gs_window_attention_bwd_workspace_bytes(ctypes.byref(d)) - delta
    assert 0 < parts <= 64 << 20


@pytest.mark.parametrize("tokens,window,sinks,heads,kv_heads,dim", [
    (40000, 64, 2500, 12, 4, 64), (40000, 300, 1200, 16, 16, 128), (40000, 16, 40000, 12, 4, 64),
    (16320, 8160, 8160, 16, 4, 128), (160000, 300, 1200, 8, 8, 64)])
def test_workspace_of_many_first_tokens_is_bounded(tokens, window, sinks, heads, kv_heads, dim):
    """First tokens that are a whole view: parts for at most 1536 workgroups (1024
    on the first tokens, 512 on the others), each two float32 tiles of 128 keys."""
    lib = nat.library()
    d = _attention(batch=1, queries=tokens, keys=tokens, window=window, sinks=sinks, heads=heads,
                   kv_heads=kv_heads, head_dim=dim)
    delta = heads * tokens * 4 + 4096
    assert lib.gs_window_attention_bwd_workspace_bytes(ctypes.byref(d)) <= delta + 1536 * 2 * 128 * dim * 4


def test_norm_backward_refuses():
    """What the kernels would read beyond: a shorter weight or inverse, one of
    another type."""
    s, w, r = torch.zeros(2, 3, 8), torch.ones(8), torch.ones(6)
    back = sequence.add_rms_norm_backward
    with pytest.raises(ValueError, match="weight .* does not fit rows"):
        back(s, w[:7], r, s, None, torch.float32)
    with pytest.raises(TypeError, match="weight is torch.float16"):
        back(s, w.half(), r, s, None, torch.float32)
    with pytest.raises(TypeError, match="inverse is torch.bfloat16"):
        back(s, w, r.bfloat16(), s, None, torch.float32)
    for bad in (r[:5], r[:1], torch.ones(7), torch.ones(())):
        with pytest.raises(ValueError, match="inverse .* rows of"):
            back(s, w, bad, s, None, torch.float32)
    with pytest.raises(TypeError, match="total is torch.float16"):
        back(s.half(), w.bfloat16(), r, s.bfloat16(), None, torch.bfloat16)
    with pytest.raises(TypeError, match="float64"):
        back(s, w, r, None, None, torch.float64)
    with pytest.raises(ValueError, match="gradient"):
        back(s, w, r, s[:1], None, torch.float32)
    for good in (r, r.view(2, 3)):
        with pytest.raises(ValueError, match="ROCm GPU"):
            back(s, w, good, s, None, torch.float32)


def test_scan_backward_refuses():
    x, starts = torch.zeros(2, 5, 8), torch.zeros(2, 1, 8)
    back = sequence.gated_scan_backward
    with pytest.raises(TypeError, match="starts is torch.bfloat16"):
        back(x, x, starts.bfloat16(), x, None)
    for bad in (starts[:1], starts[:, :, :7], torch.zeros(2, 2, 8), starts.expand(2, 1, 8)[:, :0]):
        with pytest.raises(ValueError, match="starts .* are not those"):
            back(x, x, bad, x, None)
    with pytest.raises(ValueError, match="grad_y"):
        back(x, x, starts, x[:1], None)
    with pytest.raises(ValueError, match="grad_last"):
        back(x, x, starts, x, torch.zeros(2, 8).half())
    with pytest.raises(ValueError, match="ROCm GPU"):
        back(x, x, starts, x, torch.zeros(2, 8))


def test_step_refuses_caches_beyond_its_counters():
    lib = nat.library()
    strides = (ctypes.c_int64 * 6)(*[64] * 6)
    for window, sinks in ((1 << 30, 0), ((1 << 30) - 1, 1), ((1 << 30) - 1, (1 << 30) - 1), (1, (1 << 63) - 1)):
        d = _attention(window=window, sinks=sinks)
        # Without positions: a call that the sizes do not turn away ends there.
        assert lib.gs_window_attention_step(ctypes.byref(d), FAKE, FAKE, FAKE, FAKE, FAKE, strides, NULL, FAKE,
                                            FAKE, 1 << 40, NULL) == nat.GS_ERR_OVERFLOW, (window, sinks)


def test_attention_refuses_more_workgroups_than_a_launch_holds():
    """2^24 workgroups of 256 threads; without buffers, so that a call that the
    sizes do not turn away ends at its pointers."""
    lib = nat.library()
    strides = (ctypes.c_int64 * 12)(*[64] * 12)
    d = ctypes.byref(_attention(batch=65535, queries=1024, keys=1024, heads=64, kv_heads=1, window=2, sinks=0))
    assert lib.gs_window_attention_fwd(d, NULL, NULL, NULL, strides, NULL, NULL, NULL, NULL) == nat.GS_ERR_OVERFLOW
    assert lib.gs_window_attention_bwd(d, NULL, NULL, NULL, NULL, NULL, NULL, strides, NULL, NULL, NULL, NULL, NULL,
                                       1 << 50, NULL) == nat.GS_ERR_OVERFLOW


def test_step_refuses_expanded_caches():
    """Streams that share their memory would write to it at once."""
    q, k = torch.zeros(2, 4, 16), torch.zeros(2, 2, 16)
    cache, at = torch.zeros(2, 9, 2, 16), torch.zeros(2, dtype=torch.int32)
    for bad in (cache[:1].expand(2, -1, -1, -1), cache[:, :1].expand(-1, 9, -1, -1), cache[:, :, :1].expand(-1, -1, 2, -1)):
        with pytest.raises(ValueError, match="k_cache is expanded"):
            sequence.window_attention_step(q, k, k, bad, cache, at, 8, 1)
        with pytest.raises(ValueError, match="v_cache is expanded"):
            sequence.window_attention_step(q, k, k, cache, bad, at, 8, 1)
    one = cache[:1].expand(1, -1, -1, -1).as_strided((1, 9, 2, 16), (0, 32, 16, 1))
    with pytest.raises(ValueError, match="ROCm GPU"):
        sequence.window_attention_step(q[:1], k[:1], k[:1], one, one, at[:1], 8, 1)
