"""Choices of a splat predictor: what is refused, and what the default keeps."""

from __future__ import annotations

import pytest
import torch

from gaussian_splats_hip.sequence import QuantWindowCache, WindowCache
from gaussian_splats_hip.sequence import predictor
from gaussian_splats_hip.sequence.predictor import SplatPredictor


def test_refusals():
    with pytest.raises(ValueError, match="mixer"):
        SplatPredictor(mixer="mean")
    for kv_heads in (0, 3):
        with pytest.raises(ValueError, match="key heads"):
            SplatPredictor(kv_heads=kv_heads)
    with pytest.raises(ValueError, match="cache_bits"):
        SplatPredictor().start(cache_bits=8)
    with pytest.raises(NotImplementedError, match="multiple of 32"):
        SplatPredictor(width=64, heads=4).start(cache_bits=4)


@pytest.mark.parametrize("mixer,shape", [("gated", (3, 256)), ("delta", (3, 4, 64, 64))])
def test_states(mixer, shape):
    model = SplatPredictor(mixer=mixer)
    for bits, kind in ((16, WindowCache), (4, QuantWindowCache)):
        states = model.start(3, cache_bits=bits)
        assert len(states) == 2
        for state, cache in states:
            assert state.shape == shape and state.dtype == torch.float32
            assert type(cache) is kind


def test_default_parameters_are_the_gated_ones():
    names = [n for n, _ in SplatPredictor().named_parameters()]
    assert names == [n for n, _ in SplatPredictor(mixer="delta").named_parameters()]
    block = SplatPredictor().blocks[0]
    assert block.scan_in.weight.shape == (512, 256)
    assert torch.equal(block.scan_in.bias[256:], torch.linspace(1.0, 8.0, 256).to(torch.bfloat16))


@pytest.mark.parametrize("bits", [4, 16])
@pytest.mark.parametrize("mixer", ["gated", "delta"])
def test_a_refused_prefill_changes_nothing(mixer, bits, monkeypatch):
    """One sequence into the states of several streams, or into another model's state:
    neither states nor caches are touched.  The refusals come before any kernel, so
    stand-ins do for those ahead of them."""
    monkeypatch.setattr(predictor, "add_rms_norm", lambda x, stream, weight: (x, stream))
    monkeypatch.setattr(predictor, "gated_scan", lambda value, gate: (value, value[:, -1].float()))
    monkeypatch.setattr(predictor, "delta_scan", lambda q, k, v, gate, beta, scale: (
        v, torch.ones(1, v.shape[2], q.shape[3], v.shape[3])))
    model = SplatPredictor(mixer=mixer, dtype=torch.float32)
    tokens, rays = torch.ones(5, 774), torch.ones(5, 6)

    def touched(states):
        return any(t.any() for state, cache in states
                   for t in (state, cache.positions, *(cache._tensors() if bits == 4 else (cache.k, cache.v))))

    several = model.start(3, cache_bits=bits)
    with pytest.raises(ValueError):
        model.prefill(tokens, rays, several)
    assert not touched(several)
    # A state that the sequence's would be spread over, beside a cache that fits.
    wide = [(torch.zeros(3, *state.shape[1:]), cache) for state, cache in model.start(1, cache_bits=bits)]
    with pytest.raises(ValueError, match="state"):
        model.prefill(tokens, rays, wide)
    assert not touched(wide)
