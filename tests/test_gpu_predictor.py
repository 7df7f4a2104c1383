"""The example that runs the sequence operators together: it learns, and a
stream taken token by token gives the splats that the whole one gives."""

from __future__ import annotations

import pytest
import torch

from gaussian_splats_hip.sequence import predictor
from gaussian_splats_hip.splats import rasterize

pytestmark = pytest.mark.gpu


def test_predictor_learns_and_streams():
    model, tokens, rays, losses = predictor.train(steps=40, views=3, size=96, log=lambda *_: None)
    assert losses[-1] < 0.6 * losses[0]
    for p in model.parameters():
        assert p.grad is not None and torch.isfinite(p.grad).all()
    with torch.no_grad():
        whole = model(tokens, rays)
    streamed = predictor.stream(model, tokens, rays)
    assert set(whole) == set(streamed)
    cameras, _ = predictor._views(torch.device("cuda"), 1, 96, 0)
    with torch.no_grad():
        a, b = (rasterize(predictor.splats_of(p), cameras[0], tile_size=16) for p in (whole, streamed))
    # The two forms round bfloat16 products of other shapes differently; the
    # images differ by a few of its roundings of values up to one.
    assert float((a - b).abs().mean()) < 4 * 2.0**-8


def test_float32_stream_is_exact_to_rounding():
    torch.manual_seed(1)
    model = predictor.SplatPredictor(width=64, heads=2, kv_heads=1, blocks=2, window=20, sinks=2,
                                     dtype=torch.float32).to("cuda")
    tokens, rays = torch.randn(70, 774, device="cuda"), torch.randn(70, 6, device="cuda")
    with torch.no_grad():
        whole = model(tokens, rays)
    streamed = predictor.stream(model, tokens, rays)
    for name in whole:
        # Some hundred float32 operations deep.
        torch.testing.assert_close(streamed[name], whole[name], rtol=1e-4, atol=1e-4)
