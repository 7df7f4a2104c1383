"""Splat predictors with the gated delta rule, trained with clipped gradients and
streamed over a cache in 4 bits: the operators as they are used together.

A splat and a gradient are some 40 operators deep (forwards and backwards), each of
whose results is off by at most n 2^-24 of the sum of its n terms' sizes, n up to 774
in the longest product: 40 * 774 * 2^-24 = 2e-3 of the result's size, of which
independent roundings reach the root.  Gradients are held to the 2e-3, in the 2-norm
of each parameter's; splats, half as deep, to 1e-4 element by element."""

from __future__ import annotations

import copy

import pytest
import torch

from gaussian_splats_hip.sequence import WindowCache, predictor
from gaussian_splats_hip.training import grad_norm
from oracle import sequence as oracle

pytestmark = pytest.mark.gpu


def _model(**sizes):
    torch.manual_seed(3)
    sizes = {"width": 64, "heads": 2, "kv_heads": 1, "blocks": 2, "window": 20, "sinks": 2, **sizes}
    return predictor.SplatPredictor(dtype=torch.float32, mixer="delta", **sizes).to("cuda")


def _tokens(count):
    torch.manual_seed(4)
    return torch.randn(count, 774, device="cuda"), torch.randn(count, 6, device="cuda")


def test_clipped_training_and_4_bit_streaming_run():
    limit = 0.05
    model, tokens, rays, losses = predictor.train(steps=6, views=2, size=64, log=lambda *_: None,
                                                  mixer="delta", max_norm=limit)
    assert all(l == l for l in losses)
    grads = [p.grad for p in model.parameters()]
    assert all(torch.isfinite(g).all() for g in grads)
    # The clipped ones are rounded to bfloat16 once more.
    assert float(grad_norm(grads)) <= limit * (1 + 2.0**-8 + 1e-5)
    with torch.no_grad():
        whole = model(tokens, rays)
    for bits, first in ((16, 0), (4, 0), (4, 20)):
        streamed = predictor.stream(model, tokens, rays, cache_bits=bits, first=first)
        for name in whole:
            assert streamed[name].shape == whole[name].shape and torch.isfinite(streamed[name]).all()


class _Delta(torch.autograd.Function):
    @staticmethod
    def forward(ctx, *inputs):
        ctx.save_for_backward(*inputs)
        return oracle.delta_scan(*inputs, scale=1.0)

    @staticmethod
    def backward(ctx, *grads):
        return oracle.delta_scan(*ctx.saved_tensors, scale=1.0, grads=grads)[2:7]


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, window, sinks):
        ctx.save_for_backward(q, k, v)
        ctx.sizes = window, sinks
        return oracle.window_attention(q, k, v, window, sinks)

    @staticmethod
    def backward(ctx, grad):
        return (*oracle.window_attention(*ctx.saved_tensors, *ctx.sizes, grad=grad)[1:], None, None)


@pytest.mark.parametrize("heads,kv_heads", [(2, 1), (4, 4)])
def test_gradients_are_those_of_64_bits(heads, kv_heads, monkeypatch):
    model = _model(heads=heads, kv_heads=kv_heads)
    tokens, rays = _tokens(70)
    splats = model(tokens, rays)
    weights = {name: torch.randn_like(t) for name, t in splats.items()}
    sum((splats[name] * w).sum() for name, w in weights.items()).backward()

    plain = copy.deepcopy(model).cpu().double()
    plain.dtype = torch.float64
    for p in plain.parameters():
        p.grad = None
    monkeypatch.setattr(predictor, "add_rms_norm", lambda x, s, w: oracle.add_rms_norm(x, s, w, 1e-6))
    monkeypatch.setattr(predictor, "window_attention", _Attention.apply)
    monkeypatch.setattr(predictor, "delta_scan", lambda *inputs, scale: _Delta.apply(*inputs))
    exact = plain(tokens.cpu(), rays.cpu())
    sum((exact[name] * w.cpu()).sum() for name, w in weights.items()).backward()
    for name, t in exact.items():
        torch.testing.assert_close(splats[name].detach().cpu(), t.detach().float(), rtol=1e-4, atol=1e-4)
    for (name, p), x in zip(model.named_parameters(), plain.parameters()):
        off = float((p.grad.cpu().double() - x.grad).norm() / x.grad.norm())
        assert off <= 2e-3, (name, off)


@pytest.mark.parametrize("first", [0, 1, 33])
def test_stream_goes_on_behind_a_prefill(first):
    model = _model()
    tokens, rays = _tokens(70)
    with torch.no_grad():
        whole = model(tokens, rays)
    streamed = predictor.stream(model, tokens, rays, first=first)
    for name in whole:
        torch.testing.assert_close(streamed[name], whole[name], rtol=1e-4, atol=1e-4)


class _Rounded(WindowCache):
    """A cache in float32 of keys and values that 4 bits can hold."""

    @staticmethod
    def _round(t):
        return oracle.mxfp4_decode(*oracle.mxfp4_encode(t.cpu())).to(t)

    def fill(self, k, v):
        super().fill(self._round(k), self._round(v))

    def step(self, q, k, v):
        return super().step(q, self._round(k), self._round(v))


@pytest.mark.parametrize("first", [0, 33])
def test_4_bit_stream_is_that_of_rounded_keys(first, monkeypatch):
    # One block: what a second one would round depends on the first's last bits.
    model = _model(blocks=1, width=128, heads=4, kv_heads=2)
    tokens, rays = _tokens(70)
    streamed = predictor.stream(model, tokens, rays, cache_bits=4, first=first)
    monkeypatch.setattr(predictor, "WindowCache", _Rounded)
    rounded = predictor.stream(model, tokens, rays, first=first)
    for name in rounded:
        torch.testing.assert_close(streamed[name], rounded[name], rtol=1e-4, atol=1e-4)


def test_captured_steps_of_all_together():
    """A step of several streams, replayed, gives what eager steps give."""
    model = _model(blocks=2, width=128, heads=4, kv_heads=2)
    tokens, rays = _tokens(60)
    batches = tokens.view(15, 4, -1), rays.view(15, 4, -1)
    eager = model.start(4, cache_bits=4)
    expected = [model.step(t, r, eager) for t, r in zip(*batches)]

    states = model.start(4, cache_bits=4)
    token, ray = batches[0][0].clone(), batches[1][0].clone()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        model.step(token, ray, model.start(4, cache_bits=4))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = model.step(token, ray, states)
    for t, r, want in zip(*batches, expected):
        token.copy_(t)
        ray.copy_(r)
        graph.replay()
        torch.cuda.synchronize()
        for name in want:
            torch.testing.assert_close(out[name], want[name], rtol=0, atol=0)


def test_training_clips_what_is_above_the_limit(monkeypatch):
    """A limit of half the first step's norm, as a run without one has it: training
    passes every step's gradients to the clipping, which brings the first ones down."""
    seen = []
    clip = predictor.clip_grad_norm

    def recorded(parameters, limit):
        parameters = list(parameters)
        norm = clip(parameters, limit)
        seen.append((float(norm), float(grad_norm([p.grad for p in parameters]))))
        return norm

    monkeypatch.setattr(predictor, "clip_grad_norm", recorded)
    sizes = {"views": 2, "size": 64, "log": lambda *_: None, "mixer": "delta"}
    predictor.train(steps=1, max_norm=float("inf"), **sizes)
    (first, kept), = seen
    assert first > 0.0 and kept == first
    limit = first / 2
    seen.clear()
    predictor.train(steps=3, max_norm=limit, **sizes)
    assert len(seen) == 3 and seen[0][0] > limit
    for before, after in seen:
        # The clipped ones are rounded to bfloat16 once more.
        want = min(before, limit)
        assert abs(after - want) <= want * (2.0**-8 + 1e-5)


def test_a_prefill_of_a_single_stream_only():
    """States of several streams refuse one's tokens and go on as if nothing had been asked."""
    tokens, rays = _tokens(12)
    for mixer, bits in (("gated", 16), ("delta", 16), ("delta", 4)):
        torch.manual_seed(3)
        model = predictor.SplatPredictor(width=128, heads=4, kv_heads=2, window=20, sinks=2, dtype=torch.float32,
                                         mixer=mixer).to("cuda")
        asked, other = model.start(4, cache_bits=bits), model.start(4, cache_bits=bits)
        for states in (asked, other):
            model.step(tokens[:4], rays[:4], states)
        with pytest.raises(ValueError):
            model.prefill(tokens, rays, asked)
        a, c = (model.step(tokens[4:8], rays[4:8], states) for states in (asked, other))
        for name in a:
            assert torch.equal(a[name], c[name])
