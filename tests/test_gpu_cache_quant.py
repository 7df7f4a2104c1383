"""The 4-bit window cache on the GPU against its definition in float64.

Codes and exponents are whole numbers and have to be equal: a power of two divides
exactly, and a tie is decided.  What codes stand for is exact in the inputs' type, so
the step's bound is that of a cache in the inputs' type: with u the type's unit, U
float32's, n the slots seen and d the head dimension, a score is a sum of d products
in float32, its exponent takes two more roundings of at most s = scale |q| |k|; a
probability is within e = (2 d + 16) U (1 + s) before its rounding to the type, and
the output within (3 u + 2 e + 2 n U) max|v|.
"""

from __future__ import annotations

import math

import pytest
import torch

from gaussian_splats_hip.sequence import (
    QuantWindowCache,
    window_attention_step_quant,
    window_cache_fill_quant,
)
from oracle import sequence as orc
from sequence_helpers import TINY, TYPES, U32, UNIT, assert_within, normal

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")


def _cache(b, hk, n, d, seed):
    """Random codes, powers of two around a quarter: [codes, exponents] of keys, values."""
    g = torch.Generator().manual_seed(seed)
    out = []
    for _ in range(2):
        out += [torch.randint(0, 256, (b, hk, n, d // 2), generator=g, dtype=torch.uint8),
                torch.randint(122, 127, (b, hk, n, d // 32), generator=g, dtype=torch.uint8)]
    return out


def _step(q, k, v, cache, positions, window, sinks, scale=None):
    """(out, cache) by the definition: rows are encoded, what they stand for is attended to."""
    cache = [t.clone() for t in cache]
    for i, p in enumerate(positions.tolist()):
        if p >= 0:
            at = orc.cache_slot(p, window, sinks)
            cache[0][i, :, at], cache[1][i, :, at] = orc.mxfp4_encode(k[i])
            cache[2][i, :, at], cache[3][i, :, at] = orc.mxfp4_encode(v[i])
    keys, values = orc.mxfp4_decode(*cache[:2]), orc.mxfp4_decode(*cache[2:])
    b, h, d = q.shape
    hk = k.shape[1]
    out, bound = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    scale = 1 / math.sqrt(d) if scale is None else scale
    u, tiny = UNIT[q.dtype], TINY[q.dtype]
    for i, p in enumerate(positions.tolist()):
        n = min(p + 1, sinks + window)
        for m in range(h if n > 0 else 0):
            kk, vv = keys[i, m * hk // h, :n], values[i, m * hk // h, :n]
            w = torch.softmax(kk @ q[i, m].double() * scale, 0)
            out[i, m] = w @ vv
            size = scale * float(q[i, m].double().norm() * kk.nan_to_num(0.0).norm(dim=-1).max())
            e = (2 * d + 16) * U32 * (1 + size)
            bound[i, m] = (3 * u + 2 * e + 2 * n * U32) * vv.abs().nan_to_num(0.0).amax() + tiny * (1 + n)
    return out, cache, bound


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(1, 1, 1, 32, 1, 0), (3, 4, 2, 64, 5, 2), (2, 7, 1, 96, 100, 0),
                                   (5, 8, 8, 128, 33, 4), (2, 40, 1, 64, 300, 3), (1, 70, 1, 32, 130, 1),
                                   (4, 6, 2, 96, 2000, 16), (1, 2, 1, 128, 64, 100), (1, 8, 8, 64, 2500, 4)])
def test_step_matches_definition(shape, dtype):
    """Streams at their first token, among the first tokens, with the ring partly
    filled, just full and wrapped around; slots not filled yet hold NaN."""
    print(f"[step quant] {shape} {dtype}", flush=True)
    b, h, hk, d, window, sinks = shape
    n = window + sinks
    places = [0, sinks, n - 1, n, n + window // 2 + 1, max(0, sinks - 1), n // 2]
    for turn in range(2):
        positions = torch.tensor([places[(i + 3 * turn) % len(places)] for i in range(b)], dtype=torch.int32)
        q, k, v = normal((b, h, d), dtype, 1), normal((b, hk, d), dtype, 2), normal((b, hk, d), dtype, 3)
        cache = _cache(b, hk, n, d, 4)
        for i, p in enumerate(positions.tolist()):
            cache[1][i, :, p + 1:] = 255
            cache[3][i, :, p + 1:] = 255
        want, kept, bound = _step(q, k, v, cache, positions, window, sinks)
        on = [t.to(DEV) for t in cache]
        out = window_attention_step_quant(q.to(DEV), k.to(DEV), v.to(DEV), *on, positions.to(DEV), window, sinks)
        assert out.dtype == dtype
        for got, t in zip(on, kept):
            assert torch.equal(got.cpu(), t)
        assert_within(out, want, bound, "out")


@pytest.mark.parametrize("dtype", TYPES)
def test_every_code_and_power(dtype):
    """A slot that takes all the weight comes out as the value it stands for, whatever
    its codes and power; the new token's score is so low that its weight is zero."""
    powers = list(range(0, 253)) if dtype != torch.float16 else list(range(105, 140))
    b, d = len(powers), 32
    q, k, v = torch.zeros(b, 1, d, dtype=dtype), torch.zeros(b, 1, d, dtype=dtype), torch.ones(b, 1, d, dtype=dtype)
    q[..., 0], k[..., 0] = 100.0, -96.0
    cache = [torch.zeros(b, 1, 2, d // 2, dtype=torch.uint8), torch.zeros(b, 1, 2, 1, dtype=torch.uint8),
             torch.zeros(b, 1, 2, d // 2, dtype=torch.uint8), torch.zeros(b, 1, 2, 1, dtype=torch.uint8)]
    cache[0][:, :, 0, 0], cache[1][:, :, 0] = 7, 131
    cache[2][:, :, 0] = torch.tensor([2 * (i % 8) + 16 * (2 * (i % 8) + 1) for i in range(16)], dtype=torch.uint8)
    cache[3][:, 0, 0, 0] = torch.tensor(powers, dtype=torch.uint8)
    want = orc.mxfp4_decode(cache[2], cache[3])[:, :, 0]
    on = [t.to(DEV) for t in cache]
    at = torch.ones(b, dtype=torch.int32, device=DEV)
    out = window_attention_step_quant(q.to(DEV), k.to(DEV), v.to(DEV), *on, at, 2, 0).cpu()
    # Below the smallest normal number the matrix cores may flush to zero.
    small = want.abs() < (2.0**-14 if dtype == torch.float16 else 2.0**-126)
    # The weight p, near one, multiplies the value and divides the product: two roundings
    # of float32, fl(fl(p v) / p), after which a 16-bit type has the value again.
    near = want.abs() * (2 * U32 * (1 + U32) if dtype == torch.float32 else 0.0)
    assert ((out.double() - want)[~small].abs() <= near[~small]).all()
    assert ((out.double() - want)[small].abs() <= want[small].abs()).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_encoding(dtype):
    """Rows of every size, ties, zeros, infinities and NaN, filled and stepped."""
    top = 14 if dtype == torch.float16 else 126
    x = normal((64, 128), torch.float32, 1)
    x *= torch.exp2(torch.linspace(-30 if dtype == torch.float16 else -148, top, 64))[:, None]
    x[1, :32] = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.9] * 4) * 4
    x[2, 32:64] = -torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.5] * 4)
    x[3], x[4, 96:] = 0.0, -0.0
    x = x.clamp(-60000, 60000) if dtype == torch.float16 else x
    x = x.to(dtype)
    x[5, 3], x[6, 77], x[7, 127] = float("inf"), -float("inf"), float("nan")
    rows = x[:, None, None]  # 64 streams of one token
    want = orc.mxfp4_encode(x)
    for form in ("fill", "step"):
        cache = QuantWindowCache(64, 1, 128, 3, 1, DEV)
        if form == "fill":
            cache.fill(rows.to(DEV), rows.flip(0).to(DEV))
        else:
            cache.step(x[:, None].to(DEV), x[:, None].to(DEV), x.flip(0)[:, None].to(DEV))
        assert torch.equal(cache.k_codes[:, 0, 0].cpu(), want[0]), form
        assert torch.equal(cache.k_exponents[:, 0, 0].cpu(), want[1]), form
        assert torch.equal(cache.v_codes[:, 0, 0].cpu(), want[0].flip(0)), form
        assert torch.equal(cache.v_exponents[:, 0, 0].cpu(), want[1].flip(0)), form
        assert cache.positions.tolist() == [1] * 64


@pytest.mark.parametrize("dtype", TYPES)
def test_blocks_of_nan(dtype):
    """A key with one makes its heads' outputs NaN; a value with one those elements."""
    b, hk, n, d = 2, 2, 200, 64
    q, k, v = normal((b, 4, d), dtype, 1), normal((b, hk, d), dtype, 2), normal((b, hk, d), dtype, 3)
    cache = _cache(b, hk, n, d, 4)
    cache[1][0, 1, 77, 1], cache[3][1, 0, 140, 0] = 255, 255
    positions = torch.tensor([500, 300], dtype=torch.int32)
    want, _, bound = _step(q, k, v, cache, positions, n, 0)
    assert want[0, 2:].isnan().all() and want[1, :2, :32].isnan().all() and int(want.isnan().sum()) == 192
    out = window_attention_step_quant(q.to(DEV), k.to(DEV), v.to(DEV), *(t.to(DEV) for t in cache),
                                      positions.to(DEV), n, 0)
    assert_within(out, want, bound, "out")


def test_inactive_streams():
    positions = torch.tensor([-1, 3], dtype=torch.int32, device=DEV)
    q, k = torch.ones(2, 2, 32, device=DEV), torch.ones(2, 1, 32, device=DEV)
    cache = QuantWindowCache(2, 1, 32, 8, 1, DEV)
    cache.positions.copy_(positions)
    out = cache.step(q, k, k)
    assert not out[0].any() and out[1].any() and cache.positions.tolist() == [-1, 4]
    assert not cache.k_codes[0].any() and not cache.v_exponents[0].any()
    assert cache.k_codes[1].any(-1)[0].nonzero().tolist() == [[3]]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens,window,sinks", [(1, 5, 2), (2, 5, 2), (7, 5, 2), (8, 5, 2), (40, 5, 0), (33, 40, 3)])
def test_fill(tokens, window, sinks, dtype):
    """Each slot takes the last of its tokens; slots without one stay; any strides."""
    b, hk, d, n = 3, 2, 96, window + sinks
    whole = normal((b, hk, tokens, 2 * d + 8), dtype, 1)
    k, v = whole[..., :d].transpose(1, 2), whole[..., d + 3:2 * d + 3].transpose(1, 2)
    on = whole.to(DEV)
    kd, vd = on[..., :d].transpose(1, 2), on[..., d + 3:2 * d + 3].transpose(1, 2)
    for lengths in (None, [tokens, 0, tokens // 2], [-4, tokens + 9, 1]):
        cache = _cache(b, hk, n, d, 5)
        got = [t.to(DEV) for t in cache]
        at = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device=DEV)
        window_cache_fill_quant(kd, vd, *got, window, sinks, at)
        for i in range(b):
            length = tokens if lengths is None else max(0, min(tokens, lengths[i]))
            token = orc.window_cache_fill(k[i], length, window, sinks, n)
            slots = (token >= 0).nonzero()[:, 0]
            for j, t in ((0, k), (2, v)):
                codes, exponents = orc.mxfp4_encode(t[i, token[slots]].transpose(0, 1))
                cache[j][i, :, slots], cache[j + 1][i, :, slots] = codes, exponents
        for a, c in zip(got, cache):
            assert torch.equal(a.cpu(), c)


def test_stream_goes_on_behind_a_prefill():
    """Filled and stepped caches hold what steps alone put there, and give the same."""
    b, hk, h, d, window, sinks, tokens = 3, 2, 4, 64, 20, 3, 50
    lengths = torch.tensor([50, 7, 0], dtype=torch.int32, device=DEV)
    q, k, v = (normal((b, tokens + 30, n, d), torch.bfloat16, i).to(DEV) for i, n in ((1, h), (2, hk), (3, hk)))
    filled, stepped = (QuantWindowCache(b, hk, d, window, sinks, DEV) for _ in range(2))
    filled.fill(k[:, :tokens], v[:, :tokens], lengths)
    each = torch.arange(b, device=DEV)
    for t in range(tokens):
        place = stepped.positions.clone()
        stepped.positions[lengths <= t] = -1
        stepped.step(q[:, t], k[:, t], v[:, t])
        stepped.positions.copy_(torch.where(lengths <= t, place, place + 1))
    assert torch.equal(filled.positions, lengths) and torch.equal(stepped.positions, lengths)
    for a, c in zip(filled._tensors(), stepped._tensors()):
        assert torch.equal(a, c)
    for _ in range(30):
        at = filled.positions.long()
        args = q[each, at], k[each, at], v[each, at]
        assert torch.equal(filled.step(*args), stepped.step(*args))


def test_step_in_a_graph():
    """Replays with new inputs and positions in the captured buffers, with eager work
    between them, equal eager steps."""
    b, h, hk, d, window, sinks = 2, 4, 2, 64, 600, 2
    q, k, v = (normal((b, n, d), torch.bfloat16, i).to(DEV) for i, n in ((1, h), (2, hk), (3, hk)))
    cache, twin = (QuantWindowCache(b, hk, d, window, sinks, DEV) for _ in range(2))
    for c in (cache, twin):
        for t in c._tensors():
            t.copy_(torch.randint(100, 120, t.shape, generator=torch.Generator().manual_seed(3)).to(torch.uint8))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        cache.step(q, k, v)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = cache.step(q, k, v)
    for c in (cache, twin):
        c.positions.fill_(580)
    twin.k_codes.copy_(cache.k_codes), twin.k_exponents.copy_(cache.k_exponents)
    twin.v_codes.copy_(cache.v_codes), twin.v_exponents.copy_(cache.v_exponents)
    for t in range(40):
        for i, x in enumerate((q, k, v)):
            x.copy_(normal(x.shape, torch.bfloat16, 10 * t + i))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, twin.step(q, k, v)), t
        assert torch.equal(cache.k_codes, twin.k_codes) and torch.equal(cache.positions, twin.positions)


def test_offsets_beyond_32_bits():
    """A stream of more than 2^31 bytes of codes whose last slots take all the weight
    (scores of some hundreds, all others zero) gives what those slots alone give."""
    window, near, d = (1 << 25) + 100, 100, 128
    cache = [torch.zeros((1, 1, window, w), dtype=torch.uint8, device=DEV) for w in (64, 4, 64, 4)]
    small = [torch.zeros((1, 1, near, w), dtype=torch.uint8, device=DEV) for w in (64, 4, 64, 4)]
    g = torch.Generator().manual_seed(1)
    for t, s in zip(cache, small):
        if t.shape[-1] == 64:  # positive codes
            s.copy_(torch.randint(0, 256, s.shape, generator=g, dtype=torch.uint8) & 0x77)
        else:
            s.fill_(127)
        t[:, :, -near:] = s
    q, k = torch.ones(1, 2, d, dtype=torch.bfloat16), torch.full((1, 1, d), 2.0, dtype=torch.bfloat16)
    v = normal((1, 1, d), torch.bfloat16, 3)
    want, kept, bound = _step(q, k, v, [t.cpu() for t in small], torch.tensor([near - 1]), near, 0, 1.0)
    at = torch.tensor([window - 1], dtype=torch.int32, device=DEV)
    out = window_attention_step_quant(q.to(DEV), k.to(DEV), v.to(DEV), *cache, at, window, 0, 1.0)
    assert_within(out, want, bound, "out")
    for t, s in zip(cache, kept):
        assert torch.equal(t[:, :, -near:].cpu(), s)
    # A fill that wraps around leaves a slot's last token, far from the first.
    window_cache_fill_quant(k[:, None].to(DEV), k[:, None].to(DEV), *cache, window)
    assert torch.equal(cache[0][0, 0, 0].cpu(), orc.mxfp4_encode(k[0])[0][0])
    assert torch.equal(cache[0][:, :, -near:].cpu(), kept[0])


def test_fill_in_a_graph():
    """A captured filling follows its buffers' tokens and lengths."""
    k, v = (normal((3, 90, 2, 64), torch.bfloat16, i).to(DEV) for i in (1, 2))
    lengths = torch.tensor([90, 5, 0], dtype=torch.int32, device=DEV)
    cache, twin = (QuantWindowCache(3, 2, 64, 30, 4, DEV) for _ in range(2))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        cache.fill(k, v, lengths)
    torch.cuda.current_stream().wait_stream(side)
    twin.fill(k, v, lengths)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.fill(k, v, lengths)
    for turn in range(3):
        for i, x in enumerate((k, v)):
            x.copy_(normal(x.shape, torch.bfloat16, 10 * turn + i))
        lengths.copy_(torch.tensor([turn, 90 - turn, 40]))
        graph.replay()
        torch.cuda.synchronize()
        twin.fill(k, v, lengths)
        for a, c in zip((*cache._tensors(), cache.positions), (*twin._tensors(), twin.positions)):
            assert torch.equal(a, c)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("shape", [(64, 8, 2, 64, 6, 1), (16, 34, 1, 128, 9, 0), (40, 16, 1, 96, 7, 0)])
def test_outputs_have_one_rounding(shape, dtype):
    """With values of one sign an output is as large as what is added up for it.
    Probabilities are two numbers of the type, each cut off: within 2^-15 relative in
    bfloat16 (2^-20 in float16, beside float32's scores at 2^-18), which moves a value
    over the border between two of the type, 2^-8 (2^-11) of it apart, in at most 2^-6
    (2^-6) of all places.  Probabilities rounded to the type once, 2^-9 (2^-12) off,
    moved a twelfth of them."""
    b, h, hk, d, window, sinks = shape
    n = window + sinks
    q, k, v = normal((b, h, d), dtype, 1), normal((b, hk, d), dtype, 2), normal((b, hk, d), dtype, 3).abs()
    cache = _cache(b, hk, n, d, 4)
    cache[2] &= 0x77
    positions = torch.full((b,), n - 1, dtype=torch.int32)
    want, _, _ = _step(q, k, v, cache, positions, window, sinks)
    out = window_attention_step_quant(q.to(DEV), k.to(DEV), v.to(DEV), *(t.to(DEV) for t in cache),
                                      positions.to(DEV), window, sinks).cpu()
    moved = float((out != want.to(dtype)).double().mean())
    print(f"[step quant] {shape} {dtype}: {moved:.4f} of the values moved", flush=True)
    assert moved <= 2.0**-6
