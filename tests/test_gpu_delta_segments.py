"""The gated delta rule over sequences whose chain of chunks is cut into segments
(from 2048 tokens on): the values of calls of 1536 tokens, whose chains are not cut
and which hand the state on; sequences of different lengths; tokens that are not
finite; replays of a graph.

Each side is off (2-norm) by at most 2 units of its type in 16 bits, 4 in the gates'
gradient, 2^-15 in states and 2^-17 in float32 (test_gpu_delta_scan.py); two of them
differ by at most twice that."""

from __future__ import annotations

import pytest
import torch

from gaussian_splats_hip.sequence import delta_scan, delta_scan_backward, delta_scan_forward
from oracle import sequence as oracle
from sequence_helpers import TYPES, UNIT, normal
from test_gpu_delta_scan import DEV, _inputs

pytestmark = pytest.mark.gpu


def _close(a, c, dtype, units=2):
    a, c = a.detach(), c.detach()
    off = float((a.double() - c.double()).norm() / c.double().norm())
    if dtype == torch.float32:
        most = 2.0**-17
    else:
        most = 2.0**-15 if a.dtype == torch.float32 else units * UNIT[dtype]
    assert off <= 2 * most, (off, most)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(1, 2048, 1, 1, 64, 64), (2, 4700, 3, 1, 24, 128), (1, 4160, 4, 2, 128, 64),
                                   (1, 2400, 32, 8, 128, 128)])
def test_equals_uncut_calls(shape, dtype):
    print(f"[delta] segments {shape} {dtype}", flush=True)
    b, t, h, _, d, dv = shape
    inputs = [x.to(DEV) for x in _inputs(*shape, dtype, shift=5.0)]
    state = normal((b, h, d, dv), torch.float32, 9).to(DEV)
    out, last = delta_scan(*inputs, state)
    parts = []
    for at in range(0, t, 1536):
        part, state = delta_scan(*(x[:, at:at + 1536] for x in inputs), state)
        parts.append(part)
    _close(out, torch.cat(parts, 1), dtype)
    _close(last, state, dtype)


@pytest.mark.parametrize("dtype", TYPES)
def test_lengths(dtype):
    """Sequences that end in some segment, in its first token, or at once."""
    lengths = [4700, 0, 2111, 513, 4097]
    inputs = [x.to(DEV) for x in _inputs(5, 4700, 2, 1, 64, 40, dtype, shift=5.0)]
    state = normal((5, 2, 64, 40), torch.float32, 9).to(DEV)
    do = normal((5, 4700, 2, 40), dtype, 10).to(DEV)
    dlast = normal(state.shape, torch.float32, 11).to(DEV)
    for i, n in enumerate(lengths):
        for x in (*inputs, do):
            x[i, n:] = float("nan")
    whole = [x.requires_grad_(True) for x in (*inputs, state)]
    got = delta_scan(*whole, lengths=torch.tensor(lengths, dtype=torch.int32, device=DEV))
    grads = torch.autograd.grad(got, whole, (do, dlast))
    for i, n in enumerate(lengths):
        alone = [x[i:i + 1, :n].detach().requires_grad_(True) for x in inputs]
        first = state[i:i + 1].detach().requires_grad_(True)
        want = delta_scan(*alone, first)
        assert not got[0][i, n:].any() and not any(g[i, n:].any() for g in grads[:5])
        if n == 0:
            assert torch.equal(got[1][i], state[i]) and torch.equal(grads[5][i], dlast[i])
            continue
        back = torch.autograd.grad(want, (*alone, first), (do[i:i + 1, :n], dlast[i:i + 1]))
        for a, c in ((got[0][i, :n], want[0][0]), (got[1][i], want[1][0]), (grads[5][i], back[5][0])):
            _close(a, c, dtype)
        for j, (a, c) in enumerate(zip(grads[:5], back[:5])):
            _close(a[i, :n], c[0], dtype, 4 if j == 3 else 2)


@pytest.mark.parametrize("dtype", TYPES)
def test_not_finite(dtype):
    """As in short sequences: NaN from the token on, all else keeps its bits; a
    gradient reaches other heads and sequences as before."""
    inputs = [x.to(DEV) for x in _inputs(2, 3000, 2, 2, 64, 64, dtype)]
    do = normal((2, 3000, 2, 64), dtype, 10).to(DEV)
    want, last, kept = delta_scan_forward(*inputs)
    grads = delta_scan_backward(*inputs, kept, do, None)
    for which, value in ((1, float("inf")), (2, float("nan")), (3, float("nan"))):
        bad = [x.clone() for x in inputs]
        bad[which][0, 1100, 1] = value
        out, end, kept = delta_scan_forward(*bad)
        assert out[0, 1100:, 1].isnan().all() and end[0, 1].isnan().all()
        keep = torch.ones_like(want, dtype=torch.bool)
        keep[0, 1100:, 1] = False
        assert torch.equal(out[keep], want[keep])
        assert torch.equal(end[1], last[1]) and torch.equal(end[0, 0], last[0, 0])
        for a, c in zip(delta_scan_backward(*bad, kept, do, None)[:5], grads):
            assert torch.equal(a[1], c[1]) and torch.equal(a[0, :, 0], c[0, :, 0])


def test_in_a_graph():
    """Two graphs that share no buffer of their own, replayed in turn, equal eager calls."""
    sizes = ((1, 2300, 4, 2, 64, 64), (2, 2100, 2, 1, 128, 64))
    inputs = [[x.to(DEV) for x in _inputs(*s, torch.bfloat16)] for s in sizes]
    dos = [normal(x[2].shape, torch.bfloat16, 9).to(DEV) for x in inputs]

    def run(x, do):
        out, last, kept = delta_scan_forward(*x)
        return out, last, *delta_scan_backward(*x, kept, do, None)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for x, do in zip(inputs, dos):
            run(x, do)
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for x, do in zip(inputs, dos):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            captured = run(x, do)
        graphs.append((graph, captured))
    for turn in range(3):
        for x, do, size, (graph, captured) in zip(inputs, dos, sizes, graphs):
            for t, fresh in zip(x, _inputs(*size, torch.bfloat16, 100 * turn)):
                t.copy_(fresh)
            graph.replay()
        torch.cuda.synchronize()
        for x, do, (_, captured) in zip(inputs, dos, graphs):
            for a, c in zip(captured, run(x, do)):
                assert torch.equal(a, c)


def test_two_calls_at_once():
    """Calls on two streams, cut and uncut, do not disturb one another."""
    calls = [[x.to(DEV) for x in _inputs(*s, torch.bfloat16)]
             for s in ((1, 5000, 4, 2, 64, 64), (1, 3000, 2, 2, 128, 128), (2, 700, 3, 1, 40, 72))]
    alone = [delta_scan(*x) for x in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in calls]
    for _ in range(3):
        got = []
        for x, stream in zip(calls, streams):
            with torch.cuda.stream(stream):
                got.append(delta_scan(*x))
        torch.cuda.synchronize()
        for a, c in zip(got, alone):
            assert torch.equal(a[0], c[0]) and torch.equal(a[1], c[1])


def test_one_tensor_as_query_and_key():
    """The same tensor twice, and gradients that are expanded: both sides' errors add up."""
    q, _, v, gate, beta = _inputs(1, 150, 2, 2, 16, 24, torch.float32)
    ones = torch.ones(v.shape), torch.ones(1, 2, 16, 24)
    want = oracle.delta_scan(q, q, v, gate, beta, grads=ones)
    on = [x.to(DEV).requires_grad_(True) for x in (q, v, gate, beta)]
    out, last = delta_scan(on[0], on[0], *on[1:])
    (out.sum() + last.sum()).backward()
    exact = [want[2] + want[3], *want[4:7]]
    sizes = [want[2].norm() + want[3].norm(), *(x.norm() for x in want[4:7])]
    for x, value, size in zip(on, exact, sizes):
        assert float((x.grad.cpu().double() - value).norm()) <= 2.0**-18 * float(size)
