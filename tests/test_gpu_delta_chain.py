"""delta_scan's chain over the chunks where its workgroups hold more waves than a value
has columns for, and where many heads run it with four waves a workgroup.

A wave takes sixteen columns of a state.  The bounds are those of
test_gpu_delta_scan.py; calls that run at once have to give the bits that they give alone."""

from __future__ import annotations

import pytest
import torch

from gaussian_splats_hip.sequence import delta_scan_backward, delta_scan_forward
from sequence_helpers import TYPES, normal
from test_gpu_delta_scan import DEV, _check, _inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(9, 70, 12, 4, 64, 72), (26, 70, 10, 5, 40, 24), (3, 130, 12, 3, 128, 128),
                                   (4, 66, 12, 6, 104, 96)])
def test_many_heads(shape, dtype):
    """More waves than the chain's smaller workgroups are used for: 512, and 256 with keys
    above 64; columns that fill their last workgroup and that do not."""
    print(f"[delta] many heads {shape} {dtype}", flush=True)
    b, _, h, _, d, dv = shape
    waves = b * h * -(-dv // 16)
    assert waves > (512 if d <= 64 else 256)
    _check(_inputs(*shape, dtype), normal((b, h, d, dv), torch.float32, 9))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [8, 24, 72, 104])
def test_gradients_of_calls_at_once(dim, dtype):
    """Forwards and backwards on several streams, chains whole and cut, keys of both
    tile sizes."""
    print(f"[delta] at once {dim} {dtype}", flush=True)
    shapes = [(2, 700, 3, 1, 40, dim), (2, 700, 3, 1, 128, dim), (1, 2400, 2, 2, 64, dim), (1, 2100, 2, 1, 72, dim)]
    calls = [[x.to(DEV) for x in _inputs(*s, dtype, shift=5.0)] for s in shapes]
    states = [normal((s[0], s[2], s[4], dim), torch.float32, 9).to(DEV) for s in shapes]
    dos = [normal(x[2].shape, dtype, 10).to(DEV) for x in calls]
    dlasts = [normal(s.shape, torch.float32, 11).to(DEV) for s in states]

    def run(x, state, do, dlast):
        out, last, kept = delta_scan_forward(*x, state)
        return out, last, *delta_scan_backward(*x, kept, do, dlast)

    alone = [run(*each) for each in zip(calls, states, dos, dlasts)]
    assert all(torch.isfinite(t).all() for results in alone for t in results)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in calls]
    for _ in range(3):
        got = []
        for stream, *each in zip(streams, calls, states, dos, dlasts):
            with torch.cuda.stream(stream):
                got.append(run(*each))
        torch.cuda.synchronize()
        for results, want in zip(got, alone):
            for a, c in zip(results, want):
                assert torch.equal(a, c)
