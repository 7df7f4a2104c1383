"""Shared pieces of the sequence operators' tests."""

from __future__ import annotations

import torch

#: Largest relative error of one rounding to the type.
UNIT = {torch.float32: 2.0**-24, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}
#: Half of the smallest subnormal: what a rounding may add to a tiny value.
TINY = {torch.float32: 2.0**-150, torch.float16: 2.0**-25, torch.bfloat16: 2.0**-134}
U32 = UNIT[torch.float32]
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def normal(shape, dtype, seed, scale=1.0, shift=0.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale + shift).to(dtype)


def assert_within(got, want, bound, what):
    """|got - want| <= bound, elementwise; non-finite values have to agree."""
    got, want = got.detach().cpu().double(), want.detach().cpu().double()
    bound = torch.as_tensor(bound, dtype=torch.float64).cpu().expand(want.shape)
    assert got.shape == want.shape, f"{what}: {tuple(got.shape)} and {tuple(want.shape)}"
    fine = torch.isfinite(want)
    assert torch.equal(fine, torch.isfinite(got)), f"{what}: other places are not finite"
    off = (got - want).abs()[fine]
    over = off > bound[fine]
    assert not over.any(), (
        f"{what}: {int(over.sum())} of {over.numel()} beyond the bound, worst "
        f"{float((off / bound[fine].clamp_min(1e-300)).max()):.2f} times it")
