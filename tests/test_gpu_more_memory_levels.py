"""Layer norm (nesle_amd.memory.layer_norm) of rows whose level is far above their
spread, against the definition of the very inputs in float64."""

from __future__ import annotations

import math

import pytest
import torch

from tests import more_memory_oracle as O
from tests.helpers import say
from tests.memory_oracle import off
from tests.test_gpu_more_memory import F32, NORM, dev, tol

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,level", [(torch.float32, 2.0 ** 8), (torch.float32, 2.0 ** 12), (torch.float32, -2.0 ** 16),
                                         (torch.float32, 2.0 ** 20), (torch.bfloat16, 2.0 ** 8), (torch.bfloat16, -2.0 ** 12)])
@pytest.mark.parametrize("dim", [7, 64, 201, 256, 1000, 4096, 16384])
def test_a_level_does_not_cost_precision(dim, dtype, level):
    """Elements and a mean that is rounded lie within a factor of two of each other, so
    their differences are exact; they share the mean's error, a fraction of the spread
    (at 2^20 a few of 2^-4), which goes out with their own mean, rounded relative to
    them.  What is left rounds as it does without a level: NORM, and 4 NORM of the terms
    of the gradient (tests/test_gpu_more_memory.py)."""
    from nesle_amd import memory

    say(f"[gpu] layer_norm of {dim} at {level} {dtype}")
    gen = torch.Generator().manual_seed(dim)
    spread = 1.0 if dtype == torch.float32 else abs(level) / 64       # a few steps of the type
    x = (spread * torch.randn(33, dim, generator=gen) + level).to(dtype)
    dy = torch.randn(33, dim, generator=gen).to(dtype)
    w, b = 1 + 0.3 * torch.randn(dim, generator=gen), 0.3 * torch.randn(dim, generator=gen)
    ref = [t.double().requires_grad_() for t in (x, w, b)]
    gpu = [t.to(dev()).requires_grad_() for t in (x, w, b)]
    want, got = O.layer_norm(*ref, 1e-5), memory.layer_norm(*gpu)
    assert off(got, want) <= tol(dtype, NORM)
    dw = torch.autograd.grad(want, ref, dy.double())
    dg = torch.autograd.grad(got, gpu, dy.to(dev()))
    terms = dy.double() * w.double() / torch.sqrt(x.double().var(-1, correction=0, keepdim=True) + 1e-5)
    error = off(dg[0], dw[0]) * float(dw[0].norm())
    assert error <= 4 * NORM * float(terms.norm()) + (0 if dtype == torch.float32 else 2.0 ** -9 * float(dw[0].norm()))
    for a, t in zip(dg[1:], dw[1:]):
        assert off(a, t) <= F32


@pytest.mark.parametrize("dim", [3, 201, 256, 1000])
def test_rows_of_one_value(dim):
    """Such a row is its bias, whatever its value: the differences from the mean are one
    rounding of it at most, and go out with their own mean to 2^-24 of themselves, times
    1 / sqrt(eps) = 316: 2^-48 316 of the value.  Without eps: 0 / 0, or a quotient of two
    roundings, but nothing of it in other rows."""
    from nesle_amd import memory

    say(f"[gpu] layer_norm of rows of one value, {dim}")
    x = torch.tensor([0.1, -3.3, 1e4 / 3, 2.0 ** 20 + 0.125, 0.0])[:, None].expand(5, dim).contiguous().to(dev())
    y = memory.layer_norm(x)
    assert bool((y.abs() <= 16 * 2.0 ** -48 * 316 * x.abs()).all())
    row = torch.randn(dim, generator=torch.Generator().manual_seed(1)).to(dev())
    x[1] = row
    y = memory.layer_norm(x, eps=0.0)
    assert off(y[1], O.layer_norm(row.cpu(), None, None, 0.0)) <= 4 * NORM
    x[2, 0] = math.inf
    x[3, 1] = math.nan
    y = memory.layer_norm(x)
    assert not bool(y[2:4].isfinite().any()) and bool(y[[0, 1, 4]].isfinite().all())
