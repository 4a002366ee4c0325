"""Linear attention whose decays grow (g above 0; nesle_amd.memory.decay_attention):
powers of the decay past float32's range, which no token of a chunk has, reach nothing."""

from __future__ import annotations

import pytest
import torch

from tests import more_memory_oracle as O
from tests import test_gpu_more_memory as M
from tests.helpers import say
from tests.memory_oracle import off
from tests.test_gpu_more_memory import F32, NAMES, dev, tol
from tests.test_gpu_more_memory_spans import decay_terms

pytestmark = pytest.mark.gpu

BOTH = [torch.float32, torch.bfloat16]


def check(x, resets, grads, longest):
    """Against the definition, where no episode, in a chunk, has more than `longest` tokens.
    A power exp(n g) comes from the rounded product: off by n g 2^-24 of itself, once for
    what the state carries and once for the pairs; they do not add up, as each result's
    largest terms are of one of the two.  The decay's gradient: as in
    tests/test_gpu_more_memory_spans.py, of its terms."""
    from nesle_amd import memory

    dtype, scale = x["q"].dtype, x["q"].shape[-1] ** -0.5
    room = longest * float(x["g"].max()) * 2.0 ** -24
    ref = [x[n].double().requires_grad_() for n in NAMES]
    want = O.decay(*ref, resets, scale)
    gpu = [x[n].to(dev()).requires_grad_() for n in NAMES]
    got = memory.decay_attention(*gpu[:4], state=gpu[4], resets=resets.to(dev()))
    assert off(got[0], want[0]) <= tol(dtype) + room and off(got[1], want[1]) <= F32 + room
    dw = torch.autograd.grad(want, ref, [t.double() for t in grads])
    dg = torch.autograd.grad(got, gpu, [t.to(dev()) for t in grads])
    for n, a, b in zip(NAMES, dg, dw):
        if n == "g":
            most = F32 * b.abs() + 2 * (F32 + room) * decay_terms(x, resets, grads, scale)
            assert bool(((a.double().cpu() - b).abs() <= most).all()), (a, b, most)
        else:
            assert off(a, b) <= (tol(dtype) if n in "qkv" else F32) + room, n


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("dim", [16, 64, 128])
@pytest.mark.parametrize("T,g", [(1, 3.0), (1, 20.0), (2, 10.0), (5, 6.0), (17, 3.0), (20, 2.8), (31, 1.5)])
def test_a_short_chunk_of_heads_that_grow(T, g, dim, dtype):
    """Few tokens: exp(n g) is finite for the tokens there are, not for a whole chunk."""
    say(f"[gpu] decay_attention {T} tokens of {dim} {dtype}, g = {g}")
    x, resets, grads = M.make(T, 2, 1, 2, dim, dim, dtype, T, resets=0.0)
    x["g"] = torch.tensor([g, 0.5 * g])
    check(x, resets, grads, T)


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("T", [512 + 4, 512 + 1, 96 + 3])
def test_a_short_last_chunk_after_short_episodes(T, dtype):
    """Episodes of 8 tokens keep heads that grow finite, but not the powers over a chunk of
    64; the last chunk is short and has no episode's end (the one of 516 and of 513 tokens
    is a segment of its own)."""
    say(f"[gpu] decay_attention {T} tokens {dtype}, short episodes of heads that grow")
    x, resets, grads = M.make(T, 2, 1, 2, 32, 32, dtype, 2, resets=0.0)
    x["g"] = torch.tensor([1.5, 1.45])
    resets[4::8] = True
    assert not bool(resets[T // 64 * 64 if T > 512 else T // 32 * 32:].any())
    check(x, resets, grads, 8)
