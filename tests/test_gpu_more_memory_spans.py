"""Linear attention's gradient (nesle_amd.memory.decay_attention) where the steps of some
tensors lie further apart than 32-bit offsets reach within a chunk: the states that the
forward kept are the ones that the gradient takes up.  Tolerances as in
tests/test_gpu_more_memory.py."""

from __future__ import annotations

import itertools

import pytest
import torch

from tests import more_memory_oracle as O
from tests import test_gpu_more_memory as M
from tests.helpers import say
from tests.memory_oracle import off
from tests.test_gpu_more_memory import F32, NAMES, dev, tol

pytestmark = pytest.mark.gpu


def most(dtype) -> int:
    """The largest step, in elements, at which 64 rows lie within what a 32-bit offset
    reaches, as a multiple of 8."""
    return ((1 << 31) - 4096) // 63 // dtype.itemsize // 8 * 8


def decay_terms(x, resets, grads, scale):
    """2-norms, a head, of the terms whose sum is the decay's gradient: for each token and
    console, each element of the state that reaches the token times the gradient of it."""
    q, k, v, g, S = (x[n].double() for n in NAMES)
    do, G = (t.double() for t in grads)
    which = torch.arange(v.shape[2]) // (v.shape[2] // q.shape[2])
    a, reach = torch.exp(g)[:, None, None], []
    for t in range(len(q)):
        reach.append(torch.where(resets[t][:, None, None, None], 0.0, S * a))
        S = reach[t] + k[t][:, which][..., None] * v[t][..., None, :]
    square = torch.zeros(v.shape[2], dtype=torch.float64)
    for t in reversed(range(len(q))):
        G = G + scale * q[t][:, which][..., None] * do[t][..., None, :]
        square += ((G * reach[t]) ** 2).sum((0, 2, 3))
        G = torch.where(resets[t][:, None, None, None], 0.0, G * a)
    return square.sqrt()


def check(shape, dtype, seed, far, steps):
    """Forward and gradient against the definition; the tensors named in `far` (of q, k, v,
    dout) have their steps `steps` elements apart.

    A decay's gradient is a sum of products of two factors, each of which is a float32
    result, off by F32 of itself; products off by 2 F32 of themselves, of either sign, add
    up to 2 F32 of the terms' 2-norm, however far the terms cancel in the sum (520 tokens of
    two consoles leave an eighth of it).  The sum itself rounds: F32 of the result."""
    from nesle_amd import memory

    T, N, hk, hv, dk, dv = shape
    x, resets, grads = M.make(*shape, dtype, seed, resets=0.02)
    ref = [x[n].double().requires_grad_() for n in NAMES]
    want = O.decay(*ref, resets, dk ** -0.5)
    dw = torch.autograd.grad(want, ref, [t.double() for t in grads])
    buf = torch.empty((T - 1) * steps + 4096, dtype=dtype, device=dev())
    place = itertools.count(0, 1024)

    def put(name, t):
        if name not in far:
            return t.to(dev())
        at = next(place)
        assert t[0].numel() <= 1024 and at < 4096
        cut = buf.as_strided(t.shape, (steps, *t[0].stride()), at)
        cut.copy_(t)
        return cut

    gpu = [put(n, x[n]).detach().requires_grad_() for n in NAMES]
    dout = put("dout", grads[0])
    got = memory.decay_attention(*gpu[:4], state=gpu[4], resets=resets.to(dev()))
    dg = torch.autograd.grad(got, gpu, [dout, grads[1].to(dev())])
    assert off(got[0], want[0]) <= tol(dtype) and off(got[1], want[1]) <= F32
    for n, a, b in zip(NAMES, dg, dw):
        if n == "g":
            room = F32 * b.abs() + 2 * F32 * decay_terms(x, resets, grads, dk ** -0.5)
            assert bool(((a.double().cpu() - b).abs() <= room).all()), (a, b, room)
        else:
            assert off(a, b) <= (tol(dtype) if n in "qkv" else F32), n


@pytest.mark.parametrize("far", ["dout", "v", "qkv", "qkv dout"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dim", [32, 64, 128])
@pytest.mark.parametrize("T", [33, 66, 130])
def test_gradient_where_steps_lie_far_apart(T, dim, dtype, far):
    say(f"[gpu] decay_attention {T} tokens of {dim} {dtype}, far: {far}")
    for steps in (most(dtype), most(dtype) + 8):
        check((T, 2, 1, 2, dim, dim), dtype, T + dim, set(far.split()) | (set("qkv") if "qkv" in far else set()), steps)


@pytest.mark.parametrize("far", ["dout", "qkv dout"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_segments_where_steps_lie_far_apart(dtype, far):
    """Few heads over so many tokens that they go in segments, in both directions."""
    say(f"[gpu] decay_attention segments {dtype}, far: {far}")
    check((520, 2, 1, 2, 40, 48), dtype, 3, set(far.split()) | (set("qkv") if "qkv" in far else set()), most(dtype) + 8)


def test_gradient_of_results_that_lie_far_apart():
    """133,500 heads of 64 in float32, whose results' steps lie that far apart by
    themselves: the first and the last consoles' results are those of the consoles alone.
    Both are float32 results: each off by F32 at most."""
    from nesle_amd import memory

    say("[gpu] decay_attention of 133,500 heads")
    T, N, some = 66, 133_500, 3
    x, resets, grads = M.make(T, some, 1, 1, 64, 64, torch.float32, 11, resets=0.02)
    small = [x[n].to(dev()).requires_grad_() for n in NAMES]
    grads, resets = [t.to(dev()) for t in grads], resets.to(dev())
    want = memory.decay_attention(*small[:4], state=small[4], resets=resets)
    dw = torch.autograd.grad(want, small, grads)

    def big(t, batch):
        out = torch.zeros(*t.shape[:batch], N, *t.shape[batch + 1:], dtype=t.dtype, device=dev())
        out.narrow(batch, 0, some).copy_(t)
        out.narrow(batch, N - some, some).copy_(t)
        return out

    wide = [big(t.detach(), 0 if n == "state" else 1) if n != "g" else t.detach() for n, t in zip(NAMES, small)]
    wide = [t.requires_grad_() for t in wide]
    got = memory.decay_attention(*wide[:4], state=wide[4], resets=big(resets, 1))
    d = torch.autograd.grad(got, wide, [big(grads[0], 1), big(grads[1], 0)])
    for n, a, b in zip(("out", "after", *NAMES), (*got, *d), (*want, *dw)):
        if n == "g":           # of both copies of the consoles
            assert off(a, 2 * b.double().cpu()) <= 2 * F32
            continue
        batch = 0 if n in ("after", "state") else 1
        for start in (0, N - some):
            assert off(a.narrow(batch, start, some), b.detach().double().cpu()) <= 2 * F32, (n, start)
