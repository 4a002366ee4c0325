"""Linear attention with a decay for each head, layer norm and sampling
(nesle_amd.memory) on the GPU against their definitions in float64
(tests/more_memory_oracle.py).

Tolerances, on the 2-norm of the difference over the 2-norm of the result.
Float32: a result goes through a few sums of at most 128 products, each rounding
2^-24 relative to a running sum of which about sqrt(128) random ones add up (7e-7),
over up to a handful of stages: 4e-6.  bfloat16: compared with the definition
rounded to bfloat16, from which one rounding of the float32 result differs in the
few elements that the float32 error carries over a rounding boundary: 2^-9 on top of
it.  Layer norm: statistics and the result take about six roundings an element, sums
over lanes a logarithm of that more: 16 x 2^-24 = 1e-6; the weights' gradients are sums of
up to 1,000 products a lane: 4e-6."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

from tests import more_memory_oracle as O
from tests.helpers import say
from tests.memory_oracle import off

pytestmark = pytest.mark.gpu

F32, NORM = 4e-6, 1e-6


def tol(dtype, f32=F32) -> float:
    return f32 if dtype == torch.float32 else 2.0 ** -9 + f32


def dev():
    return torch.device("cuda")


# ---- linear attention with a decay for each head ----------------------------------------

def make(T, N, hk, hv, dk, dv, dtype, seed, resets=0.1, alike=0.7):
    """Inputs on the CPU: unit queries and keys (neighbouring tokens alike), decays
    of half lives from 2 to 700 tokens, an initial state, resets, gradients."""
    gen = torch.Generator().manual_seed(seed)
    base = torch.randn(2, N, hk, dk, generator=gen)

    def unit(i):
        x = torch.randn(T, N, hk, dk, generator=gen) * (1 - alike) + base[i] * alike
        return (x / x.norm(dim=-1, keepdim=True)).to(dtype)

    x = {"q": unit(0), "k": unit(1), "v": torch.randn(T, N, hv, dv, generator=gen).to(dtype),
         "g": -torch.exp(torch.linspace(math.log(0.001), math.log(0.3), hv)), "state": torch.randn(N, hv, dk, dv, generator=gen)}
    resets = torch.rand(T, N, generator=gen) < resets
    grads = torch.randn(T, N, hv, dv, generator=gen).to(dtype), torch.randn(N, hv, dk, dv, generator=gen)
    return x, resets, grads


NAMES = ("q", "k", "v", "g", "state")


def check_decay(x, resets, grads, scale=None, train=True, move=lambda t: t.to(dev())):
    """Forward and gradient against the definition."""
    from nesle_amd import memory

    dtype = x["q"].dtype
    s = x["q"].shape[-1] ** -0.5 if scale is None else scale
    ref = {n: None if x[n] is None else x[n].double().requires_grad_() for n in NAMES}
    want = O.decay(*(ref[n] for n in NAMES), resets, s)
    gpu = {n: None if x[n] is None else move(x[n]).requires_grad_(train) for n in NAMES}
    got = memory.decay_attention(gpu["q"], gpu["k"], gpu["v"], gpu["g"], state=gpu["state"],
                                 resets=None if resets is None else resets.to(dev()), scale=scale)
    assert got[0].dtype == dtype and got[1].dtype == torch.float32
    assert off(got[0], want[0]) <= tol(dtype), "out"
    assert off(got[1], want[1]) <= F32, "state"
    if not train:
        return got
    names = [n for n in NAMES if x[n] is not None]
    dw = torch.autograd.grad(want, [ref[n] for n in names], [t.double() for t in grads], allow_unused=True)
    dg = torch.autograd.grad(got, [gpu[n] for n in names], [t.to(dev()) for t in grads])
    for n, a, b in zip(names, dg, dw):
        b = torch.zeros_like(ref[n]) if b is None else b
        assert a.dtype == x[n].dtype
        error = off(a, b)
        say(f"[gpu]   d{n} {error:.2g}")
        assert error <= (tol(dtype) if n in "qkv" else F32), f"d{n}"
    return got


SHAPES = [(1, 1, 1, 1, 8, 8), (3, 2, 2, 2, 16, 24), (31, 2, 1, 1, 32, 32), (32, 1, 2, 4, 32, 16), (33, 3, 1, 3, 48, 40),
          (64, 2, 2, 2, 64, 64), (77, 3, 2, 4, 64, 24), (130, 2, 1, 1, 64, 64), (65, 2, 1, 2, 128, 128),
          (40, 1, 1, 1, 24, 104), (96, 1, 2, 2, 128, 64), (200, 1, 1, 2, 16, 72)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", SHAPES)
def test_decay_matches_the_definition(shape, dtype):
    say(f"[gpu] decay_attention {shape} {dtype}")
    check_decay(*make(*shape, dtype, seed=sum(shape)))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("where", ["none", "all", "first", "edges", "last"])
def test_decay_resets(where, dtype):
    say(f"[gpu] decay_attention resets {where} {dtype}")
    x, resets, grads = make(150, 3, 1, 2, 32, 32, dtype, 5)
    resets[:] = where == "all"
    if where == "first":
        resets[0] = True
    if where == "last":
        resets[-1] = True
    if where == "edges":
        for n, t in enumerate((31, 63, 64)):
            resets[t, n] = True
            resets[t + 1, n] = n == 2
            resets[t + 64, n] = n != 1
    check_decay(x, resets, grads)
    check_decay(x, None if where == "none" else resets.to(torch.uint8) * 255, grads)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("decay", ["none", "strong", "off", "growing"])
def test_decay_decays(decay, dtype):
    """No decay; decays that leave nothing after a few tokens; heads of -inf and -200
    (a token sees itself alone); heads that grow."""
    say(f"[gpu] decay_attention decays {decay} {dtype}")
    x, resets, grads = make(100, 2, 2, 4, 32, 32, dtype, 6, resets=0.02)
    x["g"] = {"none": torch.zeros(4), "strong": torch.tensor([-1.0, -5.0, -20.0, -80.0]),
              "off": torch.tensor([-200.0, -0.1, -math.inf, -103.9]), "growing": torch.tensor([0.02, -0.01, 0.05, 0.0])}[decay]
    if decay != "off":
        check_decay(x, resets, grads)
        return
    # The definition has 0 x inf for the gradient of such a head's decay; it is 0.
    check_decay(x, resets, grads, train=False)
    from nesle_amd import memory

    gpu = {n: x[n].to(dev()).requires_grad_() for n in NAMES}
    got = memory.decay_attention(*(gpu[n] for n in NAMES[:4]), state=gpu["state"], resets=resets.to(dev()))
    dg = torch.autograd.grad(got, list(gpu.values()), [t.to(dev()) for t in grads])
    assert all(bool(t.isfinite().all()) for t in dg)
    assert float(dg[3][0]) == 0.0 and float(dg[3][2]) == 0.0 and float(dg[3][1]) != 0.0
    assert bool((dg[4][:, [0, 2]] == 0.0).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [(513, 1, 1, 1, 16, 16), (700, 2, 1, 2, 64, 64), (1100, 1, 2, 2, 128, 40), (2049, 1, 1, 1, 32, 32),
                                   (1029, 3, 1, 2, 24, 64)])
def test_decay_long_walks(shape, dtype):
    """Few heads over many tokens go in segments; ends of episodes in the first, the last,
    none and all of them, at their borders and inside."""
    from nesle_amd import abi

    say(f"[gpu] decay_attention segments {shape} {dtype}")
    T, N, hk, hv, dk, dv = shape
    a = abi.DecayArgs(abi.MEM_F32 if dtype == torch.float32 else abi.MEM_BF16, T, N, hk, hv, dk, dv, 1.0)
    assert abi.lib().nesle_decay_forward_scratch_floats(ctypes.byref(a)) > 0
    x, resets, grads = make(*shape, dtype, seed=T, resets=0.004)
    check_decay(x, resets, grads)
    resets[:] = False
    check_decay(x, resets, grads)
    for t in (0, 63, 64, 128, T - 1):
        resets[:] = False
        resets[t] = True
        check_decay(x, resets, grads, train=t in (64, T - 1))
    # Something that is not finite before an episode's end stays before it.
    from nesle_amd import memory

    resets[:] = False
    resets[300] = True
    gpu = {n: x[n].to(dev()) for n in NAMES}
    want = memory.decay_attention(*(gpu[n] for n in NAMES[:4]), state=gpu["state"], resets=resets.to(dev()))
    gpu["v"][200] = math.nan
    gpu["k"][100] = math.inf
    got = memory.decay_attention(*(gpu[n] for n in NAMES[:4]), state=gpu["state"], resets=resets.to(dev()))
    for a, b in ((got[0][:100], want[0][:100]), (got[0][300:], want[0][300:]), (got[1], want[1])):
        assert float((a.double() - b.double()).norm() / b.double().norm()) <= tol(dtype) + (0 if dtype == torch.float32 else 2.0 ** -9)


def test_decay_without_state_or_tokens():
    from nesle_amd import memory

    say("[gpu] decay_attention without state or tokens")
    x, resets, grads = make(70, 2, 1, 2, 64, 64, torch.float32, 7)
    x["state"] = None
    check_decay(x, resets, grads)
    for T, N in ((0, 2), (3, 0)):
        x, _, _ = make(T, N, 1, 2, 16, 16, torch.float32, 8)
        gpu = {n: x[n].to(dev()).requires_grad_() for n in NAMES}
        out, state = memory.decay_attention(*(gpu[n] for n in NAMES[:4]), state=gpu["state"])
        assert out.shape == (T, N, 2, 16)
        assert torch.equal(state.cpu(), x["state"])
        d = torch.autograd.grad((out.sum() + (2.0 * state).sum()), list(gpu.values()))
        assert bool((d[3] == 0.0).all()) and bool((d[4] == 2.0).all())


def test_decay_gradient_by_differences():
    """out is linear in each of q, k, v and the state, so differences have no error
    but rounding: 2^-24 of the loss's 10^5 terms' 2-norm, next to a derivative of the
    same terms: 1e-4 of it.  The decay's by a step of 2^-10 whose square, times the
    distances' (at most 80 tokens, mean about 20), leaves 4e-4."""
    from nesle_amd import memory

    say("[gpu] decay_attention differences")
    x, resets, grads = make(80, 2, 1, 2, 32, 32, torch.float32, 9, resets=0.02)
    gpu = {n: x[n].to(dev()).requires_grad_() for n in NAMES}
    do, ds = (t.to(dev()) for t in grads)

    def loss(args):
        out, state = memory.decay_attention(*(args[n] for n in NAMES[:4]), state=args["state"], resets=resets.to(dev()))
        return (out.double() * do).sum() + (state.double() * ds).sum()

    d = dict(zip(NAMES, torch.autograd.grad(loss(gpu), list(gpu.values()))))
    gen = torch.Generator().manual_seed(1)
    for n in NAMES:
        way = torch.randn(x[n].shape, generator=gen).to(dev()) * (2.0 ** -10 if n == "g" else 1.0)
        if n != "g":           # along the gradient as well, so that the answer is not near 0
            way = way + d[n] / d[n].norm() * way.norm()
        else:
            way = way.abs() * torch.sign(d[n])
        with torch.no_grad():
            change = (loss({**gpu, n: gpu[n] + way}) - loss({**gpu, n: gpu[n] - way})) / 2.0
        want = float((d[n].double() * way).sum())
        assert abs(float(change) - want) <= (4e-4 if n == "g" else 1e-4) * abs(want), n


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_decay_step_is_a_rollout_token_by_token(dtype):
    from nesle_amd import memory

    for shape in ((1, 1, 1, 8, 8), (5, 2, 4, 48, 40), (3, 1, 2, 128, 128), (300, 4, 4, 64, 64)):
        say(f"[gpu] decay_attention_step {shape} {dtype}")
        x, resets, _ = make(6, *shape, dtype, 3, resets=0.2)
        want = O.decay(*(x[n] for n in NAMES), resets, 0.5)
        gpu = {n: x[n].to(dev()) for n in NAMES}
        state, outs = gpu["state"].clone(), []
        for t in range(6):
            version = state._version
            outs.append(memory.decay_attention_step(gpu["q"][t], gpu["k"][t], gpu["v"][t], gpu["g"], state,
                                                    resets=resets[t].to(dev()), scale=0.5))
            assert state._version > version
        assert off(torch.stack(outs), want[0]) <= tol(dtype)
        assert off(state, want[1]) <= F32


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_decay_takes_strided_inputs(dtype):
    """Slices of one projection, off 16-byte boundaries, other orders of the leading
    dimensions, expanded heads."""
    from nesle_amd import memory

    say(f"[gpu] decay_attention strides {dtype}")
    x, resets, grads = make(70, 3, 2, 2, 24, 24, dtype, 11)
    flat = torch.cat([x[n].flatten(-2) for n in "qkv"], -1).to(dev())
    want = memory.decay_attention(*(x[n].to(dev()) for n in NAMES[:4]), resets=resets.to(dev()))
    q, k, v = flat.unflatten(-1, (3, 2, 24)).unbind(-3)
    g = x["g"].to(dev())
    for cut in (0, 1, 3):
        wide = torch.zeros(70, 3, 3 * 48 + 8, dtype=dtype, device=dev())
        wide[..., cut:cut + 3 * 48] = flat
        a, b, c = wide[..., cut:cut + 3 * 48].unflatten(-1, (3, 2, 24)).unbind(-3)
        got = memory.decay_attention(a, b, c, g, resets=resets.to(dev()))
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    swapped = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v)]
    got = memory.decay_attention(*swapped, g, resets=resets.to(dev()))
    assert torch.equal(got[0], want[0])
    leaf = q[:, :, :1].detach().clone().requires_grad_()
    out, _ = memory.decay_attention(leaf.expand(-1, -1, 2, -1), k, v, g, resets=resets.to(dev()))
    each = q[:, :, :1].expand(-1, -1, 2, -1).detach().clone().requires_grad_()
    same, _ = memory.decay_attention(each, k, v, g, resets=resets.to(dev()))
    assert torch.equal(out, same)
    do = grads[0].to(dev())
    one, two = torch.autograd.grad(out, leaf, do)[0], torch.autograd.grad(same, each, do)[0]
    assert off(one, two.double().sum(2, keepdim=True).cpu()) <= tol(dtype) + (0 if dtype == torch.float32 else 2.0 ** -8)
    # A gradient that is expanded, transposed, or a slice.
    leaves = [t.detach().clone().requires_grad_() for t in (q, k, v)]
    out, state = memory.decay_attention(*leaves, g, resets=resets.to(dev()))
    for dout in (torch.ones(1, device=dev(), dtype=dtype).expand_as(out), do.transpose(0, 1).contiguous().transpose(0, 1),
                 torch.cat((do, do), -1)[..., 24:]):
        got = torch.autograd.grad(out, leaves, dout, retain_graph=True)
        plain = torch.autograd.grad(out, leaves, dout.contiguous(), retain_graph=True)
        assert all(torch.equal(a, b) for a, b in zip(got, plain))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_decay_keeps_what_is_not_finite_where_it_belongs(dtype):
    """A value, key or query that is not finite reaches its own and later tokens of
    its episode alone, its console and its head alone; a state that is not finite
    ends with the episode."""
    from nesle_amd import memory

    say(f"[gpu] decay_attention not finite {dtype}")
    x, _, _ = make(140, 4, 1, 2, 32, 32, dtype, 12)
    resets = torch.zeros(140, 4, dtype=torch.bool)
    resets[100, 0] = resets[70, 1] = resets[30, 2] = resets[5, 3] = True
    clean = {n: x[n].to(dev()) for n in NAMES}
    want, after = memory.decay_attention(*(clean[n] for n in NAMES[:4]), state=clean["state"], resets=resets.to(dev()))
    for bad in (math.nan, math.inf, -math.inf):
        x2 = {n: t.clone() for n, t in x.items()}
        x2["v"][40, 0, 1, 3] = bad
        x2["k"][66, 1, 0, 5] = bad
        x2["state"][2] = bad
        x2["q"][90, 3] = bad
        gpu = {n: x2[n].to(dev()) for n in NAMES}
        got, state = memory.decay_attention(*(gpu[n] for n in NAMES[:4]), state=gpu["state"], resets=resets.to(dev()))
        same = torch.ones(140, 4, 2, dtype=torch.bool)
        same[40:100, 0, 1] = same[66:70, 1] = same[:30, 2] = same[90, 3] = False
        # A chunk that is cut adds its sums in another order.
        a, b = got.float().cpu()[same], want.float().cpu()[same]
        assert bool(a.isfinite().all()), bad
        assert float((a - b).norm() / b.norm()) <= tol(dtype) + (0 if dtype == torch.float32 else 2.0 ** -9), bad
        assert off(state, after.double().cpu()) <= F32, bad
        for t, n, h in ((40, 0, 1), (99, 0, 1), (66, 1, 0), (66, 1, 1), (0, 2, 0), (29, 2, 1), (90, 3, 0)):
            assert not bool(got[t, n, h].isfinite().all()), (bad, t, n, h)
        # Once the sums are over it the rest of the head's row is as before.
        rest = [c for c in range(32) if c != 3]
        assert bool(got[40:100, 0, 1][:, rest].isfinite().all())


# ---- layer norm -----------------------------------------------------------------------

DIMS = [1, 2, 7, 8, 16, 40, 64, 128, 136, 201, 256, 257, 500, 512, 1000, 1024, 1600, 2048, 2500, 4096, 5000, 8192, 9000, 16384]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dim", DIMS)
def test_layer_norm_matches_the_definition(dim, dtype):
    from nesle_amd import memory

    rows = (3, 7) if dim > 1024 else (5, 43)
    say(f"[gpu] layer_norm {rows} x {dim} {dtype}")
    gen = torch.Generator().manual_seed(dim)
    x = ((torch.randn(*rows, dim, generator=gen) + torch.randn(*rows, 1, generator=gen)) *
         (0.1 + 3 * torch.rand(*rows, 1, generator=gen))).to(dtype)
    w, b = 1 + 0.3 * torch.randn(dim, generator=gen), 0.3 * torch.randn(dim, generator=gen)
    dy = torch.randn(*rows, dim, generator=gen).to(dtype)
    for has_w, has_b in ((True, True), (False, False), (True, False), (False, True)):
        args = [x, w if has_w else None, b if has_b else None]
        ref = [None if t is None else t.double().requires_grad_() for t in args]
        gpu = [None if t is None else t.to(dev()).requires_grad_() for t in args]
        want, got = O.layer_norm(*ref, 1e-5), memory.layer_norm(*gpu)
        assert got.dtype == dtype and got.is_contiguous()
        dw = torch.autograd.grad(want, [t for t in ref if t is not None], dy.double())
        dg = torch.autograd.grad(got, [t for t in gpu if t is not None], dy.to(dev()))
        if dim == 1:           # nothing is left of a single element but the bias
            assert torch.equal(got.cpu().double(), want.detach().to(dtype).double()) and bool((dg[0] == 0).all())
            continue
        assert off(got, want) <= tol(dtype, NORM)
        # dx is rstd times the difference of d = dy w, its mean, and xh mean(d xh), each
        # of d's size: what rounds is 2^-24 of those, not of the difference, which with
        # few elements is far smaller (with two, xh is +-1 and all but eps cancels).
        terms = dy.double() * (1.0 if args[1] is None else w.double()) / torch.sqrt(x.double().var(-1, correction=0, keepdim=True) + 1e-5)
        error = off(dg[0], dw[0]) * float(dw[0].norm())
        assert error <= 4 * NORM * float(terms.norm()) + (0 if dtype == torch.float32 else 2.0 ** -9 * float(dw[0].norm()))
        for a, t in zip(dg[1:], dw[1:]):
            assert a.dtype == torch.float32 and off(a, t) <= F32


def test_layer_norm_of_a_large_level():
    """A level 4,096 times the spread: the mean is found first, so the deviations keep
    the bits that float32 inputs have of them, 12 fewer than 24."""
    from nesle_amd import memory

    say("[gpu] layer_norm of a large level")
    gen = torch.Generator().manual_seed(2)
    x = torch.randn(64, 256, generator=gen) + 4096.0
    got = memory.layer_norm(x.to(dev()))
    assert off(got, O.layer_norm(x, None, None, 1e-5)) <= 2.0 ** -12
    flat = torch.full((4, 256), 3.0, device=dev())
    assert bool((memory.layer_norm(flat) == 0.0).all())


def test_layer_norm_rows():
    """One to four dimensions, none of them rows, strided rows, many rows; rows that are
    not finite spoil no other."""
    from nesle_amd import memory

    say("[gpu] layer_norm rows")
    gen = torch.Generator().manual_seed(3)
    x = torch.randn(3, 5, 4, 64, generator=gen, ).to(dev())
    w, b = torch.randn(64, generator=gen).to(dev()), torch.randn(64, generator=gen).to(dev())
    want = memory.layer_norm(x, w, b)
    assert torch.equal(memory.layer_norm(x[0, 0, 0], w, b), want[0, 0, 0])
    assert torch.equal(memory.layer_norm(x[0, 0], w, b), want[0, 0])
    assert torch.equal(memory.layer_norm(x[0], w, b), want[0])
    for turned in (x.transpose(0, 1), x.transpose(1, 2), x.permute(2, 0, 1, 3)):
        assert torch.equal(memory.layer_norm(turned, w, b), memory.layer_norm(turned.contiguous(), w, b))
    wide = torch.randn(3, 5, 4, 200, generator=gen).to(dev())
    for cut in (0, 1, 8):
        part = wide[..., cut:cut + 64]
        assert off(memory.layer_norm(part, w, b), memory.layer_norm(part.contiguous(), w, b).double().cpu()) <= NORM
    assert torch.equal(memory.layer_norm(x[:, :1].expand(3, 5, 4, 64), w, b)[:, 3], want[:, 0])
    for shape in ((0, 64), (3, 0, 64), (0, 2, 3, 64)):
        leaf, lw, lb = (torch.zeros(s, device=dev(), requires_grad=True) for s in (shape, 64, 64))
        y = memory.layer_norm(leaf, lw, lb)
        assert y.shape == shape
        d = torch.autograd.grad(y.sum(), (leaf, lw, lb))
        assert d[0].shape == shape and bool((d[1] == 0).all()) and bool((d[2] == 0).all())
    spoiled = x.clone()
    spoiled[1, 2, 3, 7] = math.nan
    spoiled[2, 0, 0, 0] = math.inf
    got = memory.layer_norm(spoiled, w, b)
    keep = torch.ones(3, 5, 4, dtype=torch.bool)
    keep[1, 2, 3] = keep[2, 0, 0] = False
    assert torch.equal(got[keep], want[keep]) and not bool(got[1, 2, 3].isfinite().any())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_layer_norm_weight_gradients_over_many_rows(dtype):
    """Over 70,001 rows with a gradient of one sign, so that the sums are long and do
    not cancel.  Each lane adds up at most 100 rows and a fixed tree the rest: about
    120 roundings of one sign at worst, 120 x 2^-24 = 7e-6 of the sum."""
    from nesle_amd import memory

    say(f"[gpu] layer_norm many rows {dtype}")
    gen = torch.Generator(device=dev()).manual_seed(4)
    x = torch.randn(70001, 96, generator=gen, device=dev()).to(dtype).requires_grad_()
    w, b = torch.ones(96, device=dev(), requires_grad=True), torch.zeros(96, device=dev(), requires_grad=True)
    dy = torch.rand(70001, 96, generator=gen, device=dev()).to(dtype)
    y = memory.layer_norm(x, w, b)
    first = torch.autograd.grad(y, (x, w, b), dy, retain_graph=True)
    xd = x.detach().double().cpu().requires_grad_()
    ref = O.layer_norm(xd, w.detach().double().cpu().requires_grad_(), None, 1e-5)
    xh = ref.detach()
    assert off(first[1], (dy.double().cpu() * xh).sum(0)) <= 7e-6 * float((dy.double().cpu() * xh).abs().sum(0).norm() / (dy.double().cpu() * xh).sum(0).norm())
    assert off(first[2], dy.double().cpu().sum(0)) <= 7e-6
    again = torch.autograd.grad(y, (x, w, b), dy)
    assert all(torch.equal(a, c) for a, c in zip(first, again))


# ---- sampling ---------------------------------------------------------------------------

def check_sample(logits, uniform, move=lambda t: t.to(dev()), **how):
    from nesle_amd import memory

    actions, logprobs = memory.sample_actions(move(logits), uniform.to(dev()),
                                              **{n: v.to(dev()) if torch.is_tensor(v) else v for n, v in how.items()})
    assert actions.dtype == torch.int64 and logprobs.dtype == torch.float32
    assert actions.shape == uniform.shape == logprobs.shape
    rows, count = logits.double().reshape(-1, logits.shape[-1]).tolist(), uniform.numel()
    settings = [{n: (v.double().reshape(-1)[i].item() if n != "top_k" else int(v.reshape(-1)[i])) if torch.is_tensor(v) else v
                 for n, v in how.items()} for i in range(count)]
    want = [O.sample(row, u, **s) for row, u, s in zip(rows, uniform.double().reshape(-1).tolist(), settings)]
    got = list(zip(actions.reshape(-1).tolist(), logprobs.reshape(-1).tolist()))
    for i, ((a, p), (b, q)) in enumerate(zip(got, want)):
        assert a == b, (i, a, b, settings[i])
        assert (math.isnan(p) and math.isnan(q)) or abs(p - q) <= 2.0 ** -24 * abs(q) + 1e-13, (i, p, q)
    return actions, logprobs


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("count", [1, 2, 5, 7, 12, 16, 17, 64, 65, 100, 256, 257, 1000, 1024])
def test_sampling_matches_the_definition(count, dtype):
    say(f"[gpu] sample_actions {count} {dtype}")
    gen = torch.Generator().manual_seed(count)
    n = 33 if count > 256 else 101
    logits = (2 * torch.randn(n, count, generator=gen)).to(dtype)
    u = torch.rand(n, generator=gen)
    for how in ({}, {"temperature": 0.6}, {"top_k": 1}, {"top_k": 3}, {"top_k": count}, {"top_k": 10 ** 9}, {"top_p": 0.9},
                {"top_p": 0.3}, {"top_p": 1e-6}, {"min_p": 0.1}, {"min_p": 1.0}, {"temperature": 0.0},
                {"temperature": 1.7, "top_k": max(1, count // 2), "top_p": 0.8, "min_p": 0.05}):
        check_sample(logits, u, **how)


def test_sampling_of_equal_logits():
    """Equal scores: the lowest index first, at every border.  12 equal weights of 1
    have whole sums, so the borders are exact."""
    say("[gpu] sample_actions equal logits")
    u = torch.tensor([0.0, 0.25, 0.5, 0.75, 0.999, 1.0 - 2.0 ** -24])
    for count in (12, 96, 768):
        logits = torch.full((6, count), -3.5)
        for how in ({}, {"top_k": 4}, {"top_p": 0.5}, {"top_k": 8, "top_p": 0.5}, {"min_p": 1.0}, {"temperature": 0.0}):
            check_sample(logits, u, **how)
        logits[:, count // 3:] += 1.0
        logits[:, 0] = 0.0
        logits[:, 5] = -0.0
        check_sample(logits, u, top_k=3)
        check_sample(logits, u, temperature=0.0)


def test_sampling_of_masked_rows():
    """Actions masked with -inf or the type's lowest value; rows with nothing left, NaN,
    +inf; numbers on and past the ends of their range."""
    say("[gpu] sample_actions masks")
    gen = torch.Generator().manual_seed(6)
    for dtype in (torch.float32, torch.bfloat16):
        for count in (12, 100, 300):
            logits = torch.randn(14, count, generator=gen).to(dtype)
            logits[0, ::2] = -math.inf
            logits[1, 1:] = -math.inf
            logits[2] = -math.inf
            logits[3, 4] = math.nan
            logits[4, 5] = math.inf
            logits[5, :-1] = torch.finfo(dtype).min
            logits[6] = torch.finfo(dtype).min
            logits[7, 0] = torch.finfo(dtype).max
            u = torch.rand(14, generator=gen)
            u[8], u[9], u[10], u[11], u[12], u[13] = 0.0, 1.0, -3.0, math.nan, 7.0, math.inf
            for how in ({}, {"top_k": 2}, {"top_p": 0.7}, {"min_p": 0.2}, {"temperature": 0.0}, {"temperature": 1e-30}):
                if how.get("temperature") == 0.0:
                    u = torch.where(u.isnan(), 0.5, u)      # the oracle's rows without an answer are those of the logits
                check_sample(logits, u, **how)


def test_sampling_with_settings_of_each_row():
    from nesle_amd import memory

    say("[gpu] sample_actions settings")
    gen = torch.Generator().manual_seed(7)
    logits, u = torch.randn(4, 50, 30, generator=gen), torch.rand(4, 50, generator=gen)
    how = {"temperature": 0.2 + torch.rand(4, 50, generator=gen), "top_k": torch.randint(0, 32, (4, 50), generator=gen).to(torch.int32),
           "top_p": 0.3 + 0.7 * torch.rand(4, 50, generator=gen), "min_p": 0.2 * torch.rand(4, 50, generator=gen)}
    how["temperature"][0, :5] = 0.0
    how["top_p"][1, :5] = 1.0
    check_sample(logits, u, **how)
    # Another order of the leading dimensions, rows of a wider tensor.
    a = memory.sample_actions(logits.to(dev()), u.to(dev()))
    wide = torch.zeros(50, 4, 40, device=dev())
    wide[..., 3:33] = logits.transpose(0, 1).to(dev())
    b = memory.sample_actions(wide.transpose(0, 1)[..., 3:33], u.to(dev()))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    # A setting out of its range has no answer, in its row alone.
    for name, bad in (("temperature", (-1.0, math.nan, math.inf)), ("top_p", (0.0, 1.5, math.nan)), ("min_p", (-0.1, 1.1, math.nan)),
                      ("top_k", (-1,))):
        for value in bad:
            mine = {n: t.clone() for n, t in how.items()}
            mine[name][2, 7] = value
            actions, logprobs = memory.sample_actions(logits.to(dev()), u.to(dev()), **{n: t.to(dev()) for n, t in mine.items()})
            assert int(actions[2, 7]) == -1 and math.isnan(float(logprobs[2, 7]))
            assert int((actions == -1).sum()) == 1 and int(logprobs.isnan().sum()) == 1
    empty = memory.sample_actions(torch.zeros(0, 5, device=dev()), torch.zeros(0, device=dev()))
    assert empty[0].shape == (0,) and empty[1].shape == (0,)


def test_sampling_is_the_distribution():
    """Evenly spread numbers take every action as often as its probability says, to
    one number."""
    from nesle_amd import memory

    say("[gpu] sample_actions distribution")
    gen = torch.Generator().manual_seed(8)
    n = 1 << 16
    row = torch.randn(12, generator=gen)
    u = (torch.arange(n, dtype=torch.float64) + 0.5) / n
    actions, _ = memory.sample_actions(row.to(dev()).expand(n, 12), u.float().to(dev()))
    share = torch.bincount(actions.cpu(), minlength=12).double()
    assert float((share - n * torch.softmax(row.double(), 0)).abs().max()) <= 1.0
