"""The memory operators (nesle_amd.memory) on the GPU against their definition
in float64 (tests/memory_oracle.py).

Tolerances, on the 2-norm of the difference over the 2-norm of the result.
Float32: a result goes through a few sums of at most 128 products, each
rounding 2^-24 relative to a running sum of which about sqrt(128) random ones
add up (7e-7), over up to a handful of stages that the decays keep from
growing: 4e-6.  bfloat16: compared with the definition rounded to bfloat16,
from which one rounding of the float32 result differs in the few elements that
the float32 error carries over a rounding boundary: 2^-9 on top of it."""

from __future__ import annotations

import pytest
import torch

from tests import memory_oracle as O
from tests.helpers import say

pytestmark = pytest.mark.gpu

F32 = 4e-6


def tol(dtype) -> float:
    return F32 if dtype == torch.float32 else 2.0 ** -9 + F32


def dev():
    return torch.device("cuda")


# ---- gated delta rule ----------------------------------------------------------------

def make(T, N, hk, hv, dk, dv, dtype, seed, resets=0.1, alike=0.7):
    """Inputs on the CPU: unit queries and keys (neighbouring tokens alike),
    gates, an initial state, resets, gradients."""
    gen = torch.Generator().manual_seed(seed)
    base = torch.randn(2, N, hk, dk, generator=gen)

    def unit(i):
        x = torch.randn(T, N, hk, dk, generator=gen) * (1 - alike) + base[i] * alike
        return (x / x.norm(dim=-1, keepdim=True)).to(dtype)

    x = {"q": unit(0), "k": unit(1), "v": torch.randn(T, N, hv, dv, generator=gen).to(dtype),
         "g": -0.2 * torch.rand(T, N, hv, generator=gen), "beta": torch.rand(T, N, hv, generator=gen),
         "state": torch.randn(N, hv, dk, dv, generator=gen)}
    resets = torch.rand(T, N, generator=gen) < resets
    grads = torch.randn(T, N, hv, dv, generator=gen).to(dtype), torch.randn(N, hv, dk, dv, generator=gen)
    return x, resets, grads


NAMES = ("q", "k", "v", "g", "beta", "state")


def check_delta(x, resets, grads, scale=None, train=True, move=lambda t: t.to(dev())):
    """Forward and gradient against the definition."""
    from nesle_amd import memory

    dtype = x["q"].dtype
    s = x["q"].shape[-1] ** -0.5 if scale is None else scale
    ref = {n: None if x[n] is None else x[n].double().requires_grad_() for n in NAMES}
    want = O.delta(*(ref[n] for n in NAMES), resets, s)
    gpu = {n: None if x[n] is None else move(x[n]).requires_grad_(train) for n in NAMES}
    got = memory.gated_delta(gpu["q"], gpu["k"], gpu["v"], gpu["g"], gpu["beta"], state=gpu["state"],
                             resets=None if resets is None else resets.to(dev()), scale=scale)
    assert got[0].dtype == dtype and got[1].dtype == torch.float32
    assert O.off(got[0], want[0]) <= tol(dtype), "out"
    assert O.off(got[1], want[1]) <= F32, "state"
    if not train:
        return got
    names = [n for n in NAMES if x[n] is not None]
    dw = torch.autograd.grad(want, [ref[n] for n in names], [t.double() for t in grads], allow_unused=True)
    dg = torch.autograd.grad(got, [gpu[n] for n in names], [t.to(dev()) for t in grads])
    for n, a, b in zip(names, dg, dw):
        b = torch.zeros_like(ref[n]) if b is None else b
        assert a.dtype == x[n].dtype
        assert O.off(a, b) <= (tol(dtype) if n in "qkv" else F32), f"d{n}"
    return got


SHAPES = [(1, 1, 1, 1, 8, 8), (3, 2, 2, 2, 16, 24), (31, 2, 1, 1, 32, 32), (32, 1, 2, 4, 32, 16), (33, 3, 1, 3, 48, 40),
          (64, 2, 2, 2, 64, 64), (77, 3, 2, 4, 64, 24), (130, 2, 1, 1, 64, 64), (65, 2, 1, 2, 128, 128),
          (40, 1, 1, 1, 24, 104), (96, 1, 2, 2, 128, 64)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", SHAPES)
def test_delta_matches_the_definition(shape, dtype):
    say(f"[gpu] gated_delta {shape} {dtype}")
    check_delta(*make(*shape, dtype, seed=sum(shape)))


@pytest.mark.parametrize("where", ["none", "all", "first", "edges", "last"])
def test_delta_resets(where):
    say(f"[gpu] gated_delta resets {where}")
    x, resets, grads = make(70, 3, 1, 2, 32, 32, torch.float32, 5)
    resets[:] = where == "all"
    if where == "first":
        resets[0] = True
    if where == "last":
        resets[-1] = True
    if where == "edges":
        for n, t in enumerate((31, 32, 33)):
            resets[t, n] = True
            resets[t + 1, n] = n == 2
    check_delta(x, resets, grads)
    check_delta(x, None if where == "none" else resets.to(torch.uint8) * 255, grads)


@pytest.mark.parametrize("gate", ["zero", "strong", "off", "growing"])
def test_delta_gates(gate):
    """No decay; decays that leave nothing after a few tokens; gates of -inf and
    -200 among others (the state is dropped); gates above zero."""
    say(f"[gpu] gated_delta gates {gate}")
    x, resets, grads = make(70, 2, 1, 2, 32, 32, torch.float32, 6, resets=0.0)
    if gate == "zero":
        x["g"].zero_()
    elif gate == "strong":
        x["g"] = x["g"] * 250
    elif gate == "growing":
        x["g"] = x["g"] * -0.1
    else:
        x["g"][5, 0, 0], x["g"][40, 1, 1], x["g"][32, 0, 1] = -float("inf"), -200.0, -float("inf")
    check_delta(x, resets, grads)


def test_delta_equal_keys_and_full_writes():
    """One key for all tokens and beta 1, where powers of A reach thousands; and
    tokens that write nothing."""
    say("[gpu] gated_delta equal keys")
    x, resets, grads = make(96, 2, 1, 1, 64, 64, torch.float32, 7, resets=0.0, alike=1.0)
    x["beta"][:] = 1.0
    check_delta(x, resets, grads)
    x["beta"][:] = 0.0
    x["g"][:] = 0.0                                    # padding: the state comes out as it went in
    out, state = check_delta(x, resets, grads)
    assert torch.equal(state.cpu(), x["state"])


def test_delta_without_state_and_with_scale():
    say("[gpu] gated_delta without state")
    x, resets, grads = make(45, 2, 2, 2, 40, 40, torch.float32, 8)
    x["state"] = None
    check_delta(x, resets, grads, scale=1.0)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shift", [0, 1, 4])
def test_delta_strided_and_unaligned(dtype, shift):
    """Slices of one projection, from element 0, 1 (no aligned group of four)
    and 4 on, consoles and steps swapped in memory."""
    from nesle_amd import memory

    say(f"[gpu] gated_delta strided, shift {shift} {dtype}")
    T, N, hk, hv, dk, dv = 37, 3, 2, 2, 32, 40
    x, resets, _ = make(T, N, hk, hv, dk, dv, dtype, 9)
    wide = 2 * hk * dk + hv * dv + shift + 3
    buf = torch.zeros(N, T, wide, dtype=dtype, device=dev())
    at, cut = shift, {}
    for n in "qkv":
        size = x[n][0, 0].numel()
        cut[n] = buf[..., at:at + size].unflatten(-1, x[n].shape[-2:]).transpose(0, 1)
        cut[n].copy_(x[n])
        at += size
    g, beta, state = (x[n].to(dev()) for n in ("g", "beta", "state"))
    got = memory.gated_delta(cut["q"], cut["k"], cut["v"], g, beta, state=state, resets=resets.to(dev()))
    want = O.delta(*(x[n] for n in NAMES), resets, dk ** -0.5)
    assert O.off(got[0], want[0]) <= tol(dtype) and O.off(got[1], want[1]) <= F32
    out = memory.gated_delta_step(cut["q"][0], cut["k"][0], cut["v"][0], g[0], beta[0], state, resets=resets[0].to(dev()))
    want = O.delta(*(x[n][:1] for n in NAMES[:5]), x["state"], resets[:1], dk ** -0.5)
    assert O.off(out, want[0][0]) <= tol(dtype) and O.off(state, want[1]) <= F32


def test_delta_offsets_past_32_bits():
    """Queries, keys and values whose steps lie 2^31 elements apart."""
    from nesle_amd import memory

    say("[gpu] gated_delta wide strides")
    x, _, _ = make(3, 2, 1, 1, 32, 32, torch.bfloat16, 10)
    far = (1 << 31) + 64
    buf = torch.empty(2 * far + 4096, dtype=torch.bfloat16, device=dev())
    cut = {}
    for i, n in enumerate("qkv"):
        cut[n] = buf.as_strided(x[n].shape, (far, 32, 32, 1), 512 * i)
        cut[n].copy_(x[n])
    got = memory.gated_delta(cut["q"], cut["k"], cut["v"], x["g"].to(dev()), x["beta"].to(dev()), state=x["state"].to(dev()))
    want = O.delta(*(x[n] for n in NAMES), None, 32 ** -0.5)
    assert O.off(got[0], want[0]) <= tol(torch.bfloat16) and O.off(got[1], want[1]) <= F32


def test_delta_gradient_with_wide_strides():
    """Steps 2^26 elements apart: a chunk's rows span more than 2^31 bytes."""
    say("[gpu] gated_delta wide strides, gradient")
    far, T = (1 << 26) + 64, 34
    buf = torch.empty((T - 1) * far + 8192, dtype=torch.bfloat16, device=dev())
    x, resets, grads = make(T, 2, 1, 2, 32, 32, torch.bfloat16, 20)
    at = iter((0, 512, 1024))

    def move(t):
        if t.dim() != 4 or t.shape[0] != T:
            return t.to(dev())
        cut = buf.as_strided(t.shape, (far, t.shape[2] * t.shape[3], t.shape[3], 1), next(at))
        cut.copy_(t)
        return cut.detach()

    check_delta(x, resets, grads, move=move)


@pytest.mark.parametrize("far", [((1 << 31) - 4096) // 62 // 8 * 8, ((1 << 31) - 4096) // 62 // 8 * 8 + 8])
def test_delta_gradient_at_the_last_32_bit_stride(far):
    """The largest steps whose chunks' rows a 32-bit offset reaches, and the next."""
    say(f"[gpu] gated_delta steps of {far} elements, gradient")
    buf = torch.empty(33 * far + 8192, dtype=torch.bfloat16, device=dev())
    x, resets, grads = make(34, 2, 1, 2, 32, 32, torch.bfloat16, 30)
    at = iter((0, 512, 1024))

    def move(t):
        if t.dim() != 4 or t.shape[0] != 34:
            return t.to(dev())
        cut = buf.as_strided(t.shape, (far, t.shape[2] * t.shape[3], t.shape[3], 1), next(at))
        cut.copy_(t)
        return cut.detach()

    check_delta(x, resets, grads, move=move)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape,resets", [((513, 1, 1, 1, 64, 64), 0.0), ((1025, 2, 1, 2, 32, 24), 0.004),
                                          ((700, 1, 2, 2, 128, 128), 0.01), ((1500, 3, 1, 1, 16, 40), 0.5)])
def test_delta_few_heads_over_many_tokens(shape, resets, dtype):
    """Lengths at which the walk is cut into segments, with their gradient."""
    say(f"[gpu] gated_delta long {shape} {dtype}")
    check_delta(*make(*shape, dtype, seed=sum(shape), resets=resets))


def test_delta_segments_keep_what_is_not_finite():
    """A state of NaN, and tokens of NaN, end at the next reset also where it
    lies inside a later segment, and not before."""
    from nesle_amd import memory

    say("[gpu] gated_delta long, not finite")
    x, resets, _ = make(900, 2, 1, 1, 32, 32, torch.float32, 19, resets=0.0)
    clean = O.delta(*(x[n] for n in NAMES), resets, 32 ** -0.5)[0]
    resets[401, 0] = resets[777, 1] = True
    x["state"][0] = float("nan")
    x["k"][300, 1, 0, 0] = float("nan")
    got = memory.gated_delta(*(x[n].to(dev()) for n in NAMES[:5]), state=x["state"].to(dev()), resets=resets.to(dev()))
    out = got[0].cpu()
    y = {n: torch.where(torch.isfinite(t), t, torch.zeros_like(t)) for n, t in x.items()}
    want = O.delta(*(y[n] for n in NAMES), resets, 32 ** -0.5)[0]
    assert torch.isnan(out[:401, 0]).all() and O.off(out[401:, 0], want[401:, 0]) <= F32
    assert O.off(out[:300, 1], clean[:300, 1]) <= F32 and torch.isnan(out[300:777, 1]).all()
    assert O.off(out[777:, 1], want[777:, 1]) <= F32 and torch.isfinite(got[1]).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape,resets", [((6753, 1, 1, 1, 64, 64), 0.0), ((6760, 1, 1, 2, 32, 24), 0.002),
                                          ((6784, 2, 1, 1, 72, 128), 0.001)])
def test_delta_segments_in_groups(shape, resets, dtype):
    """Lengths whose segments are joined in groups, with their gradient."""
    say(f"[gpu] gated_delta in groups {shape} {dtype}")
    check_delta(*make(*shape, dtype, seed=sum(shape), resets=resets))


def test_delta_groups_keep_what_is_not_finite():
    """As above, with the resets in later groups of segments."""
    from nesle_amd import memory

    say("[gpu] gated_delta in groups, not finite")
    x, resets, _ = make(6800, 2, 1, 1, 32, 32, torch.float32, 23, resets=0.0)
    clean = O.delta(*(x[n] for n in NAMES), resets, 32 ** -0.5)[0]
    resets[4501, 0] = resets[6377, 1] = True
    x["state"][0] = float("nan")
    x["v"][2300, 1, 0, 7] = float("inf")
    got = memory.gated_delta(*(x[n].to(dev()) for n in NAMES[:5]), state=x["state"].to(dev()), resets=resets.to(dev()))
    out = got[0].cpu()
    y = {n: torch.where(torch.isfinite(t), t, torch.zeros_like(t)) for n, t in x.items()}
    want = O.delta(*(y[n] for n in NAMES), resets, 32 ** -0.5)[0]
    assert torch.isnan(out[:4501, 0]).all() and O.off(out[4501:, 0], want[4501:, 0]) <= F32
    assert O.off(out[:2300, 1], clean[:2300, 1]) <= F32 and not torch.isfinite(out[2300:6377, 1, 0, 7]).any()
    assert O.off(out[6377:, 1], want[6377:, 1]) <= F32 and torch.isfinite(got[1]).all()


def test_delta_gradient_of_a_state_that_starts_anywhere():
    """The state's gradient may come as a slice of a longer one, off every
    boundary: the same as by itself."""
    from nesle_amd import memory

    say("[gpu] gated_delta gradient of a slice")
    x, resets, grads = make(40, 2, 1, 2, 24, 16, torch.float32, 29)
    gpu = [x[n].to(dev()).requires_grad_() for n in NAMES]
    out, state = memory.gated_delta(*gpu[:5], state=gpu[5], resets=resets.to(dev()))
    whole = torch.cat((out.flatten()[:3], state.flatten()))
    weight = torch.cat((torch.zeros(3), grads[1].flatten())).to(dev())
    got = torch.autograd.grad(whole, gpu, weight, retain_graph=True)
    want = torch.autograd.grad((out, state), gpu, (torch.zeros_like(out), grads[1].to(dev())))
    for n, a, b in zip(NAMES, got, want):
        assert torch.equal(a, b), n


def test_delta_gradient_against_differences():
    """The kernel's gradient along a direction against central differences of
    the float64 definition: their own error is about h^2 = 1e-8 and 1e-16 / h =
    1e-12, so what is left is the kernel's."""
    from nesle_amd import memory

    say("[gpu] gated_delta gradient against differences")
    x, resets, grads = make(50, 2, 1, 2, 24, 16, torch.float32, 11)
    gpu = [x[n].to(dev()).requires_grad_() for n in NAMES]
    got = memory.gated_delta(*gpu[:5], state=gpu[5], resets=resets.to(dev()))
    d = torch.autograd.grad(got, gpu, [t.to(dev()) for t in grads])
    gen, h = torch.Generator().manual_seed(12), 1e-4
    for i, n in enumerate(NAMES):
        way = torch.randn(x[n].shape, generator=gen, dtype=torch.float64)

        def loss(step):
            y = [x[m].double() + (step * way if m == n else 0) for m in NAMES]
            out, state = O.delta(*y, resets, 24 ** -0.5)
            return float((out * grads[0].double()).sum() + (state * grads[1].double()).sum())

        want = (loss(h) - loss(-h)) / (2 * h)
        have = float((d[i].double().cpu() * way).sum())
        # relative to the size such a sum of random signs has
        size = float(d[i].double().norm())
        assert abs(have - want) <= 2e-5 * size, n


def test_delta_what_is_not_finite_stays_where_it_belongs():
    """A state of NaN ends at a reset; a NaN or infinite token reaches neither
    earlier tokens, nor other consoles, nor the next episode."""
    from nesle_amd import memory

    say("[gpu] gated_delta not finite")
    x, resets, _ = make(70, 4, 1, 1, 32, 32, torch.float32, 13, resets=0.0)
    clean = O.delta(*(x[n] for n in NAMES), resets, 32 ** -0.5)[0]
    resets[0, 0] = True
    x["state"][0] = float("nan")
    x["v"][20, 1, 0, 3] = float("nan")
    x["k"][41, 2, 0, 5] = float("inf")
    resets[50, 1], resets[45, 2] = True, True
    x["beta"][10, 3], x["g"][12, 3], resets[13, 3] = float("nan"), float("nan"), True
    got = memory.gated_delta(*(x[n].to(dev()) for n in NAMES[:5]), state=x["state"].to(dev()), resets=resets.to(dev()))
    out = got[0].cpu()
    # what the values would be if nothing but the resets had happened
    y = {n: torch.where(torch.isfinite(t), t, torch.zeros_like(t)) for n, t in x.items()}
    want = O.delta(*(y[n] for n in NAMES), resets, 32 ** -0.5)[0]
    assert O.off(out[:, 0], want[:, 0]) <= F32
    assert O.off(out[:20, 1], clean[:20, 1]) <= F32 and O.off(out[50:, 1], want[50:, 1]) <= F32
    assert O.off(out[:41, 2], clean[:41, 2]) <= F32 and O.off(out[45:, 2], want[45:, 2]) <= F32
    assert O.off(out[:10, 3], clean[:10, 3]) <= F32 and O.off(out[13:, 3], want[13:, 3]) <= F32
    assert torch.isnan(out[20:50, 1, 0, 3]).all() and torch.isnan(out[10:13, 3]).all()
    assert torch.isfinite(got[1]).all()


@pytest.mark.parametrize("T,N", [(0, 3), (4, 0), (0, 0)])
def test_delta_empty(T, N):
    from nesle_amd import memory

    x, resets, grads = make(T, N, 1, 2, 16, 16, torch.float32, 14)
    gpu = [x[n].to(dev()).requires_grad_() for n in NAMES]
    out, state = memory.gated_delta(*gpu[:5], state=gpu[5], resets=resets.to(dev()))
    assert out.shape == (T, N, 2, 16) and torch.equal(state.cpu(), x["state"])
    d = torch.autograd.grad((out, state), gpu, [t.to(dev()) for t in grads])
    assert torch.equal(d[5].cpu(), grads[1])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [(1, 1, 1, 8, 8), (1, 4, 4, 64, 64), (7, 3, 6, 48, 40), (130, 2, 2, 128, 128),
                                   (5, 1, 1, 16, 104), (2000, 4, 4, 64, 64)])
def test_delta_step_matches_the_definition(shape, dtype):
    from nesle_amd import memory

    say(f"[gpu] gated_delta_step {shape} {dtype}")
    N, hk, hv, dk, dv = shape
    x, resets, _ = make(1, N, hk, hv, dk, dv, dtype, 15)
    if N > 2:
        x["g"][0, 1] = -float("inf")
        x["state"][1] = float("nan")                   # dropped, so it does not matter
        resets[0, 2], x["state"][2] = True, float("inf")
    state = x["state"].to(dev())
    out = memory.gated_delta_step(*(x[n][0].to(dev()) for n in NAMES[:5]), state, resets=resets[0].to(dev()))
    if N > 2:
        x["state"][1:3] = 0.0
    want = O.delta(*(x[n] for n in NAMES), resets, dk ** -0.5)
    assert out.dtype == dtype
    assert O.off(out, want[0][0]) <= tol(dtype) and O.off(state, want[1]) <= F32


def test_delta_steps_make_the_rollout():
    """Acting token by token gives the outputs and states that training sees."""
    from nesle_amd import memory

    say("[gpu] gated_delta_step by step")
    x, resets, _ = make(70, 3, 2, 4, 64, 32, torch.float32, 16)
    gpu = [x[n].to(dev()) for n in NAMES]
    out, after = memory.gated_delta(*gpu[:5], state=gpu[5], resets=resets.to(dev()))
    state = gpu[5].clone()
    for t in range(70):
        o = memory.gated_delta_step(*(y[t] for y in gpu[:5]), state, resets=resets[t].to(dev()))
        assert O.off(o, out[t].cpu()) <= 2 * F32, t
    assert O.off(state, after.cpu()) <= 2 * F32


# ---- norm and rotation -----------------------------------------------------------------

def make_rotate(lead, hq, hk, dim, rotated, dtype, seed, weights=(True, True), rows=50):
    gen = torch.Generator().manual_seed(seed)
    q, k, dq, dk = (torch.randn(*lead, h, dim, generator=gen).to(dtype) for h in (hq, hk, hq, hk))
    wq, wk = (1 + 0.3 * torch.randn(dim, generator=gen) if w else None for w in weights)
    table = pos = None
    if rotated:
        from nesle_amd import memory

        table = memory.rotation_table(rows, rotated, device="cpu")
        pos = torch.randint(0, rows, lead, generator=gen, dtype=torch.int32)
    return q, k, wq, wk, pos, table, dq, dk


def check_rotate(q, k, wq, wk, pos, table, dq, dk, eps=1e-6, unit=False, interleaved=False, place=lambda t: t.to(dev())):
    from nesle_amd import memory

    dtype = q.dtype
    leaves = [None if t is None else place(t).requires_grad_() for t in (q, k, wq, wk)]
    where = [None if t is None else t.to(dev()) for t in (pos, table)]
    got = memory.qk_norm_rotate(*leaves, positions=where[0], table=where[1], eps=eps, unit=unit, interleaved=interleaved)
    ref = [None if t is None else t.double().requires_grad_() for t in (q, k, wq, wk)]
    want = [O.rotate(x, w, pos, table, eps, unit, interleaved) for x, w in zip(ref[:2], ref[2:])]
    for a, b, n in zip(got, want, "qk"):
        assert a.dtype == dtype and O.off(a, b) <= tol(dtype), n
    used = [i for i in range(4) if leaves[i] is not None]
    dw = torch.autograd.grad(want, [ref[i] for i in used], [dq.double(), dk.double()])
    dg = torch.autograd.grad(got, [leaves[i] for i in used], [dq.to(dev()), dk.to(dev())])
    for i, a, b in zip(used, dg, dw):
        assert O.off(a, b) <= (tol(dtype) if i < 2 else F32), ("dq", "dk", "dwq", "dwk")[i]


ROTATE = [((1,), 1, 1, 8, 8), ((5,), 4, 4, 64, 64), ((3, 7), 6, 2, 40, 16), ((2, 33), 3, 3, 48, 0), ((9, 4), 2, 1, 256, 128),
          ((4, 5), 1, 3, 80, 80), ((300, 70), 4, 4, 64, 64), ((11, 1), 16, 2, 128, 64)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("unit,interleaved", [(False, False), (True, True)])
@pytest.mark.parametrize("shape", ROTATE)
def test_rotate_matches_the_definition(shape, unit, interleaved, dtype):
    say(f"[gpu] qk_norm_rotate {shape} unit={unit} interleaved={interleaved} {dtype}")
    check_rotate(*make_rotate(*shape, dtype, sum(shape[1:])), unit=unit, interleaved=interleaved)


@pytest.mark.parametrize("weights", [(True, False), (False, True), (False, False)])
def test_rotate_weights(weights):
    say(f"[gpu] qk_norm_rotate weights {weights}")
    check_rotate(*make_rotate((6, 5), 2, 3, 24, 24, torch.float32, 3, weights=weights))


@pytest.mark.parametrize("shift", [1, 2, 4])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rotate_strided_and_unaligned(shift, dtype):
    say(f"[gpu] qk_norm_rotate shift {shift} {dtype}")

    def place(t):
        if t.dim() == 1:
            return t.to(dev())
        n = t[0, 0].numel()
        buf = torch.zeros(t.shape[1], t.shape[0], n + shift + 5, dtype=t.dtype, device=dev())
        cut = buf[..., shift:shift + n].unflatten(-1, t.shape[-2:]).transpose(0, 1)
        cut.copy_(t)
        return cut

    check_rotate(*make_rotate((6, 5), 2, 3, 24, 16, dtype, 4), place=place)


def test_rotate_zero_rows_and_large_values():
    """A head of zeros comes out zero (eps holds it), and values whose squares
    stay in float32's range come out of norm 1."""
    say("[gpu] qk_norm_rotate zero rows")
    q, k, wq, wk, pos, table, dq, dk = make_rotate((4, 3), 2, 2, 32, 32, torch.float32, 5)
    q[0, 0, 0] = 0.0
    k[1] *= 1e15
    check_rotate(q, k, wq, wk, pos, table, dq, dk, eps=1e-3, unit=True)


def test_rotate_position_outside_the_table():
    from nesle_amd import memory

    say("[gpu] qk_norm_rotate positions outside")
    q, k, wq, wk, pos, table, dq, dk = (None if t is None else t.to(dev())
                                        for t in make_rotate((6, 5), 2, 2, 32, 16, torch.float32, 6))
    pos[0, 0], pos[3, 2] = -1, 50
    q.requires_grad_()
    got = memory.qk_norm_rotate(q, k, positions=pos, table=table)
    bad = torch.zeros(6, 5, dtype=torch.bool, device=dev())
    bad[0, 0] = bad[3, 2] = True
    for out in got:
        assert torch.isnan(out[bad][..., :16]).all() and torch.isfinite(out[~bad]).all()
    (d,) = torch.autograd.grad(got, [q], [dq, dk])
    assert torch.isnan(d[bad]).all() and torch.isfinite(d[~bad]).all()


def test_rotate_gradient_against_differences():
    from nesle_amd import memory

    say("[gpu] qk_norm_rotate gradient against differences")
    q, k, wq, wk, pos, table, dq, dk = make_rotate((5, 4), 2, 1, 40, 24, torch.float32, 7)
    leaves = [t.to(dev()).requires_grad_() for t in (q, k, wq, wk)]
    got = memory.qk_norm_rotate(*leaves, positions=pos.to(dev()), table=table.to(dev()))
    d = torch.autograd.grad(got, leaves, [dq.to(dev()), dk.to(dev())])
    gen, h = torch.Generator().manual_seed(8), 1e-4
    for i, x in enumerate((q, k, wq, wk)):
        way = torch.randn(x.shape, generator=gen, dtype=torch.float64)

        def loss(step):
            y = [t.double() + (step * way if j == i else 0) for j, t in enumerate((q, k, wq, wk))]
            outs = [O.rotate(y[j], y[2 + j], pos, table, 1e-6, False, False) for j in range(2)]
            return float((outs[0] * dq.double()).sum() + (outs[1] * dk.double()).sum())

        want = (loss(h) - loss(-h)) / (2 * h)
        assert abs(float((d[i].double().cpu() * way).sum()) - want) <= 2e-5 * float(d[i].double().norm()), i


@pytest.mark.parametrize("lead", [(0,), (0, 4), (4, 0)])
def test_rotate_empty(lead):
    from nesle_amd import memory

    q, k, wq, wk, pos, table, dq, dk = (None if t is None else t.to(dev())
                                        for t in make_rotate(lead, 2, 2, 16, 16, torch.float32, 9))
    leaves = [t.requires_grad_() for t in (q, k, wq, wk)]
    got = memory.qk_norm_rotate(*leaves, positions=pos, table=table)
    assert got[0].shape == q.shape
    d = torch.autograd.grad(got, leaves, [dq, dk])
    assert float(d[2].abs().sum()) == 0.0 and float(d[3].abs().sum()) == 0.0


# ---- streams, graphs, repeatability, refusals ----------------------------------------------

def _layer(memory, x, resets, pos, table):
    """Both operators as a layer uses them, forward and gradient."""
    leaves = [t.detach().requires_grad_() for t in x]
    q, k, v, g, beta, state = leaves
    q, k = memory.qk_norm_rotate(q, k, positions=pos, table=table, unit=True)
    out, after = memory.gated_delta(q, k, v, g, beta, state=state, resets=resets)
    grads = torch.autograd.grad((out.float().square().sum() + after.square().sum()), leaves)
    return [out.detach(), after.detach(), *grads]


def _layer_inputs(dtype=torch.bfloat16):
    from nesle_amd import memory

    x, resets, _ = make(50, 5, 2, 4, 32, 32, dtype, 17)
    pos = torch.randint(0, 50, (50, 5), dtype=torch.int32, generator=torch.Generator().manual_seed(1))
    return [x[n].to(dev()) for n in NAMES], resets.to(dev()), pos.to(dev()), memory.rotation_table(50, 32)


def test_same_bits_every_time_and_on_another_stream():
    from nesle_amd import memory

    say("[gpu] memory operators: repeatability, another stream")
    args = _layer_inputs()
    first = _layer(memory, *args)
    again = _layer(memory, *args)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        other = _layer(memory, *args)
    side.synchronize()
    for a, b, c in zip(first, again, other):
        assert torch.equal(a, b) and torch.equal(a, c)


def test_captured_in_a_graph():
    """A captured layer replays to the eager result, on new inputs too, with
    eager work between the replays."""
    from nesle_amd import memory

    say("[gpu] memory operators: graph")
    x, resets, pos, table = _layer_inputs()
    step_state = x[5].clone()

    def work():
        q, k = memory.qk_norm_rotate(x[0], x[1], positions=pos, table=table, unit=True)
        out, after = memory.gated_delta(q, k, *x[2:5], state=x[5], resets=resets)
        one = memory.gated_delta_step(q[0], k[0], x[2][0], x[3][0], x[4][0], step_state, resets=resets[0])
        return out, after, one

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        captured = work()
    for i in range(4):
        x[2].copy_(torch.randn(x[2].shape, generator=torch.Generator().manual_seed(i)))
        step_state.copy_(x[5])
        want = [t.clone() for t in work()]
        step_state.copy_(x[5])
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(captured, want):
            assert torch.equal(a, b), i


def test_only_first_derivatives():
    """The gradient's own gradient is refused where it is asked for; a backward
    that keeps its graph for other reasons works."""
    from nesle_amd import memory

    x, resets, _ = make(4, 2, 1, 1, 16, 16, torch.float32, 21)
    q, k, v, g, beta = (x[n].to(dev()).requires_grad_() for n in NAMES[:5])
    w = torch.tensor(2.0, device=dev(), requires_grad=True)
    for out in (memory.gated_delta(q, k, v, g, beta)[0], memory.qk_norm_rotate(q, k)[0]):
        (d,) = torch.autograd.grad((out * w).square().sum(), [q], create_graph=True)
        with pytest.raises(RuntimeError, match="second derivative"):
            d.sum().backward()


def test_unused_outputs_have_no_gradient():
    """A loss that takes only the output, or only the state."""
    from nesle_amd import memory

    x, resets, grads = make(40, 2, 1, 2, 24, 16, torch.float32, 22)
    for used in range(2):
        ref = [x[n].double().requires_grad_() for n in NAMES]
        want = O.delta(*ref, resets, 24 ** -0.5)[used]
        dw = torch.autograd.grad(want, ref, grads[used].double(), allow_unused=True)
        gpu = [x[n].to(dev()).requires_grad_() for n in NAMES]
        got = memory.gated_delta(*gpu[:5], state=gpu[5], resets=resets.to(dev()))[used]
        dg = torch.autograd.grad(got, gpu, grads[used].to(dev()))
        for n, a, b in zip(NAMES, dg, dw):
            assert O.off(a, torch.zeros(a.shape, dtype=torch.float64) if b is None else b) <= F32, (used, n)


def test_step_marks_the_state_as_changed():
    """A state that a graph saved and a step then overwrote is noticed."""
    from nesle_amd import memory

    x, _, _ = make(1, 2, 1, 1, 16, 16, torch.float32, 23)
    q, k, v, g, beta, state = (x[n].to(dev()) for n in NAMES)
    q.requires_grad_()
    out, _ = memory.gated_delta(q, k, v, g, beta, state=state)
    memory.gated_delta_step(q[0].detach(), k[0], v[0], g[0], beta[0], state)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        out.sum().backward()


def test_refusals():
    from nesle_amd import memory

    x, resets, _ = make(4, 3, 2, 4, 16, 24, torch.float32, 18)
    q, k, v, g, beta, state = (x[n].to(dev()) for n in NAMES)
    resets = resets.to(dev())

    def delta(**kw):
        a = {"q": q, "k": k, "v": v, "g": g, "beta": beta, "state": state, "resets": resets, **kw}
        return memory.gated_delta(a["q"], a["k"], a["v"], a["g"], a["beta"], state=a["state"], resets=a["resets"])

    delta()
    for bad in ({"q": q.half(), "k": k.half(), "v": v.half()}, {"k": k.bfloat16()}, {"k": k[..., :8]}, {"k": k[:, :, :1]},
                {"v": v[:, :, :3]}, {"v": v[..., :12]}, {"v": v[:3]}, {"g": g.double()}, {"g": g[..., :2]},
                {"beta": beta.transpose(0, 1)}, {"state": state.bfloat16()}, {"state": state[:2]},
                {"resets": resets[:2]}, {"resets": resets.float()}, {"resets": 1}, {"q": q.cpu()}, {"state": state.cpu()},
                {"q": q.transpose(-1, -2)}, {"v": torch.zeros(4, 3, 4, 136, device=dev())}, {"q": q[0]},
                {"q": q[..., 0:0], "k": k[..., 0:0]}, {"g": g.tolist()}):
        with pytest.raises(ValueError, match="gated_delta"):
            delta(**bad)
    with pytest.raises(ValueError, match="gated_delta_step"):
        memory.gated_delta_step(q[0], k[0], v[0], g[0], beta[0], None)
    with pytest.raises(ValueError, match="gated_delta_step"):
        memory.gated_delta_step(q, k, v, g, beta, state)
    with pytest.raises(ValueError, match="no gradient"):
        memory.gated_delta_step(q[0].requires_grad_(), k[0], v[0], g[0], beta[0], state)
    off16 = torch.zeros(state.numel() + 1, device=dev())[1:].view(state.shape)
    with pytest.raises(ValueError, match="16-byte"):
        delta(state=off16)

    table = memory.rotation_table(10, 16)
    pos = torch.zeros(4, 3, dtype=torch.int32, device=dev())

    def rotate(**kw):
        a = {"q": q, "k": k, "q_weight": None, "k_weight": None, "positions": pos, "table": table, "eps": 1e-6, **kw}
        return memory.qk_norm_rotate(a["q"], a["k"], a["q_weight"], a["k_weight"], positions=a["positions"],
                                     table=a["table"], eps=a["eps"])

    rotate()
    for bad in ({"q": q.half(), "k": k.half()}, {"k": k[..., :8]}, {"k": k[:2]}, {"k": k.bfloat16()}, {"positions": None},
                {"positions": pos.long()}, {"positions": pos[:2]}, {"table": None}, {"table": table[:, :12]},
                {"table": table.double()}, {"table": memory.rotation_table(10, 24)}, {"eps": -1.0},
                {"q_weight": torch.ones(8, device=dev())}, {"k_weight": torch.ones(16)}, {"q": q[..., :12], "k": k[..., :12]},
                {"q": q[0, 0]}, {"q": q.cpu()}):
        with pytest.raises(ValueError):
            rotate(**bad)
    for args in ((0, 16), (4, 0), (4, 12)):
        with pytest.raises(ValueError, match="rotation_table"):
            memory.rotation_table(*args)
