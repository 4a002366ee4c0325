"""The memory operators where they can go wrong: what bfloat16 results hold; equal
keys, ended episodes, gates and values that are not finite on every kind of
products (32, 64 and 128 dimensions of either type); gates that leave nothing,
positions outside the table, calls that cannot be answered."""

from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as fwAD

from tests import memory_oracle as O
from tests import test_gpu_memory as M
from tests.helpers import say

pytestmark = pytest.mark.gpu

F32, NAMES = M.F32, M.NAMES
BOTH = [torch.float32, torch.bfloat16]
DIMS = [32, 64, 128]


def dev():
    return torch.device("cuda")


# A float32 result that is off by F32 of its norm and then rounded to bfloat16
# (steps of at most 2^-7 of an element): an element comes out a step away with
# the chance error / step, so the squares add up to at most |error| |steps| =
# F32 2^-7 of the result's.
ROUNDED = (F32 * 2.0 ** -7) ** 0.5


@pytest.mark.parametrize("shape", [(128, 16, 4, 4, 64, 64), (96, 16, 2, 4, 32, 32), (96, 8, 2, 2, 128, 128),
                                   (1024, 2, 2, 2, 64, 64)])
def test_bfloat16_results_are_float32_results_rounded(shape):
    """Outputs and the gradients of queries, keys and values hold what float32
    products give, rounded once."""
    from nesle_amd import memory

    say(f"[gpu] gated_delta bfloat16 results {shape}")
    x, resets, grads = M.make(*shape, torch.bfloat16, 31, resets=0.005)
    ref = [x[n].double().requires_grad_() for n in NAMES]
    want = O.delta(*ref, resets, shape[-2] ** -0.5)
    gpu = [x[n].to(dev()).requires_grad_() for n in NAMES]
    got = memory.gated_delta(*gpu[:5], state=gpu[5], resets=resets.to(dev()))
    dw = torch.autograd.grad(want, ref, [t.double() for t in grads])
    dg = torch.autograd.grad(got, gpu, [t.to(dev()) for t in grads])
    off = {"out": O.off(got[0], want[0]), **{f"d{n}": O.off(a, b) for n, a, b in zip("qkv", dg, dw)}}
    assert all(v <= ROUNDED for v in off.values()), off


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("dim", DIMS)
def test_equal_keys_of_every_size(dim, dtype):
    say(f"[gpu] gated_delta equal keys, {dim} {dtype}")
    x, resets, grads = M.make(96, 2, 1, 1, dim, dim, dtype, 7, resets=0.0, alike=1.0)
    x["beta"][:] = 1.0
    M.check_delta(x, resets, grads)


# exp of the first is zero in float32 (half its smallest value is 2^-150 =
# exp(-103.97208)), exp of the second is not.
GONE, HELD = -103.9721, -103.95


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("dim", [32, 64])
@pytest.mark.parametrize("T", [1, 40, 600])
def test_gate_whose_exponential_is_zero_drops_the_state(T, dim, dtype):
    """By selection: a state of NaN reaches nothing after it.  The gradient of
    the state is zero there, and the gate's."""
    from nesle_amd import memory

    say(f"[gpu] gated_delta gate of {GONE}, {T} x {dim} {dtype}")
    assert float(torch.tensor(GONE).exp()) == 0.0 and float(torch.tensor(HELD).exp()) > 0.0
    x, _, grads = M.make(T, 2, 1, 1, dim, dim, dtype, 14)
    at = T // 2
    x["g"][at, 0], x["g"][at, 1] = GONE, HELD
    y = {n: t.clone() for n, t in x.items()}
    x["state"][:] = float("nan")
    y["state"][:] = 0.0
    got = memory.gated_delta(*(x[n].to(dev()) for n in NAMES[:5]), state=x["state"].to(dev()))
    y["g"][at, 0] = -float("inf")
    want = O.delta(*(y[n] for n in NAMES), None, dim ** -0.5)
    assert O.off(got[0][at:, 0], want[0][at:, 0]) <= M.tol(dtype) and O.off(got[1][0], want[1][0]) <= F32
    assert torch.isnan(got[0][:, 1]).all() and torch.isnan(got[1][1]).all()
    if T == 1:
        state = x["state"].to(dev())
        out = memory.gated_delta_step(*(x[n][0].to(dev()) for n in NAMES[:5]), state)
        assert O.off(out[0], want[0][0, 0]) <= M.tol(dtype) and O.off(state[0], want[1][0]) <= F32
        assert torch.isnan(out[1]).all() and torch.isnan(state[1]).all()
    y["state"] = torch.randn(y["state"].shape, generator=torch.Generator().manual_seed(1))
    y["g"][at, 0] = GONE
    gpu = [y[n].to(dev()).requires_grad_() for n in NAMES]
    d = torch.autograd.grad(memory.gated_delta(*gpu[:5], state=gpu[5]), gpu, [t.to(dev()) for t in grads])
    assert float(d[3][at, 0].abs().sum()) == 0.0 and (T > 1 or float(d[5][0].abs().sum()) == 0.0)


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("rotated", [16, 32])
def test_position_outside_the_table_makes_the_whole_head_nan(rotated, dtype):
    from nesle_amd import memory

    say(f"[gpu] qk_norm_rotate positions outside, {rotated} of 32 {dtype}")
    q, k, wq, wk, pos, table, dq, dk = (t.to(dev()) for t in M.make_rotate((6, 5), 2, 3, 32, rotated, dtype, 6))
    pos[0, 0], pos[3, 2], pos[5, 4] = -1, 50, 1 << 30
    bad = (pos < 0) | (pos >= 50)
    leaves = [t.requires_grad_() for t in (q, k, wq, wk)]
    got = memory.qk_norm_rotate(*leaves, positions=pos, table=table)
    d = torch.autograd.grad(got, leaves, [dq, dk])
    for t in (*got, *d[:2]):
        assert torch.isnan(t[bad]).all() and torch.isfinite(t[~bad]).all()
    assert all(torch.isnan(t).all() for t in d[2:])


# ---- calls that cannot be answered --------------------------------------------------------

def _calls():
    """Each operator as a function of its inputs, with those inputs."""
    from nesle_amd import memory

    x, _, _ = M.make(4, 2, 1, 1, 16, 16, torch.float32, 21)
    q, k, v, g, beta, state = (x[n].to(dev()) for n in NAMES)
    w, table = torch.ones(16, device=dev()), memory.rotation_table(10, 16)
    pos = torch.zeros(4, 2, dtype=torch.int32, device=dev())
    return {
        "qk_norm_rotate": (lambda q, k, w, u, t: memory.qk_norm_rotate(q, k, w, u, positions=pos, table=t)[0],
                           [q, k, w, w.clone(), table]),
        "gated_delta": (lambda q, k, v, g, b, s: memory.gated_delta(q, k, v, g, b, state=s)[0], [q, k, v, g, beta, state]),
        "gated_delta_step": (lambda q, k, v, g, b, s: memory.gated_delta_step(q, k, v, g, b, s),
                             [q[0], k[0], v[0], g[0], beta[0], state.clone()]),
    }


@pytest.mark.parametrize("name", ["qk_norm_rotate", "gated_delta", "gated_delta_step"])
@pytest.mark.parametrize("grad", [False, True])
def test_forward_derivatives_are_refused(name, grad):
    """A tangent would be lost."""
    fn, inputs = _calls()[name]
    for i, t in enumerate(inputs):
        with fwAD.dual_level():
            args = list(inputs)
            args[i] = fwAD.make_dual(t.clone(), torch.ones_like(t))
            if grad and name != "gated_delta_step":
                args[(i + 1) % len(args)] = args[(i + 1) % len(args)].clone().requires_grad_(i + 2 < len(args))
            with pytest.raises(ValueError, match=f"{name}.*forward"):
                fn(*args)
    fn(*inputs)


@pytest.mark.parametrize("name", ["qk_norm_rotate", "gated_delta", "gated_delta_step"])
def test_tracing_is_refused(name):
    """A trace would hold an output that nobody wrote."""
    from torch.fx.experimental.proxy_tensor import make_fx

    fn, inputs = _calls()[name]
    with pytest.raises(ValueError, match=f"{name} cannot be traced"):
        torch.jit.trace(fn, tuple(inputs), check_trace=False)
    with pytest.raises(ValueError, match=f"{name} cannot be traced"):
        make_fx(fn)(*inputs)


def test_second_derivatives_are_refused_whatever_the_gradients_are():
    """Also where the gradient handed in needs none: the result depends on the
    inputs all the same."""
    for name in ("qk_norm_rotate", "gated_delta"):
        fn, inputs = _calls()[name]
        leaves = [t.requires_grad_() for t in inputs[:2]]
        (d,) = torch.autograd.grad(fn(*inputs).sum(), leaves[:1], create_graph=True)
        with pytest.raises(RuntimeError, match="second derivative"):
            d.square().sum().backward()


def test_sizes_of_more_than_32_bits_are_refused():
    """Of the other tensors too: heads of keys, heads of values."""
    from nesle_amd import memory

    x, _, _ = M.make(4, 2, 1, 1, 16, 16, torch.float32, 21)
    q, k, v, g, beta, state = (x[n].to(dev()) for n in NAMES)
    many = q.expand(4, 2, (1 << 32) + 1, 16)
    with pytest.raises(ValueError, match="k must be of sizes below"):
        memory.qk_norm_rotate(q, many)
    with pytest.raises(ValueError, match="v must be of sizes below"):
        memory.gated_delta(q, k, many, g, beta, state=state)
    with pytest.raises(ValueError, match="v must be of sizes below"):
        memory.gated_delta_step(q[0], k[0], many[0], g[0], beta[0], state)


# ---- ended episodes, gates ------------------------------------------------------------------

@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("where", ["all", "first", "edges", "last"])
def test_resets_of_every_size(where, dim, dtype):
    say(f"[gpu] gated_delta resets {where}, {dim} {dtype}")
    x, resets, grads = M.make(70, 3, 1, 2, dim, dim, dtype, 5, resets=0.0)
    resets[:] = where == "all"
    if where == "first":
        resets[0] = True
    if where == "last":
        resets[-1] = True
    if where == "edges":
        for n, t in enumerate((31, 32, 33)):
            resets[t, n] = True
            resets[t + 1, n] = n == 2
    M.check_delta(x, resets, grads)


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("gate", ["zero", "strong", "off", "growing"])
def test_gates_of_every_size(gate, dim, dtype):
    say(f"[gpu] gated_delta gates {gate}, {dim} {dtype}")
    x, resets, grads = M.make(70, 2, 1, 2, dim, dim, dtype, 6, resets=0.0)
    if gate == "zero":
        x["g"].zero_()
    elif gate == "strong":
        x["g"] = x["g"] * 250
    elif gate == "growing":
        x["g"] = x["g"] * -0.1
    else:
        x["g"][5, 0, 0], x["g"][40, 1, 1], x["g"][32, 0, 1] = -float("inf"), -200.0, -float("inf")
    M.check_delta(x, resets, grads)


# ---- what is not finite ------------------------------------------------------------------

@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("T", [70, 900])
def test_what_is_not_finite_stays_where_it_belongs(T, dim, dtype):
    """A state of NaN ends at a reset; a NaN or infinite token reaches neither
    earlier tokens, nor other consoles, nor the next episode.  900 steps of 4
    heads are walked in segments."""
    from nesle_amd import memory

    say(f"[gpu] gated_delta not finite, {T} x {dim} {dtype}")
    x, resets, _ = M.make(T, 4, 1, 1, dim, dim, dtype, 13, resets=0.0)
    s, at, tol = dim ** -0.5, T - 70, M.tol(dtype)
    clean = O.delta(*(x[n] for n in NAMES), resets, s)[0]
    resets[at, 0] = True
    x["state"][0] = float("nan")
    x["v"][at + 20, 1, 0, 3] = float("nan")
    x["k"][at + 41, 2, 0, 5] = float("inf")
    resets[at + 50, 1], resets[at + 45, 2] = True, True
    x["beta"][at + 10, 3], x["g"][at + 12, 3], resets[at + 13, 3] = float("nan"), float("nan"), True
    got = memory.gated_delta(*(x[n].to(dev()) for n in NAMES[:5]), state=x["state"].to(dev()), resets=resets.to(dev()))
    out = got[0].cpu()
    y = {n: torch.where(torch.isfinite(t), t, torch.zeros_like(t)) for n, t in x.items()}
    want = O.delta(*(y[n] for n in NAMES), resets, s)[0]
    assert O.off(out[at:, 0], want[at:, 0]) <= tol and torch.isnan(out[:at, 0]).all()
    assert O.off(out[:at + 20, 1], clean[:at + 20, 1]) <= tol and O.off(out[at + 50:, 1], want[at + 50:, 1]) <= tol
    assert O.off(out[:at + 41, 2], clean[:at + 41, 2]) <= tol and O.off(out[at + 45:, 2], want[at + 45:, 2]) <= tol
    assert O.off(out[:at + 10, 3], clean[:at + 10, 3]) <= tol and O.off(out[at + 13:, 3], want[at + 13:, 3]) <= tol
    assert torch.isnan(out[at + 20:at + 50, 1, 0, 3]).all() and torch.isnan(out[at + 10:at + 13, 3]).all()
    assert torch.isfinite(got[1]).all()
