"""Streams, graphs, far strides, repeatability and refusals of linear attention with a
decay, layer norm and sampling (nesle_amd.memory) on the GPU, and a run of them
together.  Tolerances as in tests/test_gpu_more_memory.py."""

from __future__ import annotations

import math

import pytest
import torch

from tests import more_memory_oracle as O
from tests import test_gpu_more_memory as M
from tests.helpers import say
from tests.memory_oracle import off
from tests.test_gpu_more_memory import F32, NAMES, NORM, dev, tol

pytestmark = pytest.mark.gpu

BOTH = [torch.float32, torch.bfloat16]
# A bfloat16 result is the float32 one rounded once: the few elements that the float32
# error carries over a rounding boundary, a share of F32 / 2^-8 of them on average, are
# then 2^-7 of themselves off at most: together sqrt(F32 2^-7) of the result's norm.
ROUNDED = (F32 * 2.0 ** -7) ** 0.5


@pytest.mark.parametrize("shape", [(128, 16, 4, 4, 64, 64), (100, 16, 2, 4, 32, 32), (96, 8, 2, 2, 128, 128), (1024, 2, 2, 2, 64, 64)])
def test_bfloat16_results_are_float32_results_rounded(shape):
    from nesle_amd import memory

    say(f"[gpu] decay_attention bfloat16 results {shape}")
    x, resets, grads = M.make(*shape, torch.bfloat16, 31, resets=0.005)
    ref = [x[n].double().requires_grad_() for n in NAMES]
    want = O.decay(*ref, resets, shape[-2] ** -0.5)
    gpu = [x[n].to(dev()).requires_grad_() for n in NAMES]
    got = memory.decay_attention(*gpu[:4], state=gpu[4], resets=resets.to(dev()))
    dw = torch.autograd.grad(want, ref, [t.double() for t in grads])
    dg = torch.autograd.grad(got, gpu, [t.to(dev()) for t in grads])
    error = {"out": off(got[0], want[0]), **{f"d{n}": off(a, b) for n, a, b in zip("qkv", dg, dw)}}
    # Of shared key heads' gradients too: shares are added in float32.
    assert all(v <= ROUNDED for v in error.values()), error


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("dim", [8, 32, 40, 64, 72, 128])
@pytest.mark.parametrize("T", [31, 32, 33, 63, 64, 65, 96, 97, 128, 129])
def test_decay_lengths_around_a_chunk(T, dim, dtype):
    say(f"[gpu] decay_attention {T} tokens of {dim} {dtype}")
    M.check_decay(*M.make(T, 2, 1, 2, dim, dim, dtype, T + dim, resets=0.03))


@pytest.mark.parametrize("dim", [32, 64, 128])
def test_decay_equal_keys(dim):
    """All queries alike and all keys alike: what is summed for a decay's gradient has
    one sign a head, and the pairs' products are all as large as they get."""
    for dtype in BOTH:
        say(f"[gpu] decay_attention equal keys {dim} {dtype}")
        M.check_decay(*M.make(150, 2, 1, 2, dim, dim, dtype, 7, resets=0.0, alike=1.0))


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("shape,segments", [((513, 16, 2, 4, 64, 64), 5), ((470, 32, 2, 4, 64, 48), 4), ((449, 32, 4, 4, 32, 32), 8),
                                            ((460, 8, 2, 4, 72, 128), 8), ((450, 16, 4, 4, 128, 40), 4), ((1000, 4, 4, 4, 64, 64), 16)])
def test_decay_few_segments(shape, segments, dtype):
    """2 to 16 segments: the state before one, and the gradient after one, are found in
    other ways than of many."""
    import ctypes

    from nesle_amd import abi

    say(f"[gpu] decay_attention {segments} segments {shape} {dtype}")
    a = abi.DecayArgs(abi.MEM_F32 if dtype == torch.float32 else abi.MEM_BF16, *shape, 1.0)
    floats = abi.lib().nesle_decay_forward_scratch_floats(ctypes.byref(a))
    assert floats == segments * shape[1] * shape[3] * (shape[4] * shape[5] + 1)
    x, resets, grads = M.make(*shape, dtype, 50 + segments, resets=0.002)
    M.check_decay(x, resets, grads)
    x["state"] = None
    M.check_decay(x, None, grads)


def test_decay_gradient_of_one_number():
    """One head: its decay's gradient is one number, over 64 to 6,000 terms of either sign
    that nearly cancel in places.  Each term is off by a few 2^-24 of itself, and they are
    added in float64 from 32 tokens of a lane on: 2^-22 of their 2-norm, with room for 4
    standard deviations of 20 draws.  The terms by the definition: one console's each."""
    from nesle_amd import memory

    for seed in range(10):
        for T, N in ((1, 64), (70, 30)):
            say(f"[gpu] decay_attention decay's gradient {seed} {T} {N}")
            x, _, grads = M.make(T, N, 1, 1, 48, 48, torch.float32, seed, resets=0.0)
            ref = [x[n].double() for n in NAMES]
            ref[3] = ref[3].expand(N, 1).clone().requires_grad_()
            # A decay of its own for each console.
            each = torch.stack([torch.autograd.grad(O.decay(*(t[:, n:n + 1] for t in ref[:3]), ref[3][n], ref[4][n:n + 1], None, 48 ** -0.5),
                                                    ref[3], [grads[0][:, n:n + 1].double(), grads[1][n:n + 1].double()])[0][n]
                                for n in range(N)])
            gpu = [x[n].to(dev()) for n in NAMES]
            gpu[3].requires_grad_()
            got = torch.autograd.grad(memory.decay_attention(*gpu[:4], state=gpu[4]), gpu[3], [t.to(dev()) for t in grads])[0]
            assert abs(float(got) - float(each.sum())) <= 2.0 ** -22 * float(each.norm()) + 2.0 ** -24 * abs(float(each.sum())), (seed, T)


def test_decay_offsets_past_32_bits():
    """Queries, keys and values whose steps lie 2^31 elements apart."""
    from nesle_amd import memory

    say("[gpu] decay_attention wide strides")
    x, _, _ = M.make(3, 2, 1, 1, 32, 32, torch.bfloat16, 10)
    far = (1 << 31) + 64
    buf = torch.empty(2 * far + 4096, dtype=torch.bfloat16, device=dev())
    cut = {}
    for i, n in enumerate("qkv"):
        cut[n] = buf.as_strided(x[n].shape, (far, 32, 32, 1), 512 * i)
        cut[n].copy_(x[n])
    got = memory.decay_attention(cut["q"], cut["k"], cut["v"], x["g"].to(dev()), state=x["state"].to(dev()))
    want = O.decay(*(x[n] for n in NAMES), None, 32 ** -0.5)
    assert off(got[0], want[0]) <= tol(torch.bfloat16) and off(got[1], want[1]) <= F32


@pytest.mark.parametrize("far", [((1 << 31) - 4096) // 126 // 8 * 8, ((1 << 31) - 4096) // 126 // 8 * 8 + 8, (1 << 26) + 64])
def test_decay_gradient_at_the_last_32_bit_stride(far):
    """The largest steps at which 64 rows lie within what a 32-bit offset reaches, the
    next, and larger ones; two chunks."""
    say(f"[gpu] decay_attention steps of {far} elements, gradient")
    T = 66
    buf = torch.empty((T - 1) * far + 8192, dtype=torch.bfloat16, device=dev())
    x, resets, grads = M.make(T, 2, 1, 2, 32, 32, torch.bfloat16, 30)
    at = iter((0, 512, 1024))

    def move(t):
        if t.dim() != 4 or t.shape[0] != T:
            return t.to(dev())
        cut = buf.as_strided(t.shape, (far, t.shape[2] * t.shape[3], t.shape[3], 1), next(at))
        cut.copy_(t)
        return cut.detach()

    M.check_decay(x, resets, grads, move=move)


def test_norm_and_sampling_offsets_past_32_bits():
    from nesle_amd import memory

    say("[gpu] layer_norm and sample_actions wide strides")
    far = (1 << 31) + 64
    buf = torch.empty(2 * far + 4096, dtype=torch.bfloat16, device=dev())
    x = buf.as_strided((3, 4, 96), (far, 96, 1))
    x.copy_(torch.randn(3, 4, 96, generator=torch.Generator().manual_seed(1)))
    assert torch.equal(memory.layer_norm(x), memory.layer_norm(x.contiguous()))
    u = torch.rand(3, 4, generator=torch.Generator().manual_seed(2)).to(dev())
    for count in (12, 96):
        got, want = memory.sample_actions(x[..., :count], u), memory.sample_actions(x[..., :count].contiguous(), u)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_norm_writes_past_32_bits():
    """A result of more than 2^32 bytes: its last rows."""
    from nesle_amd import memory

    say("[gpu] layer_norm of 4.6 GB")
    x = torch.randn(1, 256, device=dev()).expand(9_000_000, 256)
    y = memory.layer_norm(x.to(torch.bfloat16))
    assert bool((y[-1000:] == y[:1000]).all()) and bool((y[4_200_000:4_201_000] == y[:1000]).all())


# ---- a run of them together -------------------------------------------------------------

def _layer(x, resets, u, w, b, keep=True):
    """What a policy with such a memory does with its tokens: memory, norm of each head,
    action; and one step of the same."""
    from nesle_amd import memory

    out, after = memory.decay_attention(*x[:4], state=x[4], resets=resets)
    y = memory.layer_norm(out, w, b)
    logits = y.flatten(-2)[..., :30]
    with torch.no_grad():
        actions, logprobs = memory.sample_actions(logits.detach(), u, temperature=0.8, top_k=20, top_p=0.95, min_p=0.01)
    return y, after, actions, logprobs


def _layer_inputs(T=70, dtype=torch.float32):
    x, resets, grads = M.make(T, 6, 2, 4, 32, 32, dtype, 40, resets=0.05)
    gen = torch.Generator().manual_seed(41)
    u = torch.rand(T, 6, generator=gen)
    w, b = 1 + 0.1 * torch.randn(32, generator=gen), 0.1 * torch.randn(32, generator=gen)
    return [x[n].to(dev()) for n in NAMES], resets.to(dev()), u.to(dev()), w.to(dev()), b.to(dev()), grads


@pytest.mark.parametrize("dtype", BOTH)
def test_a_layer_and_its_gradient(dtype):
    """The operators one after the other against their definitions one after the other;
    every action against the definition of the logits that it was drawn from."""
    say(f"[gpu] a layer {dtype}")
    x, resets, u, w, b, grads = _layer_inputs(dtype=dtype)
    leaves = [t.requires_grad_() for t in (*x, w, b)]
    y, after, actions, logprobs = _layer(leaves[:5], resets, u, *leaves[5:])
    ref = [t.detach().cpu().double().requires_grad_() for t in leaves]
    out, want_after = O.decay(*ref[:5], resets.cpu(), 32 ** -0.5)
    if dtype == torch.bfloat16:        # as the norm got it
        out = out + (out.detach().bfloat16().double() - out.detach())
    want = O.layer_norm(out, ref[5], ref[6], 1e-5)
    # The norm divides by a spread that is as exact as its input: the errors add.
    assert off(y, want) <= 2 * tol(dtype) and off(after, want_after) <= F32
    d = torch.autograd.grad((y, after), leaves, [t.to(dev()) for t in grads])
    dw = torch.autograd.grad((want, want_after), ref, [t.double() for t in grads])
    for n, a, c in zip((*NAMES, "weight", "bias"), d, dw):
        # bfloat16: the gradient passes from the norm to the memory rounded, 2^-9 of each
        # of its elements, and the results are rounded again.
        assert off(a, c) <= (10 * F32 if dtype == torch.float32 else 3 * 2.0 ** -9 + 10 * F32), n
    rows = y.detach().flatten(-2)[..., :30].double().cpu().reshape(-1, 30).tolist()
    for i, (row, number) in enumerate(zip(rows, u.double().cpu().reshape(-1).tolist())):
        a, p = O.sample(row, number, 0.8, 20, 0.95, 0.01)
        assert int(actions.reshape(-1)[i]) == a and abs(float(logprobs.reshape(-1)[i]) - p) <= 2.0 ** -24 * abs(p) + 1e-13, i


def test_same_bits_every_time_and_on_another_stream():
    say("[gpu] a layer on another stream")
    for T in (70, 600):
        x, resets, u, w, b, grads = _layer_inputs(T)
        grads = [t.to(dev()) for t in grads]

        def work():
            leaves = [t.detach().requires_grad_() for t in (*x, w, b)]
            y, after, actions, logprobs = _layer(leaves[:5], resets, u, *leaves[5:])
            return (y, after, actions, logprobs, *torch.autograd.grad((y, after), leaves, grads))

        first, again = work(), work()
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            other = work()
        side.synchronize()
        for a, b2, c in zip(first, again, other):
            assert torch.equal(a, b2) and torch.equal(a, c)


def test_two_streams_at_once():
    """Calls that overlap share nothing: segments, partial sums and all."""
    from nesle_amd import memory

    say("[gpu] two streams at once")
    x, resets, u, w, b, _ = _layer_inputs(1200)
    other = [t + 0.25 for t in x[:3]] + x[3:]
    want = [_layer(a, resets, u, w, b) for a in (x, other)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, a in enumerate((x, other)):
            with torch.cuda.stream(streams[i]):
                got[i].append(_layer(a, resets, u, w, b))
    torch.cuda.synchronize()
    for i in range(2):
        for g in got[i]:
            assert all(torch.equal(a, c) for a, c in zip(g, want[i]))


@pytest.mark.parametrize("T", [40, 600])
def test_captured_in_a_graph(T):
    """A captured layer, its step, and its gradient replay to the eager result, on new
    inputs too, with eager work between the replays.  The leaves of the captured
    gradient are its own."""
    from nesle_amd import memory

    say(f"[gpu] a layer in a graph, {T} steps")
    x, resets, u, w, b, grads = _layer_inputs(T)
    grads = [t.to(dev()) for t in grads]
    held = x[4].clone()

    def work():
        leaves = [t.detach().requires_grad_() for t in (*x, w, b)]
        y, after, actions, logprobs = _layer(leaves[:5], resets, u, *leaves[5:])
        d = torch.autograd.grad((y, after), leaves, grads)
        with torch.no_grad():
            one = memory.decay_attention_step(x[0][0], x[1][0], x[2][0], x[3], held, resets=resets[0])
        return (y, after, actions, logprobs, *d, one)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs, captured = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for graph in graphs:                   # two graphs of the same work
        with torch.cuda.graph(graph, stream=side):
            captured.append(work())
    for i in range(4):
        x[2].copy_(torch.randn(x[2].shape, generator=torch.Generator().manual_seed(i)))
        u.copy_(torch.rand(u.shape, generator=torch.Generator().manual_seed(i)))
        held.copy_(x[4])
        want = [t.clone() for t in work()]
        for graph, outs in zip(graphs, captured):
            held.copy_(x[4])
            graph.replay()
            torch.cuda.synchronize()
            for a, c in zip(outs, want):
                assert torch.equal(a, c), i


# ---- gradients that are partly wanted, and of what is refused -----------------------------

def test_unused_outputs_and_inputs_without_gradient():
    from nesle_amd import memory

    say("[gpu] partly wanted gradients")
    x, resets, grads = M.make(70, 2, 1, 2, 24, 16, torch.float32, 22)
    for used in range(2):
        ref = [x[n].double().requires_grad_() for n in NAMES]
        want = O.decay(*ref, resets, 24 ** -0.5)[used]
        dw = torch.autograd.grad(want, ref, grads[used].double(), allow_unused=True)
        gpu = [x[n].to(dev()).requires_grad_() for n in NAMES]
        got = memory.decay_attention(*gpu[:4], state=gpu[4], resets=resets.to(dev()))[used]
        dg = torch.autograd.grad(got, gpu, grads[used].to(dev()))
        for n, a, c in zip(NAMES, dg, dw):
            assert off(a, torch.zeros(a.shape, dtype=torch.float64) if c is None else c) <= F32, (used, n)
    whole = torch.autograd.grad(memory.decay_attention(*gpu[:4], state=gpu[4], resets=resets.to(dev())), gpu,
                                [t.to(dev()) for t in grads])
    for i, n in enumerate(NAMES):
        alone = [t.detach().requires_grad_(j == i) for j, t in enumerate(gpu)]
        out = memory.decay_attention(*alone[:4], state=alone[4], resets=resets.to(dev()))
        assert torch.equal(torch.autograd.grad(out, alone[i], [t.to(dev()) for t in grads])[0], whole[i]), n
    # A gradient of a state that starts off a 16-byte boundary.
    pad = torch.zeros(grads[1].numel() + 1, device=dev())
    pad[1:] = grads[1].flatten().to(dev())
    out = memory.decay_attention(*gpu[:4], state=gpu[4], resets=resets.to(dev()))
    same = torch.autograd.grad(out, gpu, [grads[0].to(dev()), pad[1:].view(grads[1].shape)])
    assert all(torch.equal(a, c) for a, c in zip(same, whole))
    t = torch.randn(5, 24, device=dev())
    w, b = torch.ones(24, device=dev()), torch.zeros(24, device=dev())
    full = torch.autograd.grad(memory.layer_norm(*(leaves := [v.clone().requires_grad_() for v in (t, w, b)])).square().sum(), leaves)
    for i in range(3):
        alone = [v.clone().requires_grad_(j == i) for j, v in enumerate((t, w, b))]
        assert torch.equal(torch.autograd.grad(memory.layer_norm(*alone).square().sum(), alone[i])[0], full[i])


def test_only_first_derivatives():
    from nesle_amd import memory

    x, _, _ = M.make(4, 2, 1, 1, 16, 16, torch.float32, 21)
    q, k, v, g = (x[n].to(dev()).requires_grad_() for n in NAMES[:4])
    w = torch.tensor(2.0, device=dev(), requires_grad=True)
    for fn in (lambda: memory.decay_attention(q, k, v, g)[0], lambda: memory.layer_norm(q)):
        (d,) = torch.autograd.grad((fn() * w).square().sum(), [q], create_graph=True)
        with pytest.raises(RuntimeError, match="second derivative"):
            d.sum().backward()
        (d,) = torch.autograd.grad(fn().sum(), [q], create_graph=True)
        with pytest.raises(RuntimeError, match="second derivative"):
            d.square().sum().backward()


def test_step_marks_the_state_as_changed():
    from nesle_amd import memory

    x, _, _ = M.make(1, 2, 1, 1, 16, 16, torch.float32, 23)
    q, k, v, g, state = (x[n].to(dev()) for n in NAMES)
    out, _ = memory.decay_attention(q.requires_grad_(), k, v, g, state=state)
    memory.decay_attention_step(q[0].detach(), k[0], v[0], g, state)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        out.sum().backward()


def test_refusals():
    from nesle_amd import memory

    x, resets, _ = M.make(4, 3, 2, 4, 16, 24, torch.float32, 18)
    q, k, v, g, state = (x[n].to(dev()) for n in NAMES)
    resets = resets.to(dev())

    def decay(**kw):
        a = {"q": q, "k": k, "v": v, "g": g, "state": state, "resets": resets, **kw}
        return memory.decay_attention(a["q"], a["k"], a["v"], a["g"], state=a["state"], resets=a["resets"])

    decay()
    for bad in ({"q": q.half(), "k": k.half(), "v": v.half()}, {"k": k.bfloat16()}, {"k": k[..., :8]}, {"k": k[:, :, :1]},
                {"v": v[:, :, :3]}, {"v": v[..., :12]}, {"v": v[:3]}, {"g": g.double()}, {"g": g[:2]}, {"g": g.expand(4, 3, 4)},
                {"state": state.bfloat16()}, {"state": state[:2]}, {"resets": resets[:2]}, {"resets": resets.float()},
                {"resets": 1}, {"q": q.cpu()}, {"state": state.cpu()}, {"g": g.cpu()}, {"q": q.transpose(-1, -2)},
                {"v": torch.zeros(4, 3, 4, 136, device=dev())}, {"q": q[0]}, {"q": q[..., 0:0], "k": k[..., 0:0]}, {"g": g.tolist()},
                {"state": torch.zeros(state.numel() + 1, device=dev())[1:].view(state.shape)}):
        with pytest.raises(ValueError, match="decay_attention"):
            decay(**bad)
    for args in ((q[0], k[0], v[0], g, None), (q, k, v, g, state)):
        with pytest.raises(ValueError, match="decay_attention_step"):
            memory.decay_attention_step(*args)
    with pytest.raises(ValueError, match="no gradient"):
        memory.decay_attention_step(q[0].requires_grad_(), k[0], v[0], g, state)

    t, w = torch.zeros(3, 16, device=dev()), torch.ones(16, device=dev())
    for args in ((t.half(),), (t.double(),), (t.t(),), (t[:, :0],), (torch.zeros(2, 16385, device=dev()),), (t, w[:8]), (t, w.bfloat16()),
                 (t, w, w[:8]), (t, w.cpu()), (t, torch.ones(17, device=dev())[1:]), (t.view(1, 1, 1, 3, 16),), (torch.tensor(1.0, device=dev()),)):
        with pytest.raises(ValueError, match="layer_norm"):
            memory.layer_norm(*args)
    for eps in (-1e-5, math.nan, math.inf):
        with pytest.raises(ValueError, match="eps"):
            memory.layer_norm(t, eps=eps)

    u = torch.zeros(3, device=dev())
    for args in ((t.half(), u), (t, u.double()), (t, u[:2]), (t, u.cpu()), (t[0], u), (torch.zeros(3, 1025, device=dev()), u), (t[:, :0], u),
                 (t.t(), u), (t, torch.zeros(6, device=dev())[::2])):
        with pytest.raises(ValueError, match="sample_actions"):
            memory.sample_actions(*args)
    for how in ({"temperature": -0.1}, {"temperature": math.nan}, {"temperature": math.inf}, {"top_k": -1}, {"top_k": 2.5},
                {"top_k": "many"}, {"top_p": 0.0}, {"top_p": 1.5}, {"min_p": -0.1}, {"min_p": 1.5}, {"min_p": None},
                {"temperature": u.double()}, {"top_k": u}, {"top_p": u[:2]}, {"min_p": u.cpu()}, {"top_k": 10 ** 30}):
        with pytest.raises(ValueError, match="nesle_sample|sample_actions"):
            memory.sample_actions(t, u, **how)
    with pytest.raises(ValueError, match="no gradient"):
        memory.sample_actions(t.clone().requires_grad_(), u)
