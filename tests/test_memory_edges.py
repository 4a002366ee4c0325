"""The memory operators' binding and entry points without a GPU: calls that cannot
be answered are refused."""

from __future__ import annotations

import subprocess
import sys
from pathlib import Path

import pytest
import torch
import torch.autograd.forward_ad as fwAD

from nesle_amd import memory

ROOT = Path(__file__).resolve().parents[1]


def calls():
    """Each operator as a function of its tensors, and those tensors (on the CPU,
    which is refused last)."""
    q, g, state = torch.zeros(2, 3, 1, 16), torch.zeros(2, 3, 1), torch.zeros(3, 1, 16, 16)
    w, table = torch.ones(16), memory.rotation_table(4, 16, device="cpu")
    pos = torch.zeros(2, 3, dtype=torch.int32)
    return {
        "qk_norm_rotate": (lambda q, k, w, u, t: memory.qk_norm_rotate(q, k, w, u, positions=pos, table=t)[0],
                           [q, q.clone(), w, w.clone(), table]),
        "gated_delta": (lambda q, k, v, g, b, s: memory.gated_delta(q, k, v, g, b, state=s)[0],
                        [q, q.clone(), q.clone(), g, g.clone(), state]),
        "gated_delta_step": (lambda q, k, v, g, b, s: memory.gated_delta_step(q, k, v, g, b, s),
                             [q[0], q[1], q[0].clone(), g[0], g[1], state.clone()]),
    }


@pytest.mark.parametrize("name", ["qk_norm_rotate", "gated_delta", "gated_delta_step"])
def test_forward_derivatives_are_refused(name):
    fn, inputs = calls()[name]
    with pytest.raises(ValueError, match="GPU"):
        fn(*inputs)
    for i, t in enumerate(inputs):
        with fwAD.dual_level():
            args = list(inputs)
            args[i] = fwAD.make_dual(t.clone(), torch.ones_like(t))
            with pytest.raises(ValueError, match=f"{name} has no forward-mode derivative"):
                fn(*args)


@pytest.mark.parametrize("name", ["qk_norm_rotate", "gated_delta", "gated_delta_step"])
def test_tracing_is_refused(name):
    from torch.fx.experimental.proxy_tensor import make_fx

    fn, inputs = calls()[name]
    with pytest.raises(ValueError, match=f"{name} cannot be traced"):
        torch.jit.trace(fn, tuple(inputs), check_trace=False)
    with pytest.raises(ValueError, match=f"{name} cannot be traced"):
        make_fx(fn)(*inputs)


@pytest.mark.parametrize("name", ["qk_norm_rotate", "gated_delta", "gated_delta_step"])
def test_sizes_of_more_than_32_bits_are_refused(name):
    """An expanded tensor takes no memory, so such a size is within reach; cut to
    32 bits it would pass every later check."""
    fn, inputs = calls()[name]
    for size in (1 << 32, (1 << 32) + 2):
        for dim in range(inputs[0].dim() - 1):
            q = inputs[0][tuple(slice(0, 1) if d == dim else slice(None) for d in range(inputs[0].dim()))]
            q = q.expand(*(size if d == dim else n for d, n in enumerate(q.shape)))
            with pytest.raises(ValueError, match=f"{name}: q must be of sizes below 2\\^32"):
                fn(q, q, *inputs[2:])


@pytest.mark.parametrize("dim", [0, 264, 3000, 4096, 0xffffffff])
def test_scratch_of_dimensions_that_are_refused(dim):
    """The size asked for ends, and is nothing, where the call itself refuses (in a
    process of its own: it did not return for the largest)."""
    code = ("import ctypes; from nesle_amd import abi; a = abi.QkArgs(abi.MEM_F32, 4, 2, 2, 2, %d, 0, 0, 0, 1e-6, "
            "q_weight=16); print(abi.lib().nesle_qk_scratch_floats(ctypes.byref(a)))" % dim)
    done = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=60, cwd=ROOT)
    assert done.returncode == 0 and done.stdout.strip() == "0", done


def test_the_console_builds_without_pytorch(monkeypatch):
    from nesle_amd import build

    made = []
    monkeypatch.setitem(sys.modules, "torch", None)        # not importable
    monkeypatch.setattr(build, "build_hip", lambda: made.append("hip"))
    monkeypatch.setattr(build, "build_shim", lambda: made.append("shim"))
    monkeypatch.setattr(build, "_run", lambda cmd: made.append(cmd))
    build.build_all()
    assert made == ["hip", "shim"]


@pytest.mark.parametrize("dim,heads,tokens,cut", [
    (32, 128, 256, True), (32, 256, 256, False), (32, 256, 1024, True), (32, 260, 4096, False),
    (64, 64, 256, True), (64, 64, 224, False), (64, 128, 256, False), (64, 128, 512, True), (64, 132, 4096, False),
    (128, 32, 256, True), (128, 64, 256, False), (128, 64, 512, True), (128, 128, 1024, False), (72, 96, 512, False)])
def test_long_walks_are_cut_where_that_is_faster(dim, heads, tokens, cut):
    """Both sides of the rule, measured: with 128 dimensions 1,024 tokens of 128 heads
    take 174 us whole and 245 us in four segments."""
    import ctypes

    from nesle_amd import abi

    a = abi.DeltaArgs(abi.MEM_BF16, tokens, heads, 1, 1, dim, dim, 1.0)
    assert (abi.lib().nesle_delta_forward_scratch_floats(ctypes.byref(a)) > 0) == cut
