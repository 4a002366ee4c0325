"""Linear attention with a decay, layer norm and sampling without a GPU: the C
entry points and the binding refuse what they cannot take, and the structures are
laid out as the header has them."""

from __future__ import annotations

import ctypes
import math
import re
import shutil
import subprocess

import pytest
import torch
import torch.autograd.forward_ad as fwAD

from nesle_amd import abi, memory


def refusal(fn, args, why):
    assert fn(None if args is None else ctypes.byref(args), None) == abi.EINVAL, why
    assert why in abi.lib().nesle_last_error().decode()


def with_(a, **kw):
    for name, value in kw.items():
        setattr(a, name, value)
    return a


def decay_args(**kw):
    return with_(abi.DecayArgs(abi.MEM_F32, 4, 2, 2, 4, 16, 16, 1.0), **kw)


@pytest.mark.parametrize("entry", ["nesle_decay_forward", "nesle_decay_backward", "nesle_decay_step"])
def test_decay_entries_refuse(entry):
    fn = getattr(abi.lib(), entry)
    steps = 1 if entry == "nesle_decay_step" else 4
    refusal(fn, None, "null arguments")
    for bad, why in (({"dtype": 7}, "dtype"), ({"k_dim": 12}, "multiples of 8"), ({"v_dim": 0}, "multiples of 8"),
                     ({"v_dim": 136}, "multiples of 8"), ({"v_heads": 3}, "multiple of k_heads"),
                     ({"k_heads": 0}, "multiple of k_heads"), ({"batch": 1 << 31}, "at most"), ({}, "null device pointer")):
        refusal(fn, decay_args(**{"steps": steps, **bad}), why)
    if entry == "nesle_decay_step":
        refusal(fn, decay_args(steps=2), "steps must be 1")
    else:
        refusal(fn, decay_args(steps=(1 << 30) + 1), "2^30")
    assert fn(ctypes.byref(decay_args(steps=steps, batch=0)), None) == abi.OK
    a = decay_args(steps=steps, g=8, state=8, state_out=16, out=16)
    for n in "qkv":
        setattr(a, n, abi.Heads(16, 1, 1, 1))
    refusal(fn, a, "16-byte")
    if entry != "nesle_decay_step":        # without a token too
        refusal(fn, decay_args(steps=0, state=8, state_out=16), "16-byte")
        refusal(fn, decay_args(steps=0, state_out=16, dg=16, scratch=8), "16-byte")


def test_decay_workspaces():
    L = abi.lib()
    # The state before every span of tokens but the first.
    for dtype, dim, span in ((abi.MEM_F32, 64, 64), (abi.MEM_F32, 72, 32), (abi.MEM_BF16, 64, 64), (abi.MEM_BF16, 72, 64)):
        assert L.nesle_decay_saved_floats(ctypes.byref(decay_args(dtype=dtype, steps=span, k_dim=dim))) == 0
        assert L.nesle_decay_saved_floats(ctypes.byref(decay_args(dtype=dtype, steps=2 * span + 1, k_dim=dim))) == 2 * 2 * 4 * dim * 16
    # Shares of key heads' gradients, and one float a workgroup.
    one = L.nesle_decay_scratch_floats(ctypes.byref(decay_args(k_heads=4)))
    assert one >= 2 * 4
    assert L.nesle_decay_scratch_floats(ctypes.byref(decay_args())) == one + 2 * 4 * 2 * 4 * 16


def norm_args(**kw):
    return with_(abi.NormArgs(abi.MEM_F32, 4, 2, 3, 16, 1e-5), **kw)


@pytest.mark.parametrize("entry", ["nesle_layer_norm", "nesle_layer_norm_grad"])
def test_norm_entries_refuse(entry):
    fn = getattr(abi.lib(), entry)
    refusal(fn, None, "null arguments")
    grad = entry.endswith("grad")
    for bad, why in (({"dtype": 2}, "dtype"), ({"dim": 0}, "dim"), ({"dim": 16385}, "dim"), ({"eps": -1.0}, "eps"),
                     ({"eps": math.nan}, "eps"), ({"eps": math.inf}, "eps"), ({"steps": 1 << 16, "batch": 1 << 16}, "rows"),
                     ({"batch": (1 << 32) - 1, "heads": (1 << 32) - 1}, "rows"), ({}, "null device pointer")):
        refusal(fn, norm_args(**bad), why)
    refusal(fn, norm_args(x=abi.Heads(16, 1, 1, 1), y=16, weight=8, dy=abi.Heads(16, 1, 1, 1), dx=16), "16-byte")
    if grad:
        refusal(fn, norm_args(x=abi.Heads(16, 1, 1, 1), dy=abi.Heads(16, 1, 1, 1), dx=16, dweight=16), "null device pointer")
        refusal(fn, norm_args(steps=0, dweight=16), "null device pointer")
    for empty in ({"steps": 0}, {"batch": 0}, {"heads": 0}):
        assert fn(ctypes.byref(norm_args(**empty)), None) == abi.OK
    for dim in (0, 16385, 0xffffffff):
        assert abi.lib().nesle_norm_scratch_floats(ctypes.byref(norm_args(dim=dim))) == 0


def sample_args(**kw):
    return with_(abi.SampleArgs(abi.MEM_F32, 1, 4, 12, abi.Heads(16, 0, 12, 0), 16, 1.0, 1.0, 0.0, 0), action=16, logprob=16, **kw)


def test_sample_refuses():
    fn = abi.lib().nesle_sample
    refusal(fn, None, "null arguments")
    for bad, why in (({"dtype": 3}, "dtype"), ({"actions": 0}, "actions"), ({"actions": 1025}, "actions"),
                     ({"steps": 1 << 16, "batch": 1 << 16}, "rows"), ({"temperature": -1.0}, "temperature"),
                     ({"temperature": math.nan}, "temperature"), ({"temperature": math.inf}, "temperature"),
                     ({"top_p": 0.0}, "top_p"), ({"top_p": 1.01}, "top_p"), ({"top_p": math.nan}, "top_p"),
                     ({"min_p": -0.1}, "min_p"), ({"min_p": 1.1}, "min_p"), ({"min_p": math.nan}, "min_p"),
                     ({"uniform": None}, "null device pointer"), ({"logits": abi.Heads()}, "null device pointer")):
        refusal(fn, sample_args(**bad), why)
    for empty in ({"steps": 0}, {"batch": 0}):
        assert fn(ctypes.byref(sample_args(**empty)), None) == abi.OK


def test_structures_and_limits_match_the_header(tmp_path):
    text = (abi.INCLUDE / "nesle_memory.h").read_text()
    found = dict(re.findall(r"#define (NESLE_\w+) (\d+)u", text))
    assert int(found["NESLE_DECAY_MAX_DIM"]) == abi.DECAY_MAX_DIM
    assert int(found["NESLE_NORM_MAX_DIM"]) == abi.NORM_MAX_DIM
    assert int(found["NESLE_SAMPLE_MAX_ACTIONS"]) == abi.SAMPLE_MAX_ACTIONS
    cc = shutil.which("gcc")
    if cc is None:
        pytest.skip("no C compiler")
    structs = {"nesle_decay_args": abi.DecayArgs, "nesle_norm_args": abi.NormArgs, "nesle_sample_args": abi.SampleArgs}
    lines = []
    for name, cls in structs.items():
        lines.append(f'printf("{name} %zu\\n", sizeof({name}));')
        lines += [f'printf("{name}.{f[0]} %zu\\n", offsetof({name}, {f[0]}));' for f in cls._fields_]
    src = tmp_path / "layout.c"
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "nesle_memory.h"\nint main(void) {\n'
                   + "\n".join(lines) + "\nreturn 0;\n}\n")
    subprocess.run([cc, f"-I{abi.INCLUDE}", "-o", str(tmp_path / "layout"), str(src)], check=True)
    got = dict(line.rsplit(" ", 1) for line in subprocess.run([str(tmp_path / "layout")], check=True, capture_output=True,
                                                              text=True).stdout.splitlines())
    for name, cls in structs.items():
        assert int(got[name]) == ctypes.sizeof(cls)
        for field, _ in cls._fields_:
            assert int(got[f"{name}.{field}"]) == getattr(cls, field).offset, f"{name}.{field}"


def calls():
    """Each operator as a function of its tensors, and those tensors (on the CPU,
    which is refused last)."""
    q, g, state = torch.zeros(2, 3, 1, 16), torch.zeros(1), torch.zeros(3, 1, 16, 16)
    return {
        "decay_attention": (lambda q, k, v, g, s: memory.decay_attention(q, k, v, g, state=s)[0],
                            [q, q.clone(), q.clone(), g, state]),
        "decay_attention_step": (lambda q, k, v, g, s: memory.decay_attention_step(q, k, v, g, s),
                                 [q[0], q[1], q[0].clone(), g, state.clone()]),
        "layer_norm": (lambda x, w, b: memory.layer_norm(x, w, b), [q, torch.ones(16), torch.zeros(16)]),
        "sample_actions": (lambda x, u: memory.sample_actions(x, u)[1], [torch.zeros(2, 3, 5), torch.zeros(2, 3)]),
    }


NAMES = ["decay_attention", "decay_attention_step", "layer_norm", "sample_actions"]


@pytest.mark.parametrize("name", NAMES)
def test_what_the_binding_refuses(name):
    from torch.fx.experimental.proxy_tensor import make_fx

    fn, inputs = calls()[name]
    with pytest.raises(ValueError, match="GPU"):
        fn(*inputs)
    with pytest.raises(ValueError, match=name):
        fn(None, *inputs[1:])
    for i, t in enumerate(inputs):
        with fwAD.dual_level():
            args = list(inputs)
            args[i] = fwAD.make_dual(t.clone(), torch.ones_like(t))
            with pytest.raises(ValueError, match=f"{name} has no forward-mode derivative"):
                fn(*args)
    with pytest.raises(ValueError, match=f"{name} cannot be traced"):
        torch.jit.trace(fn, tuple(inputs), check_trace=False)
    with pytest.raises(ValueError, match=f"{name} cannot be traced"):
        make_fx(fn)(*inputs)


@pytest.mark.parametrize("name", NAMES)
def test_sizes_of_more_than_32_bits_are_refused(name):
    """An expanded tensor takes no memory, so such a size is within reach; cut to
    32 bits it would pass every later check."""
    fn, inputs = calls()[name]
    first = "qx"["norm" in name] if "sample" not in name else "logits"
    for size in (1 << 32, (1 << 32) + 2):
        for dim in range(inputs[0].dim() - 1):
            q = inputs[0][tuple(slice(0, 1) if d == dim else slice(None) for d in range(inputs[0].dim()))]
            q = q.expand(*(size if d == dim else n for d, n in enumerate(q.shape)))
            rest = [q if t.shape == inputs[0].shape else t for t in inputs[1:]]
            with pytest.raises(ValueError, match=f"{name}: {first} must be of sizes below 2\\^32"):
                fn(q, *rest)
