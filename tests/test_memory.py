"""The memory operators without a GPU: the C entry points refuse what they
cannot take, their structures are laid out as the header has them, and the
rotation table is its formula."""

from __future__ import annotations

import ctypes
import math
import re
import shutil
import subprocess
from pathlib import Path

import pytest
import torch

from nesle_amd import abi, build, memory


def _delta(**kw):
    a = abi.DeltaArgs(abi.MEM_F32, 4, 2, 2, 4, 16, 16, 1.0)
    for name, value in kw.items():
        setattr(a, name, value)
    return a


@pytest.mark.parametrize("entry", ["nesle_delta_forward", "nesle_delta_backward", "nesle_delta_step"])
def test_delta_entries_refuse(entry):
    fn = getattr(abi.lib(), entry)
    steps = 1 if entry == "nesle_delta_step" else 4
    assert fn(None, None) == abi.EINVAL
    for bad, why in (({"dtype": 7}, "dtype"), ({"k_dim": 12}, "multiples of 8"), ({"v_dim": 0}, "multiples of 8"),
                     ({"v_dim": 136}, "multiples of 8"), ({"v_heads": 3}, "multiple of k_heads"),
                     ({"k_heads": 0}, "multiple of k_heads"), ({"batch": 1 << 31}, "at most"), ({}, "null device pointer")):
        assert fn(ctypes.byref(_delta(**{"steps": steps, **bad})), None) == abi.EINVAL, bad
        assert why in abi.lib().nesle_last_error().decode()
    if entry == "nesle_delta_step":
        assert fn(ctypes.byref(_delta(steps=2)), None) == abi.EINVAL
    assert fn(ctypes.byref(_delta(steps=steps, batch=0)), None) == abi.OK
    a = _delta(steps=steps, g=8, beta=8, state=8, state_out=16, out=16)
    for n in "qkv":
        setattr(a, n, abi.Heads(16, 1, 1, 1))
    assert fn(ctypes.byref(a), None) == abi.EINVAL
    assert "16-byte" in abi.lib().nesle_last_error().decode()


def test_delta_workspaces():
    L = abi.lib()
    assert L.nesle_delta_saved_floats(ctypes.byref(_delta(steps=32))) == 0
    assert L.nesle_delta_saved_floats(ctypes.byref(_delta(steps=33, k_dim=40))) == 2 * 4 * 40 * 16
    assert L.nesle_delta_scratch_floats(ctypes.byref(_delta())) == 2 * 4 * 2 * 4 * 16
    assert L.nesle_delta_scratch_floats(ctypes.byref(_delta(k_heads=4))) == 0
    assert L.nesle_delta_forward_scratch_floats(ctypes.byref(_delta(steps=128))) == 0
    assert L.nesle_delta_forward_scratch_floats(ctypes.byref(_delta(steps=4096, batch=4096))) == 0
    assert L.nesle_delta_forward_scratch_floats(ctypes.byref(_delta(steps=4096))) > 0


@pytest.mark.parametrize("entry", ["nesle_qk_norm_rotate", "nesle_qk_norm_rotate_grad"])
def test_qk_entries_refuse(entry):
    fn = getattr(abi.lib(), entry)
    assert fn(None, None) == abi.EINVAL

    def args(**kw):
        a = abi.QkArgs(abi.MEM_F32, 4, 2, 2, 2, 16, 0, 0, 0, 1e-6)
        for name, value in kw.items():
            setattr(a, name, value)
        return a

    for bad, why in (({"dtype": 2}, "dtype"), ({"dim": 12}, "dim"), ({"dim": 264}, "dim"), ({"rotated": 24}, "rotated"),
                     ({"rotated": 4}, "rotated"), ({"rotated": 8}, "positions"), ({"eps": -1.0}, "eps"),
                     ({"eps": math.nan}, "eps"), ({"q_heads": 0, "k_heads": 0}, "heads"),
                     ({"steps": 1 << 31, "batch": 1 << 31}, "elements"), ({"q_out": 8}, "16-byte"),
                     ({"q_heads": 5000}, "heads"), ({}, "null device pointer")):
        assert fn(ctypes.byref(args(**bad)), None) == abi.EINVAL, bad
        assert why in abi.lib().nesle_last_error().decode(), bad
    if entry.endswith("grad"):
        assert fn(ctypes.byref(args(q_weight=16)), None) == abi.EINVAL
    assert fn(ctypes.byref(args(steps=0)), None) == abi.OK


def test_structures_match_the_header(tmp_path):
    """Sizes and offsets of the ctypes structures against the compiler's."""
    cc = shutil.which("gcc")
    if cc is None:
        pytest.skip("no C compiler")
    structs = {"nesle_heads": abi.Heads, "nesle_qk_args": abi.QkArgs, "nesle_delta_args": abi.DeltaArgs}
    lines = []
    for name, cls in structs.items():
        lines.append(f'printf("{name} %zu\\n", sizeof({name}));')
        lines += [f'printf("{name}.{f[0]} %zu\\n", offsetof({name}, {f[0]}));' for f in cls._fields_]
    src = tmp_path / "layout.c"
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "nesle_memory.h"\nint main(void) {\n'
                   + "\n".join(lines) + "\nreturn 0;\n}\n")
    exe = tmp_path / "layout"
    subprocess.run([cc, f"-I{abi.INCLUDE}", "-o", str(exe), str(src)], check=True)
    got = dict(line.rsplit(" ", 1) for line in subprocess.run([str(exe)], check=True, capture_output=True,
                                                              text=True).stdout.splitlines())
    for name, cls in structs.items():
        assert int(got[name]) == ctypes.sizeof(cls)
        for field, _ in cls._fields_:
            assert int(got[f"{name}.{field}"]) == getattr(cls, field).offset, f"{name}.{field}"


def test_constants_match_the_header():
    text = (abi.INCLUDE / "nesle_memory.h").read_text()
    found = dict(re.findall(r"#define (NESLE_\w+) (\d+)u", text))
    assert int(found["NESLE_MEM_F32"]) == abi.MEM_F32 and int(found["NESLE_MEM_BF16"]) == abi.MEM_BF16
    assert int(found["NESLE_QK_MAX_DIM"]) == abi.QK_MAX_DIM
    assert int(found["NESLE_DELTA_MAX_DIM"]) == abi.DELTA_MAX_DIM
    assert int(found["NESLE_DELTA_CHUNK"]) == abi.DELTA_CHUNK


def test_rotation_table():
    t = memory.rotation_table(7, 8, base=100.0, device="cpu")
    assert t.shape == (7, 8) and t.dtype == torch.float32
    for p in range(7):
        for i in range(4):
            angle = p * 100.0 ** (-2 * i / 8)
            assert abs(float(t[p, i]) - math.cos(angle)) <= 2.0 ** -24
            assert abs(float(t[p, 4 + i]) - math.sin(angle)) <= 2.0 ** -24


def test_cpu_tensors_are_refused():
    q = torch.zeros(3, 2, 16)
    with pytest.raises(ValueError, match="GPU"):
        memory.qk_norm_rotate(q, q)
    with pytest.raises(ValueError, match="GPU"):
        memory.gated_delta_step(q, q, q, q[..., 0], q[..., 0], torch.zeros(3, 2, 16, 16))


def test_delta_kernels_share_a_compute_unit(tmp_path):
    """The gradient's LDS leaves room for two workgroups of heads of 64 on a
    compute unit's 160 KB, the bfloat16 forward's for four; up to 64 dimensions
    nothing spills."""
    from test_kernel_resources import HIPCC, _kernels

    if not Path(HIPCC).exists():
        pytest.skip("hipcc not available")
    for source, lds in (("mem_delta_fwd.hip", {"IDF16bLi64": 40, "IfLi64": 80}),
                        ("mem_delta_bwd.hip", {"IDF16bLi64": 80, "IfLi64": 80})):
        kernels = {k: v for k, v in _kernels(build.CSRC / source, tmp_path).items() if "ward_kernel" in k}
        for kind, most in lds.items():
            of_kind = [v for k, v in kernels.items() if kind in k]
            assert of_kind and all(v["group_segment_fixed_size"] <= most << 10 for v in of_kind), source
        assert all(v["private_segment_fixed_size"] == 0 for k, v in kernels.items() if "Li128" not in k), source
