"""Every compiled kernel of linear attention, layer norm and sampling is one that a call
reaches, and workspaces have the sizes that the kernels use (no GPU needed)."""

from __future__ import annotations

import ctypes
import re
from pathlib import Path

import pytest

from nesle_amd import abi, build
from tests.test_kernel_resources import HIPCC, _kernels
from tests.test_more_memory import decay_args


@pytest.mark.skipif(not Path(HIPCC).exists(), reason="hipcc not available")
@pytest.mark.parametrize("source,joins", [("mem_decay_fwd.hip", {("0", "16")}), ("mem_decay_bwd.hip", {("1", "1"), ("1", "16")})])
def test_only_joins_that_are_launched(source, joins, tmp_path):
    """Forward, up to 16 segments are joined by the walk itself, so the join of few is the
    gradient's alone."""
    names = "\n".join(_kernels(build.CSRC / source, tmp_path))
    assert set(re.findall(r"decay_join_kernelILb([01])ELi(\d+)E", names)) == joins


@pytest.mark.skipif(not Path(HIPCC).exists(), reason="hipcc not available")
def test_only_shapes_of_rows_that_are_chosen(tmp_path):
    """A row takes the first shape, of (lanes, vectors a lane), that holds it in at most 32
    elements a lane."""
    shapes = [(16, 1), (16, 2), (64, 1), (64, 2), (64, 4), (64, 8), (256, 4), (256, 8), (1024, 2), (1024, 4), (1024, 16)]
    want = set()
    for dtype, vectors in (("f", (1, 4)), ("DF16b", (1, 8))):
        for v in vectors:
            for dim in range(v, abi.NORM_MAX_DIM + 1, v):
                lanes, n = next(s for s in shapes if s[0] * s[1] * v >= dim and s[1] * v <= 32)
                want |= {(kernel, dtype, str(v), str(n), str(lanes)) for kernel in ("layer_norm", "layer_norm_grad")}
    names = "\n".join(_kernels(build.CSRC / "mem_norm.hip", tmp_path))
    assert set(re.findall(r"(layer_norm|layer_norm_grad)_kernelI(f|DF16b)Li(\d+)ELi(\d+)ELi(\d+)E", names)) == want


@pytest.mark.parametrize("steps", [4, 500, 5000])
@pytest.mark.parametrize("groups", [1, 2])
def test_gradient_workspace(groups, steps):
    """Shares of key heads' gradients, segments' states with a flag each, and a float64 a
    workgroup, of a head's part in a segment, on a boundary of its own."""
    a = decay_args(steps=steps, batch=2, k_heads=4 // groups, v_heads=4, k_dim=24, v_dim=16)
    floats = abi.lib().nesle_decay_scratch_floats(ctypes.byref(a))
    heads = 2 * 4
    shares = 0 if groups == 1 else 2 * steps * heads * 24
    spans = (steps + 63) // 64
    segments = 1 if spans < 8 else -(-spans // -(-spans // min(spans, 128, 1024 // heads)))
    states = 0 if segments == 1 else segments * heads * (24 * 16 + 1)
    assert floats == shares + (states + 1) // 2 * 2 + 2 * segments * heads
