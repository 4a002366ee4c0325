"""The states that linear attention's forward keeps for its gradient lie as many tokens
apart as both count on and as the workspace is sized for, whatever the strides of the
tensors of either call (no GPU needed)."""

from __future__ import annotations

import ctypes
import itertools
import re
from pathlib import Path

import pytest

from nesle_amd import abi, build
from tests.test_kernel_resources import HIPCC, _kernels

FAR = 1 << 30          # elements from step to step: past what 32-bit offsets reach within a chunk


def span(dtype: int, dim: int) -> int:
    """Tokens between two kept states: by type and padded dimension."""
    return 32 if dtype == abi.MEM_F32 and dim > 64 else 64


@pytest.mark.parametrize("dtype", [abi.MEM_F32, abi.MEM_BF16])
@pytest.mark.parametrize("dims", [(8, 8), (32, 16), (40, 64), (64, 64), (64, 72), (128, 128)])
def test_kept_states_do_not_depend_on_strides(dims, dtype):
    every = span(dtype, max(dims))
    for T in (1, 32, 33, 64, 65, 66, 96, 97, 128, 130):
        want = (T + every - 1) // every - 1        # the state before every span but the first
        for far in itertools.product((96, FAR), repeat=4):
            a = abi.DecayArgs(dtype, T, 2, 1, 2, *dims, 1.0)
            for name, stride in zip(("q", "k", "v", "dout"), far):
                setattr(a, name, abi.Heads(16, stride, 96, 48))
            assert abi.lib().nesle_decay_saved_floats(ctypes.byref(a)) == want * 2 * 2 * dims[0] * dims[1], (T, far)


@pytest.mark.skipif(not Path(HIPCC).exists(), reason="hipcc not available")
@pytest.mark.parametrize("source,kernel", [("mem_decay_fwd.hip", "decay_forward_kernel"), ("mem_decay_bwd.hip", "decay_backward_kernel")])
def test_far_strides_have_kernels_of_each_dimension(source, kernel, tmp_path):
    """The spacing is a kernel's own, by the type and the dimension that it is made for, so
    the ones for far strides are made for the same dimensions as the others: the float32
    one of 128 dimensions in place of one of 32 or 64 counts half as many tokens."""
    names = "\n".join(_kernels(build.CSRC / source, tmp_path))
    found = set(re.findall(kernel + r"I(f|DF16b)Li(\d+)ELb([01])E", names))
    assert found == set(itertools.product(("f", "DF16b"), ("32", "64", "128"), "01"))
