"""Compiled resources of the kernels of linear attention with a decay, layer norm and
sampling (no GPU needed): the forward kernels and steps use no scratch memory, and LDS
lets two workgroups share a compute unit's 160 KB where the launches count on it: every
forward kernel, and the gradient of up to 64 bfloat16 dimensions."""

from __future__ import annotations

import re
from pathlib import Path

import pytest

from nesle_amd import build
from tests.test_kernel_resources import HIPCC, _kernels

pytestmark = pytest.mark.skipif(not Path(HIPCC).exists(), reason="hipcc not available")


@pytest.mark.parametrize("source", ["mem_decay_fwd.hip", "mem_decay_bwd.hip", "mem_decay_step.hip", "mem_norm.hip", "mem_sample.hip"])
def test_resources(source, tmp_path):
    kernels = _kernels(build.CSRC / source, tmp_path)
    assert kernels
    for name, v in kernels.items():
        lds, scratch = v["group_segment_fixed_size"], v["private_segment_fixed_size"]
        gradient = "backward" in name
        assert lds <= (80 if not gradient or re.search("DF16bLi(32|64)E", name) else 160) * 1024, (name, lds)
        if not any(n in name for n in ("backward", "grad", "sample")):
            assert scratch == 0, (name, scratch)
        assert scratch <= 256, (name, scratch)
