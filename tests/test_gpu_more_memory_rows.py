"""Sampling (nesle_amd.memory.sample_actions) of as many rows as it says it takes."""

from __future__ import annotations

import pytest
import torch

from tests.helpers import say
from tests.test_gpu_more_memory import dev

pytestmark = pytest.mark.gpu

TILE = 1 << 20


@pytest.mark.parametrize("rows,count", [((1 << 28) - 1, 12), (1 << 28, 12), ((1 << 28) + 5, 1), (1 << 30, 5), (1 << 30, 17),
                                        ((1 << 29) + 77, 70)])
def test_many_rows(rows, count):
    """2^28 rows of 16 lanes and 2^30 of a sixteenth of a wave are 2^32 threads.  All rows
    have the same logits and their numbers repeat every 2^20: so do the answers."""
    from nesle_amd import memory

    say(f"[gpu] sample_actions {rows} rows of {count}")
    gen = torch.Generator().manual_seed(count)
    logits = torch.randn(count, generator=gen).to(dev())
    some = torch.rand(TILE, generator=gen).to(dev())
    want = memory.sample_actions(logits.expand(TILE, count), some)
    u = some.repeat((rows + TILE - 1) // TILE)[:rows]
    actions, logprobs = memory.sample_actions(logits.expand(rows, count), u)
    del u
    for start in range(0, rows, 64 * TILE):
        for got, one in ((actions, want[0]), (logprobs, want[1])):
            part = got[start:start + 64 * TILE]
            whole = len(part) // TILE * TILE
            assert bool((part[:whole].view(-1, TILE) == one).all()), start
            assert torch.equal(part[whole:], one[:len(part) - whole]), start


def test_more_rows_than_that_are_refused():
    from nesle_amd import memory

    one = torch.zeros(1, device=dev())
    with pytest.raises(ValueError, match="rows must be at most 2\\^30"):
        memory.sample_actions(one[:, None].expand((1 << 30) + 1, 1), torch.empty((1 << 30) + 1, device=dev()))
