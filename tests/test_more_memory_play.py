"""What playing a policy with memory (nesle_amd.memory_ppo.play) refuses, as the trainer
does (no GPU needed)."""

from __future__ import annotations

import pytest
import torch

from nesle_amd import memory_ppo as M


@pytest.mark.parametrize("bad,why", [({"reward_mode": "smart"}, "reward_mode"), ({"reward_mode": "none"}, "reward_mode"),
                                     ({"flag_bonus": 1.0}, "flag_bonus"), ({"finish_zone_bonus": 0.0}, "finish_zone_bonus"),
                                     ({"death_penalty": 5.0}, "death_penalty")])
def test_the_shaped_reward_is_refused(bad, why):
    config = M.MemoryPPOConfig("x", **bad)
    for call in (lambda: M.play(config, 3), lambda: M.train_memory_ppo(config)):
        with pytest.raises(ValueError, match=why):
            call()


@pytest.mark.skipif(torch.cuda.is_available(), reason="there is a GPU")
def test_without_a_gpu():
    for call in (lambda: M.play(M.MemoryPPOConfig("x"), 3), lambda: M.train_memory_ppo(M.MemoryPPOConfig("x"))):
        with pytest.raises(SystemExit, match="needs a GPU"):
            call()
