"""The policy with memory and its trainer (nesle_amd.memory_ppo): acting step by
step and evaluating the rollout give the same policy, and an update learns."""

from __future__ import annotations

import math

import pytest
import torch

from nesle_amd import synthrom
from tests.helpers import say

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_acting_and_training_see_the_same_policy(dtype):
    """The log probabilities and values a rollout recorded while acting are
    those of ``forward`` over the rollout, episodes ending inside.  Float32:
    both run the same formulas in a different order (1e-5 of values of order
    1); bfloat16: the layer's inputs and outputs round to 2^-8."""
    from nesle_amd import memory_ppo as M
    from nesle_amd import native_ppo as P
    from oracle import oracle as O
    from tests.helpers import warm_snapshots

    say(f"[gpu] memory ppo {dtype}")
    checked = []

    def check(update, b):
        with torch.no_grad():
            logits, values, _ = b["model"](b["obs"], b["steps"], b["resets"], b["state"])
        logp = torch.log_softmax(logits, -1).gather(-1, b["actions"][..., None]).squeeze(-1)
        worst = max(float((logp - b["logprobs"]).abs().max()), float((values - b["values"]).abs().max()))
        assert worst <= (1e-5 if dtype == "float32" else 2.0 ** -6), (update, worst)
        assert int(b["resets"][1:].sum()) > 0 and bool(b["steps"][b["resets"]].eq(0).all())
        checked.append(update)

    reward = dict(kind="x_delta", x_lo=synthrom.X_LO, x_hi=synthrom.X_HI, done_addr=synthrom.DONE_BYTE, clip=15,
                  time_penalty=0.25)
    cfg = M.MemoryPPOConfig("synthetic.nes", num_envs=48, n_steps=40, batch_size=640, update_epochs=2,
                            total_timesteps=2 * 48 * 40, action_space="complex", reward=reward, memory_dtype=dtype, seed=4)
    rom = synthrom.make_rom(5).rom
    snaps = warm_snapshots(rom, [100, 150, 200, 250], seed=55)
    for i, s in enumerate(snaps):
        s[O.OFF["ram"] + synthrom.DONE_BYTE] = 5 + 3 * i
    stats = M.train_memory_ppo(cfg, batch=P.make_batch(cfg, rom, [bytes(s) for s in snaps]), on_rollout=check)
    assert checked == [1, 2] and stats["updates"] == 2 and all(math.isfinite(x["loss"]) for x in stats["log"])
    torch.manual_seed(cfg.seed)
    fresh = M.MemoryActorCritic(12, dtype=getattr(torch, dtype))
    still = [n for (n, a), b in zip(fresh.named_parameters(), stats["model"].parameters()) if torch.equal(a, b)]
    assert not still, still


def test_refusals():
    from nesle_amd import memory_ppo as M

    with pytest.raises(ValueError, match="batch_size"):
        M.train_memory_ppo(M.MemoryPPOConfig("x", num_envs=4, n_steps=128, batch_size=64))
    with pytest.raises(ValueError, match="reward_mode"):
        M.train_memory_ppo(M.MemoryPPOConfig("x", reward_mode="smart"))
