"""Options of the trainer of a policy with memory (nesle_amd.memory_ppo) that it
shares with native_ppo's: each is honoured."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from nesle_amd import synthrom
from oracle import oracle as O
from tests.helpers import OracleBatch, say, warm_snapshots

pytestmark = pytest.mark.gpu

REWARD = dict(kind="x_delta", x_lo=synthrom.X_LO, x_hi=synthrom.X_HI, done_addr=synthrom.DONE_BYTE, clip=15,
              time_penalty=0.25)


def trainer(**kw):
    """(config, ROM, snapshots) of a small run on the synthetic game."""
    from nesle_amd import memory_ppo as M

    rom = synthrom.make_rom(5).rom
    snaps = warm_snapshots(rom, [100, 150, 200, 250], seed=55)
    for i, s in enumerate(snaps):
        s[O.OFF["ram"] + synthrom.DONE_BYTE] = 3 + 4 * i
    return M.MemoryPPOConfig("synthetic.nes", **{**dict(
        num_envs=16, n_steps=12, batch_size=96, update_epochs=1, total_timesteps=2 * 16 * 12, action_space="complex",
        reward=REWARD, seed=4, save_checkpoints=False), **kw}), rom, [bytes(s) for s in snaps]


@pytest.mark.parametrize("most", [0, 5])
def test_episodes_end_at_the_step_limit(most):
    """Consoles, steps of the episode and resets are those of oracle consoles under
    the same actions, put back where an episode ended by itself or by the limit."""
    from nesle_amd import memory_ppo as M

    say(f"[gpu] memory ppo, max_episode_steps={most}")
    cfg, rom, snaps = trainer(max_episode_steps=most)
    seen = []
    M.train_memory_ppo(cfg, rom_bytes=rom, snapshot_bytes=snaps, on_rollout=lambda u, b: seen.append(
        {k: b[k].cpu().numpy().copy() for k in ("actions", "rewards", "steps", "resets", "obs")}))
    run = {k: np.concatenate([s[k] for s in seen]) for k in seen[0]}
    masks = np.asarray(M._actions.action_masks("complex"), dtype=np.uint8)
    n, levels = cfg.num_envs, np.arange(cfg.num_envs) % len(snaps)
    ob = OracleBatch(rom, list(range(n)), reward=dict(REWARD, kind=1))
    for e, c in enumerate(ob.cons):
        c.load(np.frombuffer(snaps[levels[e]], dtype=np.uint8))
    first_ram = np.stack([np.frombuffer(s, dtype=np.uint8)[O.OFF["ram"]:O.OFF["ram"] + 2048] for s in snaps])[levels]
    done, length, by_limit = np.ones(n, dtype=bool), np.zeros(n, dtype=np.int64), 0
    for t in range(len(run["steps"])):
        length = np.where(done, 0, length)
        np.testing.assert_array_equal(run["resets"][t], done, err_msg=f"step {t}")
        np.testing.assert_array_equal(run["steps"][t], length, err_msg=f"step {t}")
        np.testing.assert_array_equal(run["obs"][t][done], first_ram[done], err_msg=f"step {t}")
        _, want, ended = ob.step(masks[run["actions"][t]], 4)
        np.testing.assert_array_equal(run["rewards"][t], want, err_msg=f"step {t}")
        length += 1
        late = (length >= most) & ~ended.astype(bool) if most else np.zeros(n, dtype=bool)
        by_limit += int(late.sum())
        done = ended.astype(bool) | late
        for e in np.nonzero(done)[0]:
            ob.cons[e].load(np.frombuffer(snaps[levels[e]], dtype=np.uint8))
    assert (by_limit > 0) == (most > 0)


def test_checkpoints_are_written_and_read(tmp_path):
    """The model and optimizer of the last update, and a run that goes on from them."""
    from nesle_amd import memory_ppo as M

    say("[gpu] memory ppo, checkpoints")
    path = tmp_path / "made" / "memory.pt"
    cfg, rom, snaps = trainer(save_checkpoints=True, checkpoint_path=str(path))
    stats = M.train_memory_ppo(cfg, rom_bytes=rom, snapshot_bytes=snaps)
    kept = torch.load(path, weights_only=True)
    assert kept["global_step"] == stats["global_step"] == 2 * 16 * 12 and kept["config"]["heads"] == cfg.heads
    want = stats["model"].state_dict()
    assert kept["model"].keys() == want.keys() and all(torch.equal(kept["model"][k], want[k]) for k in want)

    seen = []
    cfg, _, _ = trainer(total_timesteps=3 * 16 * 12)
    after = M.train_memory_ppo(cfg, str(path), rom_bytes=rom, snapshot_bytes=snaps, on_rollout=lambda u, b: seen.append(
        {k: v.clone() for k, v in b["model"].state_dict().items()}))
    assert len(seen) == after["updates"] == 1 and after["global_step"] == 3 * 16 * 12
    assert all(torch.equal(seen[0][k], want[k].to(seen[0][k].device)) for k in want)
    assert torch.load(path, weights_only=True)["global_step"] == 2 * 16 * 12        # the second run saved nothing


@pytest.mark.parametrize("init", ["orthogonal", "xavier"])
def test_weights_start_as_asked(init):
    """Orthogonal rows, or values that reach xavier's bound and no further."""
    from nesle_amd import memory_ppo as M

    torch.manual_seed(0)
    model = M.MemoryActorCritic(12, init=init)
    w = model.encode.weight.detach().double()               # 256 x 2,048, gain sqrt(2)
    bound = 2.0 ** 0.5 * (6 / (256 + 2048)) ** 0.5
    assert (float(w.abs().max()) <= bound * (1 + 1e-6)) == (init == "xavier")
    square = w @ w.T
    square.diagonal().sub_(2.0)
    assert (float(square.abs().max()) < 1e-4) == (init == "orthogonal")


def test_log_lines_at_the_interval_and_the_end():
    from nesle_amd import memory_ppo as M

    say("[gpu] memory ppo, log_interval")
    cfg, rom, snaps = trainer(log_interval=2, total_timesteps=5 * 16 * 12, init="xavier")
    stats = M.train_memory_ppo(cfg, rom_bytes=rom, snapshot_bytes=snaps)
    assert stats["updates"] == 5 and [x["update"] for x in stats["log"]] == [2, 4, 5]


def test_options_that_would_have_no_effect_are_refused():
    from nesle_amd import memory_ppo as M

    for option in ("flag_bonus", "finish_zone_bonus", "death_penalty"):
        with pytest.raises(ValueError, match=option):
            M.train_memory_ppo(M.MemoryPPOConfig("x", **{option: 1.0}))
    with pytest.raises(ValueError, match="init"):
        M.MemoryActorCritic(12, init="zeros")


def test_observations_are_left_as_they_are():
    """Float observations too, which a cast would hand on as they lie; the policy
    sees the same."""
    from nesle_amd import memory_ppo as M

    model = M.MemoryActorCritic(12)
    ram = torch.randint(0, 256, (4, 2048), dtype=torch.uint8, generator=torch.Generator().manual_seed(1)).cuda()
    steps, resets = torch.zeros(4, dtype=torch.int32).cuda(), torch.ones(4, dtype=torch.bool).cuda()
    want = model.act(ram, steps, resets, model.new_state(4))
    obs = ram.float()
    got = model.act(obs, steps, resets, model.new_state(4))
    assert torch.equal(obs, ram.float())
    assert all(torch.equal(a, b) for a, b in zip(got, want))
