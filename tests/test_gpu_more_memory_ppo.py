"""The policy with linear attention as its memory, drawing its actions from given
random numbers (nesle_amd.memory_ppo): acting step by step and evaluating the rollout
give the same policy, an update learns, and a trained policy is played."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from nesle_amd import synthrom
from oracle import oracle as O
from tests.helpers import OracleBatch, say
from tests.test_gpu_memory_ppo_options import REWARD, trainer

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_acting_and_training_see_the_same_policy(dtype):
    """The log probabilities and values a rollout recorded while acting are those of
    ``forward`` over the rollout, episodes ending inside.

    The four heads' normed readouts have length 16 (each of its 64 elements is of mean
    square 1), and not 1; the merging layer keeps lengths, tanh shortens them and the
    critic's row has length 1 (all orthogonal at first, with gain 1), so an error of
    relative size e in the readouts moves a value by 16 e at most, and by 16 e / sqrt(256)
    = e on average where it does not favour a direction; 5 times that over a few thousand
    values.  Float32: e is 4e-6 of either side (test_gpu_more_memory.F32).  bfloat16: the
    readout and what the norm makes of it each round by 2^-9."""
    from nesle_amd import memory_ppo as M

    say(f"[gpu] memory ppo, decay, {dtype}")
    checked = []

    def check(update, b):
        with torch.no_grad():
            logits, values, _ = b["model"](b["obs"], b["steps"], b["resets"], b["state"])
        logp = torch.log_softmax(logits, -1).gather(-1, b["actions"][..., None]).squeeze(-1)
        worst = max(float((logp - b["logprobs"]).abs().max()), float((values - b["values"]).abs().max()))
        assert worst <= 5 * 2 * (4e-6 if dtype == "float32" else 2 * 2.0 ** -9), (update, worst)
        assert int(b["resets"][1:].sum()) > 0
        checked.append(update)

    cfg, rom, snaps = trainer(num_envs=48, n_steps=40, batch_size=640, update_epochs=2, total_timesteps=2 * 48 * 40,
                              memory="decay", sampler="uniform", memory_dtype=dtype)
    stats = M.train_memory_ppo(cfg, rom_bytes=rom, snapshot_bytes=snaps, on_rollout=check)
    assert checked == [1, 2] and stats["updates"] == 2 and all(math.isfinite(x["loss"]) for x in stats["log"])
    torch.manual_seed(cfg.seed)
    fresh = M.MemoryActorCritic(12, dtype=getattr(torch, dtype), memory="decay")
    still = [n for (n, a), b in zip(fresh.named_parameters(), stats["model"].parameters()) if torch.equal(a, b)]
    assert not still, still


@pytest.mark.parametrize("memory", ["delta", "decay"])
def test_a_policy_is_played(memory, tmp_path):
    """The consoles are oracle consoles under the same actions; temperature 0 and top_k 1
    are the same, likeliest actions; a checkpoint plays as the model does."""
    from nesle_amd import memory_ppo as M

    say(f"[gpu] memory ppo, play, {memory}")
    path = str(tmp_path / "policy.pt")
    cfg, rom, snaps = trainer(memory=memory, save_checkpoints=True, checkpoint_path=path, max_episode_steps=9)
    model = M.train_memory_ppo(cfg, rom_bytes=rom, snapshot_bytes=snaps)["model"]

    def run(**kw):
        seen = []
        got = M.play(cfg, 25, rom_bytes=rom, snapshot_bytes=snaps, on_step=lambda t, a, p: seen.append((a.clone(), p.clone())), **kw)
        return got, torch.stack([a for a, _ in seen]), torch.stack([p for _, p in seen])

    got, actions, logprobs = run(model=model, temperature=0.7, top_k=8, top_p=0.95)
    assert bool((logprobs <= 0).all()) and bool(logprobs.isfinite().all())
    masks = np.asarray(M._actions.action_masks("complex"), dtype=np.uint8)
    n, levels = cfg.num_envs, np.arange(cfg.num_envs) % len(snaps)
    ob = OracleBatch(rom, list(range(n)), reward=dict(REWARD, kind=1))
    for e, c in enumerate(ob.cons):
        c.load(np.frombuffer(snaps[levels[e]], dtype=np.uint8))
    total, episodes, length = np.zeros(n), np.zeros(n, dtype=np.int64), np.zeros(n, dtype=np.int64)
    for t in range(25):
        _, reward, ended = ob.step(masks[actions[t].cpu().numpy()], 4)
        total += reward
        length += 1
        over = ended.astype(bool) | (length >= 9)
        length[over] = 0
        episodes += over
        for e in np.nonzero(over)[0]:
            ob.cons[e].load(np.frombuffer(snaps[levels[e]], dtype=np.uint8))
    np.testing.assert_array_equal(got["episodes"].cpu().numpy(), episodes)
    np.testing.assert_allclose(got["rewards"].cpu().numpy(), total, atol=25 * 16 * 2.0 ** -23)
    again, same, _ = run(temperature=0.7, top_k=8, top_p=0.95)         # from the checkpoint
    assert torch.equal(actions, same) and torch.equal(again["rewards"], got["rewards"])
    greedy, narrow = run(model=model, temperature=0), run(model=model, top_k=1)
    assert torch.equal(greedy[1], narrow[1]) and bool((greedy[2] == 0).all()) and bool((narrow[2] == 0).all())


def test_undefined_logits_end_the_run(tmp_path):
    from nesle_amd import memory_ppo as M

    say("[gpu] memory ppo, logits that are not numbers")
    path = str(tmp_path / "policy.pt")
    cfg, rom, snaps = trainer(memory="decay", sampler="uniform", save_checkpoints=True, checkpoint_path=path)
    model = M.train_memory_ppo(cfg, rom_bytes=rom, snapshot_bytes=snaps)["model"]
    with torch.no_grad():
        model.actor.bias[3] = math.nan
    with pytest.raises(FloatingPointError, match="logits"):
        M.play(cfg, 2, model, rom_bytes=rom, snapshot_bytes=snaps)
    saved = torch.load(path, weights_only=True)
    saved["model"]["actor.bias"][3] = math.nan
    torch.save(saved, path)
    cfg.total_timesteps *= 2
    with pytest.raises(FloatingPointError, match="logits"):
        M.train_memory_ppo(cfg, resume_from=path, rom_bytes=rom, snapshot_bytes=snaps)


def test_options_are_checked(tmp_path):
    from nesle_amd import memory_ppo as M

    with pytest.raises(ValueError, match="sampler"):
        M.train_memory_ppo(M.MemoryPPOConfig("x", sampler="dice"))
    with pytest.raises(ValueError, match="memory"):
        M.MemoryActorCritic(12, memory="elephant")
    with pytest.raises(SystemExit, match="resume-from"):
        M.main(["x", "--play", "5"])


def test_command_plays(tmp_path, capsys):
    from nesle_amd import memory_ppo as M

    say("[gpu] memory ppo, command")
    rom, path = tmp_path / "game.nes", str(tmp_path / "p.pt")
    rom.write_bytes(synthrom.make_rom(5).rom)
    some = [str(rom), "--num-envs", "8", "--memory", "decay", "--sampler", "uniform"]
    M.main([*some, "--n-steps", "8", "--batch-size", "32", "--total-timesteps", "64", "--checkpoint-path", path])
    M.main([*some, "--resume-from", path, "--play", "6", "--temperature", "0.5", "--top-p", "0.9"])
    assert "steps=6" in capsys.readouterr().out
