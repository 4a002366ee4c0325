"""PPO with a policy that remembers its episode: the operators of
``nesle_amd.memory`` used together.

The policy of ``native_ppo`` sees one instant of RAM.  ``MemoryActorCritic``
puts a memory layer behind its first layer: queries, keys and values of 4 heads
of 64 from one projection, normed and rotated by the step of the episode
(``qk_norm_rotate``), through the gated delta rule.  It

* acts one token at a time (``act``: ``gated_delta_step``, the states of all
  consoles updated in place, dropped where an episode ended), and
* trains on whole rollouts of the consoles of a minibatch (``forward``:
  ``gated_delta`` from the states the rollout started with, gradients through
  both operators).

``train_memory_ppo`` is the trainer: the console batch, generalised advantage
estimation and the clipped loss head are ``native_ppo``'s.  Minibatches are
consoles with all their steps, as a memory's tokens belong together.

    python -m nesle_amd.memory_ppo game.nes --num-envs 512 --total-timesteps 10000000
"""

from __future__ import annotations

import argparse
import math
from dataclasses import dataclass

import torch
import torch.nn as nn
import torch.nn.functional as F

from nesle_amd import actions as _actions
from nesle_amd import memory
from nesle_amd import native_ppo as P


class MemoryActorCritic(nn.Module):
    """2,048 RAM bytes / 255 -> width tanh -> memory of ``heads`` heads -> width
    tanh -> action logits + value."""

    def __init__(self, action_dim: int, obs_dim: int = 2048, width: int = 256, heads: int = 4, head_dim: int = 64,
                 max_steps: int = 4096, dtype: torch.dtype = torch.float32, init: str = "orthogonal", device=None) -> None:
        super().__init__()
        if init not in ("orthogonal", "xavier"):
            raise ValueError(f"unknown init {init!r}: 'orthogonal' or 'xavier'")
        dev = device if device is not None else torch.device("cuda")
        self.heads, self.head_dim, self.dtype = heads, head_dim, dtype
        inner = heads * head_dim
        self.encode = nn.Linear(obs_dim, width, device=dev)
        self.project = nn.Linear(width, 3 * inner, device=dev)
        self.gates = nn.Linear(width, 2 * heads, device=dev)
        self.q_weight = nn.Parameter(torch.ones(head_dim, device=dev))
        self.k_weight = nn.Parameter(torch.ones(head_dim, device=dev))
        self.merge = nn.Linear(inner, width, device=dev)
        self.actor = nn.Linear(width, action_dim, device=dev)
        self.critic = nn.Linear(width, 1, device=dev)
        for layer, gain in ((self.encode, math.sqrt(2.0)), (self.project, 1.0), (self.gates, 0.1), (self.merge, 1.0),
                            (self.actor, 0.01), (self.critic, 1.0)):
            (nn.init.orthogonal_ if init == "orthogonal" else nn.init.xavier_uniform_)(layer.weight, gain)
            nn.init.zeros_(layer.bias)
        # Half lives of about 10 to 300 steps to begin with, one for each head.
        with torch.no_grad():
            rate = torch.logspace(math.log10(0.07), math.log10(0.0025), heads, device=dev)
            self.gates.bias[:heads] = torch.log(torch.expm1(rate))
        self.register_buffer("table", memory.rotation_table(max_steps, head_dim, device=dev), persistent=False)

    def new_state(self, num_envs: int) -> torch.Tensor:
        return torch.zeros(num_envs, self.heads, self.head_dim, self.head_dim, device=self.encode.weight.device)

    def _tokens(self, obs, steps):
        """(features, q, k, v, g, beta) of observations [..., obs_dim]."""
        x = torch.tanh(self.encode((obs / 255.0).float()))
        q, k, v = self.project(x).to(self.dtype).unflatten(-1, (3, self.heads, self.head_dim)).unbind(-3)
        # Unit norms (the rule wants keys of about unit length); the weights
        # scale the directions against each other.
        q, k = memory.qk_norm_rotate(q, k, self.q_weight, self.k_weight, positions=steps, table=self.table, unit=True)
        decay, write = self.gates(x).chunk(2, -1)
        return x, q, k, v, -F.softplus(decay), torch.sigmoid(write)

    def _heads_out(self, x, out):
        x = torch.tanh(x + self.merge(out.flatten(-2).float()))
        return self.actor(x), self.critic(x).squeeze(-1)

    def forward(self, obs, steps, resets, state):
        """(logits, values, state after) of a rollout: obs [T, N, obs_dim]
        uint8, steps int32 [T, N] (of the episode), resets [T, N] (its first
        step), state before it."""
        x, q, k, v, g, beta = self._tokens(obs, steps)
        out, state = memory.gated_delta(q, k, v, g, beta, state=state, resets=resets, scale=1.0)
        return (*self._heads_out(x, out), state)

    @torch.no_grad()
    def act(self, obs, steps, resets, state):
        """(logits, values) of one step of every console; ``state`` is updated."""
        x, q, k, v, g, beta = self._tokens(obs, steps)
        out = memory.gated_delta_step(q, k, v, g.contiguous(), beta.contiguous(), state, resets=resets, scale=1.0)
        return self._heads_out(x, out)


@dataclass
class MemoryPPOConfig(P.NativePPOConfig):
    """``native_ppo``'s configuration; ``batch_size`` counts samples and is
    rounded down to whole consoles.  Rewards are the batch's in-kernel rule, so the
    shaped reward's options are refused.  Rollouts and updates run eagerly, whatever
    ``cuda_graph`` says."""
    heads: int = 4
    head_dim: int = 64
    memory_dtype: str = "float32"
    checkpoint_path: str = "nesle_memory_ppo.pt"


def train_memory_ppo(config: MemoryPPOConfig, resume_from: str | None = None, *, rom_bytes: bytes | None = None,
                     snapshot_bytes=None, batch=None, on_rollout=None) -> dict:
    """Train; returns {"global_step", "updates", "log", "model"}.  Checkpoints, and
    ``resume_from`` one of them, as ``native_ppo``'s trainer has them.
    ``on_rollout(update, buffers)`` receives each rollout's buffers (tests)."""
    if config.reward_mode != "minimal":
        raise ValueError("the memory trainer takes reward_mode 'minimal'")
    for name in ("flag_bonus", "finish_zone_bonus", "death_penalty"):
        if getattr(config, name) is not None:
            raise ValueError(f"{name} belongs to reward_mode 'smart', which the memory trainer does not take")
    n, T = config.num_envs, config.n_steps
    consoles = config.batch_size // T
    if consoles < 1 or consoles > n:
        raise ValueError(f"batch_size {config.batch_size} must hold at least one console of {T} steps and at most {n}")
    if not torch.cuda.is_available():
        raise SystemExit("memory PPO needs a GPU")
    from torch.utils.dlpack import from_dlpack

    torch.manual_seed(config.seed)
    dev = torch.device("cuda")
    masks = _actions.action_masks(config.action_space)
    mask_table = torch.tensor(masks, dtype=torch.uint8, device=dev)
    batch = P.make_batch(config, rom_bytes, snapshot_bytes) if batch is None else batch
    batch.set_stream(torch.cuda.current_stream().cuda_stream)
    batch.reset_device()
    ram, rewards_view, dones_view = (from_dlpack(v()) for v in (batch.ram_device, batch.rewards_device,
                                                                batch.last_done_device))
    model = MemoryActorCritic(len(masks), width=config.hidden_size, heads=config.heads, head_dim=config.head_dim,
                              dtype=getattr(torch, config.memory_dtype), init=config.init)
    optimizer = torch.optim.Adam(model.parameters(), lr=config.learning_rate, eps=1e-5, fused=True)
    global_step = P._load_checkpoint(resume_from, model, optimizer)

    obs = torch.empty((T, n, 2048), dtype=torch.uint8, device=dev)
    actions = torch.empty((T, n), dtype=torch.long, device=dev)
    logprobs, rewards, dones, values = (torch.empty((T, n), device=dev) for _ in range(4))
    steps, resets = torch.empty((T, n), dtype=torch.int32, device=dev), torch.empty((T, n), dtype=torch.bool, device=dev)
    state, length = model.new_state(n), torch.zeros(n, dtype=torch.int32, device=dev)      # steps of the episode so far
    done = torch.ones(n, dtype=torch.bool, device=dev)      # every console starts an episode
    last = model.table.shape[0] - 1
    stats = {"global_step": global_step, "updates": 0, "log": [], "model": model}

    num_updates = math.ceil(max(0, config.total_timesteps - global_step) / (n * T))
    progress = P._progress_bar(config.progress_bar, global_step + num_updates * n * T, global_step)
    for update in range(1, num_updates + 1):
        before = state.clone()
        for t in range(T):
            step = torch.clamp(length, max=last)
            obs[t], dones[t], steps[t], resets[t] = ram, done.float(), step, done
            logits, values[t] = model.act(ram, step, done, state)
            logp = torch.log_softmax(logits, -1)
            action = torch.multinomial(logp.exp(), 1).squeeze(-1)
            actions[t], logprobs[t] = action, logp.gather(-1, action[:, None]).squeeze(-1)
            batch.step_device(mask_table[action], auto_reset=True, synchronize=False)
            rewards[t] = rewards_view
            done = dones_view.bool()
            length += 1
            if config.max_episode_steps > 0:
                timeout = (length >= config.max_episode_steps) & ~done
                batch.reset_envs_device(timeout.to(torch.uint8))       # consoles not in the mask are untouched
                done = done | timeout
            length.masked_fill_(done, 0)
        with torch.no_grad():
            _, next_value = model.act(ram, torch.clamp(length, max=last), done, state.clone())
            advantages, returns = P.compute_gae(rewards, dones, values, done.float(), next_value, config.gamma,
                                                config.gae_lambda)
        if on_rollout is not None:
            on_rollout(update, {"obs": obs, "actions": actions, "logprobs": logprobs, "rewards": rewards, "values": values,
                                "steps": steps, "resets": resets, "state": before, "model": model})
        sums = torch.zeros(2, device=dev)
        count = 0
        for _ in range(config.update_epochs):
            for idx in torch.randperm(n, device=dev).split(consoles):
                logits, value, _ = model(obs[:, idx], steps[:, idx].contiguous(), resets[:, idx].contiguous(), before[idx])
                loss, _ = P.ppo_head_loss(logits.flatten(0, 1), value.flatten(), *(
                    b[:, idx].flatten() for b in (actions, logprobs, advantages, returns)), config.clip_coef,
                    config.ent_coef, config.vf_coef, sums)
                optimizer.zero_grad(set_to_none=True)
                loss.backward()
                nn.utils.clip_grad_norm_(model.parameters(), config.max_grad_norm)
                optimizer.step()
                count += 1
        stats["global_step"] += n * T
        stats["updates"] = update
        if progress is not None:
            progress.update(n * T)
        if update % max(1, config.log_interval) != 0 and update != num_updates:
            continue
        loss, clipfrac = (sums / count).tolist()
        line = {"update": update, "step": stats["global_step"], "loss": loss, "clipfrac": clipfrac,
                "reward_mean": float(rewards.mean()), "episodes": int(dones.sum())}
        stats["log"].append(line)
        print(" ".join(f"{k}={v:.4f}" if isinstance(v, float) else f"{k}={v}" for k, v in line.items()), flush=True)
        if config.save_checkpoints:
            P._save_checkpoint(config.checkpoint_path, model, optimizer, config, stats["global_step"])
    if progress is not None:
        progress.close()
    return stats


def main(argv=None) -> None:
    p = argparse.ArgumentParser(description="Train a policy with memory by PPO on the MI355X console.")
    p.add_argument("rom_path")
    p.add_argument("--num-envs", type=int, default=512)
    p.add_argument("--total-timesteps", type=int, default=1_000_000)
    p.add_argument("--n-steps", type=int, default=128)
    p.add_argument("--batch-size", type=int, default=8192)
    p.add_argument("--heads", type=int, default=4)
    p.add_argument("--head-dim", type=int, default=64)
    p.add_argument("--memory-dtype", default="float32", choices=["float32", "bfloat16"])
    p.add_argument("--action-space", default="simple_with_start",
                   choices=["right_only", "simple", "simple_with_start", "complex", "mario", "raw"])
    p.add_argument("--reset-state-path", default=None)
    p.add_argument("--max-episode-steps", type=int, default=0)
    p.add_argument("--init", default="orthogonal", choices=["orthogonal", "xavier"])
    p.add_argument("--seed", type=int, default=1)
    p.add_argument("--log-interval", type=int, default=1)
    p.add_argument("--progress-bar", action="store_true")
    p.add_argument("--checkpoint-path", default="nesle_memory_ppo.pt")
    p.add_argument("--resume-from", default=None)
    a = p.parse_args(argv)
    train_memory_ppo(MemoryPPOConfig(
        rom_path=a.rom_path, num_envs=a.num_envs, total_timesteps=a.total_timesteps, n_steps=a.n_steps,
        batch_size=a.batch_size, heads=a.heads, head_dim=a.head_dim, memory_dtype=a.memory_dtype,
        action_space=a.action_space, reset_state_path=a.reset_state_path,
        max_episode_steps=a.max_episode_steps, init=a.init, seed=a.seed, log_interval=a.log_interval,
        progress_bar=a.progress_bar, checkpoint_path=a.checkpoint_path), a.resume_from)


if __name__ == "__main__":
    main()
