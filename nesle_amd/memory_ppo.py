"""PPO with a policy that remembers its episode: the operators of
``nesle_amd.memory`` used together.

The policy of ``native_ppo`` sees one instant of RAM.  ``MemoryActorCritic``
puts a memory layer behind its first layer: queries, keys and values of 4 heads
of 64 from one projection, normed and rotated by the step of the episode
(``qk_norm_rotate``), through the gated delta rule, or (``memory="decay"``) through
linear attention with a learned decay for each head, whose readout a layer norm of
each head brings to one size.  It

* acts one token at a time (``act``: ``gated_delta_step`` or
  ``decay_attention_step``, the states of all consoles updated in place, dropped
  where an episode ended), and
* trains on whole rollouts of the consoles of a minibatch (``forward``:
  ``gated_delta`` or ``decay_attention`` from the states the rollout started with,
  gradients through all of its operators).

``train_memory_ppo`` is the trainer: the console batch, generalised advantage
estimation and the clipped loss head are ``native_ppo``'s.  Minibatches are
consoles with all their steps, as a memory's tokens belong together.  ``play``
plays a trained policy, with ``sample_actions``'s temperature, top-k, top-p and
min-p.

    python -m nesle_amd.memory_ppo game.nes --num-envs 512 --total-timesteps 10000000
    python -m nesle_amd.memory_ppo game.nes --num-envs 64 --resume-from nesle_memory_ppo.pt --play 2000 --top-p 0.9
"""

from __future__ import annotations

import argparse
import math
from dataclasses import dataclass

import torch
import torch.nn as nn
import torch.nn.functional as F

from nesle_amd import actions as _actions
from nesle_amd import memory as operators
from nesle_amd import native_ppo as P


class MemoryActorCritic(nn.Module):
    """2,048 RAM bytes / 255 -> width tanh -> memory of ``heads`` heads -> width
    tanh -> action logits + value.  memory: "delta", the gated delta rule with gates
    from the features, or "decay", linear attention with one decay a head."""

    def __init__(self, action_dim: int, obs_dim: int = 2048, width: int = 256, heads: int = 4, head_dim: int = 64,
                 max_steps: int = 4096, dtype: torch.dtype = torch.float32, init: str = "orthogonal", device=None,
                 memory: str = "delta") -> None:
        super().__init__()
        if init not in ("orthogonal", "xavier"):
            raise ValueError(f"unknown init {init!r}: 'orthogonal' or 'xavier'")
        if memory not in ("delta", "decay"):
            raise ValueError(f"unknown memory {memory!r}: 'delta' or 'decay'")
        dev = device if device is not None else torch.device("cuda")
        self.heads, self.head_dim, self.dtype, self.memory = heads, head_dim, dtype, memory
        inner = heads * head_dim
        self.encode = nn.Linear(obs_dim, width, device=dev)
        self.project = nn.Linear(width, 3 * inner, device=dev)
        if memory == "delta":
            self.gates = nn.Linear(width, 2 * heads, device=dev)
        else:
            self.norm_weight = nn.Parameter(torch.ones(head_dim, device=dev))
            self.norm_bias = nn.Parameter(torch.zeros(head_dim, device=dev))
        self.q_weight = nn.Parameter(torch.ones(head_dim, device=dev))
        self.k_weight = nn.Parameter(torch.ones(head_dim, device=dev))
        self.merge = nn.Linear(inner, width, device=dev)
        self.actor = nn.Linear(width, action_dim, device=dev)
        self.critic = nn.Linear(width, 1, device=dev)
        gates = ((self.gates, 0.1),) if memory == "delta" else ()
        for layer, gain in ((self.encode, math.sqrt(2.0)), (self.project, 1.0), *gates, (self.merge, 1.0), (self.actor, 0.01),
                            (self.critic, 1.0)):
            (nn.init.orthogonal_ if init == "orthogonal" else nn.init.xavier_uniform_)(layer.weight, gain)
            nn.init.zeros_(layer.bias)
        # Half lives of about 10 to 300 steps to begin with, one for each head.
        with torch.no_grad():
            rate = torch.logspace(math.log10(0.07), math.log10(0.0025), heads, device=dev)
            if memory == "delta":
                self.gates.bias[:heads] = torch.log(torch.expm1(rate))
            else:
                self.decay = nn.Parameter(torch.log(rate))     # a head's log decay is -exp of it
        self.register_buffer("table", operators.rotation_table(max_steps, head_dim, device=dev), persistent=False)

    def new_state(self, num_envs: int) -> torch.Tensor:
        return torch.zeros(num_envs, self.heads, self.head_dim, self.head_dim, device=self.encode.weight.device)

    def _tokens(self, obs, steps):
        """(features, q, k, v, *gates) of observations [..., obs_dim]; gates: g, beta of
        the delta rule, or the heads' log decays."""
        x = torch.tanh(self.encode((obs / 255.0).float()))
        q, k, v = self.project(x).to(self.dtype).unflatten(-1, (3, self.heads, self.head_dim)).unbind(-3)
        # Unit norms (the rule wants keys of about unit length); the weights
        # scale the directions against each other.
        q, k = operators.qk_norm_rotate(q, k, self.q_weight, self.k_weight, positions=steps, table=self.table, unit=True)
        if self.memory == "decay":
            return x, q, k, v, -torch.exp(self.decay)
        decay, write = self.gates(x).chunk(2, -1)
        return x, q, k, v, -F.softplus(decay), torch.sigmoid(write)

    def _heads_out(self, x, out):
        if self.memory == "decay":         # nothing else bounds what a slow head adds up
            out = operators.layer_norm(out, self.norm_weight, self.norm_bias)
        x = torch.tanh(x + self.merge(out.flatten(-2).float()))
        return self.actor(x), self.critic(x).squeeze(-1)

    def forward(self, obs, steps, resets, state):
        """(logits, values, state after) of a rollout: obs [T, N, obs_dim]
        uint8, steps int32 [T, N] (of the episode), resets [T, N] (its first
        step), state before it."""
        x, q, k, v, *gates = self._tokens(obs, steps)
        over = operators.gated_delta if self.memory == "delta" else operators.decay_attention
        out, state = over(q, k, v, *gates, state=state, resets=resets, scale=1.0)
        return (*self._heads_out(x, out), state)

    @torch.no_grad()
    def act(self, obs, steps, resets, state):
        """(logits, values) of one step of every console; ``state`` is updated."""
        x, q, k, v, *gates = self._tokens(obs, steps)
        step = operators.gated_delta_step if self.memory == "delta" else operators.decay_attention_step
        out = step(q, k, v, *(t.contiguous() for t in gates), state, resets=resets, scale=1.0)
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
    # "delta" (the gated delta rule) or "decay" (linear attention).
    memory: str = "delta"
    # How rollouts draw their actions: "multinomial" (torch's), or "uniform": one
    # uniform number a console and step through sample_actions, which also gives the
    # log probability.  The same distribution; other random numbers.
    sampler: str = "multinomial"
    checkpoint_path: str = "nesle_memory_ppo.pt"


def _model_of(config: MemoryPPOConfig, action_dim: int) -> MemoryActorCritic:
    return MemoryActorCritic(action_dim, width=config.hidden_size, heads=config.heads, head_dim=config.head_dim,
                             dtype=getattr(torch, config.memory_dtype), init=config.init, memory=config.memory)


def _check_reward(config: MemoryPPOConfig) -> None:
    if config.reward_mode != "minimal":
        raise ValueError("the memory trainer takes reward_mode 'minimal'")
    for name in ("flag_bonus", "finish_zone_bonus", "death_penalty"):
        if getattr(config, name) is not None:
            raise ValueError(f"{name} belongs to reward_mode 'smart', which the memory trainer does not take")


@torch.no_grad()
def play(config: MemoryPPOConfig, steps: int, model: MemoryActorCritic | None = None, *, temperature=1.0, top_k=0, top_p=1.0,
         min_p=0.0, rom_bytes: bytes | None = None, snapshot_bytes=None, batch=None, on_step=None) -> dict:
    """Play ``steps`` env-steps of every console from its start with ``model`` (None:
    the one at ``config.checkpoint_path``), actions by ``sample_actions`` with the given
    settings (``temperature=0``: the likeliest).  Returns {"rewards": summed, [num_envs],
    "episodes": ended, [num_envs]}.  ``on_step(t, actions, logprobs)`` receives each
    step's tensors.  Episodes end by the game or by ``max_episode_steps``; rewards are
    the in-kernel ones, as in training, and the shaped reward's options are refused."""
    _check_reward(config)
    if not torch.cuda.is_available():
        raise SystemExit("memory PPO needs a GPU")
    from torch.utils.dlpack import from_dlpack

    dev, n = torch.device("cuda"), config.num_envs
    masks = _actions.action_masks(config.action_space)
    mask_table = torch.tensor(masks, dtype=torch.uint8, device=dev)
    if model is None:
        model = _model_of(config, len(masks))
        saved = torch.load(config.checkpoint_path, map_location=dev, weights_only=True)
        model.load_state_dict(saved["model"])
    torch.manual_seed(config.seed)         # after the weights, which draw too
    batch = P.make_batch(config, rom_bytes, snapshot_bytes) if batch is None else batch
    batch.set_stream(torch.cuda.current_stream().cuda_stream)
    batch.reset_device()
    ram, rewards_view, dones_view = (from_dlpack(v()) for v in (batch.ram_device, batch.rewards_device,
                                                                batch.last_done_device))
    state, length = model.new_state(n), torch.zeros(n, dtype=torch.int32, device=dev)
    done = torch.ones(n, dtype=torch.bool, device=dev)
    rewards, episodes = torch.zeros(n, device=dev), torch.zeros(n, dtype=torch.long, device=dev)
    undefined = torch.zeros(n, dtype=torch.bool, device=dev)
    last = model.table.shape[0] - 1
    for t in range(steps):
        logits, _ = model.act(ram, torch.clamp(length, max=last), done, state)
        action, logprob = operators.sample_actions(logits, torch.rand(n, device=dev), temperature=temperature, top_k=top_k,
                                                   top_p=top_p, min_p=min_p)
        undefined |= action < 0
        if on_step is not None:
            on_step(t, action, logprob)
        batch.step_device(mask_table[action], auto_reset=True, synchronize=False)
        rewards += rewards_view
        done = dones_view.bool()
        length += 1
        if config.max_episode_steps > 0:
            timeout = (length >= config.max_episode_steps) & ~done
            batch.reset_envs_device(timeout.to(torch.uint8))       # consoles not in the mask are untouched
            done = done | timeout
        length.masked_fill_(done, 0)
        episodes += done
    if bool(undefined.any()):
        raise FloatingPointError("the policy's logits are not finite")
    return {"rewards": rewards, "episodes": episodes}


def train_memory_ppo(config: MemoryPPOConfig, resume_from: str | None = None, *, rom_bytes: bytes | None = None,
                     snapshot_bytes=None, batch=None, on_rollout=None) -> dict:
    """Train; returns {"global_step", "updates", "log", "model"}.  Checkpoints, and
    ``resume_from`` one of them, as ``native_ppo``'s trainer has them.
    ``on_rollout(update, buffers)`` receives each rollout's buffers (tests)."""
    _check_reward(config)
    if config.sampler not in ("multinomial", "uniform"):
        raise ValueError(f"unknown sampler {config.sampler!r}: 'multinomial' or 'uniform'")
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
    model = _model_of(config, len(masks))
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
            if config.sampler == "uniform":
                action, logprobs[t] = operators.sample_actions(logits, torch.rand(n, device=dev))
            else:
                logp = torch.log_softmax(logits, -1)
                action = torch.multinomial(logp.exp(), 1).squeeze(-1)
                logprobs[t] = logp.gather(-1, action[:, None]).squeeze(-1)
            actions[t] = action
            batch.step_device(mask_table[action], auto_reset=True, synchronize=False)
            rewards[t] = rewards_view
            done = dones_view.bool()
            length += 1
            if config.max_episode_steps > 0:
                timeout = (length >= config.max_episode_steps) & ~done
                batch.reset_envs_device(timeout.to(torch.uint8))       # consoles not in the mask are untouched
                done = done | timeout
            length.masked_fill_(done, 0)
        if config.sampler == "uniform" and bool((actions < 0).any()):      # before anything reads them as indexes
            raise FloatingPointError("the policy's logits are not finite")
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
    p.add_argument("--memory", default="delta", choices=["delta", "decay"])
    p.add_argument("--sampler", default="multinomial", choices=["multinomial", "uniform"])
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
    p.add_argument("--play", type=int, default=0, metavar="STEPS",
                   help="play the policy of --resume-from for so many steps instead of training")
    p.add_argument("--temperature", type=float, default=1.0, help="of --play, as the next three")
    p.add_argument("--top-k", type=int, default=0)
    p.add_argument("--top-p", type=float, default=1.0)
    p.add_argument("--min-p", type=float, default=0.0)
    a = p.parse_args(argv)
    config = MemoryPPOConfig(
        rom_path=a.rom_path, num_envs=a.num_envs, total_timesteps=a.total_timesteps, n_steps=a.n_steps,
        batch_size=a.batch_size, heads=a.heads, head_dim=a.head_dim, memory_dtype=a.memory_dtype,
        action_space=a.action_space, reset_state_path=a.reset_state_path,
        max_episode_steps=a.max_episode_steps, init=a.init, seed=a.seed, log_interval=a.log_interval,
        progress_bar=a.progress_bar, checkpoint_path=a.checkpoint_path, memory=a.memory, sampler=a.sampler)
    if a.play < 0:
        raise SystemExit("--play takes a number of steps")
    if a.play == 0:
        train_memory_ppo(config, a.resume_from)
        return
    if a.resume_from is None:
        raise SystemExit("--play needs --resume-from, a checkpoint to play")
    config.checkpoint_path = a.resume_from
    got = play(config, a.play, temperature=a.temperature, top_k=a.top_k, top_p=a.top_p, min_p=a.min_p)
    print(f"consoles={a.num_envs} steps={a.play} reward_mean={float(got['rewards'].mean()):.4f} "
          f"episodes={int(got['episodes'].sum())}")


if __name__ == "__main__":
    main()
