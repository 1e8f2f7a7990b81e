"""GPU-resident PPO with a policy that remembers: the operators of
``nesle_b200.ops`` together, as a training program uses them.

One RAM image does not say where an episode has been; a state for every env and
head does (the gated delta rule).  The policy is

    RAM bytes -> Linear+ReLU -> Linear+ReLU -> h
    q, k, v = projections of h;  g, beta = gates of h;  S <- delta rule
    h + Linear(read of S) -> logits, value

* Rollout: the two encoder layers run as 8-bit products -- the first eats the
  core's RAM view as it is, no conversion, no copy -- and the memory advances
  one token in place (``delta_step``), envs that were reset from zero.
* Update: minibatches of whole sequences, a few envs for all steps.  The
  encoder runs in bf16 with gradients, the memory over all steps at once
  (``delta_scan``) from the state that the rollout began with.  Matrices learn
  by ``Muon``, all else by Adam; then the encoder is quantised again.

The log-probabilities of the rollout are those of the 8-bit policy that acted;
the update's ratio starts from them.  The reference's PPO (src/nesle/native_ppo.py)
has a feed-forward policy only.

    python -m nesle_b200.memory_ppo --envs 256 --steps 32 --iterations 3
"""
from __future__ import annotations

import argparse
import math
import time
from dataclasses import dataclass
from typing import Any

from . import workloads as w
from .native_ppo import NativePPOConfig, PPOTrainer, allreduce_mean_grads, compute_gae


@dataclass
class MemoryPPOConfig(NativePPOConfig):
    heads: int = 4
    head_dim: int = 64
    muon_lr: float = 0.01
    muon_momentum: float = 0.95


def make_memory_model(obs_dim: int, action_dim: int, hidden_sizes: tuple[int, int], heads: int, head_dim: int, device):
    """The recurrent actor-critic; ``step`` is its rollout form, ``forward`` its training form."""
    import torch
    import torch.nn as nn
    import torch.nn.functional as F

    from . import ops

    h1, h2 = hidden_sizes
    inner = heads * head_dim

    class MemoryActorCritic(nn.Module):
        def __init__(self) -> None:
            super().__init__()
            self.enc1, self.enc2 = nn.Linear(obs_dim, h1), nn.Linear(h1, h2)
            self.query, self.key, self.value_in = (nn.Linear(h2, inner, bias=False) for _ in range(3))
            self.gates = nn.Linear(h2, 2 * heads)
            self.read = nn.Linear(inner, h2, bias=False)
            self.actor, self.critic = nn.Linear(h2, action_dim), nn.Linear(h2, 1)
            for layer in (self.enc1, self.enc2):
                nn.init.orthogonal_(layer.weight, math.sqrt(2.0))
                nn.init.zeros_(layer.bias)
            for layer in (self.query, self.key, self.value_in, self.read):
                nn.init.orthogonal_(layer.weight)
            nn.init.zeros_(self.gates.weight)
            # decays from about 0.98 to 0.999 a step, half strength of writing
            self.gates.bias.data[:heads] = torch.linspace(-4.0, -7.0, heads)
            self.gates.bias.data[heads:] = 0.0
            nn.init.orthogonal_(self.actor.weight, 0.01)
            nn.init.zeros_(self.actor.bias)
            nn.init.orthogonal_(self.critic.weight, 1.0)
            nn.init.zeros_(self.critic.bias)
            self.packed = None

        def matrices(self):
            """The parameters that Muon takes."""
            return [self.enc1.weight, self.enc2.weight, self.query.weight, self.key.weight, self.value_in.weight,
                    self.read.weight]

        def quantize(self) -> None:
            """Lays the encoder out in 8 bits for ``step``; to be called when its weights have changed."""
            self.packed = tuple(ops.Int8Weight.from_float(x.weight) for x in (self.enc1, self.enc2))

        def _tokens(self, h):
            """q, k, v, g, beta of the memory from (..., h2) features."""
            with torch.autocast("cuda", dtype=torch.bfloat16, cache_enabled=False):
                q, k, v = (layer(h).unflatten(-1, (heads, head_dim)) for layer in (self.query, self.key, self.value_in))
                gates = self.gates(h).float()
            q, k = (F.normalize(x.float(), dim=-1).to(torch.bfloat16) for x in (q, k))
            return q, k, v, -F.softplus(gates[..., :heads]), torch.sigmoid(gates[..., heads:])

        def _heads(self, h, o):
            with torch.autocast("cuda", dtype=torch.bfloat16, cache_enabled=False):
                f = h + self.read(o.flatten(-2))
                logits, value = self.actor(f), self.critic(f).squeeze(-1)
            return logits.float(), value.float()

        @torch.no_grad()
        def step(self, obs, reset, state):
            """One step of every env: (n, obs_dim) uint8 RAM, (n,) flags of envs just reset; ``state`` in place."""
            h = ops.int8_linear(obs, self.packed[0], 1.0 / 255.0, self.enc1.bias, relu=True)
            h = ops.int8_linear(h, self.packed[1], bias=self.enc2.bias, relu=True)
            return self._heads(h, ops.delta_step(*self._tokens(h), state, reset))

        def forward(self, obs, reset, state):
            """All steps: (t, n, obs_dim) RAM, (t, n) flags, the state before; logits, values and the state after."""
            with torch.autocast("cuda", dtype=torch.bfloat16, cache_enabled=False):
                h = torch.relu(self.enc2(torch.relu(self.enc1(obs.to(torch.bfloat16) * (1.0 / 255.0)))))
            o, state = ops.delta_scan(*self._tokens(h), state, reset)
            return (*self._heads(h, o), state)

    return MemoryActorCritic().to(device)


class _Both:
    """Two optimisers as one."""

    def __init__(self, *optimizers):
        self.optimizers = optimizers

    def zero_grad(self, set_to_none: bool = True) -> None:
        for o in self.optimizers:
            o.zero_grad(set_to_none=set_to_none)

    def step(self) -> None:
        for o in self.optimizers:
            o.step()


class MemoryPPOTrainer(PPOTrainer):
    """One process (one GPU) of the recurrent PPO loop on a CudaBatch."""

    def __init__(self, config: MemoryPPOConfig, workload: w.Workload | None = None, *, device: int = 0, rank: int = 0,
                 world: int = 1):
        import torch

        if config.batch_size % config.n_steps:
            raise ValueError(f"batch_size={config.batch_size} must be whole sequences of n_steps={config.n_steps}")
        super().__init__(config, workload, device=device, rank=rank, world=world, use_graphs=False)
        shape = (config.num_envs, config.heads, config.head_dim, config.head_dim)
        self.state = torch.zeros(shape, dtype=torch.float32, device=self.dev)
        self.first_state = torch.zeros_like(self.state)
        self.model.quantize()

    def _make_model(self):
        c = self.cfg
        return make_memory_model(2048, len(w.SIMPLE_MOVEMENT_MASKS), c.hidden_sizes, c.heads, c.head_dim, self.dev)

    def _make_optimizer(self):
        import torch

        from .muon import Muon

        matrices = self.model.matrices()
        taken = {id(p) for p in matrices}
        rest = [p for p in self.model.parameters() if id(p) not in taken]
        return _Both(Muon(matrices, lr=self.cfg.muon_lr, momentum=self.cfg.muon_momentum),
                     torch.optim.Adam(rest, lr=self.cfg.learning_rate, eps=1e-5))

    def rollout(self) -> None:
        """n_steps env-steps of every env; no host synchronisation."""
        import torch

        self.first_state.copy_(self.state)
        for t in range(self.cfg.n_steps):
            self.obs_buf[t].copy_(self.obs)
            self.done_buf[t].copy_(self.next_done)
            logits, value = self.model.step(self.obs, self.next_done != 0, self.state)
            logp_all = torch.log_softmax(logits, dim=-1)
            u = torch.rand_like(logp_all).clamp_(1e-20, 1.0)  # Gumbel-max: a sample with no host round trip
            action = torch.argmax(logp_all - torch.log(-torch.log(u)), dim=-1)
            self.logp_buf[t].copy_(logp_all.gather(1, action[:, None]).squeeze(1))
            self.act_buf[t].copy_(action)
            self.val_buf[t].copy_(value)
            self.batch.step_device(self.mask_table[action], auto_reset=True, synchronize=False)
            self.rew_buf[t].copy_(self.rewards)
            self.next_done.copy_(self.dones)
        self.global_step += self.cfg.num_envs * self.cfg.n_steps * self.world

    def update(self) -> dict[str, Any]:
        """GAE and update_epochs passes over the envs' sequences; the encoder is quantised again at the end."""
        import torch

        cfg = self.cfg
        _, next_value = self.model.step(self.obs, self.next_done != 0, self.state.clone())
        adv, ret = compute_gae(self.rew_buf, self.done_buf, self.val_buf, self.next_done, next_value, cfg.gamma,
                               cfg.gae_lambda)
        reset = self.done_buf != 0
        params = list(self.model.parameters())
        per_batch = cfg.batch_size // cfg.n_steps
        losses = []
        for _ in range(cfg.update_epochs):
            perm = torch.randperm(cfg.num_envs, device=self.dev)
            for start in range(0, cfg.num_envs, per_batch):
                idx = perm[start:start + per_batch]
                logits, value, _ = self.model(self.obs_buf[:, idx], reset[:, idx], self.first_state[idx])
                loss = self._surrogate_loss(logits.flatten(0, 1), value.flatten(), self.act_buf[:, idx].flatten(),
                                            self.logp_buf[:, idx].flatten(), adv[:, idx].flatten(), ret[:, idx].flatten())
                self.opt.zero_grad(set_to_none=True)
                loss.backward()
                allreduce_mean_grads(params, self.world)
                torch.nn.utils.clip_grad_norm_(params, cfg.max_grad_norm)
                self.opt.step()
                losses.append(loss.detach())
        self.model.quantize()
        return {"loss": torch.stack(losses).mean(), "samples": cfg.num_envs * cfg.n_steps}


def train_memory_ppo(config: MemoryPPOConfig, iterations: int, workload: w.Workload | None = None,
                     device: int = 0) -> list[float]:
    """Single-GPU training loop; returns the mean loss of every iteration.  Raises where an operator's kernel has given up
    on a wait, whose outputs are invalid."""
    from . import ops

    trainer = MemoryPPOTrainer(config, workload, device=device)
    out = []
    stalls = ops.stalls(device)
    t0 = time.perf_counter()
    for it in range(iterations):
        out.append(float(trainer.iteration()["loss"]))
        if ops.stalls(device) != stalls:  # beside the read of the loss, which has waited for the device
            raise RuntimeError(f"a kernel gave up on an internal wait in iteration {it + 1}: its results are invalid")
        fps = trainer.global_step / max(1e-9, time.perf_counter() - t0)
        print(f"iteration={it + 1}/{iterations} step={trainer.global_step} loss={out[-1]:.4f} fps={fps:.0f}", flush=True)
    trainer.batch.synchronize()
    return out


def main(argv=None) -> int:
    ap = argparse.ArgumentParser(description="Recurrent PPO on the batched core")
    ap.add_argument("--envs", type=int, default=2048)
    ap.add_argument("--steps", type=int, default=128)
    ap.add_argument("--batch", type=int, default=8192, help="samples of a minibatch at most (one sequence at least): whole sequences of --steps")
    ap.add_argument("--iterations", type=int, default=4)
    ap.add_argument("--device", type=int, default=0)
    args = ap.parse_args(argv)
    sequences = max(1, min(args.batch // args.steps, args.envs))
    train_memory_ppo(MemoryPPOConfig(num_envs=args.envs, n_steps=args.steps, batch_size=sequences * args.steps),
                     args.iterations, device=args.device)
    return 0


if __name__ == "__main__":
    raise SystemExit(main())
