"""Train a token policy on the navigation scenario with the framework's own operators.

Each agent's two velocity slots are tokens: one of ``bins`` values in [-1, 1] each. An
iteration rolls the environment out with the current policy (``Environment.step``), records
the tokens' log probabilities (``token_logp``), estimates advantages (``gae``, with the values
of the observations that the steps ended in, before finished environments were reset), and takes a
few epochs of the clipped policy loss against the rollout's policy, with a divergence term
against the iteration's first policy (``policy_loss``), stepping both networks with
:class:`~swarp_b200.AdamW` (8-bit moments).

    python examples/train_navigation_tokens.py --envs 1024 --agents 1 --iterations 50
"""

from __future__ import annotations

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import swarp_b200 as swarp  # noqa: E402


class TokenPolicy(torch.nn.Module):
    """Observations ``[..., obs_dim]`` to logits ``[..., 2, bins]`` and a value ``[...]``."""

    def __init__(self, obs_dim: int, bins: int, hidden: int) -> None:
        super().__init__()
        self.bins = bins
        self.body = torch.nn.Sequential(torch.nn.Linear(obs_dim, hidden), torch.nn.Tanh(),
                                        torch.nn.Linear(hidden, hidden), torch.nn.Tanh())
        self.logits = torch.nn.Linear(hidden, 2 * bins)
        self.value = torch.nn.Linear(hidden, 1)

    def forward(self, obs):
        h = self.body(obs)
        return self.logits(h).unflatten(-1, (2, self.bins)), self.value(h).squeeze(-1)


def rollout(env, policy, obs, steps):
    """``steps`` steps of the environment: what the update needs, stacked ``[T, E, A, ...]``, and
    the observation that the next rollout starts from."""
    keep: dict[str, list] = {k: [] for k in ("obs", "tokens", "logp", "rewards", "values",
                                             "terminated", "truncated", "final")}
    with torch.no_grad():
        for _ in range(steps):
            logits, value = policy(obs)
            tokens = torch.distributions.Categorical(logits=logits).sample()
            logp, _ = swarp.token_logp(logits, tokens)
            actions = tokens.to(obs.dtype) * (2.0 / (policy.bins - 1)) - 1.0
            keep["obs"].append(obs)
            obs, reward, terminated, truncated, info = env.step(actions)
            for k, x in (("tokens", tokens), ("logp", logp), ("rewards", reward),
                         ("values", value), ("terminated", terminated), ("truncated", truncated),
                         ("final", info["final_obs"])):
                keep[k].append(x.clone())
        batch = {k: torch.stack(v) for k, v in keep.items()}
        # a step's successor is what it ended in: obs belongs to the next episode after a reset
        batch["next_values"] = policy(batch.pop("final"))[1]
    return batch, obs


def train(envs=1024, agents=8, steps=32, iterations=50, epochs=4, bins=21, hidden=64, lr=3e-3,
          gamma=0.97, lam=0.95, kl_coef=0.02, entropy_coef=0.003, state_bits=8, seed=0,
          report=print):
    """Train; returns the policy and the mean reward per step of each iteration."""
    torch.manual_seed(seed)
    env = swarp.make("navigation", n_envs=envs, n_agents=agents, device="cuda:0", dt=0.05,
                     max_steps=steps, auto_reset=True, clone_outputs=True, final_observation=True,
                     seed=seed)
    obs = env.reset(seed=seed)
    policy = TokenPolicy(obs.shape[-1], bins, hidden).to(obs.device)
    optimizer = swarp.AdamW(policy.parameters(), lr=lr, weight_decay=0.0, max_norm=1.0,
                            state_bits=state_bits, seed=seed)
    rewards = []
    for it in range(iterations):
        batch, obs = rollout(env, policy, obs, steps)
        adv, returns = swarp.gae(batch["rewards"], batch["values"], None, batch["terminated"],
                                 batch["truncated"], gamma=gamma, lam=lam,
                                 next_values=batch["next_values"])
        scaled = (adv - adv.mean()) / (adv.std() + 1e-6)
        scaled = scaled[..., None].expand_as(batch["logp"])  # both slots share it
        for _ in range(epochs):
            logits, value = policy(batch["obs"])
            out = swarp.policy_loss(logits, batch["tokens"], batch["logp"], scaled,
                                    ref_logp=batch["logp"], kl_coef=kl_coef,
                                    entropy_coef=entropy_coef)
            loss = out.loss + 0.5 * (value - returns).square().mean()
            optimizer.zero_grad()
            loss.backward()
            optimizer.step()
        rewards.append(float(batch["rewards"].mean()))
        if report:
            pg, kl, entropy, cut = out.stats.tolist()
            report(f"iteration {it:3d}  reward {rewards[-1]:+.4f}  kl {kl:.4f}  "
                   f"entropy {entropy:.3f}  cut {cut:.3f}  |g| {float(optimizer.grad_norm):.3f}")
    return policy, rewards


def main():
    p = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    for name, default in (("envs", 1024), ("agents", 8), ("steps", 32), ("iterations", 50),
                          ("epochs", 4), ("bins", 21), ("state-bits", 8), ("seed", 0)):
        p.add_argument(f"--{name}", type=int, default=default)
    p.add_argument("--lr", type=float, default=3e-3)
    train(**{k: v for k, v in vars(p.parse_args()).items()})


if __name__ == "__main__":
    main()
