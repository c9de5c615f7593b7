"""What a step ended in, before finished environments were reset, and the example's bootstrap from
it, against an environment that is never reset (GPU)."""

import pytest
import torch

import swarp_b200 as swarp
from test_gpu_learn_example import example

pytestmark = pytest.mark.gpu
KW = dict(n_envs=32, n_agents=3, device="cuda:0", dt=0.05)


def actions(steps, seed=1):
    g = torch.Generator().manual_seed(seed)
    return [(torch.rand(32, 3, 2, generator=g) * 2 - 1).cuda() for _ in range(steps)]


def test_final_observation_is_from_before_the_reset():
    env = swarp.make("navigation", max_steps=5, auto_reset=True, final_observation=True, **KW)
    twin = swarp.make("navigation", **KW)  # the same draws up to the first reset's effect
    assert torch.equal(env.reset(seed=3), twin.reset(seed=3))
    for k, a in enumerate(actions(5)):
        obs, _, terminated, truncated, info = env.step(a)
        want = twin.step(a)[0]
        assert not terminated.any() and bool(truncated.all()) == (k == 4)
        assert torch.equal(info["final_obs"], want)
        assert torch.equal(obs, want) == (k < 4)
    again = env.step(actions(1)[0])  # the next episode goes on from the returned observation
    assert not again[3].any() and torch.equal(again[4]["final_obs"], again[0])


def test_it_is_asked_for():
    env = swarp.make("navigation", max_steps=2, auto_reset=True, **KW)
    env.reset(seed=0)
    assert "final_obs" not in env.step(actions(1)[0])[4]


def test_the_example_bootstraps_from_the_episode_that_ended():
    steps = 6
    mod = example()
    torch.manual_seed(0)
    env = swarp.make("navigation", max_steps=steps, auto_reset=True, clone_outputs=True,
                     final_observation=True, **KW)
    obs = env.reset(seed=5)
    policy = mod.TokenPolicy(obs.shape[-1], 7, 16).cuda()
    batch, after = mod.rollout(env, policy, obs, steps)
    assert batch["truncated"][-1].all() and not batch["terminated"].any()
    twin = swarp.make("navigation", **KW)
    twin.reset(seed=5)
    with torch.no_grad():
        for t in range(steps):
            seen = twin.step(batch["tokens"][t].float() * (2.0 / 6) - 1.0)[0]
            # matrix products of other shapes may round otherwise
            torch.testing.assert_close(batch["next_values"][t], policy(seen)[1], rtol=1e-4, atol=1e-5)
        assert not torch.allclose(batch["next_values"][-1], policy(after)[1], rtol=1e-2)
