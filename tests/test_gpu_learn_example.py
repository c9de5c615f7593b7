"""The operators together on the simulator: a short training run of the token-policy example
raises the reward, repeats bit for bit from its seed, and with 32-bit moments too (GPU)."""

import importlib.util
import os

import pytest
import torch

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def example():
    path = os.path.join(ROOT, "examples", "train_navigation_tokens.py")
    spec = importlib.util.spec_from_file_location("train_navigation_tokens", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


@pytest.mark.parametrize("bits", [8, 32])
def test_training_raises_the_reward(bits):
    _, rewards = example().train(envs=512, agents=1, steps=32, iterations=30, state_bits=bits,
                                 report=None)
    early, late = sum(rewards[:3]) / 3, sum(rewards[-3:]) / 3
    # a step brings an agent at most dt = 0.05 nearer, and 5 at its goal; random walks bring
    # about nothing
    assert late > early + 0.05, rewards


def test_training_repeats():
    # no atomics in the framework's operators; matrix products are the same calls twice
    runs = [example().train(envs=64, agents=4, steps=8, iterations=3, report=None)
            for _ in range(2)]
    assert runs[0][1] == runs[1][1]
    for a, b in zip(runs[0][0].parameters(), runs[1][0].parameters()):
        assert torch.equal(a, b)
