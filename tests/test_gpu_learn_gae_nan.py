"""A NaN or infinite reward reaches every earlier step of its episode, however far and however
the steps are grouped (GPU)."""

import math

import pytest
import torch

import swarp_b200 as swarp

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


# one thread a column, steps in segments, and segments of runs; products of decays that stay
# (0.94), that leave float32 (0.45) and that leave float64 (1e-4) within a run of steps
@pytest.mark.parametrize("shape", [(40, 6), (900, 4), (3000, 1), (3000, 7), (2500, 130), (2048, 128),
                                   (20000, 2)])
@pytest.mark.parametrize("gamma,lam", [(0.99, 0.95), (0.9, 0.5), (0.01, 0.01), (1e-30, 1e-30)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_a_bad_reward_reaches_its_whole_episode(shape, gamma, lam, dtype, bad):
    T = shape[0]
    g = torch.Generator(device=DEV).manual_seed(T)
    r, v = (torch.randn(*shape, generator=g, device=DEV, dtype=dtype) for _ in range(2))
    last = torch.randn(*shape[1:], generator=g, device=DEV, dtype=dtype)
    start, at = T // 5, T - 2  # the episode's first step, and the bad reward
    ends = torch.zeros(*shape, dtype=torch.bool, device=DEV)
    ends[start - 1] = True
    r[at] = bad
    term, trunc = ends.clone(), ends.clone()
    term[:, 1::2] = False
    trunc[:, ::2] = False
    a, ret = swarp.gae(r, v, last, term, trunc, gamma=gamma, lam=lam)
    for x in (a, ret):
        reached = x[start:at + 1]
        if float(torch.tensor(gamma * lam, dtype=dtype)) != 0.0:  # 1e-60 is 0 in float32
            assert (reached.isnan() if math.isnan(bad) else reached.isinf()).all()
        assert x[:start].isfinite().all() and x[at + 1:].isfinite().all()

