"""The divergence e^d - d - 1 of a policy near its reference, where its terms cancel (GPU).

Bounds, relative, with eps = 2^-24 and d = ref - lp from the kernel's own lp (their difference is
exact where they are within a factor of two). Below 1/2 the series' seven steps and three
products round once each, all its terms are at most half of the first: 16 eps; its gradient
e^d - 1 is d plus it. From 1/2 on the exponential is off by 4 eps e^|d|, the sums by 2, of
a value of 0.1 (d < 0) or 0.14 at least: 100 eps covers |d| <= 1.
"""

import pytest
import torch

import swarp_b200 as swarp
from test_gpu_learn_policy import EPS, batch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


# short rows, groups of lanes, lanes with vectors, a CTA, a cluster, the loop
@pytest.mark.parametrize("V", [5, 21, 70, 777, 3000, 20000, 300007])
@pytest.mark.parametrize("d", [1e-4, 1e-3, 1e-2, 0.1, 0.45, 0.7, 1.0])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_divergence_near_the_reference(V, d, sign):
    z, tok, *_ = batch(4, V, torch.float32, seed=V)
    z[torch.arange(4), tok] += 3 + torch.log(torch.tensor(float(V)))  # lp well away from 0 and -9
    z[torch.arange(4), (tok + 1) % V] += 4 + torch.log(torch.tensor(float(V)))
    # row by row: at an odd address a short row goes through another kernel
    logp = torch.cat([swarp.token_logp(z[i:i + 1], tok[i:i + 1])[0] for i in range(4)])
    zero = torch.zeros_like(logp)
    for i in range(4):
        ref = logp[i:i + 1] + sign * d
        out, grad = swarp.policy_loss_and_grad(z[i:i + 1], tok[i:i + 1], logp[i:i + 1], zero[:1],
                                               ref_logp=ref, kl_coef=1.0)
        assert torch.equal(out.logp, logp[i:i + 1])
        x = ref.double() - out.logp.double()
        want, slope = torch.expm1(x) - x, -torch.expm1(x)
        if float(x.abs()) < 0.01:  # 64 bits cancel too
            want = x * x * (0.5 + x * (1 / 6 + x * (1 / 24 + x / 120)))
        room = (16 if float(x.abs()) < 0.5 else 100) * EPS
        for got in (out.stats[1], out.loss):
            assert abs(float(got) / float(want) - 1) <= room, (float(got), float(want))
        # the gradient of the chosen token: slope (1 - p)
        p = out.logp.double().exp()
        got = float(grad[0, tok[i]])
        assert abs(got / float(slope * (1 - p)) - 1) <= room + 64 * EPS / float(1 - p), got
