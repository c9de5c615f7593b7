"""The gradients' norm where float32 does not hold their squares, and steps that are clipped by it
(GPU). Bounds as in test_gpu_learn_adamw."""

import math

import pytest
import torch

import swarp_b200 as swarp
from test_gpu_learn_adamw import DEV, EPS, check_step, setup

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("gscale", [1e-34, 1e-28, 1e-23, 1e-20, 1e-17, 1e-15, 1e17, 1e19, 1e25, 1e33])
def test_norm_of_tiny_and_huge_gradients(gscale, dtype):
    """Whole chunks, the rest of one, an odd address and an empty tensor."""
    params, grads, m, v, w = setup([5 * 2048 + 77, 4096, 3, 0, 900], dtype, 32, gscale=gscale)
    grads[4] = torch.cat([grads[4], grads[4][:1]])[1:]
    norm = swarp.adamw_step(params, grads, m, v, step=1, lr=0.0, max_norm=1.0, masters=w)
    true = math.sqrt(sum(float(x.double().square().sum()) for x in grads))
    assert abs(float(norm) - true) <= 16 * EPS * true


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("gscale", [1e19, 1e25, 1e33])
def test_a_huge_gradient_is_clipped_and_not_lost(gscale, dtype):
    st = setup([3 * 2048 + 5, 700], dtype, 32, gscale=gscale)
    for x in st[2] + st[3]:
        x.zero_()
    check_step(st, 1, 32, max_norm=0.5)
    assert all(x.any() for x in st[2])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_one_large_element_among_zeros_and_others(dtype):
    n = 9 * 2048
    g = torch.zeros(n, device=DEV, dtype=dtype)
    g[::3] = 1e-7
    g[5000] = 6e4
    p, m, v = (torch.zeros(n, device=DEV) for _ in range(3))
    master = None if dtype == torch.float32 else [p.clone()]
    norm = swarp.adamw_step([p.to(dtype)], [g], [m], [v], step=1, lr=0.1, max_norm=1.0, masters=master)
    true = math.sqrt(float(g.double().square().sum()))
    assert abs(float(norm) - true) <= 16 * EPS * true
