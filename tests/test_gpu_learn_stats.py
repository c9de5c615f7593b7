"""The share of rows that the clip cut, and 8-bit moments of clipped gradients, against their
definitions (GPU)."""

import math

import pytest
import torch

import swarp_b200 as swarp
from test_gpu_learn_adamw import HP, hashes, rounded, setup, value
from test_gpu_learn_policy import batch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("mean", [True, False])
@pytest.mark.parametrize("clip", [(0.2, 0.2), (0.1, 0.3), (0.0, 0.0), (1.0, 5.0)])
@pytest.mark.parametrize("V", [5, 21, 70, 300, 2500, 9000, 40000, 262145])
def test_share_of_rows_that_the_clip_cut(V, clip, mean):
    """A ratio within 1e-4 of a bound is moved off it: there rounding would decide."""
    rows = 400 if V < 9000 else 60
    z, tok, _, adv, _ = batch(rows, V, torch.float32, seed=V)
    g = torch.Generator(device=DEV).manual_seed(V)
    lp = torch.log_softmax(z.double(), 1).gather(1, tok[:, None]).squeeze(1)
    t = 0.3 * torch.randn(rows, generator=g, device=DEV)
    lo, hi = clip
    for b in [math.log(x) for x in (1 - lo, 1 + hi) if x > 0]:
        t = torch.where((t - b).abs() < 1e-4, t + 3e-4, t)
    old = (lp - t).float()
    mask = torch.arange(rows, device=DEV) % 7 != 3
    adv[::11] = 0.0  # nothing to cut
    out, _ = swarp.policy_loss_and_grad(z, tok, old, adv, mask=mask, clip_low=lo, clip_high=hi,
                                        reduction="mean" if mean else "sum")
    r = (lp - old.double()).exp()
    cut = ((adv > 0) & (r > 1 + hi)) | ((adv < 0) & (r < 1 - lo))
    n = int((cut & mask).sum())
    assert 0 < n < int(mask.sum()) or clip == (1.0, 5.0)
    want = n / int(mask.sum()) if mean else float(n)
    # whole numbers, times the float 1 / count
    assert abs(float(out.stats[3]) - want) <= 2.0 ** -22 * want


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("max_norm", [1e-4, 0.05])
def test_8_bit_moments_of_clipped_gradients(max_norm, dtype):
    """Codes are exactly those of the float32 moments, whose gradient is the float32 product with
    the float32 scale; that scale is within 16 eps of the definition's."""
    sizes = [5000, 33, 2 * 2048, 70001]
    params, grads, m, v, masters = setup(sizes, dtype, 8)
    b1, b2 = HP["betas"]
    for step in (1, 2, 3):
        m0, v0 = [value(x) for x in m], [value(x) for x in v]
        norm = swarp.adamw_step(params, grads, m, v, step=step, seed=3, max_norm=max_norm,
                                masters=masters, **HP)
        true = math.sqrt(sum(float(x.double().square().sum()) for x in grads))
        scale = torch.tensor(max_norm, device=DEV) / (norm + 1e-6)
        assert abs(float(scale) / (max_norm / (true + 1e-6)) - 1) <= 16 * 2.0 ** -24 and scale < 0.5
        for i, g in enumerate(grads):
            g32 = g.float() * scale
            m32 = m0[i].float() * b1 + g32 * (1 - b1)
            v32 = v0[i].float() * b2 + (g32 * (1 - b2)) * g32
            h = hashes(g.numel(), 3, step, i)
            assert torch.equal(value(m[i]), rounded(m32.double(), h & 0xFFFF, True))
            assert torch.equal(value(v[i]), rounded(v32.double(), h >> 16, False))
