"""A parameter that is given twice is refused, by the function and by the optimizer, and empty ones
may share an address (GPU)."""

import pytest
import torch

import swarp_b200 as swarp

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def test_refused_before_the_launch():
    p = [torch.ones(3000, device=DEV), torch.ones(40, device=DEV)]
    z = lambda: [torch.zeros_like(x) for x in (*p, p[0])]  # noqa: E731
    m, v = z(), z()
    with pytest.raises(ValueError, match="the same memory"):
        swarp.adamw_step([*p, p[0]], [torch.ones_like(x) for x in (*p, p[0])], m, v, step=1, lr=0.1)
    assert all((x == 1).all() for x in p) and not any(x.any() for x in m + v)
    q = torch.nn.Parameter(torch.ones(50, device=DEV))
    q.grad = torch.ones_like(q)
    with pytest.warns(UserWarning):  # torch's own
        opt = swarp.AdamW([q, q], lr=0.1)
    with pytest.raises(ValueError, match="the same memory"):
        opt.step()
    assert (q == 1).all() and not opt.state_dict()["state"]


def test_empty_tensors():
    e = lambda: [torch.zeros(n, device=DEV) for n in (0, 5, 0, 0)]  # noqa: E731
    p = e()
    swarp.adamw_step(p, [torch.ones_like(x) for x in p], e(), e(), step=1, lr=0.1, weight_decay=0.0)
    assert torch.allclose(p[1], torch.full((5,), -0.1, device=DEV), rtol=1e-5)
