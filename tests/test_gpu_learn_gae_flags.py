"""Flags that more columns share than the C struct can count, with that limit made small (GPU)."""

import pytest
import torch

import swarp_b200 as swarp
from swarp_b200.learn import advantage

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("most", [23, 4, 3, 1])
@pytest.mark.parametrize("lead", [1, 2])
def test_flags_are_spread_over_more_dimensions(lead, most, monkeypatch):
    g = torch.Generator(device="cuda:0").manual_seed(0)
    r, v = (torch.randn(20, 6, 4, generator=g, device="cuda:0") for _ in range(2))
    u = torch.rand(r.shape[:lead], generator=g, device="cuda:0")
    for flags in ((u < 0.2, (u > 0.2) & (u < 0.4)), (u < 0.2, None), (None, u < 0.2)):
        want = swarp.gae(r, v, r[0], *flags)
        with monkeypatch.context() as m:
            m.setattr(advantage, "_MOST_PER_FLAG", most)
            got = swarp.gae(r, v, r[0], *flags)
        # columns with flags of their own may be taken one by one
        for x, y in zip(got, want):
            torch.testing.assert_close(x, y, rtol=1e-5, atol=1e-5)
