"""Rows that a cluster of CTAs shares: a wait for a part that runs out (here at once) ends the call
with NaN wherever the part is missing, and the next call is right (GPU)."""

import pytest
import torch

import swarp_b200 as swarp
from test_gpu_learn_policy import batch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("rows", [1, 5, 400])
@pytest.mark.parametrize("V", [20000, 50000, 100000])  # clusters of 2, 4 and 8
def test_a_wait_that_runs_out_is_loud(V, rows, monkeypatch):
    z, tok, old, adv, ref = batch(rows, V, torch.float32)
    mask = torch.arange(rows, device=DEV) % 3 != 1
    kw = dict(ref_logp=ref, mask=mask, kl_coef=0.1, entropy_coef=0.01)
    want = swarp.policy_loss_and_grad(z, tok, old, adv, **kw)
    monkeypatch.setenv("SWARP_POLICY_WAIT_CLOCKS", "-1")
    out, grad = swarp.policy_loss_and_grad(z, tok, old, adv, **kw)
    alone = swarp.policy_loss(z, tok, old, adv, **kw)
    logp, entropy = swarp.token_logp(z, tok)
    torch.cuda.synchronize()  # the context is as before
    assert out.loss.isnan() and alone.loss.isnan()
    assert out.logp[mask].isnan().all() and grad[mask].isnan().all()
    assert not out.logp[~mask].any() and not grad[~mask].any()
    assert logp.isnan().all() and entropy.isnan().all()
    monkeypatch.delenv("SWARP_POLICY_WAIT_CLOCKS")
    again = swarp.policy_loss_and_grad(z, tok, old, adv, **kw)
    assert torch.equal(again[1], want[1])
    assert all(torch.equal(a, b) for a, b in zip(again[0], want[0]))
