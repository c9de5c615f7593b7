"""The policy loss over logits of large finite magnitude: action masks that fill with -1e6 to
-1e37, rows that are large everywhere, rows on both sides of where the kernels change the way an
exponent is formed (|max| = 1e5), against the formulas in 64 bits (GPU).

Bounds. As in test_gpu_learn_policy: eps (2 spread + V / 32 + 64), with the spread that of the
logits within 200 of their row's maximum. Those further below have probability e^-200 at most,
which float32 holds as 0, and add nothing. A maximum up to 1e5 may shift all of a row's
exponents alike by 2^-7, which leaves the differences, and with them the bound, as they are.
"""

import math

import pytest
import torch

import swarp_b200 as swarp
from test_gpu_learn_policy import EPS, ULP, batch, close, formula

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
FILLS = [-1e6, -1e8, -1e10, -1e15, -1e20, -1e30, -1e37]
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
# short rows through shared memory, groups of lanes, lanes with vectors, a CTA, clusters, the loop
VOCABS = [9, 21, 32, 70, 130, 777, 1500, 3000, 20000, 70001, 150000, 300007]


def compare(z, tok, old, adv, ref, kl=0.05, ent=0.01, scale=1.0, mean=True):
    V, n = z.shape[-1], z.shape[0] if mean else 1
    out, grad = swarp.policy_loss_and_grad(z, tok, old, adv, ref_logp=ref, kl_coef=kl,
                                           entropy_coef=ent, grad_scale=scale,
                                           reduction="mean" if mean else "sum")
    logp, entropy = swarp.token_logp(z, tok)
    z64 = z.double().requires_grad_(True)
    loss, lp, H, stats = formula(z64, tok, old, adv, ref, None, kl, ent, mean)
    (loss * scale).backward()
    near = z64.detach() - z64.detach().amax(-1, keepdim=True)
    spread = float(-near[near > -200].min())
    tol = EPS * (2 * spread + V / 32 + 64)
    for got, want in ((out.logp, lp), (logp, lp)):
        close(got, want.detach(), tol, "logp")
    for got in (out.entropy, entropy):
        close(got, H.detach(), 2 * tol, "entropy")
    size = float(adv.abs().max()) * 8 + 8
    close(out.loss, loss.detach(), z.shape[0] / n * size * 4 * tol, "loss")
    close(out.stats[:3], stats, z.shape[0] / n * size * 4 * tol, "stats")
    p = torch.softmax(z64.detach(), -1)
    hot = torch.zeros_like(p).scatter_(-1, tok[:, None], 1.0)
    room = scale / n * (size + ent * (spread + 8)) * 8 * tol
    sub = 2.0 ** -25 if z.dtype == F16 else 0.0
    close(grad, z64.grad, room * (p + hot) + z64.grad.abs() * ULP[z.dtype] + sub + 1e-35, "grad")
    return out, grad


def at_token(z, tok):
    return torch.log_softmax(z.double(), 1).gather(1, tok[:, None]).squeeze(1)


def filled(V, dtype, fill, rows=24):
    """All but two tokens filled, all of a row filled, its second half filled, every second
    token filled, and rows without any."""
    z, tok, _, adv, _ = batch(rows, V, dtype, seed=V)
    j = torch.arange(V, device=DEV)
    other = (tok + 1 + V // 3) % V
    for i in range(rows):
        kind = i % 5
        keep = (j == tok[i]) | (j == other[i])
        if kind == 0:
            z[i, ~keep] = fill
        elif kind == 1:
            z[i] = fill
        elif kind == 2:
            z[i, (j >= V // 2) & ~keep] = fill
        elif kind == 3:
            z[i, (j % 2 == 0) & ~keep] = fill
    lp = at_token(z, tok)
    return z, tok, (lp - 0.05).float(), adv, (lp + 0.1).float()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("V", VOCABS)
@pytest.mark.parametrize("fill", FILLS)
def test_filled_tokens(fill, V, dtype):
    compare(*filled(V, dtype, fill))


@pytest.mark.parametrize("V", VOCABS)
@pytest.mark.parametrize("fill", [-1e4, -6e4])
def test_filled_tokens_float16(fill, V):
    compare(*filled(V, F16, fill), scale=1024.0)


@pytest.mark.parametrize("V", VOCABS)
@pytest.mark.parametrize("level", [1e4, 9.99e4, 1e5, 1.001e5, 1e6, 1e10, 1e30, 3e38])
def test_rows_that_are_large_everywhere(level, V):
    """Logits around +-level: about the size of its ulp apart, or all alike."""
    z, tok, _, adv, _ = batch(20, V, F32, seed=V + 1)
    sign = torch.where(torch.arange(20, device=DEV) % 2 == 0, 1.0, -1.0)[:, None]
    z = sign * level + z * (torch.arange(20, device=DEV) % 3)[:, None]
    z[::5] += 30 * torch.randn(4, V, device=DEV, generator=torch.Generator(DEV).manual_seed(V))
    lp = at_token(z, tok)
    compare(z, tok, (lp - 0.05).float(), adv, (lp + 0.1).float())


@pytest.mark.parametrize("V", VOCABS)
def test_parts_on_both_sides_of_the_change(V):
    """Stretches of a row around 9.99e4, 1e5 and 1.0001e5, so that the row's maximum and those
    of its parts are of different kinds."""
    z, tok, _, adv, _ = batch(20, V, F32, seed=V + 2)
    j = torch.arange(V, device=DEV) * 7 // V
    level = torch.tensor([99999.0, 1e5, 100001.0, 99990.0, 100010.0, 99998.0, 100002.0], device=DEV)
    for i in range(20):
        z[i] = z[i] + level[(j + i) % 7] * (1.0 if i % 2 else -1.0)
    lp = at_token(z, tok)
    compare(z, tok, (lp - 0.05).float(), adv, (lp + 0.1).float())


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("V", VOCABS)
def test_fills_near_the_end_of_the_range(V, dtype):
    """A loss scale times the entropy's coefficient must not take a finite logit's product out
    of the range, and neither may a row's maximum far above a part's."""
    z, tok, _, adv, _ = batch(12, V, dtype, seed=V + 3)
    j = torch.arange(V, device=DEV)
    for i, (fill, top) in enumerate([(-1e38, 0.0), (-2.2e38, 0.0), (-1e38, 9e37), (-2.2e38, 9e37)]):
        z[i, (j % 4 != 0) & (j != tok[i])] = fill
        if top:
            z[i, V // 2] = top
            tok[i] = V // 2
    lp = at_token(z, tok)
    compare(z, tok, (lp - 0.05).float(), adv, (lp + 0.1).float(), scale=65536.0, mean=False)


def far_below(z, V):
    """Tokens at 30, 1e4, 1e9, 1e30 and 3e38 below the rows' maximum, and their bound: each of
    the two differences is rounded once."""
    z = z.clone()
    tok = torch.full((z.shape[0],), V - 1 - V // 5, device=DEV)
    z[:, V // 2] = 3.0
    z[:, V - 1 - V // 5] = torch.tensor([-30.0, -1e4, -1e9, -1e30, -3e38],
                                        device=DEV).repeat(z.shape[0] // 5)
    lp = at_token(z, tok)
    return z, tok, lp, EPS * (2 * lp.abs() + V / 32 + 64)


@pytest.mark.parametrize("V", VOCABS)
def test_a_chosen_token_far_below(V):
    """Its log probability has no floor, and is the same from an aligned batch and a strided one,
    which short rows take through other kernels."""
    z, tok, lp, tol = far_below(batch(20, V, F32, seed=V + 4)[0], V)
    wide = torch.empty(20, V + 3, device=DEV)
    wide[:, :V] = z
    zero = torch.zeros(20, device=DEV)
    for x in (z, wide[:, :V]):
        close(swarp.token_logp(x, tok)[0], lp, tol, "logp")
        out, grad = swarp.policy_loss_and_grad(x, tok, zero, zero + 1)
        close(out.logp, lp, tol, "logp")
        assert not out.loss.isnan() and not grad.isnan().any()


@pytest.mark.parametrize("V", VOCABS)
def test_a_barred_token_in_a_row_with_nan(V):
    z, tok, *_ = batch(6, V, F32)
    z[torch.arange(6), tok] = -math.inf
    z[torch.arange(6), (tok + 1) % V] = math.nan
    assert swarp.token_logp(z, tok)[0].isnan().all()
