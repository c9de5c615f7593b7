"""Advantages against the recurrence in 64 bits, step by step (GPU).

Bound: a step's own rounding is at most about 8 eps of the magnitudes in it (reward, two
values, advantage), however the steps are grouped, and reaches earlier steps times (gamma
lam)^k: at most min(T, 1 / (1 - gamma lam)) of it. A grouped product of k decays is off by k
eps relative, times its size (gamma lam)^k, which the same bound covers.
"""

import numpy as np
import pytest
import torch

import swarp_b200 as swarp

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
EPS = {torch.float32: 2.0 ** -24, torch.float64: 2.0 ** -53}


def recurrence(r, v, nxt, last, term, trunc, gamma, lam):
    r, v = (x.cpu().numpy().astype(np.longdouble) for x in (r, v))
    nxt = None if nxt is None else nxt.cpu().numpy().astype(np.longdouble)
    follow = None if last is None else last.cpu().numpy().astype(np.longdouble)

    def flag(x):
        if x is None:
            return np.zeros(r.shape, bool)
        x = x.cpu().numpy()
        return np.broadcast_to(x.reshape(x.shape + (1,) * (r.ndim - x.ndim)), r.shape)

    term, trunc = flag(term), flag(trunc)
    A, ahead = np.zeros_like(r), np.zeros_like(r[0])
    for t in reversed(range(r.shape[0])):
        f = follow if nxt is None else nxt[t]
        d = r[t] + gamma * np.where(term[t], 0, f) - v[t]
        ahead = d + gamma * lam * np.where(term[t] | trunc[t], 0, ahead)
        A[t], follow = ahead, v[t]
    return A, A + v


def check(shape, dtype=torch.float32, gamma=0.99, lam=0.95, ends=0.05, own_next=False, lead=None,
          seed=0, nan_after_end=False):
    g = torch.Generator(device=DEV).manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=g, device=DEV, dtype=dtype)  # noqa: E731
    r, v, last = rn(*shape), 1 + rn(*shape), 1 + rn(*shape[1:])
    nxt = 1 + rn(*shape) if own_next else None
    term = trunc = None
    if ends is not None:
        u = torch.rand(*(lead or shape), generator=g, device=DEV)
        term, trunc = u < ends, (u >= ends) & (u < 2 * ends)
    a, ret = swarp.gae(r, v, last, term, trunc, gamma=gamma, lam=lam, next_values=nxt)
    assert a.shape == ret.shape == r.shape and a.dtype == dtype
    wa, wr = recurrence(r, v, nxt, last, term, trunc, gamma, lam)
    M = float(np.abs(wa).max()) + float(r.abs().max()) + 2 * float(v.abs().max()) + (
        float(nxt.abs().max()) if own_next else float(last.abs().max()))
    reach = min(shape[0], 1 / max(1e-9, 1 - gamma * lam))
    tol = 8 * EPS[dtype] * M * (1 + reach)
    for got, want in ((a, wa), (ret, wr)):
        err = np.abs(got.cpu().numpy().astype(np.longdouble) - want).max()
        assert err <= tol, (float(err), tol)
    return a


STEPS = [1, 2, 3, 7, 8, 9, 31, 32, 33, 63, 64, 65, 100, 127, 128, 129, 255, 256, 257, 511, 512, 513,
         1000, 2047, 2048, 2049, 4100]


@pytest.mark.parametrize("columns", [1, 2, 3, 6, 7, 8, 9, 31, 32, 33, 100])
@pytest.mark.parametrize("T", STEPS)
def test_steps_and_columns(T, columns):
    check((T, columns), seed=T, own_next=T % 2 == 0)


@pytest.mark.parametrize("T,E,A", [(64, 1000, 16), (65, 333, 5), (1, 70000, 2), (20, 12000, 16),
                                   (2000, 40, 3), (20000, 5, 1), (32768, 6, 1), (700, 1000, 3)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
def test_env_flags(T, E, A, dtype):
    check((T, E, A), dtype, lead=(T, E), ends=0.02)
    check((T, E, A), dtype, ends=0.02, own_next=True)  # flags per agent


@pytest.mark.parametrize("gamma,lam", [(1.0, 1.0), (0.0, 0.9), (0.9, 0.0), (0.999, 1.0)])
@pytest.mark.parametrize("shape", [(500, 3), (40, 300)])
def test_discounts(shape, gamma, lam):
    check(shape, gamma=gamma, lam=lam, ends=None)
    check(shape, gamma=gamma, lam=lam, ends=0.5)
    check(shape, torch.float64, gamma=gamma, lam=lam)


@pytest.mark.parametrize("shape", [(40, 6), (900, 4), (3000, 2), (64, 30000)])
def test_a_dropped_value_may_be_anything(shape):
    """NaN and inf values behind terminated steps, and whole episodes of NaN after the last
    end do not reach back across it."""
    g = torch.Generator(device=DEV).manual_seed(4)
    T = shape[0]
    r, v, last = (torch.randn(*s, generator=g, device=DEV) for s in (shape, shape, shape[1:]))
    term = torch.rand(*shape, generator=g, device=DEV) < 0.1
    nxt = torch.randn(*shape, generator=g, device=DEV)
    clean, _ = swarp.gae(r, v, None, term, next_values=nxt)
    dirty, _ = swarp.gae(r, v, None, term,
                         next_values=torch.where(term, torch.full_like(nxt, float("nan")), nxt))
    assert torch.equal(clean, dirty) and not clean.isnan().any()
    term[T // 2] = True  # all that comes after is rubbish
    r2, v2 = r.clone(), v.clone()
    r2[T // 2 + 1:], v2[T // 2 + 1:] = float("nan"), float("inf")
    want, _ = swarp.gae(r, v, last, term)
    got, _ = swarp.gae(r2, v2, last * float("nan"), term)
    assert torch.equal(got[:T // 2 + 1], want[:T // 2 + 1])


def test_truncation_bootstraps_and_cuts():
    r = torch.tensor([[1.0], [2.0], [4.0]], device=DEV)
    v = torch.tensor([[10.0], [20.0], [40.0]], device=DEV)
    nxt = torch.tensor([[100.0], [200.0], [400.0]], device=DEV)
    no = torch.zeros(3, 1, dtype=torch.bool, device=DEV)
    at1 = no.clone()
    at1[1] = True
    a, ret = swarp.gae(r, v, None, no, at1, gamma=0.5, lam=0.5, next_values=nxt)
    # A2 = 4 + 200 - 40; A1 = 2 + 100 - 20 (cut); A0 = 1 + 50 - 10 + 0.25 A1
    assert a[:, 0].tolist() == [41 + 0.25 * 82, 82.0, 164.0]
    a, _ = swarp.gae(r, v, None, at1, no, gamma=0.5, lam=0.5, next_values=nxt)
    assert a[:, 0].tolist() == [41 - 0.25 * 18, -18.0, 164.0]  # terminated: no 0.5 x 200
    assert torch.equal(ret, torch.tensor([[71.5], [102.0], [204.0]], device=DEV))


def test_orders_and_strides():
    g = torch.Generator(device=DEV).manual_seed(1)
    r, v = (torch.randn(50, 12, generator=g, device=DEV) for _ in range(2))
    last = torch.randn(12, generator=g, device=DEV)
    term = torch.rand(50, 12, generator=g, device=DEV) < 0.1
    want = swarp.gae(r, v, last, term)
    got = swarp.gae(r.t().contiguous().t(), v.repeat(1, 2)[:, :12],
                    last.repeat_interleave(2)[::2], term.t().contiguous().t())
    assert all(torch.equal(x, y) for x, y in zip(want, got))
    odd = torch.empty(50 * 12 + 1, device=DEV)
    odd[1:] = r.reshape(-1)
    assert torch.equal(swarp.gae(odd[1:].view(50, 12), v, last, term)[0], want[0])
    one = swarp.gae(r[:, 0].contiguous(), v[:, 0].contiguous(), last[0].clone(),
                    term[:, 0].contiguous())
    assert torch.equal(one[0], swarp.gae(r[:, :1], v[:, :1], last[:1], term[:, :1])[0][:, 0])


def test_empty():
    z = torch.zeros(0, 4, device=DEV)
    a, b = swarp.gae(z, z, torch.zeros(4, device=DEV))
    assert a.shape == b.shape == (0, 4)
    z = torch.zeros(4, 0, device=DEV)
    assert swarp.gae(z, z, z[0])[0].shape == (4, 0)


def test_same_bits_other_streams_and_graphs():
    g = torch.Generator(device=DEV).manual_seed(1)
    r, v = (torch.randn(3000, 5, generator=g, device=DEV) for _ in range(2))
    last = torch.randn(5, generator=g, device=DEV)
    want = swarp.gae(r, v, last)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = swarp.gae(r, v, last)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cap = swarp.gae(r, v, last)
    graph.replay()
    torch.cuda.synchronize()
    for x, y, z in zip(want, other, cap):
        assert torch.equal(x, y) and torch.equal(x, z)


def test_refusals():
    r = torch.zeros(4, 3, 2, device=DEV)
    last = r[0]
    no = torch.zeros(4, 3, dtype=torch.bool, device=DEV)
    with pytest.raises(TypeError):
        swarp.gae(r.half(), r.half(), last.half())
    with pytest.raises(TypeError):
        swarp.gae(r, r.double(), last)
    with pytest.raises(TypeError):
        swarp.gae(r, r, last, no.float())
    with pytest.raises(ValueError):
        swarp.gae(r, r[:3], last)
    with pytest.raises(ValueError):
        swarp.gae(r, r, None)
    with pytest.raises(ValueError):
        swarp.gae(r, r, last, no[:, :2])
    with pytest.raises(ValueError):
        swarp.gae(r, r, last, no, torch.zeros(4, 3, 2, dtype=torch.bool, device=DEV))
    with pytest.raises(ValueError):
        swarp.gae(r, r, last, gamma=1.5)
    with pytest.raises(ValueError):
        swarp.gae(r, r.clone().requires_grad_(True), last)
    with pytest.raises(ValueError):
        swarp.gae(r, r.cpu(), last)
    with pytest.raises(RuntimeError):
        swarp.gae(r.cpu(), r, last)
