"""The clipped policy loss, its gradient and token log probabilities against the formulas in
64 bits, at the rows, vocabularies, strides and masks where they can go wrong (GPU).

Bounds. With eps = 2^-24, x = z - max and S = sum e^x: an exponential is off by a few eps
and eps |x| of its argument, a sum of V terms split over at least 32 lanes by (V / 32 + 16)
eps at most, so lp = x_a - ln S is off by eps (2 max|x| + V / 32 + 64) at most, and so are
the entropy (a weighted mean of x), the ratio and p (relative). Gradients are c p and eta p
(ln p + H): three such factors, times the row's coefficient, then one rounding to the output
type (half an ulp; float16 has subnormals of 2^-24).
"""

import math

import pytest
import torch

import swarp_b200 as swarp

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
EPS = 2.0 ** -24
# half an ulp, relative: 8, 11 and 24 bits of significand
ULP = {t: torch.finfo(t).eps / 2 for t in (torch.float32, torch.bfloat16, torch.float16)}


def batch(rows, V, dtype, seed=0, spread=2.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    z = (torch.randn(rows, V, generator=g, device=DEV) * spread).to(dtype)
    tok = torch.randint(0, V, (rows,), generator=g, device=DEV)
    lp = torch.log_softmax(z.double(), 1).gather(1, tok[:, None]).squeeze(1)
    t = torch.randn(rows, generator=g, device=DEV) * 0.3
    for b in (math.log(0.8), math.log(1.2)):  # rounding must not decide what the clip does
        t = torch.where((t - b).abs() < 1e-3, t + 3e-3, t)
    old = (lp - t).float()
    adv = torch.randn(rows, generator=g, device=DEV)
    ref = (lp + 0.4 * torch.randn(rows, generator=g, device=DEV)).float()
    return z, tok, old, adv, ref


def formula(z, tok, old, adv, ref, mask, kl, ent, mean=True, lo=0.2, hi=0.2, empty=None):
    """Per-row terms and the loss in 64 bits, differentiable; z float64."""
    logs = torch.log_softmax(z, -1)
    logs = torch.where(z == -math.inf, torch.full_like(logs, -1e300), logs)
    lp = logs.gather(-1, tok[..., None]).squeeze(-1)
    H = -(logs.exp() * logs).sum(-1)
    r = (lp - old.double()).exp()
    A = adv.double()
    pg = -torch.min(r * A, r.clamp(1 - lo, 1 + hi) * A)
    k3 = torch.zeros_like(pg)
    if ref is not None:
        d = ref.double() - lp
        k3 = d.exp() - d - 1
    live = torch.ones_like(pg, dtype=torch.bool) if mask is None else mask
    n = int(live.sum()) if mean else 1
    term = pg + kl * k3 - ent * H
    return (term[live].sum() / n, lp, H,
            torch.stack([x[live].sum() / n for x in (pg, k3, H)]).detach())


def close(got, want, tol, what):
    err = (got.double() - want).abs()
    bad = ~(err <= tol)
    assert not bad.any(), (what, float(err.max()), float((tol * torch.ones_like(err)).min()))


def check(z, tok, old, adv, ref, mask=None, kl=0.05, ent=0.01, mean=True, scale=1.0, autograd=False):
    V = z.shape[-1]
    kw = dict(ref_logp=ref, mask=mask, kl_coef=kl if ref is not None else 0.0, entropy_coef=ent,
              reduction="mean" if mean else "sum")
    if autograd:
        leaf = z.detach().requires_grad_(True)
        out = swarp.policy_loss(leaf, tok, old, adv, **kw)
        (out.loss * scale).backward()
        grad = leaf.grad
    else:
        out, grad = swarp.policy_loss_and_grad(z, tok, old, adv, grad_scale=scale, **kw)
    z64 = z.detach().double().requires_grad_(True)
    loss, lp, H, stats = formula(z64, tok.long(), old, adv, ref, mask, kw["kl_coef"], ent, mean)
    (loss * scale).backward()
    live = torch.ones_like(lp, dtype=torch.bool) if mask is None else mask
    fin = z64.detach()[live]
    fin = fin[fin > -1e30]
    spread = float(fin.max() - fin.min()) if fin.numel() else 0.0
    tol = EPS * (2 * spread + V / 32 + 64)
    close(out.logp[live], lp.detach()[live], tol, "logp")
    close(out.entropy[live], H.detach()[live], 2 * tol, "entropy")
    assert not out.logp[~live].any() and not out.entropy[~live].any()
    n = max(1, int(live.sum())) if mean else 1
    # each row's terms are at most about e^1.2 |A| and e^1.6 here: 8 covers both
    size = float(adv[live].abs().max()) * 8 + 8 if live.any() else 1.0
    rows = int(live.sum()) / n
    close(out.loss, loss.detach(), rows * size * 4 * tol + 1e-12, "loss")
    close(out.stats[:3], stats, rows * size * 4 * tol + 1e-12, "stats")
    assert grad.shape == z.shape and grad.dtype == z.dtype and grad.is_contiguous()
    want = z64.grad.nan_to_num(0.0)
    room = scale / n * (size + ent * (spread + 8)) * 8 * tol
    sub = 2.0 ** -25 if z.dtype == torch.float16 else 0.0
    # the clip and KL parts cancel to some extent, so the room is that of the parts
    p = torch.softmax(z64.detach(), -1).nan_to_num(0.0)
    hot = torch.zeros_like(p).scatter_(-1, tok.long()[..., None], 1.0)
    close(grad, want, room * (p + hot) + want.abs() * ULP[z.dtype] + sub + 1e-35, "grad")
    if mask is not None:
        assert not grad[~mask].any()
    return out, grad


VOCABS = [1, 2, 3, 5, 8, 21, 25, 31, 32, 33, 64, 100, 127, 128, 200, 256, 257, 511, 512, 777,
          1000, 1024, 1025, 2048, 2049, 4095, 4096, 4099, 8191, 8192, 9001, 16384, 16385, 20011,
          32768, 40000, 65536, 70001, 131072, 262145, 300007]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("V", VOCABS)
def test_vocabularies(V, dtype):
    rows = 7 if V > 4096 else 301
    check(*batch(rows, V, dtype, seed=V))


@pytest.mark.parametrize("rows,V", [(1, 1), (1, 7), (1, 50000), (2, 3), (9999, 4), (4097, 40),
                                    (3001, 300), (2500, 1500), (100000, 21)])
@pytest.mark.parametrize("autograd", [False, True])
def test_rows_and_autograd(rows, V, autograd):
    for mean in (True, False):
        check(*batch(rows, V, torch.float32, seed=rows), mean=mean, autograd=autograd)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("V", [17, 600, 5000, 40007])
def test_masked_rows_are_not_read(V, dtype):
    rows = 57
    z, tok, old, adv, ref = batch(rows, V, dtype, seed=3)
    mask = torch.arange(rows, device=DEV) % 3 != 1
    z[~mask], tok[~mask] = math.nan, -100
    for t in (old, adv, ref):
        t[~mask] = math.nan
    zc, tc = z.clone(), tok.clone()
    zc[~mask], tc[~mask] = 0.0, 0
    fix = lambda t: torch.where(mask, t, torch.zeros_like(t))  # noqa: E731
    # the formula with harmless values in the masked places, the kernel with NaN
    out, grad = swarp.policy_loss_and_grad(z, tok, old, adv, ref_logp=ref, mask=mask, kl_coef=0.05,
                                           entropy_coef=0.01)
    want, wgrad = check(zc, tc, fix(old), fix(adv), fix(ref), mask=mask)
    assert torch.equal(grad, wgrad)
    for a, b in zip(out, want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("V", [5, 900, 30000])
def test_no_row_admitted(V):
    z, tok, old, adv, ref = batch(6, V, torch.float32)
    mask = torch.zeros(6, dtype=torch.bool, device=DEV)
    out, grad = swarp.policy_loss_and_grad(z, tok, old, adv, mask=mask, entropy_coef=0.1)
    assert float(out.loss) == 0.0 and not grad.any() and not out.stats.any()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("V", [9, 130, 1500, 3000, 20000, 150000])
def test_barred_tokens(V, dtype):
    """Logits of -inf, and of the type's lowest value, among others."""
    z, tok, old, adv, ref = batch(40, V, dtype, seed=V)
    g = torch.Generator(device=DEV).manual_seed(1)
    bar = torch.rand(40, V, generator=g, device=DEV) < 0.5
    bar.scatter_(1, tok[:, None], False)
    bar[5:9, V // 2:] = True  # long barred stretches
    bar.scatter_(1, tok[:, None], False)
    low = torch.finfo(dtype).min
    z[:20] = torch.where(bar[:20], -math.inf, z[:20])
    z[20:] = torch.where(bar[20:], low, z[20:])
    lp = torch.log_softmax(z.double(), 1).gather(1, tok[:, None]).squeeze(1)
    out, grad = check(z, tok, (lp - 0.05).float(), adv, (lp + 0.1).float())
    assert not grad[bar].any()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("V", [6, 70, 700, 2500, 30000])
def test_rows_without_an_ordinary_logit(V, dtype):
    """Rows of -inf alone, of the lowest value alone, of one lowest among -inf, of the largest
    value alone, and of a NaN or an inf among others."""
    f = torch.finfo(dtype)
    z = torch.zeros(6, V, dtype=dtype, device=DEV)
    z[0] = -math.inf
    z[1] = f.min
    z[2] = -math.inf
    z[2, V // 2] = f.min
    z[3] = f.max
    z[4, V // 3] = math.nan
    z[5, V // 3] = math.inf
    tok = torch.full((6,), V // 2, device=DEV)
    old = torch.full((6,), -math.log(V), device=DEV)
    adv = torch.ones(6, device=DEV)
    logp, ent = swarp.token_logp(z, tok)
    lnV = math.log(V)
    tol = EPS * (V / 32 + 64) * max(1.0, lnV)
    assert logp[0] == -math.inf and ent[0] == 0.0
    close(logp[[1, 3]], torch.full((2,), -lnV, dtype=torch.float64, device=DEV), tol, "uniform")
    close(ent[[1, 3]], torch.full((2,), lnV, dtype=torch.float64, device=DEV), 2 * tol, "uniform")
    assert abs(float(logp[2])) <= tol and abs(float(ent[2])) <= tol
    assert logp[4:].isnan().all()
    mask = torch.tensor([1, 1, 0, 1, 0, 0], dtype=torch.bool, device=DEV)
    out, grad = swarp.policy_loss_and_grad(z, tok, old, adv, mask=mask, entropy_coef=0.02,
                                           reduction="sum", clip_low=1.0, clip_high=9.0)
    # row 0 adds nothing; rows 1 and 3 are uniform with ratio 1: p - 1{token}, entropy flat
    assert not grad[0].any()
    want = torch.full((V,), 1.0 / V, dtype=torch.float64, device=DEV)
    want[V // 2] -= 1.0
    for i in (1, 3):
        close(grad[i], want, want.abs() * ULP[dtype] + 16 * tol + 2.0 ** -25, "uniform grad")
    close(out.loss, torch.tensor(-2.0 - 0.02 * 2 * lnV, dtype=torch.float64, device=DEV),
          64 * tol, "loss")
    bad, g4 = swarp.policy_loss_and_grad(z, tok, old, adv)
    assert bad.loss.isnan() and g4[4].isnan().all()


@pytest.mark.parametrize("V", [6, 300, 5000, 50000])
def test_token_out_of_range_is_loud(V):
    z, tok, old, adv, ref = batch(5, V, torch.float32)
    for bad in (-1, V, V + 7, -100, 1 << 40):
        tok[2] = bad
        out, _ = swarp.policy_loss_and_grad(z, tok, old, adv)
        assert out.logp[2].isnan() and out.loss.isnan()
        assert not out.logp[[0, 1, 3, 4]].isnan().any()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [21, 260, 1300, 9000, 33000])
def test_strides_and_layouts(V, dtype):
    """A sequence batch without its last step, a vocabulary with padding, steps before
    sequences, one row for all, and rows at an odd address."""
    B, T = 3, 5
    z, tok, old, adv, ref = batch(B * T, V, dtype, seed=V)
    base = swarp.policy_loss_and_grad(z, tok, old, adv, ref_logp=ref, kl_coef=0.1,
                                      entropy_coef=0.01)

    def same(zz, shape, order=lambda t: t):
        args = [order(t.reshape(B, T)).contiguous() for t in (tok, old, adv, ref)]
        out, grad = swarp.policy_loss_and_grad(zz, *args[:3], ref_logp=args[3], kl_coef=0.1,
                                               entropy_coef=0.01)
        assert grad.shape == shape
        # an alignment of its own may take another order of summation
        tol = EPS * (40 + V / 16 + 128)
        back = order(out.logp) if order(out.logp).shape == (B, T) else out.logp
        close(back.reshape(-1), base[0].logp.double(), tol, "logp")
        gback = grad.transpose(0, 1) if shape[0] == T and shape != (B, T, V) else grad
        ref_grad = base[1].double()
        close(gback.reshape(B * T, V), ref_grad, ref_grad.abs() * 2 * ULP[dtype] + 8 * tol, "grad")

    long = torch.full((B, T + 1, V), math.nan, dtype=dtype, device=DEV)
    long[:, :-1] = z.view(B, T, V)
    same(long[:, :-1], (B, T, V))
    wide = torch.full((B, T, V + 3), math.nan, dtype=dtype, device=DEV)
    wide[..., :V] = z.view(B, T, V)
    same(wide[..., :V], (B, T, V))
    wide4 = torch.full((B, T + 2, V + 5), math.nan, dtype=dtype, device=DEV)
    wide4[:, 1:-1, 2:-3] = z.view(B, T, V)
    same(wide4[:, 1:-1, 2:-3], (B, T, V))
    odd = torch.empty(B * T * V + 1, dtype=dtype, device=DEV)
    odd[1:] = z.reshape(-1)
    same(odd[1:].view(B, T, V), (B, T, V))
    steps_first = z.view(B, T, V).transpose(0, 1)
    same(steps_first, (T, B, V), lambda t: t.transpose(0, 1))
    copied = z.view(B, T, V).transpose(1, 2).contiguous().transpose(1, 2)  # V not adjacent
    same(copied, (B, T, V))
    one = z[:1].expand(6, V)  # a stride of zero
    out, grad = swarp.policy_loss_and_grad(one, tok[:6], old[:6], adv[:6])
    alone = [swarp.policy_loss_and_grad(z[:1], tok[i:i + 1], old[i:i + 1], adv[i:i + 1])[0].logp
             for i in range(6)]
    close(out.logp, torch.cat(alone).double(), EPS * (40 + V / 16 + 128), "expanded")


def test_leading_shapes_and_int32_tokens():
    z, tok, old, adv, ref = batch(2 * 3 * 4, 11, torch.float32)
    flat = swarp.policy_loss_and_grad(z, tok, old, adv)
    sh = (2, 3, 4)
    out, grad = swarp.policy_loss_and_grad(z.view(*sh, 11), tok.int().view(sh), old.view(sh),
                                           adv.view(sh))
    assert torch.equal(out.logp.reshape(-1), flat[0].logp) and out.logp.shape == sh
    assert torch.equal(grad.reshape(-1, 11), flat[1]) and torch.equal(out.loss, flat[0].loss)
    single, g1 = swarp.policy_loss_and_grad(z[0], tok[0], old[0], adv[0])  # no leading dimension
    assert single.logp.shape == () and g1.shape == (11,)
    empty, g0 = swarp.policy_loss_and_grad(z[:0], tok[:0], old[:0], adv[:0])
    assert float(empty.loss) == 0.0 and g0.shape == (0, 11)


@pytest.mark.parametrize("V", [40, 4000, 50001])
def test_gradient_against_differences(V):
    """Central differences of the 64-bit loss in random directions."""
    z, tok, old, adv, ref = batch(12, V, torch.float32, seed=8)
    mask = torch.arange(12, device=DEV) % 4 != 2
    _, grad = swarp.policy_loss_and_grad(z, tok, old, adv, ref_logp=ref, mask=mask, kl_coef=0.2,
                                         entropy_coef=0.05)
    g = torch.Generator(device=DEV).manual_seed(2)
    for _ in range(4):
        u = torch.randn(12, V, generator=g, device=DEV, dtype=torch.float64)
        u.scatter_add_(1, tok[:, None], 3 * torch.ones(12, 1, device=DEV, dtype=torch.float64))
        h = 1e-5
        f = [formula(z.double() + s * h * u, tok, old, adv, ref, mask, 0.2, 0.05)[0]
             for s in (1, -1)]
        d = float((f[0] - f[1]) / (2 * h))
        got = float((grad.double() * u).sum())
        assert abs(got - d) <= 1e-6 * (1 + float((grad.double() * u).abs().sum())), (got, d)


def test_cotangent_and_second_backward():
    z, tok, old, adv, ref = batch(33, 2000, torch.bfloat16)
    leaf = z.clone().requires_grad_(True)
    out = swarp.policy_loss(leaf, tok, old, adv, entropy_coef=0.01)
    (g1,) = torch.autograd.grad(out.loss, leaf, retain_graph=True)
    keep = g1.clone()
    (g2,) = torch.autograd.grad(out.loss, leaf, retain_graph=True)
    (g3,) = torch.autograd.grad(4.0 * out.loss, leaf)
    assert torch.equal(g1, keep) and torch.equal(g1, g2) and g1.data_ptr() != g2.data_ptr()
    assert torch.equal(g3, (4.0 * g1.float()).to(z.dtype))  # a power of two scales exactly
    assert torch.equal(g1, swarp.policy_loss_and_grad(z, tok, old, adv, entropy_coef=0.01)[1])
    assert not out.logp.requires_grad and not out.stats.requires_grad
    with pytest.raises(RuntimeError):
        out.loss.backward()


def test_float16_loss_scale_keeps_small_gradients():
    z, tok, old, adv, ref = batch(8192, 64, torch.float16)
    check(z, tok, old, adv, ref, scale=65536.0)
    check(z, tok, old, adv, ref, scale=65536.0, autograd=True)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,V", [(1, 2), (5, 100), (1, 131072), (3, 99991), (1000, 21),
                                    (64, 4100), (700, 2048)])
def test_token_logp(rows, V, dtype):
    z, tok, *_ = batch(rows, V, dtype, seed=V + 1)
    logp, ent = swarp.token_logp(z, tok)
    logs = torch.log_softmax(z.double(), 1)
    tol = EPS * (40 + V / 32 + 64)
    close(logp, logs.gather(1, tok[:, None]).squeeze(1), tol, "logp")
    close(ent, -(logs.exp() * logs).sum(1), 2 * tol, "entropy")


def test_large_offsets():
    """Rows beyond element 2^31 of the logits and of the gradient."""
    V = 131072
    rows = (1 << 31) // V + 8
    z = torch.zeros(rows, V, dtype=torch.bfloat16, device=DEV)
    small, tok, old, adv, ref = batch(16, V, torch.bfloat16)
    z[-16:] = small
    mask = torch.zeros(rows, dtype=torch.bool, device=DEV)
    mask[-16:] = True
    pad = lambda t: torch.cat([t.new_zeros(rows - 16), t])  # noqa: E731
    out, grad = swarp.policy_loss_and_grad(z, pad(tok), pad(old), pad(adv), mask=mask)
    want, wgrad = swarp.policy_loss_and_grad(small, tok, old, adv)
    assert torch.equal(grad[-16:], wgrad) and torch.equal(out.logp[-16:], want.logp)
    assert not grad[:64].any() and not grad[-64:-16].any()


def test_same_bits_other_streams_and_graphs():
    z, tok, old, adv, ref = batch(5000, 45, torch.float32)
    big = batch(9, 70000, torch.bfloat16)
    first = swarp.policy_loss_and_grad(z, tok, old, adv, ref_logp=ref, kl_coef=0.1)
    firstb = swarp.policy_loss_and_grad(*big[:4], entropy_coef=0.1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = swarp.policy_loss_and_grad(z, tok, old, adv, ref_logp=ref, kl_coef=0.1)
        againb = swarp.policy_loss_and_grad(*big[:4], entropy_coef=0.1)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cap = swarp.policy_loss_and_grad(z, tok, old, adv, ref_logp=ref, kl_coef=0.1)
        capb = swarp.policy_loss_and_grad(*big[:4], entropy_coef=0.1)
    graph.replay()
    torch.cuda.synchronize()
    for a, b in ((first, again), (first, cap), (firstb, againb), (firstb, capb)):
        assert torch.equal(a[1], b[1])
        assert all(torch.equal(x, y) for x, y in zip(a[0], b[0]))


def test_refusals():
    z, tok, old, adv, ref = batch(4, 6, torch.float32)
    call = swarp.policy_loss_and_grad
    with pytest.raises(TypeError):
        call(z.double(), tok, old, adv)
    with pytest.raises(TypeError):
        call(z, tok.float(), old, adv)
    with pytest.raises(TypeError):
        call(z, tok, old.double(), adv)
    with pytest.raises(TypeError):
        call(z, tok, old, None)
    with pytest.raises(TypeError):
        call(z, tok, old, adv, mask=torch.ones(4, device=DEV))
    with pytest.raises(ValueError):
        call(z, tok[:3], old, adv)
    with pytest.raises(ValueError):
        call(z, tok, old, adv[:, None])
    with pytest.raises(ValueError):
        call(z, tok.cpu(), old, adv)
    with pytest.raises(ValueError):
        call(z, tok, old, adv, kl_coef=0.1)
    with pytest.raises(ValueError):
        call(z, tok, old, adv, clip_low=1.5)
    with pytest.raises(ValueError):
        call(z, tok, old, adv, clip_high=-0.1)
    with pytest.raises(ValueError):
        call(z, tok, old, adv, reduction="none")
    with pytest.raises(ValueError):
        call(z[:, :0], tok, old, adv)
    with pytest.raises(ValueError):
        call(z, tok, old, adv.clone().requires_grad_(True))
    with pytest.raises(ValueError):
        swarp.token_logp(z.clone().requires_grad_(True), tok)
    with pytest.raises(RuntimeError):
        call(z.cpu(), tok, old, adv)
