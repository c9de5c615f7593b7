"""AdamW steps against the formulas in 64 bits: sizes, types, 8-bit codes, clipping (GPU).

Bounds. m and v are two products and a sum (3 eps of the larger part); the parameter takes a
handful of roundings on its two parts. 8-bit codes must stand for exactly the values that the
definition, in 64 bits, gives for the float32 moments, whose three roundings are fixed.
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
DT = [torch.float32, torch.bfloat16, torch.float16]
HP = dict(lr=1e-3, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.1)
M32 = 0xFFFFFFFF


def mix(x):
    x = x ^ (x >> 16)
    x = (x * 0xE80B5AE5) & M32
    x = x ^ (x >> 15)
    x = (x * 0xCB276749) & M32
    return x ^ (x >> 16)


def hashes(n, seed, step, tensor):
    key = mix((mix((seed + step) & M32) + tensor) & M32)
    return mix(torch.arange(n, device=DEV) ^ key)


def pow2(e):
    """2^e in 64 bits, exactly (the device's pow is not), for whole e above -1022."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def exponent(a):
    """The exponent of a, from -126 up (a float32 below has that step too)."""
    return torch.frexp(a.clamp(min=2.0 ** -126)).exponent.double() - 1


def value(m):
    """What a Moment8 stands for, in 64 bits."""
    n = m.codes.numel()
    E = m.exponents.double().repeat_interleave(256)[:n]
    f = (m.codes % 128 if m.signed else m.codes).double()
    q = f + 8 * E - (112 if m.signed else 247)
    x = pow2(torch.floor(q / 8) - 127) * (1 + (q % 8) / 8)
    x = torch.where(q < 8, q * 2.0 ** -129, x)  # float32 bits below the least exponent
    x = torch.where(f > 0, x, 0.0)
    return torch.where((m.codes > 127) & m.signed, -x, x)


def rounded(x, r16, signed):
    """x in the 8-bit format with the random bits r16, from the definition in 64 bits."""
    n = x.numel()
    a = x.abs().clamp(min=0.0)
    pad = torch.zeros(-n % 256, dtype=torch.float64, device=DEV)
    top = exponent(torch.cat([a, pad]).view(-1, 256).amax(1))
    top = top.repeat_interleave(256)[:n]
    step = pow2(exponent(a) - 3)
    y = torch.floor(a / step + r16.double() / 65536) * step
    # the format's least value, where float32 has it (a smaller block reaches down to 2^-129)
    low = pow2(top - 13) if signed else 1.25 * pow2(top - 31)
    low = torch.where(top >= (-113 if signed else -96), low, 0.0)
    if signed:
        return torch.where(y < low, 0.0, y) * torch.sign(x)
    return torch.where(a > 0, torch.maximum(y, low), 0.0)


def setup(sizes, dtype, bits, seed=0, gscale=1e-2):
    g = torch.Generator(device=DEV).manual_seed(seed)
    rn = lambda n: torch.randn(n, generator=g, device=DEV)  # noqa: E731
    params = [rn(n).to(dtype) for n in sizes]
    grads = [(gscale * rn(n) * torch.exp(rn(n))).to(dtype) for n in sizes]
    masters = None if dtype == torch.float32 else [p.float() for p in params]
    if bits == 32:
        m = [0.1 * gscale * rn(n) for n in sizes]
        v = [(gscale * rn(n)).square() for n in sizes]
    else:
        m = [swarp.Moment8.zeros(n, DEV, True) for n in sizes]
        v = [swarp.Moment8.zeros(n, DEV, False) for n in sizes]
    return params, grads, m, v, masters


def reference(p, g, m, v, step, scale, lr, betas, eps, weight_decay):
    b1, b2 = betas
    g = g.double() * scale
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    upd = (m / (1 - b1 ** step)) / ((v / (1 - b2 ** step)).sqrt() + eps)
    return p.double() * (1 - lr * weight_decay) - lr * upd, m, v, lr * upd.abs()


def near(got, want, tol, what):
    bad = ~((got.double() - want).abs() <= tol)
    assert not bad.any(), (what, int(bad.sum()), float((got.double() - want).abs().max()))


def check_step(state, step, bits, seed=3, max_norm=None, hp=HP):
    params, grads, m, v, masters = state
    before = [(masters or params)[i].clone() for i in range(len(params))]
    m0 = [value(x) if bits == 8 else x.double() for x in m]
    v0 = [value(x) if bits == 8 else x.double() for x in v]
    norm = swarp.adamw_step(params, grads, m, v, step=step, seed=seed, max_norm=max_norm,
                            masters=masters, **hp)
    scale = 1.0
    if max_norm is not None:
        true = math.sqrt(sum(float(x.double().square().sum()) for x in grads))
        assert abs(float(norm) - true) <= 16 * EPS * true
        scale = min(1.0, max_norm / (true + 1e-6))
    else:
        assert norm is None
    for i, g in enumerate(grads):
        p, m1, v1, upd = reference(before[i], g, m0[i], v0[i], step, scale, **hp)
        got = (masters or params)[i]
        near(got, p, 16 * EPS * (before[i].double().abs() + upd) + 64 * EPS * upd, "param")
        if masters:
            assert torch.equal(params[i], got.to(params[i].dtype))
        mt = 20 * EPS * (m0[i].abs() + (g.double() * scale).abs())
        vt = 20 * EPS * v1 + 1e-44
        if bits == 32:
            near(m[i], m1, mt, "m")
            near(v[i], v1, vt, "v")
            continue
        if g.numel() == 0:
            continue
        # the new moments with their roundings written out: the codes are then exactly theirs
        assert scale == 1.0
        b1, b2 = hp["betas"]
        g32 = g.float()
        m32 = m0[i].float() * b1 + g32 * (1 - b1)
        v32 = v0[i].float() * b2 + (g32 * (1 - b2)) * g32
        near(m32, m1, mt, "m before rounding")
        near(v32, v1, vt, "v before rounding")
        h = hashes(g.numel(), seed, step, i)
        for x, want, r, signed in ((m[i], m32, h & 0xFFFF, True), (v[i], v32, h >> 16, False)):
            got = value(x)
            assert torch.equal(got, rounded(want.double(), r, signed))
            assert torch.equal(x.values(torch.float32).double(), got)
            assert torch.equal(x.values().double(), got)  # bfloat16 holds them exactly


SIZES = [[1], [2, 3], [255, 256, 257], [1, 0, 5], [4096, 4095, 4097], [8192, 12345, 7],
         [100003], [1 << 20, 3]]


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("sizes", SIZES, ids=str)
def test_sizes(sizes, dtype, bits):
    st = setup(sizes, dtype, bits)
    for step in (1, 2, 3):
        check_step(st, step, bits)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("count", [383, 384, 385, 1000])
def test_many_tensors(count, bits):
    """More tensors than one launch's parameters hold."""
    sizes = [(i * 37) % 700 for i in range(count)]
    st = setup(sizes, torch.bfloat16, bits)
    check_step(st, 1, bits, max_norm=0.5 if bits == 32 else 1e6)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("max_norm", [1e-3, 0.7, 1e5])
def test_clipping(dtype, max_norm):
    check_step(setup([5000, 33, 70001], dtype, 32), 1, 32, max_norm=max_norm)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", DT)
def test_odd_addresses(dtype, bits):
    """Tensors that start off any vector boundary."""
    sizes = [1000, 513, 4099]
    params, grads, m, v, masters = setup(sizes, dtype, bits)

    def off(t):
        u = torch.empty(t.numel() + 1, dtype=t.dtype, device=DEV)
        u[1:] = t
        return u[1:]

    if bits == 8:
        m = [swarp.Moment8(off(x.codes), off(x.exponents), True) for x in m]
        v = [swarp.Moment8(off(x.codes), off(x.exponents), False) for x in v]
    else:
        m, v = [off(x) for x in m], [off(x) for x in v]
    st = ([off(x) for x in params], [off(x) for x in grads], m, v,
          None if masters is None else [off(x) for x in masters])
    for step in (1, 2):
        check_step(st, step, bits)
    # one odd tensor of the set, the others aligned; and the same bits as all aligned
    a, b = setup(sizes, dtype, bits, seed=9), setup(sizes, dtype, bits, seed=9)
    b[1][1] = off(b[1][1])
    for s in (a, b):
        swarp.adamw_step(s[0], s[1], s[2], s[3], step=1, masters=s[4], **HP)
    for i in range(3):
        assert torch.equal(a[0][i], b[0][i])
        x, y = (s[2][i] if bits == 32 else s[2][i].codes for s in (a, b))
        assert torch.equal(x, y)


def test_8_bit_rounding_is_unbiased_and_does_not_stall():
    """Constant gradients: the averages must reach g and g^2, in expectation and without
    freezing. After k steps from zero v / g^2 = 1 - b2^k. Each step's rounding is unbiased;
    its standard deviation is below half a step (1/16), and the last 1 / (1 - b2^2) of them
    add up, each with probability about (1 - b2) / (1/8): a relative deviation under 0.3 per
    element, so the mean over n elements is within 6 x 0.3 / sqrt(n)."""
    n, b1, b2, k = 65536, 0.9, 0.999, 3000
    p, g = [torch.zeros(n, device=DEV)], [torch.full((n,), 0.01, device=DEV)]
    m, v = [swarp.Moment8.zeros(n, DEV, True)], [swarp.Moment8.zeros(n, DEV, False)]
    for step in range(1, k + 1):
        swarp.adamw_step(p, g, m, v, step=step, lr=0.0, betas=(b1, b2), weight_decay=0.0)
    room = 6 * 0.3 / math.sqrt(n)
    for x, want in ((m[0], 0.01), (v[0], 1e-4 * (1 - b2 ** k))):
        got = value(x)
        assert abs(float(got.mean()) / want - 1) <= room, float(got.mean()) / want
        assert float(got.std()) / want < 0.35
    # and decay again once the gradients vanish
    g[0].zero_()
    for step in range(k + 1, 2 * k + 1):
        swarp.adamw_step(p, g, m, v, step=step, lr=0.0, betas=(b1, b2), weight_decay=0.0)
    want = 1e-4 * (1 - b2 ** k) * b2 ** k
    assert abs(float(value(v[0]).mean()) / want - 1) <= 3 * room
    assert float(value(m[0]).abs().max()) < 1e-25


def test_8_bit_range_and_zeros():
    """Within a block: 16 octaves of the first moment below its largest element, 30 of the
    second; a second moment that is not zero never becomes zero; zeros stay zeros."""
    n = 512
    g = torch.zeros(n, device=DEV)
    g[0] = 1.0
    g[1:200] = 2.0 ** -torch.arange(1, 200, device=DEV).float().clamp(max=60)
    st = ([torch.zeros(n, device=DEV)], [g], [swarp.Moment8.zeros(n, DEV, True)],
          [swarp.Moment8.zeros(n, DEV, False)], None)
    check_step(st, 1, 8)
    m, v = value(st[2][0]), value(st[3][0])
    assert (m[1:13] > 0).all() and (m[15:] == 0).all()
    assert (v[:60] > 0).all() and (v[200:] == 0).all()
    assert int(st[2][0].exponents[1]) == 0 and int(st[3][0].exponents[1]) == 0
    assert float(v[60]) == float(v[100])  # the smallest value of the block
    # tiny and huge gradients, down to second moments that are subnormal or zero
    for scale in (1e-30, 1e-22, 1e-18, 1e-15, 1e15):
        st = setup([700], torch.float32, 8, gscale=scale)
        check_step(st, 1, 8)


def test_nan_is_loud():
    for bits in (32, 8):
        p, g, m, v, w = setup([600, 600], torch.float32, bits)
        g[0][300] = math.nan
        swarp.adamw_step(p, g, m, v, step=1, **HP)
        assert p[0][300].isnan() and int(p[0].isnan().sum()) == 1 and not p[1].isnan().any()
        mm = m[0] if bits == 32 else m[0].values(torch.float32)
        assert mm[300].isnan()
        norm = swarp.adamw_step(p, g, m, v, step=2, max_norm=1.0, **HP)
        assert norm.isnan() and p[1].isnan().all()


def test_deterministic_across_streams_and_graphs():
    for bits in (32, 8):
        runs = []
        for how in ("plain", "stream", "graph"):
            st = setup([70000, 5, 333], torch.bfloat16, bits, seed=5)
            go = lambda: swarp.adamw_step(st[0], st[1], st[2], st[3], step=7,  # noqa: E731
                                          masters=st[4], max_norm=0.3, **HP)
            if how == "plain":
                norm = go()
            elif how == "stream":
                side = torch.cuda.Stream()
                side.wait_stream(torch.cuda.current_stream())
                with torch.cuda.stream(side):
                    norm = go()
            else:
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph):
                    norm = go()
                graph.replay()
            torch.cuda.synchronize()
            flat = [x if bits == 32 else x.codes for x in st[2] + st[3]]
            runs.append([norm.clone(), *st[0], *st[4], *flat])
        for other in runs[1:]:
            assert all(torch.equal(a, b) for a, b in zip(runs[0], other))


@pytest.mark.parametrize("bits", [32, 8])
def test_optimizer(bits):
    """The class against the function: groups, missing gradients, state_dict, version."""
    g = torch.Generator(device=DEV).manual_seed(0)
    make = lambda *s, dtype=torch.float32: torch.nn.Parameter(  # noqa: E731
        torch.randn(*s, generator=g, device=DEV).to(dtype))
    ps = [make(30, 20), make(20), make(7, 9, dtype=torch.bfloat16), make(5), make(300)]
    start = [p.detach().clone() for p in ps]
    opt = swarp.AdamW([{"params": ps[:3]}, {"params": ps[3:], "lr": 0.05, "weight_decay": 0.0}],
                      lr=0.01, max_norm=0.5, state_bits=bits, seed=11)
    sched = torch.optim.lr_scheduler.StepLR(opt, 1, 0.5)
    gr = [torch.randn(p.shape, generator=g, device=DEV).to(p.dtype) for p in ps]
    for p, x in zip(ps, gr):
        p.grad = x.clone()
    ps[1].grad = None  # left out
    ps[0].grad = gr[0].t().contiguous().t()  # another memory order
    version = ps[0]._version
    opt.step()
    sched.step()
    assert ps[0]._version > version and torch.equal(ps[1], start[1])
    true = math.sqrt(sum(float(x.double().square().sum()) for i, x in enumerate(gr) if i != 1))
    assert abs(float(opt.grad_norm) - true) <= 1e-5 * true
    scale = 0.5 / (true + 1e-6)
    for i in (0, 2, 3, 4):
        lr, wd = (0.01, 0.01) if i < 3 else (0.05, 0.0)
        want, _, _, _ = reference(start[i].float(), gr[i], 0.0, 0.0, 1, scale, lr, (0.9, 0.999),
                                  1e-8, wd)
        near(ps[i], want, 1e-5 * (want.abs() + lr) + want.abs() * ULP[ps[i].dtype], i)
    # a copy made from the state dict goes on with the same bits
    copies = [torch.nn.Parameter(p.detach().clone()) for p in ps]
    opt2 = swarp.AdamW([{"params": copies[:3]}, {"params": copies[3:]}], max_norm=0.5,
                       state_bits=bits, seed=11)
    import copy
    opt2.load_state_dict(copy.deepcopy(opt.state_dict()))
    assert opt2.param_groups[1]["lr"] == opt.param_groups[1]["lr"] != 0.05
    for step in range(2):
        for group in (ps, copies):
            for p, x in zip(group, gr):
                p.grad = x.clone()
        opt.step()
        opt2.step()
    for a, b in zip(ps, copies):
        assert torch.equal(a, b)
        sa, sb = opt.state[a], opt2.state[b]
        assert sa["step"] == sb["step"]
        for k in sa:
            if torch.is_tensor(sa[k]):
                assert sa[k].dtype == sb[k].dtype and torch.equal(sa[k], sb[k]), k
    want = torch.uint8 if bits == 8 else torch.float32
    assert opt.state[ps[0]]["exp_avg"].dtype == want


def test_optimizer_trains():
    g = torch.Generator(device=DEV).manual_seed(0)
    X = torch.randn(4096, 16, generator=g, device=DEV)
    Y = X @ torch.randn(16, 3, generator=g, device=DEV)
    for bits in (32, 8):
        W = torch.nn.Parameter(torch.zeros(16, 3, device=DEV))
        opt = swarp.AdamW([W], lr=0.05, weight_decay=0.0, state_bits=bits, max_norm=10.0)
        for _ in range(300):
            opt.zero_grad()
            loss = (X @ W - Y).square().mean()
            loss.backward()
            opt.step()
        assert float(loss) < 1e-2 * float(Y.square().mean()), (bits, float(loss))


def test_refusals():
    p, g, m, v, _ = setup([10, 20], torch.float32, 32)
    bad = dict(step=1, lr=1e-3)
    with pytest.raises(ValueError):
        swarp.adamw_step(p, g[:1], m, v, **bad)
    with pytest.raises(ValueError):
        swarp.adamw_step(p, [g[1], g[0]], m, v, **bad)
    with pytest.raises(TypeError):
        swarp.adamw_step(p, [x.half() for x in g], m, v, **bad)
    with pytest.raises(TypeError):
        swarp.adamw_step([x.double() for x in p], [x.double() for x in g], m, v, **bad)
    with pytest.raises(ValueError):
        swarp.adamw_step([x.half() for x in p], [x.half() for x in g], m, v, **bad)
    with pytest.raises(ValueError):
        swarp.adamw_step(p, g, m, v, masters=p, **bad)
    with pytest.raises(ValueError):
        swarp.adamw_step([p[0], p[1].expand(2, 20)[:, 0]], g, m, v, **bad)
    with pytest.raises(ValueError):
        swarp.adamw_step([p[0], p[1].repeat(2)[::2]], g, m, v, **bad)
    with pytest.raises(ValueError):
        swarp.adamw_step(p, g, m, v, step=0, lr=1e-3)
    with pytest.raises(ValueError):
        swarp.adamw_step(p, g, m, v, max_norm=0.0, **bad)
    with pytest.raises(ValueError):
        swarp.adamw_step(p, g, m, v, betas=(1.0, 0.9), **bad)
    with pytest.raises(ValueError):
        swarp.adamw_step([], [], [], [], **bad)
    m8 = [swarp.Moment8.zeros(n, DEV, True) for n in (10, 20)]
    v8 = [swarp.Moment8.zeros(n, DEV, False) for n in (10, 20)]
    with pytest.raises(TypeError):
        swarp.adamw_step(p, g, v8, m8, **bad)
    with pytest.raises(ValueError):
        swarp.adamw_step(p, g, m8, [v8[0], swarp.Moment8.zeros(21, DEV, False)], **bad)
    with pytest.raises(RuntimeError):
        swarp.adamw_step([x.cpu() for x in p], g, m, v, **bad)
    with pytest.raises(TypeError):
        m8[0].values(torch.float16)
    with pytest.raises(ValueError):
        swarp.AdamW(p, state_bits=4)
