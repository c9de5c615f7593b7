"""The policy-training operators as workloads: the token policy loss with its gradient,
advantage estimation over a rollout, and the AdamW step.

``listed()`` names the workloads, ``draw(rng)`` gives more of the same ranges,
``prepare`` makes what a training program has in hand, and ``run`` is one call of the
operator: with ``own`` the framework's kernels, otherwise the plain form in elementary
torch operations and 32 bits. ``exact`` is the definition in 64 bits.

The loss. A policy chooses one of V tokens per row with logits z. With lp the log
probability of the row's token, r = exp(lp - old), A its advantage and ref its log
probability under a reference policy,

    loss = mean over unmasked rows of  -min(r A, clip(r, 1 - lo, 1 + hi) A)
                                       + kl (exp(ref - lp) - (ref - lp) - 1)  -  ent H(z)

Advantages. A_t = r_t + g V'_t - V_t + g l A_{t+1}; V' is the next step's value, dropped
at a terminated step; A_{t+1} is dropped at a terminated or truncated one.

AdamW with the gradients clipped to a global norm; the moments in 32 bits, or in 8 bits
in blocks of 256 that share one exponent E (that of the block's largest magnitude):
with q(x) = (float bits of |x| + 16 random bits << 4) >> 20, i.e. the exponent and three
bits of mantissa rounded at random,

    first moment   code = sign << 7 | f,  f = q - (8 E - 112), zero below f = 8
    second moment  code = q - (8 E - 247), at least 1 where the value is not zero

The random bits are a hash of (seed, step, tensor, element): ``_mix`` below.
"""

import math
import random

import numpy as np
import torch

own = False

DEV = "cuda:0"
BLOCK = 256
LO, HI = 0.2, 0.2
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


# ------------------------------------------------------------------------------ cases
def listed():
    return [
        # one minibatch of the 8-agent navigation fleet (1024 envs, one step of a few envs):
        # 25 = a 5 x 5 grid of velocities; launch latency is what counts
        dict(name="loss 512x25 f32", op="loss", form="autograd", rows=512, vocab=25,
             dtype="f32", masked=0.0, barred=0.2, kl=0.05, ent=0.01, scale=1.0),
        # one step of the 16,000 x 16 fleet, two action slots of 21 bins per agent
        dict(name="loss 512000x21 f32", op="loss", form="direct", rows=512000, vocab=21,
             dtype="f32", masked=0.1, barred=0.0, kl=0.05, ent=0.01, scale=1.0),
        # odd rows and vocabulary: few rows start on a 16-byte boundary. f16 gradients are
        # those of a scaled loss
        dict(name="loss 16383x4099 f16", op="loss", form="direct", rows=16383, vocab=4099,
             dtype="f16", masked=0.1, barred=0.1, kl=0.0, ent=0.01, scale=4096.0),
        # a sequence policy's minibatch, through autograd
        dict(name="loss 4096x32768 bf16", op="loss", form="autograd", rows=4096, vocab=32768,
             dtype="bf16", masked=0.05, barred=0.0, kl=0.05, ent=0.0, scale=1.0),
        # the largest: 2.1 GB of logits, and as much of gradient
        dict(name="loss 8192x131072 bf16", op="loss", form="direct", rows=8192, vocab=131072,
             dtype="bf16", masked=0.0, barred=0.0, kl=0.05, ent=0.001, scale=1.0),
        # the log probabilities of the tokens just chosen: one decode step of 48 sequences
        dict(name="logp 48x100003 bf16", op="loss", form="logp", rows=48, vocab=100003,
             dtype="bf16", masked=0.0, barred=0.0, kl=0.0, ent=0.0, scale=1.0),
        # a small policy network: six tensors
        dict(name="adamw 6 tensors 32-bit f32", op="adamw", tensors=6, elements=41_000,
             dtype="f32", bits=32, clip=0.1),
        # a transformer policy with float32 masters of bf16 parameters
        dict(name="adamw 148 tensors 32-bit bf16", op="adamw", tensors=148,
             elements=150_000_000, dtype="bf16", bits=32, clip=1.0),
        # 8-bit moments, f32 parameters; the clip is one that an ordinary step stays under
        dict(name="adamw 37 tensors 8-bit f32", op="adamw", tensors=37, elements=40_000_001,
             dtype="f32", bits=8, clip=100.0),
        # 8-bit moments, bf16 parameters with masters: the largest update
        dict(name="adamw 90 tensors 8-bit bf16", op="adamw", tensors=90, elements=250_000_003,
             dtype="bf16", bits=8, clip=0.0),
        # the 16,000 x 16 fleet over its horizon of 64; episodes end per env
        dict(name="gae 64x16000x16", op="gae", steps=64, envs=16000, agents=16,
             ends=0.02, own_next=False),
        # six long streams: hardly any columns, a very long recurrence
        dict(name="gae 32768x6x1", op="gae", steps=32768, envs=6, agents=1, ends=0.001,
             own_next=True),
    ]


def _log_uniform(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5))))))


def draw(rng):
    kind = rng.choice(["loss", "loss", "logp", "adamw", "adamw", "gae", "gae"])
    if kind in ("loss", "logp"):
        vocab = _log_uniform(rng, 2, 131072)
        rows = _log_uniform(rng, 1, min(512000, (1 << 28) // vocab))
        train = kind == "loss"
        dtype = rng.choice(["f32", "bf16", "f16"])
        return dict(op="loss", form=rng.choice(["autograd", "direct"]) if train else "logp",
                    rows=rows, vocab=vocab, dtype=dtype,
                    scale=4096.0 if train and dtype == "f16" else 1.0,
                    masked=rng.choice([0.0, 0.2]) if train and rows > 16 else 0.0,
                    barred=rng.choice([0.0, 0.2]) if vocab > 8 else 0.0,
                    kl=rng.choice([0.0, 0.05]) if train else 0.0,
                    ent=rng.choice([0.0, 0.01]) if train else 0.0)
    if kind == "adamw":
        tensors = _log_uniform(rng, 1, 160)
        bits = rng.choice([32, 8])
        return dict(op="adamw", tensors=tensors,
                    elements=_log_uniform(rng, max(1000, 40 * tensors), 100_000_000),
                    dtype=rng.choice(["f32", "bf16", "f16"]), bits=bits,
                    clip=rng.choice([0.0, 0.1 if bits == 32 else 100.0]))
    steps = _log_uniform(rng, 1, 32768)
    columns = _log_uniform(rng, 1, min(256_000, (1 << 24) // steps))
    agents = rng.choice([1, min(columns, 4), min(columns, 16)])
    return dict(op="gae", steps=steps, envs=max(1, columns // agents), agents=agents,
                ends=rng.choice([0.0, 0.02, 0.2]), own_next=rng.random() < 0.5)


def _sizes(case):
    """Sizes of the parameter tensors: a third of them vectors, the rest matrices of spread
    sizes, none a round number; they add up to about ``elements``."""
    k, total = case["tensors"], case["elements"]
    rng = random.Random(31 * k + total)
    share = [0.0005 if i % 3 == 2 else math.exp(rng.uniform(-1.5, 1.0)) for i in range(k)]
    s = sum(share)
    return [max(1, int(total * x / s) + rng.choice([0, 1, 3])) for x in share]


def _offsets(sizes):
    at, offs = 0, []
    for n in sizes:
        offs.append(at)
        at += -(-n // BLOCK) * BLOCK
    return offs, at


def work(case):
    if case["op"] == "loss":
        cells, rows = case["rows"] * case["vocab"], case["rows"]
        wide = 4 if case["dtype"] == "f32" else 2
        if case["form"] == "logp":
            return {"bytes": cells * wide + rows * 16, "flops": 4 * cells}
        live = 1.0 - case["masked"]  # a masked row's logits need not be read
        return {"bytes": cells * wide * (1 + live) + rows * (8 + 4 * 4 + 2 * 4), "flops": 10 * cells}
    if case["op"] == "adamw":
        n = sum(_sizes(case))
        p = 8 + 4 if case["dtype"] == "f32" else 8 + 2 + 2  # parameter or master, gradient, copy
        # the 8-bit moments also come back as the bf16 values that they stand for
        s = 16 if case["bits"] == 32 else 4 + 4 + 4 / BLOCK
        return {"bytes": n * (p + s), "flops": 16 * n}
    n = case["steps"] * case["envs"] * case["agents"]
    flags = 2 * case["steps"] * case["envs"]
    return {"bytes": n * (20 if case["own_next"] else 16) + flags, "flops": 7 * n}


# ----------------------------------------------------------------------------- inputs
def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return {"loss": _prepare_loss, "adamw": _prepare_adamw, "gae": _prepare_gae}[case["op"]](case, g)


def _randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device=DEV, dtype=dtype)


def _rand(g, *shape):
    return torch.rand(*shape, generator=g, device=DEV)


def _row_chunks(rows, vocab, cells=1 << 27):
    step = max(1, cells // vocab)
    return [slice(i, min(rows, i + step)) for i in range(0, rows, step)]


def _prepare_loss(case, g):
    N, V, dtype = case["rows"], case["vocab"], DTYPES[case["dtype"]]
    logits = _randn(g, N, V, dtype=dtype)
    logits.mul_(2.0)
    tokens = (_rand(g, N) * V).long().clamp_(max=V - 1)
    rows = torch.arange(N, device=DEV)
    if case["barred"]:  # actions that the state does not allow: -inf, never the chosen one
        for s in _row_chunks(N, V):
            part = logits[s]
            part.masked_fill_(torch.rand(part.shape, generator=g, device=DEV) < case["barred"],
                              -math.inf)
        logits[rows, tokens] = _randn(g, N).to(dtype)
    # the chosen token is a likely one, as sampling makes it
    logits[rows, tokens] += (1.0 + 0.7 * math.log(V) * _rand(g, N)).to(dtype)
    lp = torch.empty(N, device=DEV)
    for s in _row_chunks(N, V):
        z = logits[s].float()
        lp[s] = z.gather(1, tokens[s, None]).squeeze(1) - z.logsumexp(1)
    # the policy has moved a little since the rollout. A ratio within 0.002 of a clip bound
    # is moved off it: there rounding alone would decide whether the row has a gradient.
    moved = 0.15 * _randn(g, N)
    for bound in (math.log(1 - LO), math.log(1 + HI)):
        moved = torch.where((moved - bound).abs() < 0.002, moved + 0.005, moved)
    st = dict(case=case, logits=logits, tokens=tokens, old_logp=lp - moved,
              advantages=0.25 + _randn(g, N), ref_logp=None, mask=None)
    if case["kl"]:
        st["ref_logp"] = lp + 0.3 * _randn(g, N)
    if case["masked"]:  # padding: zeros, as a batch is padded
        st["mask"] = _rand(g, N) >= case["masked"]
        for k in ("tokens", "old_logp", "advantages", "ref_logp"):
            if st[k] is not None:
                st[k] = torch.where(st["mask"], st[k], torch.zeros_like(st[k]))
    if case["form"] == "autograd":
        logits.requires_grad_(True)
        st["cotangent"] = torch.full((), case["scale"], device=DEV)  # of the scaled loss
    return st


def _prepare_adamw(case, g):
    sizes = _sizes(case)
    offs, total = _offsets(sizes)
    dtype = DTYPES[case["dtype"]]
    live = torch.zeros(total, device=DEV, dtype=torch.bool)
    for o, n in zip(offs, sizes):
        live[o:o + n] = True
    master = (0.02 * _randn(g, total)).mul_(live)
    grad = (1e-3 * _randn(g, total)).mul_(live).to(dtype)
    flat = {"grad": grad, "param": master if dtype == torch.float32 else master.to(dtype)}
    if dtype != torch.float32:
        flat["master"] = master
    if case["bits"] == 32:
        flat["m"] = (4e-4 * _randn(g, total)).mul_(live)
        flat["v"] = (1e-6 * (0.05 + _rand(g, total))).mul_(live)
    else:  # codes and exponents of moments of the same sizes
        flat["m"] = (torch.randint(64, 120, (total,), generator=g, device=DEV, dtype=torch.uint8)
                     + 128 * torch.randint(0, 2, (total,), generator=g, device=DEV,
                                           dtype=torch.uint8)).mul_(live)
        flat["v"] = torch.randint(200, 253, (total,), generator=g, device=DEV,
                                  dtype=torch.uint8).mul_(live)
        flat["m_exp"] = torch.full((total // BLOCK,), 117, device=DEV, dtype=torch.uint8)
        flat["v_exp"] = torch.full((total // BLOCK,), 107, device=DEV, dtype=torch.uint8)
    del live
    cut = {k: [t[o // BLOCK:o // BLOCK + -(-n // BLOCK)] if k.endswith("_exp") else t[o:o + n]
               for o, n in zip(offs, sizes)] for k, t in flat.items()}
    return dict(case=case, flat=flat, cut=cut, sizes=sizes, offs=offs, step=1000)


def _prepare_gae(case, g):
    T, E, A = case["steps"], case["envs"], case["agents"]
    value = 2.0 + _randn(g, T, E, A)
    ends = _rand(g, T, E)
    return dict(case=case, rewards=0.1 * _randn(g, T, E, A), values=value,
                last_values=2.0 + _randn(g, E, A),
                next_values=value + 0.2 * _randn(g, T, E, A) if case["own_next"] else None,
                terminated=ends < 0.5 * case["ends"],
                truncated=(ends >= 0.5 * case["ends"]) & (ends < case["ends"]))


GAMMA, LAM = 0.99, 0.95
ADAM = dict(lr=1e-4, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01)
SEED = 12345


# -------------------------------------------------------------------------------- run
def run(state):
    op = state["case"]["op"]
    if op == "loss":
        return _own_loss(state) if own else _plain_loss(state)
    if op == "adamw":
        state["step"] += 1
        return _own_adamw(state) if own else _plain_adamw(state)
    return _own_gae(state) if own else _plain_gae(state)


def _own_loss(st):
    import swarp_b200 as swarp

    case = st["case"]
    if case["form"] == "logp":
        logp, entropy = swarp.token_logp(st["logits"], st["tokens"])
        return {"logp": logp, "entropy": entropy}
    args = (st["logits"], st["tokens"], st["old_logp"], st["advantages"])
    more = dict(ref_logp=st["ref_logp"], mask=st["mask"], clip_low=LO, clip_high=HI,
                kl_coef=case["kl"], entropy_coef=case["ent"])
    if case["form"] == "autograd":
        out = swarp.policy_loss(*args, **more)
        (grad,) = torch.autograd.grad(out.loss, st["logits"], st["cotangent"])
    else:
        out, grad = swarp.policy_loss_and_grad(*args, grad_scale=case["scale"], **more)
    return {"loss": out.loss, "logp": out.logp, "entropy": out.entropy, "stats": out.stats,
            "grad": grad}


def _plain_loss(st):
    case, a = st["case"], st["tokens"][:, None]
    logits = st["logits"].detach()
    z = logits.float()
    z = z - z.amax(1, keepdim=True)
    e = z.exp()
    total = e.sum(1, keepdim=True)
    ln = total.log()
    held = torch.where(e > 0, z, torch.zeros_like(z))  # a barred token adds nothing to H
    H = ln - (e * held).sum(1, keepdim=True) / total
    lp = z.gather(1, a) - ln
    if case["form"] == "logp":
        return {"logp": lp.squeeze(1), "entropy": H.squeeze(1)}
    live = torch.ones_like(a, dtype=torch.bool) if st["mask"] is None else st["mask"][:, None]
    count = live.sum().float()
    zero = torch.zeros_like(lp)
    A = st["advantages"][:, None]
    r = (lp - st["old_logp"][:, None]).exp()
    pg = -torch.minimum(r * A, r.clamp(1 - LO, 1 + HI) * A)
    cut = ((A > 0) & (r > 1 + HI)) | ((A < 0) & (r < 1 - LO))
    c = torch.where(cut, zero, -r * A)
    k3 = zero
    if st["ref_logp"] is not None:
        d = st["ref_logp"][:, None] - lp
        k3 = d.exp() - d - 1
        c = c + case["kl"] * (1 - d.exp())
    mean = lambda x: torch.where(live, x, zero).sum() / count  # noqa: E731
    stats = torch.stack([mean(pg), mean(k3), mean(H), mean(cut.float())])
    loss = stats[0] + case["kl"] * stats[1] - case["ent"] * stats[2]
    p = e / total
    c = torch.where(live, c / count, zero)
    grad = -c * p
    if case["ent"]:
        grad += torch.where(live, case["ent"] / count, zero) * (p * (held - ln + H))
    grad.scatter_add_(1, a, c)
    if case["scale"] != 1.0:
        grad *= case["scale"]
    return {"loss": loss, "logp": torch.where(live, lp, zero).squeeze(1),
            "entropy": torch.where(live, H, zero).squeeze(1), "stats": stats,
            "grad": grad.to(logits.dtype)}


def _own_adamw(st):
    import swarp_b200 as swarp

    case, cut, flat = st["case"], st["cut"], st["flat"]
    m, v = cut["m"], cut["v"]
    if case["bits"] == 8:
        m = [swarp.Moment8(c, e, True) for c, e in zip(m, cut["m_exp"])]
        v = [swarp.Moment8(c, e, False) for c, e in zip(v, cut["v_exp"])]
    norm = swarp.adamw_step(cut["param"], cut["grad"], m, v, step=st["step"], seed=SEED,
                            max_norm=case["clip"] or None, masters=cut.get("master"), **ADAM)
    out = {k: flat[k] for k in ("param", "master") if k in flat}
    if case["bits"] == 8:
        out["m"] = swarp.Moment8(flat["m"], flat["m_exp"], True).values()
        out["v"] = swarp.Moment8(flat["v"], flat["v_exp"], False).values()
    else:
        out["m"], out["v"] = flat["m"], flat["v"]
    if norm is not None:
        out["norm"] = norm
    return out


def _mix(x):
    """A 32-bit hash, of integers or int64 tensors (whose products wrap, low bits intact)."""
    x = x ^ (x >> 16)
    x = (x * 0xE80B5AE5) & 0xFFFFFFFF
    x = x ^ (x >> 15)
    x = (x * 0xCB276749) & 0xFFFFFFFF
    return x ^ (x >> 16)


def _key(step, tensor):
    return _mix((_mix((SEED + step) & 0xFFFFFFFF) + tensor) & 0xFFFFFFFF)


def _decode8(code, exp, signed):
    exp = exp.int().repeat_interleave(BLOCK) * 8
    code = code.int()
    f = code & 127 if signed else code
    x = ((f + exp - (112 if signed else 247)) << 20).view(torch.float32)
    x = torch.where(f > 0, x, torch.zeros_like(x))
    return torch.where(code > 127, -x, x) if signed else x


def _encode8(x, r16, signed):
    bits = x.abs().view(torch.int32)
    exp = bits.view(-1, BLOCK).amax(1) >> 23
    q = ((bits + (r16 << 4)) >> 20).clamp_(max=2047)
    f = q - (exp * 8 - (112 if signed else 247)).repeat_interleave(BLOCK)
    if signed:
        f = torch.where(f < 8, torch.zeros_like(f), f) + torch.where(x < 0, 128, 0)
        f = torch.where((f & 127) == 0, torch.zeros_like(f), f)
    else:
        f = torch.maximum(f, (bits > 0).int())
    return f.to(torch.uint8), exp.to(torch.uint8)


def _plain_adamw(st):
    case, flat, t = st["case"], st["flat"], st["step"]
    lr, (b1, b2), eps, wd = ADAM["lr"], ADAM["betas"], ADAM["eps"], ADAM["weight_decay"]
    g = flat["grad"].float()
    out = {}
    if case["clip"]:
        norm = g.square().sum().sqrt()
        out["norm"] = norm
        g = g * (case["clip"] / (norm + 1e-6)).clamp(max=1.0)
    eight = case["bits"] == 8
    m = _decode8(flat["m"], flat["m_exp"], True) if eight else flat["m"]
    v = _decode8(flat["v"], flat["v_exp"], False) if eight else flat["v"]
    m = m * b1 + g * (1 - b1)
    v = v * b2 + (g * (1 - b2)) * g
    p = flat.get("master", flat["param"])
    p.copy_(p * (1 - lr * wd) - (lr / (1 - b1 ** t)) * (m / (v.sqrt() / math.sqrt(1 - b2 ** t) + eps)))
    out["param"] = flat["param"]
    if "master" in flat:
        out["master"] = p
        flat["param"].copy_(p)
    if not eight:
        flat["m"].copy_(m)
        flat["v"].copy_(v)
        out["m"], out["v"] = flat["m"], flat["v"]
        return out
    padded = torch.tensor([-(-n // BLOCK) * BLOCK for n in st["sizes"]], device=DEV)
    starts = torch.tensor(st["offs"], device=DEV)
    keys = torch.tensor([_key(t, i) for i in range(len(st["sizes"]))], device=DEV)
    element = torch.arange(g.numel(), device=DEV) - starts.repeat_interleave(padded)
    h = _mix(element ^ keys.repeat_interleave(padded)).int()
    for name, x, signed, r in (("m", m, True, h & 0xFFFF), ("v", v, False, (h >> 16) & 0xFFFF)):
        code, exp = _encode8(x, r, signed)
        flat[name].copy_(code)
        flat[name + "_exp"].copy_(exp)
        out[name] = _decode8(code, exp, signed).to(torch.bfloat16)
    return out


def _own_gae(st):
    import swarp_b200 as swarp

    advantages, returns = swarp.gae(st["rewards"], st["values"], st["last_values"],
                                    st["terminated"], st["truncated"], gamma=GAMMA, lam=LAM,
                                    next_values=st["next_values"])
    return {"advantages": advantages, "returns": returns}


def _plain_gae(st):
    V, nxt = st["values"], st["next_values"]
    if nxt is None:
        nxt = torch.cat([V[1:], st["last_values"][None]])
    term = st["terminated"][:, :, None]
    done = term | st["truncated"][:, :, None]
    A = st["rewards"] + GAMMA * torch.where(term, torch.zeros_like(nxt), nxt) - V
    c = torch.where(done, 0.0, GAMMA * LAM).expand_as(A)
    k = 1
    while k < A.shape[0]:  # after each turn A_t covers 2k steps and c_t is their product
        A = torch.cat([A[:-k] + c[:-k] * A[k:], A[-k:]])
        c = torch.cat([c[:-k] * c[k:], c[-k:]])
        k *= 2
    return {"advantages": A, "returns": A + V}


# ------------------------------------------------------------------------------ exact
def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "loss":
        return _exact_loss(st)
    return _exact_adamw(st) if case["op"] == "adamw" else _exact_gae(st)


def _exact_loss(st):
    """In 64 bits, the gradient by differentiation of the loss."""
    case, N, V = st["case"], *st["logits"].shape
    train = case["form"] != "logp"
    live = torch.ones(N, dtype=torch.bool, device=DEV) if st["mask"] is None else st["mask"]
    count = int(live.sum())
    logp, ent = (torch.zeros(N, dtype=torch.float64, device=DEV) for _ in range(2))
    grad = torch.zeros(N, V, dtype=torch.float64, device=DEV) if train else None
    sums = torch.zeros(4, dtype=torch.float64, device=DEV)
    for s in _row_chunks(N, V, 1 << 26):
        i = torch.arange(s.start, s.stop, device=DEV)[live[s]]
        if i.numel() == 0:
            continue
        z = st["logits"].detach()[i].double().requires_grad_(train)
        logs = torch.log_softmax(z, dim=1)
        lp = logs.gather(1, st["tokens"][i, None]).squeeze(1)
        H = -torch.where(z > -math.inf, logs.exp() * logs.clamp(min=-1e300), 0.0).sum(1)
        logp[i], ent[i] = lp.detach(), H.detach()
        if not train:
            continue
        A = st["advantages"][i].double()
        r = torch.exp(lp - st["old_logp"][i].double())
        pg = -torch.min(r * A, torch.clamp(r, 1 - LO, 1 + HI) * A)
        kl = torch.zeros_like(pg)
        if st["ref_logp"] is not None:
            d = st["ref_logp"][i].double() - lp
            kl = torch.expm1(d) - d
        (pg + case["kl"] * kl - case["ent"] * H).sum().mul(case["scale"] / count).backward()
        grad[i] = z.grad.nan_to_num(0.0)  # a barred token: 0 times minus infinity
        clipped = torch.where(A > 0, r > 1 + HI, r < 1 - LO) & (A != 0)
        sums += torch.stack([pg.sum(), kl.sum(), H.sum(), clipped.double().sum()]).detach() / count
    if not train:
        return {"logp": logp, "entropy": ent}
    return {"loss": sums[0] + case["kl"] * sums[1] - case["ent"] * sums[2], "logp": logp,
            "entropy": ent, "stats": sums, "grad": grad}


def _exact_adamw(st):
    """Tensor by tensor in 64 bits; a code is the value's place among the format's steps."""
    case, t = st["case"], st["step"] + 1
    lr, (b1, b2), eps, wd = ADAM["lr"], ADAM["betas"], ADAM["eps"], ADAM["weight_decay"]
    flat, cut = st["flat"], st["cut"]
    out = {k: torch.zeros(flat["grad"].numel(), dtype=torch.float64, device=DEV)
           for k in ("param", "master", "m", "v") if k in flat}
    norm = math.sqrt(sum(float(x.double().square().sum()) for x in cut["grad"]))
    scale = min(1.0, case["clip"] / (norm + 1e-6)) if case["clip"] else 1.0
    for i, (o, n) in enumerate(zip(st["offs"], st["sizes"])):
        g = cut["grad"][i].double() * scale
        m, v = cut["m"][i], cut["v"][i]
        if case["bits"] == 8:
            m = _value64(m, cut["m_exp"][i], n, True)
            v = _value64(v, cut["v_exp"][i], n, False)
        m = b1 * m.double() + (1 - b1) * g
        v = b2 * v.double() + (1 - b2) * g * g
        p = cut["master" if "master" in cut else "param"][i].double()
        p = (1 - lr * wd) * p - lr * (m / (1 - b1 ** t)) / ((v / (1 - b2 ** t)).sqrt() + eps)
        out["param"][o:o + n] = p
        if "master" in out:
            out["master"][o:o + n] = p
        if case["bits"] == 8:
            h = _mix(torch.arange(n, device=DEV) ^ _key(t, i))
            m, v = _round64(m, h & 0xFFFF, True), _round64(v, h >> 16, False)
        out["m"][o:o + n], out["v"][o:o + n] = m, v
    if case["clip"]:
        out["norm"] = torch.tensor(norm, dtype=torch.float64, device=DEV)
    return out


def _value64(code, exp, n, signed):
    code = code.double()
    f = code % 128 if signed else code
    base = exp.double().repeat_interleave(BLOCK)[:n] - (14 if signed else 31)
    f8 = f + (0 if signed else 1)  # 247 = 8 x 31 - 1
    x = 2.0 ** (base + torch.floor(f8 / 8) - 127) * (1 + (f8 % 8) / 8)
    x = torch.where(f > 0, x, 0.0)
    return torch.where(code >= 128, -x, x) if signed else x


def _round64(x, r16, signed):
    a, n = x.abs(), x.numel()
    pad = torch.zeros(-n % BLOCK, dtype=torch.float64, device=DEV)
    top = torch.cat([a, pad]).view(-1, BLOCK).amax(1).clamp(min=2.0 ** -126).log2().floor()
    top = top.repeat_interleave(BLOCK)[:n]
    e = a.clamp(min=2.0 ** -126).log2().floor()
    step = 2.0 ** (e - 3)  # three bits of mantissa
    y = torch.floor(a / step + r16.double() / 65536) * step
    low = 2.0 ** (top - (13 if signed else 31)) * (1.0 if signed else 1.25)
    if signed:
        return torch.where(y < low, 0.0, y) * torch.sign(x)
    return torch.where(a > 0, torch.maximum(y, low), 0.0)


def _exact_gae(st):
    to = lambda x: x.cpu().numpy().astype(np.float64)  # noqa: E731
    r, V = to(st["rewards"]), to(st["values"])
    ahead, last = np.zeros_like(r[0]), to(st["last_values"])
    nxt = None if st["next_values"] is None else to(st["next_values"])
    term = st["terminated"].cpu().numpy()[:, :, None]
    stop = term | st["truncated"].cpu().numpy()[:, :, None]
    A = np.empty_like(r)
    for t in reversed(range(r.shape[0])):
        follow = nxt[t] if nxt is not None else last
        ahead = (r[t] + GAMMA * np.where(term[t], 0.0, follow) - V[t]
                 + GAMMA * LAM * np.where(stop[t], 0.0, ahead))
        A[t], last = ahead, V[t]
    return {"advantages": torch.from_numpy(A), "returns": torch.from_numpy(A + V)}
