"""AdamW over many tensors in one launch, with moments in 32 or 8 bits.

    m = b1 m + (1 - b1) g        v = b2 v + (1 - b2) g^2
    p = p (1 - lr wd) - lr / (1 - b1^t) m / (sqrt(v / (1 - b2^t)) + eps)

with the gradients first scaled to a global norm of at most ``max_norm``, if one is given.
Parameters are float32, or bfloat16 / float16 with a float32 master copy. An 8-bit moment is
a :class:`Moment8`: minifloat codes in blocks of 256 that share an exponent, rounded up or
down at random so that the averages stay unbiased (to the nearest, an average that moves by
0.1% a step would never leave a code 12.5% wide). A step of float32 parameters then moves 16
bytes per element instead of 28.

The tensors' addresses travel in the launch's parameters: a step uploads nothing, never
waits for the device, and can be captured in a CUDA graph. The step number travels there too,
so a graph that is replayed repeats the one that it was captured with: its bias corrections,
which a graph captured late in training hardly notices, and with 8-bit moments the random
bits. Each element would then always round against the same threshold, which is no longer
unbiased: do not replay a captured 8-bit step in place of further steps.
"""

from __future__ import annotations

import ctypes as C
from array import array
from collections.abc import Sequence
from operator import attrgetter
from typing import Any, NamedTuple

import torch

from swarp_b200 import _lib
from swarp_b200.learn._call import DTYPES, library, on_device, require_cuda, stream

_PARAM_DTYPES = (torch.float32, torch.bfloat16, torch.float16)
BLOCK = 256  # SWARP_MOMENT_BLOCK


class Moment8(NamedTuple):
    """An 8-bit moment of a tensor of n elements: ``codes`` uint8 ``[n]``, ``exponents`` uint8
    ``[ceil(n / 256)]`` (the float32 exponent field of each block's largest magnitude),
    ``signed`` for the first moment, not for the second.

    A code's value has an exponent and three bits of mantissa. Signed: a sign bit and seven
    bits ``f``, worth ``(f + 8 E - 112) << 20`` as float32 bits, 16 octaves. Unsigned: eight
    bits, ``(f + 8 E - 247) << 20``, 32 octaves. ``f = 0`` is 0, and a signed ``f`` of 1 to 7 does
    not occur. A NaN or infinite gradient
    makes its block's exponent 255, and the block's other elements lose their moments."""

    codes: torch.Tensor
    exponents: torch.Tensor
    signed: bool

    @classmethod
    def zeros(cls, n: int, device, signed: bool) -> "Moment8":
        return cls(torch.zeros(n, dtype=torch.uint8, device=device),
                   torch.zeros(-(-n // BLOCK), dtype=torch.uint8, device=device), signed)

    def values(self, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
        """The values that the codes stand for, in bfloat16 or float32 (both exact)."""
        if dtype not in (torch.bfloat16, torch.float32):
            raise TypeError(f"dtype {dtype}: want bfloat16 or float32")
        require_cuda(self.codes, "codes")
        n, device = self.codes.numel(), self.codes.device
        _check_moment8(self, "moment", n, device)
        out = torch.empty(n, dtype=dtype, device=device)
        lib = library()
        with on_device(device):
            _lib.check(lib.swarp_moment8_values(
                self.codes.data_ptr(), self.exponents.data_ptr(), n, self.signed, DTYPES[dtype],
                out.data_ptr(), stream(device)), "swarp_moment8_values")
        return out


def _check_moment8(m: Moment8, name: str, n: int, device) -> None:
    for t, what, size in ((m.codes, "codes", n), (m.exponents, "exponents", -(-n // BLOCK))):
        if t.dtype != torch.uint8 or t.numel() != size or t.device != device \
                or not t.is_contiguous():
            raise ValueError(f"{name}: {what} must be {size} contiguous uint8 on {device}, got "
                             f"{t.dtype} {tuple(t.shape)} on {t.device}")


# a step may have hundreds of tensors: their properties are read by C loops
_numel, _ptr, _contiguous, _device = (torch.Tensor.numel, torch.Tensor.data_ptr,
                                      torch.Tensor.is_contiguous, torch.Tensor.get_device)
_dtype, _shape = attrgetter("dtype"), attrgetter("shape")


def _same(ts, name, sizes, dtype, device, sized=False):
    """The addresses of ``ts``, once each has its parameter's size and is contiguous.
    ``sized``: the sizes are known to be right."""
    if len(ts) != len(sizes):
        raise ValueError(f"{len(sizes)} params but {len(ts)} {name}")
    if not ((sized or list(map(_numel, ts)) == sizes) and set(map(_dtype, ts)) == {dtype}
            and set(map(_device, ts)) == {device.index} and all(map(_contiguous, ts))):
        for i, (t, n) in enumerate(zip(ts, sizes)):
            if t.dtype != dtype or t.numel() != n or t.device != device or not t.is_contiguous():
                kind = TypeError if t.dtype != dtype else ValueError
                raise kind(f"{name}[{i}] must be {n} contiguous {dtype} elements on {device}, "
                           f"got {t.dtype} {tuple(t.shape)} with strides {t.stride()} on "
                           f"{t.device}")
    return list(map(_ptr, ts))


def _same8(ms, name, sizes, blocks, signed, device):
    """The addresses of the codes and exponents of 8-bit moments."""
    if len(ms) != len(sizes):
        raise ValueError(f"{len(sizes)} params but {len(ms)} {name}")
    for i, x in enumerate(ms):
        if not isinstance(x, Moment8) or x.signed != signed:
            raise TypeError(f"{name}[{i}] must be a Moment8 with signed={signed}")
    codes, exps = [x.codes for x in ms], [x.exponents for x in ms]
    return (_same(codes, name + " codes", sizes, torch.uint8, device),
            _same(exps, name + " exponents", blocks, torch.uint8, device))


def _once(ptrs, sizes) -> None:
    """Refuse a parameter that is there twice: one launch steps them all, and its two updates of
    the same memory would race."""
    seen: dict[int, int] = {}
    for i, (x, n) in enumerate(zip(ptrs, sizes)):
        if n and seen.setdefault(x, i) != i:
            raise ValueError(f"params[{i}] and params[{seen[x]}] are the same memory")


class _Tensors:
    """Checked tensors of one dtype as the C array."""

    def __init__(self, params, grads, exp_avg, exp_avg_sq, masters):
        n = len(params)
        if n == 0:
            raise ValueError("no parameters")
        require_cuda(params[0], "params[0]")
        self.device, self.dtype = params[0].device, params[0].dtype
        if self.dtype not in _PARAM_DTYPES:
            raise TypeError(f"params dtype {self.dtype}: want float32, bfloat16 or float16")
        sizes = list(map(_numel, params))
        p = _same(params, "params", sizes, self.dtype, self.device, sized=True)
        if len(set(p)) < n:
            _once(p, sizes)
        alike = list(map(_shape, params)) == list(map(_shape, grads))
        g = _same(grads, "grads", sizes, self.dtype, self.device, sized=alike)
        if not alike:
            for i, (x, y) in enumerate(zip(params, grads)):
                if x.shape != y.shape:
                    raise ValueError(f"grads[{i}] has shape {tuple(y.shape)}, its parameter "
                                     f"{tuple(x.shape)}")
        if self.dtype == torch.float32:
            if masters is not None:
                raise ValueError("masters are for 16-bit parameters")
            w = None
        elif masters is None:
            raise ValueError(f"{self.dtype} parameters need float32 masters")
        else:
            w = _same(masters, "masters", sizes, torch.float32, self.device)
        self.bits = 8 if len(exp_avg) and isinstance(exp_avg[0], Moment8) else 32
        if self.bits == 32:
            m = _same(exp_avg, "exp_avg", sizes, torch.float32, self.device)
            v = _same(exp_avg_sq, "exp_avg_sq", sizes, torch.float32, self.device)
            me = ve = None
        else:
            blocks = [-(-x // BLOCK) for x in sizes]
            m, me = _same8(exp_avg, "exp_avg", sizes, blocks, True, self.device)
            v, ve = _same8(exp_avg_sq, "exp_avg_sq", sizes, blocks, False, self.device)
        self.params, self.keep = params, grads  # until the launch has read their addresses
        # swarp_adamw_tensor_t[n], in 64-bit words
        self.words = array("Q", bytes(64 * n))
        for k, column in enumerate((sizes, p, g, w, m, v, me, ve)):
            if column is not None:
                self.words[k::8] = array("Q", column)
        self.n, self.c = n, self.words.buffer_info()[0]

    def norm_partials(self, lib, out: torch.Tensor) -> None:
        _lib.check(lib.swarp_grad_norm_partials(DTYPES[self.dtype], self.c, self.n,
                                                out.data_ptr(), stream(self.device)),
                   "swarp_grad_norm_partials")

    def step(self, lib, step, lr, betas, eps, weight_decay, seed, first, partials, max_norm,
             norm) -> None:
        opt = _lib.AdamWOpt(DTYPES[self.dtype], self.bits, step, lr, *betas, eps, weight_decay,
                            seed & 0xFFFFFFFF, first, _lib.ptr(partials),
                            0 if partials is None else partials.numel(), max_norm or 0.0,
                            _lib.ptr(norm))
        _lib.check(lib.swarp_adamw_step(C.byref(opt), self.c, self.n,
                                        stream(self.device)), "swarp_adamw_step")
        # autograd must see that the parameters changed, as after torch's own in-place steps
        torch.autograd.graph.increment_version(self.params)


def _check_betas(betas) -> None:
    if not (0.0 <= betas[0] < 1.0 and 0.0 <= betas[1] < 1.0):
        raise ValueError(f"betas must be in [0, 1), got {betas}")


def _check_settings(step, lr, betas, eps, weight_decay, max_norm) -> None:
    if step < 1:
        raise ValueError(f"step counts from 1, got {step}")
    if not lr >= 0.0 or not eps >= 0.0 or not weight_decay >= 0.0:
        raise ValueError(f"lr, eps and weight_decay must be >= 0, got {lr}, {eps}, {weight_decay}")
    _check_betas(betas)
    if max_norm is not None and not max_norm > 0.0:
        raise ValueError(f"max_norm must be > 0 (None: no clipping), got {max_norm}")


def adamw_step(
    params: Sequence[torch.Tensor],
    grads: Sequence[torch.Tensor],
    exp_avg: Sequence[torch.Tensor | Moment8],
    exp_avg_sq: Sequence[torch.Tensor | Moment8],
    *,
    step: int,
    lr: float,
    betas: tuple[float, float] = (0.9, 0.999),
    eps: float = 1e-8,
    weight_decay: float = 0.01,
    max_norm: float | None = None,
    masters: Sequence[torch.Tensor] | None = None,
    seed: int = 0,
) -> torch.Tensor | None:
    """One step in place over ``params`` (contiguous, of one dtype and device, none twice) with ``grads`` of
    the same shapes and dtype. ``exp_avg`` and ``exp_avg_sq`` are float32 tensors or
    :class:`Moment8`; 16-bit parameters need float32 ``masters``, which take the step and
    are rounded into the parameters. ``step`` counts from 1. ``eps`` below 1e-19 counts as that.
    ``seed`` is that of the random
    rounding of 8-bit moments; ``(seed, step)`` repeated gives the same bits.

    With ``max_norm`` the gradients are scaled by ``min(1, max_norm / (norm + 1e-6))`` and
    their norm before that is returned (a float32 scalar on the device)."""
    _check_settings(step, lr, betas, eps, weight_decay, max_norm)
    ts = _Tensors(params, grads, exp_avg, exp_avg_sq, masters)
    lib = library()
    partials = norm = None
    with on_device(ts.device):
        if max_norm is not None:
            partials = torch.empty(lib.swarp_grad_norm_partials_count(ts.n),
                                   dtype=torch.float64, device=ts.device)
            norm = torch.empty((), dtype=torch.float32, device=ts.device)
            ts.norm_partials(lib, partials)
        ts.step(lib, step, lr, betas, eps, weight_decay, seed, 0, partials, max_norm, norm)
    return norm


class AdamW(torch.optim.Optimizer):
    """:func:`adamw_step` as a torch optimizer (parameter groups, schedulers, ``state_dict``).

    ``state_bits`` 32 or 8; 16-bit parameters get a float32 master. ``max_norm`` clips the
    norm of all groups' gradients together; :attr:`grad_norm` is then that norm of the last
    step (a device scalar). Parameters without a gradient are left out of a step.

    A master is made at the parameter's first step and is what later steps update: after a
    16-bit parameter has been changed from outside (weights loaded into the model, say),
    set ``state[p]["master"]`` too."""

    def __init__(self, params, lr: float = 1e-3, betas: tuple[float, float] = (0.9, 0.999),
                 eps: float = 1e-8, weight_decay: float = 0.01, *, max_norm: float | None = None,
                 state_bits: int = 32, seed: int = 0) -> None:
        if state_bits not in (32, 8):
            raise ValueError(f"state_bits must be 32 or 8, got {state_bits}")
        _check_settings(1, lr, betas, eps, weight_decay, max_norm)
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay))
        self.max_norm, self.state_bits, self.seed = max_norm, state_bits, seed
        self.grad_norm: torch.Tensor | None = None

    def _init_state(self, p: torch.Tensor) -> dict[str, Any]:
        st = self.state[p]
        n = p.numel()
        st["step"] = 0
        for name, signed in (("exp_avg", True), ("exp_avg_sq", False)):
            if self.state_bits == 8:
                st[name], st[name + "_exp"] = Moment8.zeros(n, p.device, signed)[:2]
            else:
                st[name] = torch.zeros(n, dtype=torch.float32, device=p.device)
        if p.dtype != torch.float32:
            st["master"] = p.detach().float().contiguous()
        return st

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        fresh: list[torch.Tensor] = []
        try:
            made, states, device = self._launches(fresh)
        except Exception:
            for p in fresh:  # a refused step leaves no trace
                del self.state[p]
            raise
        if not made:
            return loss
        lib = library()
        for st in states:
            st["step"] += 1
        partials = norm = None
        with on_device(device):
            if self.max_norm is not None:
                counts = [lib.swarp_grad_norm_partials_count(ts.n) for *_, ts in made]
                partials = torch.empty(sum(counts), dtype=torch.float64, device=device)
                norm = torch.empty((), dtype=torch.float32, device=device)
                for (*_, ts), part in zip(made, partials.split(counts)):
                    ts.norm_partials(lib, part)
            for gi, step, first, ts in made:
                g = self.param_groups[gi]
                ts.step(lib, step, g["lr"], g["betas"], g["eps"], g["weight_decay"], self.seed,
                        first, partials, self.max_norm, norm)
        self.grad_norm = norm
        return loss

    def _launches(self, fresh):
        """The launches of a step as ``(group, step, index of the first tensor, tensors)``, all
        checked, the states that it steps, and its device. Parameters whose state was made
        go to ``fresh``."""
        # (group, dtype, device, step) -> its parameters; the index numbers all of them
        sets: dict[tuple, list] = {}
        index, device = 0, None
        for gi, group in enumerate(self.param_groups):
            _check_betas(group["betas"])
            for p in group["params"]:
                g = p.grad
                if g is not None:
                    if g.is_sparse:
                        raise RuntimeError("AdamW takes dense gradients")
                    dev = p.device
                    if device is not None and dev != device:
                        raise ValueError("AdamW steps the parameters of one device")
                    device = dev
                    st = self.state.get(p)
                    if not st:
                        fresh.append(p)
                        st = self._init_state(p)
                    sets.setdefault((gi, p.dtype, dev, st["step"] + 1), []).append(
                        (index, p, g, st))
                index += 1
        made = []
        for (gi, dtype, _, step), members in sets.items():
            # a run of consecutive indices shares a launch: the 8-bit rounding counts tensors
            runs: list[list] = []
            for m in members:
                if runs and (self.state_bits == 32 or m[0] == runs[-1][-1][0] + 1):
                    runs[-1].append(m)
                else:
                    runs.append([m])
            for run in runs:
                made.append((gi, step, run[0][0], self._tensors(run, dtype)))
        return made, [m[3] for members in sets.values() for m in members], device

    def _tensors(self, run, dtype) -> _Tensors:
        params, grads, m, v, w = [], [], [], [], []
        for _, p, g, st in run:
            params.append(p)
            grads.append(g.contiguous())
            if self.state_bits == 8:
                m.append(Moment8(st["exp_avg"], st["exp_avg_exp"], True))
                v.append(Moment8(st["exp_avg_sq"], st["exp_avg_sq_exp"], False))
            else:
                m.append(st["exp_avg"])
                v.append(st["exp_avg_sq"])
            w.append(st.get("master"))
        return _Tensors(params, grads, m, v, None if dtype == torch.float32 else w)

    def load_state_dict(self, state_dict) -> None:
        """As torch's, but each state keeps its own dtype (torch's would turn codes and
        masters into the parameter's)."""
        super().load_state_dict(state_dict)
        saved = state_dict["state"]
        ids = [i for g in state_dict["param_groups"] for i in g["params"]]
        params = [p for g in self.param_groups for p in g["params"]]
        for i, p in zip(ids, params):
            if i not in saved:
                continue
            for k, x in saved[i].items():
                if isinstance(x, torch.Tensor):
                    self.state[p][k] = x.detach().clone().to(p.device)


__all__ = ["AdamW", "Moment8", "adamw_step"]
