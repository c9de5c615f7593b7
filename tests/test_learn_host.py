"""Host side of the policy-training operators (CPU): struct layouts, argument validation before
any CUDA call, row strides, the refusal of CPU tensors, and the 8-bit rounding's random bits."""

import ctypes as C
import os
import subprocess

import pytest
import torch

import swarp_b200 as swarp
from swarp_b200 import _lib, build
from swarp_b200.learn.policy import _rows

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def lib():
    build.build()
    so = C.CDLL(_lib.LIB_PATH)
    for name, (res, args) in _lib.SIGNATURES.items():
        getattr(so, name).restype, getattr(so, name).argtypes = res, args
    return so


PAIRS = [("swarp_policy_t", _lib.Policy), ("swarp_gae_t", _lib.Gae),
         ("swarp_adamw_tensor_t", _lib.AdamWTensor), ("swarp_adamw_t", _lib.AdamWOpt)]


def test_struct_layouts(tmp_path):
    lines = []
    for name, cls in PAIRS:
        lines.append(f'printf("{name} %zu\\n", sizeof({name}));')
        for field, _ in cls._fields_:
            lines.append(f'printf("{name}.{field} %zu\\n", offsetof({name}, {field.rstrip("_")}));')
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "swarp_b200.h"\n'
                   "int main(void) {" + "\n".join(lines) + "return 0;}")
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)],
                   check=True)
    out = dict(x.rsplit(" ", 1) for x in subprocess.check_output([str(exe)]).decode().split("\n")
               if x)
    for name, cls in PAIRS:
        assert int(out[name]) == C.sizeof(cls)
        for field, _ in cls._fields_:
            assert int(out[f"{name}.{field}"]) == getattr(cls, field).offset, (name, field)


def policy(**kw):
    p = _lib.Policy()
    p.rows, p.vocab, p.inner, p.stride_inner = 4, 8, 4, 8
    for k in ("logits", "tokens", "old_logp", "advantages", "logp", "entropy", "loss", "stats"):
        setattr(p, k, 256)  # placeholders, never dereferenced
    for k, x in kw.items():
        setattr(p, k, x)
    return p


def test_policy_validation(lib):
    size = lib.swarp_policy_workspace_bytes
    assert size(None) == 0 and size(C.byref(policy())) > 0
    for bad in (dict(dtype=1), dict(dtype=9), dict(rows=-1), dict(vocab=0), dict(vocab=1 << 31),
                dict(inner=0), dict(inner=3)):
        assert size(C.byref(policy(**bad))) == 0, bad
        assert lib.swarp_policy_loss(C.byref(policy(**bad)), 256, 1 << 30, None) == -1, bad
    for k in ("logits", "tokens", "old_logp", "advantages", "logp", "entropy", "loss", "stats"):
        assert lib.swarp_policy_loss(C.byref(policy(**{k: None})), 256, 1 << 30, None) == -1, k
    p = policy()
    assert lib.swarp_policy_loss(C.byref(p), None, 1 << 30, None) == -5
    assert lib.swarp_policy_loss(C.byref(p), 256, size(C.byref(p)) - 1, None) == -5
    assert lib.swarp_policy_grad(C.byref(p), None, 0, 256, 1 << 30, None) == -1
    assert lib.swarp_policy_grad(C.byref(p), 256, 0, 256, 1 << 30, None) == -1  # no grad
    assert lib.swarp_token_logp(C.byref(policy(logp=None)), 256, 1 << 30, None) == -1


def test_gae_validation(lib):
    def call(**kw):
        g = _lib.Gae(0, 1, 4, 6, 256, 256, None, 256, None, None, 0.9, 0.9, 256, 256)
        for k, x in kw.items():
            setattr(g, k, x)
        return lib.swarp_gae(C.byref(g), None, 0, None)

    assert lib.swarp_gae(None, None, 0, None) == -1
    for bad in (dict(dtype=2), dict(steps=-1), dict(columns=-1), dict(columns_per_flag=0),
                dict(columns_per_flag=4), dict(rewards=None), dict(values=None),
                dict(last_values=None), dict(advantages=None), dict(returns=None)):
        assert call(**bad) == -1, bad
    assert call(steps=0) == 0 and call(columns=0) == 0


def test_adamw_validation(lib):
    t = (_lib.AdamWTensor * 1)(_lib.AdamWTensor(4, 256, 256, None, 256, 256, None, None))

    def call(n=1, tensors=t, **kw):
        o = _lib.AdamWOpt(0, 32, 1, 1e-3, 0.9, 0.99, 1e-8, 0.0, 0, 0, None, 0, 0.0, None)
        for k, x in kw.items():
            setattr(o, k, x)
        return lib.swarp_adamw_step(C.byref(o), tensors, n, None)

    for bad in (dict(dtype=1), dict(moment_bits=16), dict(step=0), dict(beta1=1.0),
                dict(beta2=-0.1), dict(moment_bits=8), dict(dtype=2),
                dict(norm_partials=256), dict(norm_partials=256, n_norm_partials=4)):
        assert call(**bad) == -1, bad
    assert call(n=-1) == -1 and call(tensors=None) == -1
    for k in ("param", "grad", "exp_avg", "exp_avg_sq"):
        u = (_lib.AdamWTensor * 1)(_lib.AdamWTensor(4, 256, 256, None, 256, 256, None, None))
        setattr(u[0], k, None)
        assert call(tensors=u) == -1, k
    empty = (_lib.AdamWTensor * 1)()
    assert call(tensors=empty) == 0 and call(n=0) == 0
    assert lib.swarp_grad_norm_partials(0, t, 1, None, None) == -1
    assert lib.swarp_grad_norm_partials(1, t, 1, 256, None) == -1
    count = lib.swarp_grad_norm_partials_count
    assert count(1) == count(0) > 0 and count(10_000) > count(1) and count(-1) == 0
    assert lib.swarp_moment8_values(None, None, 4, 0, 0, None, None) == -1
    assert lib.swarp_moment8_values(256, 256, 4, 0, 3, 256, None) == -1
    assert lib.swarp_moment8_values(None, None, 0, 0, 0, None, None) == 0


def test_cpu_tensors_are_refused():
    z, tok = torch.zeros(4, 5), torch.zeros(4, dtype=torch.int64)
    f = torch.zeros(4)
    for call in (lambda: swarp.policy_loss(z, tok, f, f), lambda: swarp.token_logp(z, tok),
                 lambda: swarp.policy_loss_and_grad(z, tok, f, f), lambda: swarp.gae(z, z, z[0]),
                 lambda: swarp.adamw_step([f], [f], [f], [f], step=1, lr=0.1),
                 lambda: swarp.Moment8.zeros(4, "cpu", True).values()):
        with pytest.raises(RuntimeError, match="CUDA device only"):
            call()


def offsets(t):
    z, rows, inner, so, si = _rows(t)
    base = (z.data_ptr() - t.data_ptr()) // 4 if z.data_ptr() == t.data_ptr() else None
    return z is t, [(i // inner) * so + (i % inner) * si for i in range(rows)], base


@pytest.mark.parametrize("make,copied", [
    (lambda b: b, False),
    (lambda b: b[:, :-1], False),
    (lambda b: b[..., 2:5], False),
    (lambda b: b[1:, ::2], False),
    (lambda b: b.transpose(0, 1), False),
    (lambda b: b[:, :1], False),
    (lambda b: b[0], False),
    (lambda b: b[0, 0], False),
    (lambda b: b[:1].expand(6, 5, 7), False),
    (lambda b: b.transpose(1, 2), True),
    (lambda b: b.view(2, 2, 5, 7).transpose(0, 2), True),
])
def test_row_offsets(make, copied):
    base = torch.arange(4 * 5 * 7, dtype=torch.float32).view(4, 5, 7)
    t = make(base)
    same, offs, _ = offsets(t)
    assert same != copied
    if same:  # each row's first element is its offset from the tensor's first
        want = [float(x) for x in (t[..., 0] - t.reshape(-1)[0]).reshape(-1)]
        assert offs == want


def test_random_bits_are_even():
    """The rounding's hash: every one of its 32 bits is even over elements, steps and tensors,
    and changes with every bit of the element's index about half the time."""
    M = 0xFFFFFFFF

    def mix(x):
        x = x ^ (x >> 16)
        x = (x * 0xE80B5AE5) & M
        x = x ^ (x >> 15)
        x = (x * 0xCB276749) & M
        return x ^ (x >> 16)

    n = 1 << 16
    i = torch.arange(n)
    sd = 0.5 / n ** 0.5
    for step in range(3):
        for tensor in range(3):
            h = mix(i ^ mix((mix(step) + tensor) & M))
            bits = (h[:, None] >> torch.arange(32)) & 1
            # 32 x 9 means of n fair bits: six standard deviations
            assert (bits.double().mean(0) - 0.5).abs().max() < 6 * sd
    for b in range(16):
        flip = mix(i) ^ mix(i ^ (1 << b))
        bits = (flip[:, None] >> torch.arange(32)) & 1
        assert (bits.double().mean(0) - 0.5).abs().max() < 0.02
