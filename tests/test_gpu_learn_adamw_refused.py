"""A step of the optimizer that is refused leaves its state as it was (GPU)."""

import copy

import pytest
import torch

import swarp_b200 as swarp

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def state_of(opt):
    return copy.deepcopy(opt.state_dict())


def same(a, b):
    assert a["state"].keys() == b["state"].keys()
    for k in a["state"]:
        for name, x in a["state"][k].items():
            y = b["state"][k][name]
            assert torch.equal(x, y) if torch.is_tensor(x) else x == y, (k, name)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("first", [True, False])  # the refused step is the first, or a later one
@pytest.mark.parametrize("what", ["device", "sparse", "strides", "dtype", "betas"])
def test_a_refused_step_leaves_the_state(what, first, bits):
    g = torch.Generator(device=DEV).manual_seed(0)
    ps = [torch.nn.Parameter(torch.randn(40, 30, generator=g, device=DEV)) for _ in range(3)]
    opt = swarp.AdamW([{"params": ps[:2]}, {"params": ps[2:]}], lr=0.1, state_bits=bits)

    def grads():
        for p in ps:
            p.grad = torch.ones_like(p)

    grads()
    if not first:
        opt.step()
    before, values = state_of(opt), [p.detach().clone() for p in ps]
    other = None
    if what == "device":
        other = torch.nn.Parameter(torch.ones(4))
        other.grad = torch.ones(4)
        opt.add_param_group({"params": [other]})
    elif what == "sparse":
        ps[2].grad = torch.ones(40, 30, device=DEV).to_sparse()
    elif what == "strides":
        ps[2].data = ps[2].data.t()
        ps[2].grad = torch.ones(30, 40, device=DEV)
    elif what == "dtype":
        other = torch.nn.Parameter(torch.ones(4, dtype=torch.float64, device=DEV))
        other.grad = torch.ones_like(other)
        opt.add_param_group({"params": [other]})
    else:
        opt.param_groups[1]["betas"] = (0.9, 1.0)
    with pytest.raises((ValueError, RuntimeError, TypeError)):
        opt.step()
    same(state_of(opt), before)
    # mended, it goes on as if nothing had been
    if other is not None:
        other.grad = None
    if what == "strides":
        ps[2].data = ps[2].data.t()
    opt.param_groups[1]["betas"] = (0.9, 0.999)
    grads()
    opt.step()
    copies = [torch.nn.Parameter(x) for x in values]
    clean = swarp.AdamW([{"params": copies[:2]}, {"params": copies[2:]}], lr=0.1, state_bits=bits)
    clean.load_state_dict(before)
    for p in copies:
        p.grad = torch.ones_like(p)
    clean.step()
    assert all(torch.equal(a, b) for a, b in zip(ps, copies))
