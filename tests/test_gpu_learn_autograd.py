"""The policy loss in autograd: its inputs belong to the graph until the backward has run (GPU)."""

import pytest
import torch

import swarp_b200 as swarp
from test_gpu_learn_policy import batch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
NAMES = ["logits", "tokens", "old_logp", "advantages", "ref_logp", "mask"]
KW = dict(kl_coef=0.05, entropy_coef=0.01)


def inputs(rows=40, V=300, dtype=torch.float32, seed=0):
    z, tok, old, adv, ref = batch(rows, V, dtype, seed=seed)
    return dict(logits=z, tokens=tok, old_logp=old, advantages=adv, ref_logp=ref,
                mask=torch.arange(rows, device=DEV) % 4 != 1)


def loss_of(x):
    rest = {k: v for k, v in x.items() if k in ("ref_logp", "mask")}
    return swarp.policy_loss(x["logits"], x["tokens"], x["old_logp"], x["advantages"], **rest, **KW)


def grad_of(x, scale):
    rest = {k: v for k, v in x.items() if k in ("ref_logp", "mask")}
    return swarp.policy_loss_and_grad(x["logits"].detach(), x["tokens"], x["old_logp"],
                                      x["advantages"], grad_scale=scale, **rest, **KW)[1]


@pytest.mark.parametrize("scale", [1.0, 0.5])
@pytest.mark.parametrize("name", NAMES)
def test_a_changed_input_is_an_error(name, scale):
    """As in any composition of tensor operations: the gradient would be another loss's."""
    x = inputs()
    leaf = x["logits"].clone().requires_grad_(True)
    x["logits"] = leaf * 1.0
    out = loss_of(x)
    with torch.no_grad():
        x[name].copy_(x[name].roll(1, 0))
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        (out.loss * scale).backward()


def test_a_refilled_buffer_is_an_error():
    """Two losses over one static buffer, summed and divided before one backward."""
    x, y = inputs(), inputs(seed=1)
    x["logits"].requires_grad_(True)
    first = loss_of(x).loss
    for k in NAMES[1:]:
        x[k].copy_(y[k])
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        ((first + loss_of(x).loss) / 2).backward()


@pytest.mark.parametrize("scale", [1.0, 0.25])
def test_inputs_of_a_rollout_in_inference_mode(scale):
    """They cannot be saved as they are, and are used all the same; a change after the call does
    not reach the gradient."""
    with torch.inference_mode():
        rolled = inputs()
    x = {k: v for k, v in rolled.items() if k != "logits"}
    x["logits"] = rolled["logits"].clone().requires_grad_(True)
    want = grad_of(x, scale)
    out = loss_of(x)
    with torch.inference_mode():
        for k in NAMES[1:]:
            rolled[k].copy_(rolled[k].roll(1, 0))
    (out.loss * scale).backward()
    assert torch.equal(x["logits"].grad, want)


@pytest.mark.parametrize("scale", [1.0, 0.25])
def test_inputs_that_only_the_graph_holds(scale):
    """The caller's own references may go: the graph keeps what the backward reads."""
    x = inputs(rows=3000, V=50, dtype=torch.bfloat16)
    leaf = x["logits"].requires_grad_(True)
    want = grad_of(x, scale)
    loss = loss_of({k: v if k == "logits" else v.clone() for k, v in x.items()}).loss
    junk = [torch.full_like(v, 1) for k, v in x.items() for _ in range(4) if k != "logits"]
    (loss * scale).backward()
    assert torch.equal(leaf.grad, want) and junk


@pytest.mark.parametrize("V", [21, 300, 5000])
@pytest.mark.parametrize("scale", [1.0, 0.25])
def test_inputs_that_a_hook_brings_back(scale, V):
    """Saved tensors that wait on the host come back in other places, and a slice of a padded
    batch comes back without the padding."""
    B, T = 4, 10
    x = inputs(rows=B * T, V=V)
    want = grad_of(x, scale)
    wide = torch.full((B, T + 2, V + 3), float("nan"), device=DEV)
    wide[:, :T, :V] = x["logits"].view(B, T, V)
    leaf = wide.requires_grad_(True)
    y = {k: v.view(B, T) for k, v in x.items() if k != "logits"}
    y["logits"] = leaf[:, :T, :V]
    with torch.autograd.graph.save_on_cpu():
        loss = loss_of(y).loss
    (loss * scale).backward(retain_graph=True)
    first, leaf.grad = leaf.grad, None
    (loss * scale).backward()
    for g in (first, leaf.grad):
        # a row at another alignment may be summed in another order
        torch.testing.assert_close(g[:, :T, :V].reshape(B * T, V), want, rtol=1e-4, atol=1e-8)
        assert not g[:, T:].any() and not g[..., V:].any()
