"""The clipped policy loss over token logits, with its gradient, and token log probabilities.

A policy that chooses one of ``V`` tokens per row (a bin of an action slot, a word) gives
logits ``[..., V]``. With ``lp`` the log probability of the row's token, ``r =
exp(lp - old_logp)``, ``A`` its advantage, ``d = ref_logp - lp`` and ``H`` the entropy,

    row loss = -min(r A, clip(r, 1 - clip_low, 1 + clip_high) A)
               + kl_coef (exp(d) - d - 1) - entropy_coef H

and the loss is the mean (or sum) over the rows that ``mask`` admits. One kernel reads each
row once and writes its gradient; a plain composition of tensor operations passes over the
logits some twenty times. The reference has no counterpart on its step path (its trainer
composes the loss in torch).
"""

from __future__ import annotations

import ctypes as C
from typing import NamedTuple

import torch

from swarp_b200 import _lib
from swarp_b200.learn._call import (
    DTYPES,
    constant,
    library,
    like,
    on_device,
    require_cuda,
    stream,
    workspace,
)

_LOGIT_DTYPES = (torch.float32, torch.bfloat16, torch.float16)
_TOKEN_DTYPES = (torch.int64, torch.int32)
_F32 = (torch.float32,)
_BOOL = (torch.bool,)


class PolicyLoss(NamedTuple):
    """``loss`` (a scalar, differentiable in :func:`policy_loss`), per-row ``logp`` and
    ``entropy`` (float32; 0 where the mask leaves a row out) and ``stats``: the mean (or sum)
    over the admitted rows of the clipped term, of ``exp(d) - d - 1``, of the entropy, and of
    1 where the clip cut the gradient."""

    loss: torch.Tensor
    logp: torch.Tensor
    entropy: torch.Tensor
    stats: torch.Tensor


def _rows(logits: torch.Tensor):
    """``(logits, rows, inner, stride_outer, stride_inner)``: row ``i`` of the logits starts
    ``(i // inner) * stride_outer + (i % inner) * stride_inner`` elements in. Any slice of a
    contiguous ``[B, T, V]`` along ``B``, ``T`` or the end of ``V`` fits without a copy; what
    does not (``V`` not adjacent, more than two levels of strides) is copied."""
    V = logits.shape[-1]
    rows = logits.numel() // V if V else 0
    if logits.is_contiguous():
        return logits, rows, rows, 0, V
    if logits.stride(-1) == 1 or V == 1:
        levels: list[list[int]] = []  # [size, stride], innermost last
        for n, s in zip(logits.shape[:-1], logits.stride()[:-1]):
            if n == 1:
                continue
            if levels and levels[-1][1] == n * s:
                levels[-1][0] *= n
                levels[-1][1] = s
            else:
                levels.append([n, s])
        if len(levels) < 2:
            return logits, rows, rows, 0, levels[0][1] if levels else V
        if len(levels) == 2:
            return logits, rows, levels[1][0], levels[0][1], levels[1][1]
    return logits.contiguous(), rows, rows, 0, V


class _Batch:
    """Checked arguments as the C struct, and the tensors that it points to (``keep``, by the
    struct's field ``fields``, the logits first)."""

    def __init__(self, logits, tokens, old_logp=None, advantages=None, ref_logp=None, mask=None,
                 clip_low=0.0, clip_high=0.0, kl_coef=0.0, entropy_coef=0.0, mean=True,
                 grad_scale=1.0):
        require_cuda(logits, "logits")
        if logits.dtype not in _LOGIT_DTYPES:
            raise TypeError(f"logits dtype {logits.dtype}: want float32, bfloat16 or float16")
        if logits.dim() < 1 or logits.shape[-1] < 1:
            raise ValueError(f"logits must be [..., V] with V >= 1, got {tuple(logits.shape)}")
        self.shape = lead = logits.shape[:-1]
        self.device = device = logits.device
        rowed, rows, inner, outer_stride, inner_stride = _rows(logits)
        tokens = like(tokens, "tokens", lead, _TOKEN_DTYPES, device)
        self.keep = keep = [rowed, tokens]
        self.fields = fields = ["logits", "tokens"]
        self.strides = rowed.stride()
        small = []
        for t, name, dtypes in ((old_logp, "old_logp", _F32), (advantages, "advantages", _F32),
                                (ref_logp, "ref_logp", _F32), (mask, "mask", _BOOL)):
            if t is not None:
                constant(t, name)
                t = like(t, name, lead, dtypes, device)
                keep.append(t)
                fields.append(name)
            small.append(None if t is None else t.data_ptr())
        self.c = _lib.Policy(DTYPES[logits.dtype], tokens.dtype == torch.int64, rows,
                             logits.shape[-1], inner, outer_stride, inner_stride,
                             rowed.data_ptr(), tokens.data_ptr(), *small, clip_low, clip_high,
                             kl_coef, entropy_coef, mean, grad_scale)

    def outputs(self):
        logp = self.keep[0].new_empty(self.shape, dtype=torch.float32)
        entropy = torch.empty_like(logp)
        self.c.logp, self.c.entropy = logp.data_ptr(), entropy.data_ptr()
        return logp, entropy

    def reads(self, tensors) -> None:
        """Point the struct at ``tensors`` in place of ``keep``, with the same values: what a
        saved-tensor hook brings back may lie in another place and in another order."""
        keep, c = list(tensors), self.c
        if keep[0].stride() != self.strides:
            keep[0], _, c.inner, c.stride_outer, c.stride_inner = _rows(keep[0])
            self.strides = keep[0].stride()
        for k, field in enumerate(self.fields):
            if k and not keep[k].is_contiguous():
                keep[k] = keep[k].contiguous()
            setattr(c, field, keep[k].data_ptr())
        self.keep = keep

    def new_grad(self, logits):
        grad = (torch.empty_like(logits) if logits.is_contiguous() else
                logits.new_empty((*self.shape, self.c.vocab)))
        self.c.grad = grad.data_ptr()
        return grad

    def call(self, what: str, on: torch.Tensor, *args):
        lib = library()
        with on_device(self.device):
            ref = C.byref(self.c)
            n = lib.swarp_policy_workspace_bytes(ref)
            ws = workspace(n, on)
            rc = getattr(lib, what)(ref, *args, ws.data_ptr(), n, stream(self.device))
        if rc:
            _lib.check(rc, what)

    def loss(self, with_grad: bool):
        logp, entropy = self.outputs()
        loss, stats = logp.new_empty(()), logp.new_empty(4)
        self.c.loss, self.c.stats = loss.data_ptr(), stats.data_ptr()
        grad = self.new_grad(self.keep[0]) if with_grad else None
        self.call("swarp_policy_loss", logp)
        return PolicyLoss(loss, logp, entropy, stats), grad


class _PolicyLossFn(torch.autograd.Function):
    """The forward writes the gradient of the loss itself beside it, in one pass over the
    logits. The backward hands that buffer out. Where the loss's cotangent is not 1 it is
    written anew from the logits first (scaling it would round twice, and lose what a loss
    scale keeps above the smallest float16); the device decides, so the host does not wait."""

    @staticmethod
    def forward(ctx, logits, batch):
        out, ctx.grad = batch.loss(True)
        batch.out = out  # the rest of it is not differentiable and stays outside autograd
        # autograd alone keeps the inputs: a loss kept for the record frees them, and one that is
        # written to before the backward is an error. An inference tensor cannot be kept, and
        # has no version to compare: a copy takes its place
        kept = [t.clone() if t.is_inference() else t for t in batch.keep]
        if kept[0] is not logits:
            kept.append(logits)
        ctx.save_for_backward(*kept)
        batch.keep = None
        ctx.batch = batch
        return out.loss

    @staticmethod
    def backward(ctx, g_loss):
        if torch.is_grad_enabled():
            raise RuntimeError("policy_loss is differentiable once (create_graph is not supported)")
        inputs = ctx.saved_tensors
        batch, grad, ctx.grad = ctx.batch, ctx.grad, None
        skip_unit = grad is not None
        batch.reads(inputs[:len(batch.fields)])
        if grad is None:  # a second backward of a retained graph: the buffer is gone
            grad = batch.new_grad(batch.keep[0])
        batch.call("swarp_policy_grad", grad, g_loss.data_ptr(), int(skip_unit))
        batch.keep = None
        return grad, None


def _settings(clip_low, clip_high, reduction):
    if not 0.0 <= clip_low <= 1.0:
        raise ValueError(f"clip_low must be in [0, 1], got {clip_low}")
    if not clip_high >= 0.0:
        raise ValueError(f"clip_high must be >= 0, got {clip_high}")
    if reduction not in ("mean", "sum"):
        raise ValueError(f"reduction must be 'mean' or 'sum', got {reduction!r}")
    return clip_low, clip_high


def _batch(logits, tokens, old_logp, advantages, ref_logp, mask, clip_low, clip_high, kl_coef,
           entropy_coef, reduction, grad_scale=1.0):
    low, high = _settings(clip_low, clip_high, reduction)
    if ref_logp is None and kl_coef != 0.0:
        raise ValueError("kl_coef needs ref_logp")
    for t, name in ((old_logp, "old_logp"), (advantages, "advantages")):
        if t is None:
            raise TypeError(f"{name} must be a tensor, got None")
    return _Batch(logits, tokens, old_logp, advantages, ref_logp, mask, low, high, kl_coef,
                  entropy_coef, reduction == "mean", grad_scale)


def policy_loss(
    logits: torch.Tensor,
    tokens: torch.Tensor,
    old_logp: torch.Tensor,
    advantages: torch.Tensor,
    *,
    ref_logp: torch.Tensor | None = None,
    mask: torch.Tensor | None = None,
    clip_low: float = 0.2,
    clip_high: float = 0.2,
    kl_coef: float = 0.0,
    entropy_coef: float = 0.0,
    reduction: str = "mean",
) -> PolicyLoss:
    """The clipped policy loss, differentiable in ``logits`` (``[..., V]``, float32, bfloat16
    or float16, any strides). ``tokens`` (int64 or int32), ``old_logp``, ``advantages``,
    ``ref_logp`` (float32) and ``mask`` (bool) have the logits' leading shape and are
    constants. As with any autograd operation, none of them may be written to before the
    backward has run: that raises an error.

    A masked row adds nothing and its gradient is exactly 0, whatever its inputs hold. A
    logit of ``-inf`` is a token that cannot be chosen; a row of nothing else has ``logp``
    ``-inf``, entropy 0 and no loss or gradient, but counts in the mean. A token outside
    ``[0, V)`` makes the loss NaN. With no row admitted the loss is 0.
    """
    b = _batch(logits, tokens, old_logp, advantages, ref_logp, mask, clip_low, clip_high, kl_coef,
               entropy_coef, reduction)
    if logits.requires_grad and torch.is_grad_enabled():
        loss = _PolicyLossFn.apply(logits, b)
        out, b.out = b.out, None
        return out._replace(loss=loss)
    return b.loss(False)[0]


def policy_loss_and_grad(
    logits: torch.Tensor,
    tokens: torch.Tensor,
    old_logp: torch.Tensor,
    advantages: torch.Tensor,
    *,
    ref_logp: torch.Tensor | None = None,
    mask: torch.Tensor | None = None,
    clip_low: float = 0.2,
    clip_high: float = 0.2,
    kl_coef: float = 0.0,
    entropy_coef: float = 0.0,
    reduction: str = "mean",
    grad_scale: float = 1.0,
) -> tuple[PolicyLoss, torch.Tensor]:
    """:func:`policy_loss` and the gradient of ``grad_scale * loss`` w.r.t. the logits, without
    autograd: ``(PolicyLoss, grad)`` with ``grad`` contiguous in the logits' shape and dtype.
    Hand it on with ``logits.backward(grad)``. ``grad_scale`` is a loss scale (float16
    gradients of a mean over many rows underflow without one), applied before rounding."""
    b = _batch(logits, tokens, old_logp, advantages, ref_logp, mask, clip_low, clip_high, kl_coef,
               entropy_coef, reduction, grad_scale)
    return b.loss(True)


def token_logp(logits: torch.Tensor, tokens: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """``(logp, entropy)``, float32: the log probability of each row's token and the row's
    entropy, as a rollout or a reference policy records them. One pass over the logits; a
    few rows of a long vocabulary are split over several SMs. Not differentiable: with
    ``logits`` that require grad, call it under ``torch.no_grad()``."""
    constant(logits, "logits")
    b = _Batch(logits, tokens)
    out = b.outputs()
    b.call("swarp_token_logp", out[0])
    return out


__all__ = ["PolicyLoss", "policy_loss", "policy_loss_and_grad", "token_logp"]
