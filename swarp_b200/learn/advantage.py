"""Generalised advantage estimates of a rollout.

    delta_t = r_t + gamma V'_t - V_t
    A_t     = delta_t + gamma lam A_{t+1},   returns_t = A_t + V_t

with ``V'_t`` dropped at a terminated step and ``A_{t+1}`` at a terminated or truncated one:
what ``Environment.step`` returns over T steps (``V'_t`` is the value of ``info["final_obs"]``), in one launch (two for a long rollout of few
columns, which is split along time). The reference's trainer loops over the steps in torch.
"""

from __future__ import annotations

import ctypes as C
import math

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

_FLOATS = (torch.float32, torch.float64)
_BOOL = (torch.bool,)
_MOST_PER_FLAG = 2 ** 31 - 1  # swarp_gae_t.columns_per_flag is an int32


def _flag_dims(shape, dims: int) -> int:
    """Leading dimensions of ``shape`` that the flags have to have, ``dims`` at least, so that
    the number of columns that share one fits the C struct."""
    while math.prod(shape[dims:]) > _MOST_PER_FLAG:
        dims += 1
    return dims


def gae(
    rewards: torch.Tensor,
    values: torch.Tensor,
    last_values: torch.Tensor | None,
    terminated: torch.Tensor | None = None,
    truncated: torch.Tensor | None = None,
    *,
    gamma: float = 0.99,
    lam: float = 0.95,
    next_values: torch.Tensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """``(advantages, returns)`` of ``rewards`` and ``values`` ``[T, ...]`` (float32 or
    float64), fresh and contiguous.

    ``last_values`` ``[...]`` follow the last step. ``terminated`` and ``truncated`` (bool)
    have the shape of the rewards or of their leading dimensions: ``[T, n_envs]`` flags
    serve ``[T, n_envs, n_agents]`` rewards. The value that follows step ``t`` is
    ``values[t + 1]``, or ``next_values[t]`` where those are given (``last_values`` may then
    be ``None``): give them when episodes are truncated and reset inside the rollout, where
    ``values[t + 1]`` already belongs to the next episode; ``Environment(...,
    final_observation=True)`` hands out the observations that they are of. A value that a terminated step
    drops may be anything, NaN included. The results are constants: no gradient flows.
    """
    require_cuda(rewards, "rewards")
    if rewards.dim() < 1:
        raise ValueError("rewards must be [T, ...]")
    shape, device, dtype = rewards.shape, rewards.device, rewards.dtype
    if dtype not in _FLOATS:
        raise TypeError(f"rewards dtype {dtype}: want float32 or float64")
    if not (0.0 <= gamma <= 1.0 and 0.0 <= lam <= 1.0):
        raise ValueError(f"gamma and lam must be in [0, 1], got {gamma} and {lam}")
    same = (dtype,)
    r = like(rewards, "rewards", shape, same, device)
    v = like(values, "values", shape, same, device)
    for t, name in ((rewards, "rewards"), (values, "values"), (last_values, "last_values"),
                    (next_values, "next_values")):
        constant(t, name)
    nxt = last = None
    if next_values is not None:
        nxt = like(next_values, "next_values", shape, same, device)
    elif last_values is None:
        raise ValueError("gae needs last_values or next_values")
    if last_values is not None:
        last = like(last_values, "last_values", shape[1:], same, device)
    flags, lead = [], None
    for t, name in ((terminated, "terminated"), (truncated, "truncated")):
        if t is not None:
            want = shape[:t.dim()] if isinstance(t, torch.Tensor) and t.dim() >= 1 else shape
            t = like(t, name, want, _BOOL, device)
            if lead is not None and t.shape != lead:
                raise ValueError(f"terminated has shape {tuple(lead)}, truncated "
                                 f"{tuple(t.shape)}")
            lead = t.shape
        flags.append(t)
    columns = math.prod(shape[1:])
    per_flag = 1
    if lead is not None:
        dims = _flag_dims(shape, len(lead))
        if dims > len(lead):
            flags = [t if t is None else t.view(*lead, *[1] * (dims - len(lead)))
                     .expand(shape[:dims]).contiguous() for t in flags]
        per_flag = math.prod(shape[dims:])
    adv = torch.empty_like(r)
    ret = torch.empty_like(adv)
    if adv.numel() == 0:
        return adv, ret
    c = _lib.Gae(DTYPES[dtype], per_flag, shape[0], columns,
                 *(_lib.ptr(t) for t in (r, v, nxt, last, *flags)), gamma, lam, adv.data_ptr(),
                 ret.data_ptr())
    lib = library()
    with on_device(device):
        n = lib.swarp_gae_workspace_bytes(C.byref(c))
        ws = workspace(n, r) if n else None
        _lib.check(lib.swarp_gae(C.byref(c), _lib.ptr(ws), n, stream(device)), "swarp_gae")
    return adv, ret


__all__ = ["gae"]
