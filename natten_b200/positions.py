"""Rotary positions over one to three token axes, for queries and keys of the attention operators."""
from __future__ import annotations

import math
from typing import Any, Optional, Sequence, Tuple, Union

import torch
from torch import Tensor

from . import _native, ops
from .functional import _native_eligible, _require_cuda, _wants_grad

ROTARY_DTYPES = (torch.float32, torch.float16, torch.bfloat16)
MAX_HEAD_DIM = 256


def rotary_axis_dims(head_dim: int, axes: int) -> Tuple[int, ...]:
    """The channels that each of `axes` token axes gets by default: equal parts in steps of 8 channels
    (of 2 where the head has no 8 for every axis), the first axes taking what is left over."""
    step = 8 if head_dim % 8 == 0 and head_dim >= 8 * axes else 2
    n = head_dim // step
    return tuple(step * (n // axes + (a < n % axes)) for a in range(axes))


def _per_axis(x: Any, axes: int, name: str, kinds, check, what: str):
    values = list(x) if isinstance(x, Sequence) and not isinstance(x, str) else [x] * axes
    if len(values) != axes or not all(isinstance(v, kinds) and not isinstance(v, bool) and check(v)
                                      for v in values):
        raise ValueError(f"Invalid value for `{name}`; expected {what} or one for each of {axes} axes, "
                         f"got {x!r}.")
    return values


def check_rotary_args(axes: int, head_dim: int, axis_dims: Any, theta: Any, origin: Any,
                      position_scale: Any):
    """(axis_dims, theta, position_scale, origin), one of each for every axis."""
    if axis_dims is None:
        axis_dims = rotary_axis_dims(head_dim, axes)
    if (not isinstance(axis_dims, Sequence) or len(axis_dims) != axes
            or not all(isinstance(d, int) and not isinstance(d, bool) and d >= 0 and d % 2 == 0
                       for d in axis_dims) or sum(axis_dims) > head_dim):
        raise ValueError(f"`axis_dims` must hold {axes} even numbers of channels, {head_dim} together at "
                         f"most, got {axis_dims!r}.")
    theta = _per_axis(theta, axes, "theta", (int, float), lambda v: v > 0 and math.isfinite(v),
                      "a positive number")
    position_scale = _per_axis(position_scale, axes, "position_scale", (int, float), math.isfinite,
                               "a finite number")
    origin = _per_axis(origin, axes, "origin", int, lambda v: abs(v) < 2 ** 53, "an integer")
    return list(axis_dims), [float(v) for v in theta], [float(v) for v in position_scale], origin


def rotary(query: Tensor, key: Optional[Tensor] = None, axis_dims: Optional[Sequence[int]] = None,
           theta: Union[float, Sequence[float]] = 10000.0, positions: Optional[Tensor] = None,
           origin: Union[int, Sequence[int]] = 0, position_scale: Union[float, Sequence[float]] = 1.0,
           interleaved: bool = False) -> Union[Tensor, Tuple[Tensor, Tensor]]:
    """Rotary positions for ``[batch, *tokens, heads, head_dim]`` query and key with 1 to 3 token axes.

    Axis a owns ``axis_dims[a]`` consecutive channels (default: `rotary_axis_dims`); their pair i turns by
    ``position * position_scale * theta ** (-2 * i / axis_dims[a])``. Pairs are channel i of the first and
    of the second half of the axis' channels, or neighbours with ``interleaved=True``. Channels behind the
    last axis pass through. The position of a token is its coordinate along the axis plus ``origin``, or
    comes from ``positions``: ``[batch or 1, *tokens, axes]`` of int32, int64 or float32, with any number
    of axes from 1 to 3 (a flat sequence of text and image tokens can carry time, height and width). Angles
    are formed and reduced in 64 bits: off by 2e-15 of themselves at most, which fp32 does not see up to
    about 2**25 (2**32: 1e-5).

    Returns new contiguous tensors: the query alone when there is no key, else (query, key). fp32, fp16
    and bf16, head dims up to 256; differentiable in query and key, also twice (refused where
    ``NATTEN_B200_DISABLE_TORCH_OPS=1`` leaves no registered operator to hold the formula)."""
    if _native_eligible():
        result = _native.rotary(query, key, axis_dims, theta, positions, origin, position_scale, interleaved)
        if result is not None:
            return result
    for name, t in (("Query", query), ("Key", key)):
        if t is None:
            continue
        if t.is_sparse or t.is_nested:
            raise NotImplementedError("natten_b200 does not support sparse or nested tensors.")
        if t.dim() not in (4, 5, 6):
            raise ValueError(f"{name} must be [batch, *tokens, heads, head_dim] with 1 to 3 token axes, "
                             f"got {t.dim()=}.")
        if t.dtype not in ROTARY_DTYPES:
            raise ValueError(f"rotary() takes fp32, fp16 and bf16 tensors, got {t.dtype}.")
    if key is not None:
        if query.device != key.device or query.dtype != key.dtype:
            raise ValueError("Query and key must have the same device and data type, got "
                             f"{query.device}, {key.device}, {query.dtype}, {key.dtype}.")
        if (query.dim() != key.dim() or query.shape[:-2] != key.shape[:-2]
                or query.shape[-1] != key.shape[-1]):
            raise ValueError("Query and key must match in batch, token layout and head dim, got "
                             f"{tuple(query.shape)} and {tuple(key.shape)}.")
    head_dim, lead = query.shape[-1], query.shape[:-2]
    if head_dim > MAX_HEAD_DIM:
        raise NotImplementedError(f"rotary() takes head dims up to {MAX_HEAD_DIM}, got {head_dim}.")
    if not isinstance(interleaved, bool):
        raise ValueError(f"`interleaved` must be a boolean, got {interleaved!r}.")
    for t in (query, key):
        if t is not None and max(t.shape) >= 2 ** 31:
            raise NotImplementedError(f"rotary() takes axes of less than 2**31 entries, got {tuple(t.shape)}.")
    axes = query.dim() - 3
    if positions is not None:
        if positions.dtype not in ops.POSITION_CODE:
            raise ValueError(f"`positions` must be int32, int64 or float32, got {positions.dtype}.")
        if (positions.dim() != query.dim() - 1 or not 1 <= positions.shape[-1] <= 3
                or positions.shape[1:-1] != lead[1:] or positions.shape[0] not in (1, lead[0])):
            raise ValueError("`positions` must be [batch or 1, *tokens, axes] with 1 to 3 axes, got "
                             f"{tuple(positions.shape)} for a query of {tuple(query.shape)}.")
        if positions.device != query.device:
            raise ValueError(f"`positions` must be on the query's device, got {positions.device}.")
        if positions.requires_grad and torch.is_grad_enabled():
            raise NotImplementedError("rotary() has no gradient for positions.")
        axes = positions.shape[-1]
    how = check_rotary_args(axes, head_dim, axis_dims, theta, origin, position_scale)
    if positions is not None and any(how[3]):
        raise ValueError("`origin` belongs to positions that come from the layout; add it to `positions`.")
    if not ops.USE_TORCH_OPS and _wants_grad(query, key):
        raise NotImplementedError("rotary() has no gradient without registered operators "
                                  "(NATTEN_B200_DISABLE_TORCH_OPS=1).")
    _require_cuda(query, key, positions)
    out = ops.rotary(query, key, *how, positions, interleaved, False)
    return out[0] if key is None else out
