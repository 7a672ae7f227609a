"""Neighborhood-attention layers on top of the B200 operators.

Drop-in counterparts of the reference's ``NeighborhoodAttention1D/2D/3D``
(src/natten/modules.py:42-122): same constructor arguments, same parameter names (``qkv``,
``proj``), so a reference checkpoint loads unchanged. Trainable: the operator underneath is
differentiable.

Beyond the reference's layers: rotary positions (``rotary_theta``) and, for the causal 1-D layer, serving
with a paged key/value cache (``prefill`` and ``decode``).
"""
from typing import Any, Optional, Sequence, Tuple

import torch
from torch import Tensor, nn
from torch.nn.modules.module import _has_any_global_hook

from . import _native
from .checks import check_all_args
from .functional import _native_eligible, attention, neighborhood_attention_generic
from .kv_cache import KVCache, _expect_cache, _per_sequence, _refuse_grad, kv_cache_write, na1d_decode
from .positions import check_rotary_args, rotary


def _is_bare_linear(m: nn.Module) -> bool:
    """An nn.Linear that does nothing but its product: no subclass, hook or patched forward."""
    return (type(m) is nn.Linear and not m._forward_hooks and not m._forward_pre_hooks
            and not m._backward_hooks and not m._backward_pre_hooks and "forward" not in m.__dict__)


class NeighborhoodAttentionGeneric(nn.Module):
    """QKV projection -> neighborhood attention over ``na_dim`` token axes -> output projection.

    Input and output are ``[batch, *token_layout, embed_dim]``. With ``rotary_theta`` queries and keys
    get rotary positions over the token axes (`rotary`: ``rotary_axis_dims`` channels each, neighbouring
    channels paired with ``rotary_interleaved``)."""

    # (also for modules that were pickled without them)
    rotary_theta: Any = None
    rotary_axis_dims: Optional[Sequence[int]] = None
    rotary_interleaved = False

    def __init__(self, na_dim: int, embed_dim: int, num_heads: int, kernel_size: Any,
                 stride: Any = 1, dilation: Any = 1, is_causal: Any = False, qkv_bias: bool = True,
                 qk_scale: Optional[float] = None, proj_drop: float = 0.0,
                 rotary_theta: Any = None, rotary_axis_dims: Optional[Sequence[int]] = None,
                 rotary_interleaved: bool = False):
        super().__init__()
        if embed_dim % num_heads != 0:
            raise ValueError("Number of attention heads must evenly divide embedding dimension, "
                             f"got {embed_dim=}, {num_heads=}.")
        self.kernel_size, self.stride, self.dilation, self.is_causal = check_all_args(
            na_dim, kernel_size, stride, dilation, is_causal)
        self.na_dim = na_dim
        self.embed_dim = embed_dim
        self.num_heads = num_heads
        self.head_dim = embed_dim // num_heads
        self.scale = qk_scale or self.head_dim ** -0.5
        if rotary_theta is not None:
            check_rotary_args(na_dim, self.head_dim, rotary_axis_dims, rotary_theta, 0, 1.0)
        self.rotary_theta = rotary_theta
        self.rotary_axis_dims = rotary_axis_dims
        self.rotary_interleaved = bool(rotary_interleaved)
        self.qkv = nn.Linear(embed_dim, 3 * embed_dim, bias=qkv_bias)
        self.proj = nn.Linear(embed_dim, embed_dim)
        self.proj_drop = nn.Dropout(proj_drop)

    def forward(self, x: Tensor) -> Tensor:
        if x.dim() != self.na_dim + 2:
            raise ValueError(f"NeighborhoodAttention{self.na_dim}D expected a tensor with rank "
                             f"{self.na_dim + 2} (batch, {self.na_dim} token axes, embedding), "
                             f"got {x.dim()=}.")
        if x.shape[-1] != self.embed_dim:
            raise ValueError(f"Expected embedding dimension {self.embed_dim}, got {x.shape[-1]} "
                             f"({x.shape=}).")
        # One native call for projection, attention and projection where nothing hangs between them.
        # In training it is one autograd node: the attention's gradients are written straight into
        # the fused projection's gradient (no copies of q, k, v gradients), and the bias gradients
        # are summed by a kernel that reads them at the memory's rate.
        if self.rotary_theta is None and _native_eligible() and not _has_any_global_hook():
            qkv, proj = self.qkv, self.proj
            if _is_bare_linear(qkv) and _is_bare_linear(proj):
                y = _native.layer(self.na_dim, x, qkv.weight, qkv.bias, proj.weight, proj.bias,
                                  self.num_heads, self.kernel_size, self.stride, self.dilation,
                                  self.is_causal, self.scale)
                if y is not None:
                    return self.proj_drop(y)
        lead = x.shape[:-1]
        q, k, v = self._project(x)
        out = neighborhood_attention_generic(q, k, v, kernel_size=self.kernel_size,
                                             stride=self.stride, dilation=self.dilation,
                                             is_causal=self.is_causal, scale=self.scale)
        return self.proj_drop(self.proj(out.reshape(*lead, self.embed_dim)))

    def _project(self, x: Tensor, positions: Optional[Tensor] = None) -> Tuple[Tensor, Tensor, Tensor]:
        """Queries, keys and values, at the positions of the layout or at given ones."""
        # [..., 3, heads, head_dim]: q, k, v are strided views of one projection output
        q, k, v = self.qkv(x).unflatten(-1, (3, self.num_heads, self.head_dim)).unbind(-3)
        if self.rotary_theta is not None:
            q, k = rotary(q, k, axis_dims=self.rotary_axis_dims, theta=self.rotary_theta,
                          positions=positions, interleaved=self.rotary_interleaved)
        return q, k, v

    def extra_repr(self) -> str:
        rotary_repr = "" if self.rotary_theta is None else f", rotary_theta={self.rotary_theta}"
        return (f"head_dim={self.head_dim}, num_heads={self.num_heads}, "
                f"kernel_size={self.kernel_size}, stride={self.stride}, "
                f"dilation={self.dilation}, is_causal={self.is_causal}{rotary_repr}")


class NeighborhoodAttention1D(NeighborhoodAttentionGeneric):
    """1-D neighborhood attention layer on ``[batch, length, embed_dim]``."""

    def __init__(self, embed_dim: int, num_heads: int, kernel_size: Any, stride: Any = 1,
                 dilation: Any = 1, is_causal: Any = False, qkv_bias: bool = True,
                 qk_scale: Optional[float] = None, proj_drop: float = 0.0,
                 rotary_theta: Any = None, rotary_axis_dims: Optional[Sequence[int]] = None,
                 rotary_interleaved: bool = False):
        super().__init__(1, embed_dim, num_heads, kernel_size, stride, dilation, is_causal,
                         qkv_bias, qk_scale, proj_drop, rotary_theta, rotary_axis_dims,
                         rotary_interleaved)

    def _check_serving(self, x: Tensor) -> None:
        if not self.is_causal[0] or self.stride[0] != 1:
            raise ValueError("Serving with a cache needs a causal layer with stride 1, got "
                             f"is_causal={self.is_causal}, stride={self.stride}.")
        if x.dim() != 3 or x.shape[-1] != self.embed_dim:
            raise ValueError(f"Expected [batch, tokens, {self.embed_dim}], got {tuple(x.shape)}.")

    def prefill(self, x: Tensor, cache: KVCache, page_table: Tensor,
                counts: Optional[Tensor] = None) -> Tensor:
        """The layer on whole prompts ``[batch, tokens, embed_dim]``, whose keys and values go into the
        cache: token t of sequence b at position t, if ``t < counts[b]`` (prompts padded at their end;
        all without ``counts``). What lies behind a prompt may be anything, and the rows of the output there
        mean nothing. A dilated layer needs as many tokens as its window spans, like `forward`."""
        self._check_serving(x)
        _expect_cache(cache)
        counts = _per_sequence(cache, counts, x.shape[0], "counts")
        if counts is not None:
            # What lies behind a prompt may be anything: a NaN there has weight 0 for the prompt's rows, but the
            # tensor cores' products with 0 would keep it.
            behind = torch.arange(x.shape[1], device=x.device) >= counts[:, None]
            x = x.masked_fill(behind[..., None], 0.0)
        q, k, v = self._project(x)
        _refuse_grad("prefill()", q, k, v)
        if x.shape[1] < self.kernel_size[0] and self.dilation[0] == 1:      # a window over all of it
            out = attention(q, k, v, is_causal=True, scale=self.scale)
        else:
            out = neighborhood_attention_generic(q, k, v, kernel_size=self.kernel_size, stride=1,
                                                 dilation=self.dilation, is_causal=self.is_causal,
                                                 scale=self.scale)
        kv_cache_write(cache, k, v, page_table, None, counts)
        return self.proj_drop(self.proj(out.reshape(x.shape)))

    def decode(self, x: Tensor, cache: KVCache, page_table: Tensor, lengths: Tensor) -> Tensor:
        """The layer on the newest tokens ``[batch, tokens, embed_dim]`` of every sequence: they are written
        to positions ``lengths - tokens`` to ``lengths - 1`` and attend the cache (see `na1d_decode`).
        ``lengths`` (int32) counts the tokens of each sequence, these included."""
        self._check_serving(x)
        start = lengths - x.shape[1]
        positions = None
        if self.rotary_theta is not None:
            positions = (start[:, None] + torch.arange(x.shape[1], dtype=torch.int32,
                                                       device=x.device))[..., None]
        q, k, v = self._project(x, positions)
        kv_cache_write(cache, k, v, page_table, start)
        out = na1d_decode(q, cache, page_table, lengths, self.kernel_size[0], self.dilation[0], self.scale)
        return self.proj_drop(self.proj(out.reshape(x.shape)))


class NeighborhoodAttention2D(NeighborhoodAttentionGeneric):
    """2-D neighborhood attention layer on ``[batch, X, Y, embed_dim]``."""

    def __init__(self, embed_dim: int, num_heads: int, kernel_size: Any, stride: Any = 1,
                 dilation: Any = 1, is_causal: Any = False, qkv_bias: bool = True,
                 qk_scale: Optional[float] = None, proj_drop: float = 0.0,
                 rotary_theta: Any = None, rotary_axis_dims: Optional[Sequence[int]] = None,
                 rotary_interleaved: bool = False):
        super().__init__(2, embed_dim, num_heads, kernel_size, stride, dilation, is_causal,
                         qkv_bias, qk_scale, proj_drop, rotary_theta, rotary_axis_dims,
                         rotary_interleaved)


class NeighborhoodAttention3D(NeighborhoodAttentionGeneric):
    """3-D neighborhood attention layer on ``[batch, X, Y, Z, embed_dim]``."""

    def __init__(self, embed_dim: int, num_heads: int, kernel_size: Any, stride: Any = 1,
                 dilation: Any = 1, is_causal: Any = False, qkv_bias: bool = True,
                 qk_scale: Optional[float] = None, proj_drop: float = 0.0,
                 rotary_theta: Any = None, rotary_axis_dims: Optional[Sequence[int]] = None,
                 rotary_interleaved: bool = False):
        super().__init__(3, embed_dim, num_heads, kernel_size, stride, dilation, is_causal,
                         qkv_bias, qk_scale, proj_drop, rotary_theta, rotary_axis_dims,
                         rotary_interleaved)
