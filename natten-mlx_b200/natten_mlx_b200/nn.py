"""torch modules around the fused operators: the immediate callers of the hot path.

Behaviour follows the reference's MLX modules
(``src/natten_mlx/nn/na1d.py:14-154``, ``nn/na2d.py:14-154``, ``nn/na3d.py:14-158``):
channels-last input ``[B, spatial..., C]``; one fused ``qkv`` projection, or
``q_proj`` + ``kv_proj`` when ``num_kv_heads`` differs from ``num_heads``
(grouped-query attention); the fused operator on heads-last tensors
``[B, spatial..., heads, head_dim]``; with ``attn_drop > 0`` the split path
(QK → softmax → dropout → AV); with per-sample ``spatial_sizes`` the
variable-length operator; then the output projection and its dropout.

One class serves the three ranks.  The head split is a ``view`` of the projection
output: channel order ``(3, heads, head_dim)`` of the fused projection makes
q, k and v strided views of one buffer, and the operators take them without a
copy when they are already dense (q/k/v of the fused projection are not, so one
gather per tensor remains, as in the reference's ``mx.split``).

What the reference's modules leave to the model around them is here as well: ``LayerNorm``, and as options of the
attention modules the norm of every head of q and k (``qk_norm``), rotary positions over the spatial axes
(``rotary``), both of which read q and k where they lie in the projection's output, and in ``forward`` keys and values
that the whole batch shares (``prefix``).
"""

from __future__ import annotations

from typing import Optional, Sequence, Union

import torch
from torch import nn

from . import functional as F
from .norm import layer_norm
from .positions import rotary as _rotary
from .prefix import prefix_attention
from .utils.params import normalize_kernel_size, normalize_tuple_param

_IntOrSeq = Union[int, Sequence[int]]
_BoolOrSeq = Union[bool, Sequence[bool]]

_FUSED = {1: F.na1d, 2: F.na2d, 3: F.na3d}
_QK = {1: F.na1d_qk, 2: F.na2d_qk, 3: F.na3d_qk}
_AV = {1: F.na1d_av, 2: F.na2d_av, 3: F.na3d_av}
_VARLEN = {1: F.na1d_varlen, 2: F.na2d_varlen, 3: F.na3d_varlen}
_LAYOUT = {1: "[B, L, C]", 2: "[B, H, W, C]", 3: "[B, D, H, W, C]"}


class LayerNorm(nn.Module):
    """Layer norm over the last axis (``natten_mlx_b200.layer_norm``).  ``weight`` and ``bias`` keep their own dtype: the
    input's, or float32 beside inputs of 16 bits."""

    def __init__(self, dim: int, eps: float = 1e-5, elementwise_affine: bool = True, bias: bool = True, device=None,
                 dtype=None):
        super().__init__()
        if dim <= 0:
            raise ValueError(f"dim must be positive, got {dim}")
        self.dim, self.eps = int(dim), float(eps)
        kw = dict(device=device, dtype=dtype)
        self.weight = nn.Parameter(torch.ones(self.dim, **kw)) if elementwise_affine else None
        self.bias = nn.Parameter(torch.zeros(self.dim, **kw)) if elementwise_affine and bias else None

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if x.shape[-1] != self.dim:
            raise ValueError(f"Input channel dim ({x.shape[-1]}) must match dim ({self.dim})")
        return layer_norm(x, self.weight, self.bias, self.eps)

    def extra_repr(self) -> str:
        return f"{self.dim}, eps={self.eps}, elementwise_affine={self.weight is not None}, bias={self.bias is not None}"


class _NeighborhoodAttention(nn.Module):
    rank = 0

    def __init__(self, embed_dim: int, num_heads: int, kernel_size: _IntOrSeq, stride: _IntOrSeq = 1,
                 dilation: _IntOrSeq = 1, is_causal: _BoolOrSeq = False, num_kv_heads: Optional[int] = None,
                 qkv_bias: bool = True, qk_scale: Optional[float] = None, attn_drop: float = 0.0,
                 proj_drop: float = 0.0, device=None, dtype=None, *, qk_norm: bool = False, rotary: bool = False,
                 rotary_base: float = 10000.0):
        super().__init__()
        if embed_dim <= 0:
            raise ValueError(f"embed_dim must be positive, got {embed_dim}")
        if num_heads <= 0:
            raise ValueError(f"num_heads must be positive, got {num_heads}")
        if embed_dim % num_heads != 0:
            raise ValueError("embed_dim must be divisible by num_heads")
        kv_heads = num_heads if num_kv_heads is None else int(num_kv_heads)
        if kv_heads <= 0 or num_heads % kv_heads != 0:
            raise ValueError(f"num_heads ({num_heads}) must be divisible by num_kv_heads ({kv_heads})")
        rank = self.rank
        self.embed_dim, self.num_heads, self.num_kv_heads = int(embed_dim), int(num_heads), kv_heads
        self.head_dim = embed_dim // num_heads
        self.kernel_size = normalize_kernel_size(kernel_size, rank)
        self.stride = tuple(int(s) for s in normalize_tuple_param(stride, rank, "stride"))
        self.dilation = tuple(int(d) for d in normalize_tuple_param(dilation, rank, "dilation"))
        self.is_causal = tuple(bool(c) for c in normalize_tuple_param(is_causal, rank, "is_causal"))
        self.scale = float(qk_scale) if qk_scale is not None else self.head_dim ** -0.5
        kw = dict(device=device, dtype=dtype)
        if kv_heads != num_heads:
            self.q_proj = nn.Linear(embed_dim, num_heads * self.head_dim, bias=qkv_bias, **kw)
            self.kv_proj = nn.Linear(embed_dim, 2 * kv_heads * self.head_dim, bias=qkv_bias, **kw)
            self.qkv = None
        else:
            self.qkv = nn.Linear(embed_dim, 3 * embed_dim, bias=qkv_bias, **kw)
            self.q_proj = self.kv_proj = None
        self.q_norm = LayerNorm(self.head_dim, **kw) if qk_norm else None
        self.k_norm = LayerNorm(self.head_dim, **kw) if qk_norm else None
        if rotary and self.head_dim < 2 * rank:
            raise ValueError(f"rotary needs two channels of a head for each axis, head_dim is {self.head_dim}")
        self.rotary, self.rotary_base = bool(rotary), float(rotary_base)
        self.attn_drop_rate = float(attn_drop)
        self.attn_drop = nn.Dropout(self.attn_drop_rate) if self.attn_drop_rate > 0.0 else None
        self.proj = nn.Linear(embed_dim, embed_dim, **kw)
        self.proj_drop_rate = float(proj_drop)
        self.proj_drop = nn.Dropout(self.proj_drop_rate) if self.proj_drop_rate > 0.0 else None

    def _heads(self, x: torch.Tensor):
        lead = tuple(x.shape[:-1])
        if self.qkv is not None:
            qkv = self.qkv(x).view(*lead, 3, self.num_heads, self.head_dim)
            return qkv.select(-3, 0), qkv.select(-3, 1), qkv.select(-3, 2)
        q = self.q_proj(x).view(*lead, self.num_heads, self.head_dim)
        kv = self.kv_proj(x).view(*lead, 2, self.num_kv_heads, self.head_dim)
        return q, kv.select(-3, 0), kv.select(-3, 1)

    def forward(self, x: torch.Tensor, spatial_sizes: Optional[torch.Tensor] = None, *, offsets=None, prefix=None,
                prefix_lens: Optional[torch.Tensor] = None) -> torch.Tensor:
        """``offsets``: where the positions start, as in ``rotary`` (modules built with ``rotary``).  ``prefix``: keys and
        values ``[P, num_kv_heads, head_dim]`` that every query of the batch attends to besides its window, the samples
        to their first ``prefix_lens`` tokens of them; they enter as given, and without gradients (serving)."""
        rank = self.rank
        if offsets is not None and not self.rotary:
            raise ValueError("offsets need a module built with rotary=True")
        if prefix_lens is not None and prefix is None:
            raise ValueError("prefix_lens needs a prefix")
        if prefix is not None and (spatial_sizes is not None or (self.attn_drop is not None and self.training)):
            raise ValueError("a prefix cannot be combined with spatial_sizes or with attention dropout in training")
        if x.dim() != rank + 2:
            raise ValueError(f"Expected input shape {_LAYOUT[rank]}, got {tuple(x.shape)}")
        if x.shape[-1] != self.embed_dim:
            raise ValueError(f"Input channel dim ({x.shape[-1]}) must match embed_dim ({self.embed_dim})")
        q, k, v = self._heads(x)
        if self.q_norm is not None:
            q, k = self.q_norm(q), self.k_norm(k)
        if self.rotary:
            q, k = _rotary(q, k, base=self.rotary_base, offsets=offsets)
        if prefix is not None:
            window = _FUSED[rank](q, k, v, kernel_size=self.kernel_size, stride=self.stride, dilation=self.dilation,
                                  is_causal=self.is_causal, scale=self.scale, return_lse=True)
            rows = q[(slice(None),) + tuple(slice(None, None, st) for st in self.stride)]
            out = prefix_attention(rows, prefix[0], prefix[1], self.scale, prefix_lens=prefix_lens, window=window)
        elif spatial_sizes is not None:
            out = _VARLEN[rank](q, k, v, spatial_sizes, kernel_size=self.kernel_size, dilation=self.dilation,
                                scale=self.scale)
        elif self.attn_drop is not None:
            logits = _QK[rank](q, k, kernel_size=self.kernel_size, dilation=self.dilation, stride=self.stride,
                               is_causal=self.is_causal, scale=self.scale)
            attn = self.attn_drop(torch.softmax(logits, dim=-1))
            out = _AV[rank](attn, v, kernel_size=self.kernel_size, dilation=self.dilation, stride=self.stride,
                            is_causal=self.is_causal)
        else:
            out = _FUSED[rank](q, k, v, kernel_size=self.kernel_size, stride=self.stride, dilation=self.dilation,
                               is_causal=self.is_causal, scale=self.scale)
        out = self.proj(out.reshape(*out.shape[:-2], self.embed_dim))
        return out if self.proj_drop is None else self.proj_drop(out)

    def extra_repr(self) -> str:
        return (f"embed_dim={self.embed_dim}, num_heads={self.num_heads}, num_kv_heads={self.num_kv_heads}, "
                f"kernel_size={self.kernel_size}, stride={self.stride}, dilation={self.dilation}, "
                f"is_causal={self.is_causal}")


class NeighborhoodAttention1D(_NeighborhoodAttention):
    """Input ``[B, L, C]`` → output ``[B, ceil(L / stride), C]``; ``forward(x, seq_lens)`` for ragged batches."""
    rank = 1


class NeighborhoodAttention2D(_NeighborhoodAttention):
    """Input ``[B, H, W, C]`` → output ``[B, ceil(H / stride_h), ceil(W / stride_w), C]``."""
    rank = 2


class NeighborhoodAttention3D(_NeighborhoodAttention):
    """Input ``[B, D, H, W, C]`` → output with every spatial extent divided (rounding up) by its stride."""
    rank = 3


__all__ = ["LayerNorm", "NeighborhoodAttention1D", "NeighborhoodAttention2D", "NeighborhoodAttention3D"]
