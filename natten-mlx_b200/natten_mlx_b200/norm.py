"""``layer_norm``: layer norm over the last axis, for the input of a block and for the heads of q and k.

One kernel reads every element once; the backward is one kernel for the input's gradient and the sums of the weights'
gradients, and a small one that joins those sums in a fixed order.  The reference leaves the norm to its array library;
the layer between two norms is src/natten_mlx/nn/na2d.py:14-154.
"""

from __future__ import annotations

import math
from typing import Optional

import torch

from . import autograd as _ag
from ._core import cuda as _cuda


def _check_vector(name, t, x):
    if t.dim() != 1 or t.shape[0] != x.shape[-1]:
        raise ValueError(f"{name} must have shape ({x.shape[-1]},), got {tuple(t.shape)}")
    if t.dtype != x.dtype and t.dtype != torch.float32:
        raise ValueError(f"{name} must have the input's dtype {x.dtype} or float32, got {t.dtype}")
    if t.device != x.device:
        raise ValueError(f"{name} must be on the input's device {x.device}, got {t.device}")
    return t if t.is_contiguous() else t.contiguous()


def layer_norm(input: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               eps: float = 1e-5) -> torch.Tensor:
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last axis, statistics in float32.

    ``input`` ``[..., C]`` is float32, float16 or bfloat16; ``weight`` and ``bias`` ``[C]`` (either may be None) have its
    dtype or are float32, both alike.  The result has the input's dtype and is dense.  An input whose rows follow one
    or two strides, such as the queries inside the output of a fused q/k/v projection, is read where it lies.
    Differentiable (once) in all three; the weights' gradients do not depend on the order in which blocks finish.
    """
    if not input.is_cuda:
        raise RuntimeError("natten_mlx_b200 runs on CUDA tensors only (there is no CPU path)")
    if input.dtype not in _cuda._DTYPES:
        raise ValueError(f"unsupported dtype {input.dtype}; expected float32, float16 or bfloat16")
    if input.dim() < 1 or input.shape[-1] < 1:
        raise ValueError(f"layer_norm expects [..., C] with C >= 1, got {tuple(input.shape)}")
    eps = float(eps)
    if not (eps >= 0.0 and math.isfinite(eps)):
        raise ValueError(f"eps must be finite and not negative, got {eps}")
    if weight is not None:
        weight = _check_vector("weight", weight, input)
    if bias is not None:
        bias = _check_vector("bias", bias, input)
        if weight is not None and bias.dtype != weight.dtype:
            raise ValueError(f"weight and bias must have one dtype, got {weight.dtype} and {bias.dtype}")
    if torch.is_grad_enabled() and (input.requires_grad or (weight is not None and weight.requires_grad)
                                    or (bias is not None and bias.requires_grad)):
        return _ag.layer_norm_with_grad(input, weight, bias, eps)
    return _cuda.layer_norm_forward(input, weight, bias, eps)[0]


__all__ = ["layer_norm"]
