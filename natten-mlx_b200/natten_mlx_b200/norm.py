"""``layer_norm``: layer norm over the last axis, for the input of a block and for the heads of q and k.

One kernel reads every element once; the backward is one kernel for the input's gradient and the sums of the weights'
gradients, and a small one that joins those sums in a fixed order.  The reference leaves the norm to its array library;
the layer between two norms is src/natten_mlx/nn/na2d.py:14-154.
"""

from __future__ import annotations

from typing import Optional

import torch

from . import _lib


def layer_norm(input: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               eps: float = 1e-5) -> torch.Tensor:
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last axis, statistics in float32.

    ``input`` ``[..., C]`` is float32, float16 or bfloat16; ``weight`` and ``bias`` ``[C]`` (either may be None) have its
    dtype or are float32, both alike.  The result has the input's dtype and is dense.  An input whose rows follow one
    or two strides, such as the queries inside the output of a fused q/k/v projection, is read where it lies.
    Differentiable (once) in all three; the weights' gradients do not depend on the order in which blocks finish.
    """
    return (_lib._binding or _lib.binding()).layer_norm(input, weight, bias, eps)


__all__ = ["layer_norm"]
