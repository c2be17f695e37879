"""``prefix_attention``: attention of a batch's queries to keys and values that all samples share (a long prompt,
conditioning tokens), read once for the whole batch, to stand beside the window of ``na1d``, ``na2d`` and ``na3d``.

The extra tokens of those operators belong to one sample each (src/natten_mlx/functional.py:71-104); here the queries of
a key/value head, over all samples, are the rows of one product.  The result merges with that of the window as
``merge_attentions`` does (src/natten_mlx/merge.py:20-68), in the same kernel when the window's result is handed in.
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _lib
from ._core import cuda as _cuda


def prefix_attention(query: torch.Tensor, prefix_keys: torch.Tensor, prefix_values: torch.Tensor,
                     scale: Optional[float] = None, return_lse: bool = False, *,
                     prefix_lens: Optional[torch.Tensor] = None,
                     window: Optional[Tuple[torch.Tensor, torch.Tensor]] = None):
    """``softmax(scale * query . prefix_keys) . prefix_values``, the prefix shared by every sample of the batch.

    ``query`` ``[B, spatial..., heads_q, D]`` (one to three spatial axes; a single new token is ``[B, 1, heads_q, D]``),
    ``prefix_keys`` and ``prefix_values`` ``[P, heads_kv, D]`` with ``heads_kv`` dividing ``heads_q``; ``D`` up to 256.
    ``prefix_lens`` (int32/int64 ``[B]``) lets a sample see only the first tokens of the prefix (values are clamped to
    0..P); what the prefix holds past a sample's length does not reach its result.  A query that sees no token gets
    zeros, and ``-inf`` as its log-sum-exp.

    ``window`` is ``(output, lse)`` of the same queries over other keys, as ``na1d(..., return_lse=True)`` returns them:
    the result is then that over both sets of keys, without a pass of ``merge_attentions``.

    Returns ``[B, spatial..., heads_q, D]``, or ``(output, lse)`` with the float32 log-sum-exp
    ``[B, spatial..., heads_q]`` when ``return_lse`` is set.  bfloat16 and float16 with ``D`` a multiple of 8 up to 128 run
    on the tensor cores.  Forward only, for serving: inputs that need gradients are refused.
    """
    if window is not None and len(window) != 2:
        raise ValueError("window must be (output, lse).")
    if prefix_lens is not None and not torch.is_tensor(prefix_lens):
        raise ValueError("prefix_lens must be an int32 or int64 tensor.")
    out, lse = (None, None) if window is None else window
    result = _lib.binding().prefix(query, prefix_keys, prefix_values, scale, prefix_lens, out, lse, _cuda._PATHS[_cuda._fused_path])
    return result if return_lse else result[0]


__all__ = ["prefix_attention"]
