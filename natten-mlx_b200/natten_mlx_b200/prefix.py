"""``prefix_attention``: attention of a batch's queries to keys and values that all samples share (a long prompt,
conditioning tokens), read once for the whole batch, to stand beside the window of ``na1d``, ``na2d`` and ``na3d``.

The extra tokens of those operators belong to one sample each (src/natten_mlx/functional.py:71-104); here the queries of
a key/value head, over all samples, are the rows of one product.  The result merges with that of the window as
``merge_attentions`` does (src/natten_mlx/merge.py:20-68), in the same kernel when the window's result is handed in.
"""

from __future__ import annotations

import math
from typing import Optional, Tuple

import torch

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
    rank = query.dim() - 3
    if rank not in (1, 2, 3):
        raise ValueError("prefix_attention expects a query of shape [B, spatial..., heads, dim] with 1 to 3 spatial axes.")
    if prefix_keys.dim() != 3 or prefix_values.dim() != 3:
        raise ValueError("prefix_keys/prefix_values must be 3D: [P, heads_kv, dim].")
    if prefix_keys.shape != prefix_values.shape:
        raise ValueError(f"prefix_keys and prefix_values must have one shape, got {tuple(prefix_keys.shape)} and "
                         f"{tuple(prefix_values.shape)}.")
    heads_q, d = query.shape[-2:]
    if prefix_keys.shape[-1] != d:
        raise ValueError(f"Head dim must match: Q has {d}, the prefix has {prefix_keys.shape[-1]}.")
    if not 1 <= d <= 256:
        raise ValueError(f"prefix_attention takes head dims from 1 to 256, got {d}.")
    if prefix_keys.shape[1] < 1 or heads_q < 1 or heads_q % prefix_keys.shape[1] != 0:
        raise ValueError(f"heads_q ({heads_q}) must be divisible by heads_kv ({prefix_keys.shape[1]}).")
    tensors = [query, prefix_keys, prefix_values] + (list(window) if window is not None else [])
    if window is not None:
        if len(window) != 2:
            raise ValueError("window must be (output, lse).")
        out, lse = window
        if out.shape != query.shape or tuple(lse.shape) != tuple(query.shape[:-1]):
            raise ValueError(f"window must have the shapes {tuple(query.shape)} and {tuple(query.shape[:-1])}, got "
                             f"{tuple(out.shape)} and {tuple(lse.shape)}.")
        if out.dtype != query.dtype:
            raise ValueError(f"the window's output must have the query's dtype {query.dtype}, got {out.dtype}.")
    if any(t.dtype != query.dtype for t in tensors[:3]) or query.dtype not in _cuda._DTYPES:
        raise ValueError("query, prefix_keys and prefix_values must share a dtype of float32, float16 or bfloat16.")
    if scale is not None and not (float(scale) > 0.0 and math.isfinite(float(scale))):
        raise ValueError(f"scale must be positive and finite, got {scale}.")
    if torch.is_grad_enabled() and any(t.requires_grad for t in tensors):
        raise RuntimeError("prefix_attention computes no gradients: call it under torch.no_grad(), or detach its inputs")
    if not query.is_cuda:
        raise RuntimeError("natten_mlx_b200 runs on CUDA tensors only (there is no CPU path)")
    if any(t.device != query.device for t in tensors):
        raise ValueError("all tensors must be on one device")
    lens = None
    if prefix_lens is not None:
        if not torch.is_tensor(prefix_lens) or prefix_lens.dtype not in (torch.int32, torch.int64):
            raise ValueError("prefix_lens must be an int32 or int64 tensor.")
        if tuple(prefix_lens.shape) != (query.shape[0],):
            raise ValueError(f"prefix_lens must have shape ({query.shape[0]},), got {tuple(prefix_lens.shape)}.")
        if prefix_lens.device != query.device:
            raise ValueError("prefix_lens must be on the query's device")
        lens = prefix_lens.contiguous() if prefix_lens.dtype == torch.int32 else \
            prefix_lens.clamp(0, prefix_keys.shape[0]).to(torch.int32)
    w_out = w_lse = None
    if window is not None:
        w_out, w_lse = out, lse.to(torch.float32).contiguous()
    result = _cuda.prefix_forward(query, prefix_keys, prefix_values, scale, lens, w_out, w_lse)
    return result if return_lse else result[0]


__all__ = ["prefix_attention"]
