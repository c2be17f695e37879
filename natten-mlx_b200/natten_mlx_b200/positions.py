"""``rotary``: rotary positions over one to three axes, for the queries and keys of ``na1d``, ``na2d`` and ``na3d``.

One kernel turns q and k together.  It reads no table of angles: a block computes the cosines and sines of its tokens
once for all heads, from positions that wrap around at whole turns in 64-bit integers, so that far positions keep their
angles.  The gradient is the turn by the opposite angles.  No counterpart in the reference, whose positional term is the
relative bias of its allin1 ops (src/natten_mlx/extras/allin1/__init__.py:40-79).
"""

from __future__ import annotations

import ctypes
import math
from decimal import Decimal, localcontext
from functools import lru_cache
from typing import Optional, Sequence, Tuple, Union

import torch

from . import autograd as _ag
from ._core import cuda as _cuda
from .utils.params import normalize_tuple_param

_TWO_PI = Decimal("6.28318530717958647692528676655900576839433879875021164194988918461563281257241799725606965068")
_NO_ORIGIN = (ctypes.c_int64 * 3)()
_LAYOUTS = {1: "[B, L, heads, dim]", 2: "[B, H, W, heads, dim]", 3: "[B, D, H, W, heads, dim]"}


def split_axis_dims(head_dim: int, axes: int) -> Tuple[int, ...]:
    """Channels of a head for each axis: equal even parts, what is left over goes to the first axis."""
    part = 2 * (head_dim // (2 * axes))
    return (head_dim - head_dim % 2 - part * (axes - 1),) + (part,) * (axes - 1)


@lru_cache(maxsize=128)
def _phases(axis_dims: Tuple[int, ...], base: float, frequencies: Optional[Tuple[float, ...]]):
    """Angles per position as 64-bit fractions of a turn, computed with 50 digits."""
    with localcontext() as ctx:
        ctx.prec = 50
        if frequencies is not None:
            rad = [Decimal(f) for f in frequencies]
        else:
            rad = [Decimal(base) ** (Decimal(-2 * j) / Decimal(d)) for d in axis_dims for j in range(d // 2)]
        values = [int((f / _TWO_PI * (1 << 64)).to_integral_value()) % (1 << 64) for f in rad]
    return (ctypes.c_uint64 * len(values))(*values)


@lru_cache(maxsize=128)
def _spec(axis_dims: Tuple[int, ...], base: float, frequencies: Optional[Tuple[float, ...]], interleaved: bool):
    """What a call hands to the library, once for each choice of arguments."""
    dims = (ctypes.c_int32 * 3)(*axis_dims, *(0,) * (3 - len(axis_dims)))
    return len(axis_dims), dims, _phases(axis_dims, base, frequencies), int(interleaved)


def _check_positions(name, t, shape_ok, expected, query):
    if not torch.is_tensor(t) or t.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"{name} must be an int32 or int64 tensor, got {t.dtype if torch.is_tensor(t) else type(t)}")
    if not shape_ok:
        raise ValueError(f"{name} must have shape {expected}, got {tuple(t.shape)}")
    if t.device != query.device:
        raise ValueError(f"{name} must be on the query's device {query.device}, got {t.device}")
    return t.contiguous()


def rotary(query: torch.Tensor, key: torch.Tensor, axis_dims: Optional[Sequence[int]] = None, *, base: float = 10000.0,
           interleaved: bool = True, offsets: Union[None, int, Sequence[int], torch.Tensor] = None,
           positions: Optional[torch.Tensor] = None, frequencies: Optional[Sequence[float]] = None):
    """Turns the channel pairs of every head by angles that grow with the token's position; returns ``(query, key)``.

    ``query`` ``[B, spatial..., heads_q, D]`` and ``key`` ``[B, spatial..., heads_kv, D]`` (one to three spatial axes, the
    layouts of ``na1d``, ``na2d`` and ``na3d``).  The first ``sum(axis_dims)`` channels of a head are rotated,
    ``axis_dims[a]`` (even) of them by the position on axis ``a``; the default shares all channels among the spatial
    axes.  Pair ``j`` of an axis turns by ``position * base ** (-2 j / axis_dims[a])`` radians; ``frequencies`` gives the
    radians per position of all pairs instead, axis by axis.  Pairs are neighbouring channels, or with
    ``interleaved=False`` channel ``p`` of the first and of the second half of the rotated channels.

    Positions are the indices on the spatial axes, plus ``offsets``: an integer, one per axis, or an int32/int64 tensor
    ``[B, rank]`` on the device with a start for each sample (a step of cached decoding).  Or ``positions``, int32/int64
    ``[B or 1, spatial..., len(axis_dims)]`` on the device, gives the position of every token on one to three axes of
    any meaning.  Any position that fits 32 bits, negative ones too, keeps its angle.

    Inputs may be strided views, such as q and k inside a fused projection; the results are dense.  Differentiable
    (once) in query and key.
    """
    rank = query.dim() - 3
    if rank not in (1, 2, 3) or key.dim() != query.dim():
        raise ValueError("rotary expects query and key with one of the shapes " + ", ".join(_LAYOUTS.values()))
    if query.shape[:-2] != key.shape[:-2]:
        raise ValueError(f"Batch and spatial dimensions must match: Q={tuple(query.shape[:-2])}, K={tuple(key.shape[:-2])}.")
    head_dim = query.shape[-1]
    if key.shape[-1] != head_dim:
        raise ValueError(f"Head dim must match: Q has {head_dim}, K has {key.shape[-1]}.")
    if query.dtype not in _cuda._DTYPES or key.dtype != query.dtype:
        raise ValueError(f"query and key must share a dtype of float32, float16 or bfloat16, got {query.dtype} and {key.dtype}")
    if not query.is_cuda:
        raise RuntimeError("natten_mlx_b200 runs on CUDA tensors only (there is no CPU path)")
    if key.device != query.device:
        raise ValueError("query and key must be on one device")
    axes = rank if positions is None or axis_dims is not None else positions.shape[-1]
    dims = split_axis_dims(head_dim, axes) if axis_dims is None else tuple(int(d) for d in axis_dims)
    if not 1 <= len(dims) <= 3:
        raise ValueError(f"axis_dims must have 1 to 3 entries, got {dims}")
    if any(d < 0 or d % 2 for d in dims) or not 2 <= sum(dims) <= min(head_dim, 512):
        raise ValueError(f"axis_dims must be even, not negative and sum to 2..{min(head_dim, 512)}, got {dims}")
    base = float(base)
    if not (base > 0.0 and math.isfinite(base)):
        raise ValueError(f"base must be positive and finite, got {base}")
    if frequencies is not None:
        frequencies = tuple(float(f) for f in frequencies)
        if len(frequencies) != sum(dims) // 2 or not all(math.isfinite(f) for f in frequencies):
            raise ValueError(f"frequencies must be {sum(dims) // 2} finite numbers, got {len(frequencies)}")
    origin, start = _NO_ORIGIN, None
    if positions is not None:
        if offsets is not None:
            raise ValueError("offsets and positions cannot be combined")
        lead = tuple(query.shape[1:-2])
        ok = torch.is_tensor(positions) and positions.dim() == rank + 2 and positions.shape[0] in (1, query.shape[0]) \
            and tuple(positions.shape[1:-1]) == lead and positions.shape[-1] == len(dims)
        positions = _check_positions("positions", positions, ok, f"[{query.shape[0]} or 1, {lead}, {len(dims)}]", query)
    else:
        if len(dims) != rank:
            raise ValueError(f"axis_dims must have an entry for each of the {rank} spatial axes, got {dims}")
        if torch.is_tensor(offsets):
            start = _check_positions("offsets", offsets, tuple(offsets.shape) == (query.shape[0], rank),
                                     f"[{query.shape[0]}, {rank}]", query)
        elif offsets is not None:
            given = normalize_tuple_param(offsets, rank, "offsets")
            if not all(isinstance(o, int) and -2 ** 62 < o < 2 ** 62 for o in given):
                raise ValueError(f"offsets must be integers, got {offsets!r}")
            origin = (ctypes.c_int64 * 3)(*given, *(0,) * (3 - rank))
    spec = _spec(dims, base, frequencies, bool(interleaved))
    if torch.is_grad_enabled() and (query.requires_grad or key.requires_grad):
        return _ag.rotary_with_grad(query, key, spec, origin, start, positions)
    return _cuda.rotary(query, key, spec, origin, start, positions)


__all__ = ["rotary", "split_axis_dims"]
