"""``rotary``: rotary positions over one to three axes, for the queries and keys of ``na1d``, ``na2d`` and ``na3d``.

One kernel turns q and k together.  It reads no table of angles: a block computes the cosines and sines of its tokens
once for all heads, from positions that wrap around at whole turns in 64-bit integers, so that far positions keep their
angles.  The gradient is the turn by the opposite angles.  No counterpart in the reference, whose positional term is the
relative bias of its allin1 ops (src/natten_mlx/extras/allin1/__init__.py:40-79).
"""

from __future__ import annotations

import math
from decimal import Decimal, localcontext
from functools import lru_cache
from typing import Optional, Sequence, Tuple, Union

import torch

from . import _lib
from .utils.params import normalize_tuple_param

_TWO_PI = Decimal("6.28318530717958647692528676655900576839433879875021164194988918461563281257241799725606965068")


def split_axis_dims(head_dim: int, axes: int) -> Tuple[int, ...]:
    """Channels of a head for each axis: equal even parts, what is left over goes to the first axis."""
    part = 2 * (head_dim // (2 * axes))
    return (head_dim - head_dim % 2 - part * (axes - 1),) + (part,) * (axes - 1)


def _phases(axis_dims: Tuple[int, ...], base: float, frequencies: Optional[Tuple[float, ...]]):
    """Angles per position as 64-bit fractions of a turn, computed with 50 digits."""
    with localcontext() as ctx:
        ctx.prec = 50
        if frequencies is not None:
            rad = [Decimal(f) for f in frequencies]
        else:
            rad = [Decimal(base) ** (Decimal(-2 * j) / Decimal(d)) for d in axis_dims for j in range(d // 2)]
        return [int((f / _TWO_PI * (1 << 64)).to_integral_value()) % (1 << 64) for f in rad]


@lru_cache(maxsize=256)
def _spec(head_dim: int, axes: int, axis_dims: Optional[Tuple[int, ...]], base: float,
          frequencies: Optional[Tuple[float, ...]], interleaved: bool):
    """What a call hands to the library, checked and computed once for each choice of arguments."""
    dims = split_axis_dims(head_dim, axes) if axis_dims is None else axis_dims
    if not 1 <= len(dims) <= 3:
        raise ValueError(f"axis_dims must have 1 to 3 entries, got {dims}")
    if any(not isinstance(d, int) or d < 0 or d % 2 for d in dims) or not 2 <= sum(dims) <= min(head_dim, 512):
        raise ValueError(f"axis_dims must be even, not negative and sum to 2..{min(head_dim, 512)}, got {dims}")
    if not (base > 0.0 and math.isfinite(base)):
        raise ValueError(f"base must be positive and finite, got {base}")
    if frequencies is not None and (len(frequencies) != sum(dims) // 2 or not all(math.isfinite(f) for f in frequencies)):
        raise ValueError(f"frequencies must be {sum(dims) // 2} finite numbers, got {len(frequencies)}")
    return _lib.binding().RotarySpec(list(dims), _phases(dims, base, frequencies), interleaved)


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
    if not 1 <= rank <= 3:
        raise ValueError("rotary expects query and key with one of the shapes [B, L, heads, dim], [B, H, W, heads, dim], "
                         "[B, D, H, W, heads, dim]")
    origin, start = (), None
    if positions is not None:
        if offsets is not None:
            raise ValueError("offsets and positions cannot be combined")
        if not torch.is_tensor(positions) or positions.dim() < 1:
            raise ValueError("positions must be an int32 or int64 tensor with a last axis of coordinates")
    elif torch.is_tensor(offsets):
        start = offsets
    elif offsets is not None:
        origin = normalize_tuple_param(offsets, rank, "offsets")
        if not all(isinstance(o, int) and -2 ** 62 < o < 2 ** 62 for o in origin):
            raise ValueError(f"offsets must be integers, got {offsets!r}")
    spec = _spec(query.shape[-1], rank if positions is None else positions.shape[-1],
                 None if axis_dims is None else tuple(axis_dims), float(base),
                 None if frequencies is None else tuple(float(f) for f in frequencies), bool(interleaved))
    return _lib.binding().rotary(query, key, spec, origin, start, positions)


__all__ = ["rotary", "split_axis_dims"]
