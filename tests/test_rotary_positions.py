"""``rotary``: values and gradients against complex products in 64 bits, layouts, sources of positions, far positions,
strided inputs, refusals.

Tolerance.  A result is a cos - b sin.  The angle, a fraction of a turn, is truncated to 2^-32 of a turn and rounded to 24
bits of at most half a turn: 1.9e-7 radians; cosine and sine are within two units of the last place, 1.2e-7 below 1;
the products and their sum add 2^-23 (|a| + |b|).  Together less than 2^-21 (|a| + |b|), and the result is rounded once.
For 16-bit types the angle is rounded once more, as radians (1.9e-7), and cosine and sine are off by at most 2^-21.19 and
2^-21.41: 1.9e-7 + 1.9e-7 + 4.2e-7 + 1.2e-7 = 9.2e-7, less than 2^-20 (9.5e-7)."""

from __future__ import annotations

import ctypes
import math
from fractions import Fraction

import pytest
import torch

import natten_mlx_b200 as nb
from natten_mlx_b200 import _lib
from natten_mlx_b200.positions import _phases, split_axis_dims

DEV = "cuda"
U = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TURN = {torch.float32: 2.0 ** -21, torch.float16: 2.0 ** -20, torch.bfloat16: 2.0 ** -20}


def _rand(shape, seed, dtype):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed), dtype=torch.float64).to(dtype)


def _turns(positions, dims, base=10000.0, freqs=None):
    """Fractions of a turn [.., pairs] in float64, reduced exactly: positions is an int64 tensor [.., axes]."""
    cols = []
    p = 0
    for a, d in enumerate(dims):
        for j in range(d // 2):
            f = base ** (-2.0 * j / d) if freqs is None else freqs[p]
            p += 1
            # the product of a 32-bit position and a double is exact as a fraction
            turn = Fraction(f) / Fraction(math.pi + 1.2246467991473532e-16 - 1.2246467991473532e-16) / 2
            vals = [float((int(x) * turn) % 1) for x in positions[..., a].reshape(-1).tolist()]
            cols.append(torch.tensor(vals, dtype=torch.float64))
    return torch.stack(cols, -1).reshape(*positions.shape[:-1], -1)


def _turned(t, turns, interleaved, sign=1.0):
    """(result, |a| + |b| of each channel's pair) in float64; turns [B, spatial..., pairs]."""
    t = t.detach().double().cpu()
    n = turns.shape[-1]
    unit = torch.polar(torch.ones_like(turns), turns * (2 * math.pi * sign)).unsqueeze(-2)
    out, size = t.clone(), t.abs().clone()
    if interleaved:
        a, b = t[..., 0:2 * n:2], t[..., 1:2 * n:2]
    else:
        a, b = t[..., :n], t[..., n:2 * n]
    z = torch.complex(a, b) * unit
    both = a.abs() + b.abs()
    if interleaved:
        out[..., 0:2 * n:2], out[..., 1:2 * n:2] = z.real, z.imag
        size[..., 0:2 * n:2], size[..., 1:2 * n:2] = both, both
    else:
        out[..., :n], out[..., n:2 * n] = z.real, z.imag
        size[..., :n], size[..., n:2 * n] = both, both
    return out, size, 2 * n


def _check(got, t, turns, interleaved, sign=1.0, angle_err=0.0):
    want, size, width = _turned(t, turns, interleaved, sign)
    got64 = got.detach().double().cpu()
    assert got.dtype == t.dtype and got.shape == t.shape and got.is_contiguous()
    bound = U[got.dtype] * want.abs() + size * (TURN[got.dtype] + angle_err) + (2.0 ** -25 if got.dtype == torch.float16 else 0.0)
    off = (got64 - want).abs()
    assert bool((off <= bound).all()), f"{float((off / bound).max()):.3g} of the bound"
    assert torch.equal(got[..., width:].cpu(), t.detach()[..., width:].cpu())


def _grid(lead, origin=None, offsets=None):
    axes = [torch.arange(n) for n in lead[1:]]
    pos = torch.stack(torch.meshgrid(*axes, indexing="ij"), -1).unsqueeze(0).repeat(lead[0], *([1] * len(lead))).long()
    if origin is not None:
        pos = pos + torch.tensor(origin)
    if offsets is not None:
        pos = pos + offsets.long().cpu().reshape([lead[0]] + [1] * (len(lead) - 1) + [-1])
    return pos


def _case(q, k, turns, call, interleaved, angle_err=0.0):
    ql, kl = q.to(DEV).detach().requires_grad_(True), k.to(DEV).detach().requires_grad_(True)
    yq, yk = call(ql, kl)
    _check(yq, ql, turns, interleaved, 1.0, angle_err)
    _check(yk, kl, turns, interleaved, 1.0, angle_err)
    gq, gk = _rand(q.shape, 71, q.dtype).to(DEV), _rand(k.shape, 72, k.dtype).to(DEV)
    dq, dk = torch.autograd.grad((yq, yk), (ql, kl), (gq, gk))
    _check(dq, gq, turns, interleaved, -1.0, angle_err)
    _check(dk, gk, turns, interleaved, -1.0, angle_err)


CASES = [
    # batch and extents, heads, kv heads, head dim, axis dims
    ((1, 1), 1, 1, 2, (2,)), ((2, 7), 3, 1, 6, (4,)), ((1, 300), 8, 2, 64, (64,)), ((3, 33), 4, 4, 128, (96,)),
    ((2, 5, 9), 4, 4, 32, (16, 16)), ((1, 17, 4), 6, 3, 24, (10, 14)), ((2, 3, 5), 2, 2, 48, (2, 30)),
    ((2, 3, 4, 5), 4, 4, 64, (24, 20, 20)), ((1, 2, 6, 7), 5, 1, 80, (16, 24, 24)), ((1, 2, 3, 2), 2, 2, 512, (200, 156, 156)),
    ((2, 3, 4, 5), 2, 1, 16, (8, 0, 4)), ((70, 1), 16, 4, 64, (64,)),
]


@pytest.mark.gpu
@pytest.mark.parametrize("lead,hq,hk,d,dims", CASES)
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_grid_positions(lead, hq, hk, d, dims, interleaved, dtype):
    q, k = _rand(lead + (hq, d), 1, dtype), _rand(lead + (hk, d), 2, dtype)
    _case(q, k, _turns(_grid(lead), dims), lambda a, b: nb.rotary(a, b, dims, interleaved=interleaved), interleaved)


@pytest.mark.gpu
@pytest.mark.parametrize("lead,hq,hk,d,dims", [
    ((1, 5, 4), 5, 4, 512, (256, 256)),      # a token's channels take several passes of the block, fewer threads than pairs
    ((1, 700), 40, 9, 128, (128,)), ((2, 40, 41), 3, 2, 72, (36, 36)), ((1, 20011), 1, 1, 2, (2,)),
])
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_wide_tokens_and_long_runs(lead, hq, hk, d, dims, interleaved, dtype):
    q, k = _rand(lead + (hq, d), 1, dtype), _rand(lead + (hk, d), 2, dtype)
    _case(q, k, _turns(_grid(lead), dims), lambda a, b: nb.rotary(a, b, dims, interleaved=interleaved), interleaved)
    # heads that start off the 16-byte boundaries take the pairs one by one
    q1, k1 = (_rand(lead + (h, d + 1), 3, dtype).to(DEV)[..., 1:] for h in (hq, hk))
    yq, yk = nb.rotary(q1, k1, dims, interleaved=interleaved)
    _check(yq, q1, _turns(_grid(lead), dims), interleaved)
    _check(yk, k1, _turns(_grid(lead), dims), interleaved)


@pytest.mark.gpu
def test_defaults_share_the_channels_among_the_axes():
    assert split_axis_dims(64, 3) == (24, 20, 20) and split_axis_dims(128, 3) == (44, 42, 42)
    assert split_axis_dims(32, 2) == (16, 16) and split_axis_dims(64, 1) == (64,) and split_axis_dims(7, 3) == (2, 2, 2)
    q, k = _rand((2, 3, 4, 5, 2, 64), 1, torch.float32), _rand((2, 3, 4, 5, 2, 64), 2, torch.float32)
    _case(q, k, _turns(_grid((2, 3, 4, 5)), (24, 20, 20)), nb.rotary, True)
    pos = torch.randint(0, 50, (1, 3, 4, 5, 2), generator=torch.Generator().manual_seed(1))
    _case(q, k, _turns(pos.expand(2, 3, 4, 5, 2), (32, 32)), lambda a, b: nb.rotary(a, b, positions=pos.to(DEV)), True)


@pytest.mark.gpu
@pytest.mark.parametrize("ptype", [torch.int32, torch.int64])
def test_offsets(ptype):
    lead = (4, 3, 5)
    q, k = _rand(lead + (2, 24), 1, torch.float32), _rand(lead + (1, 24), 2, torch.float32)
    start = torch.tensor([[0, 0], [100, -7], [32767, 131071], [-5, 2 ** 31 - 10]], dtype=ptype)
    dims = (8, 12)
    # the definition multiplies by base ** x as a double: its last place, 2^-53, counts 2^31 times
    _case(q, k, _turns(_grid(lead, offsets=start), dims), lambda a, b: nb.rotary(a, b, dims, offsets=start.to(DEV)), True, 2.0 ** -19)
    _case(q, k, _turns(_grid(lead, origin=(11, 2000)), dims), lambda a, b: nb.rotary(a, b, dims, offsets=(11, 2000)), True)
    _case(q, k, _turns(_grid(lead, origin=(9, 9)), dims), lambda a, b: nb.rotary(a, b, dims, offsets=9), True)


@pytest.mark.gpu
@pytest.mark.parametrize("ptype,shared", [(torch.int32, False), (torch.int64, True)])
@pytest.mark.parametrize("interleaved", [True, False])
def test_given_positions(ptype, shared, interleaved):
    lead, dims = (2, 37), (16, 10, 6)
    q, k = _rand(lead + (6, 40), 1, torch.bfloat16), _rand(lead + (2, 40), 2, torch.bfloat16)
    pos = torch.randint(-1000, 40000, ((1 if shared else 2), 37, 3), generator=torch.Generator().manual_seed(4)).to(ptype)
    _case(q, k, _turns(pos.long().expand(2, 37, 3), dims),
          lambda a, b: nb.rotary(a, b, dims, interleaved=interleaved, positions=pos.to(DEV)), interleaved, 2.0 ** -30)
    # the same positions again, as a view whose last axis is not the fastest
    strided = pos.to(DEV).transpose(1, 2).contiguous().transpose(1, 2)
    a = nb.rotary(q.to(DEV), k.to(DEV), dims, positions=pos.to(DEV))
    b = nb.rotary(q.to(DEV), k.to(DEV), dims, positions=strided)
    assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.gpu
def test_base_and_frequencies():
    lead, dims = (1, 19), (12,)
    q, k = _rand(lead + (2, 16), 1, torch.float32), _rand(lead + (2, 16), 2, torch.float32)
    _case(q, k, _turns(_grid(lead), dims, base=500.0), lambda a, b: nb.rotary(a, b, dims, base=500.0), True)
    freqs = [7.5, 1.0, -0.25, 0.0, 1e-9, 3.141592653589793]
    _case(q, k, _turns(_grid(lead), dims, freqs=freqs), lambda a, b: nb.rotary(a, b, dims, frequencies=freqs), True)


def test_phases_are_fractions_of_a_turn():
    p = list(_phases((4, 2), 10000.0, None))
    pi = Fraction(314159265358979323846264338327950288419716939937510, 10 ** 50)
    for got, f in zip(p, (Fraction(1), Fraction(1, 100), Fraction(1))):
        assert abs(Fraction(got, 2 ** 64) - f / (2 * pi)) <= Fraction(1, 2 ** 64)
    assert list(_phases((2,), 1.0, (-1.0,)))[0] == (-p[0]) % 2 ** 64


@pytest.mark.gpu
@pytest.mark.parametrize("interleaved", [True, False])
def test_strided_inputs(interleaved):
    qkv = _rand((2, 5, 6, 3, 4, 32), 1, torch.float16).to(DEV)
    turns = _turns(_grid((2, 5, 6)), (16, 16))
    call = lambda a, b: nb.rotary(a, b, interleaved=interleaved)
    _case(qkv.select(-3, 0), qkv.select(-3, 1), turns, call, interleaved)
    heads_first = _rand((2, 4, 5, 6, 32), 2, torch.float16).to(DEV).permute(0, 2, 3, 1, 4)
    _case(heads_first, qkv.select(-3, 2)[..., :1, :], turns, call, interleaved)
    wide = _rand((2, 5, 6, 4, 37), 3, torch.float16).to(DEV)
    _case(wide[..., 1:33], wide[..., :2, 5:37], turns, call, interleaved)      # heads that start anywhere
    _case(qkv[:1, :1, :1, 0].expand(2, 5, 6, 4, 32), qkv.select(-3, 0)[..., 1:3, :], turns, call, interleaved)


@pytest.mark.gpu
def test_angles_do_not_depend_on_the_path_taken():
    """What a token gets depends on its position alone: the same in a long sequence, by offset and by given position."""
    q, k = _rand((1, 400, 2, 64), 1, torch.bfloat16).to(DEV), _rand((1, 400, 1, 64), 2, torch.bfloat16).to(DEV)
    whole = nb.rotary(q, k)
    part = nb.rotary(q[:, 390:], k[:, 390:], offsets=390)
    step = nb.rotary(q[:, 399:], k[:, 399:], offsets=torch.tensor([[399]], device=DEV))
    given = nb.rotary(q[:, 390:], k[:, 390:], positions=torch.arange(390, 400, device=DEV).reshape(1, 10, 1))
    for a, b, c, d in zip(whole, part, step, given):
        assert torch.equal(a[:, 390:], b) and torch.equal(a[:, 399:], c) and torch.equal(b, d)


@pytest.mark.gpu
def test_one_gradient_only_and_empty_batches():
    q = _rand((2, 9, 2, 16), 1, torch.float32).to(DEV).requires_grad_(True)
    k = _rand((2, 9, 1, 16), 2, torch.float32).to(DEV)
    yq, yk = nb.rotary(q, k)
    dq, = torch.autograd.grad(yq.square().sum(), q)
    # turning keeps lengths, so the gradient of the squared length is 2 q
    assert torch.allclose(dq, 2 * q.detach(), atol=1e-5)
    e, f = nb.rotary(torch.empty(0, 9, 2, 16, device=DEV), torch.empty(0, 9, 1, 16, device=DEV))
    assert e.shape == (0, 9, 2, 16) and f.shape == (0, 9, 1, 16)
    e, f = nb.rotary(torch.empty(2, 0, 2, 16, device=DEV), torch.empty(2, 0, 1, 16, device=DEV))
    assert e.shape == (2, 0, 2, 16)


@pytest.mark.gpu
def test_captured_and_replayed():
    q, k = _rand((3, 1, 4, 64), 1, torch.bfloat16).to(DEV), _rand((3, 1, 2, 64), 2, torch.bfloat16).to(DEV)
    at = torch.tensor([[5], [6], [7]], dtype=torch.int32, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            got = nb.rotary(q, k, offsets=at)
    torch.cuda.current_stream().wait_stream(side)
    for _ in range(3):
        at += 1                                        # a step of decoding reads the new positions
        graph.replay()
    want = nb.rotary(q, k, offsets=torch.tensor([[8], [9], [10]], device=DEV))
    assert all(torch.equal(a, b) for a, b in zip(got, want))


# ---- refusals ----------------------------------------------------------------------------------------------------

def test_python_refusals():
    q, k = torch.zeros(2, 5, 2, 8), torch.zeros(2, 5, 1, 8)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        nb.rotary(q, k)
    for args, match in [((q[0], k[0]), "shapes"), ((q, k[:, :3]), "must match"), ((q, k[..., :4]), "Head dim"),
                        ((q, k.half()), "dtype"), ((q.double(), k.double()), "dtype")]:
        with pytest.raises(ValueError, match=match):
            nb.rotary(*args)
    with pytest.raises(ValueError, match="must have heads"):
        nb.rotary(q[:, :, :0], k)
    with pytest.raises(ValueError, match="must have heads"):
        nb.rotary(q, k[:, :, :0])
    many = torch.zeros(1, 1, 1, 2).expand(1, 2 ** 32 + 5, 1, 2)
    with pytest.raises(ValueError, match="below 2"):
        nb.rotary(many, many)
    with pytest.raises(ValueError, match="positions must be"):
        nb.rotary(q, k, positions=[0, 1, 2, 3, 4])
    with pytest.raises(ValueError, match="positions must be"):
        nb.rotary(q, k, positions=torch.tensor(3))
    with torch.autograd.forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="forward-mode"):
            nb.rotary(torch.autograd.forward_ad.make_dual(q, torch.ones_like(q)), k)
    with pytest.raises(ValueError, match="rotary needs"):
        nb.nn.NeighborhoodAttention2D(12, 4, 3, rotary=True)


@pytest.mark.gpu
def test_python_refusals_of_cuda_tensors():
    q, k = torch.zeros(2, 5, 2, 8, device=DEV), torch.zeros(2, 5, 1, 8, device=DEV)
    pos = torch.zeros(2, 5, 1, dtype=torch.int32, device=DEV)
    for kw, match in [(dict(axis_dims=(3,)), "even"), (dict(axis_dims=(10,)), "sum"), (dict(axis_dims=(0,)), "sum"),
                      (dict(axis_dims=(4, 4)), "spatial axes"), (dict(axis_dims=()), "1 to 3"), (dict(base=0.0), "base"),
                      (dict(frequencies=[1.0]), "finite numbers"), (dict(frequencies=[1.0, 2.0, float("inf"), 0.0]), "finite"),
                      (dict(offsets=(1, 2)), "length"), (dict(offsets=1.5), "integers"), (dict(offsets=pos, positions=pos), "combined"),
                      (dict(offsets=torch.zeros(3, 1, dtype=torch.int32, device=DEV)), "shape"),
                      (dict(offsets=torch.zeros(2, 1, device=DEV)), "int32 or int64"),
                      (dict(offsets=torch.zeros(2, 1, dtype=torch.int32)), "device"),
                      (dict(positions=pos[:, :4]), "shape"), (dict(positions=pos.float()), "int32 or int64"),
                      (dict(positions=pos.expand(2, 5, 4)), "entries"), (dict(axis_dims=(4, 2), positions=pos), "shape")]:
        with pytest.raises(ValueError, match=match):
            nb.rotary(q, k, **kw)


def _geom(**kw):
    phases = (ctypes.c_uint64 * 256)()
    g = _lib.RotaryGeom(_lib.F32, 1, 2, _lib._I3(5, 0, 0), 2, 1, 8, 1, _lib._I3(8, 0, 0), 16, 8, 8, 8, 1, 0, 32, 0,
                        (ctypes.c_int64 * 3)(), None, ctypes.addressof(phases))
    g._keep = phases
    for name, v in kw.items():
        setattr(g, name, _lib._I3(*v) if isinstance(v, tuple) else v)
    return g


@pytest.mark.parametrize("kw,needle", [
    (dict(dtype=9), "dtype"), (dict(rank=0), "rank"), (dict(rank=4), "rank"), (dict(n_axes=0), "axes"), (dict(n_axes=4), "axes"),
    (dict(n_axes=2, axis_dims=(2, 2, 0)), "spatial dimension"), (dict(position_kind=3), "kind"), (dict(position_kind=1), "positions is null"),
    (dict(position_bits=16), "bits"), (dict(heads_q=0), "positive"), (dict(head_dim=0), "positive"), (dict(phases=None), "phases"),
    (dict(extent=(-1, 0, 0)), "extents"), (dict(batch=1 << 31), "tokens"), (dict(axis_dims=(3, 0, 0)), "even"),
    (dict(axis_dims=(-2, 0, 0)), "even"), (dict(axis_dims=(10, 0, 0)), "head_dim"), (dict(axis_dims=(0, 0, 0)), "rotated"),
    (dict(axis_dims=(514, 0, 0), head_dim=600), "rotated"), (dict(head_dim=1 << 20), "large"),
])
def test_abi_refusals(kw, needle):
    before = _lib.launch_count()
    assert _lib.load().natten_b200_rotary(_geom(**kw), 4096, 4096, 4096, 4096, 0, None) == _lib.EINVAL
    assert needle in _lib.last_error()
    assert _lib.launch_count() == before


def test_abi_pointers():
    lib = _lib.load()
    assert lib.natten_b200_rotary(None, 4096, 4096, 4096, 4096, 0, None) == _lib.EINVAL
    assert lib.natten_b200_rotary(_geom(), None, 4096, 4096, 4096, 0, None) == _lib.EINVAL
    assert lib.natten_b200_rotary(_geom(), 4096 + 2, 4096, 4096, 4096, 0, None) == _lib.EINVAL
    assert lib.natten_b200_rotary(_geom(batch=0), None, None, None, None, 0, None) == _lib.OK
    assert lib.natten_b200_rotary(_geom(position_kind=1, positions=4096 + 2), 4096, 4096, 4096, 4096, 0, None) == _lib.EINVAL
    assert lib.natten_b200_rotary(_geom(position_kind=2, position_bits=64, positions=4096 + 4), 4096, 4096, 4096, 4096, 0,
                                  None) == _lib.EINVAL and "aligned" in _lib.last_error()
