"""``layer_norm``: values and gradients against the definition in 64 bits, widths on both sides of every kernel variant,
strided inputs, types, refusals.

Tolerances.  Let u be half a step of the result's type (2^-24, 2^-11, 2^-8) and e = 2^-24.  The kernel works in float32 and
rounds once, so every bound is u |value| plus the float32 error.  A sum over C elements adds at most 32 of them in a row
in a thread and joins the threads in a tree or in 16 steps: fewer than 64 roundings deep (the kernels for very wide rows
add C / 512 in a row).  With K = 64 + C / 512 the mean is off by at most K e mean|x|, and xhat by
K e (2 + |xhat| + rstd mean|x|) up to terms of second order; the factors that follow add a few e."""

from __future__ import annotations

import pytest
import torch

import natten_mlx_b200 as nb
from natten_mlx_b200 import _lib

DEV = "cuda"
U = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
E = 2.0 ** -24


def _definition(x, w, b, g, eps):
    """y, dx, dw, db and the sizes that the bounds need, all in float64."""
    x, g = x.double().cpu(), g.double().cpu()
    c = x.shape[-1]
    w = torch.ones(c, dtype=torch.float64) if w is None else w.double().cpu()
    bb = torch.zeros(c, dtype=torch.float64) if b is None else b.double().cpu()
    mean = x.mean(-1, keepdim=True)
    rstd = 1.0 / torch.sqrt(((x - mean) ** 2).mean(-1, keepdim=True) + eps)
    xh = (x - mean) * rstd
    gw = g * w
    dx = rstd * (gw - gw.mean(-1, keepdim=True) - xh * (gw * xh).mean(-1, keepdim=True))
    rows = lambda t: t.reshape(-1, c)
    k = 64 + c / 512
    xh_err = k * E * (2 + xh.abs() + rstd * x.abs().mean(-1, keepdim=True))
    y_err = xh_err * w.abs() + 4 * E * (xh * w).abs() + 2 * E * bb.abs()
    mean_abs = lambda t: t.abs().mean(-1, keepdim=True)
    # the second mean sees the error of xhat twice: in its terms, and in the xhat it is multiplied by
    dx_err = rstd * (8 * E * gw.abs() + k * E * mean_abs(gw) + xh.abs() * (k * E * mean_abs(gw * xh) + mean_abs(gw * xh_err))
                     + xh_err * mean_abs(gw * xh)) + 4 * E * dx.abs() + dx.abs() * k * E
    n = rows(x).shape[0]
    deep = min(n, 2 * (n // 148 + 64)) + 64       # rows added in a row by one thread, then the joins
    dw_err = rows(g.abs() * xh_err).sum(0) + deep * E * rows((g * xh).abs()).sum(0)
    db_err = deep * E * rows(g.abs()).sum(0)
    return dict(y=(xh * w + bb, y_err), dx=(dx, dx_err), dw=(rows(g * xh).sum(0), dw_err), db=(rows(g).sum(0), db_err))


def _check(name, got, want):
    value, err = want
    got64 = got.detach().double().cpu()
    assert got64.shape == value.shape
    off = (got64 - value).abs()
    # a result below the smallest normal number of fp16 is rounded to a multiple of 2^-24
    tiny = 2.0 ** -25 if got.dtype == torch.float16 else 0.0
    bound = U[got.dtype] * value.abs() + err * (1 + U[got.dtype]) + tiny
    worst = (off / bound.clamp_min(1e-300)).max() if off.numel() else 0.0
    assert bool((off <= bound).all()), f"{name}: {float(worst):.3g} of the bound"


def _rand(shape, seed, dtype, scale=1.0, mean=0.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed), dtype=torch.float64) * scale + mean).to(dtype)


def _case(x, w, b, g, eps=1e-5):
    want = _definition(x, w, b, g, eps)
    x, g = x.to(DEV), g.to(DEV)
    leaves = [None if t is None else t.to(DEV).requires_grad_(True) for t in (w, b)]
    xl = x.detach().requires_grad_(True)
    y = nb.layer_norm(xl, leaves[0], leaves[1], eps=eps)
    assert y.dtype == x.dtype and y.is_contiguous()
    _check("y", y, want["y"])
    ins = [xl] + [t for t in leaves if t is not None]
    grads = torch.autograd.grad(y, ins, g)
    names = ["dx"] + [n for n, t in zip(("dw", "db"), leaves) if t is not None]
    for n, t, like in zip(names, grads, ins):
        assert t.dtype == like.dtype and t.shape == like.shape
        _check(n, t, want[n])
    return y, grads


# widths on both sides of the variants' limits, odd ones, and lengths from a single row
WIDTHS = [(5, 1), (3, 2), (37, 7), (33, 32), (70, 33), (9, 64), (19, 96), (130, 128), (3, 200), (50, 256), (2, 257),
          (17, 512), (5, 513), (31, 768), (7, 776), (40, 1000), (9, 1024), (4, 1025), (6, 1536), (7, 2048), (3, 2056), (5, 2560), (2, 2568), (2, 4096), (3, 4100), (2, 8192),
          (2, 8200), (1, 16384), (2, 16385), (3, 20000)]


@pytest.mark.gpu
@pytest.mark.parametrize("rows,c", WIDTHS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_against_the_definition(rows, c, dtype):
    wt = torch.float32 if (rows + c) % 2 else dtype
    x = _rand((rows, c), 1, dtype, 1.5, 0.4)
    _case(x, _rand((c,), 2, wt, 0.3, 1.0), _rand((c,), 3, wt, 0.3), _rand((rows, c), 4, dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("rows,c,dtype", [(4001, 96, torch.bfloat16), (3001, 1024, torch.bfloat16), (20011, 32, torch.float16),
                                          (2503, 331, torch.float32), (999, 4096, torch.float16)])
def test_many_rows(rows, c, dtype):
    _case(_rand((rows, c), 1, dtype), _rand((c,), 2, torch.float32, 0.3, 1.0), _rand((c,), 3, torch.float32), _rand((rows, c), 4, dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("c", [65, 66, 127, 130, 333, 334, 511, 514, 1026, 2001, 2046, 2050])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_narrow_accesses(c, dtype):
    """Row lengths that leave accesses of 2 and 4 bytes, and so do rows that start off the wider boundaries."""
    x = _rand((301, c), 1, dtype, 1.5, 0.4)
    w, b, g = _rand((c,), 2, torch.float32, 0.3, 1.0), _rand((c,), 3, torch.float32, 0.3), _rand((301, c), 4, dtype)
    y, grads = _case(x, w, b, g)
    xs = torch.zeros(301, c + 3, dtype=dtype, device=DEV)[:, 1:c + 1].copy_(x).requires_grad_(True)
    _check("y", nb.layer_norm(xs, w.to(DEV), b.to(DEV)), _definition(x, w, b, g, 1e-5)["y"])
    ds, = torch.autograd.grad(nb.layer_norm(xs, w.to(DEV), b.to(DEV)), xs, g.to(DEV))
    _check("dx", ds, _definition(x, w, b, g, 1e-5)["dx"])


@pytest.mark.gpu
@pytest.mark.parametrize("with_w,with_b", [(False, False), (True, False), (False, True)])
def test_without_weights(with_w, with_b):
    c = 72
    _case(_rand((2, 3, c), 1, torch.float32), _rand((c,), 2, torch.float32) if with_w else None,
          _rand((c,), 3, torch.float32) if with_b else None, _rand((2, 3, c), 4, torch.float32), eps=1e-3)


@pytest.mark.gpu
def test_rows_inside_a_fused_projection_and_other_strides():
    qkv = _rand((2, 5, 6, 3, 4, 32), 1, torch.bfloat16).to(DEV)
    w, b = _rand((32,), 2, torch.float32, 0.3, 1.0), _rand((32,), 3, torch.float32)
    for x in (qkv.select(-3, 1), qkv.select(-3, 0)[:, 1:, ::2], qkv.select(-3, 2).transpose(1, 3), qkv[..., 1:2, :, :],
              qkv[:, :, :1, 0, :1], qkv.select(-3, 0)[..., 3:30], qkv[:1, :1, :1, 0, 0].expand(4, 2, 3, 32)):
        c = x.shape[-1]
        g = _rand(x.shape, 5, torch.bfloat16)
        _case(x, w[:c].clone(), b[:c].clone(), g)
    # a base address that is aligned to the elements only
    flat = _rand((7 * 40 + 3,), 6, torch.bfloat16).to(DEV)
    for first in (1, 2, 3):
        _case(flat[first:first + 280].view(7, 40), _rand((41,), 2, torch.float32)[1:], None, _rand((7, 40), 7, torch.bfloat16))


@pytest.mark.gpu
def test_gradient_arrives_in_any_layout():
    x = _rand((6, 10, 48), 1, torch.float32).to(DEV).requires_grad_(True)
    y = nb.layer_norm(x)
    g = _rand((10, 6, 48), 2, torch.float32).to(DEV).transpose(0, 1)
    a, = torch.autograd.grad(y, x, g, retain_graph=True)
    b, = torch.autograd.grad(y, x, g.contiguous(), retain_graph=True)
    assert torch.equal(a, b)
    s, = torch.autograd.grad(y.sum(), x)          # an expanded gradient; the sum over a row does not depend on x
    assert float(s.abs().max()) < 1e-5


@pytest.mark.gpu
def test_special_rows():
    x = _rand((8, 64), 1, torch.float32).to(DEV)
    x[1] = 3.25                                    # no spread: xhat is 0
    x[2, 5] = float("inf")
    x[3, 7] = float("nan")
    x[4] = 1e4 + x[4]                              # a large mean: the variance is taken about it
    x[5] = 0
    y = nb.layer_norm(x)
    clean = nb.layer_norm(x[[0, 6, 7]])
    assert torch.equal(y[[0, 6, 7]], clean)
    assert float(y[1].abs().max()) == 0.0 and float(y[5].abs().max()) == 0.0
    assert bool(torch.isnan(y[2]).any()) and bool(torch.isnan(y[3]).all())
    x4 = x[4].double()
    want = (x4 - x4.mean()) / torch.sqrt(x4.var(correction=0) + 1e-5)
    assert float((y[4].double() - want).abs().max()) < 64 * E * 1e4 * 2 / float(x4.std()) + 1e-6


@pytest.mark.gpu
def test_same_bits_from_call_to_call_and_only_what_is_asked_for():
    x = _rand((5000, 256), 1, torch.bfloat16).to(DEV)
    w, b = (_rand((256,), s, torch.float32).to(DEV).requires_grad_(True) for s in (2, 3))
    g = _rand((5000, 256), 4, torch.bfloat16).to(DEV)
    first = torch.autograd.grad(nb.layer_norm(x, w, b), (w, b), g)          # x needs no gradient
    for _ in range(3):
        again = torch.autograd.grad(nb.layer_norm(x, w, b), (w, b), g)
        assert all(torch.equal(a, c) for a, c in zip(first, again))
    xl = x.detach().requires_grad_(True)
    dx, = torch.autograd.grad(nb.layer_norm(xl, w.detach(), b.detach()), xl, g)
    dx2, dw, db = torch.autograd.grad(nb.layer_norm(xl, w, b), (xl, w, b), g)
    assert torch.equal(dx, dx2) and torch.equal(dw, first[0]) and torch.equal(db, first[1])
    dw_only, = torch.autograd.grad(nb.layer_norm(xl, w, b.detach()), w, g)
    assert torch.equal(dw_only, dw)


@pytest.mark.gpu
def test_empty_batches():
    w, b = (torch.ones(16, device=DEV).requires_grad_(True) for _ in range(2))
    x = torch.empty(0, 5, 16, device=DEV, requires_grad=True)
    y = nb.layer_norm(x, w, b)
    assert y.shape == x.shape
    dx, dw, db = torch.autograd.grad(y.sum(), (x, w, b))
    assert dx.shape == x.shape and float(dw.abs().sum()) == 0.0 and float(db.abs().sum()) == 0.0


@pytest.mark.gpu
def test_against_differences():
    x, w, b = _rand((3, 20), 1, torch.float32), _rand((20,), 2, torch.float32), _rand((20,), 3, torch.float32)
    g = _rand((3, 20), 4, torch.float32)
    leaves = [t.to(DEV).requires_grad_(True) for t in (x, w, b)]
    grads = torch.autograd.grad(nb.layer_norm(*leaves), leaves, g.to(DEV))
    f = lambda ts: float((_definition(ts[0], ts[1], ts[2], g, 1e-5)["y"][0] * g.double()).sum())
    h = 1e-5
    for i, (t, grad) in enumerate(zip((x, w, b), grads)):
        for j in range(0, t.numel(), 7):
            args = [a.double().clone() for a in (x, w, b)]
            args[i].view(-1)[j] += h
            up = f(args)
            args[i].view(-1)[j] -= 2 * h
            # central differences of a function of order ten in 64 bits: h^2 and 1e-14 / h are far below 1e-6
            assert abs((up - f(args)) / (2 * h) - float(grad.view(-1)[j])) < 1e-5 * (1 + abs(float(grad.view(-1)[j])))


@pytest.mark.gpu
def test_captured_replayed_and_on_another_stream():
    x = _rand((700, 128), 1, torch.bfloat16).to(DEV)
    w, b = _rand((128,), 2, torch.float32).to(DEV), _rand((128,), 3, torch.float32).to(DEV)
    g = _rand((700, 128), 4, torch.bfloat16).to(DEV)
    xl, wl, bl = (t.detach().requires_grad_(True) for t in (x, w, b))

    def step():
        y = nb.layer_norm(xl, wl, bl)
        return (y,) + torch.autograd.grad(y, (xl, wl, bl), g)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            got = step()
    torch.cuda.current_stream().wait_stream(side)
    with torch.no_grad():
        x.copy_(_rand((700, 128), 9, torch.bfloat16))      # xl shares x's memory
    graph.replay()
    want = step()
    torch.cuda.synchronize()
    assert all(torch.equal(a, c) for a, c in zip(got, want))


@pytest.mark.gpu
def test_double_backward_is_refused():
    x = torch.randn(3, 8, device=DEV, requires_grad=True)
    g, = torch.autograd.grad(nb.layer_norm(x).square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.sum().backward()


# ---- refusals: nothing is launched -------------------------------------------------------------------------------

def test_tangents_are_refused():
    x, w = torch.zeros(2, 4), torch.ones(4)
    with torch.autograd.forward_ad.dual_level():
        for args in ((torch.autograd.forward_ad.make_dual(x, x), w), (x, torch.autograd.forward_ad.make_dual(w, w))):
            with pytest.raises(RuntimeError, match="forward-mode"):
                nb.layer_norm(*args)


def test_python_refusals():
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        nb.layer_norm(torch.zeros(2, 4))
    with pytest.raises(ValueError, match="dim must be positive"):
        nb.nn.LayerNorm(0)


@pytest.mark.gpu
def test_python_refusals_of_cuda_tensors():
    x = torch.zeros(2, 4, device=DEV)
    for kw, match in [(dict(weight=torch.ones(3, device=DEV)), "shape"), (dict(weight=torch.ones(4)), "device"),
                      (dict(weight=torch.ones(4, device=DEV, dtype=torch.float16)), "dtype"),
                      (dict(weight=torch.ones(4, device=DEV), eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"),
                      (dict(bias=torch.ones(4, 1, device=DEV)), "shape")]:
        with pytest.raises(ValueError, match=match):
            nb.layer_norm(x, **kw)
    with pytest.raises(ValueError, match="one dtype"):
        nb.layer_norm(x.half(), torch.ones(4, device=DEV), torch.ones(4, device=DEV).half())
    with pytest.raises(ValueError, match="unsupported dtype"):
        nb.layer_norm(x.double())
    with pytest.raises(ValueError, match="C >= 1"):
        nb.layer_norm(torch.zeros(3, 0, device=DEV))
    with pytest.raises(ValueError, match="match dim"):
        nb.nn.LayerNorm(5).to(DEV)(x)


@pytest.mark.parametrize("change,code,needle", [
    (dict(dtype=7), _lib.EINVAL, "dtype"), (dict(wdtype=_lib.F16), _lib.EINVAL, "weights"), (dict(rows=None), _lib.EINVAL, "null"),
    (dict(rows=_lib.Rows(4, 1, 8, 0, 0, 0)), _lib.EINVAL, "channels"), (dict(rows=_lib.Rows(-1, 1, 8, 0, 8, 0)), _lib.EINVAL, "rows"),
    (dict(rows=_lib.Rows(1 << 31, 1, 8, 0, 8, 0)), _lib.EINVAL, "rows"), (dict(rows=_lib.Rows(4, 0, 8, 0, 8, 0)), _lib.EINVAL, "inner"),
    (dict(x=None), _lib.EINVAL, "null"), (dict(eps=-1.0), _lib.EINVAL, "eps"), (dict(x=4096 + 1), _lib.EINVAL, "aligned"),
    (dict(mean=None), _lib.EINVAL, "null"),
])
def test_abi_refusals(change, code, needle):
    a = dict(dtype=_lib.BF16, wdtype=_lib.BF16, rows=_lib.Rows(4, 1, 8, 0, 8, 0), x=4096, eps=1e-5, mean=4096)
    a.update(change)
    before = _lib.launch_count()
    lib = _lib.load()
    assert lib.natten_b200_layer_norm_forward(a["dtype"], a["wdtype"], a["rows"], a["x"], 4096, 4096, a["eps"], 4096,
                                              a["mean"], 4096, None) == code
    assert needle in _lib.last_error()
    if "eps" not in change:
        assert lib.natten_b200_layer_norm_backward(a["dtype"], a["wdtype"], a["rows"], a["x"], 4096, a["mean"], 4096, 4096,
                                                   4096, 4096, 4096, 4096, 1 << 30, None) == code
    assert _lib.launch_count() == before


def test_abi_alignment_of_weights_and_statistics():
    lib, before = _lib.load(), _lib.launch_count()
    rows = _lib.Rows(4, 1, 8, 0, 8, 0)
    for at, off in ((3, 2), (4, 2), (7, 2), (8, 1)):         # weight, bias (float32 beside bf16), mean, rstd
        a = [_lib.BF16, _lib.F32, rows, 4096, 4096, 4096, 1e-5, 4096, 4096, 4096, None]
        a[at + 1] += off
        assert lib.natten_b200_layer_norm_forward(*a) == _lib.EINVAL and "aligned" in _lib.last_error()
    for at, off in ((4, 2), (5, 2), (6, 2), (9, 2), (10, 2)):        # weight, mean, rstd, dweight, dbias
        a = [_lib.BF16, _lib.F32, rows, 4096, 4096, 4096, 4096, 4096, 4096, 4096, 4096, 4096, 1 << 30, None]
        a[at] += off
        assert lib.natten_b200_layer_norm_backward(*a) == _lib.EINVAL and "aligned" in _lib.last_error()
    assert lib.natten_b200_layer_norm_forward(_lib.BF16, _lib.F32, _lib.Rows(4, 1, 8, 0, 8, 1), 4096, 4096, 4096, 1e-5, 4096, 4096,
                                              4096, None) == _lib.EINVAL and "reserved" in _lib.last_error()
    assert _lib.launch_count() == before


def test_abi_scratch_and_empty_calls():
    lib = _lib.load()
    rows = _lib.Rows(1000, 1, 64, 0, 64, 0)
    need = lib.natten_b200_layer_norm_backward_scratch_bytes(1000, 64)
    assert 0 < need <= 1000 * 2 * 64 * 4
    assert lib.natten_b200_layer_norm_backward(_lib.F32, _lib.F32, rows, 4096, 4096, 4096, 4096, 4096, 4096, 4096, 4096, 4096,
                                               need - 1, None) == _lib.ERESOURCE
    assert lib.natten_b200_layer_norm_backward(_lib.F32, _lib.F32, rows, 4096, 4096, 4096, 4096, 4096, 4096, 4096, 4096, None,
                                               need, None) == _lib.ERESOURCE
    assert lib.natten_b200_layer_norm_backward_scratch_bytes(0, 64) == 0
    none = _lib.Rows(0, 1, 64, 0, 64, 0)
    assert lib.natten_b200_layer_norm_forward(_lib.F32, _lib.F32, none, None, None, None, 1e-5, None, None, None, None) == _lib.OK
    # nothing is asked for
    assert lib.natten_b200_layer_norm_backward(_lib.F32, _lib.F32, rows, 4096, 4096, 4096, 4096, 4096, None, None, None, None, 0,
                                               None) == _lib.OK
