"""``prefix_attention``: both kernel families against the definition in 64 bits: head layouts, lengths from one key, odd
sizes, samples that see a part of the prefix or none, non-finite keys behind a sample's end, merging with a window's
result, splitting, strides, refusals.

Tolerances.  Let u be half a step of the type, e = 2^-24, o = sum w v with weights w that sum to 1, A = sum w |v|.
A logit is a sum of D products in float32: off by at most 2 (D + 2) e scale sum |q k| (the factor 2: the tensor core may
truncate where it adds), which with 2^-18 for the base-2 exponential (a polynomial of 2^-18.5 on the tensor
cores' path) and its argument is the relative error r of a weight.  On the tensor cores a weight is also rounded to the type (u; fp16 steps no finer than 2^-24 below 2^-14, against a
sum of at least 1: 2^-25 for each key, times |v|).  Sums over n keys are tree-like or at most 2 (n / 16 + 64) e.  So
  |out - o| <= u |o| + (2 r + u + 2 (n / 16 + 64) e) A + 2 e |o|,   |lse - l| <= r + 2 (n / 16 + 64) e + 4 e |l|."""

from __future__ import annotations

import math

import pytest
import torch

import natten_mlx_b200 as nb
from natten_mlx_b200 import _lib

DEV = "cuda"
U = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
E = 2.0 ** -24


def _rand(shape, seed, dtype, scale=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed), dtype=torch.float64) * scale).to(dtype)


def _definition(q, k, v, scale, lens=None, window=None, tc=True):
    """out, lse and their bounds, in float64 on the CPU; a sample's rows never touch what lies past its length."""
    dtype = q.dtype
    q, k, v = (t.detach().double().cpu() for t in (q, k, v))
    b, hq, d = q.shape[0], q.shape[-2], q.shape[-1]
    n, hk = k.shape[:2]
    u = U[dtype] if tc else 0.0
    flat = q.reshape(b, -1, hq, d)
    out, lse = torch.zeros_like(flat), torch.full(flat.shape[:-1], -math.inf, dtype=torch.float64)
    o_err, l_err = torch.zeros_like(flat), torch.zeros_like(lse)
    for i in range(b):
        m = n if lens is None else max(0, min(n, int(lens[i])))
        if m == 0:
            continue
        for h in range(hq):
            kh, vh = k[:m, h // (hq // hk)], v[:m, h // (hq // hk)]
            s = flat[i, :, h] @ kh.T * scale
            w = torch.softmax(s, -1)
            r = 2 * (d + 2) * E * scale * (flat[i, :, h].abs() @ kh.abs().T).amax(-1) + 2.0 ** -18
            out[i, :, h], lse[i, :, h] = w @ vh, torch.logsumexp(s, -1)
            sums = 2 * (m / 16 + 64) * E
            o_err[i, :, h] = (2 * r + u + sums).unsqueeze(-1) * (w @ vh.abs()) + 2 * E * out[i, :, h].abs()
            if tc and dtype == torch.float16:
                o_err[i, :, h] += 2.0 ** -25 * vh.abs().sum(0)
            l_err[i, :, h] = r + sums + 4 * E * lse[i, :, h].abs()
    out, lse, o_err, l_err = out.reshape(q.shape), lse.reshape(q.shape[:-1]), o_err.reshape(q.shape), l_err.reshape(q.shape[:-1])
    if window is not None:
        ow, lw = window[0].detach().double().cpu(), window[1].detach().double().cpu()
        both = torch.logaddexp(lse, lw)
        a = torch.where(lse == -math.inf, torch.zeros_like(lse), torch.exp(lse - both))
        c = torch.where(lw == -math.inf, torch.zeros_like(lw), torch.exp(lw - both))
        # the share of either part moves by the error of the lse, and by a few roundings of float32 numbers of its size
        move = (a * c * (l_err + 8 * E * (1 + lse.abs().nan_to_num(0, 0, 0) + lw.abs().nan_to_num(0, 0, 0)))).unsqueeze(-1)
        part = torch.where((c > 0).unsqueeze(-1), ow, torch.zeros_like(ow))
        o_err = o_err * a.unsqueeze(-1) + move * (out.abs() + part.abs()) + 8 * E * (out.abs() + part.abs())
        l_err = l_err + 8 * E * (1 + both.abs().nan_to_num(0, 0, 0))
        out = out * a.unsqueeze(-1) + part * c.unsqueeze(-1)
        lse = both
    return out, lse, U[dtype] * out.abs() + o_err + (2.0 ** -25 if dtype == torch.float16 else 0.0), l_err


def _check(got, want):
    out, lse = (t.detach().double().cpu() for t in got)
    o, l, o_err, l_err = want
    assert out.shape == o.shape and lse.shape == l.shape
    assert torch.equal(torch.isinf(lse), torch.isinf(l)), "rows without keys"
    off = (out - o).abs()
    assert bool((off <= o_err).all()), f"out: {float((off / o_err.clamp_min(1e-300)).max()):.3g} of the bound"
    fin = torch.isfinite(l)
    off = (lse - l).abs()[fin]
    assert bool((off <= l_err[fin]).all()), f"lse: {float((off / l_err[fin]).max()):.3g} of the bound"


def _run(q, k, v, path, scale=None, lens=None, window=None):
    q, k, v = q.to(DEV), k.to(DEV), v.to(DEV)
    lens = None if lens is None else torch.as_tensor(lens, dtype=torch.int32).to(DEV)
    nb.set_fused_path(path)
    try:
        got = nb.prefix_attention(q, k, v, scale, True, prefix_lens=lens,
                                  window=None if window is None else tuple(t.to(DEV) for t in window))
        assert _lib.last_path() == ("tcgen05" if path == "tcgen05" else "simt")
    finally:
        nb.set_fused_path("auto")
    assert got[0].dtype == q.dtype and got[1].dtype == torch.float32
    assert got[0].is_contiguous() and got[1].is_contiguous()
    assert _lib.kernel_status() == 0
    return got


def _case(shape, hk, n, dtype, path, lens=None, window=False, seed=0, scale=None):
    d = shape[-1]
    q, k, v = _rand(shape, seed + 1, dtype, 1.3), _rand((n, hk, d), seed + 2, dtype, 1.3), _rand((n, hk, d), seed + 3, dtype)
    win = (_rand(shape, seed + 4, dtype, 0.5), _rand(shape[:-1], seed + 5, torch.float32) + math.log(n + 1)) if window else None
    got = _run(q, k, v, path, scale, lens, win)
    _check(got, _definition(q, k, v, d ** -0.5 if scale is None else scale, lens, win, path == "tcgen05"))


TC = [
    # query [B, spatial..., heads, D], kv heads, prefix
    ((1, 1, 1, 64), 1, 1), ((1, 1, 1, 8), 1, 127), ((2, 1, 8, 64), 2, 128), ((3, 1, 4, 128), 4, 129), ((64, 1, 16, 64), 4, 300),
    ((1, 130, 2, 64), 2, 257), ((2, 9, 15, 4, 32), 4, 200), ((1, 5, 7, 11, 3, 24), 1, 385), ((2, 300, 6, 128), 2, 1000),
    ((1, 257, 1, 80), 1, 640), ((5, 3, 7, 128), 1, 131), ((2, 3, 130, 16), 2, 90), ((1, 2, 128, 40), 1, 77), ((1, 700, 5, 72), 5, 140),
    ((1, 1, 2, 128), 1, 20000), ((4, 1, 8, 64), 8, 6000), ((1, 2100, 18, 64), 18, 1500), ((1, 1300, 8, 104), 8, 800),
    ((40, 33, 8, 32), 8, 2000),
]


@pytest.mark.gpu
@pytest.mark.parametrize("shape,hk,n", TC)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_tensor_core_kernel(shape, hk, n, dtype):
    _case(shape, hk, n, dtype, "tcgen05", window=(n + len(shape)) % 2 == 0)


SIMT = [
    ((1, 1, 1, 1), 1, 1), ((2, 1, 8, 64), 2, 63), ((3, 1, 4, 128), 4, 65), ((2, 9, 15, 4, 32), 4, 200), ((1, 5, 7, 3, 24), 1, 385),
    ((1, 130, 2, 17), 2, 257), ((1, 70, 4, 200), 2, 99), ((1, 1, 2, 256), 1, 3001), ((1, 90, 1, 256), 1, 33), ((2, 40, 3, 130), 1, 64),
    ((16, 1, 2, 66), 2, 500), ((1, 1, 300, 12), 2, 40), ((1, 1, 1, 150), 1, 40000), ((1, 2, 2, 131), 2, 5000),
]


@pytest.mark.gpu
@pytest.mark.parametrize("shape,hk,n", SIMT)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_cuda_core_kernel(shape, hk, n, dtype):
    _case(shape, hk, n, dtype, "simt", window=(n + len(shape)) % 2 == 0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,path", [(torch.bfloat16, "tcgen05"), (torch.float16, "tcgen05"), (torch.float32, "simt")])
@pytest.mark.parametrize("window", [False, True])
def test_samples_that_see_a_part(dtype, path, window):
    _case((7, 1, 4, 64), 2, 1000, dtype, path, lens=[1000, 0, 1, 128, 129, 777, 5000], window=window)
    _case((3, 50, 6, 40), 3, 300, dtype, path, lens=[0, 300, -4], window=window)
    _case((2, 150, 2, 128), 1, 260, dtype, path, lens=[130, 3], window=window)
    _case((3, 2, 2, 32), 1, 4000, dtype, path, lens=[0, 0, 0], window=window)
    _case((9, 1, 3, 24), 3, 700, dtype, path, lens=[700, 3, 64, 65, 0, 62, 699, 1, 130], window=window)


@pytest.mark.gpu
@pytest.mark.parametrize("d", [17, 28, 60, 124, 200])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_cuda_core_kernel_with_samples_that_see_a_part(d, dtype):
    """Rows of one thread that end at different places, in head dims of every variant and at every bank of a row."""
    _case((7, 3, 6, d), 2, 300, dtype, "simt", lens=[300, 1, 64, 31, 0, 33, 298])
    _case((2, 5, 2, d), 2, 90, dtype, "simt", lens=[7, 90], window=True)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,path", [(torch.bfloat16, "tcgen05"), (torch.float16, "tcgen05"), (torch.float32, "simt")])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_what_lies_past_a_samples_end_does_not_reach_it(dtype, path, bad):
    """The other samples see the bad tokens and are not compared."""
    shape, hk = (4, 3, 4, 64), 2
    for n, lens in ((500, [100, 256, 500, 0]), (6000, [3000, 1, 6000, 0])):
        q, k, v = _rand(shape, 1, dtype), _rand((n, hk, 64), 2, dtype), _rand((n, hk, 64), 3, dtype)
        win = (_rand(shape, 4, dtype), _rand(shape[:-1], 5, torch.float32))
        for which in (k, v):
            which[lens[0] if lens[0] > lens[1] else lens[1]:] = bad
        for w in (None, win):
            got = _run(q, k, v, path, None, lens, w)
            o, l, oe, le = _definition(q, k, v, 0.125, lens, w, path == "tcgen05")
            keep = [0, 1, 3]
            _check((got[0][keep], got[1][keep]), (o[keep], l[keep], oe[keep], le[keep]))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,path", [(torch.bfloat16, "tcgen05"), (torch.float16, "tcgen05"), (torch.float32, "simt")])
def test_logits_that_grow_along_the_prefix(dtype, path):
    """The reference maximum has to follow: every chunk's logits exceed those before by far more than 2^8."""
    n, d = 900, 64
    q = _rand((2, 70, 2, d), 1, dtype)
    q[..., 0] = 4.0
    k, v = _rand((n, 1, d), 2, dtype, 0.5), _rand((n, 1, d), 3, dtype)
    k[..., 0] = torch.arange(n, dtype=torch.float64).reshape(n, 1).to(dtype) * 0.25
    for keys in (k, k.flip(0)):
        got = _run(q, keys, v, path)
        _check(got, _definition(q, keys, v, d ** -0.5, tc=path == "tcgen05"))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,path", [(torch.bfloat16, "tcgen05"), (torch.float32, "simt")])
def test_window_without_keys_and_prefix_without_tokens(dtype, path):
    shape, n = (2, 6, 2, 32), 150
    q, k, v = _rand(shape, 1, dtype), _rand((n, 1, 32), 2, dtype), _rand((n, 1, 32), 3, dtype)
    ow, lw = _rand(shape, 4, dtype), _rand(shape[:-1], 5, torch.float32)
    lw[0] = -math.inf
    ow[0] = float("nan")                              # a result over no keys counts for nothing, whatever it holds
    _check(_run(q, k, v, path, window=(ow, lw)), _definition(q, k, v, 32 ** -0.5, None, (ow, lw), path == "tcgen05"))
    got = _run(q, k, v, path, None, [0, 0], (ow, lw))
    assert float(got[0][0].abs().max()) == 0.0 and bool((got[1][0] == -math.inf).all())
    assert torch.equal(got[0][1].cpu(), ow[1]) and torch.allclose(got[1][1].cpu(), lw[1], atol=1e-6)
    none = nb.prefix_attention(q.to(DEV), k[:0].to(DEV), v[:0].to(DEV), return_lse=True)
    assert float(none[0].abs().max()) == 0.0 and bool((none[1] == -math.inf).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,path", [(torch.bfloat16, "tcgen05"), (torch.float32, "simt")])
def test_agrees_with_extra_tokens_and_merge(dtype, path):
    """The window and the prefix together: as extra tokens of every sample, by merge_attentions, and in one kernel."""
    q, k, v = (_rand((2, 12, 14, 4, 32), s, dtype).to(DEV) for s in (1, 2, 3))
    pk, pv = _rand((75, 4, 32), 4, dtype).to(DEV), _rand((75, 4, 32), 5, dtype).to(DEV)
    extra = nb.na2d(q, k, v, 5, return_lse=True, additional_keys=pk.expand(2, 75, 4, 32), additional_values=pv.expand(2, 75, 4, 32))
    win = nb.na2d(q, k, v, 5, return_lse=True)
    one = nb.prefix_attention(q, pk, pv, return_lse=True, window=win)
    two = nb.merge_attentions([win[0], nb.prefix_attention(q, pk, pv)], [win[1], nb.prefix_attention(q, pk, pv, return_lse=True)[1]])
    tol = 2e-2 if dtype == torch.bfloat16 else 1e-5
    for other in (extra, two):
        assert float((one[0].float() - other[0].float()).abs().max()) < tol
        assert float((one[1] - other[1]).abs().max()) < 1e-3 if dtype == torch.bfloat16 else 1e-5


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,path", [(torch.bfloat16, "tcgen05"), (torch.float32, "simt")])
def test_strided_tensors(dtype, path):
    qkv = _rand((2, 9, 5, 3, 4, 32), 1, dtype).to(DEV)
    cache = _rand((300, 2, 4, 32), 2, dtype).to(DEV)
    q, k, v = qkv.select(-3, 0), cache[:, 0], cache[:, 1]
    want = _definition(q, k, v, 32 ** -0.5, tc=path == "tcgen05")
    _check(_run(q, k, v, path), want)
    heads_first = cache.permute(1, 2, 0, 3).contiguous()      # [2, heads, P, D]
    _check(_run(q, heads_first[0].transpose(0, 1), heads_first[1].transpose(0, 1), path), want)
    _check(_run(q.permute(0, 1, 2, 4, 3).contiguous().permute(0, 1, 2, 4, 3), k, v, path), want)
    odd = torch.zeros(300 * 4 * 32 + 3, dtype=dtype, device=DEV)[3:].view(300, 4, 32)
    odd.copy_(k)
    _check(_run(q, odd, v, path), want)
    one = k[:1].expand(300, 4, 32)
    _check(_run(q[:, ::2], one, v, path), _definition(q[:, ::2], one, v, 32 ** -0.5, tc=path == "tcgen05"))


@pytest.mark.gpu
def test_same_bits_from_call_to_call_and_two_streams_at_once():
    q, k, v = _rand((8, 1, 8, 64), 1, torch.bfloat16).to(DEV), _rand((9000, 2, 64), 2, torch.bfloat16).to(DEV), _rand((9000, 2, 64), 3, torch.bfloat16).to(DEV)
    want = nb.prefix_attention(q, k, v, return_lse=True)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for _ in range(4):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(nb.prefix_attention(q, k, v, return_lse=True))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for g in got for a, b in zip(g, want))
    assert _lib.kernel_status() == 0


@pytest.mark.gpu
def test_captured_and_replayed():
    q, k, v = _rand((4, 1, 4, 64), 1, torch.float16).to(DEV), _rand((3000, 2, 64), 2, torch.float16).to(DEV), _rand((3000, 2, 64), 3, torch.float16).to(DEV)
    lens = torch.tensor([3000, 10, 0, 2000], dtype=torch.int32, device=DEV)
    nb.prefix_attention(q, k, v, prefix_lens=lens)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs = []
    with torch.cuda.stream(side):
        for _ in range(2):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                got = nb.prefix_attention(q, k, v, return_lse=True, prefix_lens=lens)
            graphs.append((graph, got))
    torch.cuda.current_stream().wait_stream(side)
    lens.copy_(torch.tensor([5, 3000, 700, 1]))
    q.mul_(0.5)
    for graph, _ in graphs:
        graph.replay()
    want = nb.prefix_attention(q, k, v, return_lse=True, prefix_lens=lens)
    for _, got in graphs:
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
def test_lens_in_64_bits_and_no_queries():
    q, k, v = _rand((2, 3, 2, 16), 1, torch.float32).to(DEV), _rand((40, 2, 16), 2, torch.float32).to(DEV), _rand((40, 2, 16), 3, torch.float32).to(DEV)
    a = nb.prefix_attention(q, k, v, prefix_lens=torch.tensor([7, 2 ** 40], device=DEV))
    b = nb.prefix_attention(q, k, v, prefix_lens=torch.tensor([7, 40], dtype=torch.int32, device=DEV))
    assert torch.equal(a, b)
    assert nb.prefix_attention(q[:0], k, v).shape == (0, 3, 2, 16)
    assert nb.prefix_attention(q[:, :0], k, v).shape == (2, 0, 2, 16)


# ---- refusals ----------------------------------------------------------------------------------------------------

def test_tangents_are_refused():
    q, k = torch.zeros(2, 5, 4, 8), torch.zeros(7, 2, 8)
    with torch.autograd.forward_ad.dual_level(), torch.no_grad():
        with pytest.raises(RuntimeError, match="forward-mode"):
            nb.prefix_attention(q, torch.autograd.forward_ad.make_dual(k, k), k)


def test_python_refusals():
    q, k = torch.zeros(2, 5, 4, 8), torch.zeros(7, 2, 8)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        nb.prefix_attention(q, k, k)
    with pytest.raises(RuntimeError, match="no gradients"):
        nb.prefix_attention(q.clone().requires_grad_(True), k, k)
    win = (torch.zeros(2, 5, 4, 8), torch.zeros(2, 5, 4))
    for args, kw, match in [((q[0], k, k), {}, "spatial"), ((q, k[0], k[0]), {}, "3D"), ((q, k, k[:5]), {}, "one shape"),
                            ((q, k[..., :4], k[..., :4]), {}, "Head dim"), ((q[..., :3, :], k, k), {}, "divisible"),
                            ((q, k.half(), k.half()), {}, "dtype"), ((q, k, k, 0.0), {}, "scale"), ((q, k, k, float("nan")), {}, "scale"),
                            ((q, k, k, -1.0), {}, "scale"), ((q, k, k), dict(window=(win[0][:1], win[1])), "window"),
                            ((q, k, k), dict(window=(win[0], win[1], None)), r"window must be|NoneType"),
                            ((q, k, k), dict(window=(win[0].half(), win[1])), "dtype"),
                            ((torch.zeros(1, 1, 1, 257), torch.zeros(3, 1, 257), torch.zeros(3, 1, 257)), {}, "256")]:
        with pytest.raises((ValueError, AttributeError), match=match):
            nb.prefix_attention(*args, **kw)


@pytest.mark.gpu
def test_python_refusals_of_cuda_tensors():
    q, k = torch.zeros(2, 5, 4, 8, device=DEV), torch.zeros(7, 2, 8, device=DEV)
    for kw, match in [(dict(prefix_lens=[3, 4]), "int32 or int64"), (dict(prefix_lens=torch.zeros(2, device=DEV)), "int32 or int64"),
                      (dict(prefix_lens=torch.zeros(3, dtype=torch.int32, device=DEV)), "shape"),
                      (dict(prefix_lens=torch.zeros(2, dtype=torch.int32)), "device")]:
        with pytest.raises(ValueError, match=match):
            nb.prefix_attention(q, k, k, **kw)
    nb.set_fused_path("tcgen05")
    try:
        with pytest.raises(ValueError, match="float32"):
            nb.prefix_attention(q, k, k)
    finally:
        nb.set_fused_path("auto")


def _geom(**kw):
    g = _lib.PrefixGeom(_lib.BF16, 4, 2, 64, 2, 3, 100, 256, 64, 128, 64, 128, 64, 0.125, 0, None)
    for name, v in kw.items():
        setattr(g, name, v)
    return g


@pytest.mark.parametrize("kw,needle", [
    (dict(dtype=5), "dtype"), (dict(heads_q=0), "positive"), (dict(heads_q=3), "divisible"), (dict(head_dim=0), "positive"),
    (dict(head_dim=300), "256"), (dict(batch=-1), "negative"), (dict(prefix=-1), "negative"), (dict(prefix=1 << 31), "2^31"),
    (dict(batch=1 << 20, tokens=1 << 20), "2^31"), (dict(scale=0.0), "scale"), (dict(scale=float("inf")), "scale"),
    (dict(scale=float("nan")), "scale"), (dict(path=2, head_dim=68), "tcgen05"), (dict(path=2, k_token_stride=0), "stride"),
    (dict(path=2, q_token_stride=257), "stride"), (dict(path=2, dtype=0), "float32"),
])
def test_abi_refusals(kw, needle):
    before = _lib.launch_count()
    assert _lib.load().natten_b200_prefix_forward(_geom(**kw), 4096, 4096, 4096, None, None, 4096, 4096, 4096, 1 << 40, None) == _lib.EINVAL
    assert needle in _lib.last_error()
    assert _lib.launch_count() == before


def test_abi_pointers_and_scratch():
    lib = _lib.load()
    before = _lib.launch_count()
    assert lib.natten_b200_prefix_forward(None, *([None] * 8), 0, None) == _lib.EINVAL
    assert lib.natten_b200_prefix_forward(_geom(), None, 4096, 4096, None, None, 4096, None, None, 0, None) == _lib.EINVAL
    assert lib.natten_b200_prefix_forward(_geom(), 4096, 4096, 4096, 4096, None, 4096, None, None, 0, None) == _lib.EINVAL
    assert lib.natten_b200_prefix_forward(_geom(), 4096 + 8, 4096, 4096, None, None, 4096, None, None, 0, None) == _lib.EINVAL
    for geom, wl, lse in ((_geom(lens=4096 + 2), 4096, 4096), (_geom(), 4096 + 1, 4096), (_geom(), 4096, 4096 + 2)):
        assert lib.natten_b200_prefix_forward(geom, 4096, 4096, 4096, 4096, wl, 4096, lse, 4096, 1 << 40, None) == _lib.EINVAL
        assert "aligned" in _lib.last_error()
    long = _geom(prefix=100000)
    need = lib.natten_b200_prefix_scratch_bytes(long)
    assert need > 0 and need % (65 * 4) == 0
    assert lib.natten_b200_prefix_forward(long, 4096, 4096, 4096, None, None, 4096, None, 4096, need - 1, None) == _lib.ERESOURCE
    assert lib.natten_b200_prefix_forward(long, 4096, 4096, 4096, None, None, 4096, None, None, 0, None) == _lib.ERESOURCE
    assert lib.natten_b200_prefix_forward(_geom(batch=0), None, None, None, None, None, None, None, None, 0, None) == _lib.OK
    assert lib.natten_b200_prefix_scratch_bytes(_geom(batch=0)) == 0
    assert _lib.launch_count() == before


def test_struct_layouts():
    import ctypes
    assert ctypes.sizeof(_lib.PrefixGeom) == 104 and _lib.PrefixGeom.scale.offset == 88 and _lib.PrefixGeom.lens.offset == 96
    assert ctypes.sizeof(_lib.RotaryGeom) == 144 and _lib.RotaryGeom.phases.offset == 136
    assert ctypes.sizeof(_lib.Rows) == 40 and _lib.Rows.channels.offset == 32
