"""Layer norm, rotary positions, the window and a shared prefix as a block uses them: through the modules, against the
same computation written out in 64 bits around the CPU oracle, in training (without a prefix) and in serving."""

from __future__ import annotations

import copy

import pytest
import torch

import natten_oracle as oracle

import natten_mlx_b200 as nb
from natten_mlx_b200.nn import LayerNorm, NeighborhoodAttention1D, NeighborhoodAttention2D, NeighborhoodAttention3D
from natten_mlx_b200.positions import split_axis_dims

MODS = {1: NeighborhoodAttention1D, 2: NeighborhoodAttention2D, 3: NeighborhoodAttention3D}


def test_options_add_their_parameters_and_nothing_else():
    plain, full = NeighborhoodAttention2D(16, 4, 3), NeighborhoodAttention2D(16, 4, 3, qk_norm=True, rotary=True)
    assert set(full.state_dict()) - set(plain.state_dict()) == {"q_norm.weight", "q_norm.bias", "k_norm.weight", "k_norm.bias"}
    assert full.q_norm.weight.shape == (4,)
    n = LayerNorm(8, bias=False)
    assert n.weight.shape == (8,) and n.bias is None and LayerNorm(8, elementwise_affine=False).weight is None
    assert "8" in repr(n)


def test_refusals():
    m, r = NeighborhoodAttention1D(8, 2, 3), NeighborhoodAttention1D(8, 2, 3, rotary=True, attn_drop=0.5)
    x = torch.zeros(2, 6, 8)
    kv = (torch.zeros(5, 2, 4), torch.zeros(5, 2, 4))
    for mod, kw, match in [(m, dict(offsets=3), "rotary=True"), (m, dict(prefix_lens=torch.zeros(2)), "needs a prefix"),
                           (m, dict(spatial_sizes=torch.tensor([6, 5]), prefix=kv), "combined"), (r, dict(prefix=kv), "combined")]:
        with pytest.raises(ValueError, match=match):
            mod(x, **kw)


def _norm64(x, w, b, eps=1e-5):
    mean = x.mean(-1, keepdim=True)
    return (x - mean) / torch.sqrt(((x - mean) ** 2).mean(-1, keepdim=True) + eps) * w + b


def _turn64(t, origin):
    rank, d = t.dim() - 3, t.shape[-1]
    parts = []
    for a, n in enumerate(split_axis_dims(d, rank)):
        pos = torch.arange(t.shape[1 + a], dtype=torch.float64) + origin[a]
        ang = pos[:, None] * 10000.0 ** (-torch.arange(0, n, 2, dtype=torch.float64) / n)
        parts.append(ang.reshape([1] * (1 + a) + [-1] + [1] * (rank - 1 - a) + [1, n // 2]).expand(*t.shape[:-2], 1, n // 2))
    ang = torch.cat(parts, -1)
    x, y = t[..., 0::2], t[..., 1::2]
    return torch.stack((x * ang.cos() - y * ang.sin(), x * ang.sin() + y * ang.cos()), -1).flatten(-2)


def _block64(m, norm, x, origin, prefix=None):
    """norm -> projection -> norm of the heads -> rotary -> window (and prefix) -> projection, in float64."""
    w = {n: p.detach().cpu().double().requires_grad_(True) for n, p in list(m.named_parameters()) +
         [("norm." + n, p) for n, p in norm.named_parameters()]}
    xc = x.detach().cpu().double().requires_grad_(True)
    lin = lambda name, t: torch.nn.functional.linear(t, w[name + ".weight"], w.get(name + ".bias"))
    h = _norm64(xc, w["norm.weight"], w["norm.bias"])
    lead = tuple(h.shape[:-1])
    if m.qkv is not None:
        q, k, v = lin("qkv", h).view(*lead, 3, m.num_heads, m.head_dim).unbind(-3)
    else:
        q = lin("q_proj", h).view(*lead, m.num_heads, m.head_dim)
        k, v = lin("kv_proj", h).view(*lead, 2, m.num_kv_heads, m.head_dim).unbind(-3)
    q, k = _norm64(q, w["q_norm.weight"], w["q_norm.bias"]), _norm64(k, w["k_norm.weight"], w["k_norm.bias"])
    q, k = _turn64(q, origin), _turn64(k, origin)
    extra = {}
    if prefix is not None:
        extra = dict(additional_keys=prefix[0].cpu().double().expand(lead[0], *prefix[0].shape),
                     additional_values=prefix[1].cpu().double().expand(lead[0], *prefix[1].shape))
    o = oracle.na(q, k, v, m.kernel_size, m.stride, m.dilation, m.is_causal, scale=m.scale, **extra)
    return lin("proj", o.reshape(*o.shape[:-2], m.embed_dim)), xc, w


CASES = [
    (1, (2, 19, 16), dict(embed_dim=16, num_heads=4, kernel_size=5, is_causal=True), 700),
    (2, (2, 8, 9, 32), dict(embed_dim=32, num_heads=4, kernel_size=(3, 5), dilation=(2, 1), num_kv_heads=2), (3, 40)),
    (3, (1, 4, 6, 7, 24), dict(embed_dim=24, num_heads=2, kernel_size=(3, 3, 5), is_causal=(True, False, False)), None),
]


def _make(rank, kwargs, seed=3):
    torch.manual_seed(seed)
    m = MODS[rank](qk_norm=True, rotary=True, **kwargs).to("cuda").eval()
    norm = LayerNorm(m.embed_dim).to("cuda")
    with torch.no_grad():
        for p in [m.q_norm.weight, m.q_norm.bias, m.k_norm.weight, m.k_norm.bias, norm.weight, norm.bias]:
            p.add_(torch.randn_like(p) * 0.2)
    return m, norm


def _origin(offsets, rank):
    return (0,) * rank if offsets is None else (offsets,) * rank if isinstance(offsets, int) else offsets


@pytest.mark.gpu
@pytest.mark.parametrize("rank,shape,kwargs,offsets", CASES)
def test_a_block_in_training(rank, shape, kwargs, offsets):
    m, norm = _make(rank, kwargs)
    x = torch.randn(shape, generator=torch.Generator().manual_seed(5)).to("cuda").requires_grad_(True)
    y = m(norm(x), offsets=offsets)
    y_ref, x_ref, w_ref = _block64(m, norm, x, _origin(offsets, rank))
    # float32 against float64 over a chain of about ten products of up to 32 terms: the tolerance of the module tests
    assert torch.allclose(y.detach().cpu().double(), y_ref.detach(), atol=2e-4, rtol=2e-4)
    cot = torch.randn(y_ref.shape, generator=torch.Generator().manual_seed(6), dtype=torch.float64)
    y.backward(cot.float().to("cuda"))
    y_ref.backward(cot)
    assert torch.allclose(x.grad.cpu().double(), x_ref.grad, atol=1e-3, rtol=1e-3)
    for name, p in list(m.named_parameters()) + [("norm." + n, p) for n, p in norm.named_parameters()]:
        assert torch.allclose(p.grad.cpu().double(), w_ref[name].grad, atol=2e-3, rtol=2e-3), name


@pytest.mark.gpu
@pytest.mark.parametrize("rank,shape,kwargs,offsets", CASES)
def test_a_block_in_serving_with_a_prefix(rank, shape, kwargs, offsets):
    m, norm = _make(rank, kwargs)
    gen = torch.Generator().manual_seed(8)
    x = torch.randn(shape, generator=gen).to("cuda")
    prefix = tuple(torch.randn(33, m.num_kv_heads, m.head_dim, generator=gen).to("cuda") for _ in range(2))
    with torch.no_grad():
        y = m(norm(x), offsets=offsets, prefix=prefix)
        alone = m(norm(x), offsets=offsets)
        off = m(norm(x), offsets=offsets, prefix=prefix, prefix_lens=torch.zeros(shape[0], dtype=torch.int32, device="cuda"))
    y_ref, _, _ = _block64(m, norm, x, _origin(offsets, rank), prefix)
    assert torch.allclose(y.cpu().double(), y_ref.detach(), atol=2e-4, rtol=2e-4)
    assert torch.allclose(off, alone, atol=1e-6, rtol=1e-6)        # a prefix of which no sample sees anything
    with pytest.raises(RuntimeError, match="no gradients"):
        m(norm(x), offsets=offsets, prefix=prefix)


@pytest.mark.gpu
def test_a_strided_block_with_a_prefix():
    m = NeighborhoodAttention2D(16, 4, 3, stride=(2, 3), qk_norm=True, rotary=True).to("cuda").eval()
    x = torch.randn(2, 7, 8, 16, generator=torch.Generator().manual_seed(1)).to("cuda")
    prefix = tuple(torch.randn(9, 4, 4, generator=torch.Generator().manual_seed(s)).to("cuda") for s in (2, 3))
    with torch.no_grad():
        y = m(x, prefix=prefix)
        q, k, v = m._heads(x)
        q, k = nb.rotary(m.q_norm(q), m.k_norm(k))
        o, l = nb.na2d(q, k, v, 3, stride=(2, 3), return_lse=True)
        po, pl = nb.prefix_attention(q[:, ::2, ::3], *prefix, return_lse=True)
        want = m.proj(nb.merge_attentions([o, po], [l, pl])[0].reshape(2, 4, 3, 16))
    assert y.shape == (2, 4, 3, 16) and torch.allclose(y, want, atol=1e-5, rtol=1e-5)


@pytest.mark.gpu
def test_a_block_in_bfloat16_step_by_step():
    """Serving one token at a time: norm, projection, rotary at the token's place, the shared prompt.  The prompt's keys
    were turned at positions 0..P-1, the new token sits behind them; all in 16 bits with norms in 32."""
    torch.manual_seed(2)
    b, p, heads, kv, d = 5, 300, 8, 2, 64
    norm = LayerNorm(heads * d).to("cuda")                          # float32 weights beside bfloat16 activations
    proj = torch.nn.Linear(heads * d, (heads + 2 * kv) * d).to("cuda", torch.bfloat16)
    prompt, new = torch.randn(1, p, heads * d, device="cuda", dtype=torch.bfloat16), torch.randn(b, 1, heads * d, device="cuda", dtype=torch.bfloat16)

    def heads_of(x, start):
        t = proj(norm(x)).view(*x.shape[:-1], heads + 2 * kv, d)
        q, k = nb.rotary(t[..., :heads, :], t[..., heads:heads + kv, :], offsets=start)
        return q, k, t[..., heads + kv:, :]

    with torch.no_grad():
        _, pk, pv = heads_of(prompt, 0)
        at = torch.full((b, 1), p, dtype=torch.int32, device="cuda")
        q, k, v = heads_of(new, at)
        # the token's own key is its window: an output of v and the token's logit
        own_lse = (q.float().view(b, 1, kv, heads // kv, d) * k.float().unsqueeze(-2)).sum(-1).flatten(-2) * d ** -0.5
        own = v.repeat_interleave(heads // kv, dim=-2)
        out = nb.prefix_attention(q, pk[0], pv[0], window=(own, own_lse))
        keys = torch.cat([pk.expand(b, p, kv, d), k], 1).double().repeat_interleave(heads // kv, dim=-2)
        vals = torch.cat([pv.expand(b, p, kv, d), v], 1).double().repeat_interleave(heads // kv, dim=-2)
        w = torch.softmax(torch.einsum("bqhd,bkhd->bhqk", q.double(), keys) * d ** -0.5, -1)
        want = torch.einsum("bhqk,bkhd->bqhd", w, vals)
        size = torch.einsum("bhqk,bkhd->bqhd", w, vals.abs())
    # weights and result rounded to bfloat16 once each (2^-8), float32 sums far below
    assert bool(((out.double() - want).abs() <= 2.0 ** -8 * want.abs() + (2.0 ** -8 + 2.0 ** -12) * size).all())


@pytest.mark.gpu
def test_modules_can_be_copied_and_loaded():
    m, norm = _make(2, dict(embed_dim=16, num_heads=2, kernel_size=3))
    n = copy.deepcopy(m)
    n.load_state_dict(m.state_dict())
    x = torch.randn(1, 5, 6, 16, device="cuda")
    with torch.no_grad():
        assert torch.equal(m(norm(x)), n(norm(x)))


@pytest.mark.gpu
def test_rows_further_apart_than_32_bits_reach():
    """Views whose last rows start past 2^31 elements give the bits of their dense copies."""
    far = 2 ** 30
    room = torch.empty(2 * far + 8192, dtype=torch.bfloat16, device="cuda")

    def apart(dense):
        view = room.as_strided(dense.shape, (far,) + dense.stride()[1:])
        return view.copy_(dense)

    gen = torch.Generator("cuda").manual_seed(5)
    x = torch.randn(3, 1000, generator=gen, device="cuda").bfloat16()
    w = torch.randn(1000, generator=gen, device="cuda")
    g = torch.randn(3, 1000, generator=gen, device="cuda").bfloat16()
    got, want = [], []
    for rows, results in ((apart(x), got), (x, want)):
        rows = rows.detach().requires_grad_(True)
        y = nb.layer_norm(rows, w)
        results += [y.detach(), *torch.autograd.grad(y, rows, g)]
    qk = torch.randn(3, 2, 64, generator=gen, device="cuda").bfloat16()
    got += [nb.rotary(apart(qk)[None], qk[None])[0], nb.rotary(qk[None], apart(qk)[None])[1]]
    want += [nb.rotary(qk[None], qk[None])[0]] * 2
    q = torch.randn(2, 5, 4, 64, generator=gen, device="cuda").bfloat16()
    for path in ("tcgen05", "simt"):
        nb.set_fused_path(path)
        try:
            got += [nb.prefix_attention(q, apart(qk), qk), nb.prefix_attention(q, qk, apart(qk)),
                    nb.prefix_attention(apart(qk)[None], qk, qk)]
            want += [nb.prefix_attention(q, qk, qk)] * 2 + [nb.prefix_attention(qk[None], qk, qk)]
        finally:
            nb.set_fused_path("auto")
    for i, (a, b) in enumerate(zip(got, want)):
        assert torch.equal(a, b), i
