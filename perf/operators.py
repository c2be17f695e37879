"""Cases and plain forms of the operators that stand around neighborhood attention in a block: layer norm, rotary
positions over the axes of a sequence, an image or a video, and attention to a prefix that the whole batch shares.

``run`` computes a case either in plain torch operations (``own`` false) or by the calls that a user makes of this
package (``own`` true).  ``exact`` gives the same results in 64 bits, from the definitions.
"""

from __future__ import annotations

import math
import os
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
EPS = 1e-5


def _package():
    """This repository's package; its folder is not on the path of a program that starts in the repository's root."""
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "natten-mlx_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import natten_mlx_b200
    return natten_mlx_b200


# ---------------------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------------------
# Shapes are texts, "2x32x96x96", so that a case stays a dict of plain values.

def _case(name, **values):
    return dict(values) if name is None else dict(name=name, **values)


def _norm(name, lead, channels, dtype, weights, train, packed=0):
    """``packed`` > 0: the rows are the heads of q inside the output of a fused q/k/v projection with so many heads."""
    return _case(name, op="norm", lead=lead, channels=channels, dtype=dtype, weights=weights, train=train,
                 packed=packed)


def _rotary(name, lead, heads, kv_heads, head_dim, axis_dims, dtype, source, interleaved, train, packed=False):
    """``source``: where positions come from: "grid" (the index on each axis), "offset" (the index plus a start for
    each sample) or "given" (a tensor with the position of every token on every axis)."""
    return _case(name, op="rotary", lead=lead, heads=heads, kv_heads=kv_heads, head_dim=head_dim, axis_dims=axis_dims,
                 dtype=dtype, source=source, interleaved=interleaved, train=train, packed=packed)


def _prefix(name, lead, heads, kv_heads, head_dim, tokens, dtype, lens, window):
    """``lens``: samples see only their first tokens of the prefix, some none.  ``window``: the result is merged with
    that of the queries' own window."""
    return _case(name, op="prefix", lead=lead, heads=heads, kv_heads=kv_heads, head_dim=head_dim, tokens=tokens,
                 dtype=dtype, lens=lens, window=window)


def listed():
    return [
        # one new token of 64 sequences in serving, 16 heads of 64 channels: the launch is what counts
        _norm("norm_step", "64x1", 1024, "bf16", "bf16", False),
        # the benchmark's image stage, 4 heads of 32 channels, trained with weights in 32 bits
        _norm("norm_nat_stage", "32x56x56", 128, "bf16", "f32", True),
        # half of the benchmark's video batch, 16 heads of 64 channels: the largest rows-by-channels
        _norm("norm_video", "1x32x96x96", 1024, "bf16", "bf16", True),
        # queries normalised head by head before attention, read out of the fused projection of the image stage
        _norm("norm_heads", "32x56x56x4", 32, "f16", "f32", True, packed=4),
        # an odd number of rows of an odd width in 32 bits
        _norm("norm_odd", "7x331", 1001, "f32", "f32", True),
        # one new token of 64 sequences, each at a place of its own, with grouped heads
        _rotary("rotary_step", "64x1", 16, 4, 64, "64", "bf16", "offset", True, False),
        # the image stage, q and k as they lie in the fused projection
        _rotary("rotary_nat_stage", "32x56x56", 4, 4, 32, "16x16", "bf16", "grid", True, True, packed=True),
        # the benchmark's video batch: time, height and width share the 64 channels
        _rotary("rotary_video", "2x32x96x96", 16, 16, 64, "24x20x20", "bf16", "grid", True, True),
        # text and video tokens in one sequence, a position on three axes for each token, the halves of a head paired
        _rotary("rotary_mixed", "3x4099", 12, 4, 80, "16x24x24", "f32", "given", False, True),
        # one new token of 32 sequences behind a long shared prompt, merged with the attention to their own tokens
        _prefix("prefix_step", "32x1", 16, 4, 128, 65536, "f16", False, True),
        # a piece of the video volume with conditioning tokens that the batch shares, merged with the window's result
        _prefix("prefix_video", "2x8x32x32", 16, 16, 64, 4096, "bf16", False, True),
        # images in 32 bits with an odd head size, of which one sees the whole prefix, one a part and one nothing
        _prefix("prefix_odd", "3x13x17", 6, 2, 24, 1531, "f32", True, False),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _grid(rng, rank, tokens):
    """``rank`` extents whose product is at most ``tokens``."""
    ext = []
    left = tokens
    for a in range(rank, 1, -1):
        e = _log_int(rng, 1, max(1, min(96, int(left ** (1.0 / a) * 2))))
        ext.append(e)
        left = max(1, left // e)
    ext.append(max(1, left))
    rng.shuffle(ext)
    return ext


def _text(seq):
    return "x".join(str(int(s)) for s in seq)


def draw(rng):
    op = rng.choice(["norm", "norm", "rotary", "rotary", "prefix", "prefix"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op == "norm":
        weights = rng.choice([dtype, "f32"])
        train = rng.random() < 0.6
        most = 300_000_000 // (2 if dtype == "f32" else 1)
        if rng.random() < 0.3:
            heads, dim = rng.randint(1, 16), rng.choice([16, 24, 32, 48, 64, 80, 96, 128])
            tokens = _log_int(rng, 1, min(200_000, most // (3 * heads * dim)))
            return _norm(None, _text([tokens, heads]), dim, dtype, weights, train, packed=heads)
        channels = _log_int(rng, 16, 8192)
        if rng.random() < 0.6:
            channels = max(16, channels // 16 * 16)
        rows = _log_int(rng, 1, min(400_000, most // channels))
        return _norm(None, _text(_grid(rng, rng.randint(1, 3), rows)), channels, dtype, weights, train)
    if op == "rotary":
        rank = rng.randint(1, 3)
        kv = rng.choice([1, 2, 4, 8])
        heads = kv * rng.choice([1, 1, 2, 3, 4])
        dim = rng.choice([16, 24, 32, 48, 64, 80, 96, 128])
        source = rng.choice(["grid", "grid", "offset", "given"])
        axes = rank if source != "given" else rng.randint(1, 3)
        even = [2 * rng.randint(1, max(1, dim // (2 * axes))) for _ in range(axes)]
        most = 1_200_000_000 // (4 if dtype == "f32" else 2)
        batch = _log_int(rng, 1, 64)
        tokens = _log_int(rng, 1, max(1, min(300_000, most // ((heads + kv) * dim * batch))))
        packed = heads == kv and rng.random() < 0.4
        return _rotary(None, _text([batch] + _grid(rng, rank, tokens)), heads, kv, dim, _text(even), dtype, source,
                       rng.random() < 0.5, rng.random() < 0.5, packed)
    kv = rng.choice([1, 2, 4, 8, 16])
    heads = kv * rng.choice([1, 1, 2, 3, 4, 8])
    dim = rng.choice([24, 32, 40, 64, 64, 80, 128, 128])
    tokens = _log_int(rng, 1, 65536)
    batch = _log_int(rng, 1, 64)
    most = 130e9 if dtype != "f32" else 8e9           # operations; in 32 bits a case costs far more for each
    rows = max(1, int(min(most / (4.0 * heads * dim * tokens), 5e8 / (heads * tokens), 4e7 / (heads * dim)) / batch))
    rank = rng.randint(1, 3)
    ext = [1] * rank if rng.random() < 0.4 else _grid(rng, rank, _log_int(rng, 1, min(rows, 20_000)))
    return _prefix(None, _text([batch] + ext), heads, kv, dim, tokens, dtype, rng.random() < 0.4, rng.random() < 0.5)


def _ints(text):
    return [int(s) for s in str(text).split("x")]


# ---------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------

def _inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed) * 1000003 + 17)
    dt = DTYPES[case["dtype"]]

    def normal(shape, std=1.0, mean=0.0, dtype=dt):
        return torch.empty(shape, dtype=dtype, device="cuda").normal_(mean, std, generator=gen)

    lead = _ints(case["lead"])
    s = {"op": case["op"]}
    if case["op"] == "norm":
        c, heads = case["channels"], case["packed"]
        s["train"] = case["train"]
        if heads:
            qkv = normal(lead[:-1] + [3, heads, c])
            s["x"] = qkv.select(-3, 0)
        else:
            # a residual stream: its channels differ in size and have means of their own
            s["x"] = normal(lead + [c]).mul_(normal([c], 0.5).exp_()).add_(normal([c], 0.3))
        wt = DTYPES[case["weights"]]
        s["weight"], s["bias"] = normal([c], 0.2, 1.0, wt), normal([c], 0.2, 0.0, wt)
        if s["train"]:
            s["grad"] = normal(lead + [c])
    elif case["op"] == "rotary":
        hq, hk, d = case["heads"], case["kv_heads"], case["head_dim"]
        s["train"], s["interleaved"] = case["train"], case["interleaved"]
        s["axis_dims"] = tuple(_ints(case["axis_dims"]))
        if case["packed"]:
            qkv = normal(lead + [3, hq, d])
            s["q"], s["k"] = qkv.select(-3, 0), qkv.select(-3, 1)
        else:
            s["q"], s["k"] = normal(lead + [hq, d]), normal(lead + [hk, d])
        rank, axes = len(lead) - 1, len(s["axis_dims"])
        s["offsets"] = s["positions"] = None
        if case["source"] == "offset":
            s["offsets"] = torch.randint(0, 100_000, (lead[0], rank), generator=gen, device="cuda", dtype=torch.int32)
        elif case["source"] == "given":
            s["positions"] = torch.randint(0, 32_768, lead + [axes], generator=gen, device="cuda", dtype=torch.int64)
        if s["train"]:
            s["grad_q"], s["grad_k"] = normal(lead + [hq, d]), normal(lead + [hk, d])
    else:
        hq, hk, d, n = case["heads"], case["kv_heads"], case["head_dim"], case["tokens"]
        s["q"] = normal(lead + [hq, d], 1.4)
        s["k"], s["v"] = normal([n, hk, d], 1.4), normal([n, hk, d])
        s["lens"] = s["window"] = None
        if case["lens"]:
            lens = torch.randint(0, n + 1, (lead[0],), generator=gen, device="cuda", dtype=torch.int32)
            lens[0] = n
            lens[-1] = 0
            s["lens"] = lens
        if case["window"]:
            s["window"] = (normal(lead + [hq, d], 0.5), normal(lead + [hq], 0.7, 4.0, torch.float32))
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if s.get("train"):
        for name in ("x", "weight", "bias", "q", "k"):
            if name in s:
                s[name].requires_grad_(True)
    return s


# ---------------------------------------------------------------------------------------------------------------------
# the operators
# ---------------------------------------------------------------------------------------------------------------------

def run(state):
    return {"norm": _run_norm, "rotary": _run_rotary, "prefix": _run_prefix}[state["op"]](state)


def _run_norm(s):
    x, w, b = s["x"], s["weight"], s["bias"]
    if own:
        y = _package().layer_norm(x, w, b, eps=EPS)
        if not s["train"]:
            return {"y": y}
        dx, dw, db = torch.autograd.grad(y, (x, w, b), s["grad"])
        return {"y": y, "dx": dx, "dw": dw, "db": db}
    with torch.no_grad():
        xf, wf = x.float(), w.float()
        xc = xf - xf.mean(-1, keepdim=True)
        rstd = torch.rsqrt((xc * xc).mean(-1, keepdim=True) + EPS)
        xhat = xc * rstd
        y = (xhat * wf + b.float()).to(x.dtype)
        if not s["train"]:
            return {"y": y}
        g = s["grad"].float()
        gw = g * wf
        dx = rstd * (gw - gw.mean(-1, keepdim=True) - xhat * (gw * xhat).mean(-1, keepdim=True))
        c = x.shape[-1]
        dw, db = (g * xhat).reshape(-1, c).sum(0), g.reshape(-1, c).sum(0)
        return {"y": y, "dx": dx.to(x.dtype), "dw": dw.to(w.dtype), "db": db.to(w.dtype)}


def _angles(s, sign):
    """cos and sin of every token's angles, [B or 1, spatial..., 1, pairs], float32 from angles in 64 bits."""
    lead, dev = s["q"].shape[:-2], s["q"].device
    parts = []
    for a, d in enumerate(s["axis_dims"]):
        freq = torch.pow(10000.0, torch.arange(0, d, 2, dtype=torch.float64, device=dev) / -d)
        if s["positions"] is not None:
            pos = s["positions"][..., a].double()
        else:
            pos = torch.arange(lead[1 + a], dtype=torch.float64, device=dev)
            pos = pos.reshape([1] * (1 + a) + [-1] + [1] * (len(lead) - 2 - a))
            if s["offsets"] is not None:
                pos = pos + s["offsets"][:, a].double().reshape([-1] + [1] * (len(lead) - 1))
            pos = pos.expand([pos.shape[0]] + list(lead[1:]))
        parts.append(pos.unsqueeze(-1) * freq)
    ang = torch.cat(parts, -1).unsqueeze(-2)
    return ang.cos().float(), ang.sin().float() * sign


def _rotate(t, cos, sin, width, interleaved):
    half = width // 2
    f = t.float()
    if interleaved:
        a, b = f[..., 0:width:2], f[..., 1:width:2]
        turned = torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)
    else:
        a, b = f[..., :half], f[..., half:width]
        turned = torch.cat((a * cos - b * sin, a * sin + b * cos), -1)
    return torch.cat((turned, f[..., width:]), -1).to(t.dtype)


def _run_rotary(s):
    q, k = s["q"], s["k"]
    if own:
        yq, yk = _package().rotary(q, k, s["axis_dims"], interleaved=s["interleaved"], offsets=s["offsets"],
                                   positions=s["positions"])
        if not s["train"]:
            return {"q": yq, "k": yk}
        dq, dk = torch.autograd.grad((yq, yk), (q, k), (s["grad_q"], s["grad_k"]))
        return {"q": yq, "k": yk, "dq": dq, "dk": dk}
    with torch.no_grad():
        width, il = sum(s["axis_dims"]), s["interleaved"]
        cos, sin = _angles(s, 1.0)
        res = {"q": _rotate(q, cos, sin, width, il), "k": _rotate(k, cos, sin, width, il)}
        if s["train"]:
            cos, sin = _angles(s, -1.0)
            res["dq"], res["dk"] = _rotate(s["grad_q"], cos, sin, width, il), _rotate(s["grad_k"], cos, sin, width, il)
        return res


def _run_prefix(s):
    q, k, v = s["q"], s["k"], s["v"]
    if own:
        out, lse = _package().prefix_attention(q, k, v, return_lse=True, prefix_lens=s["lens"], window=s["window"])
        return {"out": out, "lse": lse}
    hq, d = q.shape[-2:]
    n, hk, _ = k.shape
    batch, group = q.shape[0], hq // hk
    tokens = q[..., 0, 0].numel() // batch
    # [kv head, batch * tokens * group, ...]: the batch's queries of a kv head are the rows of one product
    rows = q.float().reshape(batch * tokens, hk, group, d).transpose(0, 1).reshape(hk, -1, d)
    logits = torch.matmul(rows, k.float().permute(1, 2, 0)) * d ** -0.5
    if s["lens"] is not None:
        limit = s["lens"].repeat_interleave(tokens * group)
        logits = logits.masked_fill(torch.arange(n, device=q.device) >= limit[:, None], -math.inf)
    top = logits.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    p = torch.exp(logits - top)
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p, v.float().transpose(0, 1)) / torch.where(total == 0, torch.ones_like(total), total)
    lse = (top + torch.log(total)).squeeze(-1)
    o = o.reshape(hk, batch * tokens, group, d).transpose(0, 1).reshape(q.shape)
    lse = lse.reshape(hk, batch * tokens, group).transpose(0, 1).reshape(q.shape[:-1])
    if s["window"] is not None:
        ow, lw = s["window"]
        both = torch.logaddexp(lse, lw)
        o = o * torch.exp(lse - both).unsqueeze(-1) + ow.float() * torch.exp(lw - both).unsqueeze(-1)
        lse = both
    return {"out": o.to(q.dtype), "lse": lse}


# ---------------------------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------------------------------

def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    lead = _ints(case["lead"])
    n = math.prod(lead)
    if case["op"] == "norm":
        c = case["channels"]
        wsize = 4 if case["weights"] == "f32" else 2
        forward = {"bytes": 2 * n * c * size + 2 * c * wsize, "flops": 8 * n * c}
        if not case["train"]:
            return forward
        return {"bytes": 4 * n * c * size + 4 * c * wsize, "flops": 22 * n * c}
    if case["op"] == "rotary":
        elems = n * (case["heads"] + case["kv_heads"]) * case["head_dim"]
        axes = len(_ints(case["axis_dims"]))
        extra = 8 * n * axes if case["source"] == "given" else 4 * lead[0] * axes if case["source"] == "offset" else 0
        passes = 2 if case["train"] else 1
        return {"bytes": passes * (2 * elems * size + extra), "flops": passes * 3 * elems}
    hq, hk, d, p = case["heads"], case["kv_heads"], case["head_dim"], case["tokens"]
    q_bytes = n * hq * d * size
    total = 2 * q_bytes + 2 * p * hk * d * size + n * hq * 4
    if case["window"]:
        total += q_bytes + n * hq * 4
    # lengths are drawn anew for each seed: half of the prefix on average, the first sample all, the last nothing
    seen = 1.0 if not case["lens"] else (0.0 if lead[0] == 1 else (1.0 + 0.5 * (lead[0] - 2)) / lead[0])
    if not seen:
        total -= 2 * p * hk * d * size
    return {"bytes": total, "flops": 4.0 * n * hq * p * d * seen}


# ---------------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------------------------------------------------

def exact(case, seed):
    s = _inputs(case, seed)
    return {"norm": _exact_norm, "rotary": _exact_rotary, "prefix": _exact_prefix}[s["op"]](s)


def _exact_norm(s):
    x = s["x"].double().requires_grad_(s["train"])
    w, b = s["weight"].double().requires_grad_(s["train"]), s["bias"].double().requires_grad_(s["train"])
    var, mean = torch.var_mean(x, dim=-1, correction=0, keepdim=True)
    y = (x - mean) / torch.sqrt(var + EPS) * w + b
    if not s["train"]:
        return {"y": y}
    dx, dw, db = torch.autograd.grad(y, (x, w, b), s["grad"].double())
    return {"y": y.detach(), "dx": dx, "dw": dw, "db": db}


def _exact_rotary(s):
    q = s["q"]
    lead, width, axes = list(q.shape[:-2]), sum(s["axis_dims"]), len(s["axis_dims"])
    batch, n = lead[0], math.prod(lead[1:])
    # the position of every token on every axis, [B, tokens, axes]
    if s["positions"] is not None:
        pos = s["positions"].reshape(batch, n, axes)
    else:
        idx = torch.arange(n, device=q.device)
        coords = torch.stack(torch.unravel_index(idx, lead[1:]), -1)
        pos = coords.unsqueeze(0).expand(batch, n, axes)
        if s["offsets"] is not None:
            pos = pos + s["offsets"].long().unsqueeze(1)
    pairs = [(a, 10000.0 ** (-2.0 * j / d)) for a, d in enumerate(s["axis_dims"]) for j in range(d // 2)]
    axis = torch.tensor([a for a, _ in pairs], device=q.device)
    freq = torch.tensor([f for _, f in pairs], dtype=torch.float64, device=q.device)

    def turn(t, direction):
        out = t.double().reshape(batch, n, t.shape[-2], t.shape[-1]).clone()
        for i in range(batch):
            phase = pos[i][:, axis].double() * freq * direction
            unit = torch.polar(torch.ones_like(phase), phase).unsqueeze(1)
            for first in range(0, n, 65536):
                part = out[i, first:first + 65536]
                if s["interleaved"]:
                    z = torch.view_as_complex(part[..., :width].reshape(*part.shape[:-1], width // 2, 2).contiguous())
                    part[..., :width] = torch.view_as_real(z * unit[first:first + 65536]).flatten(-2)
                else:
                    z = torch.complex(part[..., :width // 2], part[..., width // 2:width]) * unit[first:first + 65536]
                    part[..., :width] = torch.cat((z.real, z.imag), -1)
        return out.reshape(t.shape)

    res = {"q": turn(s["q"], 1.0), "k": turn(s["k"], 1.0)}
    if s["train"]:
        res["dq"], res["dk"] = turn(s["grad_q"], -1.0), turn(s["grad_k"], -1.0)
    return res


def _exact_prefix(s):
    q, k, v = s["q"], s["k"].double(), s["v"].double()
    hq, d = q.shape[-2:]
    n, hk, _ = k.shape
    flat = q.reshape(q.shape[0], -1, hq, d)
    batch, tokens = flat.shape[:2]
    out = torch.zeros(batch, tokens, hq, d, dtype=torch.float64, device=q.device)
    lse = torch.full((batch, tokens, hq), -math.inf, dtype=torch.float64, device=q.device)
    lens = [n] * batch if s["lens"] is None else s["lens"].tolist()
    step = max(1, 200_000_000 // n)
    for i in range(batch):
        m = lens[i]
        if m == 0:
            continue
        for h in range(hq):
            kh, vh = k[:m, h // (hq // hk)], v[:m, h // (hq // hk)]
            for first in range(0, tokens, step):
                x = flat[i, first:first + step, h].double() @ kh.T / math.sqrt(d)
                out[i, first:first + step, h] = torch.softmax(x, -1) @ vh
                lse[i, first:first + step, h] = torch.logsumexp(x, -1)
    if s["window"] is not None:
        ow, lw = s["window"][0].double().reshape(out.shape), s["window"][1].double().reshape(lse.shape)
        share = torch.softmax(torch.stack((lse, lw), -1), -1)
        out = out * share[..., :1] + ow * share[..., 1:]
        lse = torch.logsumexp(torch.stack((lse, lw), -1), -1)
    return {"out": out.reshape(q.shape), "lse": lse.reshape(q.shape[:-1])}
