"""Operators of a transformer around its quantized linears, as measurable cases.

A case is one pass of an operator of this package beside its plain form: elementary torch
operations in 32 bits, rounded once at the end.

  w8a8        a linear of 8-bit integers: activations quantized row by row (one scale a token),
              weights with one scale an output channel, integer sums, float epilogue
  rotary      per-head RMS norm of queries and keys, then rotary positions of several axes, read
              from a fused projection; with "train" also the gradients
  layer_norm  layer norm with a weight and bias, or with one shift and scale a group of rows (the
              adaptive form); with "train" also the gradients

Fields of a case
  op        "w8a8", "rotary" or "layer_norm"
  dtype     type of activations and outputs (weights of the norms have it too)
  rows, k, n, codes, residual       w8a8: token rows, input and output features; whether the rows
            come as codes and scales already; "none", "add" or "gate" (residual + gate * linear)
  batch, length, heads, kv_heads, dim, axes, norm, interleaved, train    rotary: the axes' share of
            the features of a head (0 for an axis left out); pairs (2i, 2i + 1), or (i, i + half)
  rows, k, form, vectors, train     layer_norm: "affine" or "modulate", groups of rows
"""

from __future__ import annotations

import math
import os
import sys

import torch

own = False

_DTYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}
_EPS = 1e-6
_W8A8 = {"op": "w8a8", "rows": 1, "k": 3072, "n": 3072, "dtype": "bfloat16", "codes": False, "residual": "none"}
_ROTARY = {"op": "rotary", "batch": 1, "length": 4608, "heads": 24, "kv_heads": 24, "dim": 128, "axis_t": 16,
           "axis_h": 56, "axis_w": 56, "dtype": "bfloat16", "norm": True, "interleaved": True, "train": False}
_NORM = {"op": "layer_norm", "rows": 512, "k": 3072, "dtype": "bfloat16", "form": "modulate", "vectors": 1,
         "train": False}


def listed() -> list[dict]:
    return [
        # An adaLN modulation layer on its single conditioning row: the smallest linear, launches and weight latency.
        {**_W8A8, "name": "w8a8 1 row", "n": 18432},
        # A few requests' single tokens through a contraction: the weights' bytes bound it.
        {**_W8A8, "name": "w8a8 24 rows float16", "rows": 24, "k": 12288, "dtype": "float16"},
        # A short prompt through a fused qkv projection: fewer rows than a tile, an odd number.
        {**_W8A8, "name": "w8a8 77 rows", "rows": 77, "n": 9216},
        # The second linear of a single block, gated back into the stream.
        {**_W8A8, "name": "w8a8 1536 rows gated", "rows": 1536, "k": 15360, "residual": "gate"},
        # The up projection at 4096 image and 512 text tokens.
        {**_W8A8, "name": "w8a8 4608 rows", "rows": 4608, "n": 12288},
        # A ragged video shape in float16 with an odd number of outputs: no dimension fills whole tiles.
        {**_W8A8, "name": "w8a8 10017 rows odd", "rows": 10017, "k": 2688, "n": 2685, "dtype": "float16"},
        # The product alone, on codes that several projections share: a video model's contraction, the largest.
        {**_W8A8, "name": "w8a8 codes 8800 rows", "rows": 8800, "k": 16384, "n": 4096, "codes": True},
        # One new token of each of 16 sequences: latency; grouped keys, 64 features, half-split pairs, no norm.
        {**_ROTARY, "name": "rotary 16 single tokens", "batch": 16, "length": 1, "heads": 32, "kv_heads": 8,
         "dim": 64, "axis_t": 16, "axis_h": 24, "axis_w": 24, "dtype": "float16", "norm": False,
         "interleaved": False},
        # The joint text and image sequence of a diffusion transformer's block.
        {**_ROTARY, "name": "rotary 4608 tokens"},
        # A training step of a video model's attention at 7800 tokens of 5120 features.
        {**_ROTARY, "name": "rotary 7800 tokens train", "length": 7800, "heads": 40, "kv_heads": 40, "axis_t": 44,
         "axis_h": 42, "axis_w": 42, "train": True},
        # The text stream's adaptive norm.
        {**_NORM, "name": "norm 512 rows modulated"},
        # A training step of a video model's norm with weight and bias.
        {**_NORM, "name": "norm 8800 rows train", "rows": 8800, "k": 5120, "form": "affine", "train": True},
    ]


_MOST = 8800 * 16384 * 4096


def draw(rng) -> dict:
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["w8a8", "w8a8", "rotary", "layer_norm"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    if op == "w8a8":
        case = {**_W8A8, "dtype": dtype, "rows": rng.choice([1, spread(1, 64), spread(1, 10017), spread(64, 10017)])}
        k = spread(512, 16384)
        k = k // 128 * 128 if rng.random() < 0.75 else k // 16 * 16
        n = spread(512, 21504)
        n = n // 64 * 64 if rng.random() < 0.7 else n
        while case["rows"] * k * n > _MOST:
            k, n = max(512, k // 32 * 16), max(512, n // 2)
        case["k"], case["n"] = k, n
        case["codes"] = rng.random() < 0.2
        case["residual"] = rng.choice(["none", "none", "add", "gate"])
        return case
    if op == "rotary":
        axes = rng.choice([(16, 56, 56), (44, 42, 42), (16, 24, 24), (0, 32, 32), (20, 30, 30), (128, 0, 0),
                           (32, 16, 16), (64, 96, 96)])
        kv = rng.choice([1, 2, 4, 8, 24, 40])
        heads = kv * rng.choice([1, 1, 2, 4]) if kv <= 8 else kv
        case = {**_ROTARY, "dtype": dtype, "axis_t": axes[0], "axis_h": axes[1], "axis_w": axes[2], "heads": heads,
                "kv_heads": kv, "norm": rng.random() < 0.7, "interleaved": rng.random() < 0.6,
                "train": rng.random() < 0.5}
        # most models turn every feature of a head; some leave a part as it is
        case["dim"] = sum(axes) if sum(axes) % 16 or rng.random() < 0.75 else 2 * sum(axes)
        case["dim"] = min(case["dim"], 256)
        case["length"] = rng.choice([1, spread(1, 64), spread(64, 8192), spread(64, 8192)])
        case["batch"] = spread(1, 64) if case["length"] <= 64 else rng.choice([1, 1, 2, 3])
        while case["batch"] * case["length"] * (heads + kv) * case["dim"] > 7800 * 80 * 128:
            case["length"] = max(1, case["length"] // 2)
        return case
    case = {**_NORM, "dtype": dtype, "form": rng.choice(["affine", "modulate"]), "train": rng.random() < 0.6}
    case["rows"] = rng.choice([spread(1, 64), spread(64, 16384), spread(64, 16384)])
    k = spread(256, 12288)
    case["k"] = k // 64 * 64 if rng.random() < 0.7 else k
    while case["rows"] * case["k"] > 8800 * 5120:
        case["rows"] //= 2
    if case["form"] == "modulate":
        case["vectors"] = rng.choice([1, 1, 2, 3])
        case["rows"] = max(1, case["rows"] // case["vectors"]) * case["vectors"]
    return case


# ------------------------------------------------------------------ inputs


def _activation(gen, rows, k, dtype):
    """N(0, 1) with one channel in 200 twenty times as large: a transformer's outlier channels."""
    gain = torch.ones(k, device="cuda")
    gain[torch.randperm(k, generator=gen, device="cuda")[: max(1, k // 200)]] = 20.0
    return (torch.randn((rows, k), generator=gen, device="cuda") * gain).to(dtype)


def _positions(case: dict, gen) -> torch.Tensor:
    """[B, L, 3] positions: frames of a 32 x 32 patch grid behind each other; a single token of each
    sequence stands at a place of its own."""
    b, length = case["batch"], case["length"]
    at = torch.arange(length, device="cuda")[None].expand(b, -1)
    if length == 1:
        at = torch.randint(0, 8192, (b, 1), generator=gen, device="cuda")
    return torch.stack([at // 1024, at // 32 % 32, at % 32], dim=-1)


def _table(case: dict, pos: torch.Tensor) -> torch.Tensor:
    """[B, L, pairs, 2] float32 cosines and sines, the angles in 64 bits (a program makes them once a step)."""
    parts = []
    for a, d in enumerate((case["axis_t"], case["axis_h"], case["axis_w"])):
        if d:
            omega = 10000.0 ** (-torch.arange(0, d, 2, dtype=torch.float64, device=pos.device) / d)
            ang = pos[..., a, None].to(torch.float64) * omega
            parts.append(torch.stack([torch.cos(ang), torch.sin(ang)], dim=-1))
    return torch.cat(parts, dim=-2).float().contiguous()


def prepare(case: dict, seed: int) -> dict:
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = _DTYPES[case["dtype"]]

    def normal(*shape, std=1.0, mean=0.0, kind=dtype):
        return (torch.randn(shape, generator=gen, device="cuda") * std + mean).to(kind)

    s = {"case": case, "dtype": dtype}
    if case["op"] == "w8a8":
        rows, k, n = case["rows"], case["k"], case["n"]
        weight = torch.randn((n, k), generator=gen, device="cuda") * 0.02
        scale = weight.abs().amax(dim=1) / 127
        s["qweight"] = torch.round(weight / scale[:, None]).clamp(-127, 127).to(torch.int8)
        s["wscales"], s["bias"] = scale, normal(n, std=0.02, kind=torch.float32)
        x = _activation(gen, rows, k, dtype)
        if case["codes"]:
            xs = x.float().abs().amax(dim=1) / 127
            s["qact"] = torch.round(x.float() / xs[:, None]).clamp(-127, 127).to(torch.int8)
            s["xscales"] = xs
        else:
            s["x"] = x
        s["residual"] = normal(rows, n) if case["residual"] != "none" else None
        s["gate"] = normal(1, n, std=0.5) if case["residual"] == "gate" else None
        return s
    if case["op"] == "rotary":
        b, length, hq, hk, d = case["batch"], case["length"], case["heads"], case["kv_heads"], case["dim"]
        qkv = normal(b, length, (hq + 2 * hk) * d, std=1.5)
        s["q"] = qkv[..., : hq * d].unflatten(-1, (hq, d)).transpose(1, 2)  # views of the projection's output
        s["k"] = qkv[..., hq * d: (hq + hk) * d].unflatten(-1, (hk, d)).transpose(1, 2)
        s["table"] = _table(case, _positions(case, gen))
        s["q_weight"], s["k_weight"] = (normal(d, std=0.1, mean=1.0) if case["norm"] else None for _ in range(2))
        if case["train"]:
            s["dq"], s["dk"] = normal(b, hq, length, d), normal(b, hk, length, d)
        return s
    rows, k = case["rows"], case["k"]
    s["x"] = _activation(gen, rows, k, dtype)
    if case["form"] == "affine":
        s["weight"], s["bias"] = normal(k, std=0.1, mean=1.0), normal(k, std=0.1)
    else:
        s["shift"], s["scale"] = (normal(case["vectors"], k, std=0.2) for _ in range(2))
    if case["train"]:
        s["dy"] = normal(rows, k)
    return s


# ------------------------------------------------------------------ the package's kernels


def _package():
    path = os.path.join(os.getcwd(), "convrot-mlx_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import convrot_mlx_amd

    return convrot_mlx_amd


def _run_own(s: dict):
    pkg, case = _package(), s["case"]
    if case["op"] == "w8a8":
        if case["codes"]:
            return pkg.hip_w8a8_matmul(s["qact"], s["qweight"], s["xscales"], s["wscales"], s["bias"],
                                       output_dtype=s["dtype"], residual=s["residual"], gate=s["gate"])
        return pkg.hip_w8a8_linear(s["x"], s["qweight"], s["wscales"], s["bias"], residual=s["residual"],
                                   gate=s["gate"])
    if case["op"] == "rotary":
        kw = dict(q_weight=s["q_weight"], k_weight=s["k_weight"], eps=_EPS, interleaved=case["interleaved"])
        out = pkg.hip_qk_rotary(s["q"], s["k"], s["table"], **kw)
        if case["train"]:
            grads = pkg.hip_qk_rotary_backward(s["dq"], s["dk"], s["q"], s["k"], s["table"], **kw)
            out = (*out, *(g for g in grads if g is not None))
        return out
    if case["form"] == "affine":
        kw, bw = dict(weight=s["weight"], bias=s["bias"]), dict(weight=s["weight"])
    else:
        kw, bw = dict(shift=s["shift"], scale=s["scale"]), dict(scale=s["scale"])
    if not case["train"]:
        return pkg.hip_layer_norm(s["x"], eps=_EPS, **kw)
    y, mean, rstd = pkg.hip_layer_norm(s["x"], eps=_EPS, return_stats=True, **kw)
    return (y, *pkg.hip_layer_norm_backward(s["dy"], s["x"], mean, rstd, **bw))


# ------------------------------------------------------------------ the plain forms


def _plain_w8a8(s: dict):
    if "x" in s:
        x = s["x"].float()
        most = x.abs().amax(dim=1, keepdim=True)
        q = torch.round(x * torch.div(torch.full_like(most, 127.0), most)).clamp(-127, 127)
        xs = most * (1.0 / 127.0)
    else:
        q, xs = s["qact"].float(), s["xscales"][:, None]
    out = torch.matmul(q, s["qweight"].float().t()) * xs * s["wscales"] + s["bias"]
    if s["gate"] is not None:
        out = out * s["gate"].float()
    if s["residual"] is not None:
        out = s["residual"].float() + out
    return out.to(s["dtype"])


def _turn(x, cos, sin, interleaved: bool):
    """Pairs of the first 2 * pairs features turned by their angles; the others stay."""
    pairs = cos.shape[-1]
    if interleaved:
        a, b = x[..., 0: 2 * pairs: 2], x[..., 1: 2 * pairs: 2]
        turned = torch.stack([a * cos - b * sin, a * sin + b * cos], dim=-1).flatten(-2)
    else:
        a, b = x[..., :pairs], x[..., pairs: 2 * pairs]
        turned = torch.cat([a * cos - b * sin, a * sin + b * cos], dim=-1)
    return torch.cat([turned, x[..., 2 * pairs:]], dim=-1)


def _plain_rotary(s: dict):
    case = s["case"]
    cos, sin = s["table"][:, None, :, :, 0], s["table"][:, None, :, :, 1]
    outs, grads, wgrads = [], [], []
    for x, w, dy in ((s["q"], s["q_weight"], s.get("dq")), (s["k"], s["k_weight"], s.get("dk"))):
        xf = x.float()
        if case["norm"]:
            r = torch.rsqrt((xf * xf).mean(dim=-1, keepdim=True) + _EPS)
            unit, wf = xf * r, w.float()
            outs.append(_turn(unit * wf, cos, sin, case["interleaved"]).to(s["dtype"]))
        else:
            outs.append(_turn(xf, cos, sin, case["interleaved"]).to(s["dtype"]))
        if dy is not None:
            g = _turn(dy.float(), cos, -sin, case["interleaved"])
            if case["norm"]:
                wgrads.append((g * unit).sum(dim=(0, 1, 2)).to(s["dtype"]))
                g = g * wf
                g = r * (g - unit * (g * unit).mean(dim=-1, keepdim=True))
            grads.append(g.to(s["dtype"]))
    return (*outs, *grads, *wgrads)


def _plain_norm(s: dict):
    x = s["x"].float()
    c = x - x.mean(dim=1, keepdim=True)
    rstd = torch.rsqrt((c * c).mean(dim=1, keepdim=True) + _EPS)
    unit = c * rstd
    vectors = s["case"]["vectors"]
    if s["case"]["form"] == "affine":
        gain, shift = s["weight"].float()[None], s["bias"].float()[None]
    else:
        gain, shift = 1 + s["scale"].float(), s["shift"].float()
    group = lambda t: t.unflatten(0, (vectors, -1))  # noqa: E731
    y = (group(unit) * gain[:, None] + shift[:, None]).flatten(0, 1).to(s["dtype"])
    if "dy" not in s:
        return y
    dy = s["dy"].float()
    dgain, dshift = group(dy * unit).sum(dim=1), group(dy).sum(dim=1)
    g = (group(dy) * gain[:, None]).flatten(0, 1)
    dx = rstd * (g - g.mean(dim=1, keepdim=True) - unit * (g * unit).mean(dim=1, keepdim=True))
    if s["case"]["form"] == "affine":
        dgain, dshift = dgain[0], dshift[0]
    return y, dx.to(s["dtype"]), dgain.to(s["dtype"]), dshift.to(s["dtype"])


def run(state: dict):
    if own:
        return _run_own(state)
    return {"w8a8": _plain_w8a8, "rotary": _plain_rotary, "layer_norm": _plain_norm}[state["case"]["op"]](state)


# ------------------------------------------------------------------ 64 bits, and the work


def _exact_w8a8(s: dict):
    case = s["case"]
    if case["codes"]:
        codes, scale = s["qact"].double(), s["xscales"].double()
    else:
        x = s["x"].double()
        scale = x.abs().max(dim=1).values / 127
        codes = torch.round(x / scale.unsqueeze(1))
    y = codes @ s["qweight"].double().t().contiguous()
    y = y * (scale.unsqueeze(1) * s["wscales"].double().unsqueeze(0)) + s["bias"].double()
    if case["residual"] == "gate":
        y = s["residual"].double() + s["gate"].double() * y
    elif case["residual"] == "add":
        y = s["residual"].double() + y
    return y


def _exact_rotary(s: dict):
    """Each pair as a complex number, its angle a unit complex factor."""
    case = s["case"]
    pairs, dim = s["table"].shape[-2], case["dim"]
    factor = torch.view_as_complex(s["table"].double()).unsqueeze(1)
    even = torch.arange(pairs, device="cuda") * (2 if case["interleaved"] else 1)
    odd = even + (1 if case["interleaved"] else pairs)

    def turned(t, by):
        z = torch.complex(t[..., even], t[..., odd]) * by
        t = t.clone()
        t[..., even], t[..., odd] = z.real, z.imag
        return t

    outs, grads, wgrads = [], [], []
    for name in ("q", "k"):
        x = s[name].double()
        size = (x.square().sum(-1, keepdim=True) / dim + _EPS).sqrt()
        w = s[name + "_weight"].double() if case["norm"] else None
        outs.append(turned(x / size * w if case["norm"] else x, factor))
        if case["train"]:
            g = turned(s["d" + name].double(), factor.conj())
            if case["norm"]:
                wgrads.append((g * x / size).flatten(0, 2).sum(0))
                along = (g * w * x).sum(-1, keepdim=True)
                g = g * w / size - x * along / (dim * size ** 3)
            grads.append(g)
    return (*outs, *grads, *wgrads)


def _exact_norm(s: dict):
    case, x = s["case"], s["x"].double()
    k = case["k"]
    var, mean = torch.var_mean(x, dim=1, correction=0, keepdim=True)
    std = (var + _EPS).sqrt()
    unit = (x - mean) / std
    each = case["rows"] // case["vectors"]
    if case["form"] == "affine":
        gain, shift = s["weight"].double(), s["bias"].double()
    else:
        gain = (s["scale"].double() + 1).repeat_interleave(each, dim=0)
        shift = s["shift"].double().repeat_interleave(each, dim=0)
    y = unit * gain + shift
    if not case["train"]:
        return y
    dy = s["dy"].double()
    g = dy * gain
    dx = (g * k - g.sum(1, keepdim=True) - unit * (g * unit).sum(1, keepdim=True)) / (k * std)
    dgain = (dy * unit).reshape(case["vectors"], each, k).sum(1)
    dshift = dy.reshape(case["vectors"], each, k).sum(1)
    if case["form"] == "affine":
        dgain, dshift = dgain.squeeze(0), dshift.squeeze(0)
    return y, dx, dgain, dshift


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    return {"w8a8": _exact_w8a8, "rotary": _exact_rotary, "layer_norm": _exact_norm}[case["op"]](s)


def work(case: dict) -> dict:
    e = 4 if case["dtype"] == "float32" else 2
    if case["op"] == "w8a8":
        m, k, n = case["rows"], case["k"], case["n"]
        values = m * k * (1 if case["codes"] else e) + (4 * m if case["codes"] else 0)
        extra = {"none": 0, "add": m * n * e, "gate": (m * n + n) * e}[case["residual"]]
        return {"bytes": values + n * k + 8 * n + m * n * e + extra, "flops": 2 * m * n * k}
    if case["op"] == "rotary":
        tokens, d = case["batch"] * case["length"], case["dim"]
        size = tokens * (case["heads"] + case["kv_heads"]) * d
        table = tokens * (case["axis_t"] + case["axis_h"] + case["axis_w"]) * 4
        weights = 2 * d * e if case["norm"] else 0
        # training: the inputs are read once for both directions where they could stay on the chip
        moved = size * e * (4 if case["train"] else 2) + table + weights * (2 if case["train"] else 1)
        return {"bytes": moved, "flops": size * (4 + 3 * case["norm"]) * (3 if case["train"] else 1)}
    size = case["rows"] * case["k"]
    params = 2 * case["vectors"] * case["k"] * e
    moved = size * e * (4 if case["train"] else 2) + params * (2 if case["train"] else 1)
    return {"bytes": moved, "flops": size * (20 if case["train"] else 8)}
