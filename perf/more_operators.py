"""Linears in 8-bit floating point and the linears of a mixture of experts, as measurable cases.

A case is one pass of an operator of this package beside its plain form: elementary torch
operations in 32 bits, rounded once at the end.

  fp8          a linear on e4m3 codes: activations with a scale for each block of 128 features of a
               row (a power of two), weights with a scale for each block of 128 x 128, float epilogue
  experts      the products of rows sorted by expert with their expert's weight, 16 bits; with
               "train" also the gradients of the rows and of every expert's weight
  fp8_experts  the same products on e4m3 codes, with the scales of "fp8"
  route        the order of the tokens' choices by expert, and the weighted sum of the experts' rows
               back to tokens; with "train" also the gradients of the rows and of the weights

Fields of a case
  op         one of these
  dtype      type of activations and outputs
  rows, k, n, codes, residual    fp8: token rows, input and output features; whether the rows come
             as codes and scales already; "none", "add" or "gate" (residual + gate * linear)
  tokens, choices, experts       the others: each token goes to `choices` different experts
  gather     experts, fp8_experts: rows are read from the tokens in place (a first linear), or lie
             sorted already (a second one)
  dropped    some choices belong to no expert (over an expert's capacity)
  k, n       input and output features (route: n features a row)
"""

from __future__ import annotations

import math
import os
import sys

import torch

own = False

_DTYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}
_FP8 = {"op": "fp8", "rows": 1, "k": 4096, "n": 4096, "dtype": "bfloat16", "codes": False, "residual": "none"}
_EXPERTS = {"op": "experts", "tokens": 8, "choices": 2, "experts": 16, "k": 2048, "n": 4096, "dtype": "bfloat16",
            "gather": True, "dropped": False, "train": False}
_FP8_EXPERTS = {"op": "fp8_experts", "tokens": 8, "choices": 2, "experts": 16, "k": 2048, "n": 4096,
                "dtype": "bfloat16", "gather": True, "dropped": False}
_ROUTE = {"op": "route", "tokens": 8, "choices": 2, "experts": 16, "n": 4096, "dtype": "bfloat16", "dropped": False,
          "train": False}


def listed() -> list[dict]:
    return [
        # A modulation or single-token linear: the weights' bytes and latency bound it.
        {**_FP8, "name": "fp8 1 row", "n": 12288},
        # A short prompt's rows, an odd number, through a fused qkv projection.
        {**_FP8, "name": "fp8 77 rows", "rows": 77, "n": 9216},
        # The closing linear of a block, gated back into the stream, in float16.
        {**_FP8, "name": "fp8 1536 rows gated", "rows": 1536, "k": 15360, "n": 5120, "dtype": "float16",
         "residual": "gate"},
        # The product alone, on codes that several projections share: a video model's sequence, the largest.
        {**_FP8, "name": "fp8 codes 8800 rows", "rows": 8800, "k": 8192, "n": 4096, "codes": True},
        # A few requests' single tokens through the experts' first linear: the weights of the experts that are met.
        {**_EXPERTS, "name": "experts 8 tokens"},
        # A prompt's rows in the experts' second linear, sizes that fill no tile, in float16.
        {**_EXPERTS, "name": "experts 1030 tokens odd", "tokens": 1030, "k": 1384, "n": 2685, "dtype": "float16",
         "gather": False, "dropped": True},
        # A training step of the experts' first linear at an image's 4096 and 512 text tokens.
        {**_EXPERTS, "name": "experts 4608 tokens train", "tokens": 4608, "experts": 8, "k": 4096, "n": 2048,
         "train": True},
        # Single tokens of a batch through many experts at 8 bits: nearly every weight is read.
        {**_FP8_EXPERTS, "name": "fp8 experts 32 tokens", "tokens": 32, "choices": 4, "experts": 64, "n": 2048},
        # A long sequence through the experts' second linear at 8 bits.
        {**_FP8_EXPERTS, "name": "fp8 experts 9216 tokens", "tokens": 9216, "experts": 16, "k": 4096,
         "gather": False},
        # The routing around one decoding step of a batch: launches.
        {**_ROUTE, "name": "route 16 tokens", "tokens": 16, "choices": 4, "experts": 64, "n": 2048},
        # The routing around a training step, some choices over capacity.
        {**_ROUTE, "name": "route 9216 tokens train", "tokens": 9216, "choices": 4, "experts": 64, "dropped": True,
         "train": True},
    ]


_MOST = 8800 * 8192 * 4096


def draw(rng) -> dict:
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["fp8", "fp8", "experts", "experts", "fp8_experts", "route"])
    if op == "fp8":
        case = {**_FP8, "dtype": rng.choice(["bfloat16", "bfloat16", "float16", "float32"])}
        case["rows"] = rng.choice([1, spread(1, 64), spread(1, 8800), spread(64, 8800)])
        k, n = spread(512, 16384), spread(512, 21504)
        k = k // 128 * 128 if rng.random() < 0.75 else k // 16 * 16
        n = n // 64 * 64 if rng.random() < 0.7 else n
        while case["rows"] * k * n > _MOST:
            k, n = max(512, k // 32 * 16), max(512, n // 2)
        case["k"], case["n"] = k, n
        case["codes"] = rng.random() < 0.2
        case["residual"] = rng.choice(["none", "none", "add", "gate"])
        return case
    experts = rng.choice([1, 2, 4, 8, 8, 16, 16, 32, 60, 64])
    size = {"experts": experts, "choices": min(experts, rng.choice([1, 2, 2, 4, 8])),
            "dtype": rng.choice(["bfloat16", "bfloat16", "float16"]), "dropped": rng.random() < 0.3}
    tokens = rng.choice([1, spread(1, 64), spread(64, 9216), spread(64, 9216)])
    if op == "route":
        case = {**_ROUTE, **size, "tokens": tokens, "train": rng.random() < 0.5}
        n = spread(256, 8192)
        case["n"] = n // 64 * 64 if rng.random() < 0.7 else n
        while case["tokens"] * case["choices"] * case["n"] > 9216 * 4 * 4096:
            case["tokens"] = max(1, case["tokens"] // 2)
        return case
    case = {**(_EXPERTS if op == "experts" else _FP8_EXPERTS), **size, "tokens": tokens, "gather": rng.random() < 0.6}
    if op == "experts":
        case["train"] = rng.random() < 0.5
    k, n = spread(256, 8192), spread(256, 8192)
    case["k"] = k // 64 * 64 if rng.random() < 0.7 else k // 16 * 16
    case["n"] = n // 64 * 64 if rng.random() < 0.7 else n
    while (case["tokens"] * case["choices"] * case["k"] * case["n"] * (3 if case.get("train") else 1) > _MOST // 2
           or experts * case["k"] * case["n"] > 64 * 2048 * 2048):
        case["k"], case["n"] = max(256, case["k"] // 32 * 16), max(256, case["n"] // 2)
        case["tokens"] = max(1, case["tokens"] * 3 // 4)
    return case


# ------------------------------------------------------------------ inputs


def _activation(gen, rows, k, dtype):
    """N(0, 1) with one channel in 200 twenty times as large: a transformer's outlier channels."""
    gain = torch.ones(k, device="cuda")
    gain[torch.randperm(k, generator=gen, device="cuda")[: max(1, k // 200)]] = 20.0
    return (torch.randn((rows, k), generator=gen, device="cuda") * gain).to(dtype)


def _spread(scales, n, k):
    """Scales of 128 x 128 blocks [.., N / 128, K / 128] at each weight [.., n, k]."""
    return scales.repeat_interleave(128, dim=-2)[..., :n, :].repeat_interleave(128, dim=-1)[..., :k]


def _fp8_weight(gen, *shape):
    """Random weights as a checkpoint holds them: e4m3 codes, and float32 scales of 128 x 128 blocks that
    take a block's largest magnitude to the type's."""
    n, k = shape[-2:]
    w = torch.randn(shape, generator=gen, device="cuda") * 0.02
    pad = torch.nn.functional.pad(w.abs(), (0, -k % 128, 0, -n % 128))
    scales = pad.unflatten(-1, (-1, 128)).amax(-1).unflatten(-2, (-1, 128)).amax(-2) / 448.0
    return (w / _spread(scales, n, k)).to(torch.float8_e4m3fn), scales


def _choices(case: dict, gen) -> torch.Tensor:
    """[T, C] int64: the experts with the largest scores, some experts liked more than others; where the case
    drops some, one choice in 32 is -1."""
    t, c, e = case["tokens"], case["choices"], case["experts"]
    score = torch.randn((t, e), generator=gen, device="cuda") + torch.randn(e, generator=gen, device="cuda") * 0.5
    ids = score.topk(c, dim=1).indices
    if case["dropped"]:
        ids = torch.where(torch.rand((t, c), generator=gen, device="cuda") < 1 / 32, -1, ids)
    return ids


def _order(ids: torch.Tensor, experts: int):
    """(offsets [E + 1], order [T C], slots [T, C]) in int32: the choices sorted by expert, those of one expert in
    their order, those of none last; where each expert's begin, which choice each is, and where each choice is."""
    flat = ids.flatten()
    key = torch.where((flat >= 0) & (flat < experts), flat, experts)
    by, order = torch.sort(key, stable=True)
    offsets = torch.searchsorted(by, torch.arange(experts + 1, device=by.device))
    slots = torch.empty_like(order)
    slots[order] = torch.arange(order.numel(), device=order.device)
    return offsets.int(), order.int(), slots.view(ids.shape).int()


def prepare(case: dict, seed: int) -> dict:
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = _DTYPES[case["dtype"]]

    def normal(*shape, std=1.0, mean=0.0, kind=dtype):
        return (torch.randn(shape, generator=gen, device="cuda") * std + mean).to(kind)

    s = {"case": case, "dtype": dtype}
    if case["op"] == "fp8":
        rows, k, n = case["rows"], case["k"], case["n"]
        s["qweight"], s["wscales"] = _fp8_weight(gen, n, k)
        s["bias"] = normal(n, std=0.02, kind=torch.float32)
        x = _activation(gen, rows, k, dtype)
        if case["codes"]:
            s["qact"], s["xscales"] = _block_codes(x)
        else:
            s["x"] = x
        s["residual"] = normal(rows, n) if case["residual"] != "none" else None
        s["gate"] = normal(1, n, std=0.5) if case["residual"] == "gate" else None
        return s
    e, slots = case["experts"], case["tokens"] * case["choices"]
    s["ids"] = _choices(case, gen)
    if case["op"] == "route":
        s["y"] = normal(slots, case["n"])
        s["weights"] = torch.rand((case["tokens"], case["choices"]), generator=gen, device="cuda") + 0.05
        s["weights"] /= s["weights"].sum(1, keepdim=True)
        if case["train"]:
            s["dout"] = normal(case["tokens"], case["n"])
        return s
    s["offsets"], s["order"], s["slots"] = _order(s["ids"], e)
    s["most"] = max(1, int(s["offsets"].diff().max()))  # rows of the largest expert, for the padded plain form
    x_rows = case["tokens"] if case["gather"] else slots
    s["x"] = _activation(gen, x_rows, case["k"], dtype)
    if case["op"] == "fp8_experts":
        s["qweight"], s["wscales"] = _fp8_weight(gen, e, case["n"], case["k"])
    else:
        s["weight"] = normal(e, case["n"], case["k"], std=0.02)
        if case["train"]:
            s["dy"] = normal(slots, case["n"])
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
    if case["op"] == "fp8":
        kw = dict(residual=s["residual"], gate=s["gate"])
        if case["codes"]:
            return pkg.hip_fp8_matmul(s["qact"], s["qweight"], s["xscales"], s["wscales"], s["bias"],
                                      output_dtype=s["dtype"], **kw)
        return pkg.hip_fp8_linear(s["x"], s["qweight"], s["wscales"], s["bias"], **kw)
    if case["op"] == "route":
        plan = pkg.expert_plan(s["ids"], case["experts"])
        out = (*plan, pkg.hip_combine_rows(s["y"], plan, s["weights"]))
        return (*out, *pkg.hip_combine_rows_backward(s["dout"], s["y"], plan, s["weights"])) if case["train"] else out
    plan = pkg.ExpertPlan(s["offsets"], s["order"], s["slots"])
    if case["op"] == "fp8_experts":
        return pkg.hip_fp8_grouped_linear(s["x"], s["qweight"], s["wscales"], plan, gather=case["gather"])
    out = pkg.hip_grouped_linear(s["x"], s["weight"], plan, gather=case["gather"])
    if not case["train"]:
        return out
    return (out, *pkg.hip_grouped_linear_backward(s["dy"], s["x"], s["weight"], plan, gather=case["gather"]))


# ------------------------------------------------------------------ the plain forms


def _block_codes(x):
    """(e4m3 codes [M, K], float32 scales [M, K / 128]): the smallest power of two that takes a block's largest
    magnitude to at most 448 = 0.875 * 2^9."""
    k = x.shape[1]
    blocks = torch.nn.functional.pad(x.float(), (0, -k % 128)).unflatten(1, (-1, 128))
    mantissa, exponent = torch.frexp(blocks.abs().amax(-1))
    exponent = exponent - 9 + (mantissa > 0.875).int()
    scales, inverse = (((127 + e) << 23).view(torch.float32) for e in (exponent, -exponent))
    codes = (blocks * inverse[..., None]).to(torch.float8_e4m3fn)
    return codes.flatten(1)[:, :k].contiguous(), scales


def _values(codes, scales):
    return codes.float() * scales.repeat_interleave(128, dim=1)[:, : codes.shape[1]]


def _plain_fp8(s: dict):
    n, k = s["qweight"].shape
    x = _values(s["qact"], s["xscales"]) if s["case"]["codes"] else _values(*_block_codes(s["x"]))
    w = s["qweight"].float() * _spread(s["wscales"], n, k)
    out = torch.matmul(x, w.t()) + s["bias"]
    if s["gate"] is not None:
        out = out * s["gate"].float()
    if s["residual"] is not None:
        out = s["residual"].float() + out
    return out.to(s["dtype"])


def _places(s: dict):
    """Of each sorted row: its expert (any for none), its place among that expert's, and 1 (0 for none)."""
    offsets = s["offsets"].long()
    row = torch.arange(s["order"].numel(), device=offsets.device)
    expert = torch.searchsorted(offsets, row, right=True) - 1
    some = row < offsets[-1]
    expert = torch.where(some, expert, 0)
    return expert, torch.where(some, row - offsets[expert], 0), some[:, None].float()


def _plain_experts(s: dict):
    """Every expert's rows padded to the most that one has, then batched products."""
    case = s["case"]
    expert, place, some = _places(s)
    token = s["order"].long() // case["choices"]

    def padded(rows):
        out = torch.zeros((case["experts"], s["most"], rows.shape[1]), device=rows.device)
        return out.index_put_((expert, place), rows * some, accumulate=True)

    if case["op"] == "fp8_experts":
        x = _values(*_block_codes(s["x"]))
        w = s["qweight"].float() * _spread(s["wscales"], case["n"], case["k"])
    else:
        x, w = s["x"].float(), s["weight"].float()
    xp = padded(x[token] if case["gather"] else x)
    out = (torch.matmul(xp, w.transpose(1, 2).contiguous())[expert, place] * some).to(s["dtype"])
    if not case.get("train"):
        return out
    dyp = padded(s["dy"].float())
    dx = torch.matmul(dyp, w)[expert, place] * some
    if case["gather"]:
        dx = dx[s["slots"].long()].sum(dim=1)
    dw = torch.matmul(dyp.transpose(1, 2).contiguous(), xp)
    return out, dx.to(s["dtype"]), dw.to(s["dtype"])


def _plain_route(s: dict):
    case, w = s["case"], s["weights"]
    offsets, order, slots = _order(s["ids"], case["experts"])
    rows = s["y"].float()[slots.long()]
    out = (offsets, order, slots, (rows * w[..., None]).sum(dim=1).to(s["dtype"]))
    if not case["train"]:
        return out
    dout, at = s["dout"].float(), order.long()
    dy = dout[at // case["choices"]] * w.flatten()[at][:, None]
    return (*out, dy.to(s["dtype"]), (rows * dout[:, None]).sum(dim=2))


def run(state: dict):
    if own:
        return _run_own(state)
    return {"fp8": _plain_fp8, "experts": _plain_experts, "fp8_experts": _plain_experts,
            "route": _plain_route}[state["case"]["op"]](state)


# ------------------------------------------------------------------ 64 bits, and the work


def _exact_values(x):
    """Rows of x as their codes stand for them: each block over its power of two, to four bits of mantissa (and
    steps of 2^-9 at the least), ties to even."""
    m, k = x.shape
    pad = torch.zeros((m, (k + 127) // 128 * 128), dtype=torch.float64, device=x.device)
    pad[:, :k] = x.double()
    b = pad.view(m, -1, 128)
    scale = torch.exp2(torch.ceil(torch.log2(b.abs().max(2, keepdim=True).values / 448)))
    v = b / scale
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -6))) - 3)
    return (torch.round(v / step) * step * scale).view(m, -1)[:, :k]


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    if case["op"] == "route":
        flat = s["ids"].flatten().tolist()
        lists = [[i for i, f in enumerate(flat) if f == e] for e in range(case["experts"])]
        order = sum(lists, []) + [i for i, f in enumerate(flat) if f < 0]
        where = {choice: at for at, choice in enumerate(order)}
        starts = [0]
        for rows in lists:
            starts.append(starts[-1] + len(rows))
        as_int = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
        slots = as_int([where[i] for i in range(len(flat))]).view(s["ids"].shape)
        w, y = s["weights"].double(), s["y"].double()
        out = torch.zeros((case["tokens"], case["n"]), dtype=torch.float64, device="cuda")
        dw = torch.zeros_like(w)
        for c in range(case["choices"]):
            rows = y[slots[:, c].long()]
            out += w[:, c:c + 1] * rows
            if case["train"]:
                dw[:, c] = (rows * s["dout"].double()).sum(1)
        if not case["train"]:
            return as_int(starts), as_int(order), slots, out
        dy = torch.empty_like(y)
        for c in range(case["choices"]):
            dy[slots[:, c].long()] = w[:, c:c + 1] * s["dout"].double()
        return as_int(starts), as_int(order), slots, out, dy, dw
    if case["op"] == "fp8":
        n, k = s["qweight"].shape
        if case["codes"]:
            x = s["qact"].double()
            for b in range(s["xscales"].shape[1]):
                x[:, 128 * b: 128 * b + 128] *= s["xscales"][:, b: b + 1].double()
        else:
            x = _exact_values(s["x"])
        w = s["qweight"].double()
        for b in range(s["wscales"].shape[0]):
            w[128 * b: 128 * b + 128] *= s["wscales"][b].double().repeat_interleave(128)[:k]
        y = x @ w.t().contiguous() + s["bias"].double()
        if case["residual"] == "gate":
            y = y * s["gate"].double()
        return y if case["residual"] == "none" else y + s["residual"].double()
    fp8 = case["op"] == "fp8_experts"
    x = _exact_values(s["x"]) if fp8 else s["x"].double()
    slots, starts = s["order"].numel(), s["offsets"].tolist()
    token = s["order"].long() // case["choices"] if case["gather"] else torch.arange(slots, device="cuda")
    out = torch.zeros((slots, case["n"]), dtype=torch.float64, device="cuda")
    dx = torch.zeros(x.shape, dtype=torch.float64, device="cuda")
    dw = []
    for e in range(case["experts"]):
        at = slice(starts[e], starts[e + 1])
        rows = x[token[at]]
        w = (s["qweight"] if fp8 else s["weight"])[e].double()
        if fp8:
            for b in range(s["wscales"].shape[1]):
                w[128 * b: 128 * b + 128] *= s["wscales"][e, b].double().repeat_interleave(128)[: case["k"]]
        out[at] = rows @ w.t().contiguous()
        if case.get("train"):
            dy = s["dy"][at].double()
            dx.index_add_(0, token[at], dy @ w)
            dw.append(dy.t().contiguous() @ rows)
    return (out, dx, torch.stack(dw)) if case.get("train") else out


def work(case: dict) -> dict:
    e = 4 if case["dtype"] == "float32" else 2
    if case["op"] == "fp8":
        m, k, n = case["rows"], case["k"], case["n"]
        blocks = (k + 127) // 128
        values = m * k + 4 * m * blocks if case["codes"] else m * k * e
        extra = {"none": 0, "add": m * n * e, "gate": (m * n + n) * e}[case["residual"]]
        return {"bytes": values + n * k + 4 * blocks * ((n + 127) // 128) + 4 * n + m * n * e + extra,
                "flops": 2 * m * n * k}
    t, c, experts = case["tokens"], case["choices"], case["experts"]
    slots = t * c
    if case["op"] == "route":
        n = case["n"]
        ints = 8 * slots + 4 * (experts + 1) + 8 * slots
        moved = (slots + t) * n * e + 4 * slots
        if case["train"]:  # the rows are read once for both directions where they could stay on the chip
            moved += (t + slots) * n * e + 4 * slots
        return {"bytes": ints + moved, "flops": slots * n * (5 if case["train"] else 2)}
    k, n, rows = case["k"], case["n"], t if case["gather"] else slots
    met = experts * (1 - (1 - c / experts) ** t)  # experts that some token goes to, were all alike
    if case["op"] == "fp8_experts":
        return {"bytes": rows * k * e + met * n * k + slots * n * e, "flops": 2 * slots * n * k}
    if not case["train"]:
        return {"bytes": (rows * k + met * n * k + slots * n) * e, "flops": 2 * slots * n * k}
    return {"bytes": (2 * rows * k + met * n * k + experts * n * k + 2 * slots * n) * e, "flops": 6 * slots * n * k}
