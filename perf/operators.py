"""The serving operators around a quantized linear, as a program calls them: the residual's addition with the RMS norm
and an 8-bit output, the rotation by positions of several axes, and the low-rank adapters of many requests beside a
shared projection.  ``run`` takes either the elementary torch form (``own`` false) or this package's calls."""
import math
import os
import sys

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_FP8 = {"e4m3": (torch.float8_e4m3fn, 448.0)}
_EPS = 1e-6


def _package():
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "comfy-kitchen_b200")
    if at not in sys.path:
        sys.path.insert(0, at)
    import comfy_kitchen

    return comfy_kitchen


# ------------------------------------------------------------------ the cases


def listed():
    return [
        # one token of one request between two layers of a language model
        {"name": "norm 1 x 4096", "op": "norm", "rows": 1, "width": 4096, "dtype": "bf16", "stream": "bf16", "codes": "mx", "keep": False, "weight": True},
        # a ragged batch of prompts; the normalised rows are kept for the adapters that read them unquantized
        {"name": "norm 333 x 5120 kept", "op": "norm", "rows": 333, "width": 5120, "dtype": "fp16", "stream": "fp16", "codes": "mx", "keep": True, "weight": True},
        # an image model's joint sequence with its residual stream in 32 bits, static per-tensor FP8 scale
        {"name": "norm 4608 x 8192 fp8", "op": "norm", "rows": 4608, "width": 8192, "dtype": "bf16", "stream": "fp32", "codes": "e4m3", "keep": False, "weight": True},
        # a long prompt through a wide layer
        {"name": "norm 16384 x 8192", "op": "norm", "rows": 16384, "width": 8192, "dtype": "bf16", "stream": "bf16", "codes": "mx", "keep": False, "weight": True},
        # one token for each of 16 requests, far into their contexts, grouped-query heads
        {"name": "rope 16 tokens", "op": "rope", "batch": 16, "tokens": 1, "heads": 32, "kv_heads": 8, "dim": 128, "axes": "32,48,48", "theta": 1000000.0,
         "dtype": "bf16", "split_half": True, "tokens_first": False, "positions": "int64", "shared": False},
        # a batch of two images behind their text
        {"name": "rope 2 x 24 x 4608", "op": "rope", "batch": 2, "tokens": 4608, "heads": 24, "kv_heads": 24, "dim": 128, "axes": "16,56,56", "theta": 10000.0,
         "dtype": "bf16", "split_half": False, "tokens_first": False, "positions": "int64", "shared": True},
        # a video's latent tokens as the projection leaves them, [batch, tokens, heads, dim]
        {"name": "rope video 25037", "op": "rope", "batch": 1, "tokens": 25037, "heads": 40, "kv_heads": 40, "dim": 128, "axes": "44,42,42", "theta": 10000.0,
         "dtype": "fp16", "split_half": False, "tokens_first": True, "positions": "int32", "shared": True},
        # a vision encoder in 32 bits: two axes over part of each head, positions between the pixels
        {"name": "rope 3 x 1377 fp32", "op": "rope", "batch": 3, "tokens": 1377, "heads": 20, "kv_heads": 5, "dim": 80, "axes": "32,32", "theta": 10000.0,
         "dtype": "fp32", "split_half": True, "tokens_first": False, "positions": "float32", "shared": False},
        # one token of one request with its adapter
        {"name": "lora 1 x 4096", "op": "lora", "rows": 1, "k": 4096, "n": 4096, "rank": 16, "adapters": 8, "requests": 1, "dtype": "bf16", "without": False, "scales": True},
        # a step of 64 requests over 16 adapters, some requests without one
        {"name": "lora 64 x 14336", "op": "lora", "rows": 64, "k": 4096, "n": 14336, "rank": 32, "adapters": 16, "requests": 64, "dtype": "fp16", "without": True, "scales": True},
        # prompts of seven requests of any length in one batch
        {"name": "lora 4608 x 12288", "op": "lora", "rows": 4608, "k": 4096, "n": 12288, "rank": 64, "adapters": 4, "requests": 7, "dtype": "bf16", "without": True, "scales": True},
        # a full batch of long prompts, adapters of a high rank
        {"name": "lora 16384 x 8192", "op": "lora", "rows": 16384, "k": 8192, "n": 8192, "rank": 128, "adapters": 8, "requests": 8, "dtype": "bf16", "without": False, "scales": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("norm", "rope", "lora"))
    if op == "norm":
        dtype = rng.choice(("bf16", "fp16", "fp32"))
        case = {"op": op, "rows": 1, "width": 32, "dtype": dtype, "stream": rng.choice((dtype, "fp32")), "codes": rng.choice(("mx", "mx", "e4m3")),
                "keep": rng.random() < 0.3, "weight": rng.random() < 0.8}
        width = _log(rng, 256, 8192)
        case["width"] = width // 32 * 32 if case["codes"] == "mx" else width
        case["rows"] = _log(rng, 1, 16384)
        while work(case)["bytes"] > 9.4e8:
            case["rows"] = _log(rng, 1, 16384)
        return case
    if op == "rope":
        dim = rng.choice((64, 80, 96, 128, 160, 256))
        count = rng.choice((1, 2, 3, 3, 4))
        turning = rng.choice((dim, dim, dim // 2))
        cuts = sorted(rng.sample(range(1, turning // 2), count - 1))
        axes = [2 * (b - a) for a, b in zip([0] + cuts, cuts + [turning // 2])]
        kv = rng.choice((1, 2, 5, 8, 24))
        case = {"op": op, "batch": 1, "tokens": 1, "heads": kv * rng.choice((1, 1, 2, 4)), "kv_heads": kv, "dim": dim, "axes": ",".join(map(str, axes)),
                "theta": rng.choice((10000.0, 1000000.0)), "dtype": rng.choice(("bf16", "bf16", "fp16", "fp32")), "split_half": rng.random() < 0.5,
                "tokens_first": rng.random() < 0.5, "positions": rng.choice(("int32", "int64", "float32")), "shared": rng.random() < 0.5}
        while True:
            case["batch"], case["tokens"] = _log(rng, 1, 16), _log(rng, 1, 25000)
            if work(case)["bytes"] <= 1.0e9:
                return case
    while True:
        rank, adapters = 8 * rng.choice((1, 2, 3, 4, 5, 8, 16)), _log(rng, 1, 32)
        rows = _log(rng, 1, 16384)
        case = {"op": op, "rows": rows, "k": 8 * _log(rng, 64, 1792), "n": 8 * _log(rng, 64, 1792), "rank": rank, "adapters": adapters,
                "requests": min(rows, _log(rng, 1, 64)), "dtype": rng.choice(("bf16", "fp16")), "without": rng.random() < 0.4, "scales": rng.random() < 0.8}
        if rank * adapters <= 1024 and work(case)["bytes"] <= 8e8 and work(case)["flops"] <= 6.8e10:
            return case


# ------------------------------------------------------------------ what a program has in hand


def _generator(seed, *more):
    g = torch.Generator(device="cuda")
    g.manual_seed((int(seed) * 1_000_003 + sum((i + 1) * int(v) for i, v in enumerate(more))) & 0x7FFFFFFF)
    return g


def _randn(g, shape, dtype, scale=1.0):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).mul_(scale).to(dtype)


def prepare(case, seed):
    return {"norm": _prepare_norm, "rope": _prepare_rope, "lora": _prepare_lora}[case["op"]](case, seed)


def _prepare_norm(case, seed):
    g = _generator(seed, case["rows"], case["width"])
    rows, width, dtype, stream = case["rows"], case["width"], _DTYPES[case["dtype"]], _DTYPES[case["stream"]]
    # a residual stream carries a few columns that dwarf the others
    column = 1.0 + 20.0 * (torch.rand(width, generator=g, device="cuda") < 0.01).float()
    state = {"case": case, "x": _randn(g, (rows, width), dtype, 0.5), "residual": _randn(g, (rows, width), torch.float32).mul_(column).to(stream), "weight": None}
    if case["weight"]:
        state["weight"] = (1.0 + 0.1 * torch.randn(width, generator=g, device="cuda")).to(dtype)
    if case["codes"] != "mx":
        # calibrated: the largest activation lands near the type's largest value
        state["scale"] = torch.rand(1, generator=g, device="cuda") * 0.02 + 0.04
    return state


def _prepare_rope(case, seed):
    g = _generator(seed, case["tokens"], case["heads"])
    axes = [int(v) for v in case["axes"].split(",")]
    batch, tokens, dim, dtype = case["batch"], case["tokens"], case["dim"], _DTYPES[case["dtype"]]

    def heads_of(heads):
        shape = (batch, tokens, heads, dim) if case["tokens_first"] else (batch, heads, tokens, dim)
        return _randn(g, shape, dtype)

    rows = 1 if case["shared"] else batch
    if tokens < 16:
        # tokens that are being generated: any place in a long context, the same on every axis
        at = torch.randint(0, 131072, (rows, 1, 1), generator=g, device="cuda") + torch.arange(tokens, device="cuda")[None, :, None]
        positions = at.expand(rows, tokens, len(axes)).contiguous()
    else:
        # text first (zeros on the grid's axes), then a grid whose last axis runs fastest
        side = max(2, int(round((tokens * 0.9) ** (1.0 / max(1, len(axes) - 1)))))
        index = torch.arange(tokens, device="cuda")
        text = tokens // 9
        start = torch.randint(0, 4096, (rows, 1), generator=g, device="cuda")
        cols = []
        for a in range(len(axes)):
            step = side ** (len(axes) - 1 - a)
            place = (index - text).clamp_min(0) // step
            place = place % side if a else place
            cols.append(place[None].expand(rows, tokens) + (start if a == 0 else 0))
        positions = torch.stack(cols, dim=-1)
    if case["positions"] == "float32":
        positions = positions.float() + 0.5 * torch.rand(positions.shape, generator=g, device="cuda")
    elif case["positions"] == "int32":
        positions = positions.int()
    # rotation per unit of position, radians, one for each pair: the table that a model keeps
    freqs = torch.cat([case["theta"] ** (-torch.arange(0, d, 2, dtype=torch.float64) / d) for d in axes]).cuda()
    return {"case": case, "q": heads_of(case["heads"]), "k": heads_of(case["kv_heads"]), "positions": positions.contiguous(), "freqs": freqs, "axes": tuple(axes)}


def _requests(case, seed):
    """Where each request's rows begin and which adapter it asks for (-1: none), on the host."""
    g = torch.Generator().manual_seed(int(seed) * 7919 + case["rows"])
    rows, requests = case["rows"], case["requests"]
    cuts = (torch.randperm(rows - 1, generator=g)[: requests - 1] + 1).sort().values if requests > 1 else torch.zeros(0, dtype=torch.int64)
    lengths = torch.diff(torch.cat([torch.zeros(1, dtype=torch.int64), cuts, torch.tensor([rows])]))
    order = torch.randperm(case["adapters"], generator=g)
    asked = order[torch.arange(requests) % case["adapters"]]
    if case["without"]:
        asked = torch.where(torch.arange(requests) % 5 == 3, torch.full_like(asked, -1), asked)
    return lengths, asked


def _prepare_lora(case, seed):
    g = _generator(seed, case["rows"], case["n"], case["k"])
    rows, k, n, rank, adapters, dtype = case["rows"], case["k"], case["n"], case["rank"], case["adapters"], _DTYPES[case["dtype"]]
    lengths, asked = _requests(case, seed)
    state = {"case": case, "x": _randn(g, (rows, k), dtype), "y": _randn(g, (rows, n), dtype),
             "a": _randn(g, (adapters, rank, k), dtype, k ** -0.5), "b": _randn(g, (adapters, n, rank), dtype, 0.3 * rank ** -0.5),
             "ids": torch.repeat_interleave(asked, lengths).int().cuda(), "scales": None}
    if case["scales"]:
        state["scales"] = 0.5 + torch.rand(adapters, generator=g, device="cuda")
    return state


# ------------------------------------------------------------------ one pass


def run(state):
    return {"norm": _run_norm, "rope": _run_rope, "lora": _run_lora}[state["case"]["op"]](state)


def _run_norm(s):
    case, x, residual, weight = s["case"], s["x"], s["residual"], s["weight"]
    if own:
        ck = _package()
        if case["codes"] == "mx":
            return ck.add_rmsnorm_quantize_mxfp8(x, residual, weight, _EPS, return_norm=case["keep"])
        return ck.add_rmsnorm_quantize_fp8(x, residual, weight, s["scale"], _EPS, _FP8[case["codes"]][0], return_norm=case["keep"])
    h = (x.float() + residual.float()).to(residual.dtype)
    hf = h.float()
    yf = hf * torch.rsqrt(hf.square().mean(-1, keepdim=True) + _EPS)
    if weight is not None:
        yf = yf * weight.float()
    y = yf.to(x.dtype)
    if case["codes"] == "mx":
        q, scales = _blocks(y.float())
        return (q, scales, h, y) if case["keep"] else (q, scales, h)
    q_dtype, most = _FP8[case["codes"]]
    inverse = (1.0 / s["scale"]).to(x.dtype).float()   # the scalar and the product are rounded to x's type
    q = (y.float() * inverse).to(x.dtype).float().clamp(-most, most).to(q_dtype)
    return (q, h, y) if case["keep"] else (q, h)


def _blocks(y):
    """32-element blocks: E4M3 values and power-of-two scales, the scales in 128-row by 4-column tiles (32 rows of 16
    bytes, which hold four rows 32 apart by four columns), zero bytes in the padding."""
    rows, width = y.shape
    blocks = y.reshape(rows, width // 32, 32)
    most = blocks.abs().amax(-1)
    mantissa, exponent = torch.frexp(torch.clamp(most / 448.0, min=2.0 ** -126))
    up = torch.where(mantissa == 0.5, exponent - 1, exponent)      # ceil(log2)
    used = most > 0
    q = torch.where(used[..., None], torch.ldexp(blocks, -up[..., None].float()), torch.zeros_like(blocks)).to(torch.float8_e4m3fn)
    byte = torch.where(used, up + 127, torch.zeros_like(up)).to(torch.uint8)
    cols = width // 32
    tall, wide = (rows + 127) // 128 * 128, (cols + 3) // 4 * 4
    padded = torch.zeros((tall, wide), dtype=torch.uint8, device=y.device)
    padded[:rows, :cols] = byte
    tiled = padded.reshape(tall // 128, 4, 32, wide // 4, 4).permute(0, 3, 2, 1, 4).reshape(tall, wide)
    return q.reshape(rows, width), tiled.view(torch.float8_e8m0fnu)


def _run_rope(s):
    case = s["case"]
    if own:
        return _package().apply_rope_axes(s["q"], s["k"], s["positions"], s["freqs"], s["axes"], split_half=case["split_half"],
                                          tokens_dim=1 if case["tokens_first"] else 2)
    freqs, axes = s["freqs"], s["axes"]
    axis = torch.repeat_interleave(torch.arange(len(axes), device=freqs.device), torch.tensor([d // 2 for d in axes], device=freqs.device), output_size=freqs.numel())
    angle = s["positions"].double()[..., axis] * freqs      # in 64 bits: positions are far
    cos, sin = angle.cos().float(), angle.sin().float()
    at = 2 if case["tokens_first"] else 1
    return _turn(s["q"], cos.unsqueeze(at), sin.unsqueeze(at), case["split_half"]), _turn(s["k"], cos.unsqueeze(at), sin.unsqueeze(at), case["split_half"])


def _turn(x, cos, sin, split_half):
    pairs = cos.shape[-1]
    xf = x.float()
    if split_half:
        a, b = xf[..., :pairs], xf[..., pairs:2 * pairs]
        turned = torch.cat([a * cos - b * sin, a * sin + b * cos], dim=-1)
    else:
        a, b = xf[..., 0:2 * pairs:2], xf[..., 1:2 * pairs:2]
        turned = torch.stack([a * cos - b * sin, a * sin + b * cos], dim=-1).flatten(-2)
    return torch.cat([turned.to(x.dtype), x[..., 2 * pairs:]], dim=-1)


def _run_lora(s):
    x, y, a, b, ids, scales = s["x"], s["y"], s["a"], s["b"], s["ids"], s["scales"]
    if own:
        return _package().lora_add(y, x, a, b, ids, scales)
    adapters, rank, k = a.shape
    # every adapter's first product at once; a row keeps its own adapter's part
    mine = (ids[:, None] == torch.arange(adapters, device=ids.device)).float()
    if scales is not None:
        mine = mine * scales
    low = (x.float() @ a.float().reshape(adapters * rank, k).t()).reshape(-1, adapters, rank) * mine[..., None]
    wide = b.float().permute(0, 2, 1).reshape(adapters * rank, -1)
    return (y.float() + low.reshape(-1, adapters * rank) @ wide).to(y.dtype)


# ------------------------------------------------------------------ what a pass cannot do without


def _size(name):
    return 4 if name == "fp32" else 2


def work(case):
    if case["op"] == "norm":
        n, width = case["rows"] * case["width"], case["width"]
        each = _size(case["dtype"]) * (2 if case["keep"] else 1) + 2 * _size(case["stream"]) + 1
        scales = (case["rows"] + 127) // 128 * 128 * ((width // 32 + 3) // 4 * 4) if case["codes"] == "mx" else 4
        return {"bytes": n * each + scales + (width * _size(case["dtype"]) if case["weight"] else 0), "flops": 6 * n}
    if case["op"] == "rope":
        axes = [int(v) for v in case["axes"].split(",")]
        heads = case["batch"] * case["tokens"] * (case["heads"] + case["kv_heads"])
        places = (1 if case["shared"] else case["batch"]) * case["tokens"] * len(axes) * (8 if case["positions"] == "int64" else 4)
        return {"bytes": heads * case["dim"] * 2 * _size(case["dtype"]) + places + 4 * sum(axes), "flops": 3 * heads * sum(axes)}
    asked = [r % case["adapters"] for r in range(case["requests"]) if not (case["without"] and r % 5 == 3)]
    rows = case["rows"] * len(asked) // case["requests"]
    weights = len(set(asked)) * case["rank"] * (case["k"] + case["n"])
    return {"bytes": 2 * (rows * case["k"] + 2 * case["rows"] * case["n"] + weights) + 4 * case["rows"], "flops": 2 * rows * case["rank"] * (case["k"] + case["n"])}


# ------------------------------------------------------------------ the definition, in 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        return _exact_norm(s)
    return _exact_rope(s) if case["op"] == "rope" else _exact_lora(s)


def _exact_norm(s):
    """The 8-bit outputs' own rounding is left out here, as every output's is.  The block scales are powers of two that
    jump at a border, and no value between them is nearer to the definition: they have none here."""
    case, dtype, stream = s["case"], s["x"].dtype, s["residual"].dtype
    h = s["x"].double() + s["residual"].double()
    stored = h.to(stream).double()                       # the norm is taken of what is stored
    y = stored / torch.sqrt((stored * stored).mean(dim=1, keepdim=True) + _EPS)
    if s["weight"] is not None:
        y = y * s["weight"].double()
    if case["codes"] == "mx":
        rows, width = y.shape
        top = y.to(dtype).double().abs().view(rows, -1, 32).max(dim=2).values   # the codes are those of the activation in x's type
        power = torch.ceil(torch.log2(torch.where(top > 0, top / 448.0, torch.ones_like(top))))
        out = ((y.view(rows, -1, 32) * torch.exp2(-power)[:, :, None]).view(rows, width), None, h)
    else:
        limit = _FP8[case["codes"]][1]
        out = ((y / s["scale"].double()).clamp(-limit, limit), h)
    return out + (y,) if case["keep"] else out


def _exact_rope(s):
    case, axes = s["case"], s["axes"]
    pairs = sum(axes) // 2
    position = torch.cat([s["positions"][..., i:i + 1].double().expand(*s["positions"].shape[:2], d // 2) for i, d in enumerate(axes)], dim=-1)
    turn = torch.polar(torch.ones_like(position), position * s["freqs"])
    turn = turn[:, :, None] if case["tokens_first"] else turn[:, None]
    got = []
    for x in (s["q"], s["k"]):
        out = x.double().clone()
        first, second = (slice(0, pairs), slice(pairs, 2 * pairs)) if case["split_half"] else (slice(0, 2 * pairs, 2), slice(1, 2 * pairs, 2))
        z = torch.complex(out[..., first].contiguous(), out[..., second].contiguous()) * turn
        out[..., first], out[..., second] = z.real, z.imag
        got.append(out)
    return tuple(got)


def _exact_lora(s):
    out = s["y"].double()
    for which in range(s["case"]["adapters"]):
        rows = (s["ids"] == which).nonzero()[:, 0]
        if rows.numel():
            low = s["x"][rows].double() @ s["a"][which].double().t()
            more = low @ s["b"][which].double().t()
            out[rows] += more if s["scales"] is None else more * s["scales"][which].double()
    return out
