"""Performance cases of the 8-bit and grouped products.

`run` computes each operator either in a plain form (elementary torch operations, `own = False`) or through the
framework's public calls (`own = True`) on the same inputs.  `exact` gives the results in 64 bits.

Operators:
  quantize    rows -> 8-bit codes and one scale per row
  ternary_a8  8-bit activations x packed ternary weights, scales per token and per channel (activations arrive in
              floating point and are quantised by the call)
  int8        8-bit activations x 8-bit weights, the same scales (activations arrive quantised)
  grouped     products grouped by expert, ragged row counts: bf16 or 8-bit activations x packed ternary weights, or
              8-bit x 8-bit
"""
import math

import torch

own = False

_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_BYTES = {"f32": 4, "bf16": 2, "f16": 2}


def listed():
    return [
        # one token's hidden state on its way into a quantised layer: launch latency
        {"name": "quantize-token", "op": "quantize", "m": 1, "k": 4096, "x": "bf16"},
        # a long prompt's activations
        {"name": "quantize-prompt", "op": "quantize", "m": 8192, "k": 8192, "x": "bf16"},
        # odd row length and count, fp32 activations (a calibration pass)
        {"name": "quantize-ragged", "op": "quantize", "m": 1037, "k": 5003, "x": "f32"},
        # decode of one token through the framework's decode matrix
        {"name": "ternary-token", "op": "ternary_a8", "m": 1, "n": 11008, "k": 4096, "x": "bf16", "y": "bf16", "bias": False},
        # a decode batch of several dozen sequences
        {"name": "ternary-batch", "op": "ternary_a8", "m": 48, "n": 11008, "k": 4096, "x": "bf16", "y": "bf16", "bias": False},
        # prefill at the framework's prefill size: the largest case
        {"name": "ternary-prompt", "op": "ternary_a8", "m": 8192, "n": 28672, "k": 8192, "x": "bf16", "y": "bf16", "bias": False},
        # odd everything, fp32 in and out, with bias
        {"name": "ternary-ragged", "op": "ternary_a8", "m": 517, "n": 1531, "k": 2051, "x": "f32", "y": "f32", "bias": True},
        # one token through a layer that stays in 8 bits (an output head)
        {"name": "int8-token", "op": "int8", "m": 1, "n": 11008, "k": 4096, "y": "bf16", "bias": False},
        # a medium prompt through such a layer
        {"name": "int8-prompt", "op": "int8", "m": 2048, "n": 4096, "k": 4096, "y": "f16", "bias": True},
        # decode of eight tokens, six experts each, out of 64
        {"name": "experts-decode", "op": "grouped", "form": "ternary_i8", "e": 64, "t": 48, "n": 2816, "k": 2048, "y": "bf16"},
        # prefill through the same experts with bf16 activations; some experts get a handful of rows, some thousands
        {"name": "experts-prompt", "op": "grouped", "form": "ternary_bf16", "e": 64, "t": 16384, "n": 2816, "k": 2048, "y": "bf16"},
        # few experts with 8-bit weights, odd sizes, fp32 out
        {"name": "experts-int8", "op": "grouped", "form": "int8", "e": 8, "t": 1501, "n": 2005, "k": 1520, "y": "f32"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["quantize", "ternary_a8", "int8", "grouped"])
    if op == "quantize":
        k = _log(rng, 16, 16384)
        return {"op": op, "m": min(_log(rng, 1, 16384), (8192 * 8192) // k), "k": k, "x": rng.choice(["bf16", "f16", "f32"])}
    if op in ("ternary_a8", "int8"):
        case = {"op": op, "m": _log(rng, 1, 8192), "n": _log(rng, 16, 28672), "k": _log(rng, 32, 8192),
                "y": rng.choice(["bf16", "f16", "f32"]), "bias": rng.random() < 0.5}
        if op == "ternary_a8":
            case["x"] = rng.choice(["bf16", "f16", "f32"])
        return case
    form = rng.choice(["ternary_i8", "ternary_bf16", "int8"])
    e = _log(rng, 1, 64)
    return {"op": op, "form": form, "e": e, "t": _log(rng, 1, 16384), "n": _log(rng, 16, 4096),
            "k": 8 * _log(rng, 4, 512), "y": rng.choice(["bf16", "f16", "f32"]) if form != "ternary_bf16" else "bf16"}


# ---- inputs ----------------------------------------------------------------------------------------------------------

def _popularity(e):
    """Share of each expert: a few are popular, most are not (Zipf with a gentle exponent)."""
    w = [1.0 / (i + 1) ** 0.8 for i in range(e)]
    s = sum(w)
    return [v / s for v in w]


def _activations(gen, m, k, dtype):
    """Hidden states: normal, a few channels an order of magnitude louder, every row at its own level."""
    x = torch.randn(m, k, generator=gen, device="cuda")
    loud = (torch.rand(1, k, generator=gen, device="cuda") < 0.004).float()
    level = torch.exp(0.5 * torch.randn(m, 1, generator=gen, device="cuda"))
    return (x * (1.0 + 9.0 * loud) * level).to(dtype)


def _ternary(gen, *shape):
    u = torch.rand(*shape, generator=gen, device="cuda")
    return (u < 0.3).to(torch.int8) - (u > 0.7).to(torch.int8)


def _codes(gen, *shape):
    """8-bit codes as quantised normal rows have them."""
    z = torch.randn(*shape, generator=gen, device="cuda") * 36.0
    return z.round().clamp(-127, 127).to(torch.int8)


def _inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))

    def uniform(lo, hi, *shape):
        return torch.rand(*shape, generator=gen, device="cuda") * (hi - lo) + lo

    op = case["op"]
    if op == "quantize":
        return {"x": _activations(gen, case["m"], case["k"], _DTYPES[case["x"]])}
    if op in ("ternary_a8", "int8"):
        m, n, k = case["m"], case["n"], case["k"]
        s = {"scale": uniform(0.01, 0.1, n), "bias": torch.randn(n, generator=gen, device="cuda") if case["bias"] else None}
        if op == "ternary_a8":
            s["x"] = _activations(gen, m, k, _DTYPES[case["x"]])
            s["w"] = _ternary(gen, n, k)
        else:
            s["row_scale"] = uniform(0.005, 0.05, m)
            s["x"] = _codes(gen, m, k)
            s["w"] = _codes(gen, n, k)
        return s
    e, t, n, k = case["e"], case["t"], case["n"], case["k"]
    pop = torch.tensor(_popularity(e), device="cuda")
    place = torch.randperm(e, generator=gen, device="cuda")          # which expert is the popular one
    expert = place[torch.multinomial(pop, t, replacement=True, generator=gen)]
    counts = torch.bincount(expert, minlength=e)
    offsets = torch.zeros(e + 1, dtype=torch.int32, device="cuda")
    offsets[1:] = torch.cumsum(counts, 0)
    s = {"offsets": offsets, "counts": counts.tolist(), "scale": uniform(0.01, 0.1, e, n), "row_scale": None}
    if case["form"] == "ternary_bf16":
        s["x"] = _activations(gen, t, k, torch.bfloat16)
    else:
        s["x"] = _codes(gen, t, k)
        s["row_scale"] = uniform(0.005, 0.05, t)
    s["w"] = _codes(gen, e, n, k) if case["form"] == "int8" else _ternary(gen, e, n, k)
    return s


def prepare(case, seed):
    """Inputs and, for the framework's calls, the weights in the layout a program keeps them in."""
    s = _inputs(case, seed)
    s["case"] = case
    if own and case["op"] != "quantize":
        from tmq_b200 import ops
        if case["op"] == "ternary_a8":
            s["wt"] = ops.prepack(ops.compactify_ternary(s["w"]), case["n"], ops.FMT_I8)
        elif case["op"] == "int8":
            s["wt"] = _padded(s["w"])
            s["x"] = _padded(s["x"])
        elif case["form"] == "int8":
            s["wt"] = _padded(s["w"])
            s["x"] = _padded(s["x"])
        else:
            fmt = ops.FMT_BF16 if case["form"] == "ternary_bf16" else ops.FMT_I8
            s["wt"] = torch.stack([ops.prepack(ops.compactify_ternary(w), case["n"], fmt) for w in s["w"].unbind(0)])
            if case["form"] == "ternary_i8":
                s["x"] = _padded(s["x"])
        del s["w"]
    return s


def _padded(codes):
    """8-bit rows with a row stride that is a multiple of 16 bytes, as the framework's quantisation writes them."""
    k = codes.shape[-1]
    if k % 16 == 0:
        return codes
    return torch.nn.functional.pad(codes, (0, -k % 16))[..., :k]


# ---- one pass ----------------------------------------------------------------------------------------------------------

def run(s):
    case = s["case"]
    return (_run_own if own else _run_plain)(case, s)


def _run_own(case, s):
    from tmq_b200 import ops
    op = case["op"]
    if op == "quantize":
        return ops.quantize_rows(s["x"])
    y = _DTYPES[case["y"]]
    if op == "ternary_a8":
        return ops.ternary_gemm_a8(s["x"], s["wt"], case["n"], scale=s["scale"], bias=s["bias"], out_dtype=y)
    if op == "int8":
        return ops.gemm_i8(s["x"], s["wt"], row_scale=s["row_scale"], scale=s["scale"], bias=s["bias"], out_dtype=y)
    if case["form"] == "int8":
        return ops.gemm_i8_grouped(s["x"], s["wt"], s["offsets"], row_scale=s["row_scale"], scales=s["scale"], out_dtype=y)
    return ops.ternary_gemm_grouped(s["x"], s["wt"], case["n"], s["offsets"], row_scale=s["row_scale"], scales=s["scale"],
                                    out_dtype=y)


def _plain_quantize(x):
    """Codes next to a rounding border are what 32 bits would get wrong: the quotient is taken in 64."""
    xd = x.double()
    amax = xd.abs().amax(dim=1, keepdim=True)
    codes = torch.where(amax > 0, (127.0 * xd / amax), torch.zeros_like(xd)).round().to(torch.int8)
    return codes, amax.float()[:, 0] / 127.0


def _product(x, w, long_sums):
    """x @ w^T; 8-bit sums pass 2^24 with 8-bit weights and are taken in 64 bits there."""
    if long_sums:
        return (x.double() @ w.double().t()).float()
    return x.float() @ w.float().t()


def _run_plain(case, s):
    op = case["op"]
    if op == "quantize":
        return _plain_quantize(s["x"])
    y = _DTYPES[case["y"]]
    if op in ("ternary_a8", "int8"):
        x, rs = _plain_quantize(s["x"]) if op == "ternary_a8" else (s["x"], s["row_scale"])
        out = _product(x, s["w"], op == "int8") * rs[:, None] * s["scale"]
        if s["bias"] is not None:
            out = out + s["bias"]
        return out.to(y)
    t, n = s["x"].shape[0], case["n"]
    out = torch.zeros(t, n, dtype=y, device="cuda")
    row = 0
    for e, count in enumerate(s["counts"]):
        if count:
            part = _product(s["x"][row:row + count], s["w"][e], case["form"] == "int8")
            if s["row_scale"] is not None:
                part = part * s["row_scale"][row:row + count, None]
            out[row:row + count] = (part * s["scale"][e]).to(y)
            row += count
    return out


def exact(case, seed):
    """The definition in 64 bits: q = round(127 x / max|x|), y = scale_n * rowscale_m * sum_k q w + bias_n."""
    s = _inputs(case, seed)
    x = s["x"].to(torch.float64)
    row_scale = s.get("row_scale")
    if case["op"] in ("quantize", "ternary_a8"):
        peak = torch.linalg.vector_norm(x, ord=float("inf"), dim=1)
        safe = torch.where(peak > 0, peak, torch.ones_like(peak))
        q = torch.round(torch.div(x * 127.0, safe[:, None]))
        row_scale = peak / 127.0
        if case["op"] == "quantize":
            return q.to(torch.int8), row_scale
        x = q
    if row_scale is not None:
        row_scale = row_scale.to(torch.float64)
        if case["op"] == "ternary_a8":
            row_scale = row_scale.to(torch.float32).to(torch.float64)     # the scale is a 32-bit number by definition
    if case["op"] != "grouped":
        y = torch.einsum("mk,nk->mn", x, s["w"].to(torch.float64))
        y = torch.einsum("mn,m,n->mn", y, row_scale, s["scale"].to(torch.float64))
        return y if s["bias"] is None else y + s["bias"].to(torch.float64)[None]
    bounds = s["offsets"].tolist()
    parts = []
    for e in range(case["e"]):
        rows = slice(bounds[e], bounds[e + 1])
        part = torch.einsum("mk,nk->mn", x[rows], s["w"][e].to(torch.float64)) * s["scale"][e].to(torch.float64)[None]
        parts.append(part if row_scale is None else part * row_scale[rows][:, None])
    return torch.cat(parts)


def work(case):
    op = case["op"]
    if op == "quantize":
        m, k = case["m"], case["k"]
        return {"bytes": m * k * (_BYTES[case["x"]] + 1) + 4 * m, "flops": 3 * m * k}
    if op in ("ternary_a8", "int8"):
        m, n, k = case["m"], case["n"], case["k"]
        xb = m * k * _BYTES[case["x"]] if op == "ternary_a8" else m * k + 4 * m
        wb = n * k // 4 if op == "ternary_a8" else n * k
        return {"bytes": xb + wb + 4 * n * (2 if case["bias"] else 1) + m * n * _BYTES[case["y"]], "flops": 2 * m * n * k}
    e, t, n, k = case["e"], case["t"], case["n"], case["k"]
    active = sum(1.0 - (1.0 - p) ** t for p in _popularity(e))       # experts that get a row, on average
    xb = t * k * (2 if case["form"] == "ternary_bf16" else 1) + (0 if case["form"] == "ternary_bf16" else 4 * t)
    wb = n * k if case["form"] == "int8" else n * k // 4
    return {"bytes": int(xb + active * (wb + 4 * n) + t * n * _BYTES[case["y"]]), "flops": 2 * t * n * k}
