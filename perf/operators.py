"""Cases of the layer-norm and 4-bit-weight operators: a norm in front of a projection with 4-bit weights, as it is
trained (norm forward and backward, weights quantised and expanded again) and as it is served (single tokens and small
batches against the 4-bit weights).

`own = False` computes every operator from elementary torch operations; `own = True` calls the library.
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
EPS = 1e-5


def listed():
    return [
        # one decoding step of eight sequences: the norm alone, no statistics kept; a call of pure latency
        {"name": "norm, 8 tokens", "op": "norm", "rows": 8, "cols": 4096, "type": "bf16", "params": "bf16", "stats": False},
        # a training batch of 16384 tokens, parameters in 32 bits, statistics kept for the backward pass
        {"name": "norm, training batch", "op": "norm", "rows": 16384, "cols": 4096, "type": "bf16", "params": "f32", "stats": True},
        # rows whose length is no multiple of any vector width, in the library's own type
        {"name": "norm gradient, odd rows", "op": "norm_grad", "rows": 5003, "cols": 1027, "type": "f32", "params": "f32"},
        # the backward pass of the training batch, with the sums over 16384 rows
        {"name": "norm gradient, training", "op": "norm_grad", "rows": 16384, "cols": 4096, "type": "bf16", "params": "f32"},
        # a small projection with a ragged last group and zero points, from 32-bit master weights
        {"name": "quantise, ragged groups", "op": "quantise", "n": 1000, "k": 2050, "group": 64, "type": "f32", "scales": "f16", "zeros": True},
        # a whole projection of a 16-bit checkpoint
        {"name": "quantise, 8192 x 8192", "op": "quantise", "n": 8192, "k": 8192, "group": 128, "type": "bf16", "scales": "bf16", "zeros": False},
        # expanded and transposed to 32 bits: the right operand of the library's SGEMM, for a batch of many rows
        {"name": "expand transposed, 6144", "op": "expand", "n": 6144, "k": 6144, "group": 128, "type": "f32", "scales": "bf16", "zeros": False, "transposed": True},
        # a projection of odd sizes to 16 bits
        {"name": "expand, odd sizes", "op": "expand", "n": 2049, "k": 1023, "group": 32, "type": "f16", "scales": "f16", "zeros": True, "transposed": False},
        # one token of one sequence
        {"name": "product, 1 token", "op": "product", "m": 1, "n": 4096, "k": 4096, "group": 128, "type": "bf16", "scales": "bf16", "zeros": False},
        # a few tokens in 32 bits against weights with zero points
        {"name": "product, 3 tokens f32", "op": "product", "m": 3, "n": 6144, "k": 6144, "group": 64, "type": "f32", "scales": "f32", "zeros": True},
        # odd sizes: rows of codes that start at any byte
        {"name": "product, odd sizes", "op": "product", "m": 5, "n": 1001, "k": 4098, "group": 64, "type": "f16", "scales": "f16", "zeros": True},
        # sixteen sequences decoded together against a wide projection (134 MB of codes)
        {"name": "product, 16 tokens", "op": "product", "m": 16, "n": 32768, "k": 8192, "group": 128, "type": "bf16", "scales": "bf16", "zeros": False},
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "norm_grad", "quantise", "expand", "product", "product"])
    kind = rng.choice(["f32", "bf16", "f16"])
    while True:
        case = {"op": op}
        if op in ("norm", "norm_grad"):
            case.update(rows=_spread(rng, 1, 65536), cols=_spread(rng, 64, 32768), type=kind, params=rng.choice(["f32", kind]))
            if rng.random() < 0.5:
                case["cols"] = -(-case["cols"] // 64) * 64
            if op == "norm":
                case["stats"] = rng.random() < 0.5
        else:
            if op == "product":
                case["m"] = _spread(rng, 1, 64)
            case.update(n=_spread(rng, 64, 32768), k=_spread(rng, 64, 16384), group=rng.choice([32, 64, 128, 256]), type=kind,
                        scales=rng.choice(["f32", kind]), zeros=rng.random() < 0.5)
            if rng.random() < 0.6:
                case["k"] = -(-case["k"] // 128) * 128
            if op == "expand":
                case["transposed"] = rng.random() < 0.5
        w = work(case)
        if w["bytes"] <= 400e6 and w["flops"] <= 8.5e9:
            return case


def work(case):
    op, t = case["op"], SIZE[case["type"]]
    if op in ("norm", "norm_grad"):
        r, c, p = case["rows"], case["cols"], SIZE[case["params"]]
        if op == "norm":
            return {"bytes": 2 * r * c * t + 2 * c * p + (8 * r if case["stats"] else 0), "flops": 8 * r * c}
        return {"bytes": 3 * r * c * t + 3 * c * p + 8 * r, "flops": 15 * r * c}
    n, k = case["n"], case["k"]
    groups = -(-k // case["group"])
    held = n * (-(-k // 2)) + n * groups * (SIZE[case["scales"]] + (1 if case["zeros"] else 0))
    if op == "product":
        return {"bytes": held + case["m"] * (k + n) * t, "flops": 2 * case["m"] * n * k}
    if op == "expand":
        return {"bytes": held + n * k * t, "flops": 2 * n * k}
    return {"bytes": held + 2 * n * k * t, "flops": 4 * n * k}   # weights in, codes and scales out, and the values they stand for


# ---- inputs -----------------------------------------------------------------------------------


def _weights(n, k, gen, dtype):
    # rows of differing scale and a few large entries, as trained projections have them
    w = torch.randn(n, k, generator=gen, device="cuda") * (0.01 + 0.02 * torch.rand(n, 1, generator=gen, device="cuda"))
    w.view(-1)[:: 997] *= 6.0
    return w.to(dtype)


def _activations(rows, cols, gen, dtype):
    # hidden states: a few columns are much larger than the others, and rows are off zero
    x = torch.randn(rows, cols, generator=gen, device="cuda")
    x[:, ::61] *= 8.0
    return x.add_(0.5 * torch.randn(rows, 1, generator=gen, device="cuda")).to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op, dtype = case["op"], TYPES[case["type"]]
    s = dict(case)
    new = lambda shape, kind: torch.empty(shape, dtype=kind, device="cuda")  # noqa: E731
    if op in ("norm", "norm_grad"):
        r, c, kind = case["rows"], case["cols"], TYPES[case["params"]]
        s["x"] = _activations(r, c, gen, dtype)
        s["gamma"] = (1.0 + 0.2 * torch.randn(c, generator=gen, device="cuda")).to(kind)
        s["beta"] = (0.1 * torch.randn(c, generator=gen, device="cuda")).to(kind)
        if op == "norm":
            s["y"] = new((r, c), dtype)
            s["mean"], s["rstd"] = (new(r, torch.float32), new(r, torch.float32)) if case["stats"] else (None, None)
            return s
        wide = s["x"].double()
        mean = wide.mean(1, keepdim=True)
        s["mean"] = mean[:, 0].float()
        s["rstd"] = ((wide - mean).square_().mean(1) + EPS).rsqrt().float()
        del wide
        s["dy"] = (0.1 * torch.randn(r, c, generator=gen, device="cuda")).to(dtype)
        s["dx"], s["dgamma"], s["dbeta"] = new((r, c), dtype), new(c, kind), new(c, kind)
        return s
    n, k, group = case["n"], case["k"], case["group"]
    groups = -(-k // group)
    if op == "quantise":
        s["w"] = _weights(n, k, gen, dtype)
        s["codes"] = new((n, -(-k // 2)), torch.uint8)
        s["scales"] = new((n, groups), TYPES[case["scales"]])
        s["zeros"] = new((n, groups), torch.uint8) if case["zeros"] else None
        s["values"] = new((n, k), dtype)
        return s
    s["codes"] = torch.randint(0, 256, (n, -(-k // 2)), generator=gen, device="cuda", dtype=torch.uint8)
    if k % 2:
        s["codes"][:, -1] &= 15
    s["scales"] = (0.002 + 0.006 * torch.rand(n, groups, generator=gen, device="cuda")).to(TYPES[case["scales"]])
    s["zeros"] = torch.randint(5, 11, (n, groups), generator=gen, device="cuda", dtype=torch.uint8) if case["zeros"] else None
    if op == "expand":
        s["w"] = new((k, n) if case["transposed"] else (n, k), dtype)
    else:
        s["x"] = _activations(case["m"], k, gen, dtype)
        s["y"] = new((case["m"], n), dtype)
    return s


# ---- one pass ---------------------------------------------------------------------------------


def run(s):
    if own:
        return _own(s)
    return {"norm": _norm, "norm_grad": _norm_grad, "quantise": _quantise, "expand": _expand, "product": _product}[s["op"]](s)


def _own(s):
    import hpcdeepneuralnetworks_b200 as b2
    op = s["op"]
    if op == "norm":
        b2.layernorm(s["rows"], s["cols"], EPS, s["x"], s["gamma"], s["beta"], s["y"], mean=s["mean"], rstd=s["rstd"])
        return [s["y"], s["mean"], s["rstd"]] if s["stats"] else [s["y"]]
    if op == "norm_grad":
        b2.layernorm_backward(s["rows"], s["cols"], s["dy"], s["x"], s["gamma"], s["mean"], s["rstd"], s["dx"], s["dgamma"], s["dbeta"])
        return [s["dx"], s["dgamma"], s["dbeta"]]
    n, k, group = s["n"], s["k"], s["group"]
    if op == "quantise":
        # quantised, and expanded again to what the codes stand for, as a check of the rounding does
        b2.w4_quantize(n, k, group, s["w"], s["codes"], s["scales"], s["zeros"])
        b2.w4_dequantize(n, k, group, s["codes"], s["scales"], s["zeros"], s["values"])
        return [s["values"], s["scales"], s["zeros"]] if s["zeros"] is not None else [s["values"], s["scales"]]
    if op == "expand":
        b2.w4_dequantize(n, k, group, s["codes"], s["scales"], s["zeros"], s["w"], transpose=s["transposed"])
        return s["w"]
    return b2.w4_matvec(s["m"], n, k, group, 1.0, s["x"], s["codes"], s["scales"], s["zeros"], 0.0, s["y"])


def _norm(s):
    x = s["x"].float()
    mean = x.mean(1, keepdim=True)
    off = x - mean
    rstd = 1.0 / torch.sqrt(off.square().mean(1, keepdim=True) + EPS)
    y = (off * rstd * s["gamma"].float() + s["beta"].float()).to(s["x"].dtype)
    return [y, mean[:, 0], rstd[:, 0]] if s["stats"] else [y]


def _norm_grad(s):
    dy, rstd = s["dy"].float(), s["rstd"][:, None]
    hat = (s["x"].float() - s["mean"][:, None]) * rstd
    u = dy * s["gamma"].float()
    dx = rstd * (u - u.mean(1, keepdim=True) - hat * (u * hat).mean(1, keepdim=True))
    kind = s["gamma"].dtype
    return [dx.to(s["x"].dtype), (dy * hat).sum(0).to(kind), dy.sum(0).to(kind)]


def _grouped(w, group, fill):
    n, k = w.shape
    pad = -k % group
    w = torch.cat([w, w.new_full((n, pad), fill)], 1) if pad else w
    return w.view(n, -1, group)


def _quantise(s):
    n, k, group, kind = s["n"], s["k"], s["group"], s["scales"].dtype
    w = _grouped(s["w"].float(), group, 0.0)
    if s["zeros"] is None:
        scale = (w.abs().amax(2) / torch.tensor(7.0, device=w.device)).to(kind)
        zero, lowest, highest = 8.0, 1, 15
    else:
        low, high = w.amin(2).clamp(max=0.0), w.amax(2).clamp(min=0.0)
        scale = ((high - low) / torch.tensor(15.0, device=w.device)).to(kind)
        lowest, highest = 0, 15
    step = scale.double()
    if s["zeros"] is not None:
        zero = torch.where(step > 0, torch.round(-low.double() / step).clamp(0, 15), 8.0)[:, :, None]
    # nearest code; the quotient in 64 bits, where values next to a border are told apart
    code = torch.where(step[:, :, None] > 0, torch.round(w.double() / step[:, :, None]), 0.0)
    code = (code + zero).clamp(lowest, highest)
    values = ((code - zero).float() * scale.float()[:, :, None]).view(n, -1)[:, :k].to(s["w"].dtype)
    return [values.contiguous(), scale] if s["zeros"] is None else [values.contiguous(), scale, zero[:, :, 0].to(torch.uint8)]


def _dense(s):
    n, k, group = s["n"], s["k"], s["group"]
    code = torch.stack([s["codes"] & 15, s["codes"] >> 4], 2).view(n, -1)[:, :k].float()
    code = _grouped(code, group, 0.0) - (8.0 if s["zeros"] is None else s["zeros"].float()[:, :, None])
    return (code * s["scales"].float()[:, :, None]).view(n, -1)[:, :k]


def _expand(s):
    w = _dense(s).to(s["w"].dtype)
    return (w.t() if s["transposed"] else w).contiguous()


def _product(s):
    return (s["x"].float() @ _dense(s).t()).to(s["x"].dtype)


# ---- the definition in 64 bits ------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "norm":
        x = s["x"].to(torch.float64)
        m = x.sum(1) / case["cols"]
        var = ((x - m.unsqueeze(1)) ** 2).sum(1) / case["cols"]
        r = (var + EPS) ** -0.5
        y = torch.addcmul(s["beta"].to(torch.float64), (x - m.unsqueeze(1)) * r.unsqueeze(1), s["gamma"].to(torch.float64))
        return [y, m, r] if case["stats"] else [y]
    if op == "norm_grad":
        # by the matrix of derivatives: dx_j = sum_i u_i r (delta_ij - 1/C - h_i h_j / C), rows in portions
        dx = torch.empty(case["rows"], case["cols"], dtype=torch.float64, device="cuda")
        dg = torch.zeros(case["cols"], dtype=torch.float64, device="cuda")
        db = torch.zeros_like(dg)
        for at in range(0, case["rows"], 4096):
            part = slice(at, at + 4096)
            g, r = s["dy"][part].to(torch.float64), s["rstd"][part].to(torch.float64).unsqueeze(1)
            h = (s["x"][part].to(torch.float64) - s["mean"][part].to(torch.float64).unsqueeze(1)) * r
            u = g * s["gamma"].to(torch.float64)
            a, b = u.sum(1, keepdim=True) / case["cols"], torch.einsum("rc,rc->r", u, h).unsqueeze(1) / case["cols"]
            dx[part] = (u - a - h * b) * r
            dg += torch.einsum("rc,rc->c", g, h)
            db += g.sum(0)
        return [dx, dg, db]
    n, k, group = case["n"], case["k"], case["group"]
    if op == "quantise":
        w = s["w"].to(torch.float64)
        values, kind = torch.empty_like(w), TYPES[case["scales"]]
        scales, points = [], []
        for at in range(0, k, group):     # group by group; the scale's two roundings belong to the format
            part = w[:, at:at + group]
            if case["zeros"]:
                low = torch.minimum(part.min(1).values, torch.zeros((), dtype=torch.float64, device="cuda"))
                high = torch.maximum(part.max(1).values, torch.zeros((), dtype=torch.float64, device="cuda"))
                d = ((high - low).to(torch.float32).to(torch.float64) / 15.0).to(torch.float32).to(kind).to(torch.float64)
                z = torch.clamp(torch.round(-low / d), 0, 15)
                z = torch.where(d == 0, torch.full_like(z, 8.0), z)
                q = torch.clamp(torch.round(part / d.unsqueeze(1)), min=-z.unsqueeze(1), max=15.0 - z.unsqueeze(1))
                points.append(z.to(torch.uint8))
            else:
                d = (part.abs().max(1).values / 7.0).to(torch.float32).to(kind).to(torch.float64)
                q = torch.clamp(torch.round(part / d.unsqueeze(1)), -7, 7)
            values[:, at:at + group] = torch.where(d.unsqueeze(1) == 0, torch.zeros_like(part), q * d.unsqueeze(1))
            scales.append(d)
        answer = [values, torch.stack(scales, 1)]
        return answer + [torch.stack(points, 1)] if case["zeros"] else answer

    # every second column from the low halves of the bytes, the others from the high halves
    def columns(first, last):
        c = s["codes"][first:last].to(torch.int16)
        w = torch.empty(c.shape[0], 2 * c.shape[1], dtype=torch.float64, device="cuda")
        w[:, 0::2], w[:, 1::2] = c.remainder(16), c.div(16, rounding_mode="floor")
        w = w[:, :k]
        at = torch.arange(k, device="cuda").div(group, rounding_mode="floor")
        if s["zeros"] is None:
            w = w - 8
        else:
            w = w - s["zeros"][first:last].to(torch.float64)[:, at]
        return w * s["scales"][first:last].to(torch.float64)[:, at]
    if op == "expand":
        w = columns(0, n)
        return w.transpose(0, 1).contiguous() if case["transposed"] else w.contiguous()
    x = s["x"].to(torch.float64)
    y = torch.empty(case["m"], n, dtype=torch.float64, device="cuda")
    for first in range(0, n, 4096):
        last = min(n, first + 4096)
        y[:, first:last] = torch.einsum("mk,nk->mn", x, columns(first, last))
    return y
