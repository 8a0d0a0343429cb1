"""Layer norm, its gradients and 4-bit weights from their formulas, in 64 bits on the CPU (torch float64).

Test infrastructure only.  Every function takes the inputs as the operators get them (already rounded to their types) and
returns float64 values (quantised ones: the exact integers and the scales' rounded values), together with the sums of
magnitudes that the tests' error bounds are stated in.
"""
import torch

D = torch.float64
LARGEST = {torch.float32: 3.4028234663852886e38, torch.bfloat16: 3.3895313892515355e38, torch.float16: 65504.0}


def half_step(dtype) -> float:
    """Largest relative error of one rounding to dtype."""
    return torch.finfo(dtype).eps / 2


def layernorm(x, gamma, beta, eps):
    """(y, mean, rstd, xhat)."""
    x = x.to(D)
    mean = x.mean(1)
    off = x - mean[:, None]
    rstd = 1.0 / torch.sqrt((off * off).mean(1) + eps)
    hat = off * rstd[:, None]
    y = hat * (1.0 if gamma is None else gamma.to(D)) + (0.0 if beta is None else beta.to(D))
    return y, mean, rstd, hat


def layernorm_backward(dy, x, gamma, mean, rstd):
    """(dx, dgamma, dbeta, and a dict of xhat, u, the rows' mean |u| and mean |u xhat|, the columns' sum |dy xhat| and |dy|)."""
    dy, x, mean, rstd = dy.to(D), x.to(D), mean.to(D)[:, None], rstd.to(D)[:, None]
    hat = (x - mean) * rstd
    u = dy * (1.0 if gamma is None else gamma.to(D))
    a, b = u.mean(1, keepdim=True), (u * hat).mean(1, keepdim=True)
    dx = rstd * (u - a - hat * b)
    sizes = {"hat": hat, "u": u, "mean_u": u.abs().mean(1, keepdim=True), "mean_uh": (u * hat).abs().mean(1, keepdim=True),
             "sum_gh": (dy * hat).abs().sum(0), "sum_g": dy.abs().sum(0)}
    return dx, (dy * hat).sum(0), dy.sum(0), sizes


def w4_quantize(W, group, scale_dtype, with_zeros):
    """(codes N x K as integers, scales N x G of scale_dtype, zeros N x G as integers): the format's definition, group by group.
    The scale's two roundings (FP32, then its type) belong to the format; everything else is exact."""
    N, K = W.shape
    W = W.to(D)
    G = -(-K // group)
    codes = torch.zeros(N, K, dtype=torch.int64)
    scales = torch.zeros(N, G, dtype=scale_dtype)
    zeros = torch.full((N, G), 8, dtype=torch.int64)
    for g in range(G):
        part = W[:, g * group:(g + 1) * group]
        bad = ~torch.isfinite(part).all(1)
        part = torch.where(bad[:, None], torch.zeros_like(part), part)
        if with_zeros:
            lo, hi = part.min(1).values.clamp(max=0.0), part.max(1).values.clamp(min=0.0)
            wide = ((hi.float() - lo.float()) / 15.0).to(D)
        else:
            wide = (part.abs().max(1).values.float() / torch.tensor(7.0)).to(D)
        s = wide.clamp(max=LARGEST[scale_dtype]).float().to(scale_dtype)
        step = s.to(D)
        live = step > 0
        safe = torch.where(live, step, torch.ones_like(step))
        if with_zeros:
            z = torch.where(live, torch.round(-lo / safe).clamp(0, 15), torch.full_like(safe, 8.0))
            c = (torch.round(part / safe[:, None]) + z[:, None]).clamp(0, 15)
        else:
            z = torch.full_like(safe, 8.0)
            c = (torch.round(part / safe[:, None]) + 8).clamp(1, 15)
        c = torch.where(live[:, None], c, z[:, None])
        z = torch.where(bad, torch.full_like(z, 8.0), z)
        c = torch.where(bad[:, None], torch.full_like(c, 8.0), c)
        codes[:, g * group:(g + 1) * group] = c.to(torch.int64)
        zeros[:, g] = z.to(torch.int64)
        scales[:, g] = torch.where(bad, torch.full_like(s, float("nan")), s)
    return codes, scales, zeros


def w4_pack(codes):
    """N x ceil(K / 2) bytes from N x K codes: even columns in the low halves."""
    N, K = codes.shape
    padded = torch.zeros(N, K + K % 2, dtype=torch.int64)
    padded[:, :K] = codes
    return (padded[:, 0::2] | (padded[:, 1::2] << 4)).to(torch.uint8)


def w4_unpack(packed, K):
    N = packed.shape[0]
    out = torch.empty(N, 2 * packed.shape[1], dtype=torch.int64)
    out[:, 0::2], out[:, 1::2] = (packed & 15).to(torch.int64), (packed >> 4).to(torch.int64)
    return out[:, :K]


def w4_values(codes, scales, zeros, group):
    """The exact matrix in float64 from integer codes (zeros None: 8)."""
    at = torch.arange(codes.shape[1]) // group
    z = 8.0 if zeros is None else zeros.to(D)[:, at]
    return (codes.to(D) - z) * scales.to(D)[:, at]
