"""GPU tests of layer norm (forward and backward) and the 4-bit-weight operators against the 64-bit reference.

Bounds.  u = 2^-24 is the largest relative error of one FP32 rounding; H = ``half_step`` of the output's type is that of the
one rounding at the store.  A sum whose terms pass through at most D additions is off by at most D*u*sum|terms| (first
order); D is taken as DEPTH(cols) = 48 + cols/256 for sums along a row: a thread adds at most max(32, cols/256) terms in a
chain and the joins of lanes, warps and blocks are at most 16 more.
Layer norm: mean is off by u*(|mean| + D*sigma) (sum of distances from a first mean), so in units of xhat by
e_m = u*(|mean|*rstd + D); rstd by (D + 4)*u relative (half of the variance's 2D, the square root, the division); then the
difference, the product, the FMA: |dy| <= H|y| + |gamma|*(e_m + u*(D + 8)*|xhat|) + 2u|y| + u*|beta|.
Gradients: mean and rstd are inputs, so xhat carries 2 roundings, u*: dx <= H|dx| + u*rstd*(6|u| + (D + 4)*mean|u| +
(D + 12)*|xhat|*mean|u xhat|); the sums over R rows D = R + 8 in whatever order.
Products: fp32 sums of exact products in chains of at most 64 + K/16 additions, two roundings' worth each because the tensor
cores cut instead of rounding; sum (c - z) x s may be formed as sum c x s - z sum x s, so each |w| = |c - z| s counts with another
z s:  H|y| + 2u*(64 + K/16)*|alpha|*sum|x|(|w| + z s) + 4u*(|alpha*acc| + |beta*y0|).
"""
import pytest
import torch

from oracle import layer as ref

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


@pytest.fixture(scope="module")
def b2(cuda):
    import hpcdeepneuralnetworks_b200 as b2
    return b2


def gen(seed):
    return torch.Generator().manual_seed(seed)


def depth(cols):
    return 48 + cols / 256


def within(got, want, tol, what):
    got = got.detach().cpu().double()
    off = (got - want).abs()
    bad = ~(off <= tol)
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} of {bad.numel()} beyond the bound, worst off {float(off[bad].max()):.3g}"


def norm_inputs(rows, cols, dtype, params, seed, offset=0.5):
    g = gen(seed)
    x = torch.randn(rows, cols, generator=g)
    x[:, ::7] *= 6.0
    x = (x + offset * torch.randn(rows, 1, generator=g)).to(dtype)
    gamma = (1 + 0.3 * torch.randn(cols, generator=g)).to(params)
    beta = (0.3 * torch.randn(cols, generator=g)).to(params)
    dy = torch.randn(rows, cols, generator=g).to(dtype)
    return x, gamma, beta, dy


def check_forward(x, gamma, beta, eps, y, mean, rstd, cols):
    wy, wm, wr, hat = ref.layernorm(x, gamma, beta, eps)
    D = depth(cols)
    sigma = 1.0 / wr
    if mean is not None:
        within(mean, wm, 2 * U * (wm.abs() + D * sigma), "mean")
        within(rstd, wr, (D + 4) * U * wr, "rstd")
    em = U * ((wm.abs() * wr)[:, None] + D)
    g = 1.0 if gamma is None else gamma.double().abs()
    b = 0.0 if beta is None else beta.double().abs()
    tol = ref.half_step(y.dtype) * wy.abs() + g * (em + U * (D + 8) * hat.abs()) + 2 * U * wy.abs() + U * b
    tol = tol + (2.0 ** -25 if y.dtype is torch.float16 else 0.0)      # half a step of FP16's subnormals
    within(y, wy, tol, "y")


SHAPES = [(1, 1), (1, 2), (3, 7), (2, 31), (5, 33), (1, 64), (17, 100), (4, 128), (300, 256), (7, 255), (33, 768), (2, 1000),
          (129, 1024), (3, 1027), (5, 2048), (6, 4096), (2, 4100), (3, 5121), (2, 8192), (2, 8200), (1, 16384), (2, 20001), (1, 32768),
          (3, 40000), (1, 70001)]


@pytest.mark.parametrize("rows,cols", SHAPES)
@pytest.mark.parametrize("kind,params", [("f32", "f32"), ("bf16", "f32"), ("bf16", "bf16"), ("f16", "f32"), ("f16", "f16")])
def test_layernorm_forward(b2, rows, cols, kind, params):
    x, gamma, beta, _ = norm_inputs(rows, cols, TYPES[kind], TYPES[params], rows * 131 + cols)
    mean, rstd = torch.full((rows,), -7.0, device="cuda"), torch.full((rows,), -7.0, device="cuda")
    y = b2.layernorm(rows, cols, 1e-5, x.cuda(), gamma.cuda(), beta.cuda(), mean=mean, rstd=rstd)
    check_forward(x, gamma, beta, 1e-5, y, mean, rstd, cols)


@pytest.mark.parametrize("given", ["none", "gamma", "beta"])
def test_layernorm_without_parameters_or_statistics(b2, given):
    x, gamma, beta, _ = norm_inputs(9, 520, torch.bfloat16, torch.float32, 5)
    gamma, beta = (gamma if given == "gamma" else None), (beta if given == "beta" else None)
    dev = lambda t: None if t is None else t.cuda()  # noqa: E731
    y = b2.layernorm(9, 520, 1e-5, x.cuda(), dev(gamma), dev(beta))
    check_forward(x, gamma, beta, 1e-5, y, None, None, 520)
    only = torch.zeros(9, device="cuda")
    b2.layernorm(9, 520, 1e-5, x.cuda(), dev(gamma), dev(beta), rstd=only)
    within(only, ref.layernorm(x, None, None, 1e-5)[2], 1e-5, "rstd alone")


@pytest.mark.parametrize("cols,pitch,shift", [(256, 300, 0), (255, 260, 1), (1024, 1025, 3), (64, 64, 5), (4096, 4104, 8), (515, 520, 2)])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_layernorm_strides_offsets_and_what_lies_between(b2, cols, pitch, shift, kind):
    rows, dtype = 11, TYPES[kind]
    x, gamma, beta, dy = norm_inputs(rows, cols, dtype, torch.float32, 77 + cols)

    def laid(values):
        base = torch.full((shift + rows * pitch + 9,), 3.0, dtype=dtype, device="cuda")
        view = base[shift:shift + rows * pitch].view(rows, pitch)[:, :cols]
        if values is not None:
            view.copy_(values.cuda())
        return base, view
    _, xv = laid(x)
    base, yv = laid(None)
    mean, rstd = torch.zeros(rows, device="cuda"), torch.zeros(rows, device="cuda")
    off = torch.cat([torch.zeros(3), gamma]).cuda()[3:], torch.cat([torch.zeros(1), beta]).cuda()[1:]
    b2.layernorm(rows, cols, 1e-5, xv, off[0], off[1], yv, mean=mean, rstd=rstd)
    check_forward(x, gamma, beta, 1e-5, yv, mean, rstd, cols)
    yv.fill_(3.0)
    assert bool((base == 3.0).all()), "something outside the rows was written"
    # the gradients of the same views
    _, gv = laid(dy)
    base, dv = laid(None)
    dgamma, dbeta = torch.zeros(cols + 1, device="cuda")[1:], torch.zeros(cols + 1, device="cuda")[1:]
    b2.layernorm_backward(rows, cols, gv, xv, off[0], mean, rstd, dv, dgamma, dbeta)
    check_backward(dy, x, gamma, mean.cpu(), rstd.cpu(), dv, dgamma, dbeta)
    dv.fill_(3.0)
    assert bool((base == 3.0).all()), "something outside the rows was written"


def test_layernorm_in_place_and_interleaved_views(b2):
    x, gamma, beta, dy = norm_inputs(6, 300, torch.float32, torch.float32, 8)
    t = x.cuda()
    assert b2.layernorm(6, 300, 1e-5, t, gamma.cuda(), beta.cuda(), t) is t
    check_forward(x, gamma, beta, 1e-5, t, None, None, 300)
    for cols in (300, 9000):      # rows held on chip and rows that are read again
        x, gamma, beta, dy = norm_inputs(6, cols, torch.bfloat16, torch.float32, 9)
        both = torch.cat([x, torch.zeros_like(x)], 1).cuda()
        b2.layernorm(6, cols, 1e-5, both[:, :cols], gamma.cuda(), beta.cuda(), both[:, cols:])
        check_forward(x, gamma, beta, 1e-5, both[:, cols:], None, None, cols)
        assert torch.equal(both[:, :cols].cpu(), x)
        mean, rstd = torch.zeros(6, device="cuda"), torch.zeros(6, device="cuda")
        b2.layernorm(6, cols, 1e-5, x.cuda(), gamma.cuda(), beta.cuda(), mean=mean, rstd=rstd)
        g = dy.cuda()
        dg, db = torch.zeros(cols, device="cuda"), torch.zeros(cols, device="cuda")
        b2.layernorm_backward(6, cols, g, x.cuda(), gamma.cuda(), mean, rstd, g, dg, db)      # dx over dy
        check_backward(dy, x, gamma, mean.cpu(), rstd.cpu(), g, dg, db)
    t = torch.zeros(6, 300, device="cuda")
    with pytest.raises(b2.B2Error, match="overlaps"):
        b2.layernorm(5, 300, 1e-5, t[:5], None, None, t[1:])
    with pytest.raises(b2.B2Error, match="overlaps"):
        b2.layernorm_backward(6, 300, t.clone(), t, None, torch.zeros(6, device="cuda"), torch.zeros(6, device="cuda"), t, None, None)


@pytest.mark.parametrize("cols", [96, 1000, 4096, 33000])
def test_layernorm_keeps_small_variance_on_a_large_mean(b2, cols):
    g = gen(cols)
    x = 1000.0 + torch.randn(4, cols, generator=g)      # FP32 holds these with 2^-14 absolute: E[x^2] - mean^2 would be lost
    mean, rstd = torch.zeros(4, device="cuda"), torch.zeros(4, device="cuda")
    y = b2.layernorm(4, cols, 0.0, x.cuda(), None, None, mean=mean, rstd=rstd)
    check_forward(x, None, None, 0.0, y, mean, rstd, cols)


@pytest.mark.parametrize("cols", [1, 96, 1000, 4096, 33000])
def test_layernorm_constant_rows_and_values_that_are_not_finite(b2, cols):
    x = torch.zeros(6, cols)
    x[0] = 4.0
    x[2, cols // 2] = float("nan")
    x[3, cols - 1] = float("inf")
    x[4, 0] = -float("inf")
    x[5] = torch.arange(cols) % 5 - 2.0
    beta = torch.linspace(-1, 1, cols)
    mean, rstd = torch.zeros(6, device="cuda"), torch.zeros(6, device="cuda")
    y = b2.layernorm(6, cols, 1e-5, x.cuda(), None, beta.cuda(), mean=mean, rstd=rstd).cpu()
    assert torch.equal(y[0], beta) and torch.equal(y[1], beta)
    assert bool(torch.isnan(y[2:5]).all()) and not bool(torch.isnan(y[[0, 1, 5]]).any())
    assert float(mean[0]) == 4.0 and abs(float(rstd[0]) - 1e-5 ** -0.5) < 1e-4


def check_backward(dy, x, gamma, mean, rstd, dx, dgamma, dbeta):
    rows, cols = x.shape
    wx, wg, wb, s = ref.layernorm_backward(dy, x, gamma, mean, rstd)
    D, r = depth(cols), rstd.double()[:, None].abs()
    if dx is not None:
        tol = U * r * (6 * s["u"].abs() + (D + 4) * s["mean_u"] + (D + 12) * s["hat"].abs() * s["mean_uh"])
        tol = tol + ref.half_step(dx.dtype) * wx.abs() + (2.0 ** -25 if dx.dtype is torch.float16 else 0.0)
        within(dx, wx, tol, "dx")
    tiny = 2.0 ** -25 if (dgamma is not None and dgamma.dtype is torch.float16) else 0.0
    if dgamma is not None:
        within(dgamma, wg, ref.half_step(dgamma.dtype) * wg.abs() + U * (rows + 10) * s["sum_gh"] + tiny, "dgamma")
    if dbeta is not None:
        within(dbeta, wb, ref.half_step(dbeta.dtype) * wb.abs() + U * (rows + 8) * s["sum_g"] + tiny, "dbeta")


def statistics(x, eps=1e-5):
    _, mean, rstd, _ = ref.layernorm(x, None, None, eps)
    return mean.float(), rstd.float()


@pytest.mark.parametrize("rows,cols", SHAPES + [(1000, 64), (777, 257), (2500, 96), (1500, 1024), (600, 2050)])
@pytest.mark.parametrize("kind,params", [("f32", "f32"), ("bf16", "f32"), ("bf16", "bf16"), ("f16", "f32"), ("f16", "f16")])
def test_layernorm_backward(b2, rows, cols, kind, params):
    x, gamma, _, dy = norm_inputs(rows, cols, TYPES[kind], TYPES[params], rows * 17 + cols)
    mean, rstd = statistics(x)
    dx = torch.full_like(x, 9.0).cuda()
    dgamma, dbeta = torch.full_like(gamma, 9.0).cuda(), torch.full_like(gamma, 9.0).cuda()
    b2.layernorm_backward(rows, cols, dy.cuda(), x.cuda(), gamma.cuda(), mean.cuda(), rstd.cuda(), dx, dgamma, dbeta)
    check_backward(dy, x, gamma, mean, rstd, dx, dgamma, dbeta)


@pytest.mark.parametrize("cols", [128, 129, 131, 242, 255, 257, 515, 1027, 2050, 2053, 4095, 5121, 8170, 8183, 16366, 16383])
@pytest.mark.parametrize("kind,params", [("f32", "f32"), ("bf16", "f32"), ("f16", "f16")])
@pytest.mark.parametrize("pads", [(0, 0), (3, 3), (5, 13), (1, 4)])
def test_layernorm_rows_that_start_anywhere(b2, cols, kind, params, pads):
    """Many rows of lengths and pitches off the 16-byte boundaries, alike (mod 8 elements) or not between input and output, with NaN
    between the input's rows and in one of them: nothing of a row's neighbours counts or is written."""
    if cols > 5121 and pads != (0, 0):
        pytest.skip("the longest rows are taken without padding alone")
    rows, dtype = 601, TYPES[kind]
    x, gamma, beta, dy = norm_inputs(rows, cols, dtype, TYPES[params], 3 * cols + pads[0])
    hole = 77
    mean, rstd = statistics(x)

    def laid(values, pad, between):
        base = torch.full((rows * (cols + pad),), between, dtype=dtype, device="cuda")
        view = base.view(rows, cols + pad)[:, :cols]
        if values is not None:
            view.copy_(values.cuda())
            view[hole] = float("nan")
        return base, view
    others = [r for r in range(rows) if r != hole]
    _, xv = laid(x, pads[0], float("nan"))
    base, yv = laid(None, pads[1], 3.0)
    m, r = torch.zeros(rows, device="cuda"), torch.zeros(rows, device="cuda")
    b2.layernorm(rows, cols, 1e-5, xv, gamma.cuda(), beta.cuda(), yv, mean=m, rstd=r)
    assert bool(torch.isnan(yv[hole]).all())
    check_forward(x[others], gamma, beta, 1e-5, yv[others], m[others], r[others], cols)
    _, gv = laid(dy, pads[0], float("nan"))
    for inplace in (False, True):
        dbase, dv = (None, gv) if inplace else laid(None, pads[1], 3.0)
        gm = torch.zeros(cols, dtype=gamma.dtype, device="cuda")
        if not inplace:      # the columns' sums need a row that is finite
            gv[hole], xv[hole] = dy[hole].cuda(), x[hole].cuda()
            dbeta = torch.zeros_like(gm)
            b2.layernorm_backward(rows, cols, gv, xv, gamma.cuda(), mean.cuda(), rstd.cuda(), dv, gm, dbeta)
            check_backward(dy, x, gamma, mean, rstd, dv, gm, dbeta)
            gv[hole] = float("nan")
        b2.layernorm_backward(rows, cols, gv, xv, gamma.cuda(), mean.cuda(), rstd.cuda(), dv, None, None)
        check_backward(dy[others], x[others], gamma, mean[others], rstd[others], dv[others], None, None)
        if dbase is not None:
            dv.fill_(3.0)
            assert bool((dbase == 3.0).all()), "something outside the rows was written"
    yv.fill_(3.0)
    assert bool((base == 3.0).all()), "something outside the rows was written"
    b2.layernorm(rows, cols, 1e-5, xv, gamma.cuda(), None, xv)
    check_forward(x, gamma, None, 1e-5, xv, None, None, cols)


@pytest.mark.parametrize("cols", [64, 1000, 5000])
@pytest.mark.parametrize("parts", ["dx", "dgamma", "dbeta", "sums", "dx+dbeta", "no gamma"])
def test_layernorm_backward_in_parts(b2, cols, parts):
    rows = 37
    x, gamma, _, dy = norm_inputs(rows, cols, torch.bfloat16, torch.float32, 55 + cols)
    mean, rstd = statistics(x)
    gamma = None if parts == "no gamma" else gamma
    dx = torch.zeros_like(x).cuda() if parts in ("dx", "dx+dbeta", "no gamma") else None
    dg = torch.zeros(cols, device="cuda") if parts in ("dgamma", "sums", "no gamma") else None
    db = torch.zeros(cols, device="cuda") if parts in ("dbeta", "sums", "dx+dbeta", "no gamma") else None
    got = b2.layernorm_backward(rows, cols, dy.cuda(), x.cuda(), None if gamma is None else gamma.cuda(), mean.cuda(), rstd.cuda(), dx, dg, db)
    assert got[0] is dx and got[1] is dg and got[2] is db
    check_backward(dy, x, gamma, mean, rstd, dx, dg, db)


@pytest.mark.parametrize("rows,cols", [(5000, 64), (3001, 515), (900, 4096), (20000, 40)])
def test_layernorm_parameter_gradients_of_whole_numbers_are_exact(b2, rows, cols):
    """With mean 0 and rstd 1 given, and small whole numbers, every partial sum is a whole number below 2^24: no row may be
    lost, counted twice or rounded."""
    g = gen(rows)
    x = torch.randint(-8, 9, (rows, cols), generator=g).float()
    dy = torch.randint(-4, 5, (rows, cols), generator=g).float()
    dg, db = torch.zeros(cols, device="cuda"), torch.zeros(cols, device="cuda")
    b2.layernorm_backward(rows, cols, dy.cuda(), x.cuda(), None, torch.zeros(rows, device="cuda"), torch.ones(rows, device="cuda"), None, dg, db)
    assert torch.equal(dg.cpu(), (dy * x).double().sum(0).float())
    assert torch.equal(db.cpu(), dy.double().sum(0).float())


def test_layernorm_backward_of_no_rows_and_of_rows_that_are_not_finite(b2):
    e, v = torch.zeros(0, 40, device="cuda"), torch.zeros(0, device="cuda")
    dg, db = torch.full((40,), 5.0, device="cuda"), torch.full((40,), 5.0, device="cuda")
    b2.layernorm_backward(0, 40, e, e, None, v, v, e.clone(), dg, db)
    assert float(dg.abs().sum()) == 0 and float(db.abs().sum()) == 0
    x, gamma, _, dy = norm_inputs(5, 600, torch.float32, torch.float32, 3)
    dy[2, 100] = float("inf")
    mean, rstd = statistics(x)
    dx = torch.zeros(5, 600, device="cuda")
    dg, db = torch.zeros(600, device="cuda"), torch.zeros(600, device="cuda")
    b2.layernorm_backward(5, 600, dy.cuda(), x.cuda(), gamma.cuda(), mean.cuda(), rstd.cuda(), dx, dg, db)
    keep = [0, 1, 3, 4]
    assert bool(torch.isfinite(dx[keep]).all()) and not bool(torch.isfinite(dx[2]).any())
    assert not bool(torch.isfinite(dg[100])) and int(torch.isfinite(dg).sum()) == 599 and int(torch.isfinite(db).sum()) == 599


def test_layernorm_gradients_against_differences(b2):
    """The gradient of sum(y * dy) by central differences of the GPU's own forward pass.  A difference over 2e is off by the
    third derivative, (e*rstd)^2/6 times sums of |dy*gamma| of order 10 (below 2e-3 here), and by the roundings of y,
    u*(D + 8)*sum|dy|*max|y| / e = 6e-8 * 60 * 200 * 4 / 0.03 < 0.1 at the very worst and a hundredth of that in root mean
    square; 0.02 absolute separates it from any wrong term, whose size is that of the gradients, 0.5 and more."""
    rows, cols, e = 2, 48, 0.03
    x, gamma, beta, dy = norm_inputs(rows, cols, torch.float32, torch.float32, 12)
    dev = [t.cuda() for t in (x, gamma, beta)]
    mean, rstd = torch.zeros(rows, device="cuda"), torch.zeros(rows, device="cuda")
    b2.layernorm(rows, cols, 1e-5, *dev, mean=mean, rstd=rstd)
    dx, dg, db = torch.zeros_like(dev[0]), torch.zeros_like(dev[1]), torch.zeros_like(dev[2])
    b2.layernorm_backward(rows, cols, dy.cuda(), dev[0], dev[1], mean, rstd, dx, dg, db)

    def loss(args):
        return float((b2.layernorm(rows, cols, 1e-5, *args).double() * dy.cuda().double()).sum())
    for which, grad in enumerate((dx, dg, db)):
        for i in range(grad.numel()):
            up, down = [t.clone() for t in dev], [t.clone() for t in dev]
            up[which].view(-1)[i] += e
            down[which].view(-1)[i] -= e
            assert abs((loss(up) - loss(down)) / (2 * e) - float(grad.view(-1)[i])) < 0.02, (which, i)


# ---- 4-bit weights --------------------------------------------------------------------------------
def weights(N, K, seed, dtype=torch.float32):
    g = gen(seed)
    w = torch.randn(N, K, generator=g) * torch.exp2(torch.randint(-6, 4, (N, 1), generator=g).float())
    return w.to(dtype)


def held(N, K, group, scale_dtype, with_zeros, seed, pad=0):
    """(integer codes, scales, zeros, device tensors) of random 4-bit weights; codes' rows `pad` bytes apart if pad."""
    g = gen(seed)
    G = -(-K // group)
    codes = torch.randint(0, 16, (N, K), generator=g)
    scales = ((0.5 + torch.rand(N, G, generator=g)) / 64).to(scale_dtype)
    zeros = torch.randint(0, 16, (N, G), generator=g) if with_zeros else None
    packed = ref.w4_pack(codes)
    width = packed.shape[1]
    pitch = max(pad, width)
    room = torch.randint(0, 256, (max(0, N * pitch),), generator=g, dtype=torch.uint8).view(N, pitch).cuda()   # junk between the rows
    room[:, :width] = packed.cuda()
    if K % 2:
        room[:, width - 1] |= 0xA0                 # the half byte behind an odd row is ignored
    return codes, scales, zeros, (room[:, :width], scales.cuda(), None if zeros is None else zeros.to(torch.uint8).cuda())


W4_SHAPES = [(1, 1), (3, 2), (2, 31), (5, 33), (4, 64), (7, 127), (16, 128), (33, 256), (9, 300), (130, 1000), (64, 1024), (17, 2050),
             (257, 515), (5, 8200), (40, 4096)]


@pytest.mark.parametrize("N,K", W4_SHAPES)
@pytest.mark.parametrize("group", [32, 64, 128, 256])
@pytest.mark.parametrize("kind,scales,with_zeros", [("f32", "f32", False), ("f32", "f16", True), ("bf16", "bf16", False), ("bf16", "f32", True),
                                                     ("f16", "f16", True), ("f16", "bf16", False)])
def test_w4_quantize_is_the_definition_bit_for_bit(b2, N, K, group, kind, scales, with_zeros):
    W = weights(N, K, N * 1009 + K, TYPES[kind])
    want, ws, wz = ref.w4_quantize(W, group, TYPES[scales], with_zeros)
    codes, s, z = b2.w4_empty(N, K, group, TYPES[scales], with_zeros)
    base = codes.as_strided((N, codes.stride(0)), (codes.stride(0), 1))
    base.fill_(0x77)
    b2.w4_quantize(N, K, group, W.cuda(), codes, s, z)
    assert torch.equal(codes.cpu(), ref.w4_pack(want))
    assert torch.equal(s.cpu(), ws)
    if with_zeros:
        assert torch.equal(z.cpu().long(), wz)
    assert bool((base[:, (K + 1) // 2:] == 0x77).all()), "bytes between the rows were written"


@pytest.mark.parametrize("with_zeros", [False, True])
def test_w4_quantize_ties_borders_and_values_that_are_not_finite(b2, with_zeros):
    W = torch.zeros(14, 64)
    ties = torch.arange(-14, 15).float() / 2          # scale 1: every half is a tie
    W[0, :29] = ties
    W[1, :29] = ties * 3.0
    W[2, :29] = torch.nextafter(ties, torch.tensor(100.0))
    W[3, :29] = torch.nextafter(ties, torch.tensor(-100.0))
    W[4, :29] = torch.nextafter(ties * 0.3, torch.tensor(100.0))
    W[5, 7] = float("nan")
    W[6, 40] = float("inf")
    W[7, 3] = -float("inf")
    W[8, :3] = torch.tensor([2.0 ** -149, -2.0 ** -147, 2.0 ** -146])       # subnormals
    W[9] = torch.linspace(-3e38, 3.4e38, 64)                              # its own step overflows: infinities and a NaN
    W[10] = torch.linspace(1.0, 2.0, 64)                                  # one sign only
    W[11] = -torch.linspace(1.0, 2.0, 64)
    W[12] = torch.linspace(-1e-30, 1e-31, 64)
    W[13] = 1e6 * torch.linspace(-1, 1, 64)                                 # beyond FP16's largest scale
    for scale in ("f32", "bf16", "f16"):
        use = W.clone()
        if with_zeros:
            use[9] = 0      # the reference forms hi - lo in FP32; its overflow is tested below
        for group in (32, 64):
            want, ws, wz = ref.w4_quantize(use, group, TYPES[scale], with_zeros)
            codes, s, z = b2.w4_empty(14, 64, group, TYPES[scale], with_zeros)
            b2.w4_quantize(14, 64, group, use.cuda(), codes, s, z)
            assert torch.equal(s.cpu().isnan(), ws.isnan())
            assert torch.equal(s.cpu().nan_to_num(-1.0), ws.nan_to_num(-1.0))
            assert torch.equal(codes.cpu(), ref.w4_pack(want)), (scale, group)
            if with_zeros:
                assert torch.equal(z.cpu().long(), wz)


def test_w4_quantize_where_the_span_passes_the_range_of_fp32(b2):
    """hi - lo is infinite in FP32, the scale (hi - lo) / 15 is not.  The codes' values are taken in 64 bits: the largest,
    (15 - 7) * 4.2667e37 = 3.4133e38, is itself beyond FP32's 3.4028e38."""
    W = torch.linspace(-3.0, 3.4, 64, dtype=torch.float64).mul(1e38).float()[None]
    assert bool(torch.isfinite(W).all())
    codes, s, z = b2.w4_empty(1, 64, 64, torch.float32, True)
    b2.w4_quantize(1, 64, 64, W.cuda(), codes, s, z)
    back = ref.w4_values(ref.w4_unpack(codes.cpu(), 64), s.cpu(), z.cpu(), 64)
    # half a step for the code, half a step for the zero point
    assert float((back - W.double()).abs().max()) <= 1.001 * float(s.double())


@pytest.mark.parametrize("N,K", W4_SHAPES)
@pytest.mark.parametrize("transpose", [False, True])
@pytest.mark.parametrize("group,kind,scales,with_zeros,pad", [(32, "f32", "bf16", False, 0), (64, "bf16", "bf16", True, 0), (128, "f16", "f16", True, 4112),
                                                              (256, "f32", "f32", True, 4200), (64, "f32", "f16", False, 4101)])
def test_w4_dequantize(b2, N, K, transpose, group, kind, scales, with_zeros, pad):
    codes, s, z, dev = held(N, K, group, TYPES[scales], with_zeros, N * 7 + K, pad)
    want = ref.w4_values(codes, s, z, group).float().to(TYPES[kind])      # one FP32 product, one rounding to the type
    want = want.t() if transpose else want
    rows, cols = want.shape
    base = torch.full((rows, cols + 5), 3.0, dtype=TYPES[kind], device="cuda")
    b2.w4_dequantize(N, K, group, *dev, base[:, :cols], transpose=transpose)
    assert torch.equal(base[:, :cols].cpu(), want)
    assert bool((base[:, cols:] == 3.0).all())
    assert torch.equal(b2.w4_dequantize(N, K, group, *dev, transpose=transpose, dtype=TYPES[kind]).cpu(), want)


def check_matvec(b2, M, N, K, group, kind, scales, with_zeros, alpha=1.0, beta=0.0, pad=0, seed=0):
    codes, s, z, dev = held(N, K, group, TYPES[scales], with_zeros, N * 3 + K + seed, pad)
    g = gen(M * 37 + K)
    x = torch.randn(M, K, generator=g).to(TYPES[kind])
    y0 = torch.randn(M, N, generator=g).to(TYPES[kind])
    y = y0.cuda() if beta != 0 else torch.full((M, N), float("nan"), dtype=TYPES[kind], device="cuda")
    b2.w4_matvec(M, N, K, group, alpha, x.cuda(), *dev, beta, y)
    w = ref.w4_values(codes, s, z, group)
    acc, size = x.double() @ w.t(), x.double().abs() @ w.abs().t()
    want = alpha * acc + beta * y0.double()
    # the kernel may take the zero point off before or after the sums: the magnitudes of both forms, |c - z| + z at most
    at = torch.arange(K) // group
    size = size + x.double().abs() @ ((8.0 if z is None else z.double()[:, at]) * s.double()[:, at]).t()
    tol = ref.half_step(y.dtype) * want.abs() + 2 * U * (64 + K / 16) * abs(alpha) * size
    tol = tol + 4 * U * ((alpha * acc).abs() + (beta * y0.double()).abs()) + (2.0 ** -25 if kind == "f16" else 0.0)
    within(y, want, tol, "y")


MATVEC_SHAPES = [(1, 1), (1, 2), (3, 31), (2, 33), (8, 64), (15, 130), (16, 128), (17, 256), (100, 300), (129, 1000), (64, 1024), (33, 2050),
                 (1000, 515), (40, 4096), (24, 8200), (257, 1536)]


@pytest.mark.parametrize("N,K", MATVEC_SHAPES)
@pytest.mark.parametrize("M", [1, 2, 5, 8, 9, 16, 33, 64])
@pytest.mark.parametrize("group,kind,scales,with_zeros", [(32, "bf16", "bf16", False), (64, "f16", "f16", True), (128, "f32", "f32", True),
                                                          (256, "bf16", "f32", True), (128, "f32", "bf16", False)])
def test_w4_matvec(b2, M, N, K, group, kind, scales, with_zeros):
    check_matvec(b2, M, N, K, group, kind, scales, with_zeros)


@pytest.mark.parametrize("M", [3, 4, 6, 7, 10, 11, 12, 15, 17, 24, 25, 31, 32, 40, 48, 63])
@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
def test_w4_matvec_every_count_of_rows(b2, M, kind):
    check_matvec(b2, M, 50, 416, 32, kind, kind, M % 2 == 0)


@pytest.mark.parametrize("pad", [256, 260, 257, 272])
@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("alpha,beta", [(0.5, 0.0), (1.0, 1.0), (-2.0, 0.25)])
def test_w4_matvec_pitches_alpha_and_beta(b2, pad, kind, alpha, beta):
    check_matvec(b2, 3, 70, 500, 64, kind, "f32", True, alpha, beta, pad)
    check_matvec(b2, 1, 33, 512, 128, kind, kind, False, alpha, beta, pad)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_w4_matvec_strided_rows_and_what_lies_between(b2, kind):
    M, N, K, group, dtype = 5, 37, 200, 64, TYPES[kind]
    codes, s, z, dev = held(N, K, group, dtype, True, 4)
    x = torch.randn(M, K, generator=gen(1)).to(dtype)
    xb = torch.full((M, K + 3), float("nan"), dtype=dtype, device="cuda")       # NaN next to the rows must not be read into them
    xb[:, 1:K + 1] = x.cuda()
    yb = torch.full((M, N + 4), 3.0, dtype=dtype, device="cuda")
    b2.w4_matvec(M, N, K, group, 1.0, xb[:, 1:K + 1], *dev, 0.0, yb[:, 2:N + 2])
    w = ref.w4_values(codes, s, z, group)
    want = x.double() @ w.t()
    within(yb[:, 2:N + 2], want, ref.half_step(dtype) * want.abs() + 2 * U * (64 + K / 16) * (x.double().abs() @ (w.abs().t() + 0.5)), "y")
    assert bool((yb[:, :2] == 3.0).all()) and bool((yb[:, N + 2:] == 3.0).all())


@pytest.mark.parametrize("M,N,K", [(1, 700, 4096), (4, 130, 8192), (16, 64, 2080), (2, 2000, 384), (33, 40, 1000)])
@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
def test_w4_matvec_of_whole_numbers_is_exact(b2, M, N, K, kind):
    """Whole activations and scales that are powers of two: every partial sum is exact in FP32, so the result is."""
    g = gen(K + N)
    group = 32
    G = -(-K // group)
    codes = torch.randint(0, 16, (N, K), generator=g)
    zeros = torch.randint(0, 16, (N, G), generator=g)
    scales = torch.exp2(torch.randint(-1, 2, (N, G), generator=g).float())
    x = torch.randint(-7, 8, (M, K), generator=g).to(TYPES[kind])
    want = x.double() @ ref.w4_values(codes, scales, zeros, group).t()
    y = b2.w4_matvec(M, N, K, group, 1.0, x.cuda(), ref.w4_pack(codes).cuda(), scales.cuda(), zeros.to(torch.uint8).cuda(), 0.0)
    assert torch.equal(y.cpu(), want.float().to(TYPES[kind]))


def test_w4_matvec_f32_keeps_large_small_and_not_finite_values(b2):
    """FP32 activations from 1e-20 to FLT_MAX in rows of their own; infinities and NaN reach only their own row."""
    N, K, group = 40, 96, 32
    codes, s, z, dev = held(N, K, group, torch.float32, False, 11)
    w = ref.w4_values(codes, s, z, group)
    x = torch.randn(8, K, generator=gen(2))
    x[1] *= 1e-20
    x[2] *= 1e30
    x[3] = 0
    x[3, 5] = 3.4028234e38
    x[4, 7] = float("inf")
    x[5, 9] = float("nan")
    x[6] = 0
    x[7] = 1.0 + 2.0 ** -23
    y = b2.w4_matvec(8, N, K, group, 1.0, x.cuda(), *dev, 0.0).cpu()
    want = x.double() @ w.t()
    size = x.double().abs() @ (w.abs().t() + 8 * s.double()[:, torch.arange(K) // group].t())
    for m in (0, 1, 2, 3, 6, 7):
        within(y[m], want[m], 2 * U * (64 + K / 16) * size[m] + U * want[m].abs(), f"row {m}")
    hit = codes[:, 7] != 8
    assert bool((y[4][hit] == torch.where(codes[:, 7] > 8, 1.0, -1.0)[hit] * float("inf")).all()) and bool(y[4][~hit].isnan().all())
    assert bool(y[5].isnan().all())


@pytest.mark.parametrize("M,N,K", [(4, 200, 2304), (1, 40, 700), (16, 300, 2304), (40, 150, 1000), (8, 2500, 8200)])
@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
def test_w4_matvec_infinities_and_nan_anywhere(b2, M, N, K, kind):
    """Elements that are not finite, in one row or several and at both ends of K, meet their exact weights: their row's outputs
    are +-inf by the sign of the weight, NaN where it is 0 or two infinities differ; the other rows keep their bound."""
    dtype, group = TYPES[kind], 64
    codes, s, z, dev = held(N, K, group, torch.float32, True, M + K)
    w = ref.w4_values(codes, s, z, group)
    x = torch.randn(M, K, generator=gen(M)).to(dtype)
    x[0, K - 1] = float("inf")
    if M > 3:
        x[2, 0], x[2, K // 2] = -float("inf"), float("inf")
        x[3, K // 3] = float("nan")
    y = b2.w4_matvec(M, N, K, group, 1.0, x.cuda(), *dev, 0.0).cpu().double()
    want = x.double() @ w.t()                   # 0 * inf and inf - inf are NaN here too
    assert torch.equal(y.isnan(), want.isnan()) and torch.equal(y == float("inf"), want == float("inf"))
    assert torch.equal(y == -float("inf"), want == -float("inf"))
    fine = torch.isfinite(want).all(1)
    assert int(fine.sum()) == M - (3 if M > 3 else 1)
    at = torch.arange(K) // group
    size = x[fine].double().abs() @ (w.abs() + 16.0 * s.double()[:, at]).t()
    tol = ref.half_step(dtype) * want[fine].abs() + 2 * U * (64 + K / 16) * size + (2.0 ** -25 if kind == "f16" else 0.0)
    within(y[fine], want[fine], tol, "the other rows")


@pytest.mark.parametrize("M", [3, 12])
def test_w4_matvec_rows_of_very_different_size(b2, M):
    """Each row is scaled by itself: rows of 1e-30, 1 and 1e30 in one product, and elements 2^-20 of their row's largest."""
    N, K, group = 60, 1600, 128
    codes, s, z, dev = held(N, K, group, torch.bfloat16, False, 8)
    w = ref.w4_values(codes, s, z, group)
    x = torch.randn(M, K, generator=gen(5))
    x[:, 5::7] *= 2.0 ** -20
    x = (x * torch.tensor([1e-30, 1.0, 1e30])[torch.arange(M) % 3][:, None]).to(torch.bfloat16)
    y = b2.w4_matvec(M, N, K, group, 1.0, x.cuda(), *dev, 0.0)
    want = x.double() @ w.t()
    size = x.double().abs() @ (w.abs() + 8.0 * s.double()[:, torch.arange(K) // group]).t()
    within(y, want, ref.half_step(torch.bfloat16) * want.abs() + 2 * U * (64 + K / 16) * size, "y")
    # a row whose elements are all tiny but one: the tiny ones still count
    one = torch.full((1, K), 2.0 ** -16, dtype=torch.bfloat16)
    one[0, 0] = 1024.0
    y = b2.w4_matvec(1, N, K, group, 1.0, one.cuda(), *dev, 0.0)
    want = one.double() @ w.t()
    size = one.double() @ (w.abs() + 8.0 * s.double()[:, torch.arange(K) // group]).t()
    within(y, want, ref.half_step(torch.bfloat16) * want.abs() + 2 * U * (64 + K / 16) * size, "y")


@pytest.mark.parametrize("M", [1, 20])
def test_w4_a_bad_weight_shows_in_its_output_alone(b2, M):
    N, K, group = 50, 640, 128
    W = weights(N, K, 3)
    W[7, 200], W[30, 639] = float("nan"), float("inf")
    codes, s, z = b2.w4_empty(N, K, group, torch.bfloat16)
    b2.w4_quantize(N, K, group, W.cuda(), codes, s, z)
    y = b2.w4_matvec(M, N, K, group, 1.0, torch.randn(M, K, generator=gen(1)).cuda(), codes, s, z, 0.0).cpu()
    bad = torch.zeros(N, dtype=torch.bool)
    bad[[7, 30]] = True
    assert bool(y[:, bad].isnan().all()) and bool(torch.isfinite(y[:, ~bad]).all())


@pytest.mark.parametrize("rows,cols", [(40, 9000), (5, 100000), (700, 8200), (3, 8193)])
def test_layernorm_backward_of_the_longest_rows(b2, rows, cols):
    x, gamma, _, dy = norm_inputs(rows, cols, torch.bfloat16, torch.float32, rows)
    mean, rstd = statistics(x)
    dx, dg, db = torch.zeros_like(x).cuda(), torch.zeros(cols, device="cuda"), torch.zeros(cols, device="cuda")
    b2.layernorm_backward(rows, cols, dy.cuda(), x.cuda(), gamma.cuda(), mean.cuda(), rstd.cuda(), dx, dg, db)
    check_backward(dy, x, gamma, mean, rstd, dx, dg, db)
    dx2 = torch.zeros_like(dx)
    b2.layernorm_backward(rows, cols, dy.cuda(), x.cuda(), gamma.cuda(), mean.cuda(), rstd.cuda(), dx2, None, None)
    assert torch.equal(dx, dx2)


def test_w4_matvec_short_cuts(b2):
    codes, s, z, dev = held(20, 64, 32, torch.float32, False, 1)
    x = torch.full((3, 64), float("nan"), device="cuda")
    y = torch.arange(60, device="cuda").float().view(3, 20)
    want = (0.5 * y).clone()
    b2.w4_matvec(3, 20, 64, 32, 0.0, x, *dev, 0.5, y)                 # alpha = 0: x is not read
    assert torch.equal(y, want)
    b2.w4_matvec(3, 20, 64, 32, 0.0, x, *dev, 0.0, y)
    assert float(y.abs().sum()) == 0
    y.fill_(2.0)
    none = torch.zeros(20, 0, dtype=torch.uint8, device="cuda"), torch.zeros(20, 0, device="cuda")
    b2.w4_matvec(3, 20, 0, 32, 1.0, torch.zeros(3, 0, device="cuda"), *none, None, 0.25, y)      # K = 0: y = beta * y
    assert bool((y == 0.5).all())
    assert b2.w4_matvec(0, 20, 64, 32, 1.0, torch.zeros(0, 64, device="cuda"), *dev, 0.0).shape == (0, 20)
    with pytest.raises(b2.B2Error, match="exceeds"):
        b2.w4_matvec(65, 20, 64, 32, 1.0, torch.zeros(65, 64, device="cuda"), *dev, 0.0)
    with pytest.raises(ValueError, match="beta"):
        b2.w4_matvec(1, 20, 64, 32, 1.0, torch.zeros(1, 64, device="cuda"), *dev, 1.0)
    with pytest.raises(TypeError, match="codes"):
        b2.w4_matvec(1, 20, 64, 32, 1.0, torch.zeros(1, 64, device="cuda"), dev[0].to(torch.int8), dev[1], None, 0.0)
    with pytest.raises(TypeError, match="y"):
        b2.w4_matvec(1, 20, 64, 32, 1.0, torch.zeros(1, 64, device="cuda"), *dev, 0.0, torch.zeros(1, 20, dtype=torch.float16, device="cuda"))


# ---- a run of them together; streams and graphs ----------------------------------------------------
def test_norm_and_quantised_projection_served_and_tuned(b2):
    """One layer: y = W * LN(x) with 4-bit W.  Served: norm, then the product of a few rows.  Tuned with W frozen: the expanded
    weights in the library's SGEMM both ways, and the norm's gradients."""
    rows, cols, N, group = 6, 320, 200, 64
    x, gamma, beta, _ = norm_inputs(rows, cols, torch.float32, torch.float32, 21)
    W = weights(N, cols, 22)
    codes, s, z = b2.w4_empty(N, cols, group, torch.float32, True)
    b2.w4_quantize(N, cols, group, W.cuda(), codes, s, z)
    icodes = ref.w4_unpack(codes.cpu(), cols)
    w = ref.w4_values(icodes, s.cpu(), z.cpu(), group)
    mean, rstd = torch.zeros(rows, device="cuda"), torch.zeros(rows, device="cuda")
    h = b2.layernorm(rows, cols, 1e-5, x.cuda(), gamma.cuda(), beta.cuda(), mean=mean, rstd=rstd)
    served = b2.w4_matvec(rows, N, cols, group, 1.0, h, codes, s, z, 0.0)
    wt = b2.w4_dequantize(N, cols, group, codes, s, z, transpose=True)
    tuned = torch.zeros(rows, N, device="cuda")
    b2.sgemm(rows, N, cols, 1.0, h, wt, 0.0, tuned)
    wy = ref.layernorm(x, gamma, beta, 1e-5)[0]
    want = wy @ w.t()
    size = wy.abs() @ (w.abs().t() + 8 * s.cpu().double()[:, torch.arange(cols) // group].t())
    # the norm's bound is below 200u of each |y|, the product's 2u*(64 + K/16), the SGEMM's K*u
    within(served, want, U * (400 + 2 * (64 + cols / 16)) * size, "served")
    within(tuned, want, U * (400 + cols + 2) * size, "tuned")
    # backward: dh = dy * W, then the norm's gradients
    dy = torch.randn(rows, N, generator=gen(23))
    wn = b2.w4_dequantize(N, cols, group, codes, s, z)
    dh = torch.zeros(rows, cols, device="cuda")
    b2.sgemm(rows, cols, N, 1.0, dy.cuda(), wn, 0.0, dh)
    dx, dg, db = torch.zeros(rows, cols, device="cuda"), torch.zeros(cols, device="cuda"), torch.zeros(cols, device="cuda")
    b2.layernorm_backward(rows, cols, dh, x.cuda(), gamma.cuda(), mean, rstd, dx, dg, db)
    check_backward(dh.cpu(), x, gamma, mean.cpu(), rstd.cpu(), dx, dg, db)
    xd = x.double().requires_grad_()
    gd, bd = gamma.double().requires_grad_(), beta.double().requires_grad_()
    off = xd - xd.mean(1, keepdim=True)
    out = (off / torch.sqrt((off * off).mean(1, keepdim=True) + 1e-5) * gd + bd) @ w.t()
    (out * dy.double()).sum().backward()
    for got, whole in ((dx, xd.grad), (dg, gd.grad), (db, bd.grad)):
        assert float((got.cpu().double() - whole).norm() / whole.norm()) < 1e-5


def test_streams_at_once_and_graphs_that_replay_at_once(b2):
    """Two streams with their own tensors, and two captured graphs replayed at once, give the bits of calls made alone."""
    rows, cols, N, group = 700, 1000, 300, 32
    sets = []
    for seed in (1, 2):
        x, gamma, beta, dy = [t.cuda() for t in norm_inputs(rows, cols, torch.bfloat16, torch.float32, seed)]
        _, s, z, dev = held(N, cols, group, torch.bfloat16, True, seed)
        sets.append(dict(x=x, gamma=gamma, beta=beta, dy=dy, w=dev, y=torch.zeros_like(x), mean=torch.zeros(rows, device="cuda"),
                         rstd=torch.zeros(rows, device="cuda"), dx=torch.zeros_like(x), dg=torch.zeros(cols, device="cuda"),
                         db=torch.zeros(cols, device="cuda"), out=torch.zeros(8, N, dtype=torch.bfloat16, device="cuda"),
                         back=torch.zeros(N, cols, device="cuda"), ws=None))

    def step(d):
        b2.layernorm(rows, cols, 1e-5, d["x"], d["gamma"], d["beta"], d["y"], mean=d["mean"], rstd=d["rstd"])
        b2.layernorm_backward(rows, cols, d["dy"], d["x"], d["gamma"], d["mean"], d["rstd"], d["dx"], d["dg"], d["db"], workspace=d["ws"])
        b2.w4_matvec(8, N, cols, group, 1.0, d["y"][:8], *d["w"], 0.0, d["out"])
        b2.w4_dequantize(N, cols, group, *d["w"], d["back"])
    names = ("y", "mean", "rstd", "dx", "dg", "db", "out", "back")
    want = []
    for d in sets:
        step(d)
        torch.cuda.synchronize()
        want.append({n: d[n].clone() for n in names})

    def same_and_clear():
        torch.cuda.synchronize()
        for d, w in zip(sets, want):
            for n in names:
                assert torch.equal(d[n], w[n]), n
                d[n].fill_(-1.0)
        torch.cuda.synchronize()
    same_and_clear()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        for d, st in zip(sets, streams):
            with torch.cuda.stream(st):
                step(d)
    same_and_clear()
    need = b2.layernorm_backward_workspace_bytes(rows, cols)
    graphs = []
    for d, st in zip(sets, streams):
        d["ws"] = torch.empty(need, dtype=torch.uint8, device="cuda")
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st):
            step(d)
        graphs.append(graph)
    torch.cuda.synchronize()
    for _ in range(3):
        for graph, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                graph.replay()
    same_and_clear()


def test_results_repeat_bit_for_bit(b2):
    x, gamma, beta, dy = [t.cuda() for t in norm_inputs(3000, 520, torch.float32, torch.float32, 31)]
    mean, rstd = torch.zeros(3000, device="cuda"), torch.zeros(3000, device="cuda")
    _, s, z, dev = held(500, 520, 64, torch.float32, True, 5)
    first = None
    for _ in range(4):
        dx, dg, db = torch.zeros_like(x), torch.zeros_like(gamma), torch.zeros_like(gamma)
        y = b2.layernorm(3000, 520, 1e-5, x, gamma, beta, mean=mean, rstd=rstd)
        b2.layernorm_backward(3000, 520, dy, x, gamma, mean, rstd, dx, dg, db)
        out = b2.w4_matvec(3, 500, 520, 64, 1.0, y[:3], *dev, 0.0)
        now = [y, dx, dg, db, out]
        first = first or now
        assert all(torch.equal(a, b) for a, b in zip(first, now))


def test_offsets_beyond_32_bits(b2):
    """Rows that start beyond 2^32 bytes and beyond 2^32 elements: only the first and the last are filled and compared."""
    if torch.cuda.get_device_properties(0).total_memory < 40 << 30:
        pytest.skip("needs 24 GB")
    cols, pitch, rows = 128, 1 << 22, 1030                  # 4.3e9 elements, 8.6 GB
    big = torch.empty(rows * pitch, dtype=torch.bfloat16, device="cuda")
    view = big.view(rows, pitch)[:, :cols]
    x, gamma, beta, _ = norm_inputs(rows, cols, torch.bfloat16, torch.float32, 3)
    view.copy_(x.cuda())
    y = b2.layernorm(rows, cols, 1e-5, view, gamma.cuda(), beta.cuda())
    check_forward(x, gamma, beta, 1e-5, y, None, None, cols)
    del big, view
    N, K, group, pitch = 1100, 256, 128, 1 << 22             # 4.6e9 bytes of codes
    big = torch.empty(N * pitch, dtype=torch.uint8, device="cuda").view(N, pitch)[:, :K // 2]
    codes, s, z, dev = held(N, K, group, torch.bfloat16, True, 9)
    big.copy_(dev[0])
    xs = torch.randn(2, K, generator=gen(2)).to(torch.bfloat16).cuda()
    assert torch.equal(b2.w4_matvec(2, N, K, group, 1.0, xs, big, dev[1], dev[2], 0.0), b2.w4_matvec(2, N, K, group, 1.0, xs, *dev, 0.0))
    want = b2.w4_dequantize(N, K, group, *dev)
    assert torch.equal(b2.w4_dequantize(N, K, group, big, dev[1], dev[2]), want)
    big.fill_(0)
    c2, s2, z2 = b2.w4_empty(N, K, group, torch.float32, True)
    b2.w4_quantize(N, K, group, want, c2, s2, z2)
    b2.w4_quantize(N, K, group, want, big, s2, z2)
    assert torch.equal(big, c2)


def test_w4_rows_as_long_as_they_may_be(b2):
    """One row of nearly 2^31 weights, whole numbers that the codes reproduce, and a product of 2^27 of them."""
    if torch.cuda.get_device_properties(0).total_memory < 40 << 30:
        pytest.skip("needs 24 GB")
    K, group = 2 ** 31 - 9, 256
    codes = torch.randint(1, 16, (1, (K + 1) // 2), dtype=torch.uint8, device="cuda") * 16 + 1     # odd elements 1..15, even ones 1: -7
    codes[0, -1] = 1
    scales = torch.ones(1, -(-K // group), dtype=torch.float16, device="cuda")
    W = b2.w4_dequantize(1, K, group, codes, scales, dtype=torch.float16)
    for at in (0, 2 ** 28 - 4, 2 ** 30 - 4, K - 1001):
        at -= at % 2
        want = torch.stack([(codes[0, at // 2:at // 2 + 500] & 15), codes[0, at // 2:at // 2 + 500] >> 4], 1).view(-1).to(torch.int16) - 8
        assert torch.equal(W[0, at:at + 1000][:K - at], want.to(torch.float16)[:K - at])
    again, s2, _ = b2.w4_quantize(1, K, group, W, torch.empty_like(codes), torch.empty_like(scales))
    assert torch.equal(again, codes) and bool((s2 == 1).all())
    del W, again
    K = 2 ** 27
    x = torch.zeros(1, K, dtype=torch.float16, device="cuda")
    x[0, 1::2 ** 12] = 1.0
    got = b2.w4_matvec(1, 1, K, group, 1.0, x, codes[:, :K // 2], scales[:, :K // group].contiguous(), None, 0.0)
    want = ((codes[0, :K // 2:2 ** 11] >> 4).double() - 8).sum()
    assert abs(float(got) - float(want)) <= 2.0 ** -11 * abs(float(want)) + 1e-3


def test_handles_and_devices(b2):
    x, gamma, beta, _ = [t.cuda() for t in norm_inputs(4, 64, torch.float32, torch.float32, 2)]
    own = b2.Handle()
    assert torch.equal(b2.layernorm(4, 64, 1e-5, x, gamma, beta, handle=own), b2.layernorm(4, 64, 1e-5, x, gamma, beta))
    own.close()


def test_short_and_long_calls_agree(b2, monkeypatch):
    """Usual calls go through the extension, others (a pitch by name, a handle of the caller's that is not the default, tensors that
    are slices) through the checks in Python: the same bits, the same errors."""
    from hpcdeepneuralnetworks_b200 import layer
    b2.default_handle()
    layer._load()
    quick = layer._quick
    x, gamma, beta, dy = [t.cuda() for t in norm_inputs(33, 300, torch.bfloat16, torch.float32, 4)]
    W = weights(70, 500, 9, torch.bfloat16).cuda()
    xs = torch.randn(9, 500, generator=gen(3)).to(torch.bfloat16).cuda()

    def everything(pitch):
        ld = dict(ldx=300) if pitch else {}
        mean, rstd = torch.zeros(33, device="cuda"), torch.zeros(33, device="cuda")
        y = b2.layernorm(33, 300, 1e-5, x, gamma, beta, torch.empty_like(x), mean=mean, rstd=rstd, **ld)
        dx, dg, db = torch.empty_like(x), torch.empty_like(gamma), torch.empty_like(gamma)
        b2.layernorm_backward(33, 300, dy, x, gamma, mean, rstd, dx, dg, db, **ld)
        codes, scales, zeros = b2.w4_empty(70, 500, 64, zeros=True)
        ldq = dict(ldq=codes.stride(0)) if pitch else {}
        b2.w4_quantize(70, 500, 64, W, codes, scales, zeros, **ldq)
        out = torch.empty(500, 70, device="cuda")
        b2.w4_dequantize(70, 500, 64, codes, scales, zeros, out, transpose=True, **ldq)
        p = b2.w4_matvec(9, 70, 500, 64, 1.0, xs, codes, scales, zeros, 0.0, torch.empty(9, 70, dtype=xs.dtype, device="cuda"), **ldq)
        return [y, mean, rstd, dx, dg, db, codes.clone(), scales, zeros, out, p]

    taken = []

    class Spy:
        def __getattr__(self, name):
            def f(*args):
                taken.append((name, getattr(quick, name)(*args)))
                return taken[-1][1]
            return f
    monkeypatch.setattr(layer, "_quick", Spy())
    short = everything(False)
    assert taken == [(n, True) for n in ("layernorm", "layernorm_backward", "w4_quantize", "w4_dequantize", "w4_matvec")]
    taken.clear()
    long = everything(True)
    assert not taken
    for a, b in zip(short, long):
        assert torch.equal(a, b)
    # a batch of sequences, by its leading dimensions
    three = b2.layernorm(33, 300, 1e-5, x.view(3, 11, 300), gamma, beta, torch.empty(3, 11, 300, dtype=x.dtype, device="cuda"))
    assert taken.pop() == ("layernorm", True) and torch.equal(three.view(33, 300), short[0])
    # what the library refuses, and what is no usual call, is said as before
    with pytest.raises(b2.B2Error, match="overlaps"):
        flat = torch.zeros(34 * 300, dtype=x.dtype, device="cuda")
        b2.layernorm(33, 300, 1e-5, flat[:33 * 300].view(33, 300), gamma, beta, flat[300:].view(33, 300))
    with pytest.raises(b2.B2Error, match="workspace"):
        b2.layernorm_backward(33, 300, dy, x, gamma, short[1], short[2], None, short[4], None, workspace=torch.empty(8, device="cuda"))
    with pytest.raises(TypeError):
        b2.layernorm(33, 300, 1e-5, x, gamma.double(), beta, torch.empty_like(x))
    with pytest.raises(ValueError):
        b2.layernorm(34, 300, 1e-5, x, gamma, beta, torch.empty_like(x))
    with pytest.raises(ValueError, match="group 33"):
        b2.w4_quantize(70, 500, 33, W, short[6], short[7])
    sliced = b2.layernorm(33, 200, 1e-5, x[:, :200], gamma[:200], beta[:200], torch.empty(33, 200, dtype=x.dtype, device="cuda"))
    check_forward(x[:, :200].cpu(), gamma[:200].cpu(), beta[:200].cpu(), 1e-5, sliced, None, None, 200)
    assert all(ok is False for _, ok in taken)
    other = b2.Handle()
    assert torch.equal(b2.layernorm(33, 300, 1e-5, x, gamma, beta, torch.empty_like(x), handle=other), short[0]) and taken.pop()[1] is True


def test_first_calls_ever_inside_a_capture():
    """A process whose first calls are captured: nothing that the first call of a kernel sets up may break the capture."""
    import subprocess
    import sys
    code = """
import torch, hpcdeepneuralnetworks_b200 as b2
b2.default_handle()
x = torch.randn(40, 512, device="cuda"); g = torch.randn(512, device="cuda"); y = torch.empty_like(x)
m, r = torch.empty(40, device="cuda"), torch.empty(40, device="cuda"); dx = torch.empty_like(x); dg, db = torch.empty_like(g), torch.empty_like(g)
codes, s, _ = b2.w4_empty(256, 512, 64); W = torch.randn(256, 512, device="cuda"); back = torch.empty_like(W); p = torch.empty(40, 256, device="cuda")
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    b2.layernorm(40, 512, 1e-5, x, g, None, y, mean=m, rstd=r)
    b2.layernorm_backward(40, 512, y, x, g, m, r, dx, dg, db)
    b2.w4_quantize(256, 512, 64, W, codes, s)
    b2.w4_dequantize(256, 512, 64, codes, s, None, back)
    b2.w4_matvec(40, 256, 512, 64, 1.0, y, codes, s, None, 0.0, p)
graph.replay()
torch.cuda.synchronize()
want = torch.nn.functional.layer_norm(x.double(), (512,), g.double())
assert float((y - want).abs().max()) < 1e-4
assert float((p - y.double() @ back.double().t()).abs().max()) < 1e-2
print("captured")
"""
    import os
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300,
                       cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
    assert r.returncode == 0 and "captured" in r.stdout, r.stderr[-2000:]
