"""GPU tests of the layer operators where sums cancel, overflow or meet values that are not finite, and of launches that the sizes
of the other tests do not reach.  u = 2^-24 is the largest relative error of one FP32 rounding."""
import pytest
import torch

from oracle import layer as ref
from test_gpu_layer import TYPES, U, check_backward, check_forward, depth, gen, held, norm_inputs, within

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def b2(cuda):
    import hpcdeepneuralnetworks_b200 as b2
    return b2


CONSTANTS = [0.1, 1.0 / 3.0, 6.6125484e7, -1e9, 6.734e8, 8.5e9, -3e15]


@pytest.mark.parametrize("cols", [1000, 1027, 2000, 4095, 14336, 16390, 33000, 200003])
@pytest.mark.parametrize("rows", [7, 601])
@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
def test_layernorm_constant_rows_of_any_value(b2, rows, cols, kind):
    """All elements equal some c whose sums are not exact.  A first mean is off by at most D*u*|c|, the mean of the equal distances
    from it is right to D*u, so together they are off by (D*u)^2*|c|, less than half a step of c while D^2*u < 1 (D = 829 at 200003
    columns): the second mean is c itself, every distance 0, rstd 1/sqrt(eps) but for its rounding, y beta."""
    if cols > 40000 and rows > 7:
        pytest.skip("the longest rows are taken a few at a time")
    dtype = TYPES[kind]
    values = torch.tensor(CONSTANTS if kind != "f16" else [0.1, 1.0 / 3.0, 4097.0, -65504.0, 1.1e-5, 777.7, 6e4]).to(dtype)
    assert depth(cols) ** 2 * U < 1
    c = values[torch.arange(rows) % 7]
    x = c[:, None].expand(rows, cols).contiguous()
    beta = torch.linspace(-1, 1, cols).to(dtype)
    mean, rstd = torch.zeros(rows, device="cuda"), torch.zeros(rows, device="cuda")
    y = b2.layernorm(rows, cols, 1e-5, x.cuda(), None, beta.cuda(), mean=mean, rstd=rstd).cpu()
    assert torch.equal(mean.cpu(), c.float())
    within(rstd, torch.full((rows,), float(torch.tensor(1e-5)) ** -0.5, dtype=torch.float64), 4 * U * 1e-5 ** -0.5, "rstd")
    assert torch.equal(y, beta.expand(rows, cols))


@pytest.mark.parametrize("cols", [1000, 1027, 2000, 4096, 14336, 33000])
@pytest.mark.parametrize("rows", [6, 602])
def test_layernorm_of_rows_a_few_steps_around_a_large_mean(b2, rows, cols):
    """Values a few FP32 steps around -1e9 and around 6.7e8: what the first mean is off by is larger than the distances themselves."""
    g = gen(cols + rows)
    step = torch.tensor([64.0, 64.0])[torch.arange(rows) % 2]
    base = torch.tensor([-1e9, 6.734e8])[torch.arange(rows) % 2]
    x = base[:, None] + step[:, None] * torch.randint(-2, 3, (rows, cols), generator=g)
    mean, rstd = torch.zeros(rows, device="cuda"), torch.zeros(rows, device="cuda")
    y = b2.layernorm(rows, cols, 1e-5, x.cuda(), None, None, mean=mean, rstd=rstd)
    check_forward(x, None, None, 1e-5, y, mean, rstd, cols)


@pytest.mark.parametrize("cols", [3, 1000, 1027, 4096, 14336, 33000])
@pytest.mark.parametrize("rows", [5, 600])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_layernorm_of_rows_near_the_largest_values(b2, rows, cols, kind):
    """Rows of a type's lowest value, as masks leave them, alone or beside ordinary elements: sums stay within FP32.  Constant rows
    keep their value as the mean (as above) and give beta; in the others the squares of the distances pass FP32, so that rstd is 0
    and the outputs are beta too.  The mean is right within D*u of the mean magnitude."""
    dtype = TYPES[kind]
    low = float(torch.finfo(torch.bfloat16).min)
    x = torch.randn(rows, cols, generator=gen(rows + cols))
    at = torch.arange(rows) % 5
    x[at == 0] = low
    x[at == 1, cols // 2:] = -8e37
    x[at == 2, ::3] = 8e37
    x[at == 3] = 2.0 ** 126
    x = x.to(dtype)
    beta = torch.linspace(-1, 1, cols).to(dtype)
    mean, rstd = torch.zeros(rows, device="cuda"), torch.full((rows,), -1.0, device="cuda")
    y = b2.layernorm(rows, cols, 1e-5, x.cuda(), None, beta.cuda(), mean=mean, rstd=rstd).cpu()
    wide = x.double()
    within(mean, wide.mean(1), (depth(cols) + 4) * U * wide.abs().mean(1) + 2.0 ** -140, "mean")
    assert torch.equal(mean.cpu()[at == 0], x[at == 0, 0].float()) and torch.equal(mean.cpu()[at == 3], x[at == 3, 0].float())
    assert torch.equal(y[at != 4], beta.expand(int((at != 4).sum()), cols))
    assert bool(torch.isfinite(rstd).all()) and float(rstd[(at == 1).cuda()].abs().max()) == 0 == float(rstd[(at == 2).cuda()].abs().max())


@pytest.mark.parametrize("cols", [64, 1000, 1027, 4096, 9000])
@pytest.mark.parametrize("rows", [4, 700])
def test_layernorm_backward_of_very_small_and_very_large_rows(b2, rows, cols):
    """Rows of spread 1e-18 with rstd 1e18 .. 1e20, whose square passes FP32, and rows whose elements lie so far apart that the
    forward pass gave rstd 0: dx is finite, 0 for the latter, and within the bound of every other row."""
    x, gamma, _, dy = norm_inputs(rows, cols, torch.float32, torch.float32, cols + rows)
    at = torch.arange(rows) % 4
    x[at == 1] *= 1e-20
    x[at == 2] *= 1e-18
    x[at == 3, ::2] = 1e38
    wide = x.double()
    mean = wide.mean(1).float()
    rstd = ((wide - mean.double()[:, None]) ** 2).mean(1).rsqrt().float()
    rstd[at == 3] = 0.0
    dx, dg, db = torch.full((rows, cols), 7.0, device="cuda"), torch.zeros(cols, device="cuda"), torch.zeros(cols, device="cuda")
    b2.layernorm_backward(rows, cols, dy.cuda(), x.cuda(), gamma.cuda(), mean.cuda(), rstd.cuda(), dx, dg, db)
    assert float(rstd.max()) > 1.9e19 and bool((dx[(at == 3).cuda()] == 0).all())
    check_backward(dy, x, gamma, mean, rstd, dx, dg, db)


# ---- products with 4-bit weights --------------------------------------------------------------------
def product_bound(x, w, want, dtype, K):
    """The product of exact weights: FP32 sums of exact products x (c - z), in chains of at most 64 + K/16 additions of two roundings'
    worth each (the tensor cores cut), scaled and added in FP32, rounded once.  Only what has a weight counts: no term for the zero
    point."""
    size = x.double().abs() @ w.abs().t()
    return ref.half_step(dtype) * want.abs() + 2 * U * (64 + K / 16) * size + 4 * U * want.abs() + (2.0 ** -25 if dtype is torch.float16 else 0.0)


@pytest.mark.parametrize("M", [1, 2, 8, 12, 20, 64])
@pytest.mark.parametrize("N,K", [(70, 4096), (33, 1000), (40, 16640), (17, 515)])
@pytest.mark.parametrize("group,kind,with_zeros", [(32, "bf16", True), (64, "f16", True), (128, "f16", False), (128, "bf16", False), (256, "bf16", True),
                                                    (64, "f32", True)])
def test_w4_matvec_where_a_large_element_meets_weight_zero(b2, M, N, K, group, kind, with_zeros):
    """One element of a row, at an even or odd place, is up to 2^100 (FP16: 2^27, FP32: 2^30) times the others, and all its weights are
    0: it takes no part in the result, and must not take the digits of what does."""
    dtype = TYPES[kind]
    codes, s, z, _ = held(N, K, group, torch.float32, with_zeros, N + K)
    x = torch.randn(M, K, generator=gen(M + K))
    large, small = {"bf16": (2.0 ** 60, 2.0 ** -40), "f16": (16384.0, 2.0 ** -13), "f32": (2.0 ** 20, 2.0 ** -10)}[kind]
    x = (x * small).to(dtype)
    for m in range(M):
        k = (37 * m + 6 + m % 2) % K
        x[m, k] = large
        codes[:, k] = 8 if z is None else z[:, k // group]
    w = ref.w4_values(codes, s, z, group)
    want = x.double() @ w.t()
    y = b2.w4_matvec(M, N, K, group, 1.0, x.cuda(), ref.w4_pack(codes).cuda(), s.cuda(), None if z is None else z.to(torch.uint8).cuda(), 0.0)
    within(y, want, product_bound(x, w, want, dtype, K), "y")


@pytest.mark.parametrize("M", [1, 3, 8, 16, 33, 64])
@pytest.mark.parametrize("N,K", [(129, 1000), (1000, 515), (40, 4096), (24, 8200)])
@pytest.mark.parametrize("group,kind,scales,with_zeros,pad", [(32, "bf16", "bf16", False, 0), (64, "f16", "f16", True, 0), (128, "f32", "f32", True, 0),
                                                              (256, "bf16", "f32", True, 4112), (128, "f16", "bf16", False, 4101)])
def test_w4_matvec_within_the_bound_of_its_weights(b2, M, N, K, group, kind, scales, with_zeros, pad):
    dtype = TYPES[kind]
    codes, s, z, dev = held(N, K, group, TYPES[scales], with_zeros, N * 3 + K, pad)
    x = torch.randn(M, K, generator=gen(M * 41 + K)).to(dtype)
    w = ref.w4_values(codes, s, z, group)
    want = x.double() @ w.t()
    within(b2.w4_matvec(M, N, K, group, 1.0, x.cuda(), *dev, 0.0), want, product_bound(x, w, want, dtype, K), "y")


@pytest.mark.parametrize("M,N,K", [(1, 40, 512), (20, 40, 512)])
@pytest.mark.parametrize("kind", ["bf16", "f16"])
def test_w4_matvec_carries_every_element_of_16_bits_exactly(b2, M, N, K, kind):
    """Rows with one element of each size a type has, a step above a power of two, against weights that pick a single one: the result is
    that element, whatever stands beside it."""
    dtype, group = TYPES[kind], 32
    g = torch.finfo(dtype)
    codes = torch.full((N, K), 8)
    pick = torch.randint(0, K, (N,), generator=gen(K))
    codes[torch.arange(N), pick] = 9
    scales = torch.ones(N, K // group)
    sizes = torch.linspace(-120, 100, K).round() if kind == "bf16" else torch.linspace(-14, 14, K).round()
    x = (torch.exp2(sizes) * (1 + g.eps))[torch.randperm(K, generator=gen(3))].to(dtype).expand(M, K).contiguous()
    x[:, :3] = torch.tensor([g.max, 2.0 ** (-133 if kind == "bf16" else -24), -g.tiny], dtype=dtype)
    pick[:3] = torch.arange(3)
    codes[:3] = 8
    codes[torch.arange(3), torch.arange(3)] = 9
    y = b2.w4_matvec(M, N, K, group, 1.0, x.cuda(), ref.w4_pack(codes).cuda(), scales.cuda(), None, 0.0).cpu()
    want = x[:, pick].clone()
    if kind == "bf16":      # 2^-133 beside 2^128 is below what a row scaled by its largest element holds (2^-250 of it)
        assert bool((y[:, 1] == 0).all() or torch.equal(y[:, 1], want[:, 1]))
        y[:, 1] = want[:, 1]
    assert torch.equal(y, want)


@pytest.mark.parametrize("M,N,K,kind", [(64, 50304, 512, "bf16"), (64, 20000, 1000, "f32"), (3, 130, 1 << 20, "f16"), (9, 300, 70000, "f32"),
                                        (1, 2000, 4096, "bf16"), (2, 5000, 1001, "f16")])
def test_w4_matvec_whole_rows_that_are_not_finite(b2, M, N, K, kind):
    """Rows of nothing but NaN, and single infinities at even and odd places, beside finite rows, in long rows and in more row blocks
    than the device holds at once: no wait runs out, the finite rows keep their bound, an infinity meets its exact weight."""
    dtype, group = TYPES[kind], 64
    g = torch.Generator(device="cuda").manual_seed(M + N)
    codes = torch.randint(0, 256, (N, (K + 1) // 2), generator=g, device="cuda", dtype=torch.uint8)
    scales = (0.5 + torch.rand(N, -(-K // group), generator=g, device="cuda")) / 64
    zeros = torch.randint(0, 16, scales.shape, generator=g, device="cuda", dtype=torch.uint8)
    x = torch.randn(M, K, generator=g, device="cuda").to(dtype)
    x[0] = float("nan")
    if M > 1:
        x[1, K // 3], x[M - 1, K - 1] = -float("inf"), float("inf")
        x[1, K // 3 + 1] = -float("inf")
    y = b2.w4_matvec(M, N, K, group, 1.0, x, codes, scales, zeros, 0.0).double()
    b2.check_status()
    want, size = torch.zeros(M, N, dtype=torch.float64, device="cuda"), torch.zeros(M, N, dtype=torch.float64, device="cuda")
    for at in range(0, K, 1 << 14):         # the definition in 64 bits, in portions of K
        end = min(K, at + (1 << 14))
        part = codes[:, at // 2:(end + 1) // 2]
        w = torch.stack([part & 15, part >> 4], 2).view(N, -1)[:, :end - at].double()
        groups = torch.arange(at, end, device="cuda") // group
        w = (w - zeros[:, groups].double()) * scales[:, groups].double()
        want += x[:, at:end].double() @ w.t()
        size += x[:, at:end].double().abs() @ w.abs().t()
    assert bool(y[0].isnan().all())
    assert torch.equal(y.isnan(), want.isnan()) and torch.equal(y.isinf(), want.isinf())
    assert torch.equal(y[y.isinf()], want[want.isinf()])
    fine = torch.isfinite(want).all(1)
    assert int(fine.sum()) == max(M - 3, 0)
    tol = ref.half_step(dtype) * want.abs() + 2 * U * (64 + K / 16) * size + 4 * U * want.abs() + (2.0 ** -25 if kind == "f16" else 0.0)
    within(y[fine], want[fine].cpu(), tol[fine].cpu(), "the other rows")


def product_on_device(x, codes, scales, zeros, group):
    """(x W^T, |x| |W|^T) in 64 bits on the device, in portions of rows."""
    N, K = codes.shape[0], x.shape[1]
    at = torch.arange(K, device="cuda") // group
    want, size = torch.empty(x.shape[0], N, dtype=torch.float64, device="cuda"), torch.empty(x.shape[0], N, dtype=torch.float64, device="cuda")
    for n in range(0, N, 2048):
        part = codes[n:n + 2048]
        w = torch.stack([part & 15, part >> 4], 2).view(part.shape[0], -1)[:, :K].double()
        w = (w - (8.0 if zeros is None else zeros[n:n + 2048][:, at].double())) * scales[n:n + 2048][:, at].double()
        want[:, n:n + 2048], size[:, n:n + 2048] = x.double() @ w.t(), x.double().abs() @ w.abs().t()
    return want, size


@pytest.mark.parametrize("M,N,K,kind", [(1, 50304, 4096, "bf16"), (16, 50304, 1024, "f16"), (64, 8192, 2048, "f32"), (33, 40000, 768, "bf16"),
                                        (1, 50304, 256, "bf16"), (1, 19200, 1024, "f16"), (8, 50300, 255, "bf16"), (2, 75000, 130, "f32"),
                                        (5, 19111, 1023, "bf16")])
@pytest.mark.parametrize("group,with_zeros", [(64, True), (256, False)])
def test_w4_matvec_of_more_row_blocks_than_the_device_holds(b2, M, N, K, kind, group, with_zeros):
    """Each CTA, or cluster of CTAs, takes several row blocks one behind the other: a vocabulary head, FP32 rows in several items, small
    products that lay x out themselves (one CTA to a row block and two), rows of codes that start anywhere; twice, for equal bits."""
    dtype = TYPES[kind]
    g = torch.Generator(device="cuda").manual_seed(N + K)
    codes = torch.randint(0, 256, (N, (K + 1) // 2), generator=g, device="cuda", dtype=torch.uint8)
    scales = (0.5 + torch.rand(N, -(-K // group), generator=g, device="cuda")) / 64
    zeros = torch.randint(0, 16, scales.shape, generator=g, device="cuda", dtype=torch.uint8) if with_zeros else None
    x = torch.randn(M, K, generator=g, device="cuda").to(dtype)
    y = torch.full((M, N), float("nan"), dtype=dtype, device="cuda")
    b2.w4_matvec(M, N, K, group, 1.0, x, codes, scales, zeros, 0.0, y)
    want, size = product_on_device(x, codes, scales, zeros, group)
    tol = ref.half_step(dtype) * want.abs() + 2 * U * (64 + K / 16) * size + 4 * U * want.abs() + (2.0 ** -25 if kind == "f16" else 0.0)
    within(y, want.cpu(), tol.cpu(), "y")
    assert torch.equal(y, b2.w4_matvec(M, N, K, group, 1.0, x, codes, scales, zeros, 0.0))
    b2.check_status()


@pytest.mark.parametrize("N,K", [(3, 2), (5, 33), (33, 254), (130, 1000), (17, 2050), (257, 515), (9, 8206), (40, 4096)])
@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("group,with_zeros", [(32, True), (128, False), (256, True)])
@pytest.mark.parametrize("pad,packed", [(0, True), (1, True), (2, False), (7, True), (8, True)])
def test_w4_quantize_packed_codes_and_pitched_weights(b2, N, K, kind, group, with_zeros, pad, packed):
    """Rows of codes directly behind one another (starting at any byte), rows of W `pad` elements apart from one that starts off the
    16-byte boundaries: the definition bit for bit, and nothing beside the rows is read into them or written."""
    dtype = TYPES[kind]
    W = (torch.randn(N, K, generator=gen(N + K)) * 0.1).to(dtype)
    base = torch.full((N * (K + pad) + pad + 8,), float("nan"), dtype=dtype, device="cuda")
    at = base[pad:pad + N * (K + pad)].view(N, K + pad)[:, :K]
    at.copy_(W.cuda())
    width = (K + 1) // 2
    want, ws, wz = ref.w4_quantize(W, group, torch.float32, with_zeros)
    room = torch.full((N * width + 64,), 0x77, dtype=torch.uint8, device="cuda")
    codes = room[32:32 + N * width].view(N, width) if packed else b2.w4_empty(N, K, group)[0]
    s = torch.empty(N, -(-K // group), device="cuda")
    z = torch.empty(s.shape, dtype=torch.uint8, device="cuda") if with_zeros else None
    b2.w4_quantize(N, K, group, at, codes, s, z)
    assert torch.equal(codes.cpu(), ref.w4_pack(want)) and torch.equal(s.cpu(), ws)
    assert z is None or torch.equal(z.cpu().long(), wz)
    assert bool((room[:32] == 0x77).all()) and bool((room[32 + N * width:] == 0x77).all())
    back = b2.w4_dequantize(N, K, group, codes, s, z, dtype=dtype)
    assert torch.equal(back.cpu(), ref.w4_values(want, ws, wz if with_zeros else None, group).float().to(dtype))
