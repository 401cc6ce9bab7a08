"""Layer norm, 8-bit rows and their products where they can go wrong: what the backward pass reads of kept rows, means far from zero,
types of gradients, sums that cancel, and the largest sizes and values (tests/rows8_oracle.py in 64 bits).

Tolerances as in test_layernorm_gpu.py and test_rows8_gpu.py; where one is new, its test derives it."""
import pytest
import torch

from tests import rows8_oracle as oracle
from tests.test_layernorm_gpu import U, TYPES, inputs
from tests.test_rows8_gpu import assert_product, assert_wgrad, spread

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------------------------------------- layer norm kept in 8 bits


def check_kept(x, ln, dy, kind):
    """Gradients of every row and column, against the formula at the codes that the forward pass kept; each code is the nearest to a
    value within the forward's own error of xh."""
    from gaussianavatar_amd import fused
    x = x.detach().requires_grad_(True)
    M, C = x.shape
    y = fused.layernorm_act(x, ln, kind, checkpoint8=True)
    codes = y.grad_fn.saved_tensors[4][:, :C].view(torch.float8_e4m3fn).cpu().double()
    dx, dw, db = (t.double().cpu() for t in torch.autograd.grad(y, (x, ln.weight, ln.bias), dy))
    w, b = ln.weight.detach().double().cpu(), ln.bias.detach().double().cpu()
    g = dy.double().cpu()
    _, xh, rstd = oracle.layer_norm(x.detach().cpu(), w, b, ln.eps, kind)
    size = x.detach().double().cpu().abs().amax(1, keepdim=True) * rstd
    s = oracle.kept_scale(C)
    off = 64 * U * (xh.abs() + size) / s
    assert (codes >= oracle.grid(xh / s - off, "e4m3")).all() and (codes <= oracle.grid(xh / s + off, "e4m3")).all()
    xh = codes * s
    want = oracle.layer_norm_grads(xh, rstd, w, b, kind, g)
    gw = (g * w).abs().amax(1, keepdim=True) * (1 + xh.abs().amax(1, keepdim=True) ** 2) * (1 + w.abs().max())
    ph, deep = oracle.half_step(ln.weight.dtype), (M / 256 + 128) * U
    tols = (256 * U * rstd * gw * (1 + size) + oracle.half_step(x.dtype) * want[0].abs() + 1e-37,
            deep * (g * xh).abs().sum(0) + 2.0 ** -21 * (g * xh).abs().sum(0) + ph * want[1].abs() + 1e-37,
            deep * g.abs().sum(0) + 2.0 ** -21 * g.abs().sum(0) + ph * want[2].abs() + 1e-37)
    for got, o, tol in zip((dx, dw, db), want, tols):
        assert got.isfinite().all() and ((got - o).abs() <= tol).all(), float(((got - o).abs() / tol).max())


@pytest.mark.parametrize("kind", ["identity", "softplus", "relu"])
@pytest.mark.parametrize("C,dtype", [(8193, torch.float32), (10001, torch.float32), (16385, torch.bfloat16), (17001, torch.float16), (130, torch.float32),
                                     (1030, torch.bfloat16), (4099, torch.float16)])
def test_kept_rows_that_end_inside_a_vector_far_from_zero(C, dtype, kind):
    """Rows whose mean is hundreds of deviations: what lies past a row's end in its last vector must not reach the row's sums."""
    _, ln, dy = inputs(5, C, dtype, torch.float32, C)
    gen = torch.Generator().manual_seed(C)
    # 300 with one element in twenty at 302 (a step of bf16 there): a deviation of 0.44; fp32 rows: 300 +- 0.3
    x = 300.0 + (0.3 * torch.randn(5, C, generator=gen) if dtype == torch.float32 else 2.0 * (torch.rand(5, C, generator=gen) < 0.05))
    x[1] -= 600.0
    check_kept(x.to(dtype).cuda(), ln, dy, kind)


KEPT_WIDTHS = [1, 5, 66, 128, 300, 771, 1030, 2047, 4096, 5000, 9000, 16384, 17000, 40000]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("C", KEPT_WIDTHS)
def test_kept_gradients_of_every_width(C, dtype):
    x, ln, dy = inputs(11, C, dtype, dtype, C)
    check_kept(x, ln, dy, "softplus" if C % 2 else "identity")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,C", [(1, 100), (4097, 100), (1500, 2048), (900, 4096), (20000, 128)])
def test_kept_gradients_of_many_rows(M, C, dtype):
    x, ln, dy = inputs(M, C, dtype, torch.float32, M)
    check_kept(x, ln, dy, "softplus")


# ---------------------------------------------------------------------------------------------- means


@pytest.mark.parametrize("C", [3, 100, 300, 771, 4096, 12000])
@pytest.mark.parametrize("value", [12345.678, -0.1, 1.0e6])
def test_rows_of_equal_values_that_do_not_add_up_exactly(C, value):
    """No deviation: xh = 0. The first sum's mean is off by at most 64 u |x| (a tree of 40 additions, the rounded 1 / C); what is left after
    its residual is taken off is as much of that: 2 (64 u)^2 |x| rstd, rstd <= eps^-1/2 = 316. For dx, the mean that the backward
    pass reads is the fp32 number nearest to the value, the value itself: xh = 0 there."""
    from gaussianavatar_amd import fused
    ln = torch.nn.LayerNorm(C, device="cuda")
    x = torch.full((3, C), value, device="cuda", requires_grad=True)
    y = fused.layernorm_act(x, ln, "identity")
    assert float(y.detach().abs().max()) <= 2 * (64 * U) ** 2 * abs(value) * 317
    dy = torch.randn(3, C, generator=torch.Generator().manual_seed(C)).cuda()
    dx, dw = torch.autograd.grad(y, (x, ln.weight), dy)
    assert not dw.any()
    g = dy.double().cpu()
    want = (g - g.mean(1, keepdim=True)) / ln.eps ** 0.5
    assert ((dx.double().cpu() - want).abs() <= 256 * U * g.abs().max() / ln.eps ** 0.5).all()


@pytest.mark.parametrize("C,dtype", [(77, torch.float32), (1000, torch.float32), (5000, torch.float32), (20000, torch.float32), (300, torch.bfloat16),
                                     (300, torch.float16)])
def test_the_forward_of_rows_far_from_zero(C, dtype):
    """The residual of the mean is taken off: what is left of the mean's error is that of the sum of the deviations, 64 u of their mean size (one, in
    units of the deviation at most), and as much of the first mean's own error, 64 u (64 u max|x|) rstd. y is rounded once more."""
    from gaussianavatar_amd import fused
    gen = torch.Generator().manual_seed(C)
    x = (3000.0 + torch.randn(9, C, generator=gen) * (1.0 if dtype == torch.float32 else 40.0)).to(dtype).cuda()
    ln = torch.nn.LayerNorm(C, device="cuda")
    with torch.no_grad():
        y = fused.layernorm_act(x, ln, "identity").double().cpu()
    want, xh, rstd = oracle.layer_norm(x.cpu(), 1.0, 0.0, ln.eps, "identity")
    tol = 64 * U * (xh.abs() + 1 + 64 * U * x.double().cpu().abs().amax(1, keepdim=True) * rstd) + oracle.half_step(dtype) * want.abs()
    assert ((y - want).abs() <= tol).all(), float(((y - want).abs() / tol).max())


# ---------------------------------------------------------------------------------------------- softplus


def test_softplus_is_accurate_relative_to_itself():
    """w = 0 leaves act(b). fp32: exp with its argument's rounding taken back, a reciprocal, a polynomial, five operations more: sixteen
    roundings of half a step at most, 2^-20 of the value, everywhere above the smallest normal numbers."""
    from gaussianavatar_amd import fused
    b = torch.cat([torch.linspace(-86, 86, 6001), torch.linspace(-6, 6, 2191)])
    ln = torch.nn.LayerNorm(len(b), device="cuda")
    with torch.no_grad():
        ln.weight.zero_(), ln.bias.copy_(b)
        y = fused.layernorm_act(torch.randn(2, len(b), device="cuda"), ln, "softplus")[1].double().cpu()
    want = torch.log1p(torch.exp(b.double()))
    assert ((y - want).abs() <= 2.0 ** -20 * want).all(), float(((y - want).abs() / want).max() * 2 ** 20)


@pytest.mark.parametrize("dtype", TYPES)
def test_softplus_of_no_number_and_of_infinities(dtype):
    from gaussianavatar_amd import fused
    ln = torch.nn.LayerNorm(5, device="cuda", dtype=dtype)
    with torch.no_grad():
        ln.weight.zero_(), ln.bias.copy_(torch.tensor([float("nan"), float("inf"), -float("inf"), 0.0, -200.0]))
        y = fused.layernorm_act(torch.randn(2, 5, device="cuda").to(dtype), ln, "softplus")[0]
    assert torch.isnan(y[0]) and y[1] == float("inf") and y[2] == 0 and y[4] == 0


# ---------------------------------------------------------------------------------------------- types of gradients


@pytest.mark.parametrize("form", ["linear8", "checkpoint8"])
@pytest.mark.parametrize("wt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M", [40, 3000, 30000])
def test_a_bias_gradient_is_rounded_once_to_the_bias_own_type(M, wt, form):
    """A 16-bit weight and an fp32 bias: the sums of the columns in fp32, beyond the largest fp16 too."""
    from gaussianavatar_amd import fused, rows8
    x, w = spread(M, 64, wt, 1), spread(9, 64, wt, 2).requires_grad_(True)
    g = spread(M, 9, wt, 4)
    g[:, 3] = 300.0                                             # 3000 of them: past 65504
    for bt in (torch.float32, wt):
        b = torch.zeros(9, device="cuda", dtype=bt, requires_grad=True)
        if form == "linear8":
            y = rows8.linear8(x, w, b)
        elif bt == wt:
            y = fused.linear(x, w, b, checkpoint8=True)
        else:
            with torch.autocast("cuda", wt):
                y = fused.linear(x, w, b, checkpoint8=True)
        dw, db = torch.autograd.grad(y, (w, b), g)
        assert dw.dtype == wt and db.dtype == bt
        want, size = g.double().cpu().sum(0), g.double().cpu().abs().sum(0)
        if bt == torch.float16:
            want = torch.where(want.abs() < 65520, want, want.sign() * float("inf"))
        tol = (M + 600) * U * size + oracle.half_step(bt) * want.abs()
        fine = torch.isfinite(want)
        assert torch.equal(db.double().cpu()[~fine], want[~fine]) and ((db.double().cpu() - want).abs() <= tol)[fine].all()


# ---------------------------------------------------------------------------------------------- products


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,N,K", [(40, 130, 8200), (33, 20, 16500), (150, 70, 24577)])
def test_products_over_more_blocks_than_lds_holds_exponents_of(M, N, K, dtype):
    """Beyond 64 blocks of 128 the exponents are fetched again inside the loop. Every block has a size of its own."""
    from gaussianavatar_amd import rows8
    sizes = torch.exp2(torch.randint(-3, 4, (1, -(-K // 128)), generator=torch.Generator().manual_seed(K)).float()).repeat_interleave(128, 1)[:, :K].cuda()
    x, w = (spread(M, K, torch.float32, 1) * sizes).to(dtype), (spread(N, K, torch.float32, 2, K ** -0.5) / sizes.flip(1)).to(dtype)
    w8 = rows8.quantize8_weight(w)
    xo, wo = oracle.rows(x.cpu())[0], oracle.weight(w.cpu())[0]
    assert_product(rows8.linear8(x, w8), xo, wo, None, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,N", [(1, 20), (16, 20), (32, 20), (33, 20), (200, 150), (4096, 3000)])
def test_products_add_in_fp32_whatever_the_result_is(M, N, dtype):
    """256 * 256 + 1 * 4 - 256 * 256 in three products of one group: fp32 sums hold the 4."""
    from gaussianavatar_amd import rows8
    x, w = torch.zeros(M, 260, device="cuda", dtype=dtype), torch.zeros(N, 260, device="cuda", dtype=dtype)
    for at in (0, 132, 256):                                     # the last one in a block that is not full
        for p, (a, b) in enumerate(((256.0, 256.0), (1.0, 4.0), (256.0, -256.0))):
            x[:, at + p], w[:, at + p] = a, b
    w8 = rows8.quantize8_weight(w)
    assert (rows8.linear8(x, w8) == 12).all() and (rows8.matmul8(rows8.quantize8(x), w8, None, dtype) == 12).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,N,K", [(1, 300, 4096), (20, 250, 384), (45, 231, 1000), (130, 128, 66), (200, 500, 2110), (4100, 4090, 640)])
def test_products_are_fp32_sums_rounded_once(M, N, K, dtype):
    """In every form, forward and for the input gradient: within K u sum|terms| and half a step of the result's type."""
    from gaussianavatar_amd import rows8
    x, w, b = spread(M, K, dtype, 1), spread(N, K, dtype, 2, K ** -0.5), spread(1, N, torch.float32, 3)[0]
    at = torch.arange(M) if M < 1000 else torch.cat([torch.arange(0, M, 97), torch.arange(M - 40, M)])
    xo, wo = oracle.rows(x.cpu()[at])[0], oracle.weight(w.cpu())[0]

    def check(y, p, q, bias):
        want, size = p @ q.t(), p.abs() @ q.abs().t()
        if bias is not None:
            want, size = want + bias, size + bias.abs()
        tol = (p.shape[1] + 2) * U * size + oracle.half_step(dtype) * want.abs() + torch.finfo(dtype).smallest_normal * 2.0 ** -8
        off = (y[at.cuda()].double().cpu() - want).abs()
        assert (off <= tol).all(), float((off / tol).max())

    check(rows8.linear8(x, rows8.quantize8_weight(w), b), xo, wo, b.double().cpu())
    x.requires_grad_(True)
    y, g = rows8.linear8(x, w, b), spread(M, N, dtype, 4)
    check(y.detach(), xo, wo, b.double().cpu())
    check(torch.autograd.grad(y, x, g)[0], oracle.rows(g.cpu()[at])[0], wo.t().contiguous(), None)


@pytest.mark.parametrize("M,N,K", [(40, 300, 1000), (64, 128, 4096), (4100, 4096, 640)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_what_the_8_bit_instructions_lose_of_a_sum(M, N, K, dtype):
    """fast=True. Equal rows, and minus the exact result as an fp32 bias, with which the sums start: what is left is the sums' own error. In a group of
    eight adjacent k a product that is no multiple of 2^-13 of the largest one's power of two loses less than one such unit, and no
    other product loses anything; fp32 sums of K terms and the bias' rounding come on top."""
    from gaussianavatar_amd import rows8
    row, w = spread(1, K, dtype, 1), spread(N, K, dtype, 2, K ** -0.5)
    p = oracle.rows(row.cpu())[0] * oracle.weight(w.cpu())[0]                        # the products, [N, K]
    exact = p.sum(1)
    groups = torch.nn.functional.pad(p, (0, -K % 8)).unflatten(1, (-1, 8))
    most = groups.abs().amax(2, keepdim=True)
    unit = torch.where(most > 0, oracle._two_to((torch.frexp(most).exponent - 14).clamp_min(-900)), torch.ones_like(most))
    tol = (unit * (torch.remainder(groups, unit) != 0)).sum((1, 2)) + (K + 2) * U * (p.abs().sum(1) + exact.abs())
    tol = tol + oracle.half_step(dtype) * tol
    y = rows8.linear8(row.expand(M, K).contiguous(), rows8.quantize8_weight(w), (-exact).float().cuda(), fast=True).double().cpu()
    assert torch.equal(y, y[:1].expand(M, N))
    assert (y[0].abs() <= tol + torch.finfo(dtype).smallest_normal).all(), float((y[0].abs() / tol).max())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,N,K", [(5, 40, 300), (70, 130, 300), (4100, 4096, 640)])
def test_fast_products_and_their_gradients(M, N, K, dtype):
    """What fast allows for y and dx (assert_product's bound), and nothing else: dW, db, fp32 results and few rows have the same bits."""
    from gaussianavatar_amd import rows8
    x, w, b = (t.requires_grad_(True) for t in (spread(M, K, dtype, 1), spread(N, K, dtype, 2, K ** -0.5), spread(1, N, dtype, 3)[0]))
    g = spread(M, N, dtype, 4)
    y, full = rows8.linear8(x, w, b, fast=True), rows8.linear8(x, w, b)
    grads, want = torch.autograd.grad(y, (x, w, b), g), torch.autograd.grad(full, (x, w, b), g)
    assert torch.equal(grads[1], want[1]) and torch.equal(grads[2], want[2])
    if M <= 32 or dtype == torch.float32:
        assert torch.equal(y, full) and torch.equal(grads[0], want[0])
    at = torch.arange(M) if M < 1000 else torch.cat([torch.arange(0, M, 97), torch.arange(M - 40, M)])
    xo, wo = oracle.rows(x.detach().cpu()[at])[0], oracle.weight(w.detach().cpu())[0]
    assert_product(y.detach()[at.cuda()], xo, wo, b.detach().double().cpu(), dtype)
    assert_product(grads[0][at.cuda()], oracle.rows(g.cpu()[at])[0], wo.t().contiguous(), None, dtype)
    w8 = rows8.quantize8_weight(w)
    with torch.no_grad():
        assert torch.equal(rows8.linear8(x, w8, b, fast=True), y) and torch.equal(rows8.matmul8(rows8.quantize8(x), w8, b, dtype, fast=True), y)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("M", [5, 40])
def test_the_types_largest_numbers_stay_finite_beside_zeros(M, dtype):
    """A masked place that holds the type's lowest value: its code stands for -2^128, past bf16's range. Times zero it is zero, in
    products and weight gradients, and times a small number it is finite."""
    from gaussianavatar_amd import rows8
    x, w = torch.ones(M, 200, device="cuda", dtype=dtype), torch.zeros(3, 200, device="cuda", dtype=dtype)
    x[2, 7] = torch.finfo(dtype).min
    x[2, 8:128] = 0
    w[1, 1], w[2, 7] = 2.0, 2.0 ** -10
    y = rows8.linear8(x, rows8.quantize8_weight(w), torch.ones(3, device="cuda"))
    assert (y[:, 0] == 1).all() and y[2, 2].double() == -2.0 ** 118 and y[1, 1] == 3
    g = torch.ones(M, 4, device="cuda", dtype=dtype)
    g[2] = 0
    g[2, 1] = 2.0 ** -12
    dW, db = rows8.wgrad8(g, rows8.quantize8(x), torch.float32)
    assert dW.isfinite().all() and dW[0, 7] == M - 1 and dW[1, 7].double() == -2.0 ** 116 and db[0] == M - 1


@pytest.mark.parametrize("M", [5, 40])
def test_the_smallest_numbers_count_beside_large_ones(M):
    """Blocks whose exponent is the least one, -126, times large numbers, in products and weight gradients."""
    from gaussianavatar_amd import rows8
    x, w = torch.zeros(M, 200, device="cuda"), torch.zeros(3, 200, device="cuda")
    x[:, 5], x[:, 130], x[3, 131] = 2.0 ** -120, 2.0 ** -126, 2.0 ** -129
    w[0, 5], w[1, 130], w[2, 131] = 2.0 ** 110, 2.0 ** 111, 2.0 ** 111
    r, w8 = rows8.quantize8(x), rows8.quantize8_weight(w)
    assert (r.exps[:, :2] == 1).all()
    y = rows8.matmul8(r, w8)
    want = (x.double() @ w.double().t())
    assert want[0, 0] == 2.0 ** -10 and torch.equal(y.double(), want)
    g = torch.full((M, 2), 2.0 ** 100, device="cuda")
    dW, _ = rows8.wgrad8(g, r)
    want = g.double().t() @ x.double()
    assert torch.equal(dW.double(), want) and want[0, 131] == 2.0 ** -29


def test_the_transposed_side_of_the_largest_numbers():
    """The same in an input gradient: dx = Q(g) Q(W)."""
    from gaussianavatar_amd import rows8
    for M in (5, 40):
        x, w = torch.zeros(M, 150, device="cuda").requires_grad_(True), torch.ones(20, 150, device="cuda")
        g = torch.zeros(M, 20, device="cuda")
        g[1, 3] = torch.finfo(torch.float32).max
        w[3, 4:] = 0
        w[3, 2] = 2.0 ** -10
        dx = torch.autograd.grad(rows8.linear8(x, w), x, g)[0]
        assert dx[1, 2].double() == 2.0 ** 118 and not dx[1, 4:].any() and not dx[0].any() and not dx[2:].any()


# ---------------------------------------------------------------------------------------------- refusals


def test_what_the_backward_pass_cannot_do_is_refused_forward():
    from gaussianavatar_amd import fused, rows8
    K = 1 << 22
    x, w = torch.ones(1, K, device="cuda", dtype=torch.bfloat16), torch.ones(1, K, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    for call in (lambda: rows8.linear8(x, w), lambda: fused.linear(x, w, None, checkpoint8=True)):
        with pytest.raises(ValueError, match="columns"):
            call()
        with torch.no_grad():
            assert float(call()) == K
    assert float(rows8.linear8(x, w.detach())) == K
