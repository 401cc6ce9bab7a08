"""Layer norm + activation on the GPU, forward and backward, against 64-bit arithmetic (tests/rows8_oracle.py).

Tolerances, u = 2^-24. A row's mean and variance are trees of at most 40 additions: xh is off by at most 64 u (|xh| + max|x| rstd) (the
second term: the mean's error, in units of the deviation). y = act(w xh + b): |act'| <= 1, and the activation's own functions give
2^-21 of 1 + |u|. dx: three terms of the size rstd max|g w| (1 + max|xh|^2), each from sums of 40 additions and from xh: 256 u of that times
(1 + max|x| rstd). dw, db: sums over M rows, at most M / 256 + 64 additions deep plus the error of xh. Rounding adds half a step."""
import pytest
import torch

from tests import rows8_oracle as oracle

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def inputs(M, C, dtype, ptype, seed, offset=0.0):
    gen = torch.Generator().manual_seed(seed)
    x = (torch.randn(M, C, generator=gen) * torch.exp(0.5 * torch.randn(1, C, generator=gen)) + offset).to(dtype).cuda()
    ln = torch.nn.LayerNorm(C, device="cuda", dtype=ptype)
    with torch.no_grad():
        ln.weight.copy_(torch.rand(C, generator=gen) + 0.5), ln.bias.copy_(torch.randn(C, generator=gen))
    return x, ln, torch.randn(M, C, generator=gen).to(dtype).cuda()


def check(x, ln, dy, kind, kept8=False):
    from gaussianavatar_amd import fused
    x = x.detach().requires_grad_(True)
    M, C = x.reshape(-1, x.shape[-1]).shape
    y = fused.layernorm_act(x, ln, kind, checkpoint8=kept8)
    params = [p for p in (ln.weight, ln.bias) if p is not None]
    got = torch.autograd.grad(y, (x, *params), dy)
    assert y.shape == x.shape and y.dtype == x.dtype and got[0].shape == x.shape
    one = torch.ones(C, dtype=torch.float64)
    w = one if ln.weight is None else ln.weight.detach().double().cpu()
    b = 0 * one if ln.bias is None else ln.bias.detach().double().cpu()
    xc, g = x.detach().cpu().reshape(M, C).double(), dy.cpu().reshape(M, C).double()
    want, xh, rstd = oracle.layer_norm(xc, w, b, ln.eps, kind)
    if M == 0:
        assert all(not t.any() for t in got[1:])
        return
    size = xc.abs().amax(1, keepdim=True) * rstd                                 # max|x| rstd
    u = xh * w + b
    half = oracle.half_step(x.dtype)
    tol = 64 * U * w.abs() * (xh.abs() + size) + 2.0 ** -21 * (1 + u.abs()) + half * want.abs() + 1e-37
    off = (y.detach().double().cpu().reshape(M, C) - want).abs()
    assert (off <= tol).all(), float((off / tol).max())
    sure_rows, sure_cols, dxh = slice(None), slice(None), 64 * U * (xh.abs() + size)
    if kept8:
        s = oracle.kept_scale(C)
        near = oracle.near_a_border(xh / s, "e4m3", 1e-4)                          # such codes may go either way: leave their rows and columns out
        sure_rows, sure_cols = ~near.any(1), ~near.any(0)
        xh = oracle.grid(xh / s, "e4m3") * s
        dxh = 0 * dxh
    dx, dw, db = oracle.layer_norm_grads(xh, rstd, w, b, kind, g)
    gw = (g * w).abs().amax(1, keepdim=True) * (1 + xh.abs().amax(1, keepdim=True) ** 2) * (1 + w.abs().max())
    tol = 256 * U * rstd * gw * (1 + size) + half * dx.abs() + 1e-37
    off = (got[0].double().cpu().reshape(M, C) - dx).abs()
    assert (off <= tol)[sure_rows].all(), float((off / tol)[sure_rows].max())
    if ln.weight is None:
        return
    deep = (M / 256 + 128) * U
    ph = oracle.half_step(ln.weight.dtype)
    # (softplus' is taken at u: it moves with xh's error too, by at most a quarter of it times |w|)
    tol = (deep * (g.abs() * xh.abs()).sum(0) + (g.abs() * dxh * (1 + w.abs() * xh.abs())).sum(0) + 2.0 ** -21 * (g * xh).abs().sum(0)
           + ph * dw.abs() + 1e-37)
    off = (got[1].double().cpu() - dw).abs()
    assert (off <= tol)[sure_cols].all(), float((off / tol)[sure_cols].max())
    if ln.bias is not None:
        tol = deep * g.abs().sum(0) + (g.abs() * dxh * w.abs()).sum(0) + 2.0 ** -21 * g.abs().sum(0) + ph * db.abs() + 1e-37
        off = (got[2].double().cpu() - db).abs()
        assert (off <= tol)[sure_cols].all(), float((off / tol)[sure_cols].max())


# one vector, odd tails, every lane-group width, four vectors a lane, a workgroup a row (three widths), beyond
WIDTHS = [1, 2, 3, 7, 8, 9, 31, 66, 128, 200, 513, 771, 1024, 1500, 2048, 2500, 4096, 5000, 8192, 10001, 16384, 40000]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("C", WIDTHS)
def test_widths(C, dtype):
    x, ln, dy = inputs(13, C, dtype, dtype, C)
    check(x, ln, dy, "softplus" if C % 2 else "identity")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("C", [1, 5, 66, 128, 300, 1030, 4096, 9000, 17000, 40000])
def test_widths_kept_in_8_bits(C, dtype):
    x, ln, dy = inputs(11, C, dtype, dtype, C)
    check(x, ln, dy, "softplus", kept8=True)


@pytest.mark.parametrize("kind", ["identity", "softplus", "relu"])
@pytest.mark.parametrize("M", [0, 1, 2, 255, 4097])
def test_rows_and_activations(M, kind):
    x, ln, dy = inputs(M, 100, torch.float32, torch.float32, M)
    check(x, ln, dy, kind)
    check(x, ln, dy, kind, kept8=True)


@pytest.mark.parametrize("dtype,ptype", [(torch.bfloat16, torch.float32), (torch.float16, torch.float32), (torch.float32, torch.bfloat16)])
def test_parameters_of_another_type(dtype, ptype):
    x, ln, dy = inputs(300, 129, dtype, ptype, 1)
    check(x, ln, dy, "softplus")


def test_a_mean_far_from_zero():
    x, ln, dy = inputs(64, 256, torch.float32, torch.float32, 1, offset=3000.0)
    check(x, ln, dy, "identity")


def test_without_parameters():
    from gaussianavatar_amd import fused
    for affine, bias in ((False, False), (True, False)):
        x, _, dy = inputs(40, 96, torch.float32, torch.float32, 2)
        ln = torch.nn.LayerNorm(96, elementwise_affine=affine, bias=bias, device="cuda")
        check(x, ln, dy, "softplus")
        with torch.no_grad():
            assert torch.equal(fused.layernorm_act(x, ln, "softplus"), fused.layernorm_act(x.clone().requires_grad_(True), ln, "softplus"))


def test_strided_shaped_and_unaligned_rows():
    base, _, _ = inputs(60, 700, torch.bfloat16, torch.bfloat16, 3)
    for x in (base[:, 1:400], base[::2, 3:99], base.t()[:50], base[7].expand(5, 700), base.view(3, 20, 700), base[4], base[:, 5:6]):
        _, ln, _ = inputs(1, x.shape[-1], torch.bfloat16, torch.bfloat16, 4)
        dy = torch.randn(x.shape, device="cuda").to(x.dtype)
        check(x, ln, dy, "identity")
        check(x, ln, dy.mT.contiguous().mT if dy.dim() > 1 else dy, "softplus")
        check(x, ln, torch.ones((), device="cuda", dtype=x.dtype).expand(x.shape), "softplus")


def test_rows_of_equal_values_and_of_no_number():
    """No deviation: xh = 0, rstd = eps^-1/2. A NaN or an infinity makes its own row NaN and no other."""
    from gaussianavatar_amd import fused
    x, ln, dy = inputs(8, 200, torch.float32, torch.float32, 5)
    x[2] = 7.0
    check(x, ln, dy, "softplus")
    x[4, 3], x[6, 0] = float("nan"), float("inf")
    for C in (200,):
        y = fused.layernorm_act(x, ln, "softplus")
        rows = torch.isnan(y).all(1)
        assert rows[4] and rows[6] and int(torch.isnan(y).any(1).sum()) == 2


def test_softplus_far_on_both_sides():
    """w = 0 leaves act(b): every size of argument, against the function in 64 bits: 2^-20 of the value."""
    from gaussianavatar_amd import fused
    ln = torch.nn.LayerNorm(512, device="cuda")
    with torch.no_grad():
        ln.weight.zero_(), ln.bias.copy_(torch.linspace(-80, 80, 512))
        y = fused.layernorm_act(torch.randn(3, 512, device="cuda"), ln, "softplus")[1].double().cpu()
    b = ln.bias.detach().double().cpu()
    want = torch.where(b < -30, torch.exp(b), torch.log1p(torch.exp(b)))
    assert ((y - want).abs() <= 2.0 ** -16 * want).all()       # exp of a number up to 80 in fp32: 80 * 2^-24 of the value, and log1p's


def test_gradients_equal_differences():
    """The loss along a direction, central differences in 64 bits of the oracle and of the kernel's own forward: step h = 2^-7, whose
    own error is of the order h^2, and the forward's rounding over h: 2^-24 / 2^-7 of the summed sizes."""
    from gaussianavatar_amd import fused
    x, ln, dy = inputs(32, 64, torch.float32, torch.float32, 6)
    x.requires_grad_(True)
    loss = lambda x: float((fused.layernorm_act(x, ln, "softplus").double() * dy.double()).sum())
    (dx,) = torch.autograd.grad(fused.layernorm_act(x, ln, "softplus"), x, dy)
    v = torch.randn_like(x)
    h = 2.0 ** -7
    with torch.no_grad():
        diff = (loss(x + h * v) - loss(x - h * v)) / (2 * h)
    size = float((dx.abs() * v.abs()).sum())
    assert abs(diff - float((dx.double() * v.double()).sum())) <= (4 * h * h + 64 * U / h) * max(size, float(dy.abs().sum()))


def test_the_same_inputs_give_the_same_bits_and_a_padded_batch_does_not_matter():
    from gaussianavatar_amd import fused
    x, ln, dy = inputs(5000, 300, torch.bfloat16, torch.bfloat16, 7)
    x.requires_grad_(True)
    run = lambda: torch.autograd.grad(fused.layernorm_act(x, ln, "softplus"), (x, ln.weight, ln.bias), dy)
    a, b = run(), run()
    assert all(torch.equal(s, t) for s, t in zip(a, b))
    with torch.no_grad():
        y, part = fused.layernorm_act(x, ln, "softplus"), fused.layernorm_act(x[:77], ln, "softplus")
    assert torch.equal(y[:77], part)


def test_what_the_kernels_do_not_take_runs_on_torch():
    from gaussianavatar_amd import fused
    x = torch.randn(5, 12, device="cuda", dtype=torch.float64)
    ln = torch.nn.LayerNorm(12, device="cuda", dtype=torch.float64)
    assert torch.equal(fused.layernorm_act(x, ln, "relu"), torch.relu(ln(x)))
    with pytest.raises(ValueError):
        fused.layernorm_act(x.cpu(), ln)
    with pytest.raises(TypeError):
        fused.layernorm_act(x, ln, checkpoint8=True)


def test_strided_parameters():
    from gaussianavatar_amd import fused
    x, ln, dy = inputs(50, 72, torch.float32, torch.float32, 7)
    want = fused.layernorm_act(x, ln, "softplus")
    grads = torch.autograd.grad(want, (ln.weight, ln.bias), dy)
    far = torch.nn.LayerNorm(72, device="cuda")
    base = torch.full((72, 2, 3), 9.0, device="cuda")
    base[:, 0, 0], base[:, 1, 2] = ln.weight.detach(), ln.bias.detach()
    far.weight, far.bias = torch.nn.Parameter(base[:, 0, 0]), torch.nn.Parameter(base[:, 1, 2])
    got = fused.layernorm_act(x, far, "softplus")
    assert torch.equal(got, want)
    with torch.no_grad():
        assert torch.equal(fused.layernorm_act(x, far, "softplus"), want)
    for a, b in zip(torch.autograd.grad(got, (far.weight, far.bias), dy), grads):
        assert torch.equal(a, b)


@pytest.mark.parametrize("kept8", [False, True])
def test_rows_behind_2_to_the_32_elements(kept8):
    """A row's results do not depend on where it lies."""
    from gaussianavatar_amd import fused
    M, C = 2 ** 22 + 3, 1030
    ln = torch.nn.LayerNorm(C, device="cuda")
    x = torch.empty(M, C, dtype=torch.bfloat16, device="cuda").normal_().requires_grad_(True)
    dy = torch.empty(M, C, dtype=torch.bfloat16, device="cuda").normal_()
    y = fused.layernorm_act(x, ln, "relu", checkpoint8=kept8)
    (dx,) = torch.autograd.grad(y, (x,), dy)
    for lo, hi in ((0, 300), (2 ** 21, 2 ** 21 + 300), (M - 300, M)):
        part = x.detach()[lo:hi].clone().requires_grad_(True)
        want = fused.layernorm_act(part, ln, "relu", checkpoint8=kept8)
        assert torch.equal(y[lo:hi], want)
        assert torch.equal(dx[lo:hi], torch.autograd.grad(want, (part,), dy[lo:hi])[0])


@pytest.mark.parametrize("kept8", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,C", [(1500, 2048), (900, 4096), (700, 1030), (5, 2047)])
def test_several_rows_to_a_workgroup(M, C, dtype, kept8):
    x, ln, dy = inputs(M, C, dtype, torch.float32, M)
    check(x, ln, dy, "softplus", kept8)
