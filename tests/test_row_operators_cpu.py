"""Layer norm, 8-bit rows and their products on the CPU where they can go wrong."""
import pytest
import torch

from gaussianavatar_amd import _native, fused, rows8


@pytest.mark.parametrize("kind", ["softplus", "identity", "relu"])
def test_one_row_without_leading_dimensions_kept_in_8_bits(kind):
    """x [C] gives what x [1, C] gives."""
    torch.manual_seed(0)
    x, dy, ln = torch.randn(50), torch.randn(50), torch.nn.LayerNorm(50)
    got = []
    for shape in ((50,), (1, 50)):
        t = x.reshape(shape).requires_grad_(True)
        y = fused.layernorm_act(t, ln, kind, checkpoint8=True)
        got.append([y] + list(torch.autograd.grad(y, (t, ln.weight, ln.bias), dy.reshape(shape))))
    for a, b in zip(*got):
        assert torch.equal(a.flatten(), b.flatten())
    assert got[0][2].shape == (50,)


@pytest.mark.parametrize("form", ["linear8", "checkpoint8"])
@pytest.mark.parametrize("wt", [torch.bfloat16, torch.float16])
def test_a_bias_gradient_is_rounded_once_to_the_bias_own_type(wt, form):
    """A 16-bit weight and an fp32 bias: the columns' sums in 64 bits, one rounding to fp32."""
    torch.manual_seed(1)
    x, w, b = torch.randn(3000, 64).to(wt), torch.randn(9, 64).to(wt).requires_grad_(True), torch.zeros(9, requires_grad=True)
    g = torch.randn(3000, 9).to(wt)
    g[:, 3] = 300.0                                             # past 65504
    if form == "linear8":
        y = rows8.linear8(x, w, b)
    else:
        with torch.autocast("cpu", wt):
            y = fused.linear(x, w, b, checkpoint8=True)
    dw, db = torch.autograd.grad(y, (w, b), g)
    assert dw.dtype == wt and torch.equal(db, g.double().sum(0).float())
    dW, db = rows8.wgrad8(g, rows8.quantize8(x), bias_dtype=torch.float32)
    assert dW.dtype == wt and torch.equal(db, g.double().sum(0).float())
    with pytest.raises(TypeError):
        rows8.wgrad8(g, rows8.quantize8(x), bias_dtype=torch.float64)


def test_the_bias_gradients_type_at_the_c_entry_points():
    """otype carries the type of dW and, where it is another, GANET_DB_TYPE (type + 1 in bits 8 ..) of db."""
    lib = _native.ganet()
    A = 1 << 20                                                    # an aligned address that nobody reads
    for otype in (3, 0x400, 0x501, 0x10001, -1):
        assert lib.ganet_wgrad8(4, 8, 8, 0, 0, A, 8, A, 16, A, 4, A, None, otype, None, 0, None) == 4
        assert b"ganet_wgrad8" in lib.ganet_last_error()


@pytest.mark.parametrize("value", [12345.678, -0.1, 1.0e6])
def test_rows_of_equal_values_kept_in_8_bits(value):
    """No deviation: xh = 0. The mean is off by at most 16 u |x| (pairwise sums), what is left of it by as much of that again, rstd <= 317."""
    for C in (3, 100, 771, 4096):
        ln, x = torch.nn.LayerNorm(C), torch.full((2, C), value, requires_grad=True)
        y = fused.layernorm_act(x, ln, "identity", checkpoint8=True)
        assert float(y.detach().abs().max()) <= 2 * (16 * 2.0 ** -24) ** 2 * abs(value) * 317


def test_the_types_largest_numbers_stay_finite_beside_zeros():
    """A value past fp32's range is the largest number in a product too: times zero it is zero."""
    x = torch.full((2, 4), torch.finfo(torch.float32).min)
    r = rows8.quantize8(x)
    y = rows8.matmul8(r, rows8.quantize8_weight(torch.tensor([[0.0, 0, 0, 0], [2.0 ** -10, 0, 0, 0]])))
    dW, _ = rows8.wgrad8(torch.zeros(2, 3), r)
    assert not y[:, 0].any() and torch.allclose(y[:, 1], torch.tensor(-2.0 ** 118), rtol=2 ** -22) and not dW.any()


def _net(norm, bits8=False):
    from gaussianavatar_amd.network import POP_no_unet
    torch.manual_seed(0)
    net = POP_no_unet(c_geom=64, hsize=32, decoder_norm=norm, decoder_bits8=bits8)
    u = (torch.arange(16) + 0.5) / 16
    return net, torch.randn(1, 64, 8, 8), torch.stack(torch.meshgrid(u, u, indexing="ij"), -1).reshape(1, 256, 2)


@pytest.mark.parametrize("bits8", [False, True])
def test_a_share_of_the_texels_through_the_layer_norm_decoder(bits8):
    """Shares of the rows, each by itself: the outputs are the whole's, and the gradients add up to the whole's. Sums over the rows are in
    another order: 16 * 2^-24 of the largest, through the layers; a code next to a border may go the other way for it."""
    net, geom, uv = _net("layer", bits8)
    geom.requires_grad_(True)
    params = [geom] + list(net.parameters())
    weights = torch.randn(256, 7)

    def run(r0, r1, rows):
        y = torch.cat(net.forward_points(None, geom, uv, raw_heads=True, rows=rows, m_global=256), 2)[0]
        assert y.shape == (r1 - r0, 7)
        return y, torch.autograd.grad((y * weights[r0:r1]).sum(), params)

    whole, want = run(0, 256, None)
    got = [run(a, b, (a, b)) for a, b in ((0, 100), (100, 101), (101, 256))]
    assert torch.allclose(torch.cat([y for y, _ in got]), whole, rtol=0, atol=2.0 ** -16 * float(whole.detach().abs().max()))
    for i, w in enumerate(want):
        assert float((sum(g[i] for _, g in got) - w).norm()) <= (2.0 ** -6 if bits8 else 2.0 ** -16) * float(w.norm()) + 1e-6


def test_a_share_of_the_texels_through_a_batch_norm_decoder_that_does_not_run_fused_is_refused():
    net, geom, uv = _net("batch")
    with pytest.raises(NotImplementedError):
        net.forward_points(None, geom, uv, rows=(0, 100), m_global=256)


def test_fast_sums_at_the_entry_points():
    """GANET_FAST (0x100) beside a type: workspaces are the type's, an unknown type is refused all the same; the CPU's sums are what they are."""
    lib = _native.ganet()
    A = 1 << 20                                                    # an aligned address that nobody reads
    for ytype in (0x103, 0x201, -1, 3):
        assert lib.ganet_gemm8(4, 8, 8, 0, A, 16, A, 4, A, 16, A, 4, None, 0, A, 8, ytype, None) == 4
        assert lib.ganet_linear8_held(4, 8, 8, ytype, A, 8, A, 16, A, 4, None, 0, A, None, 0, None) == 4
    for M, N, K in ((1, 64, 64), (1, 4096, 8192), (40, 100, 300)):
        for t in range(3):
            assert lib.ganet_linear8_held_workspace(M, N, K, t | 0x100) == lib.ganet_linear8_held_workspace(M, N, K, t)
            assert lib.ganet_linear8_bwd_workspace(M, N, K, t | 0x100) == lib.ganet_linear8_bwd_workspace(M, N, K, t)
    torch.manual_seed(0)
    x, w = torch.randn(40, 70, requires_grad=True), torch.randn(9, 70, requires_grad=True)
    got, want = rows8.linear8(x, w, fast=True), rows8.linear8(x, w)
    assert torch.equal(got, want)
    for a, b in zip(torch.autograd.grad(got.sum(), (x, w)), torch.autograd.grad(want.sum(), (x, w))):
        assert torch.equal(a, b)
