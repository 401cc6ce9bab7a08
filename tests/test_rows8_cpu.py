"""8-bit rows, weights, products and layer norm on the CPU: the definitions against 64-bit arithmetic, and what is refused."""
import pytest
import torch

from gaussianavatar_amd import _native, fused, rows8
from gaussianavatar_amd.network import ShapeDecoder
from tests import rows8_oracle as oracle


def special_rows(fmt):
    most = oracle.FORMATS[fmt][0]
    x = torch.zeros(9, 130)
    x[1] = 1.0
    x[2, :3] = torch.tensor([float("nan"), float("inf"), 3.0])
    x[3, 128:] = torch.tensor([-1e-40, 2e-38])
    x[4] = torch.linspace(-most, most, 130)                     # the block's largest is the format's: e = 0
    x[5] = x[4] * (1 + 2 ** -7)                                 # just above: e = 1
    x[6, 5], x[6, 129] = -3.0e38, 1e30
    x[7] = 0.8125 * 2.0 ** torch.arange(130).sub(65)            # every size, ties among them
    x[8] = torch.tensor([1.0, -1.0]).repeat(65) * 1.1875
    return x


@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
def test_rows_follow_their_definition(fmt):
    torch.manual_seed(0)
    for x in (special_rows(fmt), torch.randn(40, 300) * torch.exp(4 * torch.randn(40, 1)), torch.randn(3, 1), torch.randn(0, 17)):
        r = rows8.quantize8(x, fmt)
        v, e = oracle.rows(x, fmt)
        assert torch.equal(r.exps[:, :e.shape[1]].long() - 127, e)
        got = r.codes[:, :x.shape[1]].double() * oracle._two_to(e).repeat_interleave(128, 1)[:, :x.shape[1]]
        assert torch.equal(torch.isnan(got), torch.isnan(v)) and torch.equal(got[~torch.isnan(v)], v[~torch.isnan(v)])
        assert r.codes.shape[1] % 16 == 0 and not r.codes[:, x.shape[1]:].float().any()


def test_values_beyond_the_type_become_its_largest():
    x = torch.tensor([[65504.0, 1.0, -65504.0, float("nan")]])
    v = rows8.quantize8(x).dequantize(torch.float16)            # 65504 is nearer to 65536 than to the value below
    assert v[0, 0] == 65504 and v[0, 2] == -65504 and torch.isnan(v[0, 3]) and rows8.quantize8(x).dequantize()[0, 0] == 65536


def test_weight_and_its_transpose_hold_the_same_values():
    torch.manual_seed(1)
    w = torch.randn(200, 150) * torch.exp(2 * torch.randn(200, 1))
    w8 = rows8.quantize8_weight(w, transposed=True)
    v, _ = oracle.weight(w)
    assert torch.equal(w8.dequantize().double(), v) and torch.equal(w8.transposed().dequantize().double(), v.t())
    with pytest.raises(ValueError, match="transposed"):
        rows8.quantize8_weight(w).transposed()


def test_linear8_and_its_gradients_are_exact_on_numbers_that_the_format_holds():
    """Small whole numbers are their own codes: the layer is then linear in each argument, and the gradients can be had exactly from
    differences of the loss."""
    torch.manual_seed(2)
    ints = lambda *s: torch.randint(-3, 4, s).float()
    x, w, b, g = ints(6, 140), ints(9, 140), ints(9), ints(6, 9)
    for t in (x, w, b):
        t.requires_grad_(True)
    loss = lambda x, w, b: (rows8.linear8(x, w, b).double() * g).sum()
    gx, gw, gb = torch.autograd.grad(loss(x, w, b), (x, w, b))
    for k, t in enumerate((x, w, b)):
        d = torch.randint(-1, 2, t.shape).float()
        args = [a.detach() for a in (x, w, b)]
        up, down = list(args), list(args)
        up[k], down[k] = args[k] + d, args[k] - d
        diff = (loss(*up) - loss(*down)) / 2
        assert float(diff) == float(((gx, gw, gb)[k].double() * d).sum())


def test_kept8_layer_norm_gradients():
    torch.manual_seed(3)
    x, ln = torch.randn(20, 50, requires_grad=True), torch.nn.LayerNorm(50)
    with torch.no_grad():
        ln.weight.uniform_(0.5, 1.5), ln.bias.uniform_(-1, 1)
    dy = torch.randn(20, 50)
    for kind in ("softplus", "identity", "relu"):
        y = fused.layernorm_act(x, ln, kind, checkpoint8=True)
        got = torch.autograd.grad(y, (x, ln.weight, ln.bias), dy)
        w, b = ln.weight.detach().double(), ln.bias.detach().double()
        yo, xh, rstd = oracle.layer_norm(x.detach(), w, b, ln.eps, kind)
        s = oracle.kept_scale(50)
        assert not oracle.near_a_border(xh / s, "e4m3", 1e-5).any()
        want = oracle.layer_norm_grads(oracle.grid(xh / s, "e4m3") * s, rstd, w, b, kind, dy)
        # fp32 arithmetic on a few dozen terms: 128 roundings of the largest term in sight
        assert (y.double() - yo).abs().max() <= 128 * 2 ** -24 * 8
        for a, o in zip(got, want):
            assert (a.double() - o).abs().max() <= 128 * 2 ** -24 * 20 * 8
    assert _native.ganet().ganet_ln_code_exponent(50) == -5        # sqrt(50) = 7.07 <= 448 / 32 = 14; / 64 = 7 is too small


def test_decoder_with_layer_norm_and_8_bits():
    """The options change no default: parameters of the batch decoder stay what they are, and the 8-bit layer-norm decoder stays near the
    fp32 one."""
    torch.manual_seed(4)
    names = set(ShapeDecoder(66, 32).state_dict())
    assert "bn1.running_mean" in names and not any(n.startswith("ln") for n in names)
    plain, small = ShapeDecoder(66, 32, norm="layer"), ShapeDecoder(66, 32, norm="layer", bits8=True)
    small.load_state_dict(plain.state_dict())
    x = torch.randn(64, 66)
    outs = [d.forward_points(x, raw_heads=True, m_global=128) for d in (plain, small)]        # rows are independent: no exchange
    for a, b in zip(*outs):
        assert a.shape == b.shape and (a - b).abs().max() < 0.5 * a.detach().abs().max()
    with pytest.raises(ValueError, match="norm"):
        ShapeDecoder(66, 32, norm="group")


def test_refusals_of_the_python_entry_points():
    x, w = torch.randn(4, 64), torch.randn(8, 64)
    for call, error in ((lambda: rows8.quantize8(x, "e3m4"), ValueError), (lambda: rows8.quantize8(x.double()), TypeError),
                        (lambda: rows8.quantize8(torch.randn(3, 0)), ValueError), (lambda: rows8.quantize8(torch.tensor(1.0)), ValueError),
                        (lambda: rows8.quantize8_weight(w[0]), ValueError), (lambda: rows8.quantize8_weight(w.long()), TypeError),
                        (lambda: rows8.linear8(x, w[:, :5]), ValueError), (lambda: rows8.linear8(x, w, torch.zeros(7)), ValueError),
                        (lambda: rows8.linear8(x.double(), w), TypeError), (lambda: rows8.linear8(x, w.double()), TypeError),
                        (lambda: rows8.linear8(x, w, torch.zeros(8).double()), TypeError),
                        (lambda: rows8.linear8(torch.randn(4, 63), rows8.quantize8_weight(w)), ValueError),
                        (lambda: rows8.linear8(x.requires_grad_(True), rows8.quantize8_weight(w)), RuntimeError),
                        (lambda: rows8.matmul8(rows8.quantize8(torch.randn(2, 60)), rows8.quantize8_weight(w)), ValueError),
                        (lambda: rows8.matmul8(rows8.quantize8(x), rows8.quantize8_weight(w), dtype=torch.float64), TypeError),
                        (lambda: rows8.matmul8(rows8.quantize8(x), rows8.quantize8_weight(w), torch.zeros(3)), ValueError),
                        (lambda: rows8.wgrad8(torch.randn(5, 8), rows8.quantize8(x)), ValueError),
                        (lambda: rows8.wgrad8(torch.randn(4, 8).double(), rows8.quantize8(x)), TypeError),
                        (lambda: rows8.quantize8(x).dequantize(torch.float64), TypeError),
                        (lambda: fused.layernorm_act(x, torch.nn.LayerNorm(63)), ValueError),
                        (lambda: fused.layernorm_act(x, torch.nn.LayerNorm(64), "gelu"), ValueError),
                        (lambda: fused.layernorm_act(x, torch.nn.LayerNorm((4, 64))), ValueError),
                        (lambda: fused.layernorm_act(x.double(), torch.nn.LayerNorm(64).double(), checkpoint8=True), TypeError)):
        with pytest.raises(error):
            call()


def test_refusals_of_held_codes():
    codes, exps = torch.zeros(8, 64, dtype=torch.float8_e4m3fn), torch.full((1, 4), 127, dtype=torch.uint8)
    rows8.Weight8(codes, exps, 64)
    for args in ((codes, exps, 65), (codes, exps, 0), (codes[:, :40], exps, 40), (codes, exps[:, :3], 64), (codes.view(torch.uint8), exps, 64),
                 (codes.view(torch.float8_e5m2), exps, 64), (codes, exps.int(), 64), (codes[::2], exps, 64),
                 (torch.zeros(200, 64, dtype=torch.float8_e4m3fn), exps, 64), (codes, exps, 64, codes, exps)):
        with pytest.raises((TypeError, ValueError)):
            rows8.Weight8(*args)
    with pytest.raises(ValueError):
        rows8.Rows8(codes, exps, 64)                               # one row of exponents for eight of codes


def test_refusals_of_the_c_entry_points():
    """Error code and text, nothing launched (no GPU needed)."""
    lib = _native.ganet()
    A = 1 << 20                                                    # an aligned address that nobody reads
    cases = [
        (lib.ganet_rows8_pack(-1, 8, 0, 0, A, 8, A, 16, A, 4, None), 4, b"ganet_rows8_pack"),
        (lib.ganet_rows8_pack(4, 0, 0, 0, A, 8, A, 16, A, 4, None), 4, b"ganet_rows8_pack"),
        (lib.ganet_rows8_pack(4, 8, 3, 0, A, 8, A, 16, A, 4, None), 4, b"ganet_rows8_pack"),
        (lib.ganet_rows8_pack(4, 8, 0, 2, A, 8, A, 16, A, 4, None), 4, b"ganet_rows8_pack"),
        (lib.ganet_rows8_pack(4, 8, 0, 0, None, 8, A, 16, A, 4, None), 1, b"ganet_rows8_pack"),
        (lib.ganet_rows8_pack(4, 8, 0, 0, A, 7, A, 16, A, 4, None), 1, b"ganet_rows8_pack"),
        (lib.ganet_rows8_pack(4, 8, 0, 0, A, 8, A, 24, A, 4, None), 1, b"ganet_rows8_pack"),
        (lib.ganet_rows8_pack(4, 8, 0, 0, A, 8, A + 8, 16, A, 4, None), 1, b"ganet_rows8_pack"),
        (lib.ganet_rows8_pack(4, 513, 0, 0, A, 513, A, 528, A, 4, None), 1, b"ganet_rows8_pack"),
        (lib.ganet_rows8_unpack(4, 8, 0, 0, A, 16, A, 4, None, None), 1, b"ganet_rows8_unpack"),
        (lib.ganet_weight8_pack(0, 8, 0, A, 8, A, 16, A, 4, None, 0, None, 0, None), 4, b"ganet_weight8_pack"),
        (lib.ganet_weight8_pack(8, 8, 0, A, 8, A, 16, A, 4, A, 8, A, 4, None), 1, b"ganet_weight8_pack"),
        (lib.ganet_gemm8(4, 0, 8, 0, A, 16, A, 4, A, 16, A, 4, None, 0, A, 8, 0, None), 4, b"ganet_gemm8"),
        (lib.ganet_gemm8(4, 8, 8, 0, A, 16, A, 4, A, 16, A, 4, None, 0, A, 7, 0, None), 1, b"ganet_gemm8"),
        (lib.ganet_gemm8(4, 8, 8, 0, A, 16, A, 4, None, 16, A, 4, None, 0, A, 8, 0, None), 1, b"ganet_gemm8"),
        (lib.ganet_wgrad8(4, 8, 1 << 22, 0, 0, A, 8, A, 16, A, 4, A, None, 0, None, 0, None), 4, b"ganet_wgrad8"),
        (lib.ganet_wgrad8(4096, 8, 8, 0, 0, A, 8, A, 16, A, 4, A, None, 0, None, 0, None), 1, b"ganet_wgrad8"),
        (lib.ganet_linear8_held(64, 8, 8, 0, A, 8, A, 16, A, 4, None, 0, A, None, 0, None), 1, b"ganet_linear8_held"),
        (lib.ganet_linear8_fwd(4, 8, 8, 0, A, 8, 0, A, 8, None, 0, A, None, A, None, None), 4, b"ganet_linear8_fwd"),
        (lib.ganet_linear8_bwd(4, 8, 8, 0, A, 8, A, None, A, A, None, 0, A, 1 << 20, None), 4, b"ganet_linear8_bwd"),
        (lib.ganet_ln_fwd(4, 8, 0, 0, A, 8, None, None, 1e-5, 3, A, None, None, None, 0, None), 4, b"ganet_ln_fwd"),
        (lib.ganet_ln_fwd(4, 8, 0, 0, A, 4, None, None, 1e-5, 0, A, None, None, None, 0, None), 1, b"ganet_ln_fwd"),
        (lib.ganet_ln_fwd(4, 24, 0, 0, A, 24, None, None, 1e-5, 0, A, None, None, A, 24, None), 1, b"ganet_ln_fwd"),
        (lib.ganet_ln_bwd(4, 8, 0, 0, None, 8, A, None, 0, A, None, None, 0, A, 8, A, None, None, None, 0, None), 1, b"ganet_ln_bwd"),
        (lib.ganet_ln_bwd(4, 8, 0, 0, A, 8, A, None, 0, A, None, None, 0, A, 8, A, A, A, None, 0, None), 1, b"ganet_ln_bwd"),
    ]
    for rc, want, _ in cases:
        assert rc == want
    rc, _, text = (lib.ganet_ln_fwd(-1, 8, 0, 0, A, 8, None, None, 1e-5, 0, A, None, None, None, 0, None), 4, b"ganet_ln_fwd")
    assert rc == 4 and text in lib.ganet_last_error()
    # sizes of what cannot be are zero; of no rows: nothing to do
    assert lib.ganet_rows8_bytes(-1, 8) == 0 and lib.ganet_rows8_bytes(3, 66) == 3 * 80 + 3 * 4 and lib.ganet_weight8_bytes(130, 66) == 130 * 80 + 2 * 4
    assert lib.ganet_wgrad8_workspace(4, 8, 1 << 22, 0) == 0 and lib.ganet_ln_bwd_workspace(-1, 8, 0) == 0
    assert lib.ganet_rows8_pack(0, 8, 0, 0, None, 8, None, 16, None, 4, None) == 0


def test_refusals_of_row_strides_beyond_32_bit_offsets():
    lib = _native.ganet()
    A, far = 1 << 20, (1 << 24) + 16
    for ldg, ldc, lde in ((far, 16, 4), (8, far, 4), (8, 16, far)):
        assert lib.ganet_wgrad8(4, 8, 8, 0, 0, A, ldg, A, ldc, A, lde, A, None, 0, None, 0, None) == 1
        assert b"ganet_wgrad8" in lib.ganet_last_error()


def test_linear_with_an_8_bit_checkpoint_under_autocast_on_the_cpu():
    x, w = torch.randn(6, 20, requires_grad=True), torch.randn(5, 20, requires_grad=True)
    with torch.autocast("cpu", torch.bfloat16):
        y = fused.linear(x, w, None, checkpoint8=True)
    dx, dw = torch.autograd.grad(y.sum(), (x, w))
    assert y.dtype == torch.bfloat16 and dx.dtype == dw.dtype == torch.float32
    with torch.no_grad():
        assert torch.equal(fused.linear(x, w, None, checkpoint8=True), torch.nn.functional.linear(x, w))


def test_a_decoder_unpickled_from_before_it_had_a_norm_runs():
    dec = ShapeDecoder(4, 16)
    x = torch.randn(1, 4, 12)
    want = dec.eval()(x)
    del dec.norm, dec.bits8
    for a, b in zip(dec(x), want):
        assert torch.equal(a, b)
