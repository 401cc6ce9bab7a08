"""Activations and weights in 8-bit floating point, and the linear layers that work on them (include/ganet.h: ganet_rows8_*,
ganet_weight8_pack, ganet_gemm8, ganet_wgrad8).

    rows = quantize8(x)               x [..., K] as codes, a power of two for every 128 columns of a row: 8 bits and a bit
    rows.dequantize(dtype)            the values that the codes stand for
    dW, db = wgrad8(g, rows)          a linear layer's weight gradient straight from its packed input
    w8 = quantize8_weight(w)          a weight [N, K], a power of two for every 128 x 128 block
    matmul8(rows, w8, bias)           their product (fast: on the 8-bit matrix instructions)
    linear8(x, w, bias)               a linear layer on these: forward and backward in training, or with a held Weight8

With a = the largest finite magnitude of a block and F the largest value of the format (e4m3: 448, e5m2: 57344), the block's exponent e
is the smallest integer >= -126 with a <= F 2^e (a = 0: 0); code = x 2^-e rounded to nearest, ties to even. A NaN stays one, an
infinity becomes NaN in e4m3 and stays infinite in e5m2; neither moves the exponent of its block.

fp32, bf16 and fp16 tensors on a HIP device run on the kernels; on the CPU the same definitions run as plain torch operations.
"""
from __future__ import annotations

import torch

from . import _native

FORMATS = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
_FMT_CODE = {torch.float8_e4m3fn: 0, torch.float8_e5m2: 1}
_TYPE_CODE = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_FAST = 1 << 8                                                       # GANET_FAST
_DB_TYPE = {t: c + 1 << 8 for t, c in _TYPE_CODE.items()}          # GANET_DB_TYPE
BLOCK = 128


def _ptr(t):
    return None if t is None else t.data_ptr()


def _call(device, fn, *args):
    """fn(*args, stream) on `device`'s current stream; the launch happens with that device current."""
    index = device.index
    if index is None or index == torch._C._cuda_getDevice():
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(torch._C._cuda_getDevice() if index is None else index))
    else:
        with torch.cuda.device(device):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    if rc:
        _native.ganet_check(rc)


def _type_code(t, what):
    code = _TYPE_CODE.get(t.dtype)
    if code is None:
        raise TypeError(f"{what}: float32, bfloat16 or float16 expected, got {t.dtype}")
    return code


def _rows2d(x):
    """x as [M, K] whose rows are adjacent in memory, do not overlap and lie at most 2^24 elements apart (a copy only where they are not)."""
    x2 = x if x.dim() == 2 else x.reshape(-1, x.shape[-1])
    K = x2.shape[1]
    if (K > 1 and x2.stride(1) != 1) or (x2.shape[0] > 1 and not K <= x2.stride(0) <= 1 << 24):
        x2 = x2.contiguous()
    return x2


def _ld(x2):
    return max(x2.stride(0), x2.shape[1]) if x2.shape[0] > 1 else x2.shape[1]


def _same_device(what, first, *others):
    for t in others:
        if t is not None and t.device != first.device:
            raise ValueError(f"{what}: tensors on {first.device} and {t.device}")


def _pad(n, to):
    return (n + to - 1) // to * to


def _check_codes(what, codes, exps, cols, kinds):
    if codes.dtype not in kinds or codes.dim() != 2 or exps.dtype != torch.uint8 or exps.dim() != 2:
        raise TypeError(f"{what}: codes [., .] in {' or '.join(str(k) for k in kinds)} and uint8 exponents [., .] expected, got "
                        f"{codes.dtype} {tuple(codes.shape)} and {exps.dtype} {tuple(exps.shape)}")
    if cols < 1 or codes.shape[1] < _pad(cols, 16) or codes.shape[1] % 16 or exps.shape[1] * BLOCK < cols or exps.shape[1] % 4:
        raise ValueError(f"{what}: {cols} columns need codes of a width >= {_pad(max(cols, 1), 16)} and a multiple of 16, and exponents of a "
                         f"width >= {_pad((max(cols, 1) + BLOCK - 1) // BLOCK, 4)} and a multiple of 4; got {codes.shape[1]} and {exps.shape[1]}")
    if not codes.is_contiguous() or not exps.is_contiguous():
        raise ValueError(f"{what}: contiguous codes and exponents expected")
    _same_device(what, codes, exps)


class Rows8:
    """Rows in 8 bits. codes [M, K up to a multiple of 16] (float8_e4m3fn or float8_e5m2, zero past column K), exps [M, K / 128 up to
    a multiple of 4] uint8 (the exponent of each 128 columns + 127: 1 to 254), cols = K, lead = the leading dimensions of what was packed."""
    __slots__ = ("codes", "exps", "cols", "lead")

    def __init__(self, codes, exps, cols, lead=None):
        _check_codes("Rows8", codes, exps, int(cols), tuple(_FMT_CODE))
        if exps.shape[0] != codes.shape[0]:
            raise ValueError(f"Rows8: {codes.shape[0]} rows of codes and {exps.shape[0]} of exponents")
        self.codes, self.exps, self.cols = codes, exps, int(cols)
        self.lead = (codes.shape[0],) if lead is None else tuple(lead)

    def dequantize(self, dtype=torch.float32):
        """The values, [*lead, K] in `dtype`; one beyond its range becomes its largest number."""
        if dtype not in _TYPE_CODE:
            raise TypeError(f"dequantize: float32, bfloat16 or float16 expected, got {dtype}")
        M, K = self.codes.shape[0], self.cols
        if not self.codes.is_cuda:
            return _plain_values(self.codes, self.exps, K, dtype).reshape(*self.lead, K)
        y = torch.empty((M, K), dtype=dtype, device=self.codes.device)
        _call(y.device, _native.ganet().ganet_rows8_unpack, M, K, _TYPE_CODE[dtype], _FMT_CODE[self.codes.dtype], _ptr(self.codes),
              self.codes.stride(0), _ptr(self.exps), self.exps.stride(0), _ptr(y))
        return y.reshape(*self.lead, K)


class Weight8:
    """A weight [N, K] in 8 bits: codes [N, K up to a multiple of 16] in float8_e4m3fn, zero past column K, exps [N / 128, K / 128 up to a
    multiple of 4] uint8 (exponents + 127: 1 to 254), cols = K. t_codes, t_exps: the same for the transposed weight, or None."""
    __slots__ = ("codes", "exps", "cols", "t_codes", "t_exps")

    def __init__(self, codes, exps, cols, t_codes=None, t_exps=None):
        _check_codes("Weight8", codes, exps, int(cols), (torch.float8_e4m3fn,))
        if exps.shape[0] * BLOCK < codes.shape[0] or codes.shape[0] < 1:
            raise ValueError(f"Weight8: {codes.shape[0]} rows of codes and {exps.shape[0]} rows of exponents (one per {BLOCK})")
        if t_codes is not None:
            _check_codes("Weight8 (transposed)", t_codes, t_exps, codes.shape[0], (torch.float8_e4m3fn,))
            if t_codes.shape[0] != int(cols) or t_exps.shape[0] * BLOCK < int(cols):
                raise ValueError(f"Weight8: the transposed weight has {t_codes.shape[0]} rows of codes and {t_exps.shape[0]} of exponents")
            _same_device("Weight8", codes, t_codes)
        self.codes, self.exps, self.cols, self.t_codes, self.t_exps = codes, exps, int(cols), t_codes, t_exps

    @property
    def shape(self):
        return (self.codes.shape[0], self.cols)

    def transposed(self):
        if self.t_codes is None:
            raise ValueError("Weight8: made without its transposed codes (quantize8_weight(w, transposed=True))")
        return Weight8(self.t_codes, self.t_exps, self.codes.shape[0], self.codes, self.exps)

    def dequantize(self, dtype=torch.float32):
        """The values, [N, K] in `dtype` (as a check or a copy: the products read the codes)."""
        N = self.codes.shape[0]
        exps = self.exps.repeat_interleave(BLOCK, 0)[:N]
        return Rows8(self.codes, exps, self.cols).dequantize(dtype)


# ------------------------------------------------------------------------------------------------ the definitions, in torch


def _plain_exponent(a, kind):
    m, p = torch.frexp(a)                                    # a = m 2^p, 1/2 <= m < 1; F = 7/8 2^(9 or 16)
    e = (p - (9 if kind == torch.float8_e4m3fn else 16) + (m > 0.875).to(p.dtype)).clamp_min(-126)
    return torch.where(a > 0, e, torch.zeros_like(e))


def _finite_abs(x):
    return torch.where(torch.isfinite(x), x.abs(), torch.zeros_like(x))


def _plain_rows(x2, kind):
    M, K = x2.shape
    KB = (K + BLOCK - 1) // BLOCK
    blocks = torch.nn.functional.pad(x2.float(), (0, KB * BLOCK - K)).reshape(M, KB, BLOCK)
    e = _plain_exponent(_finite_abs(blocks).amax(2), kind)
    codes = torch.ldexp(blocks, -e[..., None]).reshape(M, KB * BLOCK)[:, :_pad(K, 16)].to(kind).contiguous()
    exps = torch.nn.functional.pad(e + 127, (0, _pad(KB, 4) - KB), value=127).to(torch.uint8)
    return codes, exps.contiguous()


def _plain_weight(w):
    N, K = w.shape
    NB, KB = (N + BLOCK - 1) // BLOCK, (K + BLOCK - 1) // BLOCK
    blocks = torch.nn.functional.pad(w.float(), (0, KB * BLOCK - K, 0, NB * BLOCK - N)).reshape(NB, BLOCK, KB, BLOCK)
    e = _plain_exponent(_finite_abs(blocks).amax((1, 3)), torch.float8_e4m3fn)
    codes = torch.ldexp(blocks, -e[:, None, :, None]).reshape(NB * BLOCK, KB * BLOCK)[:N, :_pad(K, 16)]
    exps = torch.nn.functional.pad(e + 127, (0, _pad(KB, 4) - KB), value=127).to(torch.uint8)
    return codes.to(torch.float8_e4m3fn).contiguous(), exps.contiguous()


def _plain_values(codes, exps, cols, dtype=torch.float32):
    e = (exps.int() - 127).repeat_interleave(BLOCK, 1)[:, :cols]
    v = codes[:, :cols].double()
    most = torch.finfo(dtype).max
    r = torch.ldexp(v, e)
    return torch.where(torch.isfinite(v), r.clamp(-most, most), r).to(dtype)


# ------------------------------------------------------------------------------------------------ the operators


def quantize8(x, fmt="e4m3"):
    """x [..., K] -> Rows8. Not differentiable by itself: linear8, fused.linear and fused.layernorm_act use it inside their own backward."""
    if fmt not in FORMATS:
        raise ValueError(f"quantize8: format {fmt!r} (known: {', '.join(FORMATS)})")
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"quantize8: [..., K] with K >= 1 expected, got {tuple(x.shape)}")
    code = _type_code(x, "quantize8")
    kind = FORMATS[fmt]
    x2 = _rows2d(x.detach())
    M, K = x2.shape
    lead = x.shape[:-1]
    if not x.is_cuda:
        return Rows8(*_plain_rows(x2, kind), K, lead)
    codes = torch.empty((M, _pad(K, 16)), dtype=kind, device=x.device)
    exps = torch.empty((M, _pad((K + BLOCK - 1) // BLOCK, 4)), dtype=torch.uint8, device=x.device)
    _call(x.device, _native.ganet().ganet_rows8_pack, M, K, code, _FMT_CODE[kind], _ptr(x2), _ld(x2), _ptr(codes), codes.stride(0),
          _ptr(exps), exps.stride(0))
    return Rows8(codes, exps, K, lead)


def quantize8_weight(w, transposed=False):
    """w [N, K] -> Weight8; transposed: with the codes of w^T too (products with the other side: an input gradient)."""
    if w.dim() != 2 or w.shape[0] < 1 or w.shape[1] < 1:
        raise ValueError(f"quantize8_weight: [N, K] expected, got {tuple(w.shape)}")
    code = _type_code(w, "quantize8_weight")
    w2 = _rows2d(w.detach())
    N, K = w2.shape
    if not w.is_cuda:
        t = _plain_weight(w2.t()) if transposed else (None, None)
        return Weight8(*_plain_weight(w2), K, *t)
    NB, KB = (N + BLOCK - 1) // BLOCK, (K + BLOCK - 1) // BLOCK
    make = lambda rows, cols: torch.empty((rows, cols), dtype=torch.uint8, device=w.device)
    codes, exps = make(N, _pad(K, 16)), make(NB, _pad(KB, 4))
    t_codes, t_exps = (make(K, _pad(N, 16)), make(KB, _pad(NB, 4))) if transposed else (None, None)
    _call(w.device, _native.ganet().ganet_weight8_pack, N, K, code, _ptr(w2), _ld(w2), _ptr(codes), codes.stride(0), _ptr(exps),
          exps.stride(0), _ptr(t_codes), t_codes.stride(0) if transposed else 0, _ptr(t_exps), t_exps.stride(0) if transposed else 0)
    as8 = lambda t: None if t is None else t.view(torch.float8_e4m3fn)
    return Weight8(as8(codes), exps, K, as8(t_codes), t_exps)


def matmul8(rows, w8, bias=None, dtype=torch.float32, fast=False):
    """rows [..., K] times w8 [N, K] transposed, plus bias [N]: [..., N] in `dtype`. Sums are fp32, rounded once. Not differentiable by
    itself (linear8 is). fast: 16-bit results of more than 32 rows on a HIP device are summed by the 8-bit matrix instructions, up to 1.8 times as
    fast; they first cut each product to 2^-13 of the largest power of two among eight adjacent columns' products: 3e-5 to 6e-5 of the result's norm, and 2^-13 of
    large products that cancel."""
    if rows.cols != w8.cols:
        raise ValueError(f"matmul8: rows of {rows.cols} columns, a weight of {w8.cols}")
    if dtype not in _TYPE_CODE:
        raise TypeError(f"matmul8: float32, bfloat16 or float16 expected, got {dtype}")
    N, K = w8.shape
    if bias is not None and tuple(bias.shape) != (N,):
        raise ValueError(f"matmul8: a bias of {tuple(bias.shape)} for {N} columns")
    btype = 0 if bias is None else _type_code(bias, "matmul8: bias")
    _same_device("matmul8", rows.codes, w8.codes, bias)
    M = rows.codes.shape[0]
    if not rows.codes.is_cuda:
        y = _plain_values(rows.codes, rows.exps, K) @ w8.dequantize().t()
        return (y if bias is None else y + bias.float()).to(dtype).reshape(*rows.lead, N)
    y = torch.empty((M, N), dtype=dtype, device=rows.codes.device)
    bias = None if bias is None else bias.detach().contiguous()
    _call(y.device, _native.ganet().ganet_gemm8, M, N, K, _FMT_CODE[rows.codes.dtype], _ptr(rows.codes), rows.codes.stride(0),
          _ptr(rows.exps), rows.exps.stride(0), _ptr(w8.codes), w8.codes.stride(0), _ptr(w8.exps), w8.exps.stride(0), _ptr(bias), btype,
          _ptr(y), N, _TYPE_CODE[dtype] | (_FAST if fast else 0))
    return y.reshape(*rows.lead, N)


def wgrad8(g, rows, dtype=None, bias_dtype=None):
    """(dW [N, K], db [N]) = (g^T rows, column sums of g) for g [..., N] over the same rows, in `dtype` (g's own by default), db in
    `bias_dtype` (dtype by default). g enters with all its bits (of an fp32 value, those down to 2^-133), sums are fp32, each result is
    rounded once. A non-finite g makes its row of dW non-finite."""
    code = _type_code(g, "wgrad8")
    dtype = g.dtype if dtype is None else dtype
    bias_dtype = dtype if bias_dtype is None else bias_dtype
    for t in (dtype, bias_dtype):
        if t not in _TYPE_CODE:
            raise TypeError(f"wgrad8: float32, bfloat16 or float16 expected, got {t}")
    if g.dim() < 1 or g.shape[-1] < 1:
        raise ValueError(f"wgrad8: [..., N] with N >= 1 expected, got {tuple(g.shape)}")
    g2 = _rows2d(g.detach())
    M, N = g2.shape
    K = rows.cols
    if M != rows.codes.shape[0]:
        raise ValueError(f"wgrad8: {M} rows of gradient, {rows.codes.shape[0]} packed rows")
    _same_device("wgrad8", g, rows.codes)
    if not g.is_cuda:
        gf = g2.double()
        return (gf.t() @ _plain_values(rows.codes, rows.exps, K).double()).to(dtype), gf.sum(0).to(bias_dtype)
    lib = _native.ganet()
    dW = torch.empty((N, K), dtype=dtype, device=g.device)
    db = torch.empty(N, dtype=bias_dtype, device=g.device)
    nbytes = lib.ganet_wgrad8_workspace(M, N, K, code)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=g.device) if nbytes else None
    _call(g.device, lib.ganet_wgrad8, M, N, K, _FMT_CODE[rows.codes.dtype], code, _ptr(g2), _ld(g2), _ptr(rows.codes),
          rows.codes.stride(0), _ptr(rows.exps), rows.exps.stride(0), _ptr(dW), _ptr(db), _TYPE_CODE[dtype] | _DB_TYPE[bias_dtype], _ptr(ws), nbytes)
    return dW, db


def check_trains(what, K, N, *params):
    """Raises where a weight gradient on the kernels will be asked for that they do not take (columns: K < 2^22, N < 2^24)."""
    if (K >= 1 << 22 or N >= 1 << 24) and torch.is_grad_enabled() and any(p is not None and p.requires_grad for p in params):
        raise ValueError(f"{what}: a weight gradient of {N} x {K} (fewer than 2^22 columns in and 2^24 out expected); under torch.no_grad() the product itself runs")


def _bytes(n, like):
    return torch.empty(n, dtype=torch.uint8, device=like.device)


class _Linear8Fn(torch.autograd.Function):
    """y = Q(x) Q(W)^T + b; dx = Q(g) Q(W); dW = g^T Q(x); db = sum g. The packed input of the product is what the backward pass keeps of x."""

    @staticmethod
    def forward(ctx, x, weight, bias, fast):
        x2, w2 = _rows2d(x), _rows2d(weight)
        M, K = x2.shape
        N = w2.shape[0]
        lib = _native.ganet()
        y = torch.empty((M, N), dtype=x.dtype, device=x.device)
        rows, held = _bytes(max(16, lib.ganet_rows8_bytes(M, K)), x), _bytes(lib.ganet_weight8_bytes(N, K), x)
        back = _bytes(lib.ganet_weight8_bytes(K, N), x) if ctx.needs_input_grad[0] else None
        b = None if bias is None else bias.contiguous()
        ctx.code = _TYPE_CODE[x.dtype] | (_FAST if fast else 0)
        _call(x.device, lib.ganet_linear8_fwd, M, N, K, ctx.code, x2.data_ptr(), _ld(x2), _TYPE_CODE[weight.dtype],
              w2.data_ptr(), _ld(w2), _ptr(b), 0 if b is None else _TYPE_CODE[b.dtype], y.data_ptr(), rows.data_ptr(),
              held.data_ptr(), _ptr(back))
        ctx.save_for_backward(rows, back)
        ctx.dims, ctx.shape = (M, N, K), x.shape
        ctx.types = (x.dtype, weight.dtype, None if bias is None else bias.dtype)
        return y if x.dim() == 2 else y.reshape(*x.shape[:-1], N)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):
        rows, back = ctx.saved_tensors
        M, N, K = ctx.dims
        xt, wt, bt = ctx.types
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        need_b = need_b and bt is not None
        lib = _native.ganet()
        g2 = _rows2d(g)
        new = lambda shape, t: torch.empty(shape, dtype=t, device=g.device)
        dx = new((M, K), xt) if need_x else None
        dW = new((N, K), wt) if need_w or need_b else None
        db = new(N, bt) if need_b else None
        code = ctx.code
        ws = _bytes(max(16, lib.ganet_linear8_bwd_workspace(M, N, K, code)), g)
        _call(g.device, lib.ganet_linear8_bwd, M, N, K, code, g2.data_ptr(), _ld(g2), rows.data_ptr(), _ptr(back), _ptr(dx), _ptr(dW),
              _ptr(db), _TYPE_CODE[wt] | _DB_TYPE[bt or wt], ws.data_ptr(), ws.numel())
        if need_x and len(ctx.shape) != 2:
            dx = dx.reshape(ctx.shape)
        return dx, dW if need_w else None, db, None


class _Linear8Plain(torch.autograd.Function):
    """The same in torch operations (CPU)."""

    @staticmethod
    def forward(ctx, x, weight, bias, fast):
        rows = quantize8(x)
        w8 = quantize8_weight(weight)
        ctx.save_for_backward(rows.codes, rows.exps, w8.codes, w8.exps)
        ctx.shape, ctx.types = x.shape, (x.dtype, weight.dtype, None if bias is None else bias.dtype)
        return matmul8(rows, w8, bias, x.dtype)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):
        codes, exps, w_codes, w_exps = ctx.saved_tensors
        xt, wt, bt = ctx.types
        w = Weight8(w_codes, w_exps, ctx.shape[-1]).dequantize()
        q = quantize8(g)
        dx = (q.dequantize() @ w).to(xt)
        dW, db = wgrad8(g, Rows8(codes, exps, ctx.shape[-1], ctx.shape[:-1]), wt, bt)
        return dx, dW, None if bt is None else db, None


def linear8(x, weight, bias=None, fast=False):
    """x [..., K] -> [..., N] in x's type, in 8-bit floating point (see matmul8). weight: a tensor [N, K] (training: differentiable in x, weight
    and bias, K < 2^22 on a HIP device; the weight is packed in the call) or a Weight8 held by the caller (evaluation: not differentiable).
    fast: as matmul8's, for the result and the input gradient."""
    if x.dim() < 1:
        raise ValueError("linear8: [..., K] expected")
    K = x.shape[-1]
    if isinstance(weight, Weight8):
        if K != weight.cols:
            raise ValueError(f"linear8: {K} columns for a weight of {weight.cols}")
        if torch.is_grad_enabled() and (x.requires_grad or (bias is not None and bias.requires_grad)):
            raise RuntimeError("linear8: a held Weight8 is for evaluation (torch.no_grad()); pass the weight itself to train")
        if not x.is_cuda:
            return matmul8(quantize8(x), weight, bias, x.dtype)
        N = weight.codes.shape[0]
        if bias is not None and tuple(bias.shape) != (N,):
            raise ValueError(f"linear8: a bias of {tuple(bias.shape)} for {N} columns")
        code = _type_code(x, "linear8") | (_FAST if fast else 0)
        btype = 0 if bias is None else _type_code(bias, "linear8: bias")
        _same_device("linear8", x, weight.codes, bias)
        x2 = _rows2d(x.detach())
        M = x2.shape[0]
        lib = _native.ganet()
        y = torch.empty((M, N), dtype=x.dtype, device=x.device)
        nbytes = lib.ganet_linear8_held_workspace(M, N, K, code)
        ws = _bytes(nbytes, x) if nbytes else None
        bias = None if bias is None else bias.detach().contiguous()
        _call(x.device, lib.ganet_linear8_held, M, N, K, code, x2.data_ptr(), _ld(x2), weight.codes.data_ptr(), weight.codes.stride(0),
              weight.exps.data_ptr(), weight.exps.stride(0), _ptr(bias), btype, y.data_ptr(), _ptr(ws), nbytes)
        return y if x.dim() == 2 else y.reshape(*x.shape[:-1], N)
    if weight.dim() != 2 or weight.shape[1] != K:
        raise ValueError(f"linear8: {K} columns for a weight of {tuple(weight.shape)}")
    if bias is not None and tuple(bias.shape) != (weight.shape[0],):
        raise ValueError(f"linear8: a bias of {tuple(bias.shape)} for {weight.shape[0]} columns")
    _type_code(x, "linear8")
    _type_code(weight, "linear8: weight")
    if bias is not None:
        _type_code(bias, "linear8: bias")
    _same_device("linear8", x, weight, bias)
    if x.is_cuda:
        check_trains("linear8", K, weight.shape[0], weight, bias)
    return (_Linear8Fn if x.is_cuda else _Linear8Plain).apply(x, weight, bias, fast)
