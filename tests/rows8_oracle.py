"""The 8-bit row formats, layer norm and their products from their definitions, in 64 bits and without the package."""
import torch

BLOCK = 128
FORMATS = {"e4m3": (448.0, 3, -6), "e5m2": (57344.0, 2, -14)}          # largest value, mantissa bits, smallest normal exponent


def half_step(dtype):
    """The largest relative error of one rounding to `dtype`."""
    return torch.finfo(dtype).eps / 2


def _two_to(e):
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def grid(v, fmt):
    """The format's nearest value (ties to even); infinities and NaN as they are."""
    _, mant, low = FORMATS[fmt]
    fine = torch.where(torch.isfinite(v), v, torch.zeros_like(v))
    step = _two_to((torch.frexp(fine).exponent - 1).clamp_min(low) - mant)
    return torch.where(torch.isfinite(v), torch.round(fine / step) * step, v)


def exponent(a, fmt):
    """The smallest e >= -126 with a <= F 2^e; 0 for a = 0."""
    most = FORMATS[fmt][0]
    e = torch.frexp(a / most).exponent.to(torch.int64)
    e = torch.where(_two_to(e - 1) * most >= a, e - 1, e)
    return torch.where(a > 0, e.clamp_min(-126), torch.zeros_like(e))


def _amax(x, dims):
    return torch.where(torch.isfinite(x), x.abs(), torch.zeros_like(x)).amax(dims)


def rows(x, fmt="e4m3"):
    """x [M, K] -> (values in 64 bits, exponents [M, K / 128])."""
    M, K = x.shape
    kb = -(-K // BLOCK)
    b = torch.nn.functional.pad(x.double(), (0, kb * BLOCK - K)).reshape(M, kb, BLOCK)
    e = exponent(_amax(b, 2), fmt)
    v = grid(b / _two_to(e)[..., None], fmt)
    if fmt == "e4m3":
        v = torch.where(torch.isinf(v), torch.full_like(v, float("nan")), v)
    return (v * _two_to(e)[..., None]).reshape(M, kb * BLOCK)[:, :K], e


def weight(w):
    """w [N, K] -> (values in 64 bits, exponents [N / 128, K / 128])."""
    N, K = w.shape
    nb, kb = -(-N // BLOCK), -(-K // BLOCK)
    b = torch.nn.functional.pad(w.double(), (0, kb * BLOCK - K, 0, nb * BLOCK - N)).reshape(nb, BLOCK, kb, BLOCK)
    e = exponent(_amax(b, (1, 3)), "e4m3")
    s = _two_to(e)[:, None, :, None]
    return (grid(b / s, "e4m3") * s).reshape(nb * BLOCK, kb * BLOCK)[:N, :K], e


def near_a_border(v, fmt, rel):
    """Where v lies within rel |v| of the middle between two values of the format: a value computed in fewer bits may round the other way."""
    return grid(v * (1 + rel), fmt) != grid(v * (1 - rel), fmt)


def act(u, kind):
    return torch.logaddexp(u, torch.zeros_like(u)) if kind == "softplus" else torch.relu(u) if kind == "relu" else u


def act_grad(u, kind):
    return torch.sigmoid(u) if kind == "softplus" else (u > 0).to(u.dtype) if kind == "relu" else torch.ones_like(u)


def kept_scale(C):
    """2^e with the smallest e such that sqrt(C) <= 448 2^e."""
    return float(_two_to(exponent(torch.tensor(C, dtype=torch.float64).sqrt(), "e4m3")))


def layer_norm(x, w, b, eps, kind):
    """-> (y, xh, rstd) in 64 bits."""
    x = x.double()
    mean = x.mean(1, keepdim=True)
    rstd = 1 / torch.sqrt(((x - mean) ** 2).mean(1, keepdim=True) + eps)
    xh = (x - mean) * rstd
    return act(xh * w + b, kind), xh, rstd


def layer_norm_grads(xh, rstd, w, b, kind, dy):
    """-> (dx, dw, db) of sum(dy y), for the given xh."""
    g = dy.double() * act_grad(xh * w + b, kind)
    gw = g * w
    dx = rstd * (gw - gw.mean(1, keepdim=True) - xh * (gw * xh).mean(1, keepdim=True))
    return dx, (g * xh).sum(0), g.sum(0)
