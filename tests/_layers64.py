"""64-bit definitions of the 8-bit checkpoint, the checkpointed activations and LayerNorm, for the tests of those operators.
Nothing here imports the library."""
import math

import torch

LARGEST = {torch.float8_e4m3fn: 448.0, torch.float8_e5m2: 57344.0, torch.int8: 127.0}
CODES = (torch.float8_e4m3fn, torch.float8_e5m2, torch.int8)
HALF_ULP = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}  # torch.finfo(t).eps / 2
assert all(HALF_ULP[t] == torch.finfo(t).eps / 2 for t in HALF_ULP)
F32 = 2.0**-24


def pitch(cols):
    return -(-cols // 16) * 16


def blocks_of(x, fill=0.0):
    """[rows, cols] -> [rows, ceil(cols / 32), 32], padded with `fill`."""
    rows, cols = x.shape
    wide = -(-cols // 32) * 32
    out = torch.full((rows, wide), fill, dtype=x.dtype, device=x.device)
    out[:, :cols] = x
    return out.reshape(rows, wide // 32, 32)


def step_of(q, code):
    """Distance of neighbouring codes at magnitude |q| (q in units of the scale)."""
    if code == torch.int8:
        return torch.ones_like(q)
    bits, lowest = (3, -6) if code == torch.float8_e4m3fn else (2, -14)
    return torch.exp2((torch.frexp(q).exponent - 1).double().clamp(min=lowest) - bits)


def exponent_of(largest, code):
    """log2 of the smallest power of two s >= 2^-127 with largest <= s * M."""
    mantissa, power = torch.frexp(largest / LARGEST[code])
    power = (power - (mantissa == 0.5).to(power.dtype)).double().clamp(min=-127)
    return torch.where(largest == 0, -127.0, power)


def pack64(x, code):
    """fp64 [rows, cols] -> (codes as fp64 [rows, pitch], scale bytes uint8)."""
    rows, cols = x.shape
    p = blocks_of(x)
    broken = ~torch.isfinite(p).all(-1)
    p = torch.where(broken[..., None], 0.0, p)
    power = exponent_of(p.abs().amax(-1), code)
    q = p * torch.exp2(-power)[..., None]
    step = step_of(q, code)
    codes = torch.round(q / step) * step
    bytes_ = torch.where(broken, 255, (power + 127).to(torch.int64)).to(torch.uint8)
    return codes.reshape(rows, -1)[:, :pitch(cols)], bytes_


def unpack64(codes, scales, cols):
    b = scales.view(torch.uint8).double()
    s = torch.where(b == 255, math.nan, torch.exp2(b - 127))
    return codes.double()[:, :cols] * s.repeat_interleave(32, 1)[:, :cols]


def activation64(x, kind):
    """act(x), act'(x), and the magnitude that the rounding errors of act' refer to (its terms do not cancel there)."""
    if kind == "swish":
        s = torch.sigmoid(x)
        return x * s, s * (1 + x * (1 - s)), s * (1 + x.abs() * (1 - s))
    phi = 0.5 * torch.erfc(x * -math.sqrt(0.5))  # special.ndtr is 1 + erf: no relative accuracy in the tail
    pdf = torch.exp(-0.5 * x * x) / math.sqrt(2 * math.pi)
    return x * phi, phi + x * pdf, phi + x.abs() * pdf


def activation_error(x, kind, dtype):
    """Relative error allowed to act, sigma, Phi and phi before the last rounding.  fp32 tensors: 16 units of 2^-24 (two hardware
    approximations of up to 4 units each, the polynomial's 3.6 and the products), plus what the exponent's argument (x for swish, x^2 / 2
    for gelu) carries: one rounding of the product and a quarter for the constant's, 2 units allowed.  16-bit tensors: the polynomial of
    Phi is off by 4.8e-6 < 2^-17.5 of the value, and the rounding of x^2 is not carried (one unit more)."""
    argument = x.abs() if kind == "swish" else 0.5 * x * x
    if dtype == torch.float32 or kind == "swish":
        return 16 * F32 + 2 * F32 * argument
    return 16 * F32 + 2.0**-17.5 + 3 * F32 * argument


def layernorm64(h, gamma, beta, eps):
    """mean, rstd, normalised, output"""
    mean = h.mean(1)
    d = h - mean[:, None]
    rstd = 1 / torch.sqrt((d * d).mean(1) + eps)
    n = d * rstd[:, None]
    return mean, rstd, n, n * gamma + beta


def layernorm_grads64(grad, n, rstd, gamma):
    w = grad * gamma
    c1, c2 = w.mean(1, keepdim=True), (w * n).mean(1, keepdim=True)
    return rstd[:, None] * (w - c1 - n * c2), (grad * n).sum(0), grad.sum(0)
