"""How near GELU of fp32 tensors comes to its definition, in units u = 2^-24, where only the arithmetic's own errors are allowed.

Phi(-a) = R(t) t e with t = 1 / (1 + p a): the fit with its evaluation is off by 2.1e-7 (3.6 u) for an exact t; t itself by 1 u (1 + p a) and 2 u (reciprocal), which R, falling
like t, passes on once; e = 2^y by 4 u (2^-22) and 1 u for the multiply-add that carries what y lacks; two products: 3.6 + 3 + 5 + 2 < 14 u.  gelu(-a) = -a Phi(-a): 15 u.
gelu(a) = a (1 - Phi(-a)): at most 14 u of Phi(-a), which is at most half of 1 or below 1 - Phi, and 2 u of the value: 16 u.
gelu'(-a) = (R t - a phi(0)) e: 3.6 + 3 + 1 u of the first term, 1 u of the constant, 1 u of the multiply-add, 6 u of e and the last product: 15 u of Phi + a phi;
gelu'(a) = 1 - that: 1 u more.  Left of x = -12 the steps of 2^-149 of Phi as a subnormal number come in; the exponential is flushed to zero below 2^-126."""
import pytest
import torch

from _layers64 import F32, activation64, unpack64
from thor_b200 import DataType
from thor_b200.activation import CheckpointedActivation, CheckpointedActivationBackward, CheckpointedActivationKind as Kind

pytestmark = pytest.mark.gpu


def test_values():
    x = torch.cat([torch.linspace(-12, 100, 600000, device="cuda"), torch.linspace(-12, 0, 600000, device="cuda"), -torch.logspace(-30, 0, 2048, device="cuda"),
                   torch.logspace(-30, 38, 4096, device="cuda")])
    x = x[:x.numel() // 32 * 32].reshape(-1, 32).contiguous()
    y = CheckpointedActivation(Kind.Gelu).stamp(x).run()
    want, _, _ = activation64(x.double(), "gelu")
    assert ((y.double() - want).abs() <= 16 * F32 * want.abs() + 2.0**-149).all()


@pytest.mark.parametrize("width", [32, 2049])  # aligned rows, and long odd ones
def test_slopes(width):
    sizes = torch.linspace(0.001, 1, 3000, device="cuda")[:, None]  # every block of its own size
    for size in (1.0, 4.0, 8.0, 12.0, 100.0):
        x = (sizes * torch.linspace(-1, 1, width, device="cuda")[None] * size).contiguous()
        forward = CheckpointedActivation(Kind.Gelu, DataType.int8).stamp(x)
        forward.run()
        got = CheckpointedActivationBackward(Kind.Gelu).stamp(torch.ones_like(x), forward.checkpoint).run()
        xk = unpack64(forward.checkpoint.codes, forward.checkpoint.scales, width)
        _, want, magnitude = activation64(xk, "gelu")
        assert ((got.double() - want).abs() <= 16 * F32 * magnitude + torch.where(xk < -12, (1 + xk.abs()) * 2.0**-126, 0.0)).all()
