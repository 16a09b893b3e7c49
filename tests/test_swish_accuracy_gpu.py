"""How near Swish of fp32 tensors comes to its definition, in units u = 2^-24, where only the arithmetic's own errors are allowed.

e = exp(-|x|): 2 units in the last place, 4 u.  1 + e: 1 u, its reciprocal 2 u, and e's error enters by e / (1 + e): sigma(|x|) is off by at most 5 u, sigma(-|x|) = e / (1 + e)
by 4 / (1 + e) + 1 + 2 + 1: 8 u.  swish = x sigma: 9 u.  swish' = sigma + swish (1 - sigma): 8 u of sigma, 9 + 5 u of the other term, 1 u each for the multiply-add's
two parts: 16 u of their size.  Where e is a subnormal number it is off by up to 2 of its steps of 2^-149, sigma by 3, and the results by (1 + |x|) as much."""
import pytest
import torch

from _layers64 import F32, activation64, unpack64
from thor_b200 import DataType
from thor_b200.activation import CheckpointedActivation, CheckpointedActivationBackward, CheckpointedActivationKind as Kind

pytestmark = pytest.mark.gpu


def steps(x):
    return 3 * (1 + x.abs()) * 2.0**-149 + 2.0**-149


def test_values():
    x = torch.cat([torch.linspace(-110, 110, 600000, device="cuda"), torch.linspace(-8, 8, 200000, device="cuda"), -torch.logspace(-30, 0, 2048, device="cuda"),
                   torch.logspace(-30, 38, 4096, device="cuda")])
    x = x[:x.numel() // 32 * 32].reshape(-1, 32).contiguous()
    y = CheckpointedActivation(Kind.Swish).stamp(x).run()
    want, _, _ = activation64(x.double(), "swish")
    assert ((y.double() - want).abs() <= 9 * F32 * want.abs() + steps(x.double())).all()


@pytest.mark.parametrize("width", [32, 2049])  # aligned rows, and long odd ones
def test_slopes(width):
    sizes = torch.linspace(0.001, 1, 3000, device="cuda")[:, None]  # every block of its own size
    for size in (1.0, 6.0, 14.0, 60.0, 110.0):
        x = (sizes * torch.linspace(-1, 1, width, device="cuda")[None] * size).contiguous()
        forward = CheckpointedActivation(Kind.Swish, DataType.int8).stamp(x)
        forward.run()
        got = CheckpointedActivationBackward(Kind.Swish).stamp(torch.ones_like(x), forward.checkpoint).run()
        xk = unpack64(forward.checkpoint.codes, forward.checkpoint.scales, width)
        _, want, magnitude = activation64(xk, "swish")
        assert ((got.double() - want).abs() <= 16 * F32 * magnitude + steps(xk)).all()
