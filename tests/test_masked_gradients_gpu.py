"""Gradients of activations where the input or the gate is masked with the type's lowest number."""
import math

import pytest
import torch

from _layers64 import CODES, F32, HALF_ULP, activation64, unpack64
from thor_b200 import DataType
from thor_b200.activation import CheckpointedActivation, CheckpointedActivationBackward, CheckpointedActivationKind as Kind
from thor_b200.checkpoint import CheckpointUnpack
from thor_b200.dtypes import from_torch

pytestmark = pytest.mark.gpu
KINDS = {"gelu": Kind.Gelu, "swish": Kind.Swish}


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("cols", [64, 2049, 2064])
@pytest.mark.parametrize("lowest_in", ["x", "gate"])
def test_masked_with_the_lowest_number(code, dtype, kind, cols, lowest_in):
    """The type's lowest number rounds to the code of -2^128, which no fp32 number holds: its gradients are those of a number that large, not NaN.
    (A place that is masked gives act = 0 and slope 0, and a gradient of zero stays zero whatever it is multiplied with.)"""
    gen = torch.Generator(device="cuda").manual_seed(3)
    x, gate, grad = (torch.randn(6, cols, device="cuda", generator=gen).to(dtype) for _ in range(3))
    lowest = torch.finfo(dtype).min
    (x if lowest_in == "x" else gate)[:, ::5] = lowest
    grad[3:] = 0
    forward = CheckpointedActivation(KINDS[kind], from_torch(code)).stamp(x, gate)
    forward.run()
    odd = [torch.empty(6 * (cols + 7) + 3, device="cuda", dtype=dtype) for _ in range(2)]  # the gradients beside 32 bytes, so that every kernel has its turn
    for places in (None, [o.as_strided((6, cols), (cols + 7, 1), 3) for o in odd]):
        back = CheckpointedActivationBackward(KINDS[kind]).stamp(grad, forward.checkpoint, forward.gate_checkpoint, *(places or ()))
        back.run()
        xk, gk = (unpack64(c.codes, c.scales, cols) for c in (forward.checkpoint, forward.gate_checkpoint))
        value, slope, size = activation64(xk.clamp(-2.0**128, 2.0**128), kind)
        g = grad.double()
        for got, want, scale in ((back.grad_input, g * gk * slope, (g * gk * size).abs()), (back.grad_gate, g * value, (g * value).abs())):
            assert not torch.isnan(got).any()
            ok = ((got.double() - want).abs() <= (40 * F32 + 2.0**-17 + 1.01 * HALF_ULP[dtype]) * scale + torch.finfo(dtype).tiny * torch.finfo(dtype).eps)
            assert (ok | (torch.isinf(got) & (want.abs() > torch.finfo(dtype).max * (1 - 2.0**-8)) & (got.sign() == want.sign()))).all()


def test_the_unpacked_lowest_number_is_infinite():
    """What CheckpointUnpack says of such a code."""
    x = torch.full((1, 32), torch.finfo(torch.bfloat16).min, device="cuda", dtype=torch.bfloat16)
    forward = CheckpointedActivation(Kind.Swish).stamp(x)
    assert not forward.run().any()
    assert (CheckpointUnpack(DataType.fp32).stamp(forward.checkpoint).run() == -math.inf).all()
