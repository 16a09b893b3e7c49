"""Swish where sigma(x) passes below the smallest normal number (x < -87.3), but x sigma(x) and the slope do not.

Allowed relative error in 16-bit types: half a unit of the type and 2^-16.  The exponent's argument is at most 134 in magnitude (x = -92.5): its rounding and that of
log2 e before it are below 2^-17 + 2e-6 of an exponent, 6.7e-6 of the result with ln 2; the instructions add less than 2^-20, the second rounding of half a unit to
itself less than 2^-16 - 2^-17.  A subnormal sigma is off by up to 3 steps of 2^-149 (fp32: two of the exponential and one of the product) and its results by (1 + |x|)
as much."""
import pytest
import torch

from _layers64 import HALF_ULP, activation64, unpack64
from thor_b200 import DataType
from thor_b200.activation import CheckpointedActivation, CheckpointedActivationBackward, CheckpointedActivationKind as Kind

pytestmark = pytest.mark.gpu
SMALLEST = {torch.float32: 2.0**-149, torch.bfloat16: 2.0**-133, torch.float16: 2.0**-24}


def tensors(dtype, rows, cols, start):
    """x: integers from 0 down to -126, which int8 codes keep as they are where a block holds one below -63."""
    at = torch.arange(rows * cols, device="cuda").reshape(rows, cols) % 127
    stride = cols + (3 if start else 0)
    x, gate, grad = (torch.empty(start + rows * stride, device="cuda", dtype=dtype).as_strided((rows, cols), (stride, 1), start) for _ in range(3))
    x.copy_(-at)
    gate.copy_((at % 5 + 1) / 4)
    grad.copy_(3 - at % 7)
    return x, gate, grad


def close(got, want, size, x, weight, dtype):
    return ((got.double() - want).abs() <= (2.0**-16 + HALF_ULP[dtype]) * size + 3 * (1 + x.abs()) * weight * 2.0**-149 + SMALLEST[dtype]).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("cols,start", [(32, 0), (97, 1), (2048, 0), (2049, 0), (2064, 5)])
def test_values_and_gradients(dtype, gated, cols, start):
    x, gate, grad = tensors(dtype, 40, cols, start)
    out, dx, dgate = tensors(dtype, 40, cols, start)
    forward = CheckpointedActivation(Kind.Swish, DataType.int8).stamp(x, gate if gated else None, output=out)
    forward.run()
    value, _, _ = activation64(x.double(), "swish")
    weight = gate.double() if gated else torch.ones_like(value)
    assert close(out, value * weight, (value * weight).abs(), x.double(), weight, dtype)
    xk = unpack64(forward.checkpoint.codes, forward.checkpoint.scales, cols)
    value, slope, size = activation64(xk, "swish")
    if gated:
        weight = unpack64(forward.gate_checkpoint.codes, forward.gate_checkpoint.scales, cols)
    CheckpointedActivationBackward(Kind.Swish).stamp(grad, forward.checkpoint, forward.gate_checkpoint, grad_input=dx, grad_gate=dgate if gated else None).run()
    g = grad.double()
    assert close(dx, g * weight * slope, (g * weight * size).abs(), xk, (g * weight).abs(), dtype)
    if gated:
        assert close(dgate, g * value, (g * value).abs(), xk, g.abs(), dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("at", [-88.0, -89.0, -91.0])
def test_places_that_an_approximation_would_flush(dtype, at):
    x = torch.full((1, 32), at, device="cuda", dtype=dtype)
    forward = CheckpointedActivation(Kind.Swish, DataType.int8).stamp(x)
    y = forward.run()
    value, slope, _ = activation64(x.double(), "swish")
    got = CheckpointedActivationBackward(Kind.Swish).stamp(torch.ones_like(x), forward.checkpoint).run()
    assert (unpack64(forward.checkpoint.codes, forward.checkpoint.scales, 32) == at).all()
    for a, b in ((y, value), (got, slope)):
        assert (b.abs() > 2.0**-126).all() and ((a.double() - b).abs() <= (2.0**-14 + HALF_ULP[dtype]) * b.abs()).all()
