"""Activation backward on long odd rows from every code type, against the definition."""
import pytest
import torch

from _layers64 import CODES, F32, activation64, activation_error, unpack64
from test_checkpointed_activation_gpu import close, values
from thor_b200.activation import CheckpointedActivation, CheckpointedActivationBackward, CheckpointedActivationKind as Kind
from thor_b200.dtypes import from_torch

pytestmark = pytest.mark.gpu
KINDS = {"gelu": Kind.Gelu, "swish": Kind.Swish}


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("gated", [False, True])
def test_long_odd_rows_of_every_code(code, dtype, kind, gated):
    """The kernel that walks odd rows on the tensor's own 32 bytes, against the definition: every code type, offsets and widths of both parities."""
    rows, cols = 7, 2083
    x, gate = (values(rows, cols, dtype, 40 + i) * torch.exp2(torch.arange(cols, device="cuda") // 32 % 5 - 2.0).to(dtype) for i in range(2))
    forward = CheckpointedActivation(KINDS[kind], from_torch(code)).stamp(x, gate if gated else None)
    forward.run()
    xk = unpack64(forward.checkpoint.codes, forward.checkpoint.scales, cols)
    gk = unpack64(forward.gate_checkpoint.codes, forward.gate_checkpoint.scales, cols) if gated else torch.ones_like(xk)
    value, slope, size = activation64(xk, kind)
    for start, width in ((0, cols), (5, cols + 2), (8, cols + 13)):
        grad, dx, dgate = (torch.zeros(start + rows * width, device="cuda", dtype=dtype).as_strided((rows, cols), (width, 1), start) for _ in range(3))
        grad.copy_(values(rows, cols, dtype, 42))
        CheckpointedActivationBackward(KINDS[kind]).stamp(grad, forward.checkpoint, forward.gate_checkpoint, grad_input=dx, grad_gate=dgate if gated else None).run()
        g = grad.double()
        close(dx, g * gk * slope, activation_error(xk, kind, dtype) + 4 * F32, dtype, (g * gk * size).abs(), factor=(1 + xk.abs()) * (g * gk).abs())
        if gated:
            close(dgate, g * value, activation_error(xk, kind, dtype) + 4 * F32, dtype, factor=(1 + xk.abs()) * g.abs())
