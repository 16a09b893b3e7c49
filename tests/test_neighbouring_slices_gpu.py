"""Inputs and outputs that are column slices of one buffer, side by side at odd places: a kernel may read the words at a slice's ends whole, its neighbour's elements
among them, and the next kernel, which is placed before the first has ended, reads what the first has written there."""
import pytest
import torch

from thor_b200 import DataType
from thor_b200.activation import CheckpointedActivation, CheckpointedActivationBackward, CheckpointedActivationKind as Kind
from thor_b200.checkpoint import CheckpointPack
from thor_b200.normalization import LayerNorm, LayerNormBackward

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,cols", [(600, 33), (600, 257), (400, 2051)])
def test_a_chain_of_kernels_over_one_buffer(rows, cols, dtype):
    buffer = torch.zeros(rows, 3 + 5 * cols, device="cuda", dtype=dtype)
    x, y, z, dy, dx = (buffer[:, 3 + i * cols:3 + (i + 1) * cols] for i in range(5))
    gamma = torch.linspace(0.5, 1.5, cols, device="cuda").to(dtype)
    act = CheckpointedActivation(Kind.Gelu).stamp(x, output=y)
    norm = LayerNorm(checkpoint_dtype=DataType.fp8_e4m3).stamp(y, gamma, output=z)
    pack = CheckpointPack().stamp(z)
    back = CheckpointedActivationBackward(Kind.Gelu).stamp(dy, act.checkpoint, grad_input=dx)
    norm_back = LayerNormBackward().stamp(dx, norm.rstd, gamma=gamma, checkpoint=norm.checkpoint)
    repack = CheckpointPack().stamp(dx)
    plans = (act, norm, pack, back, norm_back, repack)
    results = lambda: [y, z, dx, norm.rstd, norm_back.grad_input, norm_back.grad_gamma] + [c.codes.view(torch.uint8) for c in (act.checkpoint, norm.checkpoint, pack.checkpoint, repack.checkpoint)]
    for turn in range(30):
        gen = torch.Generator(device="cuda").manual_seed(turn)
        x.copy_(torch.randn(rows, cols, device="cuda", generator=gen))
        dy.copy_(torch.randn(rows, cols, device="cuda", generator=gen))
        torch.cuda.synchronize()
        for plan in plans:
            plan.run()
        torch.cuda.synchronize()
        together = [t.clone() for t in results()]
        for plan in plans:  # one at a time
            plan.run()
            torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(together, results())), turn
