"""Far to the right GELU and Swish are x itself, with slope 1: exactly, up to the largest number and for an infinite input."""
import math

import pytest
import torch

from thor_b200 import DataType
from thor_b200.activation import CheckpointedActivation, CheckpointedActivationBackward, CheckpointedActivationKind as Kind

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kind", [Kind.Gelu, Kind.Swish])
@pytest.mark.parametrize("cols", [32, 2049])
def test_the_function_is_its_argument(dtype, kind, cols):
    top = 16 if dtype == torch.float16 else 128
    x = torch.full((top - 5, cols), 1.0, device="cuda")
    x = (x * torch.exp2(torch.arange(5, top, device="cuda"))[:, None]).to(dtype)  # 32, 64, ..; one power of two a row
    x = torch.cat([x, torch.full((1, cols), torch.finfo(dtype).max, device="cuda", dtype=dtype)])
    grad = (3 - torch.arange(x.numel(), device="cuda").reshape(x.shape) % 7).to(dtype)
    forward = CheckpointedActivation(kind, DataType.fp8_e4m3).stamp(x)
    assert torch.equal(forward.run(), x)
    assert torch.equal(CheckpointedActivationBackward(kind).stamp(grad, forward.checkpoint).run(), grad)
    infinite = torch.full((2, 32), math.inf, device="cuda", dtype=dtype)
    assert torch.equal(CheckpointedActivation(kind).stamp(infinite).run(), infinite)
