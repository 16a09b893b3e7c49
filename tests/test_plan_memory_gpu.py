"""What a stamped plan writes and reads stays allocated while the plan lives, whatever becomes of its attributes."""
import gc

import pytest
import torch

from thor_b200 import DataType
from thor_b200.activation import CheckpointedActivation, CheckpointedActivationBackward, CheckpointedActivationKind as Kind
from thor_b200.checkpoint import CheckpointPack, CheckpointUnpack
from thor_b200.normalization import LayerNorm, LayerNormBackward

pytestmark = pytest.mark.gpu


def allocated(address):
    blocks = [b for segment in torch.cuda.memory_snapshot() for b in segment["blocks"] if b["address"] <= address < b["address"] + b["size"]]
    return len(blocks) == 1 and blocks[0]["state"] == "active_allocated"


def activation_backward():
    forward = CheckpointedActivation(Kind.Swish).stamp(torch.randn(64, 96, device="cuda"), torch.randn(64, 96, device="cuda"))
    return CheckpointedActivationBackward(Kind.Swish).stamp(torch.randn(64, 96, device="cuda"), forward.checkpoint, forward.gate_checkpoint)


def norm_backward():
    forward = LayerNorm(checkpoint_dtype=DataType.int8).stamp(torch.randn(600, 96, device="cuda"))
    return LayerNormBackward().stamp(torch.randn(600, 96, device="cuda"), forward.rstd, gamma=torch.ones(96, device="cuda"), checkpoint=forward.checkpoint)


@pytest.mark.parametrize("make,names", [
    (lambda: CheckpointPack().stamp(torch.randn(64, 96, device="cuda")), ("checkpoint",)),
    (lambda: CheckpointUnpack().stamp(CheckpointPack().stamp(torch.randn(64, 96, device="cuda")).run()), ("checkpoint", "output")),
    (lambda: CheckpointedActivation(Kind.Swish).stamp(torch.randn(64, 96, device="cuda"), torch.randn(64, 96, device="cuda")), ("output", "checkpoint", "gate_checkpoint")),
    (activation_backward, ("grad_input", "grad_gate")),
    (lambda: LayerNorm().stamp(torch.randn(64, 96, device="cuda"), residual=torch.randn(64, 96, device="cuda")), ("output", "sum", "mean", "rstd")),
    (lambda: LayerNorm(checkpoint_dtype=DataType.int8).stamp(torch.randn(64, 96, device="cuda")), ("output", "rstd", "checkpoint")),
    (norm_backward, ("grad_input", "grad_gamma", "grad_beta")),
])
def test_a_plan_keeps_what_its_attributes_name(make, names):
    plan, places = make(), []
    for name in names:
        value = getattr(plan, name)
        if name.endswith("checkpoint"):
            places += [value.codes.data_ptr(), value.scales.data_ptr()]
            value.codes = value.scales = None
        else:
            places.append(value.data_ptr())
        setattr(plan, name, None)
    del value
    gc.collect()
    assert all(allocated(p) for p in places)
    plan.run()
    torch.cuda.synchronize()
    del plan
    gc.collect()
    assert not any(allocated(p) for p in places)  # and no longer than the plan lives
