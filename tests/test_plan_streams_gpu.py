"""A plan stamped for a stream owns memory of that stream: what is still pending on another one does not write into its outputs."""
import pytest
import torch

from thor_b200 import DataType
from thor_b200.activation import CheckpointedActivation, CheckpointedActivationBackward, CheckpointedActivationKind as Kind
from thor_b200.checkpoint import CheckpointPack, CheckpointUnpack
from thor_b200.normalization import LayerNorm, LayerNormBackward

pytestmark = pytest.mark.gpu


def owned(plan):
    for name in ("output", "sum", "mean", "rstd", "grad_input", "grad_gate", "grad_gamma", "grad_beta", "checkpoint", "gate_checkpoint"):
        value = getattr(plan, name, None)
        if value is not None:
            yield from (value.codes, value.scales) if name.endswith("checkpoint") else (value,)


def stream_of(tensor):
    """Stream of the caching allocator's segment that holds a tensor."""
    at = tensor.data_ptr()
    return next(s["stream"] for s in torch.cuda.memory_snapshot() if s["address"] <= at < s["address"] + s["total_size"])


def test_outputs_belong_to_the_stream_of_the_plan():
    x, r = torch.randn(600, 96, device="cuda"), torch.randn(600, 96, device="cuda")
    gamma = torch.ones(96, device="cuda")
    kept = CheckpointPack().stamp(x).run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    norm = LayerNorm(checkpoint_dtype=DataType.int8).stamp(x, gamma, residual=r, stream=side)
    made = [CheckpointPack().stamp(x, stream=side), CheckpointedActivation(Kind.Gelu).stamp(x, r, stream=side), norm, LayerNorm().stamp(x, gamma, stream=side)]
    backward = LayerNormBackward().stamp(r, norm.rstd, gamma=gamma, checkpoint=norm.checkpoint, stream=side)
    for plan in made + [CheckpointedActivationBackward(Kind.Gelu).stamp(r, kept, kept, stream=side), backward]:
        assert plan.run() is not None
        assert all(stream_of(t) == side.cuda_stream for t in owned(plan) if t is not kept.codes and t is not kept.scales)
    unpack = CheckpointUnpack().stamp(kept, stream=side)
    unpack.run()
    assert stream_of(unpack.output) == side.cuda_stream
    assert [stream_of(t) for t in backward._keep if isinstance(t, torch.Tensor) and t.dtype == torch.uint8] == [side.cuda_stream]  # the workspace
    torch.cuda.synchronize()


def test_pending_work_of_another_stream_leaves_the_outputs_alone():
    """A block freed on the current stream while that stream still writes it is not what a plan of another stream gets."""
    x = torch.randn(1 << 12, 1 << 12, device="cuda")
    want = LayerNorm().stamp(x).run().clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    torch.cuda.synchronize()
    pending = torch.empty_like(x)
    torch.cuda._sleep(200_000_000)  # a tenth of a second of spinning, then the write
    pending.fill_(7)
    del pending
    plan = LayerNorm().stamp(x, stream=side)
    plan.run()
    torch.cuda.synchronize()
    assert torch.equal(plan.output, want)
