"""NaN between the rows of every input, before the first and behind the last: the same bits as dense tensors give, and nothing written beside the outputs' rows."""
import pytest
import torch

from _layers64 import CODES
from thor_b200 import DataType
from thor_b200.activation import CheckpointedActivation, CheckpointedActivationBackward, CheckpointedActivationKind as Kind
from thor_b200.checkpoint import CheckpointPack, CheckpointUnpack
from thor_b200.dtypes import from_torch
from thor_b200.normalization import LayerNorm, LayerNormBackward

pytestmark = pytest.mark.gpu


def placed(rows, cols, dtype, start, gap, seed=None):
    """A view at `start` with `gap` elements between rows in a buffer of NaN (inputs: random values from `seed`) or of sevens (outputs)."""
    buffer = torch.full((start + rows * (cols + gap) + 40,), 7.0 if seed is None else float("nan"), device="cuda", dtype=dtype)
    view = buffer.as_strided((rows, cols), (cols + gap, 1), start)
    if seed is not None:
        view.copy_(torch.randn(rows, cols, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)))
    return buffer, view


def untouched(buffer, view):
    copy = buffer.clone()
    copy.as_strided(view.shape, view.stride(), view.storage_offset()).fill_(7.0)
    return bool((copy == 7.0).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,cols", [(70, 1), (70, 17), (600, 33), (40, 250), (30, 512), (20, 1001), (530, 1040), (9, 2050), (7, 8191), (5, 9000), (3, 20000)])
@pytest.mark.parametrize("start,gap", [(0, 16), (1, 3), (8, 24), (13, 1)])
def test_every_operator(rows, cols, dtype, start, gap):
    (_, x), (_, r), (_, d) = (placed(rows, cols, dtype, start + i % 2, gap, 10 + i) for i in range(3))
    dense_x, dense_r, dense_d = (t.contiguous() for t in (x, r, d))
    code = from_torch(CODES[(rows + cols + start) % 3])

    def same(a, b):
        assert torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))

    def same_checkpoint(a, b):
        same(a.codes, b.codes)
        same(a.scales, b.scales)

    ck = CheckpointPack(code).stamp(x).run()
    same_checkpoint(ck, CheckpointPack(code).stamp(dense_x).run())
    out, view = placed(rows, cols, dtype, start, gap)
    CheckpointUnpack(from_torch(dtype)).stamp(ck, view).run()
    same(view, CheckpointUnpack(from_torch(dtype)).stamp(ck).run())
    assert untouched(out, view)
    for kind in (Kind.Gelu, Kind.Swish):
        out, view = placed(rows, cols, dtype, start, gap)
        a = CheckpointedActivation(kind, code).stamp(x, r, output=view)
        b = CheckpointedActivation(kind, code).stamp(dense_x, dense_r)
        same(a.run(), b.run())
        same_checkpoint(a.checkpoint, b.checkpoint)
        same_checkpoint(a.gate_checkpoint, b.gate_checkpoint)
        assert untouched(out, view)
        (out, view), (gate_out, gate_view) = (placed(rows, cols, dtype, start, gap) for _ in range(2))
        CheckpointedActivationBackward(kind).stamp(d, a.checkpoint, a.gate_checkpoint, grad_input=view, grad_gate=gate_view).run()
        q = CheckpointedActivationBackward(kind).stamp(dense_d, a.checkpoint, a.gate_checkpoint)
        same(q.run(), view)
        same(q.grad_gate, gate_view)
        assert untouched(out, view) and untouched(gate_out, gate_view)
    gamma, beta = (torch.linspace(a, b, cols, device="cuda").to(dtype) for a, b in ((0.5, 2), (-1, 1)))
    for keep in (None, code):
        out, view = placed(rows, cols, dtype, start, gap)
        a = LayerNorm(checkpoint_dtype=keep).stamp(x, gamma, beta, residual=r, output=view)
        b = LayerNorm(checkpoint_dtype=keep).stamp(dense_x, gamma, beta, residual=dense_r)
        same(a.run(), b.run())
        same(a.sum, b.sum)
        same(a.rstd, b.rstd)
        assert untouched(out, view)
        if keep is not None:
            same_checkpoint(a.checkpoint, b.checkpoint)
        saved = lambda t: dict(checkpoint=a.checkpoint) if keep is not None else dict(x=t, mean=a.mean)
        p = LayerNormBackward(DataType.fp32).stamp(d, a.rstd, gamma=gamma, grad_sum=r, **saved(x))
        q = LayerNormBackward(DataType.fp32).stamp(dense_d, a.rstd, gamma=gamma, grad_sum=dense_r, **saved(dense_x))
        same(p.run(), q.run())
        same(p.grad_gamma, q.grad_gamma)
        same(p.grad_beta, q.grad_beta)
