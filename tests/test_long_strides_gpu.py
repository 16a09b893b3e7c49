"""Elements past 2^32: rows far apart in one buffer, and dense tensors of more than 2^32 elements, in every kernel that reads or writes checkpoints."""
import pytest
import torch

from _layers64 import pack64, unpack64
from thor_b200 import DataType
from thor_b200.activation import CheckpointedActivation, CheckpointedActivationBackward, CheckpointedActivationKind as Kind
from thor_b200.checkpoint import ActivationCheckpoint, CheckpointPack, CheckpointUnpack
from thor_b200.normalization import LayerNorm, LayerNormBackward

pytestmark = pytest.mark.gpu
ROWS = 3


def room(gigabytes):
    if torch.cuda.mem_get_info()[0] < gigabytes << 30:
        pytest.skip(f"needs {gigabytes} GB")


@pytest.fixture(scope="module")
def far():
    """Three rows 2^31 elements and more apart: the last starts past 2^32.  far(i, cols, stride): tensor i of one buffer."""
    room(12)
    buffer = torch.zeros(2 * ((1 << 31) + 16) + (1 << 20), dtype=torch.bfloat16, device="cuda")
    yield lambda i, cols, odd: buffer.as_strided((ROWS, cols), ((1 << 31) + (1 if odd else 16), 1), i * 131072 + (3 if odd else 0))
    del buffer
    torch.cuda.empty_cache()


def fill(t, seed):
    t.copy_(torch.randn(t.shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)))
    return t


def same(a, b):
    return torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


@pytest.mark.parametrize("cols,odd", [(96, False), (4096, False), (97, True), (2049, True), (9001, True), (16400, False), (20001, True)])
def test_rows_far_apart(far, cols, odd):
    x, r, out, other, third = (far(i, cols, odd) for i in range(5))
    fill(x, 1), fill(r, 2)
    dense_x, dense_r = x.contiguous(), r.contiguous()
    ck = CheckpointPack().stamp(x).run()
    assert same(ck.codes, CheckpointPack().stamp(dense_x).run().codes)
    CheckpointUnpack().stamp(ck, out).run()
    assert same(out, CheckpointUnpack().stamp(ck).run())
    for kind in (Kind.Gelu, Kind.Swish):
        for gated in (False, True):
            a = CheckpointedActivation(kind).stamp(x, r if gated else None, output=out)
            b = CheckpointedActivation(kind).stamp(dense_x, dense_r if gated else None)
            assert same(a.run(), b.run()) and same(a.checkpoint.codes, b.checkpoint.codes)
            back = CheckpointedActivationBackward(kind)
            p = back.stamp(r, a.checkpoint, a.gate_checkpoint, grad_input=other, grad_gate=third if gated else None)
            q = back.stamp(dense_r, a.checkpoint, a.gate_checkpoint)
            assert same(p.run(), q.run()) and (not gated or same(p.grad_gate, q.grad_gate))
    gamma, beta = torch.randn(2, cols, device="cuda").bfloat16()
    gamma, beta = gamma.clone(), beta.clone()
    for code in (None, DataType.fp8_e4m3):
        a = LayerNorm(checkpoint_dtype=code).stamp(x, gamma, beta, residual=r, output=out)
        b = LayerNorm(checkpoint_dtype=code).stamp(dense_x, gamma, beta, residual=dense_r)
        assert same(a.run(), b.run()) and same(a.sum, b.sum) and same(a.rstd, b.rstd)
        kept = lambda far_x, plan: dict(checkpoint=plan.checkpoint) if code is not None else dict(x=far_x, mean=plan.mean)
        p = LayerNormBackward().stamp(r, a.rstd, gamma=gamma, grad_sum=x, **kept(x, a))
        q = LayerNormBackward().stamp(dense_r, a.rstd, gamma=gamma, grad_sum=dense_x, **kept(dense_x, a))
        assert same(p.run(), q.run()) and same(p.grad_gamma, q.grad_gamma) and same(p.grad_beta, q.grad_beta)


def test_more_than_2_to_32_elements():
    """Dense outputs (the sum, the input's gradient) and codes whose last rows lie past 2^32."""
    room(64)
    rows, cols, last = (1 << 28) + 21, 16, 40
    gen = torch.Generator(device="cuda").manual_seed(5)
    x = torch.zeros(rows, cols, dtype=torch.bfloat16, device="cuda")
    x[-last:] = torch.randn(last, cols, device="cuda", generator=gen).bfloat16()
    gamma = torch.linspace(0.5, 2, cols, device="cuda").bfloat16()
    whole = LayerNorm(checkpoint_dtype=DataType.int8).stamp(x, gamma, residual=x)
    part = LayerNorm(checkpoint_dtype=DataType.int8).stamp(x[-last:], gamma, residual=x[-last:])
    part.run()
    assert same(whole.run()[-last:], part.output) and same(whole.sum[-last:], part.sum) and same(whole.checkpoint.codes[-last:], part.checkpoint.codes)
    assert not whole.output[:-last:100003].any()
    rstd, ck = whole.rstd, whole.checkpoint
    del whole
    back = LayerNormBackward().stamp(x, rstd, gamma=gamma, checkpoint=ck, grad_sum=x)
    assert same(back.run()[-last:], LayerNormBackward().stamp(x[-last:], part.rstd, gamma=gamma, checkpoint=part.checkpoint, grad_sum=x[-last:]).run())
    assert not back.grad_input[:-last:100003].any()
    n = unpack64(part.checkpoint.codes, part.checkpoint.scales, cols)
    want = (n * x[-last:].double()).sum(0)  # every other row's gradient is zero
    assert ((back.grad_gamma.double() - want).abs() <= 2.0**-8 * want.abs() + 2.0**-18 * (n * x[-last:].double()).abs().sum(0)).all()
