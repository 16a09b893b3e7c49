"""The operators together, as a training step uses them: residual add and LayerNorm (normalised rows kept in 8 bits), a projection, the gated
activation (both factors kept in 8 bits), a projection back; then the backward pass from what was kept.  The products are torch's; every
operator's result is checked against its 64-bit definition on the inputs that it was given, and the gradient of the whole against that of
the block with the rounded intermediates put in, by 64-bit autograd."""
import pytest
import torch

from _layers64 import activation64, layernorm_grads64, unpack64
from thor_b200 import DataType, _native
from thor_b200.activation import CheckpointedActivation, CheckpointedActivationBackward, CheckpointedActivationKind as Kind
from thor_b200.checkpoint import ActivationCheckpoint, CheckpointPack, CheckpointUnpack
from thor_b200.normalization import LayerNorm, LayerNormBackward

pytestmark = pytest.mark.gpu
ROWS, COLS, INNER = 96, 256, 320


class Block:
    """One feed-forward block with static buffers, stamped once."""

    def __init__(self, dtype, code, kind):
        gen = torch.Generator(device="cuda").manual_seed(1)
        r = lambda *s, scale=1.0: (scale * torch.randn(*s, device="cuda", generator=gen)).to(dtype)
        self.x, self.residual, self.grad_out, self.grad_stream = r(ROWS, COLS), r(ROWS, COLS), r(ROWS, COLS, scale=0.1), r(ROWS, COLS, scale=0.1)
        self.gamma, self.beta = 1 + r(COLS, scale=0.1), r(COLS, scale=0.1)
        self.w1, self.w2 = r(COLS, 2 * INNER, scale=COLS**-0.5), r(INNER, COLS, scale=INNER**-0.5)
        self.norm = LayerNorm(checkpoint_dtype=code).stamp(self.x, self.gamma, self.beta, residual=self.residual)
        self.h = torch.empty(ROWS, 2 * INNER, dtype=dtype, device="cuda")
        self.act = CheckpointedActivation(kind, code).stamp(self.h[:, :INNER], self.h[:, INNER:])
        self.grad_a, self.grad_h = torch.empty(ROWS, INNER, dtype=dtype, device="cuda"), torch.empty(ROWS, 2 * INNER, dtype=dtype, device="cuda")
        self.act_back = CheckpointedActivationBackward(kind).stamp(self.grad_a, self.act.checkpoint, self.act.gate_checkpoint, grad_input=self.grad_h[:, :INNER],
                                                                   grad_gate=self.grad_h[:, INNER:])
        self.grad_y = torch.empty(ROWS, COLS, dtype=dtype, device="cuda")
        self.norm_back = LayerNormBackward(DataType.fp32).stamp(self.grad_y, self.norm.rstd, gamma=self.gamma, checkpoint=self.norm.checkpoint, grad_sum=self.grad_stream)

    def step(self):
        self.norm.run()
        torch.matmul(self.norm.output, self.w1, out=self.h)
        self.act.run()
        out = torch.matmul(self.act.output, self.w2)
        torch.matmul(self.grad_out, self.w2.t(), out=self.grad_a)
        self.act_back.run()
        torch.matmul(self.grad_h, self.w1.t(), out=self.grad_y)
        self.norm_back.run()
        return out

    def results(self):
        return [self.norm.output, self.norm.sum, self.act.output, self.grad_h, self.norm_back.grad_input, self.norm_back.grad_gamma, self.norm_back.grad_beta]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("code", [DataType.fp8_e4m3, DataType.int8])
@pytest.mark.parametrize("kind", [Kind.Gelu, Kind.Swish])
def test_one_step(dtype, code, kind):
    b = Block(dtype, code, kind)
    before = _native.lib.thor_b200_launch_count()
    b.step()
    torch.cuda.synchronize()
    assert _native.lib.thor_b200_launch_count() - before == 4  # one each
    name = "gelu" if kind == Kind.Gelu else "swish"
    # the backward chain in 64 bits, from the unpacked checkpoints; each operator's rounding to the tensors' type enters the next by its true value
    half = torch.finfo(dtype).eps / 2
    xk = unpack64(b.act.checkpoint.codes, b.act.checkpoint.scales, INNER)
    gk = unpack64(b.act.gate_checkpoint.codes, b.act.gate_checkpoint.scales, INNER)
    value, slope, size = activation64(xk, name)
    g = b.grad_a.double()
    want = torch.cat([g * gk * slope, g * value], 1)
    scale = torch.cat([(g * gk * size).abs(), (g * value).abs()], 1)
    assert ((b.grad_h.double() - want).abs() <= 2.0**-15 * scale + half * 1.01 * want.abs() + 2.0**-126).all()  # 2^-15: the bound of the activation's own test for |x| < 9
    n = unpack64(b.norm.checkpoint.codes, b.norm.checkpoint.scales, COLS)
    dx, dg, db = layernorm_grads64(b.grad_y.double(), n, b.norm.rstd.double(), b.gamma.double())
    dx = dx + b.grad_stream.double()
    assert ((b.norm_back.grad_input.double() - dx).abs() <= half * 1.01 * dx.abs() + 2.0**-15 * dx.abs().max()).all()  # sums of 256 fp32 terms: far below 2^-15
    for got, exact in ((b.norm_back.grad_gamma, dg), (b.norm_back.grad_beta, db)):
        assert ((got.double() - exact).abs() <= 2.0**-15 * exact.abs().max()).all()


@pytest.mark.parametrize("code,bits", [(DataType.fp8_e4m3, 2.0**-4), (DataType.int8, 2.0**-5)])
def test_the_whole_gradient_is_that_of_the_block_up_to_the_kept_bits(code, bits):
    """fp32 block against 64-bit autograd without any checkpoint: what differs is the rounding of the three kept values (x, gate, normalised rows).
    e4m3: an error of at most 2^-4 of a value, uniform within the step: 2^-4 / sqrt 3 in the mean square.  int8: at most half a unit, a unit is at most
    1 / 63.5 of the block's largest value, and the largest of 32 normal values is below 3.5 times their root mean square in the mean: 0.5 * 3.5 / 63.5
    / sqrt 3 = 0.016 < 2^-5 / sqrt 3.  Three independent ones: sqrt 3 times that, 2^-4 and 2^-5 of the gradient's norm.  A wrong sign, factor or
    operand is off by its whole norm."""
    b = Block(torch.float32, code, Kind.Swish)
    b.step()
    leaves = [t.double().detach().requires_grad_() for t in (b.x, b.gamma, b.beta)]
    x, gamma, beta = leaves
    s = x + b.residual.double()
    d = s - s.mean(1, keepdim=True)
    y = d / torch.sqrt((d * d).mean(1, keepdim=True) + 1e-5) * gamma + beta
    h = y @ b.w1.double()
    a = h[:, :INNER] * torch.sigmoid(h[:, :INNER]) * h[:, INNER:]
    loss = ((a @ b.w2.double()) * b.grad_out.double()).sum() + (s * b.grad_stream.double()).sum()
    loss.backward()
    for got, leaf in zip((b.norm_back.grad_input, b.norm_back.grad_gamma, b.norm_back.grad_beta), leaves):
        assert ((got.double() - leaf.grad).norm() <= bits * leaf.grad.norm()).item()


def test_captured_step_and_eager_step_agree_while_both_live():
    b = Block(torch.bfloat16, DataType.fp8_e4m3, Kind.Gelu)
    eager = Block(torch.bfloat16, DataType.fp8_e4m3, Kind.Gelu)
    b.step()  # torch's products choose their algorithms outside of the capture
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        b.step()
    for seed in (2, 3):
        fresh = torch.randn(ROWS, COLS, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)).bfloat16()
        b.x.copy_(fresh)
        eager.x.copy_(fresh)
        graph.replay()
        eager.step()
        torch.cuda.synchronize()
        for got, want in zip(b.results(), eager.results()):
            assert torch.equal(got, want)


def test_kept_tensor_between_steps_of_other_sizes():
    """Checkpoints of several sizes live at once and come back as what they were, whatever ran in between."""
    kept = []
    for rows, cols in ((7, 33), (128, 1000), (1, 8192), (300, 96)):
        x = torch.randn(rows, cols, device="cuda", generator=torch.Generator(device="cuda").manual_seed(cols))
        ck = CheckpointPack(DataType.int8).stamp(x).run()
        kept.append((ck, unpack64(ck.codes, ck.scales, cols).float()))
    Block(torch.bfloat16, DataType.fp8_e4m3, Kind.Swish).step()
    for ck, want in kept:
        assert torch.equal(CheckpointUnpack(DataType.fp32).stamp(ck).run(), want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,cols", [(5, 33), (9, 2049), (600, 1001), (3, 8193)])
def test_padding_is_not_read_and_a_broken_block_stays_a_block(dtype, rows, cols):
    """Whatever bytes lie in a checkpoint's padding, results are the same; a block whose scale is NaN gives NaN in its own columns only."""
    gen = torch.Generator(device="cuda").manual_seed(rows)
    x, grad = (torch.randn(rows, cols, device="cuda", generator=gen).to(dtype) for _ in range(2))
    gamma, rstd = 1 + 0.1 * torch.randn(cols, device="cuda", generator=gen), 1 + torch.rand(rows, device="cuda", generator=gen)
    for code in (DataType.fp8_e4m3, DataType.int8):
        clean = CheckpointPack(code).stamp(x).run()
        dirty = ActivationCheckpoint(clean.codes.clone(), clean.scales.clone(), cols)
        dirty.codes.view(torch.uint8)[:, cols:] = 0x7F  # NaN in e4m3, 127 in int8
        results = []
        for ck in (clean, dirty):
            norm = LayerNormBackward().stamp(grad, rstd, gamma=gamma, checkpoint=ck)
            act = CheckpointedActivationBackward(Kind.Gelu).stamp(grad, ck, ck)
            results.append([CheckpointUnpack(DataType.fp32).stamp(ck).run(), norm.run(), norm.grad_gamma, norm.grad_beta, act.run(), act.grad_gate])
        assert all(torch.equal(a, b) for a, b in zip(*results))
        block = (cols - 1) // 32 // 2
        dirty.scales.view(torch.uint8)[rows // 2, block] = 255
        broken = torch.zeros(rows, cols, dtype=torch.bool, device="cuda")
        broken[rows // 2, 32 * block:32 * block + 32] = True
        act = CheckpointedActivationBackward(Kind.Gelu).stamp(grad, dirty, dirty)
        act.run()
        for got, want in ((CheckpointUnpack(DataType.fp32).stamp(dirty).run(), results[0][0]), (act.grad_input, results[0][4]), (act.grad_gate, results[0][5])):
            assert torch.equal(torch.isnan(got), broken) and torch.equal(got[~broken], want[~broken])
        norm = LayerNormBackward().stamp(grad, rstd, gamma=gamma, checkpoint=dirty)
        got = norm.run()
        others = torch.arange(rows, device="cuda") != rows // 2
        assert torch.isnan(got[rows // 2]).all() and torch.equal(got[others], results[0][1][others])
        assert torch.equal(torch.isnan(norm.grad_gamma), broken[rows // 2]) and torch.equal(norm.grad_beta, results[0][3])
