"""GELU and Swish, plain and gated, that write checkpoints and read them back, against their 64-bit definitions and against differences."""
import math

import pytest
import torch

from _layers64 import CODES, F32, HALF_ULP, activation64, activation_error, pack64, unpack64
from thor_b200 import ThorB200InvalidArgument
from thor_b200.activation import CheckpointedActivation, CheckpointedActivationBackward, CheckpointedActivationKind as Kind
from thor_b200.checkpoint import ActivationCheckpoint, CheckpointPack
from thor_b200.dtypes import from_torch

pytestmark = pytest.mark.gpu
DTYPES = (torch.float32, torch.float16, torch.bfloat16)
KINDS = {"gelu": Kind.Gelu, "swish": Kind.Swish}
SHAPES = [(1, 1), (3, 9), (16, 64), (5, 96), (1, 4096), (65, 257), (128, 1000), (300, 33), (9, 2049)]


def close(got, want, relative, dtype, scale=None, factor=1.0):
    """|got - want| <= relative * scale + half a unit of the output's type (and of its smallest subnormal step).  The exponential is flushed
    to zero below 2^-126, which changes act(x) by less than |x| 2^-126 and act'(x) by less than (1 + |x|) 2^-126; `factor` is the largest number that
    these are multiplied with, 1 + |x| included."""
    got, scale = got.double(), want.abs() if scale is None else scale
    smallest = {torch.float32: 2.0**-149, torch.float16: 2.0**-24, torch.bfloat16: 2.0**-133}[dtype]
    error, allowed = (got - want).abs(), relative * scale * (1 + 2 * HALF_ULP[dtype]) + HALF_ULP[dtype] * want.abs() + smallest + factor * 2.0**-126
    if dtype == torch.float16:  # past 65504 the rounded result is an infinity
        error = torch.where(torch.isinf(got) & (want.abs() > 65504) & (got.sign() == want.sign()), 0.0, error)
    assert (error <= allowed).all(), (error - allowed).max().item()


def values(rows, cols, dtype, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return (3 * torch.randn(rows, cols, device="cuda", generator=gen)).to(dtype)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_forward_and_backward(rows, cols, dtype, gated, kind):
    code = CODES[(rows + cols) % 3]
    x, gate = values(rows, cols, dtype, 1), values(rows, cols, dtype, 2) if gated else None
    plan = CheckpointedActivation(KINDS[kind], from_torch(code)).stamp(x, gate)
    y = plan.run()
    value, _, _ = activation64(x.double(), kind)
    want = value * gate.double() if gated else value
    close(y, want, activation_error(x.double(), kind, x.dtype) + F32, dtype, factor=(1 + x.double().abs()) * (1 + (gate.double().abs() if gated else 0)))
    for ck, t in ((plan.checkpoint, x), (plan.gate_checkpoint, gate)):
        if t is not None:
            codes, scales = pack64(t.double(), code)
            assert torch.equal(ck.codes.double(), codes) and torch.equal(ck.scales.view(torch.uint8), scales)
    grad = values(rows, cols, dtype, 3)
    back = CheckpointedActivationBackward(KINDS[kind]).stamp(grad, plan.checkpoint, plan.gate_checkpoint)
    back.run()
    xk = unpack64(plan.checkpoint.codes, plan.checkpoint.scales, cols)
    gk = unpack64(plan.gate_checkpoint.codes, plan.gate_checkpoint.scales, cols) if gated else torch.ones_like(xk)
    value, slope, size = activation64(xk, kind)
    g = grad.double()
    close(back.grad_input, g * gk * slope, activation_error(xk, kind, x.dtype) + 4 * F32, dtype, (g * gk * size).abs(), factor=(1 + xk.abs()) * (g * gk).abs())
    if gated:
        close(back.grad_gate, g * value, activation_error(xk, kind, x.dtype) + 4 * F32, dtype, factor=(1 + xk.abs()) * g.abs())
    else:
        assert back.grad_gate is None


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("cols,width", [(2047, 2047), (2049, 2096), (4097, 4099), (2064, 2080)])
def test_backward_of_long_odd_rows(dtype, kind, gated, cols, width):
    """The same rows through tensors that all start at one place of 32 bytes, whichever it is, and through tensors that do not: the same bits, and
    nothing beside the rows is written.  (Aligned tensors of the next width that 16 divides give the values to compare with.)"""
    rows, padded = 19, (cols + 15) // 16 * 16
    x, gate, grad = (torch.zeros(rows, padded, device="cuda", dtype=dtype) for _ in range(3))
    for i, t in enumerate((x, gate, grad)):
        t[:, :cols] = values(rows, cols, dtype, 30 + i) * torch.exp2(torch.arange(cols, device="cuda") // 32 % 5 - 2.0).to(dtype)
    forward = CheckpointedActivation(KINDS[kind]).stamp(x, gate if gated else None)
    forward.run()
    plain = CheckpointedActivationBackward(KINDS[kind]).stamp(grad, forward.checkpoint, forward.gate_checkpoint)
    plain.run()
    kept = [ActivationCheckpoint(c.codes, c.scales, cols) if c is not None else None for c in (forward.checkpoint, forward.gate_checkpoint)]
    starts = [(s, s, s) for s in range(17)] + [(3, 4, 3), (3, 3, 4), (0, 16, 5)]
    for starts_of in starts:
        buffers = [torch.full((s + rows * width + 40,), 7.0, device="cuda", dtype=dtype) for s in starts_of]
        views = [b.as_strided((rows, cols), (width, 1), s) for b, s in zip(buffers, starts_of)]
        views[0].copy_(grad[:, :cols])
        CheckpointedActivationBackward(KINDS[kind]).stamp(views[0], *kept, grad_input=views[1], grad_gate=views[2] if gated else None).run()
        for b, s, want in zip(buffers[1:], starts_of[1:], (plain.grad_input, plain.grad_gate)):
            whole = torch.full_like(b, 7.0)
            if want is not None:
                whole.as_strided((rows, cols), (width, 1), s).copy_(want[:, :cols])
            assert torch.equal(b, whole), starts_of


@pytest.mark.parametrize("kind", KINDS)
def test_the_whole_range_of_the_function(kind):
    """From where the result underflows to where it is x itself, both signs; fp32 so that nothing is hidden by a rounding."""
    x = torch.cat([torch.linspace(-100, 100, 40001, device="cuda"), torch.logspace(-30, 30, 4096, device="cuda"), -torch.logspace(-30, 1, 4096, device="cuda")])
    x = x[:x.numel() // 32 * 32].reshape(-1, 32).contiguous()
    plan = CheckpointedActivation(KINDS[kind]).stamp(x)
    value, _, _ = activation64(x.double(), kind)
    floor = torch.full_like(value, 2.0**-126)  # what underflows in fp32 may be flushed to zero on the way
    error = (plan.run().double() - value).abs()
    assert (error <= (activation_error(x.double(), kind, x.dtype) + F32) * value.abs() + x.abs().double() * floor + floor).all()
    back = CheckpointedActivationBackward(KINDS[kind]).stamp(torch.ones_like(x), plan.checkpoint)
    xk = unpack64(plan.checkpoint.codes, plan.checkpoint.scales, 32)
    _, slope, size = activation64(xk, kind)
    error = (back.run().double() - slope).abs()
    assert (error <= (activation_error(xk, kind, x.dtype) + 4 * F32) * size + (1 + xk.abs()) * 2.0**-126).all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("gated", [False, True])
def test_gradients_against_differences(kind, gated):
    """The gradient of sum(c * act(x) * gate) by central differences of the 64-bit function at the unpacked values."""
    x, gate = values(4, 64, torch.float32, 5) * 0.5, values(4, 64, torch.float32, 6) if gated else None
    plan = CheckpointedActivation(KINDS[kind]).stamp(x, gate)
    plan.run()
    c = values(4, 64, torch.float32, 7)
    back = CheckpointedActivationBackward(KINDS[kind]).stamp(c, plan.checkpoint, plan.gate_checkpoint)
    back.run()
    xk = unpack64(plan.checkpoint.codes, plan.checkpoint.scales, 64)
    gk = unpack64(plan.gate_checkpoint.codes, plan.gate_checkpoint.scales, 64) if gated else torch.ones_like(xk)
    h = 2.0**-13  # third derivatives are below 2: the difference is off by h^2 / 3, and by 2^-52 / h of the values
    f = lambda v, g: c.double() * activation64(v, kind)[0] * g
    tolerance = (h * h + 2.0**-36) * (1 + c.double().abs() * (1 + gk.abs()) * (1 + xk.abs()))
    assert ((f(xk + h, gk) - f(xk - h, gk)) / (2 * h) - back.grad_input.double()).abs().le(tolerance + 32 * F32 * (c.double() * gk).abs() * 2).all()
    if gated:
        assert ((f(xk, gk + h) - f(xk, gk - h)) / (2 * h) - back.grad_gate.double()).abs().le(tolerance + 32 * F32 * (c.double() * xk).abs()).all()


def test_infinities_and_nan_reach_the_output_and_the_gradient():
    for kind in KINDS:
        x = torch.randn(4, 64, device="cuda")
        x[0, 3], x[1, 40], x[2, 0] = math.inf, math.nan, -math.inf
        plan = CheckpointedActivation(KINDS[kind]).stamp(x)
        y = plan.run()
        assert y[0, 3] == math.inf and torch.isnan(y[1, 40]) and torch.isnan(y[2, 0])  # -inf * 0, as the expression has it
        assert torch.isfinite(y).sum() == 4 * 64 - 3
        grad = CheckpointedActivationBackward(KINDS[kind]).stamp(torch.ones_like(x), plan.checkpoint).run()
        bad = torch.zeros_like(x, dtype=torch.bool)
        bad[0, :32] = bad[1, 32:] = bad[2, :32] = True
        assert torch.equal(torch.isnan(grad), bad)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cols", [64, 100, 33])
def test_halves_of_one_projection(dtype, cols):
    h = values(12, 2 * cols, dtype, 8).reshape(3, 4, 2 * cols)
    plan = CheckpointedActivation(Kind.Swish).stamp(h[..., :cols], h[..., cols:])
    apart = CheckpointedActivation(Kind.Swish).stamp(h[..., :cols].contiguous(), h[..., cols:].contiguous())
    assert torch.equal(plan.run(), apart.run())
    grad, grad_h = values(12, cols, dtype, 9).reshape(3, 4, cols), torch.full_like(h, 3.0)
    back = CheckpointedActivationBackward(Kind.Swish)
    back.stamp(grad, plan.checkpoint, plan.gate_checkpoint, grad_input=grad_h[..., :cols], grad_gate=grad_h[..., cols:]).run()
    other = back.stamp(grad, apart.checkpoint, apart.gate_checkpoint)
    other.run()
    assert torch.equal(grad_h, torch.cat([other.grad_input, other.grad_gate], -1))


def test_capture():
    x, gate = values(32, 96, torch.bfloat16, 10), values(32, 96, torch.bfloat16, 11)
    plan = CheckpointedActivation(Kind.Gelu).stamp(x, gate)
    back = CheckpointedActivationBackward(Kind.Gelu).stamp(values(32, 96, torch.bfloat16, 12), plan.checkpoint, plan.gate_checkpoint)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan.run()
        back.run()
    x.copy_(values(32, 96, torch.bfloat16, 13))
    graph.replay()
    replayed = [t.clone() for t in (plan.output, back.grad_input, back.grad_gate)]
    plan.run()
    back.run()
    assert all(torch.equal(a, b) for a, b in zip(replayed, (plan.output, back.grad_input, back.grad_gate)))


def test_no_rows_and_refusals():
    empty = torch.empty(0, 64, device="cuda")
    plan = CheckpointedActivation(Kind.Gelu).stamp(empty)
    assert plan.run().shape == (0, 64) and CheckpointedActivationBackward(Kind.Gelu).stamp(empty, plan.checkpoint).run().shape == (0, 64)
    x = values(8, 64, torch.bfloat16, 1)
    act, back = CheckpointedActivation(Kind.Gelu), CheckpointedActivationBackward(Kind.Gelu)
    ck = CheckpointPack().stamp(x).run()

    def refused(make, text):
        with pytest.raises(ThorB200InvalidArgument, match=text):
            make()

    refused(lambda: act.stamp(x, x.float()), "gate must have")
    refused(lambda: act.stamp(x, x[:4]), "gate must have")
    refused(lambda: act.stamp(x, output=x), "output overlaps x")
    refused(lambda: act.stamp(x, x.clone(), checkpoint=ck, gate_checkpoint=ck), "overlaps")
    refused(lambda: act.stamp(x, gate_checkpoint=ck), "without a gate")
    refused(lambda: act.stamp(x, checkpoint=ActivationCheckpoint.allocate(8, 96)), "not \\[8, 64\\]")
    refused(lambda: back.stamp(x, ActivationCheckpoint.allocate(7, 64)), "not \\[8, 64\\]")
    refused(lambda: back.stamp(x, ck, grad_gate=x.clone()), "without the gate's checkpoint")
    refused(lambda: back.stamp(x, ck, grad_input=x), "overlaps")
    refused(lambda: back.stamp(x, ck, CheckpointPack(from_torch(torch.int8)).stamp(x).run()), "same code dtype")
    h = torch.empty(8, 128, dtype=torch.bfloat16, device="cuda")
    refused(lambda: back.stamp(x, ck, ck, grad_input=h[:, :64], grad_gate=h[:, 63:127]), "overlaps")
