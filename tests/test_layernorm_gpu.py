"""LayerNorm forward and backward against the 64-bit definition, at lengths on both sides of those where the kernels change (a group of lanes up to 512
columns, whole warps above; loops above 16384 columns forward, 8192 backward).

Bounds.  A sum of n fp32 values in any order whose longest chain of additions is D has error at most D 2^-24 sum|v|; every sum here is taken
per thread, per row group and (column sums) per slab in turn, with D below 512 for the shapes tested."""
import pytest
import torch

from _layers64 import CODES, F32, HALF_ULP, LARGEST, blocks_of, layernorm64, layernorm_grads64, pack64, pitch, step_of, unpack64
from thor_b200 import DataType, ThorB200InvalidArgument
from thor_b200.checkpoint import ActivationCheckpoint, CheckpointPack
from thor_b200.dtypes import from_torch
from thor_b200.normalization import LayerNorm, LayerNormBackward

pytestmark = pytest.mark.gpu
# half the smallest subnormal step, which a rounding to the type may cost near zero
TINY = {torch.float32: 2.0**-150, torch.float16: 2.0**-25, torch.bfloat16: 2.0**-134}
DTYPES = (torch.float32, torch.float16, torch.bfloat16)
SHAPES = [(1, 8), (3, 31), (7, 64), (130, 33), (1000, 40), (64, 256), (5, 1000), (37, 1024), (9, 1025), (4, 1032), (33, 4096), (3, 4097), (2, 8192), (300, 2048), (1, 12345),
          (2, 16384), (3, 20000), (2, 32768), (1, 32769), (2, 40000)]
D = 512


def tensors(rows, cols, dtype, param, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed * 7919 + rows * 131 + cols)
    r = lambda *s: torch.randn(*s, device="cuda", generator=gen)
    x = (r(rows, cols) * (0.5 + torch.rand(rows, 1, device="cuda", generator=gen)) + 2 * r(rows, 1)).to(dtype)
    return x, r(rows, cols).to(dtype), (1 + 0.2 * r(cols)).to(param), (0.3 * r(cols)).to(param)


def normal_error(h, n, rstd, eps):
    """Bound of the fp32 error of the normalised values: the mean's error reaches all of them, the variance's scales them."""
    mean_error = D * F32 * h.abs().mean(1, keepdim=True) * rstd[:, None]
    return mean_error + (D + 8) * F32 * n.abs() + mean_error * mean_error * n.abs() + 4 * F32 * (n.abs() + h.abs().mean(1, keepdim=True) * rstd[:, None])


def assert_codes(ck, n, error, code):
    """The checkpoint of values known to within `error`: a scale that one of the possible largest values calls for, and codes within half a step
    of the values plus that error."""
    rows, cols = n.shape
    s = ck.scales.float().double()
    top, slack = blocks_of(n).abs().amax(-1), blocks_of(error).amax(-1)
    assert (s * LARGEST[code] >= top - slack).all()
    assert ((s / 2 * LARGEST[code] <= top + slack) | (s == 2.0**-127)).all()
    unit = s.repeat_interleave(32, 1)[:, :cols]
    value = unpack64(ck.codes, ck.scales, cols)
    assert ((value - n).abs() <= 0.5 * step_of((n.abs() + error) / unit, code) * unit + error).all()
    assert not ck.codes[:, cols:].view(torch.uint8).any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", SHAPES)
@pytest.mark.parametrize("residual", [False, True])
def test_forward(rows, cols, dtype, residual):
    eps = 1e-5
    param = torch.float32 if (rows + cols) % 2 else dtype
    code = CODES[(rows + cols) % 3]
    x, r, gamma, beta = tensors(rows, cols, dtype, param)
    h = x
    if residual:
        h = (x.float() + r.float()).to(dtype)
    mean, rstd, n, y = layernorm64(h.double(), gamma.double(), beta.double(), eps)
    error = normal_error(h.double(), n, rstd, eps)
    for keep in (None, from_torch(code)):
        plan = LayerNorm(eps, keep).stamp(x, gamma, beta, residual=r if residual else None)
        got = plan.run().double()
        assert ((got - y).abs() <= gamma.double().abs() * error + 4 * F32 * (n * gamma.double()).abs() + 2 * F32 * beta.double().abs() + HALF_ULP[dtype] * 1.01 * y.abs() + TINY[dtype]).all()
        assert ((plan.rstd.double() - rstd).abs() <= rstd * (D + 8) * F32 + rstd**3 * (D * F32 * h.double().abs().mean(1))**2).all()
        if residual:
            assert torch.equal(plan.sum, h)
        else:
            assert plan.sum is None
        if keep is None:
            assert plan.checkpoint is None and ((plan.mean.double() - mean).abs() <= (D + 2) * F32 * h.double().abs().mean(1)).all()
        else:
            assert plan.mean is None
            assert_codes(plan.checkpoint, n, error, code)
    quiet = LayerNorm(eps, save_statistics=False).stamp(x, gamma, beta, residual=r if residual else None)
    assert torch.equal(quiet.run(), plan.output) and quiet.rstd is None and quiet.mean is None


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", SHAPES)
@pytest.mark.parametrize("source", ["x", "e4m3", "int8"])
def test_backward(rows, cols, dtype, source):
    param = torch.float32 if (rows + cols) % 2 else dtype
    x, r, gamma, beta = tensors(rows, cols, dtype, param, 1)
    grad = tensors(rows, cols, dtype, param, 2)[1]
    forward = LayerNorm(1e-5, {"x": None, "e4m3": DataType.fp8_e4m3, "int8": DataType.int8}[source]).stamp(x, gamma, beta)
    forward.run()
    rstd = forward.rstd.double()
    if source == "x":
        n = (x.double() - forward.mean.double()[:, None]) * rstd[:, None]
        slip = 2 * F32 * n.abs() + F32 * (x.double().abs() + forward.mean.double().abs()[:, None]) * rstd[:, None]
        kept = dict(x=x, mean=forward.mean)
    else:
        n = unpack64(forward.checkpoint.codes, forward.checkpoint.scales, cols)
        slip = torch.zeros_like(n)
        kept = dict(checkpoint=forward.checkpoint)
    g = grad.double()
    dx, dg, db = layernorm_grads64(g, n, rstd, gamma.double())
    w = g * gamma.double()
    row1, row2 = w.abs().mean(1, keepdim=True), (w * n).abs().mean(1, keepdim=True)
    error = rstd[:, None] * (D * F32 * (row1 + n.abs() * row2) + n.abs() * (w.abs() * slip).mean(1, keepdim=True) + slip * row2 + 8 * F32 * (w.abs() + row1 + n.abs() * row2))
    for grad_sum in (None, r):
        plan = LayerNormBackward().stamp(grad, forward.rstd, gamma=gamma, grad_sum=grad_sum, **kept)
        plan.run()
        want = dx if grad_sum is None else dx + r.double()
        assert ((plan.grad_input.double() - want).abs() <= error + 4 * F32 * want.abs() + HALF_ULP[dtype] * 1.01 * want.abs() + TINY[dtype]).all()
        for got, exact, size, extra in ((plan.grad_gamma, dg, (g * n).abs().sum(0), (g.abs() * slip).sum(0)), (plan.grad_beta, db, g.abs().sum(0), 0.0)):
            assert got.dtype == param
            assert ((got.double() - exact).abs() <= (D + 2) * F32 * size + extra + HALF_ULP[param] * 1.01 * exact.abs() + TINY[param]).all()
    bare = LayerNormBackward().stamp(grad, forward.rstd, grad_sum=r, **kept)  # no gamma: weights of one, no parameter gradients
    assert bare.run().shape == x.shape and bare.grad_gamma is None and bare.kernel_launches == 1
    ones = LayerNormBackward().stamp(grad, forward.rstd, gamma=torch.ones(cols, device="cuda", dtype=dtype), grad_sum=r, **kept)
    assert torch.allclose(ones.run().float(), bare.grad_input.float(), rtol=4 * HALF_ULP[dtype], atol=1e-5)


def test_many_rows_and_their_column_sums():
    """Column sums of 20011 rows.  A chain of D additions, D the rows of a slab by one thread plus the slabs: below 512 still."""
    for rows, cols, dtype in ((20011, 256, torch.bfloat16), (20011, 72, torch.float32), (5003, 2056, torch.bfloat16)):
        x, _, gamma, beta = tensors(rows, cols, dtype, torch.float32, 3)
        grad = tensors(rows, cols, dtype, torch.float32, 4)[1]
        forward = LayerNorm(checkpoint_dtype=DataType.fp8_e4m3).stamp(x, gamma, beta)
        forward.run()
        plan = LayerNormBackward().stamp(grad, forward.rstd, gamma=gamma, checkpoint=forward.checkpoint)
        plan.run()
        n = unpack64(forward.checkpoint.codes, forward.checkpoint.scales, cols)
        g = grad.double()
        for got, want, size in ((plan.grad_gamma, (g * n).sum(0), (g * n).abs().sum(0)), (plan.grad_beta, g.sum(0), g.abs().sum(0))):
            assert ((got.double() - want).abs() <= (D + 2) * F32 * size + F32 * want.abs()).all()
        first = [t.clone() for t in (plan.grad_input, plan.grad_gamma, plan.grad_beta)]
        plan.run()
        assert all(torch.equal(a, b) for a, b in zip(first, (plan.grad_input, plan.grad_gamma, plan.grad_beta)))  # a fixed order


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", [(513, 16), (1201, 33), (613, 500), (2001, 1024), (700, 1032), (601, 3008), (513, 4095), (519, 4112), (741, 5001), (741, 5120), (889, 6144), (520, 6160),
                                       (513, 8191), (600, 8192), (513, 8208), (515, 9001)])
@pytest.mark.parametrize("source", ["x", "e4m3", "e5m2"])
def test_backward_of_many_rows(rows, cols, dtype, source):
    """More rows than one launch takes: teams that walk several rows one at a time or two at once, with a last turn that not every team has a row
    for, partial rows and their fold.  A column's sum is a chain of at most 2001 / 148 + 512 / 2 teams + 148 / 8 + 8 additions: below 512."""
    x, r, gamma, beta = tensors(rows, cols, dtype, torch.float32, 5)
    grad = tensors(rows, cols, dtype, torch.float32, 6)[1]
    forward = LayerNorm(1e-5, {"x": None, "e4m3": DataType.fp8_e4m3, "e5m2": DataType.fp8_e5m2}[source]).stamp(x, gamma, beta)
    forward.run()
    rstd = forward.rstd.double()
    if source == "x":
        n = (x.double() - forward.mean.double()[:, None]) * rstd[:, None]
        slip = 2 * F32 * n.abs() + F32 * (x.double().abs() + forward.mean.double().abs()[:, None]) * rstd[:, None]
        kept = dict(x=x, mean=forward.mean)
    else:
        n = unpack64(forward.checkpoint.codes, forward.checkpoint.scales, cols)
        slip = torch.zeros_like(n)
        kept = dict(checkpoint=forward.checkpoint)
    g = grad.double()
    dx, dg, db = layernorm_grads64(g, n, rstd, gamma.double())
    w = g * gamma.double()
    row1, row2 = w.abs().mean(1, keepdim=True), (w * n).abs().mean(1, keepdim=True)
    error = rstd[:, None] * (D * F32 * (row1 + n.abs() * row2) + n.abs() * (w.abs() * slip).mean(1, keepdim=True) + slip * row2 + 8 * F32 * (w.abs() + row1 + n.abs() * row2))
    for grad_sum in (None, r):
        plan = LayerNormBackward().stamp(grad, forward.rstd, gamma=gamma, grad_sum=grad_sum, **kept)
        plan.run()
        want = dx if grad_sum is None else dx + r.double()
        assert ((plan.grad_input.double() - want).abs() <= error + 4 * F32 * want.abs() + HALF_ULP[dtype] * 1.01 * want.abs() + TINY[dtype]).all()
        for got, exact, size, extra in ((plan.grad_gamma, dg, (g * n).abs().sum(0), (g.abs() * slip).sum(0)), (plan.grad_beta, db, g.abs().sum(0), 0.0)):
            assert ((got.double() - exact).abs() <= (D + 2) * F32 * size + extra + F32 * exact.abs()).all()


def test_gradients_against_differences():
    """sum(c * layernorm(x)) by central differences of the 64-bit function, in x, gamma and beta."""
    rows, cols, eps = 3, 40, 1e-5
    x, _, gamma, beta = tensors(rows, cols, torch.float32, torch.float32, 5)
    c = tensors(rows, cols, torch.float32, torch.float32, 6)[1]
    forward = LayerNorm(eps).stamp(x, gamma, beta)
    forward.run()
    plan = LayerNormBackward().stamp(c, forward.rstd, gamma=gamma, x=x, mean=forward.mean)
    plan.run()
    h = 2.0**-14

    def loss(xx, gg, bb):
        return (c.double() * layernorm64(xx, gg, bb, eps)[3]).sum().item()

    X, G, B = x.double(), gamma.double(), beta.double()
    for tensor, got in ((X, plan.grad_input), (G, plan.grad_gamma), (B, plan.grad_beta)):
        flat = tensor.view(-1)
        for i in range(0, flat.numel(), 7):
            old = flat[i].item()
            flat[i] = old + h
            up = loss(X, G, B)
            flat[i] = old - h
            down = loss(X, G, B)
            flat[i] = old
            # h^2 / 6 times a third derivative (rstd^3 times sums of c: below 2^9 here), plus the fp32 gradient's own error
            assert abs((up - down) / (2 * h) - got.view(-1)[i].item()) <= 2.0**-19 + 2.0**-15 * abs(got.view(-1)[i].item())


def test_a_row_with_an_infinity_or_nan_stays_in_its_row():
    x, _, gamma, beta = tensors(6, 96, torch.float32, torch.float32, 7)
    x[1, 5], x[4, 90] = float("inf"), float("nan")
    forward = LayerNorm(checkpoint_dtype=DataType.fp8_e4m3).stamp(x, gamma, beta)
    y = forward.run()
    bad = torch.tensor([False, True, False, False, True, False], device="cuda")
    assert torch.isnan(y[bad]).all() and torch.isfinite(y[~bad]).all()
    assert (forward.checkpoint.scales.view(torch.uint8)[bad] == 255).all() and (forward.checkpoint.scales.view(torch.uint8)[~bad] != 255).all()
    plan = LayerNormBackward().stamp(torch.ones_like(x), forward.rstd, gamma=gamma, checkpoint=forward.checkpoint)
    dx = plan.run()
    assert torch.isnan(dx[bad]).all() and torch.isfinite(dx[~bad]).all() and torch.isnan(plan.grad_gamma).all() and torch.isfinite(plan.grad_beta).all()


def test_constant_rows():
    """Variance zero: with eps the normalised values are zero (up to the mean's rounding times 1 / sqrt(eps))."""
    for value in (0.0, 3.0):
        x = torch.full((4, 512), value, device="cuda")
        forward = LayerNorm(1e-5).stamp(x)
        assert torch.equal(forward.run(), torch.zeros_like(x)) and torch.allclose(forward.rstd, torch.full((4,), 1e-5**-0.5, device="cuda"), rtol=8 * F32)


def test_values_far_from_zero():
    """mean 1000, spread 1: the squared differences are taken from the mean, not from zero."""
    gen = torch.Generator(device="cuda").manual_seed(8)
    for cols in (500, 5000):
        x = 1000 + torch.randn(16, cols, device="cuda", generator=gen)
        forward = LayerNorm(0.0).stamp(x)
        mean, rstd, n, y = layernorm64(x.double(), torch.ones(cols, device="cuda").double(), torch.zeros(cols, device="cuda").double(), 0.0)
        # the mean is within 1000 D 2^-24 in theory; 24 units of 2^-24 * 1000 cover the log2(cols) levels and 32 values of a thread
        assert (forward.run().double() - y).abs().max() <= 64 * F32 * 1000 * rstd.max() + 1e-5


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("first,cols,width", [(0, 64, 96), (8, 1000, 1024), (3, 257, 300), (1, 2048, 2050)])
def test_column_slices_and_leading_axes(dtype, first, cols, width):
    full, res, gamma, beta = tensors(24, width, dtype, dtype, 9)
    cut = lambda t: t.reshape(4, 6, width)[:, :, first:first + cols]
    dense = lambda t: cut(t).contiguous()
    gamma, beta = gamma[:cols].contiguous(), beta[:cols].contiguous()
    op = LayerNorm(checkpoint_dtype=DataType.fp8_e4m3)
    a, b = op.stamp(cut(full), gamma, beta, residual=cut(res)), op.stamp(dense(full), gamma, beta, residual=dense(res))
    assert torch.equal(a.run(), b.run()) and torch.equal(a.sum, b.sum) and a.rstd.shape == (4, 6)
    assert torch.equal(a.checkpoint.codes.view(torch.uint8), b.checkpoint.codes.view(torch.uint8))
    wide = torch.full_like(full, 5.0)
    op.stamp(cut(full), gamma, beta, residual=cut(res), output=cut(wide)).run()
    assert torch.equal(cut(wide), a.output) and (wide[:, :first] == 5).all() and (wide[:, first + cols:] == 5).all()
    back = LayerNormBackward()
    p = back.stamp(cut(res), a.rstd, gamma=gamma, checkpoint=a.checkpoint, grad_sum=cut(full))
    q = back.stamp(dense(res), a.rstd, gamma=gamma, checkpoint=a.checkpoint, grad_sum=dense(full))
    assert torch.equal(p.run(), q.run()) and torch.equal(p.grad_gamma, q.grad_gamma) and torch.equal(p.grad_beta, q.grad_beta)
    mean = a.rstd.clone()
    p = back.stamp(cut(res), a.rstd, gamma=gamma, x=cut(full), mean=mean)
    q = back.stamp(dense(res), a.rstd, gamma=gamma, x=dense(full), mean=mean)
    assert torch.equal(p.run(), q.run()) and torch.equal(p.grad_gamma, q.grad_gamma)


def test_unaligned_parameters():
    x, _, gamma, beta = tensors(5, 96, torch.bfloat16, torch.bfloat16, 10)
    odd = torch.empty(2 * 96 + 2, dtype=torch.bfloat16, device="cuda")
    g, b = odd[1:97], odd[97:193]
    g.copy_(gamma)
    b.copy_(beta)
    assert torch.equal(LayerNorm().stamp(x, g, b).run(), LayerNorm().stamp(x, gamma, beta).run())


def test_shards_of_the_rows_add_up():
    """fp32 parameter gradients of two halves of the rows, added, against those of the whole (the order differs: D additions)."""
    x, _, gamma, beta = tensors(513, 640, torch.bfloat16, torch.bfloat16, 11)
    grad = tensors(513, 640, torch.bfloat16, torch.bfloat16, 12)[1]
    forward = LayerNorm(checkpoint_dtype=DataType.fp8_e4m3).stamp(x, gamma, beta)
    forward.run()
    op = LayerNormBackward(DataType.fp32)
    whole = op.stamp(grad, forward.rstd, gamma=gamma, checkpoint=forward.checkpoint)
    whole.run()
    assert whole.grad_gamma.data_ptr() + 640 * 4 == whole.grad_beta.data_ptr()  # one [2, cols] tensor: one allreduce
    parts = []
    for a, b in ((0, 200), (200, 513)):
        p = op.stamp(grad[a:b], forward.rstd[a:b], gamma=gamma, checkpoint=forward.checkpoint.row_range(a, b))
        assert torch.equal(p.run(), whole.grad_input[a:b])
        parts.append(p)
    n = unpack64(forward.checkpoint.codes, forward.checkpoint.scales, 640)
    g = grad.double()
    assert ((parts[0].grad_gamma + parts[1].grad_gamma - whole.grad_gamma).double().abs() <= 2 * D * F32 * (g * n).abs().sum(0)).all()
    assert ((parts[0].grad_beta + parts[1].grad_beta - whole.grad_beta).double().abs() <= 2 * D * F32 * g.abs().sum(0)).all()


def test_capture_streams_and_two_plans_at_once():
    x, r, gamma, beta = tensors(200, 512, torch.bfloat16, torch.float32, 13)
    grad = tensors(200, 512, torch.bfloat16, torch.float32, 14)[1]
    forward = LayerNorm(checkpoint_dtype=DataType.fp8_e4m3).stamp(x, gamma, beta, residual=r)
    forward.run()
    plan = LayerNormBackward().stamp(grad, forward.rstd, gamma=gamma, checkpoint=forward.checkpoint)
    plan.run()
    want = [t.clone() for t in (forward.output, plan.grad_input, plan.grad_gamma, plan.grad_beta)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        forward.run()
        plan.run()
    for t in (forward.output, plan.grad_input, plan.grad_gamma, plan.grad_beta, forward.rstd):
        t.zero_()
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(want, (forward.output, plan.grad_input, plan.grad_gamma, plan.grad_beta)))
    # two plans have workspaces of their own and may run at the same time
    plans = [LayerNormBackward().stamp(grad, forward.rstd, gamma=gamma, checkpoint=forward.checkpoint) for _ in range(2)]
    streams = [torch.cuda.Stream() for _ in plans]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(20):
        for p, s in zip(plans, streams):
            with torch.cuda.stream(s):
                p.run()
    torch.cuda.synchronize()
    for p in plans:
        assert all(torch.equal(a, b) for a, b in zip(want[1:], (p.grad_input, p.grad_gamma, p.grad_beta)))


def test_no_rows():
    x = torch.empty(0, 64, device="cuda")
    gamma = torch.ones(64, device="cuda")
    forward = LayerNorm(checkpoint_dtype=DataType.fp8_e4m3).stamp(x, gamma)
    assert forward.run().shape == (0, 64)
    plan = LayerNormBackward().stamp(x, forward.rstd, gamma=gamma, checkpoint=forward.checkpoint)
    plan.grad_gamma.fill_(1)
    plan.grad_beta.fill_(1)
    plan.run()
    assert not plan.grad_gamma.any() and not plan.grad_beta.any()


def test_refusals():
    x, r, gamma, beta = tensors(8, 64, torch.bfloat16, torch.bfloat16, 15)
    rstd = torch.ones(8, device="cuda")
    ck = CheckpointPack().stamp(x).run()
    norm, back = LayerNorm(), LayerNormBackward()

    def refused(make, text):
        with pytest.raises(ThorB200InvalidArgument, match=text):
            make()

    refused(lambda: norm.stamp(x, gamma[:32]), "gamma must be")
    refused(lambda: norm.stamp(x, gamma, beta.float()), "all of one dtype")
    refused(lambda: norm.stamp(x, gamma.double()), "fp32, fp16 or bf16")
    refused(lambda: norm.stamp(x, gamma, residual=r.float()), "residual must have")
    refused(lambda: norm.stamp(x, gamma, output=x), "overlaps x")
    refused(lambda: norm.stamp(x, gamma, checkpoint=ck), "without a checkpoint")
    refused(lambda: norm.stamp(x[:, ::2], gamma[:32]), "adjacent")
    refused(lambda: back.stamp(x, rstd, gamma=gamma), "either the checkpoint")
    refused(lambda: back.stamp(x, rstd, gamma=gamma, x=x), "either the checkpoint")
    refused(lambda: back.stamp(x, rstd, gamma=gamma, x=r, mean=rstd, checkpoint=ck), "either the checkpoint")
    refused(lambda: back.stamp(x, rstd[:4], gamma=gamma, checkpoint=ck), "rstd must be")
    refused(lambda: back.stamp(x, rstd.double(), gamma=gamma, checkpoint=ck), "rstd must be")
    refused(lambda: back.stamp(x, rstd, gamma=gamma, x=r, mean=rstd[:2]), "mean must be")
    refused(lambda: back.stamp(x, rstd, gamma=gamma, checkpoint=ActivationCheckpoint.allocate(8, 32)), "not \\[8, 64\\]")
    refused(lambda: back.stamp(x, rstd, gamma=gamma, checkpoint=ck, grad_sum=r[:4]), "grad_sum must have")
    refused(lambda: norm.stamp(x.cpu()), "CUDA tensor")
