"""LayerNorm forward where a team of threads takes several rows one after the other, and on both sides of the widths where its kernels change
(a group of lanes holds a row of up to 512 columns, a CTA's registers up to 8192 with one chunk of sixteen columns a thread and up to 16384 with
two; longer rows are looped over).

Bounds.  A row's sum is a tree: 4 levels in a thread's sixteen columns, 1 for its second chunk, 5 over the lanes, 4 or 5 over the warps; the loop adds a
chain of one step per 8192 columns (5 at 40000).  D = 24 covers each.  E = D + 4 units of the largest magnitude bound the error of a mean, of the
row or of one warp's columns; the variance is a sum of squares of differences from such means, so E (relative to the spread) enters once by the
difference and once squared."""
import pytest
import torch

from _layers64 import F32, HALF_ULP, LARGEST, blocks_of, layernorm64, step_of, unpack64
from thor_b200 import DataType
from thor_b200.normalization import LayerNorm

pytestmark = pytest.mark.gpu
D = 24
TINY = {torch.float32: 2.0**-150, torch.float16: 2.0**-25, torch.bfloat16: 2.0**-134}
# (rows, columns): every one more rows than the kernel has teams on 148 SMs, and twice as many for most
TURNS = [(200003, 8), (40009, 33), (20011, 72), (9001, 512), (5003, 513), (3001, 2056), (1501, 4096), (1501, 5001), (901, 8192), (601, 8193), (601, 12345), (601, 16384)]


def tensors(rows, cols, dtype, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed * 7919 + rows * 131 + cols)
    r = lambda *s: torch.randn(*s, device="cuda", generator=gen)
    x = (r(rows, cols) * (0.5 + torch.rand(rows, 1, device="cuda", generator=gen)) + 2 * r(rows, 1)).to(dtype)
    return x, r(rows, cols).to(dtype), (1 + 0.2 * r(cols)).to(dtype), (0.3 * r(cols)).to(dtype)


def bounds(h, n, rstd):
    """Errors allowed to mean, rstd (relative) and the normalised values."""
    largest = h.abs().amax(1)
    mean = (D + 2) * F32 * h.abs().mean(1)
    e = (D + 4) * F32 * largest * rstd
    scale = (D + 8) * F32 + e + e * e
    normal = (mean * rstd)[:, None] + n.abs() * (scale[:, None] + 3 * F32)
    return mean, scale, normal


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,cols", TURNS)
@pytest.mark.parametrize("residual", [False, True])
def test_forward_of_many_rows(rows, cols, dtype, residual):
    eps = 1e-5
    x, r, gamma, beta = tensors(rows, cols, dtype, 1)
    r = r if residual else None
    h = (x.float() + r.float()).to(dtype) if residual else x
    mean, rstd, n, y = layernorm64(h.double(), gamma.double(), beta.double(), eps)
    mean_error, scale_error, error = bounds(h.double(), n, rstd)
    saved = LayerNorm(eps).stamp(x, gamma, beta, residual=r)
    kept = LayerNorm(eps, DataType.fp8_e4m3).stamp(x, gamma, beta, residual=r)
    for plan in (saved, kept):
        got = plan.run().double()
        assert ((got - y).abs() <= gamma.double().abs() * error + 2 * F32 * (y.abs() + beta.double().abs()) + HALF_ULP[dtype] * 1.01 * y.abs() + TINY[dtype]).all()
        assert ((plan.rstd.double() - rstd).abs() <= rstd * scale_error).all()
        assert plan.sum is None if not residual else torch.equal(plan.sum, h)
    assert ((saved.mean.double() - mean).abs() <= mean_error).all()
    ck, code = kept.checkpoint, torch.float8_e4m3fn
    s, slack = ck.scales.float().double(), blocks_of(error).amax(-1)
    top = blocks_of(n).abs().amax(-1)
    assert (s * LARGEST[code] >= top - slack).all() and ((s / 2 * LARGEST[code] <= top + slack) | (s == 2.0**-127)).all()
    unit = s.repeat_interleave(32, 1)[:, :cols]
    assert ((unpack64(ck.codes, ck.scales, cols) - n).abs() <= 0.5 * step_of((n.abs() + error) / unit, code) * unit + error).all()
    assert not ck.codes[:, cols:].view(torch.uint8).any()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,cols", TURNS[2:])
@pytest.mark.parametrize("residual", [False, True])
def test_a_row_does_not_depend_on_the_rows_before_it(rows, cols, dtype, residual):
    """The same rows in launches of 100, one row a team: the same bits, whatever turn a row had."""
    x, r, gamma, beta = tensors(rows, cols, dtype, 2)
    whole = LayerNorm(checkpoint_dtype=DataType.int8).stamp(x, gamma, beta, residual=r if residual else None)
    whole.run()
    for first in (0, rows // 2 // 100 * 100, rows - 100):
        some = slice(first, first + 100)
        part = LayerNorm(checkpoint_dtype=DataType.int8).stamp(x[some], gamma, beta, residual=r[some] if residual else None)
        assert torch.equal(part.run(), whole.output[some]) and torch.equal(part.rstd, whole.rstd[some])
        assert torch.equal(part.checkpoint.codes, whole.checkpoint.codes[some])
        assert torch.equal(part.checkpoint.scales.view(torch.uint8), whole.checkpoint.scales[some].view(torch.uint8))
        if residual:
            assert torch.equal(part.sum, whole.sum[some])


@pytest.mark.parametrize("cols", [1, 2, 31, 32, 33, 511, 512, 513, 1024, 1025, 8191, 8192, 8193, 16384, 16385, 32768, 32769])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_whose_sums_are_exact(cols, dtype):
    """Neighbours of opposite sign, small integers: every mean is zero and every sum of squares an integer below 2^24, so what is left in rstd are the
    division (1 unit), the addition of eps (1 unit), halved by the root, and the root: half a unit from v * y in its Newton step and one from the last
    rounding.  2.5 units; 3 are allowed."""
    rows, eps = 700, 2.0**-20
    x = torch.zeros(rows, cols, device="cuda")
    pairs = torch.arange(cols // 2, device="cuda")
    for k in range(2):
        x[:, k:cols // 2 * 2:2] = ((pairs[None] + torch.arange(rows, device="cuda")[:, None]) % 7 + 1) * (1 - 2 * k)
    plan = LayerNorm(eps).stamp(x.to(dtype))
    plan.run()
    assert not plan.mean.any()
    want = 1 / torch.sqrt((x.double()**2).sum(1) / cols + eps)
    assert ((plan.rstd.double() - want).abs() <= 3 * F32 * want).all()
