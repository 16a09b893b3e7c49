"""Packing and unpacking 8-bit checkpoints against the 64-bit definition.  Scaling by a power of two is exact, so codes and scales are
compared bit for bit, and an unpacked value is the exact product rounded once (exact in fp32)."""
import math

import pytest
import torch

from _layers64 import CODES, LARGEST, pack64, pitch, unpack64
from thor_b200 import DataType, ThorB200InvalidArgument
from thor_b200.checkpoint import ActivationCheckpoint, CheckpointPack, CheckpointUnpack
from thor_b200.dtypes import from_torch

pytestmark = pytest.mark.gpu
DTYPES = (torch.float32, torch.float16, torch.bfloat16)


def same(a, b):
    """Equal everywhere, NaN where the other is NaN."""
    return torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(torch.nan_to_num(a, 0.0, math.inf, -math.inf), torch.nan_to_num(b, 0.0, math.inf, -math.inf))


def assert_packed(ck, x, code):
    codes, scales = pack64(x.reshape(-1, x.shape[-1]).double(), code)
    assert ck.codes.shape == codes.shape and ck.scales.shape == scales.shape
    assert torch.equal(ck.scales.view(torch.uint8), scales)
    assert torch.equal(ck.codes.double(), codes)  # -0 and 0 are equal; padding is zero


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 7), (5, 8), (4, 24), (7, 31), (2, 32), (9, 33), (1, 4096), (130, 40), (33, 1000), (64, 1024), (17, 4097), (1000, 96)])
def test_round_trip(rows, cols, dtype, code):
    gen = torch.Generator(device="cuda").manual_seed(rows * 131 + cols)
    x = (torch.randn(rows, cols, device="cuda", generator=gen) * torch.exp(3 * torch.randn(rows, 1, device="cuda", generator=gen))).to(dtype)
    pack = CheckpointPack(from_torch(code)).stamp(x)
    pack.checkpoint.codes.view(torch.uint8).fill_(0x55)  # whatever was there is overwritten, the padding included
    ck = pack.run()
    assert_packed(ck, x, code)
    want = unpack64(ck.codes, ck.scales, cols)
    for out in DTYPES:
        assert same(CheckpointUnpack(from_torch(out)).stamp(ck).run(), want.to(out))  # NaN where an fp16 input overflowed
    # a code is off by at most half a step: 2^-4 of the value (e4m3) or 2^-3 (e5m2) where it is normal, half a unit of the scale's grid below
    # that (2^-10 and 2^-17 of the scale) and for int8 (1 / 2)
    relative, absolute = {torch.float8_e4m3fn: (2.0**-4, 2.0**-10), torch.float8_e5m2: (2.0**-3, 2.0**-17), torch.int8: (0.0, 0.5)}[code]
    unit = ck.scales.float().double().repeat_interleave(32, 1)[:, :cols]
    whole = ~torch.isnan(want)
    assert ((want - x.double()).abs() <= torch.maximum(relative * x.double().abs(), absolute * unit))[whole].all()


@pytest.mark.parametrize("code", CODES)
def test_every_bf16_value_alone_in_its_block(code):
    """All 65536 bit patterns of bf16 as the largest value of a block: thresholds, subnormals, infinities, NaN."""
    x = torch.zeros(65536, 32, device="cuda")
    patterns = torch.arange(65536, device="cuda", dtype=torch.int32)
    x[:, 5] = (patterns << 16).view(torch.float32)
    x = x.bfloat16()
    finite = torch.isfinite(x[:, 5].float())
    ck = CheckpointPack(from_torch(code)).stamp(x).run()
    assert_packed(ck, x, code)
    assert (ck.scales.view(torch.uint8)[~finite] == 255).all()
    back = CheckpointUnpack(DataType.fp32).stamp(ck).run()
    # the codes above the largest finite one by half a step stand for 2^128, an infinity in fp32: bf16 values above 1.75 * 2^127 reach it
    inside = x[:, 5].float().abs() <= 1.75 * 2.0**127
    assert torch.isnan(back[~finite]).all() and torch.isfinite(back[inside]).all() and not torch.isnan(back[finite]).any()


def test_ties_and_thresholds_of_the_scale():
    """Just at and just above M * 2^k the scale doubles; codes at midpoints go to the even neighbour."""
    for code in CODES:
        m = LARGEST[code]
        rows = []
        for k in (-20, 0, 3):
            for v in (m, math.nextafter(m, 0), m * (1 + 2.0**-23), m * (1 - 2.0**-22), 1.0, 2.0 - 2.0**-23, 1.0 + 2.0**-23):
                row = torch.zeros(32, dtype=torch.float64)
                row[0] = v * 2.0**k
                row[1:] = torch.linspace(-1, 1, 31, dtype=torch.float64) * v * 2.0**k
                row[2] = 0.5 * 2.0**k
                row[3], row[4] = 17 / 16 * 2.0**k, 19 / 16 * 2.0**k  # midpoints of e4m3
                rows.append(row.clamp(-row[0], row[0]))
        x = torch.stack(rows).float().cuda()
        assert_packed(CheckpointPack(from_torch(code)).stamp(x).run(), x, code)


def test_a_broken_block_is_nan_and_its_neighbours_are_not():
    x = torch.randn(8, 100, device="cuda")
    x[1, 40] = math.inf
    x[2, 99] = -math.inf
    x[3, 0] = math.nan
    for code in CODES:
        ck = CheckpointPack(from_torch(code)).stamp(x).run()
        assert_packed(ck, x, code)
        back = CheckpointUnpack(DataType.fp32).stamp(ck).run()
        bad = torch.zeros(8, 128, dtype=torch.bool, device="cuda")
        bad[1, 32:64] = bad[2, 96:] = bad[3, :32] = True
        assert torch.equal(torch.isnan(back), bad[:, :100])
    ck = ActivationCheckpoint.allocate(4, 40)  # a scale of 255 is NaN whatever the codes say
    ck.codes.view(torch.uint8).fill_(0x30)
    ck.scales.view(torch.uint8).fill_(255)
    assert torch.isnan(CheckpointUnpack(DataType.bf16).stamp(ck).run()).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("first,cols,width", [(0, 64, 80), (8, 96, 160), (3, 64, 100), (1, 33, 35), (16, 1000, 1024), (5, 257, 513)])
def test_column_slices_and_leading_axes(dtype, first, cols, width):
    gen = torch.Generator(device="cuda").manual_seed(cols)
    full = torch.randn(6, 5, width, device="cuda", generator=gen).to(dtype)
    x = full[:, :, first:first + cols]
    ck = CheckpointPack().stamp(x).run()
    assert (ck.rows, ck.cols) == (30, cols)
    assert_packed(ck, x, torch.float8_e4m3fn)
    target = torch.full_like(full, 7.0)
    CheckpointUnpack(from_torch(dtype)).stamp(ck, target[:, :, first:first + cols]).run()
    want = torch.full_like(full, 7.0)
    want[:, :, first:first + cols] = unpack64(ck.codes, ck.scales, cols).to(dtype).reshape(6, 5, cols)
    assert torch.equal(target, want)  # nothing beside the slice is written


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("cols,width", [(2033, 2049), (2047, 2047), (2048, 2065), (2049, 2096), (2064, 2081), (4097, 4097), (8193, 8195)])
def test_long_odd_rows(dtype, code, cols, width):
    """Rows that start at every place of 32 bytes in turn (odd widths), at one place (2096) and at every start of the first; each block has a magnitude
    of its own, so that a code with a neighbour's scale shows; nothing beside the rows is written."""
    gen = torch.Generator(device="cuda").manual_seed(cols)
    x = torch.randn(35, cols, device="cuda", generator=gen)
    x *= torch.exp2(torch.randint(-8, 8, (35, cols // 32 + 1), device="cuda", generator=gen).float()).repeat_interleave(32, 1)[:, :cols]
    ck = CheckpointPack(from_torch(code)).stamp(x).run()
    want = unpack64(ck.codes, ck.scales, cols).to(dtype)
    for start in range(18):
        buffer = torch.full((start + 35 * width + 40,), 7.0, device="cuda", dtype=dtype)
        whole = buffer.clone()
        CheckpointUnpack(from_torch(dtype)).stamp(ck, buffer.as_strided((35, cols), (width, 1), start)).run()
        whole.as_strided((35, cols), (width, 1), start).copy_(want)
        assert torch.equal(buffer, whole), start


def test_a_range_of_rows_is_a_checkpoint():
    x = torch.randn(50, 70, device="cuda").bfloat16()
    whole = CheckpointPack().stamp(x).run()
    part = CheckpointPack().stamp(x[10:23]).run()
    view = whole.row_range(10, 23)
    assert torch.equal(view.codes.view(torch.uint8), part.codes.view(torch.uint8)) and torch.equal(view.scales.view(torch.uint8), part.scales.view(torch.uint8))
    assert torch.equal(CheckpointUnpack().stamp(view).run(), CheckpointUnpack().stamp(whole).run()[10:23])


def test_packing_an_unpacked_checkpoint_gives_it_back():
    x = torch.randn(40, 128, device="cuda")
    for code in CODES:
        a = CheckpointPack(from_torch(code)).stamp(x).run()
        b = CheckpointPack(from_torch(code)).stamp(CheckpointUnpack(DataType.fp32).stamp(a).run()).run()
        va, vb = unpack64(a.codes, a.scales, 128), unpack64(b.codes, b.scales, 128)
        assert torch.equal(va, vb)


def test_offsets_past_32_bits():
    """More than 2^32 bytes of codes and of the tensor: rows behind that are read and written where they lie."""
    rows, cols = 33000, 131072 + 16
    free, _ = torch.cuda.mem_get_info()
    assert free > 40 << 30
    x = torch.zeros(rows, cols, dtype=torch.bfloat16, device="cuda")
    gen = torch.Generator(device="cuda").manual_seed(1)
    x[-3:] = torch.randn(3, cols, device="cuda", generator=gen).bfloat16()
    ck = CheckpointPack().stamp(x).run()
    assert not ck.codes[:-3:4099].view(torch.uint8).any()
    codes, scales = pack64(x[-3:].double(), torch.float8_e4m3fn)
    assert torch.equal(ck.codes[-3:].double(), codes) and torch.equal(ck.scales[-3:].view(torch.uint8), scales)
    x.fill_(1.0)
    CheckpointUnpack().stamp(ck, x).run()
    assert torch.equal(x[-3:], unpack64(codes, scales, cols).bfloat16()) and not x[:-3:4099].any()


def test_capture_and_streams():
    x = torch.randn(64, 200, device="cuda").bfloat16()
    pack = CheckpointPack().stamp(x)
    unpack = CheckpointUnpack().stamp(pack.checkpoint)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        pack.run()
        unpack.run()
    for seed in (1, 2):
        x.copy_(torch.randn(64, 200, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)))
        graph.replay()
        assert_packed(pack.checkpoint, x, torch.float8_e4m3fn)
        assert torch.equal(unpack.output, unpack64(pack.checkpoint.codes, pack.checkpoint.scales, 200).bfloat16())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for plan in (pack, CheckpointPack().stamp(x, stream=side)):  # the stream of the moment, and one given at stamp time
        plan.checkpoint.codes.view(torch.uint8).zero_()
        side.wait_stream(torch.cuda.current_stream())
        if plan is pack:
            with torch.cuda.stream(side):
                plan.run()
        else:
            plan.run()
        side.synchronize()
        assert_packed(plan.checkpoint, x, torch.float8_e4m3fn)


def test_no_rows():
    ck = CheckpointPack().stamp(torch.empty(0, 64, device="cuda")).run()
    assert (ck.rows, ck.cols) == (0, 64) and CheckpointUnpack().stamp(ck).run().shape == (0, 64)


def test_row_strides_past_32_bits_are_refused():
    x = torch.empty((1 << 32) + 16, dtype=torch.float16, device="cuda")
    with pytest.raises(ThorB200InvalidArgument, match="2\\^32 elements between rows"):
        CheckpointPack().stamp(x.as_strided((2, 16), (1 << 32, 1)))
    CheckpointPack().stamp(x.as_strided((2, 16), ((1 << 32) - 1, 1)))


def test_refusals():
    x = torch.randn(8, 64, device="cuda")
    ck = CheckpointPack().stamp(x).checkpoint

    def refused(make, text):
        with pytest.raises(ThorB200InvalidArgument, match=text):
            make()

    refused(lambda: CheckpointPack().stamp(x.double()), "fp32, fp16 or bf16")
    refused(lambda: CheckpointPack().stamp(x.to(torch.float8_e4m3fn)), "fp32, fp16 or bf16")
    refused(lambda: CheckpointPack().stamp(x[:, ::2]), "adjacent")
    refused(lambda: CheckpointPack().stamp(x.t()), "adjacent")
    refused(lambda: CheckpointPack().stamp(x[:1].expand(8, 64)), "overlap")
    refused(lambda: CheckpointPack().stamp(x.reshape(2, 4, 64)[:, :3]), "evenly spaced")
    refused(lambda: CheckpointPack().stamp(torch.empty(4, 0, device="cuda")), "at least one column")
    refused(lambda: CheckpointPack().stamp(x, ActivationCheckpoint.allocate(8, 65)), "not \\[8, 64\\]")
    refused(lambda: CheckpointPack(DataType.int8).stamp(x, ck), "codes, not int8")
    refused(lambda: CheckpointUnpack(DataType.fp32).stamp(ck, torch.empty(8, 16, device="cuda")), "not \\[8, 16\\]")
    refused(lambda: CheckpointUnpack(DataType.bf16).stamp(ck, x), "output must be bf16")
    refused(lambda: CheckpointUnpack().stamp(x), "ActivationCheckpoint")
    refused(lambda: ActivationCheckpoint(ck.codes, ck.scales, 63 - 16), "columns need")
    refused(lambda: ActivationCheckpoint(ck.codes, ck.scales[:4], 64), "columns need")
    refused(lambda: ActivationCheckpoint(ck.codes.view(torch.uint8), ck.scales, 64), "codes must be")
    refused(lambda: ActivationCheckpoint(ck.codes, ck.scales.float(), 64), "scales must be")
    shared = torch.zeros(8 * 16, device="cuda")
    refused(lambda: CheckpointPack().stamp(shared.reshape(8, 16), ActivationCheckpoint(shared.view(torch.float8_e4m3fn)[:128].reshape(8, 16), ck.scales[:, :1].contiguous(), 16)),
            "overlaps")


def test_more_rows_than_a_grid_dimension_holds():
    """Rows of 2048 columns and more have CTAs of their own up to 65535 rows; beyond that they share them."""
    rows, cols = 65536 + 3, 2050
    x = torch.randn(rows, cols, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3)).bfloat16()
    ck = CheckpointPack().stamp(x).run()
    for part in (slice(0, 5), slice(65530, rows)):
        codes, scales = pack64(x[part].double(), torch.float8_e4m3fn)
        assert torch.equal(ck.codes[part].double(), codes) and torch.equal(ck.scales[part].view(torch.uint8), scales)
    back = CheckpointUnpack().stamp(ck).run()
    assert torch.equal(back[-9:], unpack64(ck.codes[-9:], ck.scales[-9:], cols).bfloat16())


def test_more_chunks_than_32_bits_count():
    """2^31 + 5 rows of one column: two chunks a row, so their number passes 2^32."""
    rows = (1 << 31) + 5
    free, _ = torch.cuda.mem_get_info()
    if free < 60 << 30:
        pytest.skip("needs 60 GB")
    x = torch.zeros(rows, 1, dtype=torch.float16, device="cuda")
    x[-4:, 0] = torch.tensor([1.5, -3.0, 0.0, 100.0], dtype=torch.float16, device="cuda")
    ck = CheckpointPack().stamp(x).run()
    codes, scales = pack64(x[-4:].double(), torch.float8_e4m3fn)
    assert torch.equal(ck.codes[-4:].double(), codes) and torch.equal(ck.scales[-4:].view(torch.uint8), scales)
    assert not ck.codes[-(1 << 20):-4].view(torch.uint8).any() and not ck.scales[-(1 << 20):-4].view(torch.uint8).any()
