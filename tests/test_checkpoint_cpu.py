"""Checkpoints, checkpointed activations and LayerNorm: what the library refuses, and the sizes it reports, without a GPU."""
import ctypes as C

import pytest
import torch

import thor_b200._native as native
from thor_b200 import DataType, ThorB200InvalidArgument
from thor_b200.activation import CheckpointedActivation, CheckpointedActivationKind, _ActivationDesc
from thor_b200.checkpoint import ActivationCheckpoint, CheckpointPack, CheckpointUnpack, _CheckpointDesc, code_pitch, scale_pitch
from thor_b200.normalization import LayerNorm, LayerNormBackward, _LayerNormDesc

lib = native.lib
BF16, E4M3 = int(DataType.bf16), int(DataType.fp8_e4m3)


def refused(status, text):
    assert status == 1
    with pytest.raises(ThorB200InvalidArgument, match=text):
        native.check(status)


def test_pitches():
    assert [code_pitch(c) for c in (1, 15, 16, 17, 4097)] == [16, 16, 16, 32, 4112]
    assert [scale_pitch(c) for c in (1, 32, 33, 4096, 4097)] == [1, 1, 2, 128, 129]


@pytest.mark.parametrize("change,text", [
    (dict(dtype=int(DataType.fp64)), "fp32, fp16 or bf16"), (dict(dtype=E4M3), "fp32, fp16 or bf16"), (dict(code_dtype=int(DataType.uint8)), "fp8_e4m3, fp8_e5m2 or int8"),
    (dict(cols=0), "columns"), (dict(cols=1 << 31), "columns"), (dict(stride=63), "row stride"), (dict(stride=-64), "row stride"), (dict(stride=1 << 32), "2\\^32"), (dict(rows=1 << 61), "overflows"),
    (dict(rows=1 << 32), "2\\^32 - 1 rows"),
])
def test_pack_and_unpack_descriptions(change, text):
    d = _CheckpointDesc(**{**dict(dtype=BF16, code_dtype=E4M3, rows=4, cols=64, stride=64), **change})
    refused(lib.thor_b200_checkpoint_pack_launch(C.byref(d), 16, 16, 16, None), text)
    refused(lib.thor_b200_checkpoint_unpack_launch(C.byref(d), 16, 16, 16, None), text)


def test_pack_pointers():
    d = _CheckpointDesc(BF16, E4M3, 4, 64, 64)
    refused(lib.thor_b200_checkpoint_pack_launch(None, 16, 16, 16, None), "null description")
    refused(lib.thor_b200_checkpoint_pack_launch(C.byref(d), None, 16, 16, None), "null tensor")
    refused(lib.thor_b200_checkpoint_pack_launch(C.byref(d), 16, None, 16, None), "null checkpoint")
    refused(lib.thor_b200_checkpoint_pack_launch(C.byref(d), 16, 24, 16, None), "16-byte aligned")
    refused(lib.thor_b200_checkpoint_unpack_launch(C.byref(d), 16, 16, None, None), "null tensor")
    d.rows = 0  # nothing to do, nothing is looked at
    native.check(lib.thor_b200_checkpoint_pack_launch(C.byref(d), None, None, None, None))
    native.check(lib.thor_b200_checkpoint_unpack_launch(C.byref(d), None, None, None, None))


@pytest.mark.parametrize("change,text", [
    (dict(kind=2), "unknown activation"), (dict(dtype=int(DataType.int8)), "fp32, fp16 or bf16"), (dict(code_dtype=0), "fp8_e4m3"), (dict(x_stride=1), "stride of x"),
    (dict(gate_stride=1), "stride of gate"), (dict(y_stride=1), "stride of y"), (dict(cols=0), "columns"), (dict(gate_stride=1 << 33), "2\\^32"),
])
def test_activation_descriptions(change, text):
    d = _ActivationDesc(**{**dict(kind=0, gated=1, dtype=BF16, code_dtype=E4M3, rows=4, cols=64, x_stride=128, gate_stride=128, y_stride=64), **change})
    refused(lib.thor_b200_checkpointed_activation_launch(C.byref(d), *([16] * 7), None), text)
    refused(lib.thor_b200_checkpointed_activation_backward_launch(C.byref(d), *([16] * 7), None), text)


def test_activation_pointers():
    d = _ActivationDesc(0, 1, BF16, E4M3, 4, 64, 64, 64, 64)
    for missing, text in ((0, "null tensor"), (1, "null tensor"), (2, "null tensor"), (3, "null checkpoint"), (4, "null checkpoint"), (5, "null checkpoint"), (6, "null checkpoint")):
        args = [16] * 7
        args[missing] = None
        refused(lib.thor_b200_checkpointed_activation_launch(C.byref(d), *args, None), text)
    for missing, text in ((0, "null tensor"), (1, "null checkpoint"), (2, "null checkpoint"), (3, "null checkpoint"), (4, "null checkpoint"), (5, "null tensor"), (6, "null tensor")):
        args = [16] * 7
        args[missing] = None
        refused(lib.thor_b200_checkpointed_activation_backward_launch(C.byref(d), *args, None), text)


def norm_desc(**change):
    return _LayerNormDesc(**{**dict(dtype=BF16, param_dtype=BF16, grad_param_dtype=BF16, code_dtype=0, eps=1e-5, reserved=0, rows=4, cols=64, x_stride=64, residual_stride=64,
                                    y_stride=64), **change})


@pytest.mark.parametrize("change,text", [
    (dict(dtype=E4M3), "tensors must be"), (dict(param_dtype=int(DataType.fp64)), "parameters must be"), (dict(code_dtype=int(DataType.uint8)), "codes must be"),
    (dict(reserved=1), "reserved"), (dict(cols=0), "columns"), (dict(rows=1 << 31), "rows"), (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"),
    (dict(x_stride=63), "stride of x"), (dict(y_stride=63), "row stride of"), (dict(x_stride=1 << 32), "2\\^32"),
])
def test_layernorm_descriptions(change, text):
    d = norm_desc(**change)
    refused(lib.thor_b200_layernorm_launch(C.byref(d), 16, None, 16, 16, 16, None, None, None, None, None, None), text)
    refused(lib.thor_b200_layernorm_backward_launch(C.byref(d), 16, 16, 16, 16, None, None, 16, None, 16, 16, 16, 16, 1 << 40, None), text)


def test_layernorm_pointers():
    fwd = lib.thor_b200_layernorm_launch
    d = norm_desc()
    refused(fwd(C.byref(d), None, None, 16, 16, 16, None, None, None, None, None, None), "null tensor")
    refused(fwd(C.byref(d), 16, None, 16, 16, 16, 16, None, None, None, None, None), "sum without residual")
    refused(fwd(C.byref(d), 16, None, 16, 16, 16, None, None, None, 16, 16, None), "code_dtype")
    refused(fwd(C.byref(norm_desc(code_dtype=E4M3)), 16, None, 16, 16, 16, None, None, None, 16, None, None), "code_dtype")
    refused(fwd(C.byref(norm_desc(code_dtype=E4M3)), 16, None, 16, 16, 16, None, None, None, 8, 16, None), "16-byte aligned")
    bwd = lib.thor_b200_layernorm_backward_launch
    refused(bwd(C.byref(d), 16, None, None, 16, None, None, 16, None, 16, 16, 16, 16, 1 << 30, None), "either the saved input")
    refused(bwd(C.byref(d), 16, 16, None, 16, None, None, 16, None, 16, 16, 16, 16, 1 << 30, None), "either the saved input")
    refused(bwd(C.byref(norm_desc(code_dtype=E4M3)), 16, 16, 16, 16, 16, 16, 16, None, 16, 16, 16, 16, 1 << 30, None), "either the saved input")
    refused(bwd(C.byref(d), 16, 16, 16, 16, None, None, 16, None, 16, 16, None, 16, 1 << 30, None), "go together")
    refused(bwd(C.byref(d), 16, 16, 16, 16, None, None, 16, None, 16, 16, 16, None, 0, None), "workspace of")
    refused(bwd(C.byref(d), 16, 16, 16, 16, None, None, 16, None, 16, 16, 16, 24, 1 << 30, None), "workspace of")
    refused(bwd(C.byref(d), 16, 16, 16, None, None, None, 16, None, 16, 16, 16, 16, 1 << 30, None), "null tensor")
    size = C.c_size_t()
    native.check(lib.thor_b200_layernorm_backward_workspace_bytes(C.byref(d), C.byref(size)))
    refused(bwd(C.byref(d), 16, 16, 16, 16, None, None, 16, None, 16, 16, 16, 16, size.value - 1, None), f"{size.value} bytes")


@pytest.mark.parametrize("rows,cols", [(0, 1), (1, 1), (7, 33), (4096, 4096), (32768, 8192), (1 << 20, 8), (3, 1 << 20)])
def test_backward_workspace_holds_two_partial_rows_per_slab_and_stays_small(rows, cols):
    size = C.c_size_t()
    native.check(lib.thor_b200_layernorm_backward_workspace_bytes(C.byref(norm_desc(rows=rows, cols=cols)), C.byref(size)))
    one = 2 * ((cols + 7) // 8 * 8) * 4
    few = rows <= 512 and cols <= 8192  # one launch, no partial rows
    assert size.value == 16 if few else one <= size.value <= max(one, 64 << 20)


def test_python_refusals_without_a_gpu():
    x = torch.zeros(4, 64)
    for make in (lambda: CheckpointPack().stamp(x), lambda: LayerNorm().stamp(x), lambda: CheckpointedActivation(CheckpointedActivationKind.Gelu).stamp(x),
                 lambda: LayerNormBackward().stamp(x, x[:, 0])):
        with pytest.raises(ThorB200InvalidArgument, match="CUDA tensor"):
            make()
    for make, text in ((lambda: CheckpointPack(DataType.uint8), "codes must be"), (lambda: CheckpointUnpack(DataType.int8), "must be fp32"), (lambda: LayerNorm(eps=-1.0), "eps"),
                       (lambda: LayerNorm(checkpoint_dtype=DataType.fp8_e4m3, save_statistics=False), "saved statistics"), (lambda: LayerNormBackward(DataType.int8), "must be fp32"),
                       (lambda: ActivationCheckpoint(x, x, 64), "CUDA device")):
        with pytest.raises(ThorB200InvalidArgument, match=text):
            make()
    with pytest.raises(ValueError):
        CheckpointedActivation(2)


def test_pointers_off_their_elements():
    d = _CheckpointDesc(BF16, E4M3, 4, 64, 64)
    refused(lib.thor_b200_checkpoint_pack_launch(C.byref(d), 17, 16, 16, None), "not aligned to its elements")
    refused(lib.thor_b200_checkpoint_unpack_launch(C.byref(d), 16, 16, 17, None), "not aligned to its elements")
    a = _ActivationDesc(0, 1, int(DataType.fp32), E4M3, 4, 64, 64, 64, 64)
    for at in (0, 1, 2):
        args = [16] * 7
        args[at] = 18
        refused(lib.thor_b200_checkpointed_activation_launch(C.byref(a), *args, None), "not aligned to its elements")
    for at in (0, 5, 6):
        args = [16] * 7
        args[at] = 18
        refused(lib.thor_b200_checkpointed_activation_backward_launch(C.byref(a), *args, None), "not aligned to its elements")
    n = norm_desc(dtype=int(DataType.fp32), param_dtype=int(DataType.fp32), grad_param_dtype=int(DataType.fp32))
    for at in range(8):
        args = [16] * 8
        args[at] = 18
        refused(lib.thor_b200_layernorm_launch(C.byref(n), *args, None, None, None), "not aligned to its elements")
    for at in (0, 1, 2, 3, 6, 7, 8, 9, 10):
        args = [16, 16, 16, 16, None, None, 16, 16, 16, 16, 16]
        args[at] = 18
        refused(lib.thor_b200_layernorm_backward_launch(C.byref(n), *args, 16, 1 << 30, None), "not aligned to its elements")


def test_launch_counts():
    count = lib.thor_b200_layernorm_backward_launch_count
    assert [count(C.byref(norm_desc(rows=r, cols=c)), p) for r, c, p in ((4, 64, 0), (4, 64, 1), (513, 64, 0), (513, 64, 1), (512, 8192, 1), (513, 8192, 1), (4, 8193, 1),
                                                                         (4, 8193, 0))] == [1, 1, 1, 2, 1, 2, 3, 1]
    assert count(C.byref(norm_desc(rows=0)), 1) == 0 and count(None, 1) == 0
