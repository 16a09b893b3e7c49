"""8-bit activation checkpoints: packing a tensor for its backward pass and unpacking it (include/thor_b200.h).

An operator is described once, stamped on its tensors (checks, output allocation) and run as often as the step repeats; run()
is one call into the library on the stream given at stamp time or, without one, on the current stream, and allocates nothing, so it can be
captured into a CUDA graph.  A stamped operator owns its outputs and workspace, which belong to the stream given at stamp time or, without one, to the
one that was current then (a run on another stream is ordered behind that one by the caller, as for any tensor): two runs of one plan (direct or as replays of graphs that hold
it) must not overlap in time, and a plan must outlive the work and the graphs that use it; plans of the same operator are independent of one another."""
from __future__ import annotations

import contextlib
import ctypes as C
from typing import Optional

import torch

from . import _native
from .dtypes import DataType, from_torch, to_torch

_lib = _native.lib

BLOCK = 32  # columns that share a scale
CODE_DTYPES = (DataType.fp8_e4m3, DataType.fp8_e5m2, DataType.int8)
VALUE_DTYPES = (DataType.fp32, DataType.fp16, DataType.bf16)


class _CheckpointDesc(C.Structure):
    _fields_ = [("dtype", C.c_int32), ("code_dtype", C.c_int32), ("rows", C.c_uint64), ("cols", C.c_uint64), ("stride", C.c_int64)]


_lib.thor_b200_checkpoint_code_pitch.argtypes = [C.c_uint64]
_lib.thor_b200_checkpoint_code_pitch.restype = C.c_uint64
_lib.thor_b200_checkpoint_scale_pitch.argtypes = [C.c_uint64]
_lib.thor_b200_checkpoint_scale_pitch.restype = C.c_uint64
_lib.thor_b200_checkpoint_pack_launch.argtypes = [C.POINTER(_CheckpointDesc), C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p]
_lib.thor_b200_checkpoint_unpack_launch.argtypes = [C.POINTER(_CheckpointDesc), C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p]


def refuse(message: str):
    raise _native.ThorB200InvalidArgument(message)


def as_rows(t: torch.Tensor, what: str) -> tuple[int, int, int]:
    """(rows, cols, elements between rows) of a CUDA tensor whose last axis is dense and whose leading axes are one evenly spaced run of rows."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        refuse(f"{what} must be a CUDA tensor (no CPU path in this library)")
    if t.dtype not in (torch.float32, torch.float16, torch.bfloat16):
        refuse(f"{what} must be fp32, fp16 or bf16, got {t.dtype}")
    if t.dim() == 0 or t.shape[-1] == 0:
        refuse(f"{what} needs a last axis of at least one column")
    cols = t.shape[-1]
    rows = t.numel() // cols
    if rows == 0:
        return 0, cols, cols
    if cols > 1 and t.stride(-1) != 1:
        refuse(f"{what}: neighbouring columns must be adjacent in memory")
    lead = [(n, s) for n, s in zip(t.shape[:-1], t.stride()[:-1]) if n != 1]
    for (_, outer), (n, inner) in zip(lead, lead[1:]):
        if outer != inner * n:
            refuse(f"{what}: the leading axes must be one evenly spaced run of rows")
    stride = lead[-1][1] if lead else cols
    if rows > 1 and stride < cols:
        refuse(f"{what}: rows overlap (row stride {stride}, {cols} columns)")
    if cols >= 1 << 31 or rows >= 1 << 32 or (rows > 1 and stride >= 1 << 32):
        refuse(f"{what}: fewer than 2^31 columns, 2^32 rows and 2^32 elements between rows are taken")
    return rows, cols, stride


def same_rows(t: torch.Tensor, what: str, like: torch.Tensor) -> int:
    """The row stride of a tensor that must have another one's shape, dtype and device."""
    if t.shape != like.shape or t.dtype != like.dtype or t.device != like.device:
        refuse(f"{what} must have shape {tuple(like.shape)}, dtype {like.dtype} and device {like.device}")
    return as_rows(t, what)[2]


def _span(t: torch.Tensor) -> tuple[int, int]:
    if t.numel() == 0:
        return 0, 0
    last = sum((n - 1) * s for n, s in zip(t.shape, t.stride()))
    return t.data_ptr(), t.data_ptr() + (last + 1) * t.element_size()


def _disjoint(a: torch.Tensor, b: torch.Tensor) -> bool:
    (a0, a1), (b0, b1) = _span(a), _span(b)
    if a1 <= b0 or b1 <= a0:
        return True
    # two column slices of one buffer: rows of the same spacing, columns that do not meet
    lead = [i for i in range(a.dim() - 1) if a.shape[i] != 1]
    size, offset = a.element_size(), b0 - a0
    if not lead or a.shape[:-1] != b.shape[:-1] or a.dtype != b.dtype or offset % size or a.stride(-1) != 1 or b.stride(-1) != 1:
        return False
    spacing = a.stride(lead[-1])
    if any(a.stride(i) != b.stride(i) or a.stride(i) % spacing for i in lead):
        return False
    offset = offset // size % spacing
    return a.shape[-1] <= offset and offset + b.shape[-1] <= spacing


def check_outputs(outputs: dict, inputs: dict) -> None:
    """Refuses outputs that share memory with an input or with one another."""
    out = [(n, t) for n, t in outputs.items() if t is not None]
    for i, (name, t) in enumerate(out):
        for other, u in out[i + 1:] + [(n, u) for n, u in inputs.items() if u is not None]:
            if t.device == u.device and not _disjoint(t, u):
                refuse(f"{name} overlaps {other}")


def memory_of(stream):
    """Context in which a plan allocates what it owns: memory of the stream that it will run on, so that nothing still pending on another one uses it."""
    return torch.cuda.stream(stream) if stream is not None else contextlib.nullcontext()


class Stamped:
    """What the stamped operators share: run() is one call of `launch` with arguments resolved at stamp time (integers: the addresses of the
    description and of tensors, all of which `keep` keeps alive, outputs and the tensors of checkpoints among them) and the stream of the moment."""

    def __init__(self, launch, args: tuple, device: torch.device, stream, keep: tuple):
        # a function object of its own that takes every argument as a pointer-sized integer: the description's pointer type and the conversions cost 0.3 us a call
        self._launch = _lib[launch.__name__]
        self._launch.argtypes = [C.c_void_p] * (len(args) + 1)
        self._args, self._device = args, device.index if device.index is not None else torch.cuda.current_device()
        self._stream = stream
        self._keep = [(k.codes, k.scales) if isinstance(k, ActivationCheckpoint) else k for k in keep]
        if stream is not None and stream.device.index != self._device:
            refuse("the stream must belong to the tensors' device")

    def _call(self) -> None:
        if torch._C._cuda_getDevice() != self._device:
            with torch.cuda.device(self._device):
                self._call()
            return
        stream = self._stream.cuda_stream if self._stream is not None else torch._C._cuda_getCurrentRawStream(self._device)
        status = self._launch(*self._args, stream)
        if status:
            _native.check(status)


class ActivationCheckpoint:
    """Codes and scales of a [rows, cols] tensor: codes [rows, cols rounded up to 16] of an 8-bit dtype, scales [rows, ceil(cols / 32)] as
    float8_e8m0fnu (powers of two; a plain uint8 tensor of the same bytes is taken too).  Built around a caller's tensors, or `allocate`d."""

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, cols: int):
        if not (codes.is_cuda and scales.is_cuda) or codes.device != scales.device:
            refuse("ActivationCheckpoint: codes and scales must live on one CUDA device")
        if codes.dtype not in (torch.float8_e4m3fn, torch.float8_e5m2, torch.int8):
            refuse(f"ActivationCheckpoint: codes must be fp8_e4m3, fp8_e5m2 or int8, got {codes.dtype}")
        if scales.dtype not in (torch.float8_e8m0fnu, torch.uint8):
            refuse(f"ActivationCheckpoint: scales must be float8_e8m0fnu or uint8, got {scales.dtype}")
        cols = int(cols)
        if cols < 1 or codes.dim() != 2 or tuple(codes.shape[1:]) != (code_pitch(cols),) or tuple(scales.shape) != (codes.shape[0], scale_pitch(cols)):
            refuse(f"ActivationCheckpoint: {cols} columns need codes [rows, {code_pitch(max(cols, 1))}] and scales [rows, {scale_pitch(max(cols, 1))}]")
        if not (codes.is_contiguous() and scales.is_contiguous()) or codes.data_ptr() % 16:
            refuse("ActivationCheckpoint: codes and scales must be contiguous, codes 16-byte aligned")
        self.codes, self.scales, self.rows, self.cols = codes, scales, codes.shape[0], cols

    @staticmethod
    def allocate(rows: int, cols: int, dtype: DataType = DataType.fp8_e4m3, device="cuda") -> "ActivationCheckpoint":
        code_dtype(dtype)
        return ActivationCheckpoint(torch.empty(rows, code_pitch(cols), dtype=to_torch(dtype), device=device),
                                    torch.empty(rows, scale_pitch(cols), dtype=torch.float8_e8m0fnu, device=device), cols)

    @property
    def dtype(self) -> DataType:
        return from_torch(self.codes.dtype)

    @property
    def device(self) -> torch.device:
        return self.codes.device

    def row_range(self, first: int, last: int) -> "ActivationCheckpoint":
        """The checkpoint of rows [first, last): rows are independent, nothing is copied."""
        return ActivationCheckpoint(self.codes[first:last], self.scales[first:last], self.cols)


def code_pitch(cols: int) -> int:
    return int(_lib.thor_b200_checkpoint_code_pitch(cols))


def scale_pitch(cols: int) -> int:
    return int(_lib.thor_b200_checkpoint_scale_pitch(cols))


def code_dtype(dtype) -> DataType:
    dtype = DataType(dtype)
    if dtype not in CODE_DTYPES:
        refuse(f"checkpoint codes must be fp8_e4m3, fp8_e5m2 or int8, got {dtype.name}")
    return dtype


def target_checkpoint(given: Optional[ActivationCheckpoint], rows: int, cols: int, dtype: DataType, device: torch.device, what: str) -> ActivationCheckpoint:
    if given is None:
        return ActivationCheckpoint.allocate(rows, cols, dtype, device)
    matching_checkpoint(given, rows, cols, device, what)
    if given.dtype != dtype:
        refuse(f"{what} holds {given.dtype.name} codes, not {dtype.name}")
    return given


def matching_checkpoint(given: ActivationCheckpoint, rows: int, cols: int, device: torch.device, what: str) -> ActivationCheckpoint:
    if not isinstance(given, ActivationCheckpoint):
        refuse(f"{what} must be an ActivationCheckpoint")
    if (given.rows, given.cols) != (rows, cols) or given.device != device:
        refuse(f"{what} holds [{given.rows}, {given.cols}] on {given.device}, not [{rows}, {cols}] on {device}")
    return given


class StampedCheckpointPack(Stamped):
    def __init__(self, x: torch.Tensor, checkpoint: ActivationCheckpoint, stream):
        rows, cols, stride = as_rows(x, "CheckpointPack: the tensor")
        check_outputs({"codes": checkpoint.codes, "scales": checkpoint.scales}, {"the tensor": x})
        self.checkpoint = checkpoint
        desc = _CheckpointDesc(int(from_torch(x.dtype)), int(checkpoint.dtype), rows, cols, stride)
        super().__init__(_lib.thor_b200_checkpoint_pack_launch, (C.addressof(desc), x.data_ptr(), checkpoint.codes.data_ptr(), checkpoint.scales.data_ptr()), x.device, stream,
                         (x, checkpoint, desc))

    def run(self) -> ActivationCheckpoint:
        self._call()
        return self.checkpoint


class CheckpointPack:
    """Packs a tensor (any leading shape; its last axis are the columns) into a checkpoint of `dtype` codes."""

    def __init__(self, dtype: DataType = DataType.fp8_e4m3):
        self.dtype = code_dtype(dtype)

    def stamp(self, x: torch.Tensor, checkpoint: Optional[ActivationCheckpoint] = None, stream=None) -> StampedCheckpointPack:
        rows, cols, _ = as_rows(x, "CheckpointPack: the tensor")
        with memory_of(stream):
            checkpoint = target_checkpoint(checkpoint, rows, cols, self.dtype, x.device, "CheckpointPack: checkpoint")
        return StampedCheckpointPack(x, checkpoint, stream)


class StampedCheckpointUnpack(Stamped):
    def __init__(self, checkpoint: ActivationCheckpoint, output: torch.Tensor, stream):
        rows, cols, stride = as_rows(output, "CheckpointUnpack: output")
        matching_checkpoint(checkpoint, rows, cols, output.device, "CheckpointUnpack: checkpoint")
        check_outputs({"output": output}, {"codes": checkpoint.codes, "scales": checkpoint.scales})
        self.checkpoint, self.output = checkpoint, output
        desc = _CheckpointDesc(int(from_torch(output.dtype)), int(checkpoint.dtype), rows, cols, stride)
        super().__init__(_lib.thor_b200_checkpoint_unpack_launch, (C.addressof(desc), checkpoint.codes.data_ptr(), checkpoint.scales.data_ptr(), output.data_ptr()), output.device, stream,
                         (checkpoint, output, desc))

    def run(self) -> torch.Tensor:
        self._call()
        return self.output


class CheckpointUnpack:
    """Writes the values that a checkpoint stands for as fp32, fp16 or bf16 (bf16 and fp32 hold every one of them exactly down to
    their subnormal numbers; a code that stands for 2^128, half a step above the largest numbers, unpacks as infinity.  fp16 rounds once, and values
    from 65520 on are infinite there)."""

    def __init__(self, dtype: DataType = DataType.bf16):
        self.dtype = DataType(dtype)
        if self.dtype not in VALUE_DTYPES:
            refuse(f"CheckpointUnpack: dtype must be fp32, fp16 or bf16, got {self.dtype.name}")

    def stamp(self, checkpoint: ActivationCheckpoint, output: Optional[torch.Tensor] = None, stream=None) -> StampedCheckpointUnpack:
        if not isinstance(checkpoint, ActivationCheckpoint):
            refuse("CheckpointUnpack: needs an ActivationCheckpoint")
        if output is None:
            with memory_of(stream):
                output = torch.empty(checkpoint.rows, checkpoint.cols, dtype=to_torch(self.dtype), device=checkpoint.device)
        elif output.dtype != to_torch(self.dtype):
            refuse(f"CheckpointUnpack: output must be {self.dtype.name}")
        return StampedCheckpointUnpack(checkpoint, output, stream)
