"""Activations that keep their input as an 8-bit checkpoint in the forward pass and read it in the backward pass (include/thor_b200.h).
The functions are those of Expression.gelu and Expression.swish; plain or gated (act(x) * gate)."""
from __future__ import annotations

import ctypes as C
import enum
from typing import Optional

import torch

from . import _native
from .checkpoint import ActivationCheckpoint, Stamped, as_rows, check_outputs, code_dtype, matching_checkpoint, memory_of, refuse, same_rows, target_checkpoint
from .dtypes import DataType, from_torch

_lib = _native.lib


class _ActivationDesc(C.Structure):
    _fields_ = [("kind", C.c_int32), ("gated", C.c_int32), ("dtype", C.c_int32), ("code_dtype", C.c_int32), ("rows", C.c_uint64), ("cols", C.c_uint64),
                ("x_stride", C.c_int64), ("gate_stride", C.c_int64), ("y_stride", C.c_int64)]


_lib.thor_b200_checkpointed_activation_launch.argtypes = [C.POINTER(_ActivationDesc)] + [C.c_void_p] * 8
_lib.thor_b200_checkpointed_activation_backward_launch.argtypes = [C.POINTER(_ActivationDesc)] + [C.c_void_p] * 8


class CheckpointedActivationKind(enum.IntEnum):
    Gelu = 0
    Swish = 1


class StampedCheckpointedActivation(Stamped):
    def __init__(self, kind, x, gate, output, checkpoint, gate_checkpoint, stream):
        rows, cols, x_stride = as_rows(x, "CheckpointedActivation: x")
        gate_stride = same_rows(gate, "CheckpointedActivation: gate", x) if gate is not None else 0
        y_stride = same_rows(output, "CheckpointedActivation: output", x)
        kept = {"codes": checkpoint.codes, "scales": checkpoint.scales}
        if gate is not None:
            kept.update({"gate codes": gate_checkpoint.codes, "gate scales": gate_checkpoint.scales})
        check_outputs({"output": output, **kept}, {"x": x, "gate": gate})
        self.output, self.checkpoint, self.gate_checkpoint = output, checkpoint, gate_checkpoint
        desc = _ActivationDesc(int(kind), int(gate is not None), int(from_torch(x.dtype)), int(checkpoint.dtype), rows, cols, x_stride, gate_stride, y_stride)
        super().__init__(_lib.thor_b200_checkpointed_activation_launch,
                         (C.addressof(desc), x.data_ptr(), gate.data_ptr() if gate is not None else None, output.data_ptr(), checkpoint.codes.data_ptr(), checkpoint.scales.data_ptr(),
                          gate_checkpoint.codes.data_ptr() if gate is not None else None, gate_checkpoint.scales.data_ptr() if gate is not None else None),
                         x.device, stream, (x, gate, output, checkpoint, gate_checkpoint, desc))

    def run(self) -> torch.Tensor:
        self._call()
        return self.output


class CheckpointedActivation:
    """output = act(x), or act(x) * gate; the checkpoints of x and of gate are written in the same pass."""

    def __init__(self, kind: CheckpointedActivationKind, checkpoint_dtype: DataType = DataType.fp8_e4m3):
        self.kind, self.checkpoint_dtype = CheckpointedActivationKind(kind), code_dtype(checkpoint_dtype)

    def stamp(self, x: torch.Tensor, gate: Optional[torch.Tensor] = None, output: Optional[torch.Tensor] = None, checkpoint: Optional[ActivationCheckpoint] = None,
              gate_checkpoint: Optional[ActivationCheckpoint] = None, stream=None) -> StampedCheckpointedActivation:
        rows, cols, _ = as_rows(x, "CheckpointedActivation: x")
        if gate is None and gate_checkpoint is not None:
            refuse("CheckpointedActivation: gate_checkpoint without a gate")
        with memory_of(stream):
            if output is None:
                output = torch.empty(x.shape, dtype=x.dtype, device=x.device)
            checkpoint = target_checkpoint(checkpoint, rows, cols, self.checkpoint_dtype, x.device, "CheckpointedActivation: checkpoint")
            if gate is not None:
                gate_checkpoint = target_checkpoint(gate_checkpoint, rows, cols, self.checkpoint_dtype, x.device, "CheckpointedActivation: gate_checkpoint")
        return StampedCheckpointedActivation(self.kind, x, gate, output, checkpoint, gate_checkpoint, stream)


class StampedCheckpointedActivationBackward(Stamped):
    def __init__(self, kind, grad_output, checkpoint, gate_checkpoint, grad_input, grad_gate, stream):
        rows, cols, y_stride = as_rows(grad_output, "CheckpointedActivationBackward: grad_output")
        x_stride = same_rows(grad_input, "CheckpointedActivationBackward: grad_input", grad_output)
        gated = gate_checkpoint is not None
        gate_stride = same_rows(grad_gate, "CheckpointedActivationBackward: grad_gate", grad_output) if gated else 0
        kept = {"codes": checkpoint.codes, "scales": checkpoint.scales}
        if gated:
            kept.update({"gate codes": gate_checkpoint.codes, "gate scales": gate_checkpoint.scales})
        check_outputs({"grad_input": grad_input, "grad_gate": grad_gate}, {"grad_output": grad_output, **kept})
        self.grad_input, self.grad_gate = grad_input, grad_gate
        desc = _ActivationDesc(int(kind), int(gated), int(from_torch(grad_output.dtype)), int(checkpoint.dtype), rows, cols, x_stride, gate_stride, y_stride)
        super().__init__(_lib.thor_b200_checkpointed_activation_backward_launch,
                         (C.addressof(desc), grad_output.data_ptr(), checkpoint.codes.data_ptr(), checkpoint.scales.data_ptr(),
                          gate_checkpoint.codes.data_ptr() if gated else None, gate_checkpoint.scales.data_ptr() if gated else None,
                          grad_input.data_ptr(), grad_gate.data_ptr() if gated else None), grad_output.device, stream,
                         (grad_output, checkpoint, gate_checkpoint, grad_input, grad_gate, desc))

    def run(self) -> torch.Tensor:
        self._call()
        return self.grad_input


class CheckpointedActivationBackward:
    """grad_input = grad_output * act'(x) with x from its checkpoint; with the gate's checkpoint too, grad_input = grad_output * gate * act'(x)
    and grad_gate = grad_output * act(x).  The gradients may be column slices of one buffer.  Where x was masked with its type's lowest number, whose
    code stands for 2^128, both gradients are zero."""

    def __init__(self, kind: CheckpointedActivationKind):
        self.kind = CheckpointedActivationKind(kind)

    def stamp(self, grad_output: torch.Tensor, checkpoint: ActivationCheckpoint, gate_checkpoint: Optional[ActivationCheckpoint] = None,
              grad_input: Optional[torch.Tensor] = None, grad_gate: Optional[torch.Tensor] = None, stream=None) -> StampedCheckpointedActivationBackward:
        rows, cols, _ = as_rows(grad_output, "CheckpointedActivationBackward: grad_output")
        matching_checkpoint(checkpoint, rows, cols, grad_output.device, "CheckpointedActivationBackward: checkpoint")
        if gate_checkpoint is not None:
            matching_checkpoint(gate_checkpoint, rows, cols, grad_output.device, "CheckpointedActivationBackward: gate_checkpoint")
            if gate_checkpoint.dtype != checkpoint.dtype:
                refuse("CheckpointedActivationBackward: both checkpoints must hold the same code dtype")
        elif grad_gate is not None:
            refuse("CheckpointedActivationBackward: grad_gate without the gate's checkpoint")
        with memory_of(stream):
            if grad_input is None:
                grad_input = torch.empty(grad_output.shape, dtype=grad_output.dtype, device=grad_output.device)
            if gate_checkpoint is not None and grad_gate is None:
                grad_gate = torch.empty(grad_output.shape, dtype=grad_output.dtype, device=grad_output.device)
        return StampedCheckpointedActivationBackward(self.kind, grad_output, checkpoint, gate_checkpoint, grad_input, grad_gate, stream)
