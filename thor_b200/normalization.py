"""LayerNorm over the last axis, forward and backward, with the residual add, the saved statistics and the normalised rows as an 8-bit
checkpoint (include/thor_b200.h)."""
from __future__ import annotations

import ctypes as C
from typing import Optional

import torch

from . import _native
from .checkpoint import ActivationCheckpoint, Stamped, VALUE_DTYPES, as_rows, check_outputs, code_dtype, matching_checkpoint, memory_of, refuse, same_rows, target_checkpoint
from .dtypes import DataType, from_torch, to_torch

_lib = _native.lib


class _LayerNormDesc(C.Structure):
    _fields_ = [("dtype", C.c_int32), ("param_dtype", C.c_int32), ("grad_param_dtype", C.c_int32), ("code_dtype", C.c_int32), ("eps", C.c_float), ("reserved", C.c_uint32),
                ("rows", C.c_uint64), ("cols", C.c_uint64), ("x_stride", C.c_int64), ("residual_stride", C.c_int64), ("y_stride", C.c_int64)]


_lib.thor_b200_layernorm_launch.argtypes = [C.POINTER(_LayerNormDesc)] + [C.c_void_p] * 11
_lib.thor_b200_layernorm_backward_workspace_bytes.argtypes = [C.POINTER(_LayerNormDesc), C.POINTER(C.c_size_t)]
_lib.thor_b200_layernorm_backward_launch.argtypes = [C.POINTER(_LayerNormDesc)] + [C.c_void_p] * 12 + [C.c_size_t, C.c_void_p]
_lib.thor_b200_layernorm_backward_launch_count.argtypes = [C.POINTER(_LayerNormDesc), C.c_int]


def _ptr(t: Optional[torch.Tensor]):
    return t.data_ptr() if t is not None else None


def _check_params(who: str, like: torch.Tensor, **params) -> DataType:
    """The common dtype of the parameters that are given (the tensor's own when none is)."""
    dtype = None
    for name, p in params.items():
        if p is None:
            continue
        if p.device != like.device or tuple(p.shape) != (like.shape[-1],) or not p.is_contiguous():
            refuse(f"{who}: {name} must be a contiguous [{like.shape[-1]}] tensor on {like.device}")
        if p.dtype not in (torch.float32, torch.float16, torch.bfloat16) or (dtype is not None and p.dtype != dtype):
            refuse(f"{who}: parameters must be fp32, fp16 or bf16, all of one dtype, got {p.dtype}")
        dtype = p.dtype
    return from_torch(dtype if dtype is not None else like.dtype)


def _check_statistic(who: str, name: str, t: torch.Tensor, rows: int, device: torch.device) -> None:
    if t.dtype != torch.float32 or t.numel() != rows or not t.is_contiguous() or t.device != device:
        refuse(f"{who}: {name} must be {rows} contiguous fp32 values on {device}")


class StampedLayerNorm(Stamped):
    """output, and as described: sum, mean, rstd, checkpoint (None where not produced)."""

    def __init__(self, desc, x, gamma, beta, residual, output, total, mean, rstd, checkpoint, stream):
        self.output, self.sum, self.mean, self.rstd, self.checkpoint = output, total, mean, rstd, checkpoint
        super().__init__(_lib.thor_b200_layernorm_launch,
                         (C.addressof(desc), _ptr(x), _ptr(residual), _ptr(gamma), _ptr(beta), _ptr(output), _ptr(total), _ptr(mean), _ptr(rstd),
                          _ptr(checkpoint.codes) if checkpoint is not None else None, _ptr(checkpoint.scales) if checkpoint is not None else None),
                         x.device, stream, (x, gamma, beta, residual, output, total, mean, rstd, checkpoint, desc))

    def run(self) -> torch.Tensor:
        self._call()
        return self.output


class LayerNorm:
    """output = (h - mean(h)) * rstd(h) * gamma + beta over the last axis; h = x, or x + residual rounded to the tensors' dtype, which is the
    second output `sum`.  With save_statistics the backward pass's needs are kept: mean and rstd (fp32, one a row) or, with a
    checkpoint_dtype, rstd and the checkpoint of the normalised rows.  save_statistics = False is the form for answering."""

    def __init__(self, eps: float = 1e-5, checkpoint_dtype: Optional[DataType] = None, save_statistics: bool = True):
        if not eps >= 0.0:
            refuse("LayerNorm: eps must not be negative")
        if checkpoint_dtype is not None and not save_statistics:
            refuse("LayerNorm: a checkpoint needs the saved statistics")
        self.eps, self.save_statistics = float(eps), bool(save_statistics)
        self.checkpoint_dtype = code_dtype(checkpoint_dtype) if checkpoint_dtype is not None else None

    def stamp(self, x: torch.Tensor, gamma: Optional[torch.Tensor] = None, beta: Optional[torch.Tensor] = None, residual: Optional[torch.Tensor] = None,
              output: Optional[torch.Tensor] = None, checkpoint: Optional[ActivationCheckpoint] = None, stream=None) -> StampedLayerNorm:
        rows, cols, x_stride = as_rows(x, "LayerNorm: x")
        residual_stride = same_rows(residual, "LayerNorm: residual", x) if residual is not None else 0
        param = _check_params("LayerNorm", x, gamma=gamma, beta=beta)
        if checkpoint is not None and self.checkpoint_dtype is None:
            refuse("LayerNorm: described without a checkpoint")
        with memory_of(stream):
            if output is None:
                output = torch.empty(x.shape, dtype=x.dtype, device=x.device)
            total = torch.empty(x.shape, dtype=x.dtype, device=x.device) if residual is not None else None
            if self.checkpoint_dtype is not None:
                checkpoint = target_checkpoint(checkpoint, rows, cols, self.checkpoint_dtype, x.device, "LayerNorm: checkpoint")
            statistic = lambda: torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device)
            rstd = statistic() if self.save_statistics else None
            mean = statistic() if self.save_statistics and checkpoint is None else None
        y_stride = same_rows(output, "LayerNorm: output", x)
        check_outputs({"output": output, "codes": checkpoint.codes if checkpoint else None, "scales": checkpoint.scales if checkpoint else None},
                      {"x": x, "residual": residual, "gamma": gamma, "beta": beta})
        desc = _LayerNormDesc(int(from_torch(x.dtype)), int(param), 0, int(self.checkpoint_dtype or 0), self.eps, 0, rows, cols, x_stride, residual_stride, y_stride)
        return StampedLayerNorm(desc, x, gamma, beta, residual, output, total, mean, rstd, checkpoint, stream)


class StampedLayerNormBackward(Stamped):
    """grad_input, grad_gamma, grad_beta (the last two None without a gamma).  The plan owns its workspace."""

    def __init__(self, desc, grad_output, rstd, gamma, x, mean, checkpoint, grad_sum, grad_input, grad_params, workspace, stream):
        self.grad_input = grad_input
        self.grad_gamma, self.grad_beta = (grad_params[0], grad_params[1]) if grad_params is not None else (None, None)
        self.kernel_launches = int(_lib.thor_b200_layernorm_backward_launch_count(C.byref(desc), int(grad_params is not None)))
        super().__init__(_lib.thor_b200_layernorm_backward_launch,
                         (C.addressof(desc), _ptr(grad_output), _ptr(x), _ptr(mean), _ptr(rstd), _ptr(checkpoint.codes) if checkpoint is not None else None,
                          _ptr(checkpoint.scales) if checkpoint is not None else None, _ptr(gamma), _ptr(grad_sum), _ptr(grad_input), _ptr(self.grad_gamma), _ptr(self.grad_beta),
                          _ptr(workspace), workspace.numel() if workspace is not None else 0),
                         grad_output.device, stream, (grad_output, rstd, gamma, x, mean, checkpoint, grad_sum, grad_input, grad_params, workspace, desc))

    def run(self) -> torch.Tensor:
        self._call()
        return self.grad_input


class LayerNormBackward:
    """Gradients of a LayerNorm from what its forward pass kept: the normalised rows' checkpoint, or x (the sum, where there was a residual) with
    mean.  grad_sum is the gradient that reaches the layer's input by the residual stream; it is added in the same pass.
    grad_gamma and grad_beta come in `grad_dtype` (gamma's by default); they are the two rows of one [2, cols] tensor, and in fp32 they are the
    unrounded column sums that the shards of a batch add up."""

    def __init__(self, grad_dtype: Optional[DataType] = None):
        self.grad_dtype = DataType(grad_dtype) if grad_dtype is not None else None
        if self.grad_dtype is not None and self.grad_dtype not in VALUE_DTYPES:
            refuse(f"LayerNormBackward: parameter gradients must be fp32, fp16 or bf16, got {self.grad_dtype.name}")

    def stamp(self, grad_output: torch.Tensor, rstd: torch.Tensor, gamma: Optional[torch.Tensor] = None, x: Optional[torch.Tensor] = None,
              mean: Optional[torch.Tensor] = None, checkpoint: Optional[ActivationCheckpoint] = None, grad_sum: Optional[torch.Tensor] = None,
              stream=None) -> StampedLayerNormBackward:
        who = "LayerNormBackward"
        rows, cols, y_stride = as_rows(grad_output, f"{who}: grad_output")
        device = grad_output.device
        if (checkpoint is not None) == (x is not None) or (x is not None) != (mean is not None):
            refuse(f"{who}: needs either the checkpoint or x with its mean")
        _check_statistic(who, "rstd", rstd, rows, device)
        x_stride = 0
        if x is not None:
            x_stride = same_rows(x, f"{who}: x", grad_output)
            _check_statistic(who, "mean", mean, rows, device)
        else:
            matching_checkpoint(checkpoint, rows, cols, device, f"{who}: checkpoint")
        sum_stride = same_rows(grad_sum, f"{who}: grad_sum", grad_output) if grad_sum is not None else 0
        param = _check_params(who, grad_output, gamma=gamma)
        grad_param = self.grad_dtype if self.grad_dtype is not None else param
        with memory_of(stream):
            grad_input = torch.empty(grad_output.shape, dtype=grad_output.dtype, device=device)
            grad_params = torch.empty(2, cols, dtype=to_torch(grad_param), device=device) if gamma is not None else None
        desc = _LayerNormDesc(int(from_torch(grad_output.dtype)), int(param), int(grad_param), int(checkpoint.dtype) if checkpoint is not None else 0, 0.0, 0, rows, cols, x_stride,
                              sum_stride, y_stride)
        workspace = None
        if gamma is not None:
            size = C.c_size_t()
            _native.check(_lib.thor_b200_layernorm_backward_workspace_bytes(C.byref(desc), C.byref(size)))
            with memory_of(stream):
                workspace = torch.empty(size.value, dtype=torch.uint8, device=device)
        return StampedLayerNormBackward(desc, grad_output, rstd, gamma, x, mean, checkpoint, grad_sum, grad_input, grad_params, workspace, stream)
