"""Activations kept in 8 bits for the backward pass.

    checkpoint_activation(x)      -> ActivationCheckpoint: x in blocks of 32 columns, float8 values and a power of two each
    ActivationCheckpoint.decode() -> the values that are kept
    checkpoint_weight_gradient(g, checkpoint) -> the gradients of a linear layer's weight and bias, from its input as it was kept

What a layer keeps of its input between the two passes is most of a training step's memory.  A checkpoint takes 33/64 of a 16-bit
matrix, and a gradient formed from it differs from the exact one by what rounding to 4 bits of mantissa does to the input
(at most 2^-4 of each element, 2^-5.6 of the whole in the mean).  The layers keep one of their input when asked to (SparseLinearTranspose,
SoftThresholdLinear, GELUglu with checkpoint=True); the operators in front of a layer write one along with their output
(block_norm, residual_norm, GELUglu), which saves the pass that reads the input again.  The reference keeps its activations
as they are.
"""
import warnings

import torch

from . import _native as N

__all__ = ["ActivationCheckpoint", "checkpoint_activation", "checkpoint_weight_gradient"]

_BLOCK = 32
_TYPES = (torch.float32, torch.float16, torch.bfloat16)


class ActivationCheckpoint:
    """A tensor kept in 8 bits: `values` (float8_e4m3fn, [rows, 32 * blocks]) times 2^(`scales` - 127) (uint8, [rows, blocks]); a
    row is one of the tensor's last dimension, filled up with zeros.  `shape` and `dtype` are the tensor's.  Infinities and NaNs
    are kept as NaNs.  It is data: no gradient passes through it."""

    __slots__ = ("values", "scales", "shape", "dtype")

    def __init__(self, values, scales, shape, dtype):
        self.values, self.scales, self.shape, self.dtype = values, scales, torch.Size(shape), dtype
        self._check()

    def _check(self):
        values, scales, shape, dtype = self.values, self.scales, self.shape, self.dtype
        rows, blocks = shape[:-1].numel(), (shape[-1] + _BLOCK - 1) // _BLOCK if len(shape) else 0
        if (not blocks or values.shape != (rows, _BLOCK * blocks) or scales.shape != (rows, blocks) or values.dtype != torch.float8_e4m3fn
                or scales.dtype != torch.uint8 or values.device != scales.device or not values.is_contiguous() or not scales.is_contiguous()
                or dtype not in _TYPES):
            raise RuntimeError(f"ActivationCheckpoint: values {tuple(values.shape)} {values.dtype} and scales {tuple(scales.shape)} {scales.dtype} "
                               f"do not hold a tensor {tuple(shape)} {dtype}")

    @classmethod
    def _of(cls, values, scales, shape, dtype):
        """One of tensors that were made for it."""
        self = object.__new__(cls)
        self.values, self.scales, self.shape, self.dtype = values, scales, shape, dtype
        return self

    @property
    def device(self):
        return self.values.device

    @property
    def nbytes(self):
        return self.values.numel() + self.scales.numel()

    def decode(self, dtype=None):
        """The kept values, in the type of the tensor that was kept (exact) or in another one (rounded)."""
        dtype = self.dtype if dtype is None else dtype
        if dtype not in _TYPES:
            raise RuntimeError(f"ActivationCheckpoint.decode: dtype {dtype} is not supported")
        calls = N.torch_calls()
        if calls is not None:
            out = calls.checkpoint_decode(self.values, self.scales, self.shape, N.dtype_codes[dtype])
            if out is not None:
                return out
        self._check()
        if not self.values.is_cuda:
            raise RuntimeError("ActivationCheckpoint.decode: only CUDA tensors are supported")
        out = torch.empty(self.shape, dtype=dtype, device=self.values.device)
        rows, cols = self.values.shape[0], self.shape[-1]
        N.launch(out, N.lib().tf24_checkpoint_decode, self.values.data_ptr(), self.scales.data_ptr(), rows, cols, out.data_ptr(), N.dtype_code(dtype), cols)
        return out

    def __repr__(self):
        return f"ActivationCheckpoint(shape={tuple(self.shape)}, dtype={self.dtype}, device={self.device})"


def empty_checkpoint(rows, cols, device):
    """(values, scales) for a matrix of rows x cols"""
    blocks = (cols + _BLOCK - 1) // _BLOCK
    return (torch.empty((rows, _BLOCK * blocks), dtype=torch.float8_e4m3fn, device=device),
            torch.empty((rows, blocks), dtype=torch.uint8, device=device))


def checkpoint_activation(x):
    """x (float32, float16 or bfloat16, on a GPU, at least one dimension and one column) kept in 8 bits."""
    calls = N.torch_calls()
    if calls is not None and N.plain_eager():
        kept = calls.checkpoint_encode(x)
        if kept is not None:
            return ActivationCheckpoint._of(*kept, x.shape, x.dtype)
    if not x.is_cuda:
        raise RuntimeError("checkpoint_activation: only CUDA tensors are supported")
    if x.dtype not in _TYPES:
        raise RuntimeError(f"checkpoint_activation: dtype {x.dtype} is not supported")
    if x.dim() == 0 or x.shape[-1] == 0:
        raise RuntimeError(f"checkpoint_activation: shape {tuple(x.shape)} has no columns")
    flat, ld = N.as_rows(x)
    cols = x.shape[-1]
    rows = x.shape[:-1].numel()
    values, scales = empty_checkpoint(rows, cols, x.device)
    N.launch(x, N.lib().tf24_checkpoint_encode, flat.data_ptr(), N.dtype_code(x.dtype), ld, rows, cols, values.data_ptr(), scales.data_ptr())
    return ActivationCheckpoint._of(values, scales, x.shape, x.dtype)


def kept_of_input(given, setting):
    """What a layer is to keep of its input: the checkpoint that was given to the call, with a setting of its own (or given=True) one to be made where a
    graph is recorded, or None (given=False, whatever the setting): the input as it is."""
    kept = bool(setting) if given is None else given
    return None if kept is False or (kept is True and not torch.is_grad_enabled()) else kept


def says_that_nothing_is_kept(layer, given, why):
    """A layer that was asked for it (setting, True or a checkpoint for one call) cannot keep its input in 8 bits: what was asked for this call is
    refused; what its setting asks for is left out with a warning, where there will be a backward pass."""
    name = type(layer).__name__
    if given is not None and given is not False:
        raise RuntimeError(f"{name}: a checkpoint of the input is taken {why}")
    if given is None and layer.checkpoint and torch.is_grad_enabled() and layer.weight.requires_grad:
        warnings.warn(f"{name}: checkpoint=True has no effect on this call, the input is kept as it is: in 8 bits it is kept {why}", stacklevel=3)


def as_checkpoint(x, given):
    """What a layer keeps of its input x: the checkpoint that came with it, or with given=True one made here."""
    if given is True:
        return checkpoint_activation(x)
    if not isinstance(given, ActivationCheckpoint):
        raise RuntimeError(f"{type(given).__name__} is not a checkpoint of the input")
    if given.shape != x.shape or given.dtype != x.dtype or given.values.get_device() != x.get_device():
        raise RuntimeError(f"the checkpoint of a tensor {tuple(given.shape)} {given.dtype} on {given.device} is not one of {tuple(x.shape)} {x.dtype} on {x.device}")
    return given


def checkpoint_weight_gradient(grad_output, checkpoint, bias=False, dtype=None):
    """(dW, db) of y = x W^T + b: dW = grad_output^T x with x as `checkpoint` keeps it, db the sum of grad_output's rows with bias=True, otherwise None.
    grad_output [..., out_features] is float16 or bfloat16, x of the same type and leading dimensions; dW [out_features, in_features] and db
    are of that type or, with dtype=torch.float32, float32 (sums that are not rounded).  Without a graph: for backward passes."""
    g = grad_output.detach()
    if not g.is_cuda or g.get_device() != checkpoint.values.get_device():
        raise RuntimeError(f"checkpoint_weight_gradient: grad_output on {g.device} and a checkpoint on {checkpoint.device} are not on one GPU")
    if g.dtype not in (torch.float16, torch.bfloat16) or g.dtype != checkpoint.dtype:
        raise RuntimeError(f"checkpoint_weight_gradient: grad_output {g.dtype} with a checkpoint of {checkpoint.dtype} is not supported (float16 or bfloat16, both the same)")
    dtype = g.dtype if dtype is None else dtype
    if dtype not in (g.dtype, torch.float32):
        raise RuntimeError(f"checkpoint_weight_gradient: results of {dtype} are not supported ({g.dtype}, float32)")
    shape = checkpoint.shape
    if g.dim() == 0 or g.shape[:-1] != shape[:-1] or g.shape[-1] == 0:
        raise RuntimeError(f"checkpoint_weight_gradient: grad_output {tuple(g.shape)} does not suit a checkpoint of {tuple(shape)}")
    tokens, m, n = checkpoint.values.shape[0], g.shape[-1], shape[-1]
    calls = N.torch_calls()
    if calls is not None and N.plain_eager():
        grads = calls.checkpoint_weight_grad(g, checkpoint.values, checkpoint.scales, n, bias, N.dtype_codes[dtype])
        if grads is not None:
            return grads
    checkpoint._check()
    if tokens == 0:
        return torch.zeros((m, n), dtype=dtype, device=g.device), torch.zeros(m, dtype=dtype, device=g.device) if bias else None
    g, ld = N.as_rows(g)
    padded = (m + 7) // 8 * 8
    if padded != m:                                                # (the kernel's outputs come in eights)
        g = torch.nn.functional.pad(g.reshape(tokens, m), (0, padded - m))
        ld = padded
    elif ld < m or ld % 8 or g.data_ptr() % 16:
        g, ld = g.reshape(tokens, m).clone(memory_format=torch.contiguous_format), m
    dw = torch.empty((padded, n), dtype=dtype, device=g.device)
    db = torch.empty(padded, dtype=dtype, device=g.device) if bias else None
    lib = N.lib()
    nbytes = lib.tf24_checkpoint_weight_grad_workspace_bytes(tokens, padded, n)
    workspace = torch.empty(nbytes, dtype=torch.uint8, device=g.device) if nbytes else None
    N.launch(g, lib.tf24_checkpoint_weight_grad, g.data_ptr(), ld, N.dtype_codes[g.dtype], checkpoint.values.data_ptr(), checkpoint.scales.data_ptr(), tokens, padded, n,
             dw.data_ptr(), N.ptr(db), N.dtype_codes[dtype], N.ptr(workspace), nbytes)
    return dw[:m] if padded != m else dw, db[:m] if bias and padded != m else db
