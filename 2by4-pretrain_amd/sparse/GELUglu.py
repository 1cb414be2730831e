"""GELUglu / gelu_glu: out = gelu_tanh(gate) * x for an input whose last dimension is [x | gate].

Mirror of the reference module (sparse/GELUglu.py:156-243): an autograd function over a 3-d input
and the nn.Module around it.  Inputs whose last dimension is contiguous take the row-major kernel
(:161-177); inputs stored with the last dimension strided (a transposed 2-d view: :178-197) take
the column-major one and, like the reference, return an output stored the same way.
"""
import torch
from torch import autograd

from . import _native as N
from .activation_checkpoint import ActivationCheckpoint, empty_checkpoint

__all__ = ["GELUglu", "gelu_glu", "gelu_glu_checkpoint"]


def _as_2d(t):
    """(2-d view [rows, cols], layout, ld) the kernels can address, copying when neither
    dimension of the flattened tensor is contiguous."""
    t2 = (t.resolve_neg() if t.is_neg() else t).reshape(-1, t.shape[-1])
    lay = N.layout_of(t2)
    if lay is None:
        t2 = t2.contiguous()
        lay = N.layout_of(t2)
    return t2, lay[0], lay[1]


def _ld(t, layout):
    return t.stride(0) if layout == N.ROW_MAJOR else t.stride(1)


def _empty_like_layout(rows, cols, layout, like):
    if layout == N.ROW_MAJOR:
        return torch.empty((rows, cols), dtype=like.dtype, device=like.device)
    return torch.empty((cols, rows), dtype=like.dtype, device=like.device).t()


class gelu_glu(autograd.Function):
    @staticmethod
    def forward(ctx, input):
        assert input.dim() == 3, 'input must be 3D'
        if not input.is_cuda:
            raise RuntimeError("gelu_glu: only CUDA tensors are supported")
        if input.shape[-1] % 2:
            raise RuntimeError(f"gelu_glu: the last dimension ({input.shape[-1]}) must be even")
        x2, layout, ld = _as_2d(input)
        rows, cols = x2.shape
        out = _empty_like_layout(rows, cols // 2, layout, x2)
        N.check(N.lib().tf24_gelu_glu_forward(x2.data_ptr(), N.dtype_code(x2.dtype), layout, ld, rows, cols,
                                              out.data_ptr(), _ld(out, layout), N.stream_ptr()))
        ctx.save_for_backward(x2)
        ctx.layout, ctx.shape = layout, input.shape
        return out.view(*input.shape[:-1], cols // 2)

    @staticmethod
    def backward(ctx, grad_output):
        assert grad_output.dim() == 3, 'grad_output must be 3D'
        (x2,) = ctx.saved_tensors
        layout = ctx.layout
        rows, cols = x2.shape
        go = (grad_output.resolve_neg() if grad_output.is_neg() else grad_output).reshape(rows, cols // 2).to(x2.dtype)
        want = _empty_like_layout(rows, cols // 2, layout, x2)
        if go.stride() != want.stride():          # bring the gradient to the layout of the forward output
            want.copy_(go)
            go = want
        grad_in = _empty_like_layout(rows, cols, layout, x2)
        N.check(N.lib().tf24_gelu_glu_backward(go.data_ptr(), _ld(go, layout), x2.data_ptr(), N.dtype_code(x2.dtype), layout,
                                               _ld(x2, layout), rows, cols, grad_in.data_ptr(), _ld(grad_in, layout),
                                               N.stream_ptr()))
        return grad_in.view(ctx.shape)


class _gelu_glu_checkpoint(autograd.Function):
    @staticmethod
    def forward(ctx, input, keep_output, keep_input):
        if not input.is_cuda:
            raise RuntimeError("gelu_glu_checkpoint: only CUDA tensors are supported")
        if input.dim() == 0 or input.shape[-1] == 0 or input.shape[-1] % 2:
            raise RuntimeError(f"gelu_glu_checkpoint: the last dimension of {tuple(input.shape)} must be even")
        if input.dtype not in (torch.float32, torch.float16, torch.bfloat16):
            raise RuntimeError(f"gelu_glu_checkpoint: dtype {input.dtype} is not supported")
        x2, ld = N.as_rows(input)
        rows, cols = input.shape[:-1].numel(), input.shape[-1]
        half = cols // 2
        out = torch.empty((*input.shape[:-1], half), dtype=input.dtype, device=input.device)
        values, scales = empty_checkpoint(2 * rows, half, input.device) if keep_input else (None, None)
        out_values, out_scales = empty_checkpoint(rows, half, input.device) if keep_output else (None, None)
        if rows > 1 and ld < cols:                                 # rows that overlap
            x2, ld = x2.contiguous(), cols
        N.launch(input, N.lib().tf24_gelu_glu_forward_checkpoint, x2.data_ptr(), N.dtype_code(input.dtype), ld, rows, cols, out.data_ptr(), half,
                 N.ptr(values), N.ptr(scales), N.ptr(out_values), N.ptr(out_scales))
        if keep_input:
            ctx.save_for_backward(values, scales)
        ctx.shape, ctx.dtype, ctx.device = input.shape, input.dtype, input.device
        if not keep_output:
            return out
        ctx.mark_non_differentiable(out_values, out_scales)
        ctx.set_materialize_grads(False)
        return out, out_values, out_scales

    @staticmethod
    def backward(ctx, grad_output, *_):
        if torch.is_grad_enabled():
            raise RuntimeError("a graph of the gradients of gelu_glu_checkpoint is not supported")
        if grad_output is None:
            return None, None, None
        values, scales = ctx.saved_tensors
        cols = ctx.shape[-1]
        rows, half = ctx.shape[:-1].numel(), cols // 2
        blocks = N.lib().tf24_checkpoint_blocks(half)

        def as_it_was(t, shape, dtype):
            return N.as_it_was("gelu_glu_checkpoint", t, shape, dtype, ctx.device)

        values = as_it_was(values, (2 * rows, 32 * blocks), torch.float8_e4m3fn).contiguous()
        scales = as_it_was(scales, (2 * rows, blocks), torch.uint8).contiguous()
        go, ld = N.as_rows(as_it_was(grad_output if grad_output.dtype == ctx.dtype else grad_output.to(ctx.dtype), (*ctx.shape[:-1], half), ctx.dtype))
        if rows > 1 and ld < half:
            go, ld = go.contiguous(), half
        grad_in = torch.empty(ctx.shape, dtype=ctx.dtype, device=values.device)
        N.launch(values, N.lib().tf24_gelu_glu_backward_checkpoint, go.data_ptr(), ld, values.data_ptr(), scales.data_ptr(), N.dtype_code(ctx.dtype), rows, cols,
                 grad_in.data_ptr(), cols)
        return grad_in, None, None


class gelu_glu_checkpoint:
    """gelu_glu that keeps its input in 8 bits for the backward pass (as in ActivationCheckpoint, x and gate of a row one after the
    other) and gives the gradient at the kept values: 1.03 bytes an element in place of 2, for an input that nothing else holds.  The
    output is the same.  apply(input) -> out; apply(input, True) -> (out, values, scales), the last two being out kept in 8 bits.  Any
    input with a last dimension of an even size; the output is row-major.  Where no graph is recorded nothing is kept of the input."""

    @staticmethod
    def apply(input, keep_output=False):
        calls = N.torch_calls()
        if calls is not None and N.plain_eager():
            result = calls.gelu_glu_checkpoint(input, keep_output)
            if result is not None:
                return result
        return _gelu_glu_checkpoint.apply(input, keep_output, torch.is_grad_enabled() and input.requires_grad)


class GELUglu(torch.nn.Module):
    """checkpoint=True: the input is kept in 8 bits for the backward pass (gelu_glu_checkpoint).  output_checkpoint=True as well: forward
    returns (out, ActivationCheckpoint of out), for a layer that takes its input with one."""

    checkpoint = output_checkpoint = False

    def __init__(self, checkpoint=False, output_checkpoint=False):
        super().__init__()
        if output_checkpoint and not checkpoint:
            raise RuntimeError("GELUglu: output_checkpoint without checkpoint is not supported")
        if checkpoint:
            self.checkpoint, self.output_checkpoint = True, bool(output_checkpoint)

    def forward(self, x):
        if not self.checkpoint:
            return gelu_glu.apply(x)
        if not self.output_checkpoint:
            return gelu_glu_checkpoint.apply(x)
        out, values, scales = gelu_glu_checkpoint.apply(x, True)
        return out, ActivationCheckpoint._of(values, scales, out.shape, out.dtype)
