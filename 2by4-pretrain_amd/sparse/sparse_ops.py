"""Linear modules built on the dense-shaped 2:4 operators.

    MyLinear, my_linear          plain linear as an autograd.Function          (sparse/sparse_ops.py:8-46)
    SparseLinear, sparse_linear  same forward; dX uses an MVUE24 estimate of W  (sparse/sparse_ops.py:49-87)
    SoftThreshold                S-STE: soft-thresholded 2:4 weight x scale,
                                 straight-through gradient                      (README.md:233-243)
    SoftThresholdLinear          nn.Linear on SoftThreshold with the frozen
                                 scale of README.md:245-266 (the README calls
                                 this class SparseLinear as well)
    Sparse24                     STE magnitude pruning of the STEP recipe       (README.md:286-295)

The matrix products are torch's dense ones, as in the reference, except in SoftThresholdLinear under mixed precision: its weight and bias
gradients (`_linear16`), and its forward product and input gradient where their tiles fill the compute units (`_product16`).  There it
may keep its input in 8 bits for the backward pass (checkpoint=True, or a checkpoint that the operator in front made).
"""
from contextlib import nullcontext

import torch
import torch.nn.functional as F
from torch import autograd, nn
from torch.amp import custom_bwd, custom_fwd

from . import _native as N
from .activation_checkpoint import ActivationCheckpoint, as_checkpoint, checkpoint_weight_gradient, kept_of_input, says_that_nothing_is_kept
from .dense_ops import MVUE24_approx, soft_threshold24, sparse24

__all__ = ["MyLinear", "my_linear", "SparseLinear", "sparse_linear", "SoftThreshold", "SoftThresholdLinear", "Sparse24"]


def _forward(ctx, input, weight, bias):
    ctx.save_for_backward(input, weight, bias)
    ctx.shape = input.shape
    out = torch.mm(input.view(-1, input.shape[-1]), weight.t()).view(*input.shape[:-1], -1)
    return out if bias is None else out + bias


def _backward(ctx, grad_output, weight_for_dx):
    input, weight, bias = ctx.saved_tensors
    grad_input = grad_weight = grad_bias = None
    g2 = grad_output.reshape(-1, grad_output.shape[-1])
    if ctx.needs_input_grad[0]:
        grad_input = torch.mm(g2, weight_for_dx(weight)).view(ctx.shape)
    if ctx.needs_input_grad[1]:
        grad_weight = torch.mm(g2.t(), input.view(-1, input.shape[-1]))
    if ctx.needs_input_grad[2]:
        grad_bias = g2.sum(0)
    return grad_input, grad_weight, grad_bias


class my_linear(autograd.Function):
    @staticmethod
    @custom_fwd(device_type="cuda")
    def forward(ctx, input, weight, bias):
        return _forward(ctx, input, weight, bias)

    @staticmethod
    @custom_bwd(device_type="cuda")
    def backward(ctx, grad_output):
        return _backward(ctx, grad_output, lambda w: w)


class sparse_linear(autograd.Function):
    """dX = dY . MVUE24(W^T)^T: the weight is pruned 2:4 along its output axis, unbiasedly."""

    @staticmethod
    @custom_fwd(device_type="cuda")
    def forward(ctx, input, weight, bias):
        return _forward(ctx, input, weight, bias)

    @staticmethod
    @custom_bwd(device_type="cuda")
    def backward(ctx, grad_output):
        return _backward(ctx, grad_output, lambda w: MVUE24_approx(w.t()).t())


class MyLinear(nn.Linear):
    def forward(self, x):
        return my_linear.apply(x, self.weight, self.bias)


class SparseLinear(nn.Linear):
    def forward(self, x):
        return sparse_linear.apply(x, self.weight, self.bias)


class SoftThreshold(autograd.Function):
    @staticmethod
    def forward(ctx, weight, scale):
        weight_sparse, _ = soft_threshold24(weight.detach())
        return weight_sparse * scale

    @staticmethod
    def backward(ctx, grad_output):
        return grad_output, None


class _soft_threshold16(autograd.Function):
    """SoftThreshold followed by the cast of its result to a 16-bit dtype, in one pass over the float32 weight
    (three operators move 26 bytes per element, this one 6)."""

    @staticmethod
    def forward(ctx, weight, scale, dtype):
        out = torch.empty_like(weight, dtype=dtype)
        N.check(N.lib().tf24_soft_threshold24_scaled(weight.data_ptr(), weight.shape[0], weight.shape[1], scale.data_ptr() if scale.is_cuda else None,
                                                     0.0 if scale.is_cuda else scale.item(), out.data_ptr(), N.dtype_code(dtype), N.stream_ptr()))
        return out

    @staticmethod
    def backward(ctx, grad_output):
        return grad_output.float(), None, None


def _rows_for_kernels(t):
    """t [rows, cols] is an operand that tf24_grad_weight takes: rows contiguous, 16-byte aligned, of at most 2^20 columns.  (A
    batch of gradients that autograd maps over, is_grads_batched, has no storage of its own.)"""
    rows, cols = t.shape
    return (torch._C._has_storage(t) and not t.is_neg() and t.stride(1) == 1 and cols <= t.stride(0) <= 1 << 23 and t.stride(0) % 8 == 0
            and cols % 8 == 0 and cols <= 1 << 20 and t.data_ptr() % 16 == 0)


def _on_current_gpu(*tensors):
    """All of them are plain tensors on the GPU to whose stream the kernels go.  (What a saved-tensor hook hands back, or an overridden
    get_sparse_weights, may be anything; torch's operators say what they do not take.)"""
    device = tensors[0].device
    return device.index == torch.cuda.current_device() and all(type(t) in (torch.Tensor, nn.Parameter) and t.device == device for t in tensors if t is not None)


def _product16(x, weight, bias, transposed=False):
    """F.linear(x, weight, bias) of 16-bit operands, or (transposed) of a matrix x @ weight: by tf24_linear16 where it is the faster one, by the
    library otherwise.  Not seen by autograd."""
    rows, k = weight.shape[::-1 if transposed else 1] if weight.dim() == 2 else (0, 0)
    if (x.shape[-1] == k and x.numel() and x.dtype == weight.dtype and type(x) is torch.Tensor and N.lib().tf24_linear16_suits(rows, k, x.numel() // k)
            and _on_current_gpu(x, weight, bias) and _rows_for_kernels(weight)
            and (bias is None or (bias.dtype == x.dtype and bias.shape == (rows,) and bias.is_contiguous() and not bias.is_neg()))):
        flat = x.reshape(-1, k)
        if _rows_for_kernels(flat) and max(flat.stride(0), weight.stride(0)) <= 1 << 22:
            out = torch.empty((*x.shape[:-1], rows), dtype=x.dtype, device=x.device)
            N.check(N.lib().tf24_linear16(weight.data_ptr(), weight.stride(0), transposed, flat.data_ptr(), flat.stride(0), N.dtype_code(x.dtype), rows, k,
                                          flat.shape[0], out.data_ptr(), rows, N.ptr(bias), N.stream_ptr()))
            return out
    return torch.mm(x, weight) if transposed else F.linear(x, weight, bias)


class _straight_through(autograd.Function):
    """`value`, which was made from the float32 `weight`, with the gradient of the weight."""

    @staticmethod
    def forward(ctx, weight, value):
        return value.view_as(value)

    @staticmethod
    def backward(ctx, grad_output):
        return grad_output.float(), None


class _place_of(autograd.Function):
    """One element, expanded to the shape of `weight`, from which gradients go where the weight's do: kept in the weight's place by
    a graph that leads to it but does not need its values (which may change, or be freed, before the backward pass)."""

    @staticmethod
    def forward(ctx, weight):
        return weight.new_empty(()).expand(weight.shape)

    @staticmethod
    def backward(ctx, grad_output):
        return grad_output


class _linear16(autograd.Function):
    """y = x W^T + b of 16-bit operands, with dW = dY^T x and db = sum(dY) from one pass of tf24_grad_weight.

    The products of dW are short and wide (3072 x 768 over 12288 tokens), for which the library's kernel cuts no pieces
    along the tokens and leaves 40 % of the compute units idle: 110 to 140 us and 20 to 29 us for db, 62 to 70 us together here.
    With db the pass over dY that is saved decides from 256 tokens on (GPU time, bf16, here and in the library: 512 x 512 over 256
    tokens 8.7 and 15.5 us, 1024 x 1024 over 1024 18.6 and 21.5, 768 x 3072 over 1024 19.1 and 25.1, 11008 x 4096 over 12288 901
    and 1199).  Without it, with float32 results and the library's cast, every output measured from 512 x 512 to 11008 x 4096 is the
    faster one here from 4096 tokens on (4096 x 1024 50.0 and 51.0; with 16-bit results 48.9 and 45.6, the one exception); below
    that some are the library's (1024 x 1024 over 1024 17.0 and 14.4, over 2048 21.0 and 19.1) and some are not (3072 x 768 over
    1024 17.6 and 20.0, over 3000 26.7 and 42.7)."""

    MIN_TOKENS, MIN_TOKENS_NO_BIAS = 256, 4096

    @staticmethod
    def forward(ctx, x, weight, bias, kept=None):
        needs = ctx.needs_input_grad
        ctx.save_for_backward(*_keep(ctx, x, kept, needs[1]), weight if needs[0] else None)
        return _product16(x, weight, bias)

    @staticmethod
    def backward(ctx, grad_output):
        x, weight = _kept(ctx)
        return *_linear16_backward(grad_output, x, weight, *ctx.needs_input_grad[:3]), None


def _keep(ctx, x, kept, needed):
    """The tensors that are saved of a layer's input x for its weight gradient: x, or what is kept of it in 8 bits (kept: True, or its checkpoint)."""
    ctx.kept = None
    if not needed or kept is None:
        return (x if needed else None,)
    kept = as_checkpoint(x, kept)
    ctx.kept = kept.shape, kept.dtype
    return kept.values, kept.scales


def _kept(ctx):
    """The saved tensors with the input as _keep took it in front: itself, its checkpoint or None."""
    if ctx.kept is None:
        return ctx.saved_tensors
    values, scales, *others = ctx.saved_tensors
    return ActivationCheckpoint(values, scales, *ctx.kept), *others


def _linear16_backward(grad_output, x, weight, need_input, need_weight, need_bias, dtype=None):
    """dtype: of the gradients of weight and bias, the operands' (None) or float32"""
    grad_input = grad_weight = grad_bias = None
    g = grad_output.reshape(-1, grad_output.shape[-1])
    # where a graph of the gradients is wanted (double backward), or a tangent, mode or transform has come up since the
    # forward pass: torch's operators, which those know
    kernels = not torch.is_grad_enabled() and N.plain_eager() and type(g) is torch.Tensor
    if need_weight and isinstance(x, ActivationCheckpoint):
        if torch.is_grad_enabled():
            raise RuntimeError("a graph of the gradients of a layer that keeps its input in 8 bits is not supported")
        grad_weight, grad_bias = checkpoint_weight_gradient(grad_output, x, need_bias, dtype)
    elif need_weight:
        x = x.reshape(-1, x.shape[-1])
        if (kernels and g.dtype == x.dtype and g.shape[0] == x.shape[0] and _on_current_gpu(g, x) and _rows_for_kernels(g) and _rows_for_kernels(x)
                and g.shape[0] >= (_linear16.MIN_TOKENS if need_bias else _linear16.MIN_TOKENS_NO_BIAS)):
            grad_weight, grad_bias = _grad_weight(g, x, need_bias, dtype)
    # (entered only where autocast is on: two layers' backward passes 186 -> 172 us of host time)
    with torch.autocast(device_type="cuda", enabled=False) if torch.is_autocast_enabled("cuda") else nullcontext():
        if need_input:
            grad_input = _product16(g, weight, None, True) if kernels else torch.mm(g, weight)
            grad_input = grad_input.view(*grad_output.shape[:-1], weight.shape[1])
        if need_weight and grad_weight is None:
            grad_weight = torch.mm(g.t(), x)
            if dtype is not None:
                grad_weight = grad_weight.to(dtype)
        if need_bias and grad_bias is None:
            grad_bias = g.sum(0)
            if dtype is not None:
                grad_bias = grad_bias.to(dtype)
    return grad_input, grad_weight, grad_bias


class _soft_threshold_linear16(autograd.Function):
    """_linear16 on the soft threshold of a float32 weight, with a float32 bias: _soft_threshold16, the cast of the bias and
    _linear16 in one.  The threshold's kernel rounds the bias as well, and the gradients leave the kernels in float32, with
    the values that 16-bit ones would be widened to: four casts of 3 to 5 us a layer less."""

    @staticmethod
    def forward(ctx, x, weight, scale, bias, dtype, kept=None):
        rows, cols = weight.shape
        weight16 = torch.empty_like(weight, dtype=dtype)
        bias16 = None if bias is None else torch.empty_like(bias, dtype=dtype)
        on_device = scale.data_ptr() if scale.is_cuda else None
        value, code, lib = 0.0 if scale.is_cuda else scale.item(), N.dtype_code(dtype), N.lib()
        if bias is None:
            N.check(lib.tf24_soft_threshold24_scaled(weight.data_ptr(), rows, cols, on_device, value, weight16.data_ptr(), code, N.stream_ptr()))
        else:
            N.check(lib.tf24_soft_threshold24_scaled_bias(weight.data_ptr(), rows, cols, on_device, value, weight16.data_ptr(), bias.data_ptr(),
                                                          bias16.data_ptr(), code, N.stream_ptr()))
        needs = ctx.needs_input_grad
        source = None
        if needs[0] and needs[1] and weight.grad_fn is not None:
            with torch.enable_grad():
                source = _place_of.apply(weight)
        ctx.save_for_backward(*_keep(ctx, x, kept, needs[1]), weight16 if needs[0] else None, source)
        return _product16(x, weight16, bias16)

    @staticmethod
    def backward(ctx, grad_output):
        x, weight16, source = _kept(ctx)
        needs = ctx.needs_input_grad
        if weight16 is not None and needs[1] and torch.is_grad_enabled():
            # a graph of the gradients leads on to the weight (a parameter is held by the graph itself)
            weight16 = _straight_through.apply(ctx.next_functions[1][0].variable if source is None else source, weight16)
        grad_input, grad_weight, grad_bias = _linear16_backward(grad_output, x, weight16, needs[0], needs[1], needs[3], torch.float32)
        return grad_input, grad_weight, None, grad_bias, None, None


def _grad_weight(g, x, with_bias, dtype=None):
    """dtype: the operands' (None), or float32 for the same values widened"""
    tokens, m = g.shape
    n = x.shape[1]
    lib = N.lib()
    grad_weight = torch.empty((m, n), dtype=dtype or g.dtype, device=g.device)
    grad_bias = torch.empty(m, dtype=dtype or g.dtype, device=g.device) if with_bias else None
    nbytes = lib.tf24_grad_weight_workspace_bytes(tokens, m, n)
    workspace = torch.empty(nbytes, dtype=torch.uint8, device=g.device) if nbytes else None
    call = lib.tf24_grad_weight_f32 if dtype is torch.float32 else lib.tf24_grad_weight
    N.check(call(g.data_ptr(), g.stride(0), x.data_ptr(), x.stride(0), N.dtype_code(g.dtype), tokens, m, n,
                 grad_weight.data_ptr(), N.ptr(grad_bias), N.ptr(workspace), nbytes, N.stream_ptr()))
    return grad_weight, grad_bias


def _takes_linear16(x, weight, bias):
    """F.linear(x, weight, bias) is a product of 16-bit matrices once autocast has cast its arguments, of plain tensors on one GPU."""
    return (torch.is_autocast_enabled("cuda") and torch.get_autocast_dtype("cuda") in (torch.float16, torch.bfloat16)
            and all(type(t) in (torch.Tensor, nn.Parameter) and t.is_cuda and t.get_device() == weight.get_device() and t.dtype in (torch.float32, torch.float16, torch.bfloat16)
                    for t in (x, weight, bias) if t is not None)
            and x.dim() >= 2 and x.numel() > 0 and x.is_contiguous() and x.shape[-1] == weight.shape[1] and N.plain_eager())


class SoftThresholdLinear(nn.Linear):
    """checkpoint=True: where autocast makes the layer's products 16-bit ones, its input is kept in 8 bits for the weight's gradient
    (which is the one at the kept values).  forward(x, checkpoint) takes the ActivationCheckpoint of x (as autocast casts it) that the operator
    in front made, True or False for this call, whatever the layer's own setting."""

    checkpoint = False

    def __init__(self, in_features: int, out_features: int, bias: bool = True, device=None, dtype=None, checkpoint: bool = False):
        super().__init__(in_features, out_features, bias=bias, device=device, dtype=dtype)
        if checkpoint:
            self.checkpoint = True
        self.register_buffer("scale", torch.tensor(0.0))

    def get_sparse_weights(self):
        return SoftThreshold.apply(self.weight, self.scale)

    @torch.no_grad()
    def init_scale(self):
        """scale = <w, S(w)> / <S(w), S(w)>: the least-squares fit of scale * S(w) to w."""
        weight = self.weight.detach()
        weight_sparse, _ = soft_threshold24(weight)
        ws = torch.flatten(weight_sparse).float()
        scale = torch.dot(torch.flatten(weight).float(), ws) / torch.dot(ws, ws)
        self.scale.copy_(scale)
        self.weight.scale = self.scale

    def forward(self, x, checkpoint=None):
        weight, scale, bias = self.weight, self.scale, self.bias
        if not _takes_linear16(x, weight, bias):
            says_that_nothing_is_kept(self, checkpoint, "with contiguous GPU tensors under autocast to 16 bits only, and where no mode or transform stands around "
                                      "the call (torch.set_default_device is one)")
            return F.linear(x, self.get_sparse_weights(), bias)
        kept = kept_of_input(checkpoint, self.checkpoint)
        dtype = torch.get_autocast_dtype("cuda")                   # (what autocast does to the arguments of F.linear)
        if (getattr(self.get_sparse_weights, "__func__", None) is SoftThresholdLinear.get_sparse_weights and weight.dtype == torch.float32
                and weight.is_contiguous() and not weight.is_neg() and weight.shape[1] % 8 == 0 and weight.data_ptr() % 16 == 0
                and type(scale) is torch.Tensor and scale.dtype == torch.float32 and scale.dim() == 0 and scale.device in (weight.device, torch.device("cpu"))
                and not scale.requires_grad and not scale.is_neg()):
            if bias is None or (bias.dtype == torch.float32 and bias.is_contiguous() and not bias.is_neg() and bias.shape == weight.shape[:1]):
                return _soft_threshold_linear16.apply(x.to(dtype), weight, scale, bias, dtype, *(() if kept is None else (kept,)))
            weight = _soft_threshold16.apply(weight, scale, dtype)
        else:
            weight = self.get_sparse_weights().to(dtype)
        return _linear16.apply(x.to(dtype), weight, None if bias is None else bias.to(dtype), *(() if kept is None else (kept,)))


class Sparse24(autograd.Function):
    @staticmethod
    def forward(ctx, weight):
        weight_sparse, _ = sparse24(weight)
        return weight_sparse

    @staticmethod
    def backward(ctx, grad_output):
        return grad_output
