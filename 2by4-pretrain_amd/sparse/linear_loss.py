"""A language model's head together with its loss: the logits of a vocabulary are never kept.

    linear_cross_entropy(x, weight, target, ...)                 softmax cross entropy of the logits x W^T + b
    linear_distillation(x, weight, indices, teacher_logits, ...) divergence from a teacher of which the largest logits of each token are known
    VocabularyLinear                                             the head as a module: logits, or one of the two losses

The logits of 12 sequences of 1024 tokens over 50304 words are 2.5 GB in float32, and torch's own loss keeps them, their
softmax and the gradient of both.  Here the forward pass keeps the logarithm of the sum of exponentials of each token, and the backward pass forms the
logits once more, a piece of the vocabulary at a time (2 GiB of 16-bit gradients at most, which are gone when it returns).  Tokens that do not count take no part
in the products.
The reference has no such operators; its recipe trains models that bring their own head (README.md:56-118).
"""
from contextlib import nullcontext

import torch
from torch import autograd, nn

from . import _native as N

__all__ = ["linear_cross_entropy", "linear_distillation", "VocabularyLinear"]

_REDUCTIONS = {"mean": N.REDUCE_MEAN, "sum": N.REDUCE_SUM, "none": N.REDUCE_NONE}
_HALF = (torch.float16, torch.bfloat16)
_TYPES = (torch.float32, torch.float16, torch.bfloat16)
_MAX_ENTRIES = 1024


def _on_device_of(t):
    """The tensor's device as the current one, for the sizes of workspaces and the launches that they are for."""
    return nullcontext() if t.get_device() == torch.cuda.current_device() else torch.cuda.device(t.device)


class _linear_loss(autograd.Function):
    """`dtype` is the operands'; a float32 weight is cast to it here, and gets a float32 gradient."""

    @staticmethod
    def forward(ctx, x, weight, bias, dtype, target, ignore_index, indices, teacher_logits, teacher_lse, smoothing, z_loss, temperature, reduction):
        weight16 = weight.to(dtype)
        flat, ldx = N.as_rows(x)
        w, ldw = N.as_rows(weight16)
        bias = None if bias is None else bias.resolve_neg().contiguous()
        tokens, width, words = x.shape[:-1].numel(), x.shape[-1], weight.shape[0]
        entries = 0 if indices is None else indices.shape[-1]
        loss = torch.empty(x.shape[:-1] if reduction == N.REDUCE_NONE else (), dtype=torch.float32, device=x.device)
        ctx.call = x.shape, dtype, x.device, weight.shape, weight.dtype, None if bias is None else (bias.shape, bias.dtype), entries, smoothing, z_loss, temperature, reduction
        if tokens == 0:
            ctx.save_for_backward()
            return loss.zero_()
        lib, code, ptr = N.lib(), N.dtype_codes, N.ptr
        state = torch.empty(lib.tf24_linear_loss_state_bytes(tokens, entries), dtype=torch.uint8, device=x.device)
        ld_indices = ld_teacher = 0
        if entries:
            indices, ld_indices = N.as_rows(indices)
            teacher_logits, ld_teacher = N.as_rows(teacher_logits)
        with _on_device_of(x):
            nbytes = lib.tf24_linear_loss_forward_workspace_bytes(tokens, width, words, entries, smoothing != 0.0, w.data_ptr(), ldw)
            workspace = torch.empty(nbytes, dtype=torch.uint8, device=x.device)
            N.check(lib.tf24_linear_loss_forward(
                flat.data_ptr(), ldx, w.data_ptr(), ldw, ptr(bias), N.F32 if bias is None else code[bias.dtype], code[dtype], tokens, width, words, ptr(target),
                ignore_index, ptr(indices), ld_indices, ptr(teacher_logits), ld_teacher, code[teacher_logits.dtype] if entries else N.F32, ptr(teacher_lse), entries,
                smoothing, z_loss, 1.0 / temperature, reduction, loss.data_ptr(), state.data_ptr(), state.numel(), workspace.data_ptr(), nbytes, N.stream_ptr()))
        if any(ctx.needs_input_grad[:3]):
            ctx.save_for_backward(x, weight16, bias, state)
        return loss

    @staticmethod
    def backward(ctx, grad_loss):
        if torch.is_grad_enabled():
            raise RuntimeError("a graph of the gradients of linear_cross_entropy and linear_distillation is not supported")
        shape, dtype, device, weight_shape, weight_dtype, bias_as, entries, smoothing, z_loss, temperature, reduction = ctx.call
        needs = ctx.needs_input_grad
        tokens, width, words = shape[:-1].numel(), shape[-1], weight_shape[0]
        make = torch.empty if tokens else torch.zeros
        dx = make(shape, dtype=dtype, device=device) if needs[0] else None
        dw = make(weight_shape, dtype=weight_dtype, device=device) if needs[1] else None
        db = make(bias_as[0], dtype=bias_as[1], device=device) if needs[2] else None
        if tokens:
            x, weight, bias, state = ctx.saved_tensors
            lib, code, ptr, what = N.lib(), N.dtype_codes, N.ptr, "linear_cross_entropy and linear_distillation"
            grad_loss = N.as_it_was(what, grad_loss, shape[:-1] if reduction == N.REDUCE_NONE else (), torch.float32, device).resolve_neg().contiguous()
            flat, ldx = N.as_rows(N.as_it_was(what, x, shape, dtype, device))
            w, ldw = N.as_rows(N.as_it_was(what, weight, weight_shape, dtype, device))
            if bias is not None:
                bias = N.as_it_was(what, bias, *bias_as, device).resolve_neg().contiguous()
            state = N.as_it_was(what, state, (lib.tf24_linear_loss_state_bytes(tokens, entries),), torch.uint8, device).contiguous()
            with _on_device_of(flat):
                nbytes = lib.tf24_linear_loss_backward_workspace_bytes(tokens, width, words, entries, smoothing != 0.0, w.data_ptr(), ldw, needs[0], needs[1], needs[2])
                workspace = torch.empty(nbytes, dtype=torch.uint8, device=device)
                N.check(lib.tf24_linear_loss_backward(
                    grad_loss.data_ptr(), flat.data_ptr(), ldx, w.data_ptr(), ldw, ptr(bias), N.F32 if bias is None else code[bias.dtype], code[dtype], tokens, width,
                    words, entries, smoothing, z_loss, 1.0 / temperature, reduction, state.data_ptr(), state.numel(), ptr(dx), ptr(dw), code[weight_dtype], ptr(db),
                    workspace.data_ptr(), nbytes, N.stream_ptr()))
        return dx, dw, db, *(None,) * 10


def _operands(fn, x, weight, bias):
    """(x, the type of the products): under autocast x is cast to its type, and the weight inside; without it both have one 16-bit type."""
    named = (("x", x), ("weight", weight)) + ((("bias", bias),) if bias is not None else ())
    for name, t in named:
        if not isinstance(t, torch.Tensor):
            raise RuntimeError(f"{fn}: {name} is {type(t).__name__}, not a tensor")
    for name, t in named:
        if not t.is_cuda:
            raise RuntimeError(f"{fn}: only CUDA tensors are supported ({name} is on {t.device})")
        if t.dtype not in _TYPES:
            raise RuntimeError(f"{fn}: dtype {t.dtype} of {name} is not supported")
    if x.dim() == 0 or weight.dim() != 2 or x.shape[-1] != weight.shape[1] or not 1 <= x.shape[-1] <= 1 << 16 or not 1 <= weight.shape[0] <= 1 << 22:
        raise RuntimeError(f"{fn}: x {tuple(x.shape)} does not suit a weight {tuple(weight.shape)} (up to 2^16 columns, 2^22 words)")
    if bias is not None and bias.shape != weight.shape[:1]:
        raise RuntimeError(f"{fn}: a bias {tuple(bias.shape)} does not suit a weight {tuple(weight.shape)}")
    if any(t is not None and t.device != x.device for t in (weight, bias)):
        raise RuntimeError(f"{fn}: x, weight and bias are on different devices")
    if x.shape[:-1].numel() > 1 << 22:
        raise RuntimeError(f"{fn}: {x.shape[:-1].numel()} tokens, at most 2^22 are supported")
    if torch.is_autocast_enabled("cuda") and torch.get_autocast_dtype("cuda") in _HALF:
        dtype = torch.get_autocast_dtype("cuda")
        if weight.dtype not in (dtype, torch.float32):
            weight = weight.to(dtype)
        return x.to(dtype), weight, dtype
    if x.dtype not in _HALF or weight.dtype not in (x.dtype, torch.float32):
        raise RuntimeError(f"{fn}: x {x.dtype} with a weight {weight.dtype} is not supported: float16 or bfloat16, the weight of that type or float32 (or autocast)")
    return x, weight, x.dtype


def _number(fn, name, value, low, high):
    if isinstance(value, torch.Tensor) or not isinstance(value, (int, float)) or not low <= value <= high:
        raise RuntimeError(f"{fn}: {name} {value!r} is not a number between {low} and {high}")
    return float(value)


def _beside(fn, name, t, shape, device, floating):
    if not isinstance(t, torch.Tensor):
        raise RuntimeError(f"{fn}: {name} is {type(t).__name__}, not a tensor")
    if t.shape != shape or t.device != device:
        raise RuntimeError(f"{fn}: {name} {tuple(t.shape)} on {t.device} does not suit tokens {tuple(shape)} on {device}")
    if t.dtype not in _TYPES if floating else (t.dtype.is_floating_point or t.dtype.is_complex or t.dtype == torch.bool):
        raise RuntimeError(f"{fn}: dtype {t.dtype} of {name} is not supported")
    if floating and t.requires_grad and torch.is_grad_enabled():
        raise RuntimeError(f"{fn}: no gradient goes to {name}, detach it")
    return t


def _reduction(fn, reduction):
    if reduction not in _REDUCTIONS:
        raise RuntimeError(f"{fn}: reduction {reduction!r} is not supported (mean, sum, none)")
    return _REDUCTIONS[reduction]


def linear_cross_entropy(x, weight, target, bias=None, *, ignore_index=-100, label_smoothing=0.0, z_loss=0.0, reduction="mean"):
    """Softmax cross entropy of the logits z = x W^T + b, float32, with lse = log(sum(exp(z))) of a token

        (1 - label_smoothing) (lse - z[target]) + label_smoothing (lse - mean(z)) + z_loss lse^2

    x [..., columns] and weight [words, columns] are float16 or bfloat16 (up to 2^16 columns, 2^22 words, 2^22 tokens); a float32 weight is cast to x's
    type and gets a float32 gradient, and under autocast x is cast as well.  bias [words] of any floating type (-inf: a word that is never
    expected, as behind the end of a padded vocabulary), target [...] of whole numbers.  Tokens whose target is ignore_index do not count: their loss and
    gradient are zero, and nothing of their x is read.  reduction "mean" is over the tokens that count (of none: 0), "sum", or "none": [...].  A target that is no
    word's number makes its loss and the gradients NaN.  Gradients (once) for x, weight and bias, from the logits' rounded to 16 bits."""
    fn = "linear_cross_entropy"
    x, weight, dtype = _operands(fn, x, weight, bias)
    target = _beside(fn, "target", target, x.shape[:-1], x.device, False)
    reduction = _reduction(fn, reduction)
    smoothing, z_loss = _number(fn, "label_smoothing", label_smoothing, 0.0, 1.0), _number(fn, "z_loss", z_loss, 0.0, 1e30)
    if not isinstance(ignore_index, int) or not -2**63 <= ignore_index < 2**63:
        raise RuntimeError(f"{fn}: ignore_index {ignore_index!r} is not a whole number of 64 bits")
    return _linear_loss.apply(x, weight, bias, dtype, target.long().resolve_neg().contiguous(), ignore_index, None, None, None, smoothing, z_loss, 1.0, reduction)


def linear_distillation(x, weight, indices, teacher_logits, bias=None, *, teacher_lse=None, temperature=1.0, reduction="mean"):
    """Divergence of the student's distribution, softmax of u = (x W^T + b) / temperature, from a teacher's of which some words are listed:

        sum_k q_k (log q_k - u[index_k] + lse(u)),    q_k = exp(logit_k / temperature - teacher_lse)

    indices [..., entries] (whole numbers) and teacher_logits [..., entries] are the words and the teacher's logits of each token, in any order, 1 to 1024
    of them.  teacher_lse [...] is the logarithm of the sum of exponentials of all of the teacher's logits / temperature; without it the listed words
    share all of the probability.  An entry with a negative word is unused, one with a word past the last makes its token's loss and the gradients NaN; a token without a used entry above -inf does not count: loss and gradient
    zero, nothing of its x read.  A word listed twice has the probability of both.  x, weight, bias, reduction and gradients as in linear_cross_entropy; none for
    the teacher's.  (A loss that is to keep its size over temperatures is multiplied by temperature^2 by the caller.)"""
    fn = "linear_distillation"
    x, weight, dtype = _operands(fn, x, weight, bias)
    lead = x.shape[:-1]
    if not isinstance(indices, torch.Tensor) or indices.dim() == 0 or not 1 <= indices.shape[-1] <= _MAX_ENTRIES:
        raise RuntimeError(f"{fn}: indices must be a tensor with 1 to {_MAX_ENTRIES} entries of each token")
    shape = (*lead, indices.shape[-1])
    indices = _beside(fn, "indices", indices, shape, x.device, False)
    teacher_logits = _beside(fn, "teacher_logits", teacher_logits, shape, x.device, True)
    if teacher_lse is not None:
        teacher_lse = _beside(fn, "teacher_lse", teacher_lse, lead, x.device, True).detach().float().resolve_neg().contiguous()
    reduction = _reduction(fn, reduction)
    temperature = _number(fn, "temperature", temperature, 1e-6, 1e6)
    return _linear_loss.apply(x, weight, bias, dtype, None, 0, indices.long(), teacher_logits.detach(), teacher_lse, 0.0, 0.0, temperature, reduction)


class VocabularyLinear(nn.Linear):
    """A language model's head.  forward(x) are its logits; forward(x, target, ...) is linear_cross_entropy, forward(x, indices=, teacher_logits=, ...)
    linear_distillation with its weight and bias.  The weight may be tied to an embedding's."""

    def __init__(self, in_features: int, out_features: int, bias: bool = False, device=None, dtype=None):
        super().__init__(in_features, out_features, bias=bias, device=device, dtype=dtype)

    def forward(self, x, target=None, *, indices=None, teacher_logits=None, **how):
        if (target is not None and indices is not None) or (indices is None) != (teacher_logits is None):
            raise RuntimeError("VocabularyLinear: either a target, or indices with teacher_logits")
        if target is not None:
            return linear_cross_entropy(x, self.weight, target, self.bias, **how)
        if indices is not None:
            return linear_distillation(x, self.weight, indices, teacher_logits, self.bias, **how)
        if how:
            raise RuntimeError(f"VocabularyLinear: {', '.join(how)} without a target or a teacher")
        return super().forward(x)
