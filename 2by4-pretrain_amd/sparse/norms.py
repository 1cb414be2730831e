"""Norms before and behind the blocks of a transformer, with the gate and the residual addition between them.

    residual_norm(residual, y, ...)   out = residual_scale * residual + gate * N_post(y),  n = N_pre(out)
    block_norm(x, weight, ...)        n = N(x): the norm before the first block
    ResidualNorm, BlockNorm           the modules around them

One pass over memory each way where a model's own modules take four or more (norm, gate, addition, norm).  The residual stream may be
float32 between 16-bit blocks, or of the blocks' type; `out` has the stream's type and is rounded to it before it is normalised, `n` has
the block's.  With checkpoint=True n is also kept in 8 bits (ActivationCheckpoint) in the same pass, for a layer that takes one.
The reference has no such operators; its recipe trains models that bring their own (README.md:56-118).
"""
import torch
from torch import autograd, nn

from . import _native as N
from .activation_checkpoint import ActivationCheckpoint, empty_checkpoint

__all__ = ["block_norm", "residual_norm", "BlockNorm", "ResidualNorm"]

_KINDS = {None: N.NORM_NONE, "rms": N.NORM_RMS, "layer": N.NORM_LAYER}
_TYPES = (torch.float32, torch.float16, torch.bfloat16)
_MAX_COLS = 16384


def _forward(x, y, gate, rows_per_gate, post_weight, post_bias, pre_weight, pre_bias, scale, post_kind, pre_kind, eps, block_dtype, keep, with_stats):
    """(out, n, stats, values, scales), None for what is not formed"""
    flat, ld = N.as_rows(x)
    shape = x.shape
    rows, cols = shape[:-1].numel(), shape[-1]
    y2 = out = n = stats = values = scales = None
    ld_y = ld_gate = 0
    param = post_weight if post_weight is not None else post_bias if post_bias is not None else pre_weight if pre_weight is not None else pre_bias
    if y is not None:
        y2, ld_y = N.as_rows(y)
        out = torch.empty_like(x) if flat is x else torch.empty(shape, dtype=x.dtype, device=x.device)
    if gate is not None:
        gate, ld_gate = N.as_rows(gate)
    if pre_kind:
        n = torch.empty_like(y) if y is not None and y2 is y else torch.empty(shape, dtype=block_dtype, device=x.device)
        if keep:
            values, scales = empty_checkpoint(rows, cols, x.device)
    if with_stats and (post_kind or pre_kind):
        stats = torch.empty((4, rows), dtype=torch.float32, device=x.device)
    code, ptr = N.dtype_codes, N.ptr
    N.launch(x, N.lib().tf24_block_norm_forward, flat.data_ptr(), ld, ptr(y2), ld_y, code[x.dtype], code[block_dtype], rows, cols,
             ptr(gate), N.F32 if gate is None else code[gate.dtype], ld_gate, rows_per_gate, ptr(post_weight), ptr(post_bias), ptr(pre_weight),
             ptr(pre_bias), N.F32 if param is None else code[param.dtype], post_kind, pre_kind, scale, eps, ptr(out), ptr(n), ptr(stats),
             ptr(values), ptr(scales))
    return out, n, stats, values, scales


class _block_norm(autograd.Function):
    @staticmethod
    def forward(ctx, x, y, gate, post_weight, post_bias, pre_weight, pre_bias, rows_per_gate, scale, post_kind, pre_kind, eps, block_dtype, keep):
        ctx.set_materialize_grads(False)
        out, n, stats, values, scales = _forward(x, y, gate, rows_per_gate, post_weight, post_bias, pre_weight, pre_bias, scale, post_kind, pre_kind, eps,
                                                 block_dtype, keep, True)
        residual = y is not None
        ctx.save_for_backward((out if residual else x) if pre_kind else None, y if post_kind or (gate is not None and ctx.needs_input_grad[2]) else None, gate,
                              post_weight, post_bias, pre_weight, stats)
        param = next((p for p in (post_weight, post_bias, pre_weight, pre_bias) if p is not None), None)
        ctx.call = (x.shape, x.dtype, x.device, block_dtype, None if param is None else param.dtype, None if gate is None else (gate.shape, gate.dtype), residual,
                    rows_per_gate, scale, post_kind, pre_kind)
        if values is not None:
            ctx.mark_non_differentiable(values, scales)
        return out, n, values, scales

    @staticmethod
    def backward(ctx, grad_out, grad_n, _values, _scales):
        if torch.is_grad_enabled():
            raise RuntimeError("a graph of the gradients of block_norm and residual_norm is not supported")
        h, y, gate, post_weight, post_bias, pre_weight, stats = ctx.saved_tensors
        shape, stream_dtype, device, block_dtype, param_dtype, gate_as, residual, rows_per_gate, scale, post_kind, pre_kind = ctx.call
        needs = ctx.needs_input_grad
        if grad_n is None:
            pre_kind = N.NORM_NONE                                 # only the stream goes on
            if grad_out is None:
                return (None,) * 14
        rows, cols = shape[:-1].numel(), shape[-1]

        def as_it_was(t, shape, dtype):
            return N.as_it_was("block_norm and residual_norm", t, shape, dtype, device)

        grad_out = None if grad_out is None else as_it_was(grad_out if grad_out.dtype == stream_dtype else grad_out.to(stream_dtype), shape, stream_dtype)
        grad_n = None if grad_n is None else as_it_was(grad_n if grad_n.dtype == block_dtype else grad_n.to(block_dtype), shape, block_dtype)
        h, y = as_it_was(h, shape, stream_dtype), as_it_was(y, shape, block_dtype)
        gate = None if gate is None else as_it_was(gate, *gate_as)
        post_weight, post_bias, pre_weight = (None if t is None else as_it_was(t, (cols,), param_dtype).resolve_neg().contiguous() for t in (post_weight, post_bias, pre_weight))
        stats = None if stats is None else as_it_was(stats, (4, rows), torch.float32).contiguous()
        make = torch.empty if rows else torch.zeros                # (sums over no rows)
        grad_x = grad_y = grad_gate = None
        if needs[0]:
            grad_x = torch.empty(shape, dtype=stream_dtype, device=device)
        if needs[1]:
            grad_y = torch.empty(shape, dtype=block_dtype, device=device)
        if needs[2]:
            grad_gate = make(gate.shape, dtype=gate.dtype, device=device)
        grads = [None] * 4
        for i, kind in enumerate((post_kind, post_kind, pre_kind, pre_kind)):
            if needs[3 + i] and kind:
                grads[i] = make(cols, dtype=param_dtype, device=device)
        sums = needs[2] or needs[3] or needs[4] or needs[5] or needs[6]
        if rows:
            lib, code, ptr = N.lib(), N.dtype_codes, N.ptr
            dout = dn = h2 = y2 = gate2 = workspace = None
            ld_dout = ld_dn = ld_h = ld_y = ld_gate = nbytes = 0
            if grad_out is not None:
                dout, ld_dout = N.as_rows(grad_out)
            if pre_kind:
                dn, ld_dn = N.as_rows(grad_n)
                h2, ld_h = N.as_rows(h)
            if y is not None:
                y2, ld_y = N.as_rows(y)
            if gate is not None:
                gate2, ld_gate = N.as_rows(gate)
            if sums:
                nbytes = lib.tf24_block_norm_backward_workspace_bytes(rows, cols, rows if gate is None else rows_per_gate)
                workspace = torch.empty(nbytes, dtype=torch.uint8, device=device)
            N.launch(dout if dn is None else dn, lib.tf24_block_norm_backward,
                     ptr(dout), ld_dout, ptr(dn), ld_dn, ptr(h2), ld_h, ptr(y2), ld_y,
                     code[stream_dtype], code[block_dtype], rows, cols, ptr(gate2), N.F32 if gate is None else code[gate.dtype],
                     ld_gate, rows_per_gate, ptr(post_weight), ptr(post_bias), ptr(pre_weight),
                     N.F32 if param_dtype is None else code[param_dtype], post_kind, pre_kind, residual, scale, ptr(stats), ptr(grad_x),
                     ptr(grad_y), ptr(grad_gate), ptr(grads[0]), ptr(grads[1]), ptr(grads[2]), ptr(grads[3]), ptr(workspace), nbytes)
        return grad_x, grad_y, grad_gate, *grads, None, None, None, None, None, None, None


def _parameters(fn, x, *params):
    """The parameters, contiguous and all of one type (float32 where they differ)."""
    cols, device, dtype, plain = x.shape[-1], x.get_device(), None, True
    for p in params:
        if p is None:
            continue
        own = p.dtype
        if p.shape != (cols,) or own not in _TYPES or p.get_device() != device:
            raise RuntimeError(f"{fn}: a weight or bias {tuple(p.shape)} {p.dtype} on {p.device} does not suit {cols} columns on {x.device}")
        plain = plain and (dtype is None or own == dtype) and p.is_contiguous() and not p.is_neg()
        dtype = own
    if plain:
        return params
    mixed = any(p is not None and p.dtype != dtype for p in params)
    return [None if p is None else (p.float() if mixed else p).resolve_neg().contiguous() for p in params]


def _wide(gate):
    """A gate that is spelled out, in float32 where it gets a gradient: that of every element is added up behind the kernel, and rounded to the gate's type then."""
    return gate.float() if gate.requires_grad and torch.is_grad_enabled() else gate


def _gate(fn, gate, y):
    """(gate as rows of columns, the number of adjacent rows of y that each is for)"""
    cols, lead = y.shape[-1], y.shape[:-1]
    if gate.dtype not in _TYPES or gate.device != y.device:
        raise RuntimeError(f"{fn}: a gate {gate.dtype} on {gate.device} does not suit a tensor on {y.device}")
    if gate.shape == (cols,):
        return gate, lead.numel()
    if gate.dim() > y.dim() or any(g not in (1, s) for g, s in zip(gate.shape[::-1], y.shape[::-1])):
        raise RuntimeError(f"{fn}: a gate {tuple(gate.shape)} does not broadcast to {tuple(y.shape)}")
    if gate.dim() == 0 or gate.shape[-1] != cols:
        gate = _wide(gate).expand(*gate.shape[:-1], cols)
    own = (1,) * (y.dim() - gate.dim()) + gate.shape[:-1]
    # dimensions that the gate follows, then dimensions that share it; any other order is spelled out row by row
    shared = len(lead)
    while shared and own[shared - 1] == 1:
        shared -= 1
    if own[:shared] != lead[:shared]:
        gate, shared = _wide(gate).expand(y.shape), len(lead)
    return gate, lead[shared:].numel()


def _call(x, y, gate, rows_per_gate, post_weight, post_bias, pre_weight, pre_bias, scale, post_kind, pre_kind, eps, block_dtype, keep):
    """(out, n, checkpoint of n)"""
    graph = False
    if torch.is_grad_enabled():
        for t in (x, y, gate, post_weight, post_bias, pre_weight, pre_bias):
            if t is not None and t.requires_grad:
                graph = True
                break
    if graph or not N.plain_eager():
        out, n, values, scales = _block_norm.apply(x, y, gate, post_weight, post_bias, pre_weight, pre_bias, rows_per_gate, scale, post_kind, pre_kind, eps, block_dtype,
                                                   keep)
    else:
        out, n, _, values, scales = _forward(x, y, gate, rows_per_gate, post_weight, post_bias, pre_weight, pre_bias, scale, post_kind, pre_kind, eps, block_dtype,
                                             keep, False)
    return out, n, ActivationCheckpoint._of(values, scales, n.shape, n.dtype) if keep else None


def _ordinary(x, y, gate, post_weight, post_bias, pre_weight, pre_bias, scale, post_kind, pre_kind, eps, block_code, checkpoint):
    """_call from torch's C++ side, or None: a call to be looked at more closely."""
    calls = N.torch_calls()
    if calls is None or not N.plain_eager():
        return None
    post, pre = _KINDS.get(post_kind), _KINDS.get(pre_kind)
    if (post is None or pre is None or (not post and (post_weight is not None or post_bias is not None))
            or (not pre and (checkpoint or pre_weight is not None or pre_bias is not None))):
        return None
    result = calls.block_norm(x, y, gate, post_weight, post_bias, pre_weight, pre_bias, scale, post, pre, eps, block_code, bool(checkpoint))
    if result is None:
        return None
    out, n, values, scales = result
    return out, n, ActivationCheckpoint._of(values, scales, n.shape, n.dtype) if checkpoint else None


def _check_rows(fn, name, t):
    if not t.is_cuda:
        raise RuntimeError(f"{fn}: only CUDA tensors are supported")
    if t.dtype not in _TYPES:
        raise RuntimeError(f"{fn}: dtype {t.dtype} of {name} is not supported")
    if t.dim() == 0 or not 1 <= t.shape[-1] <= _MAX_COLS:
        raise RuntimeError(f"{fn}: {name} {tuple(t.shape)} must have 1 to {_MAX_COLS} columns")


def _kind(fn, kind, weight, bias):
    if kind not in _KINDS:
        raise RuntimeError(f"{fn}: kind of norm {kind!r} is not supported (None, rms, layer)")
    if kind is None and (weight is not None or bias is not None):
        raise RuntimeError(f"{fn}: a weight or bias without a norm")
    return _KINDS[kind]


def block_norm(x, weight=None, bias=None, kind="layer", eps=1e-5, out_dtype=None, checkpoint=False):
    """The norm before a block: "layer" (x - mean) / sqrt(var + eps) * weight + bias or "rms" x / sqrt(mean(x^2) + eps) * weight + bias over
    the last dimension (1 to 16384 columns), of type `out_dtype` (default: x's; a 16-bit x gives its own type only).  With checkpoint=True
    the result is (n, ActivationCheckpoint of n)."""
    fn = "block_norm"
    done = None if kind is None else _ordinary(x, None, None, None, None, weight, bias, 1.0, None, kind, eps, N.dtype_codes.get(out_dtype or x.dtype, -1), checkpoint)
    if done is not None:
        return done[1:] if checkpoint else done[1]
    _check_rows(fn, "x", x)
    if kind is None:
        raise RuntimeError(f"{fn}: kind of norm None is not supported (rms, layer)")
    pre_kind = _kind(fn, kind, weight, bias)
    block_dtype = x.dtype if out_dtype is None else out_dtype
    if block_dtype not in _TYPES or (x.dtype != torch.float32 and block_dtype != x.dtype):
        raise RuntimeError(f"{fn}: {x.dtype} to {block_dtype} is not supported")
    weight, bias = _parameters(fn, x, weight, bias)
    _, n, kept = _call(x, None, None, 1, None, None, weight, bias, 1.0, N.NORM_NONE, pre_kind, float(eps), block_dtype, checkpoint)
    return (n, kept) if checkpoint else n


def residual_norm(residual, y, gate=None, residual_scale=1.0, *, post_kind=None, post_weight=None, post_bias=None, pre_kind=None, pre_weight=None,
                  pre_bias=None, eps=1e-5, checkpoint=False):
    """What follows a block with output y and precedes the next one:

        out = residual_scale * residual + gate * N_post(y)      n = N_pre(out)

    residual and y have the same shape (last dimension 1 to 16384); residual is float32, or of y's type; residual_scale is a number.  A kind is None (post: y as it is;
    pre: no n is formed), "rms" or "layer"; weights and biases [columns].  `gate` is a tensor that broadcasts to y: of one element, a channel's [C],
    a sequence's [B, 1, C], a token's [B, S, C].  Returns out, with a pre_kind (out, n), with checkpoint=True (out, n, ActivationCheckpoint
    of n).  Gradients (once) for residual, y, gate, weights and biases, where no more than 2^22 gates are shared by rows; their sums take 16 bytes of
    scratch memory for each column of every such gate."""
    fn = "residual_norm"
    if not isinstance(y, torch.Tensor):
        raise RuntimeError(f"{fn}: y is {type(y).__name__}, not a tensor")
    if gate is not None and not isinstance(gate, torch.Tensor):
        raise RuntimeError(f"{fn}: gate is {type(gate).__name__}, not a tensor")
    if isinstance(residual_scale, torch.Tensor) and residual_scale.requires_grad:
        raise RuntimeError(f"{fn}: residual_scale is a number, no gradient goes to it")
    done = _ordinary(residual, y, gate, post_weight, post_bias, pre_weight, pre_bias, residual_scale, post_kind, pre_kind, eps, 0, checkpoint)
    if done is not None:
        return done if checkpoint else done[:2] if pre_kind else done[0]
    _check_rows(fn, "residual", residual)
    if residual.shape != y.shape or residual.get_device() != y.get_device():
        raise RuntimeError(f"{fn}: residual {tuple(residual.shape)} on {residual.device} and y {tuple(y.shape)} on {y.device} differ")
    if y.dtype not in _TYPES or (residual.dtype != torch.float32 and residual.dtype != y.dtype):
        raise RuntimeError(f"{fn}: a stream of {residual.dtype} with a block of {y.dtype} is not supported")
    post, pre = _kind(fn, post_kind, post_weight, post_bias), _kind(fn, pre_kind, pre_weight, pre_bias)
    if checkpoint and not pre:
        raise RuntimeError(f"{fn}: a checkpoint without a norm before the next block")
    post_weight, post_bias, pre_weight, pre_bias = _parameters(fn, y, post_weight, post_bias, pre_weight, pre_bias)
    rows_per_gate = 1
    if gate is not None:
        gate, rows_per_gate = _gate(fn, gate, y)
    out, n, kept = _call(residual, y, gate, rows_per_gate, post_weight, post_bias, pre_weight, pre_bias, float(residual_scale), post, pre, float(eps), y.dtype,
                         checkpoint)
    return (out, n, kept) if checkpoint else (out, n) if pre else out


def _make(module, name, wanted, cols, value, factory):
    module.register_parameter(name, nn.Parameter(torch.full((cols,), float(value), **factory)) if wanted else None)


class BlockNorm(nn.Module):
    """The norm before a block as a module: weight (ones) and, of a layer norm or with bias=True, bias (zeros)."""

    def __init__(self, dim, kind="layer", eps=1e-5, bias=None, out_dtype=None, device=None, dtype=None):
        super().__init__()
        if kind not in ("rms", "layer"):
            raise RuntimeError(f"BlockNorm: kind of norm {kind!r} is not supported (rms, layer)")
        self.kind, self.eps, self.out_dtype = kind, eps, out_dtype
        factory = {"device": device, "dtype": dtype}
        _make(self, "weight", True, dim, 1.0, factory)
        _make(self, "bias", kind == "layer" if bias is None else bias, dim, 0.0, factory)

    def forward(self, x, checkpoint=False):
        return block_norm(x, self.weight, self.bias, self.kind, self.eps, self.out_dtype, checkpoint)


class ResidualNorm(nn.Module):
    """What stands between two blocks as a module.  `post` and `pre` are kinds of norm or None; `gate` is None or the first value of a
    learned gate per channel.  forward(residual, y, gate=None, checkpoint=False): a gate given there takes the place of the learned one."""

    def __init__(self, dim, post=None, pre="layer", gate=None, residual_scale=1.0, eps=1e-5, bias=None, device=None, dtype=None):
        super().__init__()
        for kind in (post, pre):
            _kind("ResidualNorm", kind, None, None)
        self.post, self.pre, self.residual_scale, self.eps = post, pre, residual_scale, eps
        factory = {"device": device, "dtype": dtype}
        for name, kind in (("post", post), ("pre", pre)):
            _make(self, name + "_weight", kind is not None, dim, 1.0, factory)
            _make(self, name + "_bias", kind is not None and (kind == "layer" if bias is None else bias), dim, 0.0, factory)
        _make(self, "gate", gate is not None, dim, gate, factory)

    def forward(self, residual, y, gate=None, checkpoint=False):
        return residual_norm(residual, y, self.gate if gate is None else gate, self.residual_scale, post_kind=self.post, post_weight=self.post_weight,
                             post_bias=self.post_bias, pre_kind=self.pre, pre_weight=self.pre_weight, pre_bias=self.pre_bias, eps=self.eps, checkpoint=checkpoint)
