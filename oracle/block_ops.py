"""Oracle: block norms with gate and residual, activations kept in 8 bits.

TEST INFRASTRUCTURE ONLY -- never imported by the shipped package.  The reference has no such operators; these are the formulas in
float64.

Pinned by: kept() by torch's own float8_e4m3fn cast on blocks scaled by hand and by known values; the norms by
torch.nn.functional.layer_norm / rms_norm in float64, their gradients by autograd of those.
"""
import torch

_HELD = {torch.float16: 61440.0, torch.bfloat16: 1.875 * 2.0 ** 127, torch.float32: 1.875 * 2.0 ** 127}
_E4M3 = torch.tensor([(m / 8.0) * 2.0 ** -6 if e == 0 else (1.0 + m / 8.0) * 2.0 ** (e - 7) for e in range(16) for m in range(8) if (e, m) != (15, 7)],
                     dtype=torch.float64)                          # the magnitudes, by code


def kept_scale(block):
    """The exponent of the scale of a block (a 1-d tensor): the largest finite magnitude lies in (224, 448] * 2^exponent."""
    limit = _HELD[block.dtype]
    finite = [min(abs(float(v)), limit) for v in block if torch.isfinite(v)]
    top = max(finite, default=0.0)
    exponent = -117
    while top > 448.0 * 2.0 ** exponent:
        exponent += 1
    return exponent


def kept(x):
    """x [rows, cols] as it is kept in 8 bits, float64: blocks of 32 columns, round to nearest, ties to the even code."""
    rows, cols = x.shape
    out = torch.empty(rows, cols, dtype=torch.float64)
    limit = _HELD[x.dtype]
    for r in range(rows):
        for c in range(0, cols, 32):
            block = x[r, c:c + 32]
            unit = 2.0 ** kept_scale(block)
            v = block.double().clamp(-limit, limit) / unit
            at = torch.searchsorted(_E4M3, v.abs().contiguous()).clamp(1, len(_E4M3) - 1)
            below, above = _E4M3[at - 1], _E4M3[at]
            middle = (below + above) / 2
            up = (v.abs() > middle) | ((v.abs() == middle) & (at % 2 == 0))
            q = torch.where(up, above, below).copysign(v) * unit
            out[r, c:c + 32] = torch.where(torch.isfinite(block), q, torch.nan)
    return out


def kept_fast(x):
    """kept() for large finite matrices: the same by torch's cast."""
    rows, cols = x.shape
    v = torch.nn.functional.pad(x.double().clamp(-_HELD[x.dtype], _HELD[x.dtype]), (0, -cols % 32)).view(rows, -1, 32)
    mantissa, exponent = torch.frexp(v.abs().amax(-1, keepdim=True))
    exponent = torch.where(mantissa > 0.875, exponent - 8, exponent - 9).clamp(min=-117)
    unit = torch.ldexp(torch.ones_like(mantissa), exponent)
    return ((v / unit).float().to(torch.float8_e4m3fn).double() * unit).flatten(1)[:, :cols]


def statistics(v, kind, eps):
    """(mean, 1 / sqrt(variance or mean square + eps)) of each row, float64"""
    v = v.double()
    mean = v.mean(-1, keepdim=True) if kind == "layer" else torch.zeros(*v.shape[:-1], 1, dtype=torch.float64)
    return mean, 1.0 / torch.sqrt((v - mean).square().mean(-1, keepdim=True) + eps)


def norm(v, kind, weight, bias, eps):
    mean, r = statistics(v, kind, eps)
    out = (v.double() - mean) * r
    if weight is not None:
        out = out * weight.double()
    return out if bias is None else out + bias.double()


def norm_backward(grad, v, kind, weight, eps):
    """(gradient of v, terms of weight's gradient, terms of bias's gradient), the terms row by row"""
    mean, r = statistics(v, kind, eps)
    hat = (v.double() - mean) * r
    q = grad.double() if weight is None else grad.double() * weight.double()
    out = q - hat * (q * hat).mean(-1, keepdim=True)
    if kind == "layer":
        out = out - q.mean(-1, keepdim=True)
    return out * r, grad.double() * hat, grad.double()
