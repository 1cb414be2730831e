"""linear_cross_entropy and linear_distillation where their parts meet: a constant level in the gradient of the logits, whole and cut tiles over several pieces of the
vocabulary, numbers of tokens and words at the ends of tiles, rows that do not count, weights and gradients at the ends of float32.

Tolerances as in test_gpu_linear_loss (u = eps / 2 of the operands' type, E = 2^-24), or derived beside the test.
"""
import pytest
import torch

import oracle.linear_loss as definition
from test_gpu_linear_loss import BF16, E, F16, F32, ce_check, ce_step, draw, kd_check, kd_step, operands

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("reduction", ["mean", "none"])
@pytest.mark.parametrize("cols", [128, 600])
def test_smoothing_of_words_that_are_not_expected(cuda, dtype, reduction, cols):
    """Where nearly all words are far less probable than smoothing / words, that level is nearly all of their gradient, the same for each of them and of each token:
    an error in it does not average out.  It comes through exactly, here 0.125 / 32641, which is half a step from what bfloat16 holds, times a sum over words whose
    weights have a large mean (dx), over tokens (dW, db).

    The target's logit is more than 40 above all others: its probability is 1 in float32 (it is the largest logit, and the sum of exponentials 1), its part of the
    gradient g (0.125 - 0.125 / words) with g a power of two.  g / 8 is a number of 16 bits, so the nearest one is no further away than that: at most by the level.  What else there is
    are sums in float32, over at most all words (dx) or all tokens (dW, db), of the magnitudes added, up to 16 roundings of the level, its unit and the scale, and the rounding of the
    results.  Without the rest of the level bfloat16's dx is off by 0.0156 g, against a bound of 0.0078 g + u |dx|."""
    words, tokens, smoothing = 32641, 512, 0.125
    gen = torch.Generator().manual_seed(cols)
    w = (32 + draw(gen, words, cols)).to(dtype)
    target = torch.randint(0, words, (tokens,), generator=gen)
    x = w[target].float()
    x = (2 * (x - x.mean(1, keepdim=True))).to(dtype)
    x, w, target = x.to(cuda), w.float().to(cuda), target.to(cuda)   # a float32 weight of 16-bit values: its gradient is float32
    b = torch.zeros(words, device=cuda)
    grad = torch.tensor(1.0, device=cuda) if reduction == "mean" else torch.tensor([1.0, 0.5, -0.25, 0.0], device=cuda).repeat(tokens // 4)
    z = definition.logits(x, w, b)
    _, slope, counts = definition.cross_entropy(z, target, label_smoothing=smoothing)
    p = torch.softmax(z, 1)
    p[torch.arange(tokens, device=cuda), target] = 0
    assert p.amax() < 1e-20
    loss, (dx, dw, db) = ce_step(x, w, b, target, grad, label_smoothing=smoothing, reduction=reduction)
    *want, _ = definition.gradients(slope, counts, grad, reduction, x, w, b)
    g = (grad.double() / tokens if reduction == "mean" else grad.double()).expand(tokens).abs()
    u, size = torch.finfo(dtype).eps / 2, w.double().abs()
    level = g * smoothing / words
    bound = u * want[0].abs() + level[:, None] * (words + 64) * E * size.sum(0) + (level + 8 * E * g * smoothing)[:, None] * size[target] + (2.0 ** -25 if dtype == F16 else 0.0)
    assert ((dx.double() - want[0]).abs() <= bound).all(), ((dx.double() - want[0]).abs() - bound).max()
    listed = torch.zeros(words, cols, dtype=torch.float64, device=cuda).index_add_(0, target, x.double().abs() * g[:, None])
    bound = (tokens + 16) * E * (smoothing * listed + (level[:, None] * x.double().abs()).sum(0)) + smoothing / words * listed
    assert ((dw.double() - want[1]).abs() <= bound).all(), ((dw.double() - want[1]).abs() - bound).max()
    bound = (tokens + 16) * E * (level.sum() + torch.zeros(words, dtype=torch.float64, device=cuda).index_add_(0, target, g * smoothing))
    assert ((db.double() - want[2]).abs() <= bound).all(), ((db.double() - want[2]).abs() - bound).max()
