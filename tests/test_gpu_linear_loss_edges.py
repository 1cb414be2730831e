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


@pytest.mark.parametrize("tokens,cols", [(32768, 512), (30011, 600)])
@pytest.mark.parametrize("smoothing", [0.0, 0.1])
def test_whole_tiles_over_pieces_of_the_vocabulary(cuda, tokens, cols, smoothing):
    """The gradient of x from several pieces of the vocabulary: 256 tiles, each in one piece of k on a card of 256 compute units, and 354, some of which are cut."""
    gen, x, w, b = operands(cuda, tokens, tokens, cols, 40000, BF16, F32)
    target = torch.where(torch.rand(tokens, generator=gen) < 0.001, -100, torch.randint(0, 40000, (tokens,), generator=gen)).to(cuda)
    ce_check(cuda, x, w, b, target, label_smoothing=smoothing)


@pytest.mark.parametrize("words", [95, 96, 97, 255, 256, 257, 512, 671, 672, 673])
@pytest.mark.parametrize("tokens", [255, 256, 257, 511, 512, 513])
def test_ends_of_tiles(cuda, tokens, words):
    """Tiles of 256 tokens and 256 words, stages of 64 words of which half may lie behind the last."""
    gen, x, w, b = operands(cuda, tokens + words, tokens, 64 if words % 2 else 136, words, BF16 if tokens % 2 else F16, F32)
    target = torch.randint(0, words, (tokens,), generator=gen).to(cuda)
    ce_check(cuda, x, w, b, target, label_smoothing=0.1 if words % 3 else 0.0)
    indices = torch.randint(-1, words, (tokens, 5), generator=gen).to(cuda)
    kd_check(cuda, x, w, b, indices, draw(gen, tokens, 5).to(cuda))


@pytest.mark.parametrize("counted", [0, 1, 63, 64, 65, 255, 256, 257, 512])
def test_numbers_of_tokens_that_count(cuda, counted):
    gen, x, w, b = operands(cuda, counted, 700, 320, 900, BF16, F32)
    counts = torch.zeros(700, dtype=torch.bool)
    counts[torch.randperm(700, generator=gen)[:counted]] = True
    target = torch.where(counts, torch.randint(0, 900, (700,), generator=gen), -100).to(cuda)
    ce_check(cuda, x, w, b, target, "none", label_smoothing=0.1)
    ce_check(cuda, x, w, b, target)
    indices = torch.where(counts[:, None], torch.randint(0, 900, (700, 7), generator=gen), -1).to(cuda)
    kd_check(cuda, x, w, b, indices, draw(gen, 700, 7).to(cuda), "none")


@pytest.mark.parametrize("tokens", [1, 40, 64, 300])
def test_rows_that_do_not_count_are_not_read(cuda, tokens):
    """Infinities and NaN in them reach neither the losses nor a gradient, through any kernel and both losses."""
    gen, x, w, b = operands(cuda, tokens, tokens, 128, 1000, F16, F32)
    skipped = torch.rand(tokens, generator=gen) < 0.5
    skipped[0] = True
    target = torch.where(skipped, -100, torch.randint(0, 1000, (tokens,), generator=gen)).to(cuda)
    indices = torch.where(skipped[:, None], -1, torch.randint(0, 1000, (tokens, 6), generator=gen)).to(cuda)
    logits = draw(gen, tokens, 6).to(cuda)
    grad = torch.rand(tokens, generator=gen).to(cuda)
    dirty = x.clone()
    dirty[skipped.to(cuda)] = torch.tensor([torch.nan, torch.inf, -torch.inf, 65504.0], dtype=F16, device=cuda).repeat(32)
    for step in (lambda v: ce_step(v, w, b, target, grad, reduction="none", label_smoothing=0.1), lambda v: kd_step(v, w, b, indices, logits, grad, reduction="none")):
        clean, got = step(x), step(dirty)
        assert torch.equal(clean[0], got[0]) and all(torch.equal(a, c) for a, c in zip(clean[1], got[1]))
        assert all(t.isfinite().all() for t in (got[0], *got[1])) and not got[1][0][skipped.to(cuda)].any()


@pytest.mark.parametrize("tokens", [3, 100, 300])
def test_nothing_counts_before_weights_that_are_not_finite(cuda, tokens):
    """Tokens that do not count give no gradient, whatever the weights and the bias have become."""
    gen, x, w, b = operands(cuda, tokens, tokens, 72, 500, BF16, F32)
    for value in (torch.nan, torch.inf, -torch.inf):
        w[3, 5], b[7] = value, value
        for reduction in ("mean", "none"):
            grad = torch.ones(tokens if reduction == "none" else (), device=cuda)
            for smoothing in (0.0, 0.1):
                loss, grads = ce_step(x, w, b, torch.full((tokens,), -100, device=cuda), grad, reduction=reduction, label_smoothing=smoothing)
                assert not loss.any() and not any(g.any() for g in grads[1:]) and not grads[0].any(), (value, reduction)
            loss, grads = kd_step(x, w, b, torch.full((tokens, 2), -1, device=cuda), torch.zeros(tokens, 2, device=cuda), grad, reduction=reduction)
            assert not loss.any() and not any(g.any() for g in grads), (value, reduction)


@pytest.mark.parametrize("tokens", [3, 100, 256, 300])
def test_words_with_a_logit_of_minus_infinity(cuda, tokens):
    """A weight of -inf against positive x takes its word out as a bias of -inf does: probability 0, and a gradient of 0 for its row, as of a word whose bias is -inf."""
    gen, x, w, _ = operands(cuda, tokens, tokens, 64, 300, BF16)
    x[:, 7] = x[:, 7].abs() + 0.5
    target = torch.randint(0, 200, (tokens,), generator=gen).to(cuda)
    b = torch.zeros(300, device=cuda)
    b[250] = -torch.inf
    leaf = w.clone().requires_grad_()
    import sparse
    loss = sparse.linear_cross_entropy(x, leaf, target, b)
    want, = torch.autograd.grad(loss, leaf)
    w[250, 7] = -torch.inf
    leaf = w.clone().requires_grad_()
    got = sparse.linear_cross_entropy(x, leaf, target, torch.zeros_like(b))
    assert torch.equal(got, loss) and torch.equal(torch.autograd.grad(got, leaf)[0], want) and not want[250].any()


def test_gradients_at_the_ends_of_float32(cuda):
    """Upstream gradients far below float32's normal numbers give gradients that are no larger, and no NaN; ones near its largest number the gradients that 16 bits hold."""
    gen, x, w, b = operands(cuda, 3, 70, 64, 300, F16, F32)
    target, indices, logits = torch.randint(0, 300, (70,), generator=gen).to(cuda), torch.randint(0, 300, (70, 4), generator=gen).to(cuda), draw(gen, 70, 4).to(cuda)
    for dtype in (F16, BF16):
        for size in (1e-37, 1e-40, 1e-44):
            for reduction in ("sum", "none"):
                grad = torch.tensor(size, device=cuda) if reduction == "sum" else torch.full((70,), size, device=cuda)
                for _, grads in (ce_step(x.to(dtype), w.to(dtype), b, target, grad, reduction=reduction), kd_step(x.to(dtype), w.to(dtype), b, indices, logits, grad, reduction=reduction)):
                    # (70 tokens, or 300 words, of at most 4 or so)
                    assert all((g.double().abs() <= 2000 * size).all() for g in grads), (dtype, size, reduction)
    # probabilities of a teacher that add up to e^0.5, the largest gradient of a token's loss times that past float32's largest number, that of the operands below it
    x, w = x.to(BF16), w.to(BF16) * 2.0 ** -20
    lse = torch.logsumexp(logits, 1) - 0.5
    kw = dict(reduction="none", teacher_lse=lse)
    unit, = (g[0] for _, g in (kd_step(x, w, None, indices, logits, torch.ones(70, device=cuda), **kw),))
    large, = (g[0] for _, g in (kd_step(x, w, None, indices, logits, torch.full((70,), 2.0 ** 127, device=cuda), **kw),))
    # (units that are a power of two apart: the same roundings)
    assert torch.equal(large.double(), unit.double() * 2.0 ** 127)


def test_order_of_tokens(cuda):
    """Permuted tokens give the same loss and the same gradients up to the order of float32 sums: at most as many additions as there are tokens or words, of the magnitudes
    added, and a rounding of x's gradient.  The products that are added are the same."""
    gen, x, w, b = operands(cuda, 71, 300, 64, 500, BF16, F32)
    target = torch.randint(0, 40, (300,), generator=gen).to(cuda)
    z = definition.logits(x, w, b)
    _, slope, counts = definition.cross_entropy(z, target)
    order = torch.randperm(300, generator=gen).to(cuda)
    one = torch.tensor(1.0, device=cuda)
    loss, (dx, dw, db) = ce_step(x, w.float(), b, target, one, reduction="sum")
    other, (dx2, dw2, db2) = ce_step(x[order], w.float(), b, target[order], one, reduction="sum")
    assert abs(loss - other) <= 2 * E * loss                       # (summed in float64, rounded once)
    assert torch.equal(dx2, dx[order])
    # (a factor of 1.01 for probabilities that are rounded to 8 bits)
    assert ((dw - dw2).abs().double() <= 1.01 * 600 * E * (slope.abs().t() @ x.double().abs())).all()
    assert ((db - db2).abs().double() <= 1.01 * 600 * E * slope.abs().sum(0)).all()


def test_what_the_workspace_held_does_not_matter(cuda):
    """NaN, zeros and large numbers in the memory that workspaces, states and results are made in: the same bits."""
    gen, x, w, b = operands(cuda, 5, 333, 200, 5003, BF16, F32)
    target = torch.where(torch.rand(333, generator=gen) < 0.3, -100, torch.randint(0, 5003, (333,), generator=gen)).to(cuda)
    indices, logits = torch.where(torch.rand(333, 9, generator=gen) < 0.5, -1, torch.randint(0, 5003, (333, 9), generator=gen)).to(cuda), draw(gen, 333, 9).to(cuda)
    grad = torch.rand(333, generator=gen).to(cuda)
    first = None
    for fill in (0, 255, 126):
        torch.cuda.empty_cache()
        held = [torch.full((1 << 28,), fill, dtype=torch.uint8, device=cuda)] + [torch.full((1 << 19,), fill, dtype=torch.uint8, device=cuda) for _ in range(64)]
        del held
        got = []
        for some in (slice(None), slice(0, 50)):
            for loss, grads in (ce_step(x[some], w, b, target[some], grad[some], reduction="none", label_smoothing=0.1, z_loss=1e-3), kd_step(x[some], w, b, indices[some], logits[some], grad[some], reduction="none")):
                got += [loss, *grads]
        if first is None:
            first = got
        assert all(torch.equal(a, c) for a, c in zip(got, first)), fill


@pytest.mark.parametrize("tokens,cols,words", [(70, 65536, 300), (3, 65536, 97), (100, 24, 1 << 22), (3, 24, 1 << 22), (1 << 22, 24, 100)])
def test_largest_sizes(cuda, tokens, cols, words):
    """2^16 columns, 2^22 words, 2^22 tokens; the last word and the last token among those that matter."""
    gen, x, w, b = operands(cuda, 9, tokens, cols, words, BF16, F32)
    target = torch.where(torch.rand(tokens, generator=gen) < 0.3, -100, torch.randint(0, words, (tokens,), generator=gen))
    target[-1] = words - 1
    target = target.to(cuda)
    ce_check(cuda, x, w, b, target, label_smoothing=0.1)
    indices = torch.randint(0, words, (tokens, 3), generator=gen)
    indices[-1, 1] = words - 1
    kd_check(cuda, x, w, b, indices.to(cuda), draw(gen, tokens, 3).to(cuda))


def test_smoothing_of_any_layout_each_gradient_alone_and_replayed(cuda):
    """Weights in wider rows, in the middle of a dword, expanded; gradients one by one; a captured step with eager work between its replays: the same bits."""
    import sparse
    gen, x, w, b = operands(cuda, 13, 300, 128, 3000, BF16, F32)
    target = torch.where(torch.rand(300, generator=gen) < 0.3, -100, torch.randint(0, 3000, (300,), generator=gen)).to(cuda)
    grad = torch.rand(300, generator=gen).to(cuda)
    kw = dict(reduction="none", label_smoothing=0.1, z_loss=1e-3)
    want = ce_step(x, w, b, target, grad, **kw)
    for start, ld in ((24, 200), (3, 200), (1, 129)):
        held = torch.full((3000 * ld + start,), torch.nan, dtype=BF16, device=cuda).as_strided((3000, 128), (ld, 1), start)
        held.copy_(w)
        got = ce_step(x, held, b, target, grad, **kw)
        assert torch.equal(got[0], want[0]) and all(torch.equal(a, c) for a, c in zip(got[1], want[1]))
    for i in range(3):
        leaves = [t.detach().requires_grad_(i == n) for n, t in enumerate((x, w, b))]
        got, = torch.autograd.grad(sparse.linear_cross_entropy(leaves[0], leaves[1], target, leaves[2], **kw), leaves[i], grad)
        assert torch.equal(got, want[1][i])
    same = w[:1].expand(3000, 128)
    for a, c in zip(ce_step(x, same, b, target, grad, **kw)[1], ce_step(x, same.contiguous(), b, target, grad, **kw)[1]):
        assert torch.equal(a, c)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ce_step(x, w, b, target, grad, **kw)
    torch.cuda.synchronize()
    held = [x.clone(), target.clone(), grad.clone()]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ce_step(held[0], w, b, held[1], held[2], **kw)
    for n in range(4):
        batch = [t.roll(n, 0) for t in (x, target, grad)]
        if n == 2:
            batch[1] = torch.full_like(target, -100)
        for h, t in zip(held, batch):
            h.copy_(t)
        graph.replay()
        eager = ce_step(batch[0], w, b, batch[1], batch[2], **kw)
        torch.cuda.synchronize()
        assert torch.equal(out[0], eager[0]) and all(torch.equal(a, c) for a, c in zip(out[1], eager[1])), n
