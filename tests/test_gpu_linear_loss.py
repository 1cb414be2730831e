"""linear_cross_entropy and linear_distillation against their definitions in float64.

Tolerances (u = eps / 2 of the operands' type, e = 2^-24): a logit is off by at most
    dz = (columns + 4) e (|x| |W|^T + |b|),   and what follows from it in float32 by a few dozen e of the numbers that are added up;
the gradient of the logits by 2 dz |P| from the logits, and by u |P| from its rounding; a product with it by that, by its number of terms times e and by u of
its result.  The same in the norm: roundings of P and of the result are independent, so the whole is off by less than 2 u of the whole.
"""
import pytest
import torch

import oracle.linear_loss as definition

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
E = 2.0 ** -24


def draw(gen, *shape, std=1.0, dtype=F32):
    return (torch.randn(shape, generator=gen) * std).to(dtype)


def operands(cuda, seed, tokens, cols, words, dtype, bias=None):
    gen = torch.Generator().manual_seed(seed)
    x, w = draw(gen, tokens, cols, dtype=dtype), draw(gen, words, cols, std=2.0 / cols ** 0.5, dtype=dtype)
    b = None if bias is None else draw(gen, words, std=0.5, dtype=bias)
    return gen, x.to(cuda), w.to(cuda), None if b is None else b.to(cuda)


def logit_error(x, w, b, counts):
    rows = torch.where(counts[:, None], x.double().reshape(-1, x.shape[-1]), 0.0)
    size = rows.abs() @ w.double().abs().t()
    if b is not None:
        size = size + torch.where(b.isfinite(), b.double().abs(), 0.0)
    return (x.shape[-1] + 4) * E * size.amax(1)


def check_loss(loss, want, z, counts, x, w, b, reduction, scale=1.0):
    dz = logit_error(x, w, b, counts) / scale
    top = torch.where(counts[:, None] & z.isfinite(), z, 0.0).abs().amax(1) / scale
    tol = torch.where(counts, 4 * dz + 64 * E * (1 + top + torch.log(torch.tensor(float(z.shape[1])))) * (1 + top), 0.0)
    tol = definition.reduced(tol, counts, reduction) + 4 * E * want.abs()
    assert loss.dtype == F32 and loss.shape == want.shape
    assert ((loss.double() - want).abs() <= tol).all(), (loss.double() - want).abs().max()


def check_grads(got, want, p, x, w, b, counts, dtype):
    """got, want: dx, dW, db"""
    u = torch.finfo(dtype).eps / 2
    dz = logit_error(x, w, b, counts)[:, None]
    size = p.abs()
    dp = size * (u + 4 * dz + 64 * E) + size.amax() * 2.0 ** -38
    rows = torch.where(counts[:, None], x.double().reshape(-1, x.shape[-1]), 0.0)
    tols = (dp @ w.double().abs() + (w.shape[0] + 64) * E * (size @ w.double().abs()),
            dp.t() @ rows.abs() + (x.shape[0] + 64) * E * (size.t() @ rows.abs()), dp.sum(0) + (x.shape[0] + 64) * E * size.sum(0))
    for name, g, v, tol in zip(("x", "weight", "bias"), got, want, tols):
        if g is None:
            continue
        own = torch.finfo(g.dtype).eps / 2
        floor = 2.0 ** -25 if g.dtype == F16 else 0.0              # half a step of float16's subnormal numbers
        error = (g.double() - v).abs().reshape(tol.shape)
        bound = tol * (1 + own) + own * v.abs().reshape(tol.shape) + floor
        assert (error <= bound).all(), (name, (error - bound).max(), error.max())
        if v.norm() > 0:
            assert error.norm() <= 2 * u * v.norm() + floor * error.numel() ** 0.5 + tol.norm() * 1e-2, (name, error.norm() / v.norm(), u)


def ce_step(x, w, b, target, grad, **how):
    import sparse
    leaves = [t.detach().requires_grad_() for t in (x, w, b) if t is not None]
    loss = sparse.linear_cross_entropy(leaves[0], leaves[1], target, *leaves[2:], **how)
    return loss.detach(), torch.autograd.grad(loss, leaves, grad)


def ce_check(cuda, x, w, b, target, reduction="mean", scale=1.0, seed=5, **how):
    gen = torch.Generator().manual_seed(seed)
    z = definition.logits(torch.where((target.reshape(-1) == how.get("ignore_index", -100))[:, None], 0.0, x.reshape(-1, x.shape[-1]).double()), w, b)
    want, slope, counts = definition.cross_entropy(z, target, **how)
    grad = torch.tensor(scale, device=cuda) if reduction != "none" else (draw(gen, *target.shape) * scale).to(cuda)
    loss, grads = ce_step(x, w, b, target, grad, reduction=reduction, **how)
    check_loss(loss.reshape(-1) if reduction == "none" else loss, definition.reduced(want, counts, reduction), z, counts, x, w, b, reduction)
    *wanted, p = definition.gradients(slope, counts, grad, reduction, x, w, b)
    check_grads(grads, wanted, p, x, w, b, counts, x.dtype)
    assert not grads[0].reshape(-1, x.shape[-1])[~counts].any()
    return loss, grads


SIZES = [(1, 1, 1), (1, 64, 256), (2, 7, 3), (3, 8, 97), (37, 1601, 257), (193, 64, 191), (192, 128, 192), (385, 100, 1000), (700, 768, 5003), (50, 200, 384)]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("tokens,cols,words", SIZES)
def test_cross_entropy(cuda, tokens, cols, words, dtype):
    gen, x, w, _ = operands(cuda, tokens + words, tokens, cols, words, dtype)
    target = torch.randint(0, words, (tokens,), generator=gen).to(cuda)
    ce_check(cuda, x, w, None, target)


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("smoothing,z_loss", [(0.0, 0.0), (0.1, 0.0), (0.0, 1e-3), (0.2, 1e-2), (1.0, 0.0)])
@pytest.mark.parametrize("bias", [None, F32, BF16])
@pytest.mark.parametrize("ignored", [0.0, 0.6, 1.0])
def test_cross_entropy_terms(cuda, reduction, smoothing, z_loss, bias, ignored):
    gen, x, w, b = operands(cuda, 17, 210, 136, 500, BF16, bias)
    target = torch.where(torch.rand(210, generator=gen) < ignored, -1, torch.randint(0, 500, (210,), generator=gen)).to(cuda)
    ce_check(cuda, x, w, b, target, reduction, ignore_index=-1, label_smoothing=smoothing, z_loss=z_loss)


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_large_vocabulary(cuda, dtype):
    """Scoring: a vocabulary of many tiles, tokens of one to a few tiles."""
    import sparse
    for tokens in (1, 3, 65, 200):
        gen, x, w, b = operands(cuda, tokens, tokens, 256, 50257, dtype, F32)
        target = torch.randint(0, 50257, (tokens,), generator=gen).to(cuda)
        z = definition.logits(x, w, b)
        want, _, counts = definition.cross_entropy(z, target)
        with torch.no_grad():
            check_loss(sparse.linear_cross_entropy(x, w, target, b, reduction="none"), want, z, counts, x, w, b, "none")


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("cols", [1, 31, 33, 64, 95, 257, 766])
def test_few_tokens(cuda, cols, dtype):
    """1 to 64 tokens, whose weight is read as it lies: every number of tokens that a variant begins and ends with, rows that start in the middle of a dword, tensors that
    end with their last row, in front of which and behind which there are NaN."""
    import sparse
    words = 391
    for tokens in (1, 2, 16, 17, 32, 33, 48, 49, 63, 64, 65):
        gen, x, w, b = operands(cuda, tokens + cols, tokens, cols, words, dtype, BF16)
        around = torch.full(((words + 2) * (cols + 1) + 2,), torch.nan, dtype=dtype, device=cuda)
        for start, ld in ((1, cols), (2, cols), (1, cols + 1), (2, cols + 1)):
            held = around.clone().as_strided((words, cols), (ld, 1), start)
            held.copy_(w)
            target = torch.randint(-1, words, (tokens,), generator=gen).to(cuda)
            z = definition.logits(torch.where(target[:, None] == -1, 0, x), w, b)
            want, _, counts = definition.cross_entropy(z, target, -1, 0.1, 1e-3)
            with torch.no_grad():
                loss = sparse.linear_cross_entropy(x, held, target, b, ignore_index=-1, label_smoothing=0.1, z_loss=1e-3, reduction="none")
            check_loss(loss, want, z, counts, x, w, b, "none")
            indices, logits = torch.randint(-1, words, (tokens, 70), generator=gen).to(cuda), draw(gen, tokens, 70).to(cuda)
            z = definition.logits(x, w, b)
            want, _, counts = definition.distillation(z, indices, logits, temperature=2.0)
            with torch.no_grad():
                check_loss(sparse.linear_distillation(x, held, indices, logits, b, temperature=2.0, reduction="none"), want, z, counts, x, w, b, "none", 2.0)


@pytest.mark.parametrize("tokens,cols,words", [(520, 1100, 9000), (70, 264, 66000), (2100, 520, 700), (300, 40, 400)])
def test_pieces_along_k(cuda, tokens, cols, words):
    """Products of which some tiles are whole and others cut along k, all whole, all cut, and (few tokens count) another share of them than there is room for."""
    for ignored in (0.0, 0.7, 0.995):
        gen, x, w, b = operands(cuda, tokens, tokens, cols, words, BF16, F32)
        target = torch.where(torch.rand(tokens, generator=gen) < ignored, -100, torch.randint(0, words, (tokens,), generator=gen)).to(cuda)
        ce_check(cuda, x, w, b, target, "none")


def test_gradient_of_a_bias_is_that_of_the_unrounded_logits(cuda):
    """Of few tokens it is one listed word's probability mostly, rounded once and not twice; the order in which tokens come does not matter to the bit."""
    gen, x, w, b = operands(cuda, 71, 90, 64, 50, BF16, F32)
    target = torch.randint(0, 50, (90,), generator=gen).to(cuda)
    z = definition.logits(x, w, b)
    _, slope, counts = definition.cross_entropy(z, target)
    grad = torch.tensor(1.0, device=cuda)
    want = definition.gradients(slope, counts, grad, "sum", x, w, b)[2]
    got = ce_step(x, w, b, target, grad, reduction="sum")[1][2]
    # what is not listed is rounded to 8 bits: 2^-9 of each at most, about its root mean square over 90 tokens together; the listed words to 2^-32
    others = slope.clone()
    others[torch.arange(90, device=cuda), target] = 0
    assert ((got.double() - want).abs() <= 2.0 ** -8 * others.abs().sum(0) + 2.0 ** -20).all()
    again = [ce_step(x, w, b, target, grad, reduction="sum")[1][2] for _ in range(3)]
    assert all(torch.equal(a, got) for a in again)


def test_pieces_of_the_vocabulary(cuda):
    """More tokens than the gradient of all logits at once is formed for."""
    tokens, cols, words = 30011, 72, 40000
    gen, x, w, b = operands(cuda, 3, tokens, cols, words, BF16, BF16)
    target = torch.where(torch.rand(tokens, generator=gen) < 0.1, -100, torch.randint(0, words, (tokens,), generator=gen)).to(cuda)
    ce_check(cuda, x, w, b, target)
    indices = torch.randint(0, words, (tokens, 3), generator=gen).to(cuda)
    kd_check(cuda, x, w, b, indices, draw(gen, tokens, 3).to(cuda))


def kd_step(x, w, b, indices, logits, grad, **how):
    import sparse
    leaves = [t.detach().requires_grad_() for t in (x, w, b) if t is not None]
    loss = sparse.linear_distillation(leaves[0], leaves[1], indices, logits, *leaves[2:], **how)
    return loss.detach(), torch.autograd.grad(loss, leaves, grad)


def kd_check(cuda, x, w, b, indices, logits, reduction="mean", seed=6, temperature=1.0, **how):
    gen = torch.Generator().manual_seed(seed)
    z = definition.logits(x, w, b)
    want, slope, counts = definition.distillation(z, indices, logits, temperature=temperature, **how)
    grad = torch.tensor(1.0, device=cuda) if reduction != "none" else draw(gen, *indices.shape[:-1]).to(cuda)
    loss, grads = kd_step(x, w, b, indices, logits, grad, reduction=reduction, temperature=temperature, **how)
    # (the probabilities of a teacher may add up to more than one)
    mass = max(1.0, float((slope.abs().sum(1) * temperature).max()))
    check_loss(loss.reshape(-1) / mass if reduction == "none" else loss / mass, definition.reduced(want, counts, reduction) / mass, z, counts, x, w, b, reduction, temperature)
    *wanted, p = definition.gradients(slope, counts, grad, reduction, x, w, b)
    check_grads(grads, wanted, p, x, w, b, counts, x.dtype)
    assert not grads[0].reshape(-1, x.shape[-1])[~counts].any()


def test_more_than_2_31_elements(cuda):
    """Rows of x, dx and the teacher's entries past 2^31 elements: few of the tokens count, the first and the last, and all of them."""
    import sparse
    tokens, cols, words = 2200003, 1000, 200
    rows = torch.cat([torch.arange(1500), torch.arange(tokens - 1500, tokens)]).to(cuda)
    gen, _, w, _ = operands(cuda, 77, 1, cols, words, BF16)
    x = torch.empty(tokens, cols, dtype=BF16, device=cuda).normal_().requires_grad_()
    target = torch.full((tokens,), -100, device=cuda)
    target[rows] = torch.randint(0, words, (3000,), generator=gen).to(cuda)
    one = torch.tensor(1.0, device=cuda)
    few = x.detach()[rows]
    for some in (True, False):
        if not some:
            target[target == -100] = 7
        leaf = w.clone().requires_grad_()
        loss = sparse.linear_cross_entropy(x, leaf, target, reduction="none")
        z = definition.logits(few, w)
        want, slope, counts = definition.cross_entropy(z, target[rows])
        check_loss(loss.detach()[rows], want, z, counts, few, w, None, "none")
        dx, dw = torch.autograd.grad(loss, (x, leaf), one.expand(tokens))
        *wanted, p = definition.gradients(slope, counts, torch.ones(3000, device=cuda), "none", few, w)
        check_grads((dx[rows], dw if some else None, None), wanted, p, few, w, None, counts, BF16)
        if some:
            assert not loss.detach()[1500:-1500].any() and not dx[1500:-1500].any()
        del loss, dx, dw
    indices = torch.randint(-1, words, (tokens, cols), device=cuda)
    logits = torch.empty(tokens, cols, dtype=BF16, device=cuda).normal_()
    loss = sparse.linear_distillation(x, w, indices, logits, reduction="none")
    want, slope, counts = definition.distillation(z, indices[rows], logits[rows])
    check_loss(loss.detach()[rows], want, z, counts, few, w, None, "none")
    dx, = torch.autograd.grad(loss, x, one.expand(tokens))
    *wanted, p = definition.gradients(slope, counts, torch.ones(3000, device=cuda), "none", few, w)
    check_grads((dx[rows], None, None), wanted, p, few, w, None, counts, BF16)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("tokens,cols,words", SIZES)
def test_distillation(cuda, tokens, cols, words, dtype):
    gen, x, w, _ = operands(cuda, tokens + words, tokens, cols, words, dtype)
    entries = min(words, 33)
    indices = torch.stack([torch.randperm(words, generator=gen)[:entries] for _ in range(tokens)]).to(cuda)
    kd_check(cuda, x, w, None, indices, draw(gen, tokens, entries, std=3.0).to(cuda))


@pytest.mark.parametrize("reduction", ["mean", "none"])
@pytest.mark.parametrize("temperature", [0.5, 1.0, 3.0])
@pytest.mark.parametrize("with_lse", [False, True])
@pytest.mark.parametrize("entries,teacher", [(1, F32), (2, BF16), (64, F16), (100, F32), (1024, BF16)])
def test_distillation_terms(cuda, reduction, temperature, with_lse, entries, teacher):
    """Words listed twice (1024 entries of 700 words), unused entries, tokens without any."""
    gen, x, w, b = operands(cuda, 23, 150, 136, 700, BF16, F32)
    indices = torch.randint(0, 700, (150, entries), generator=gen)
    indices[torch.rand(150, entries, generator=gen) < 0.3] = -1
    indices[7] = -5
    logits = draw(gen, 150, entries, std=2.0, dtype=teacher)
    logits[indices < 0] = torch.nan                                # (nothing of an unused entry is looked at)
    logits[9, :] = -torch.inf                                      # a token whose words are all impossible does not count
    if entries > 1:
        logits[11, 0] = -torch.inf
    finite = torch.where(indices < 0, -torch.inf, logits.double() / temperature)
    lse = (torch.logsumexp(finite, 1).nan_to_num(neginf=0.0) + torch.rand(150, generator=gen)).float().to(cuda) if with_lse else None
    kd_check(cuda, x, w, b, indices.to(cuda), logits.to(cuda), reduction, temperature=temperature, **({"teacher_lse": lse} if with_lse else {}))


def test_rows_that_do_not_count_are_not_read(cuda):
    """Infinities and NaN in them reach neither the loss nor a gradient."""
    gen, x, w, b = operands(cuda, 29, 300, 128, 1000, F16, F32)
    target = torch.where(torch.rand(300, generator=gen) < 0.5, -100, torch.randint(0, 1000, (300,), generator=gen)).to(cuda)
    clean = ce_check(cuda, x, w, b, target)
    dirty = x.clone()
    dirty[target == -100] = torch.tensor([torch.nan, torch.inf, -torch.inf, 65504.0], dtype=F16, device=cuda).repeat(32)
    loss, grads = ce_step(dirty, w, b, target, torch.tensor(1.0, device=cuda))
    assert torch.equal(loss, clean[0]) and all(torch.equal(g, c) for g, c in zip(grads, clean[1]))


def test_masked_words(cuda):
    """A bias of -inf, or of float16's lowest number, takes words out: a padded vocabulary, whole tiles of it, all but one."""
    gen, x, w, _ = operands(cuda, 31, 200, 128, 700, BF16)
    for first, value in ((650, -torch.inf), (100, -torch.inf), (1, -torch.inf), (300, -65504.0)):
        b = torch.zeros(700, device=cuda)
        b[first:] = value
        target = torch.randint(0, first, (200,), generator=gen).to(cuda)
        _, grads = ce_check(cuda, x, w, b, target)
        assert not grads[1][first:].any() and not grads[2][first:].any()


def test_targets_that_are_no_words(cuda):
    gen, x, w, _ = operands(cuda, 37, 20, 64, 300, BF16)
    target = torch.randint(0, 300, (20,), generator=gen).to(cuda)
    for bad in (300, -1, 1 << 40, -(1 << 40)):
        target[4] = bad
        loss, grads = ce_step(x, w, None, target, torch.ones(20, device=cuda), reduction="none")
        assert loss[4].isnan() and loss.isnan().sum() == 1 and grads[0][4].isnan().all() and not grads[0][:4].isnan().any() and grads[1].isnan().all()
    indices, logits = torch.randint(0, 300, (20, 4), generator=gen).to(cuda), draw(gen, 20, 4).to(cuda)
    indices[3, 2] = 300
    loss, grads = kd_step(x, w, None, indices, logits, torch.ones(20, device=cuda), reduction="none")
    assert loss[3].isnan() and loss.isnan().sum() == 1 and grads[0][3].isnan().all() and not grads[0][4:].isnan().any()
    bad = x.clone()
    bad[2, 5] = torch.nan
    target[4] = 1
    loss, _ = ce_step(bad, w, None, target, torch.ones(20, device=cuda), reduction="none")
    assert loss[2].isnan() and loss.isnan().sum() == 1


def test_nothing_counts(cuda):
    import sparse
    gen, x, w, b = operands(cuda, 41, 5, 64, 300, BF16, F32)
    none = torch.full((5,), -100, device=cuda)
    for reduction in ("mean", "sum", "none"):
        loss, grads = ce_step(x, w, b, none, torch.ones(5 if reduction == "none" else (), device=cuda), reduction=reduction)
        assert not loss.any() and not any(g.any() for g in grads)
    empty = x[:0]
    loss, grads = ce_step(empty, w, b, none[:0], torch.tensor(1.0, device=cuda))
    assert loss == 0 and grads[0].shape == (0, 64) and not grads[1].any() and not grads[2].any()
    assert sparse.linear_cross_entropy(empty, w, none[:0], reduction="none").shape == (0,)
    loss, grads = kd_step(x, w, b, torch.full((5, 3), -1, device=cuda), torch.zeros(5, 3, device=cuda), torch.tensor(1.0, device=cuda))
    assert loss == 0 and not any(g.any() for g in grads)


def test_small_gradients_in_float16(cuda):
    """A mean over many tokens without a loss scale: probabilities of 1e-4 / 3000 are far below float16's smallest number, their products are not lost."""
    gen, x, w, _ = operands(cuda, 43, 3000, 64, 6000, F16)
    target = torch.randint(0, 6000, (3000,), generator=gen).to(cuda)
    ce_check(cuda, x, w, None, target)
    ce_check(cuda, x, w, None, target, scale=1e6)


def test_strides_and_shapes(cuda):
    """Batches, rows apart, columns apart, unaligned, transposed, negated, expanded: as contiguous ones."""
    gen, x, w, b = operands(cuda, 47, 60, 128, 300, BF16, F32)
    target = torch.randint(0, 300, (60,), generator=gen).to(cuda)
    grad = torch.rand(60, generator=gen).to(cuda)
    want = ce_step(x, w, b, target, grad, reduction="none")

    def same(x2, w2, b2, t2, g2):
        loss, grads = ce_step(x2, w2, b2, t2, g2, reduction="none")
        assert torch.equal(loss.reshape(-1), want[0]) and all(torch.equal(a.reshape(c.shape), c) for a, c in zip(grads, want[1]))

    wide = torch.zeros(60, 200, dtype=BF16, device=cuda)
    wide[:, 24:152] = x
    odd = torch.zeros(60, 131, dtype=BF16, device=cuda)
    odd[:, 3:] = x
    apart = torch.zeros(300, 256, dtype=BF16, device=cuda)
    apart[:, ::2] = w
    off = torch.zeros(300 * 128 + 1, dtype=BF16, device=cuda)
    off[1:] = w.reshape(-1)
    same(x.view(3, 4, 5, 128), w, b, target.view(3, 4, 5).int(), grad.view(3, 4, 5))
    same(wide[:, 24:152], w, b, target, grad)
    same(odd[:, 3:], w, b, target, grad)
    same(x, apart[:, ::2], b, target, grad)
    same(x, off[1:].view(300, 128), b, target, grad)
    same(x.t().contiguous().t(), w.t().contiguous().t(), b, torch.stack([target, target], 1)[:, 0], torch.stack([grad, grad], 1)[:, 0])
    same(torch._neg_view(-x), torch._neg_view(-w), torch._neg_view(-b), target, torch._neg_view(-grad))
    loss, grads = ce_step(x[:1].expand(60, 128), w, None, target[:1].expand(60), torch.ones((), device=cuda), reduction="sum")
    one, ones = ce_step(x[:1], w, None, target[:1], torch.ones((), device=cuda), reduction="sum")
    assert (loss - 60 * one).abs() <= 1e-5 * loss and torch.equal(grads[0][7], ones[0][0])
    # a width that is no multiple of anything: operands brought into whole stages, gradients in rows that are not aligned
    gen, x, w, b = operands(cuda, 48, 60, 71, 301, F16, F16)
    ce_check(cuda, x, w, b, target)
    indices = torch.randint(0, 301, (8, 60), generator=gen).to(cuda).t()
    kd_check(cuda, x, w, b, indices, torch.randn(60, 16, generator=gen).to(cuda)[:, 4:12])


def test_float32_weights_and_autocast(cuda):
    """A float32 weight takes part with its values in 16 bits; its gradient is float32, and not rounded to 16 bits on the way."""
    import sparse
    gen = torch.Generator().manual_seed(53)
    x, w, b = draw(gen, 250, 192).to(cuda), draw(gen, 500, 192, std=0.1).to(cuda), draw(gen, 500).to(cuda)
    target = torch.randint(0, 500, (250,), generator=gen).to(cuda)
    grad = torch.tensor(1.0, device=cuda)
    for dtype in (F16, BF16):
        want = ce_step(x.to(dtype), w.to(dtype), b, target, grad)
        mixed = ce_step(x.to(dtype), w, b, target, grad)
        leaves = [t.clone().requires_grad_() for t in (x, w, b)]
        with torch.autocast("cuda", dtype=dtype):
            loss = sparse.linear_cross_entropy(leaves[0], leaves[1], target, leaves[2])
        assert [t.dtype for t in (loss, *mixed[1])] == [F32, dtype, F32, F32]
        grads = torch.autograd.grad(loss, leaves, grad)
        for a in (mixed, (loss.detach(), grads)):
            assert torch.equal(a[0], want[0]) and torch.equal(a[1][0].to(dtype), want[1][0]) and torch.equal(a[1][1].to(dtype), want[1][1]) and torch.equal(a[1][2], want[1][2])
        assert not torch.equal(grads[1], grads[1].to(dtype).float())
    with pytest.raises(RuntimeError, match="autocast"):
        sparse.linear_cross_entropy(x, w, target)


def test_gradients_of_some(cuda):
    """Each gradient alone is the one among all; the same call again is the same to the bit."""
    import sparse
    gen, x, w, b = operands(cuda, 59, 400, 320, 2000, BF16, BF16)
    target = torch.randint(0, 2000, (400,), generator=gen).to(cuda)
    _, grads = ce_step(x, w, b, target, torch.tensor(2.0, device=cuda))
    again = ce_step(x, w, b, target, torch.tensor(2.0, device=cuda))[1]
    assert all(torch.equal(a, c) for a, c in zip(again, grads))
    for i in range(3):
        leaves = [t.detach().requires_grad_(i == n) for n, t in enumerate((x, w, b))]
        loss = sparse.linear_cross_entropy(leaves[0], leaves[1], target, leaves[2])
        first, = torch.autograd.grad(loss, leaves[i], torch.tensor(2.0, device=cuda), retain_graph=True)
        assert torch.equal(first, grads[i]) and torch.equal(torch.autograd.grad(loss, leaves[i], torch.tensor(2.0, device=cuda))[0], grads[i])
    leaf = x.detach().requires_grad_()
    loss = sparse.linear_cross_entropy(leaf, w, target)
    with pytest.raises(RuntimeError, match="graph of the gradients"):
        torch.autograd.grad(loss, leaf, create_graph=True)
    loss = sparse.linear_cross_entropy(leaf, w, target)
    w.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_differences(cuda):
    """The gradient is the slope of the loss: along the gradient of each operand, from losses of both sides."""
    import sparse
    gen = torch.Generator().manual_seed(61)
    x, w = draw(gen, 96, 64, dtype=F16).to(cuda), draw(gen, 400, 64, std=0.25, dtype=F16).to(cuda)
    target = torch.randint(0, 400, (96,), generator=gen).to(cuda)
    indices, logits = torch.randint(0, 400, (96, 8), generator=gen).to(cuda), draw(gen, 96, 8).to(cuda)
    losses = (lambda x, w: sparse.linear_cross_entropy(x, w, target, label_smoothing=0.1, z_loss=1e-3, reduction="sum"),
              lambda x, w: sparse.linear_distillation(x, w, indices, logits, temperature=2.0, reduction="sum"))
    for loss in losses:
        leaves = [x.detach().requires_grad_(), w.detach().requires_grad_()]
        grads = torch.autograd.grad(loss(*leaves), leaves)
        for i in range(2):
            step = 2.0 ** -5 * torch.sign(grads[i])
            sides = [[t if n != i else (t + s * step).detach() for n, t in enumerate((x, w))] for s in (1, -1)]
            moved = (sides[0][i].double() - sides[1][i].double())
            slope = (loss(*sides[0]).double() - loss(*sides[1]).double()).item()
            want = (grads[i].double() * moved).sum().item()
            # x moves a logit by at most about 64 * 0.2 / 32 = 0.4 (w: 0.8 / 32 * 64 of the one token): the cubes that a central difference leaves are 0.4^3 / 3 =
            # 0.02 of a token's loss, against a slope of about 64 * 0.2 / 16 = 0.8
            assert abs(slope - want) <= 0.05 * abs(want), (slope, want)


def test_streams_and_graphs(cuda):
    """On another stream, and captured: both passes replayed with new inputs, eager work between the replays, two graphs at once."""
    import sparse
    gen, x, w, b = operands(cuda, 67, 300, 256, 3000, BF16, F32)
    batches = []
    for i in range(4):
        t = torch.where(torch.rand(300, generator=gen) < 0.2 * i, -100, torch.randint(0, 3000, (300,), generator=gen)).to(cuda)
        idx = torch.where(torch.rand(300, 5, generator=gen) < 0.2 * i, -1, torch.randint(0, 3000, (300, 5), generator=gen)).to(cuda)
        batches.append((draw(gen, 300, 256, dtype=BF16).to(cuda), t, idx, draw(gen, 300, 5).to(cuda)))
    one = torch.tensor(1.0, device=cuda)
    want = [(ce_step(v, w, b, t, one), kd_step(v, w, b, i, l, one)) for v, t, i, l in batches]
    flat = lambda r: [r[0], *r[1]]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        on_side = ce_step(batches[1][0], w, b, batches[1][1], one)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, c) for a, c in zip(flat(on_side), flat(want[1][0])))
    held = [t.clone() for t in batches[0]]
    graphs = []
    for step in (lambda: ce_step(held[0], w, b, held[1], one), lambda: kd_step(held[0], w, b, held[2], held[3], one)):
        with torch.cuda.stream(side):
            step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        graphs.append((graph, flat(out)))
    for n in (0, 2, 1, 3, 0):
        for h, t in zip(held, batches[n]):
            h.copy_(t)
        for graph, _ in graphs:
            graph.replay()
        ce_step(batches[3][0], w, b, batches[3][1], one)
        torch.cuda.synchronize()
        for (_, out), r in zip(graphs, want[n]):
            assert all(torch.equal(a, c) for a, c in zip(out, flat(r))), n


def test_head_of_a_model(cuda):
    """Norm, 2:4 layer, gated activation, layer, residual, norm and the tied head with both losses, as a model runs them: gradients of all
    parameters against the same model with a dense head and torch's own loss of its float32 logits."""
    import sparse
    import torch.nn.functional as F
    torch.manual_seed(3)
    embedding = torch.nn.Embedding(1003, 128, device=cuda)
    torch.nn.init.normal_(embedding.weight, std=0.08)
    head = sparse.VocabularyLinear(128, 1003, device=cuda)
    head.weight = embedding.weight
    before, between = sparse.BlockNorm(128, "rms", out_dtype=F32, device=cuda), sparse.ResidualNorm(128, pre="rms", device=cuda)
    up, down = (sparse.SoftThresholdLinear(*d, device=cuda) for d in ((128, 512), (256, 128)))
    up.init_scale(), down.init_scale()
    words = torch.randint(0, 1003, (4, 65), device=cuda)
    words[1, 40:] = 7
    tokens, target = words[:, :-1], words[:, 1:].clone()
    target[1, 39:] = -100
    indices, logits = torch.randint(0, 1003, (4, 64, 6), device=cuda), torch.randn(4, 64, 6, device=cuda)
    params = [embedding.weight, before.weight, up.weight, up.bias, down.weight, down.bias, between.pre_weight]

    def step(losses):
        with torch.autocast("cuda", dtype=BF16):
            h = embedding(tokens)
            y = down(sparse.gelu_glu_checkpoint.apply(up(before(h))))
            _, n = sparse.residual_norm(h, y.float(), pre_kind="rms", pre_weight=between.pre_weight)
            loss = losses(n)
        return loss.detach(), torch.autograd.grad(loss, params)

    def fused(n):
        return head(n, target) + 0.5 * head(n, indices=indices, teacher_logits=logits, temperature=2.0)

    def dense(n):
        z = head(n).float()
        q, u = torch.softmax(logits / 2, -1), torch.log_softmax(z / 2, -1)
        return F.cross_entropy(z.view(-1, 1003), target.reshape(-1)) + 0.5 * (q * (q.log() - u.gather(-1, indices))).sum(-1).mean()

    loss, grads = step(fused)
    want, wanted = step(dense)
    assert (loss - want).abs() <= 2.0 ** -8 * want                 # (the dense head rounds its logits to bfloat16)
    for g, v in zip(grads, wanted):
        assert (g - v).norm() <= 2.0 ** -4 * v.norm(), (v.shape, (g - v).norm() / v.norm())
    assert head(before(embedding(tokens)).detach()).shape == (4, 64, 1003)
    with pytest.raises(RuntimeError, match="either a target"):
        head(embedding(tokens), target, indices=indices, teacher_logits=logits)


def test_two_threads(cuda):
    """Calls at once from two threads, on streams of their own."""
    import threading
    gen, x, w, b = operands(cuda, 73, 500, 200, 3000, BF16, F32)
    target = torch.randint(0, 3000, (500,), generator=gen).to(cuda)
    indices, logits = torch.randint(0, 3000, (500, 9), generator=gen).to(cuda), draw(gen, 500, 9).to(cuda)
    one = torch.tensor(1.0, device=cuda)
    steps = (lambda: ce_step(x, w, b, target, one), lambda: kd_step(x, w, b, indices, logits, one))
    want = [step() for step in steps]
    torch.cuda.synchronize()
    got = [[], []]

    def run(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(5):
                got[i].append(steps[i]())
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    for i in range(2):
        assert len(got[i]) == 5 and all(torch.equal(r[0], want[i][0]) and all(torch.equal(a, c) for a, c in zip(r[1], want[i][1])) for r in got[i])


def test_called_from_compiled_code(cuda):
    """What the compiler cannot trace it leaves to Python."""
    import sparse
    gen, x, w, _ = operands(cuda, 79, 130, 64, 300, BF16)
    target = torch.randint(0, 300, (130,), generator=gen).to(cuda)
    want = ce_step(x, w, None, target, torch.tensor(2.0, device=cuda))
    torch._dynamo.reset()
    leaves = [x.clone().requires_grad_(), w.clone().requires_grad_()]
    loss = torch.compile(lambda x, w: sparse.linear_cross_entropy(x, w, target) * 2, backend="eager")(*leaves)
    loss.backward()
    torch._dynamo.reset()
    assert torch.equal(loss.detach(), want[0] * 2) and all(torch.equal(t.grad, g) for t, g in zip(leaves, want[1]))


def test_saved_tensors_are_looked_at(cuda):
    """What a hook hands back instead of a saved tensor is not read as what it is not; what it brings back from the host is."""
    gen, x, w, _ = operands(cuda, 83, 40, 64, 300, BF16)
    target = torch.randint(0, 300, (40,), generator=gen).to(cuda)
    one = torch.tensor(1.0, device=cuda)
    want = ce_step(x, w, None, target, one)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu(), lambda t: t.to(cuda)):
        got = ce_step(x, w, None, target, one)
    assert all(torch.equal(a, c) for a, c in zip(got[1], want[1]))
    for spoil in (lambda t: t[:1], lambda t: t.cpu(), lambda t: t.float()):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, spoil), pytest.raises(RuntimeError, match="saved"):
            ce_step(x, w, None, target, one)


def test_refusals(cuda):
    import sparse
    x, w, t = torch.zeros(4, 64, dtype=BF16, device=cuda), torch.zeros(10, 64, dtype=BF16, device=cuda), torch.zeros(4, dtype=torch.long, device=cuda)
    i, l = torch.zeros(4, 2, dtype=torch.long, device=cuda), torch.zeros(4, 2, device=cuda)
    ce, kd = sparse.linear_cross_entropy, sparse.linear_distillation
    for call, what in ((lambda: ce(x.cpu(), w, t), "CUDA"), (lambda: ce(x, w.cpu(), t), "CUDA"), (lambda: ce(x, w, t.cpu()), "target"), (lambda: ce(x, w[:, :32], t), "suit"),
                       (lambda: ce(x, w, t[:3]), "target"), (lambda: ce(x, w, t.float()), "dtype"), (lambda: ce(x.float(), w, t), "not supported"),
                       (lambda: ce(x.half(), w, t), "not supported"), (lambda: ce(x, w, t, torch.zeros(9, device=cuda)), "bias"), (lambda: ce(x, w, t, reduction="max"), "reduction"),
                       (lambda: ce(x, w, t, label_smoothing=1.5), "label_smoothing"), (lambda: ce(x, w, t, z_loss=-1.0), "z_loss"), (lambda: ce(x, w, t, z_loss=float("nan")), "z_loss"),
                       (lambda: ce(x, w, t, ignore_index=None), "ignore_index"), (lambda: ce(x, w, t, ignore_index=1 << 64), "ignore_index"), (lambda: ce(x, w, None), "target"), (lambda: ce(x.long(), w, t), "dtype"),
                       (lambda: kd(x, w, i[:, :0], l[:, :0]), "entries"), (lambda: kd(x, w, i, l[:, :1]), "teacher_logits"), (lambda: kd(x, w, i, l.requires_grad_()), "gradient"),
                       (lambda: kd(x, w, i, l.detach(), temperature=0.0), "temperature"), (lambda: kd(x, w, i, l.detach(), teacher_lse=l[:, 0][:2]), "teacher_lse"),
                       (lambda: kd(x, w, i.expand(4, 2).repeat(1, 600), l.detach().repeat(1, 600)), "entries")):
        with pytest.raises(RuntimeError, match=what):
            call()
