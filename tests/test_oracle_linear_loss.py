"""The oracle of the vocabulary head's losses against torch's own losses in float64 and autograd's gradients of them."""
import pytest
import torch
import torch.nn.functional as F

from oracle import linear_loss as definition


def _operands(seed, tokens=30, cols=12, words=50):
    gen = torch.Generator().manual_seed(seed)
    make = lambda *shape: torch.randn(*shape, generator=gen, dtype=torch.float64)
    return gen, make(tokens, cols), make(words, cols), make(words)


def _same(got, want):
    assert all((a - b).abs().max() <= 1e-12 * max(1.0, b.abs().max()) for a, b in zip(got, want))


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("smoothing", [0.0, 0.3])
def test_cross_entropy(reduction, smoothing):
    gen, x, w, b = _operands(1)
    target = torch.where(torch.rand(30, generator=gen) < 0.3, -100, torch.randint(0, 50, (30,), generator=gen))
    leaves = [t.requires_grad_() for t in (x, w, b)]
    loss = F.cross_entropy(F.linear(x, w, b), target, label_smoothing=smoothing, reduction=reduction)
    grad = torch.randn(30, generator=gen, dtype=torch.float64) if reduction == "none" else torch.tensor(0.7, dtype=torch.float64)
    wanted = torch.autograd.grad(loss, leaves, grad)
    own, slope, counts = definition.cross_entropy(definition.logits(x, w, b).detach(), target, label_smoothing=smoothing)
    _same([definition.reduced(own, counts, reduction), *definition.gradients(slope, counts, grad, reduction, *(t.detach() for t in leaves))[:3]], [loss, *wanted])


def test_z_loss():
    gen, x, w, b = _operands(2)
    leaves = [t.requires_grad_() for t in (x, w, b)]
    target = torch.randint(0, 50, (30,), generator=gen)
    z = F.linear(x, w, b)
    loss = F.cross_entropy(z, target) + 0.01 * torch.logsumexp(z, 1).square().mean()
    wanted = torch.autograd.grad(loss, leaves)
    own, slope, counts = definition.cross_entropy(z.detach(), target, z_loss=0.01)
    _same([definition.reduced(own, counts, "mean"), *definition.gradients(slope, counts, torch.tensor(1.0), "mean", *(t.detach() for t in leaves))[:3]], [loss, *wanted])


@pytest.mark.parametrize("temperature", [1.0, 2.0])
def test_distillation(temperature):
    """All words listed: the divergence of two softmaxes."""
    gen, x, w, b = _operands(3)
    leaves = [t.requires_grad_() for t in (x, w, b)]
    teacher = torch.randn(30, 50, generator=gen, dtype=torch.float64)
    indices = torch.stack([torch.randperm(50, generator=gen) for _ in range(30)])
    z = F.linear(x, w, b)
    loss = F.kl_div(torch.log_softmax(z / temperature, 1), torch.log_softmax(teacher / temperature, 1), log_target=True, reduction="batchmean")
    wanted = torch.autograd.grad(loss, leaves)
    own, slope, counts = definition.distillation(z.detach(), indices, teacher.gather(1, indices), temperature=temperature)
    _same([definition.reduced(own, counts, "mean"), *definition.gradients(slope, counts, torch.tensor(1.0), "mean", *(t.detach() for t in leaves))[:3]], [loss, *wanted])


def test_entries():
    """Unused entries are not there; one that is listed twice counts twice; probabilities may be parts of a larger whole."""
    z = _operands(4)[2].t().contiguous()
    indices, logits = torch.tensor([[3, 5, -1, 3]] * 12), torch.tensor([[0.1, 0.7, float("nan"), -0.4]] * 12)
    lse = torch.full((12,), 2.0)
    loss, slope, counts = definition.distillation(z, indices, logits, lse)
    q = torch.exp(logits[0].double() - 2.0)
    logp = torch.log_softmax(z, 1)
    want = sum(q[k] * (logits[0, k].double() - 2.0 - logp[:, indices[0, k]]) for k in (0, 1, 3))
    assert counts.all() and torch.allclose(loss, want, rtol=1e-14, atol=0)
    p = torch.exp(logp) * (q[0] + q[1] + q[3])
    p[:, 3] -= q[0] + q[3]
    p[:, 5] -= q[1]
    assert torch.allclose(slope, p, rtol=1e-13, atol=1e-15)
