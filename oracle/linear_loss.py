"""Oracle: the losses of a vocabulary head, loss of each token, gradient of the logits and gradients of the operands.

TEST INFRASTRUCTURE ONLY -- never imported by the shipped package.  The reference has no such operators; these are the formulas in
float64.

Pinned by: torch's cross_entropy and kl_div in float64 and autograd's gradients of them.
"""
import torch


def logits(x, weight, bias=None):
    z = x.double().reshape(-1, x.shape[-1]) @ weight.double().t()
    return z if bias is None else z + bias.double()


def cross_entropy(z, target, ignore_index=-100, label_smoothing=0.0, z_loss=0.0):
    """(loss of each token, its gradient with respect to the logits z, which tokens count)"""
    target = target.reshape(-1)
    counts = target != ignore_index
    lse = torch.logsumexp(z, 1)
    at = torch.where(counts, target, 0)[:, None]
    loss = (1 - label_smoothing) * (lse - z.gather(1, at)[:, 0]) + z_loss * lse ** 2
    slope = torch.exp(z - lse[:, None]) * (1 + 2 * z_loss * lse[:, None])
    if label_smoothing:
        loss = loss + label_smoothing * (lse - z.mean(1))
        slope = slope - label_smoothing / z.shape[1]
    slope = slope.scatter_add(1, at, torch.full_like(at, label_smoothing - 1, dtype=torch.float64))
    return torch.where(counts, loss, 0.0), torch.where(counts[:, None], slope, 0.0), counts


def distillation(z, indices, teacher_logits, teacher_lse=None, temperature=1.0):
    """The same, against the words that a teacher lists; what is listed with a negative word is unused."""
    entries = indices.shape[-1]
    indices, t = indices.reshape(-1, entries), teacher_logits.double().reshape(-1, entries) / temperature
    used = indices >= 0
    t = torch.where(used, t, -torch.inf)
    counts = (t != -torch.inf).any(1)
    of_teacher = torch.logsumexp(t, 1) if teacher_lse is None else teacher_lse.double().reshape(-1)
    logq = t - torch.where(counts, of_teacher, 0.0)[:, None]
    q = torch.exp(logq)
    u = z / temperature
    lse = torch.logsumexp(u, 1)
    at = indices.clamp(min=0)
    loss = torch.where(q > 0, q * (logq - u.gather(1, at) + lse[:, None]), 0.0).sum(1)
    slope = torch.exp(u - lse[:, None]) * q.sum(1, keepdim=True)
    slope = slope.scatter_add(1, at, -q) / temperature
    return torch.where(counts, loss, 0.0), torch.where(counts[:, None], slope, 0.0), counts


def reduced(loss, counts, reduction):
    return loss if reduction == "none" else loss.sum() / counts.sum().clamp(min=1) if reduction == "mean" else loss.sum()


def gradients(slope, counts, grad, reduction, x, weight, bias=None):
    """(dx, dW, db, gradient of the logits) for the gradient `grad` of the reduced loss; rows of x that do not count are not looked at"""
    g = grad.double().reshape(-1) if reduction == "none" else grad.double() / (counts.sum().clamp(min=1) if reduction == "mean" else 1)
    p = slope * torch.where(counts, g, 0.0)[:, None]
    rows = torch.where(counts[:, None], x.double().reshape(-1, x.shape[-1]), 0.0)
    return (p @ weight.double()).view(x.shape), p.t() @ rows, None if bias is None else p.sum(0), p
