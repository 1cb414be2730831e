"""The head of a language model together with its loss, as cases that can be timed.

  cross_entropy  linear_cross_entropy: the head's product, softmax cross entropy over the vocabulary with label smoothing and a term in the
                 square of the log-sum-exp, tokens that do not count; the loss alone (scoring a text) or with its gradients (training)
  distillation   linear_distillation: the same product, against the largest logits of a teacher; with or without gradients

With z = x W^T + b, u = z / temperature and lse the logarithm of the sum of exponentials over the vocabulary:

  cross_entropy   lse - (1 - s) z[target] - s mean(z) + c lse^2
  distillation    sum_k q_k (log q_k - u[i_k] + lse(u)),  q = exp(t / temperature - teacher's lse), or the softmax of the t / temperature given

Each has a plain form (elementary operations in float32, rounded once at the end), the framework's call (`own`), and `exact`, the definition in
float64.
"""
import os
import sys

import torch

own = False

_DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def _sparse():
    """The package of the tree this runs in."""
    at = os.path.join(os.getcwd(), "2by4-pretrain_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    import sparse
    return sparse


_PLAIN = {"train": False, "dtype": "bf16", "bias": False, "grad": 1.0}
_CE = dict(_PLAIN, kind="cross_entropy", ignored=0.0, smoothing=0.0, z_loss=0.0, reduction="mean")
_KD = dict(_PLAIN, kind="distillation", k=64, used=1.0, temperature=1.0, teacher_lse=False, reduction="mean")


def listed():
    return [
        # the probability of the next token while text is generated or scored one token at a time: GPT-2's head
        dict(_CE, name="ce_score_token", tokens=1, d=768, v=50304, reduction="none"),
        # a few ragged continuations scored together: a vocabulary and a width that are no multiple of anything
        dict(_CE, name="ce_score_ragged", tokens=37, d=1601, v=50257, dtype="fp16", reduction="none"),
        # evaluating a held-out text: loss of full sequences, no gradients
        dict(_CE, name="ce_evaluate", tokens=8192, d=1024, v=50304),
        # a training step on one sequence of GPT-2
        dict(_CE, name="ce_train_sequence", tokens=1024, d=768, v=50304, train=True),
        # GPT-2's training step: 12 sequences of 1024
        dict(_CE, name="ce_train_batch", tokens=12288, d=768, v=50304, train=True),
        # fine-tuning on answers: the prompts' tokens do not count; smoothing, bias, a loss scale for float16
        dict(_CE, name="ce_finetune_masked", tokens=5003, d=1280, v=50257, dtype="fp16", train=True, bias=True, ignored=0.6, smoothing=0.1, z_loss=1e-4, grad=1024.0),
        # a wide model with a large vocabulary
        dict(_CE, name="ce_train_large", tokens=8192, d=4096, v=128000, train=True, z_loss=1e-4),
        # how far a pruned model is from its teacher, on a ragged batch
        dict(_KD, name="kd_score_ragged", tokens=333, d=1601, v=50257, dtype="fp16", k=100, used=0.7, teacher_lse=True, reduction="none"),
        # a distillation step on one sequence
        dict(_KD, name="kd_train_sequence", tokens=1024, d=768, v=50304, k=16, train=True, temperature=2.0),
        # a distillation step of a batch, 64 logits of the teacher a token
        dict(_KD, name="kd_train_batch", tokens=8192, d=1024, v=50304, k=64, train=True, teacher_lse=True),
        # the same of a wide model with a large vocabulary, each token with a weight of its own
        dict(_KD, name="kd_train_large", tokens=4096, d=4096, v=128000, k=128, train=True, temperature=1.5, reduction="none"),
    ]


def _log(rng, lo, hi):
    """An integer spread over the logarithm of [lo, hi]."""
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    d = _log(rng, 64, 4096)
    if rng.random() < 0.6:                                         # most models' widths are multiples of 64
        d = max(64, d // 64 * 64)
    v = _log(rng, 256, 131072)
    if rng.random() < 0.5:                                         # many vocabularies are padded
        v = max(256, v // 64 * 64)
    tokens = _log(rng, 1, max(1, min(16384, 8192 * 4096 * 128000 // (d * v))))
    case = {"tokens": tokens, "d": d, "v": v, "train": rng.random() < 0.7, "dtype": rng.choice(["bf16", "fp16"]),
            "bias": rng.random() < 0.3, "reduction": rng.choice(["mean", "sum", "none"])}
    case["grad"] = 1.0 if case["dtype"] == "bf16" else 64.0 if case["reduction"] == "mean" else 1.0
    if rng.random() < 0.6:
        return dict(_CE, **case, ignored=rng.choice([0.0, 0.0, 0.3, 0.8]), smoothing=rng.choice([0.0, 0.0, 0.1]), z_loss=rng.choice([0.0, 1e-4, 1e-3]))
    return dict(_KD, **case, k=_log(rng, 1, 256), used=rng.choice([1.0, 1.0, 0.6]), temperature=rng.choice([1.0, 0.7, 2.0]), teacher_lse=rng.random() < 0.5)


# ------------------------------------------------------------------ what a program holds before the call
def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    t, d, v, dtype = case["tokens"], case["d"], case["v"], _DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=gen)

    def uniform(*shape):
        return torch.rand(*shape, device="cuda", generator=gen)

    # logits of a few units beside the one that the model has learned to expect, which is up to 12 above
    weight = normal(v, d).mul_(2.0 / d ** 0.5)
    x = normal(t, d) * torch.exp(0.5 * normal(d) - 0.25)
    frequent = (v ** uniform(t)).long().clamp_(1, v) - 1           # words are used in proportion to one over their rank
    for at in range(0, t, 4096):
        rows = weight[frequent[at:at + 4096]]
        x[at:at + 4096] += rows * (12.0 * uniform(rows.shape[0], 1) / rows.square().sum(-1, keepdim=True))
    state = {"case": case, "x": x.to(dtype), "weight": weight.to(dtype), "bias": None}
    if case["bias"]:
        state["bias"] = (0.5 * normal(v)).to(dtype)
    if case["kind"] == "cross_entropy":
        state["target"] = torch.where(uniform(t) < case["ignored"], -100, frequent)
    else:
        # the teacher's k words, denser among the frequent ones; none twice
        k = min(case["k"], v)
        edges = torch.linspace(0, 1, k + 1, device="cuda", dtype=torch.float64)
        edges = torch.maximum((edges * torch.log(torch.tensor(float(v + 1)))).exp().sub(1).long(), torch.arange(k + 1, device="cuda")).clamp_(max=v)
        edges = torch.minimum(edges, v - k + torch.arange(k + 1, device="cuda"))
        low, width = edges[:-1], edges[1:] - edges[:-1]
        indices = low + torch.minimum((uniform(t, k) * width).long(), width - 1)
        indices = indices.gather(1, uniform(t, k).argsort(1))
        logits = (4.0 * normal(t, k)).sort(1, descending=True).values
        if case["used"] < 1.0:                                     # a teacher that kept fewer words where it was sure; for some tokens none
            kept = (uniform(t, 1) * (k + 1) * 2 * case["used"]).long()
            indices = torch.where(torch.arange(k, device="cuda") < kept, indices, -1)
        state["indices"], state["teacher_logits"] = indices, logits.to(dtype)
        state["teacher_lse"] = None
        if case["teacher_lse"]:
            state["teacher_lse"] = torch.logsumexp(state["teacher_logits"].float() / case["temperature"], 1) + 0.2 * uniform(t)
    state["leaves"] = [s for s in (state["x"], state["weight"], state["bias"]) if s is not None]
    if case["train"]:
        for s in state["leaves"]:
            s.requires_grad_()
        state["grad"] = torch.tensor(case["grad"], device="cuda") if case["reduction"] != "none" else case["grad"] * (0.5 + uniform(t)) / t
    return state


# ------------------------------------------------------------------ plain forms
def _plain(state):
    case = state["case"]
    dtype = _DTYPES[case["dtype"]]
    x, w = state["x"].detach().float(), state["weight"].detach().float()
    u = torch.mm(x, w.t())
    if case["bias"]:
        u = u + state["bias"].detach().float()
    if case["kind"] == "cross_entropy":
        target, smoothing, z_loss = state["target"], case["smoothing"], case["z_loss"]
        counts = target != -100
        at, q = torch.where(counts, target, 0)[:, None], None
    else:
        indices = state["indices"]
        u = u / case["temperature"]
        used, at = indices >= 0, indices.clamp(min=0)
        counts = used.any(1)
        logq = torch.where(used, state["teacher_logits"].float() / case["temperature"], -torch.inf)
        if case["teacher_lse"]:
            logq = logq - state["teacher_lse"][:, None]
        else:
            top = torch.where(counts[:, None], logq.amax(1, keepdim=True), 0.0)
            logq = logq - top - (torch.exp(logq - top).sum(1, keepdim=True)).log()
        q = torch.where(used, torch.exp(logq), 0.0)
    top = u.amax(1, keepdim=True)
    e = torch.exp(u - top)
    total = e.sum(1, keepdim=True)
    lse = (top + total.log())[:, 0]
    picked = u.gather(1, at)
    if q is None:
        loss = lse - (1.0 - smoothing) * picked[:, 0] + z_loss * lse * lse
        if smoothing:
            loss = loss - smoothing * u.mean(1)
    else:
        loss = torch.where(q > 0, q * (logq - picked + lse[:, None]), 0.0).sum(1)
    loss = torch.where(counts, loss, 0.0)
    n = counts.sum().clamp(min=1)
    out = loss.sum() / n if case["reduction"] == "mean" else loss.sum() if case["reduction"] == "sum" else loss
    if not case["train"]:
        return {"loss": out}
    g = state["grad"] / n if case["reduction"] == "mean" else state["grad"]
    g = torch.where(counts, g, 0.0)[:, None]
    p = e.div_(total)
    if q is None:
        p = p * (g * (1.0 + 2.0 * z_loss * lse[:, None]))
        if smoothing:
            p = p - g * (smoothing / case["v"])
        p.scatter_add_(1, at, -(1.0 - smoothing) * g)
    else:
        g = g / case["temperature"]
        p = p * (g * q.sum(1, keepdim=True))
        p.scatter_add_(1, at, -g * q)
    grads = [torch.mm(p, w).to(dtype), torch.mm(p.t(), x).to(dtype)]
    if case["bias"]:
        grads.append(p.sum(0).to(dtype))
    return {"loss": out, "grads": grads}


# ------------------------------------------------------------------ one pass
def run(state):
    case = state["case"]
    if not own:
        return _plain(state)
    sparse = _sparse()
    if case["kind"] == "cross_entropy":
        loss = sparse.linear_cross_entropy(state["x"], state["weight"], state["target"], state["bias"], label_smoothing=case["smoothing"],
                                           z_loss=case["z_loss"], reduction=case["reduction"])
    else:
        loss = sparse.linear_distillation(state["x"], state["weight"], state["indices"], state["teacher_logits"], state["bias"],
                                          teacher_lse=state["teacher_lse"], temperature=case["temperature"], reduction=case["reduction"])
    if not case["train"]:
        return {"loss": loss}
    return {"loss": loss.detach(), "grads": list(torch.autograd.grad(loss, state["leaves"], state["grad"]))}


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    """Inputs read once, outputs written once; the products of the tokens that count."""
    t, d, v = case["tokens"], case["d"], case["v"]
    counting = t * (1.0 - case.get("ignored", 0.0))
    entries = 8 * t if case["kind"] == "cross_entropy" else 10 * t * case["k"]
    moved = 2 * t * d + 2 * v * (d + case["bias"]) + entries + 4 * t
    if case["train"]:
        moved += 2 * t * d + 2 * v * (d + case["bias"])
    return {"bytes": int(moved), "flops": int((6 if case["train"] else 2) * counting * d * v)}


# ------------------------------------------------------------------ the definitions in float64
def exact(case, seed):
    state = prepare(case, seed)
    v = case["v"]
    x = state["x"].detach().double()
    w = state["weight"].detach().double()
    scores = x @ w.T
    if state["bias"] is not None:
        scores += state["bias"].detach().double()
    soft = {"cross_entropy": 1.0, "distillation": case.get("temperature")}[case["kind"]]
    logp = torch.log_softmax(scores / soft, dim=-1)
    rows = torch.arange(case["tokens"], device=x.device)
    # wanted: the distribution that the student is held against, one column of it per listed word
    if case["kind"] == "cross_entropy":
        counting = (state["target"] != -100).double()
        words = state["target"].clamp(min=0)[:, None]
        wanted = torch.ones(case["tokens"], 1, dtype=torch.float64, device=x.device)
        lse = torch.logsumexp(scores, -1)
        loss = -(1 - case["smoothing"]) * logp[rows, words[:, 0]] - case["smoothing"] * logp.mean(-1) + case["z_loss"] * lse ** 2
        wanted, level, pull = wanted * (1 - case["smoothing"]), case["smoothing"] / v, 1 + 2 * case["z_loss"] * lse
    else:
        listed_words = state["indices"] >= 0
        counting = listed_words.any(-1).double()
        words = state["indices"].clamp(min=0)
        t = state["teacher_logits"].double() / soft
        t = t.masked_fill(~listed_words, float("-inf"))
        lse = torch.logsumexp(t, -1) if state["teacher_lse"] is None else state["teacher_lse"].double()
        wanted = torch.exp(t - lse[:, None]).masked_fill(~listed_words, 0.0)
        loss = (torch.special.xlogy(wanted, wanted) - wanted * torch.gather(logp, 1, words)).sum(-1)
        level, pull = 0.0, wanted.sum(-1)
    loss = torch.nan_to_num(loss) * counting
    many = max(1.0, counting.sum().item())
    result = {"mean": loss.sum() / many, "sum": loss.sum(), "none": loss}[case["reduction"]]
    if not case["train"]:
        return {"loss": result}
    upstream = state["grad"].double() * counting / soft / (many if case["reduction"] == "mean" else 1.0)
    slope = torch.exp(logp, out=logp)
    slope *= pull[:, None]
    if level:
        slope -= level
    for column in range(words.shape[1]):
        slope[rows, words[:, column]] -= wanted[:, column]
    slope *= torch.nan_to_num(upstream)[:, None]
    grads = [slope @ w, slope.T @ x]
    if state["bias"] is not None:
        grads.append(slope.sum(0))
    return {"loss": result, "grads": grads}
