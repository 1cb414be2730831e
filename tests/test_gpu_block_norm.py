"""residual_norm / block_norm against float64.

Tolerances.  u = 2^-24.  A row's sums are trees of at most 16 sequential additions in a lane, 6 in a wave and 16 over waves, so a mean is off by at
most 40 u times the mean magnitude; with the products, the reciprocal root (1 unit) and the final multiply-adds every term below is off by
less than 64 u of the magnitudes that enter it, 128 u where an error of the statistics and one of the terms meet.  A centred value is off by u of
its own and of the mean's magnitude, which the factor 1 + |mean| r of a row stands for.  Sums over rows add at most rows / pieces + 32
terms in sequence, pieces in parallel: 256 u of the sum of the magnitudes.  Then one rounding to the output's type: eps / 2 of the value, plus half of
the smallest float16 (2^-25).
n and the gradients are those of `out` as it was returned (rounded): the formulas get it as it is."""
import itertools

import pytest
import torch

import oracle

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
U = 2.0 ** -24


@pytest.fixture(autouse=True, params=["torchcall", "python"])
def calls(request, monkeypatch):
    """Everything twice: with the module that makes ordinary calls from torch's C++ side, and with Python making all of them."""
    from sparse import _native as N
    if request.param == "python":
        monkeypatch.setattr(N, "_calls", None)
    elif N.torch_calls() is None:
        pytest.skip("_torchcall is not built for this torch")



def draw(seed, *shape, dtype=F32, std=1.0, mean=0.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed), dtype=torch.float64) * std + mean).to(dtype)


def close(name, got, want, magnitude, factor):
    """|got - want| within factor * u * magnitude and one rounding to got's type"""
    got64 = got.detach().cpu().double()
    tolerance = factor * U * magnitude + torch.finfo(got.dtype).eps / 2 * want.abs() * 1.01 + 2.0 ** -25 * (got.dtype == F16) + 1e-40
    off = (got64 - want).abs()
    bad = ~(off <= tolerance)
    assert not bad.any(), (name, int(bad.sum()), (off / tolerance)[bad].max().item(), torch.nonzero(bad)[0].tolist())


def check(cuda, lead, cols, stream, block, post, pre, gate, bias=True, param=None, scale=0.75, eps=1e-5, seed=0, mean=0.3, strided=False, gate_shape=None):
    import sparse
    param = param or stream
    rows = torch.Size(lead).numel()
    residual, y = draw(seed, *lead, cols, dtype=stream, mean=mean), draw(seed + 1, *lead, cols, dtype=block, mean=-mean)
    weights = {}
    for i, (which, kind) in enumerate((("post", post), ("pre", pre))):
        if kind:
            weights[which + "_weight"] = draw(seed + 2 + i, cols, dtype=param, std=0.2, mean=1.0)
            if bias:
                weights[which + "_bias"] = draw(seed + 4 + i, cols, dtype=param, std=0.2)
    if gate == "channel":
        gate_shape = (cols,)
    elif gate == "sequence":
        gate_shape = (lead[0],) + (1,) * (len(lead) - 1) + (cols,)
    elif gate == "token":
        gate_shape = (*lead, cols)
    g = None if gate is None else draw(seed + 6, *gate_shape, dtype=stream, std=0.3, mean=0.5)
    dout, dn = draw(seed + 7, *lead, cols, dtype=stream, std=0.1), draw(seed + 8, *lead, cols, dtype=block, std=0.1)

    def on(t):
        if t is None:
            return None
        if strided and t.dim() > 1:                                # rows that start anywhere, with something behind them
            wide = torch.full((*t.shape[:-1], t.shape[-1] + 5), float("nan"), dtype=t.dtype, device=cuda)
            wide[..., 3:-2] = t.to(cuda)
            return wide[..., 3:-2].detach()
        return t.to(cuda)

    leaves = {"residual": on(residual), "y": on(y), **{k: on(v) for k, v in weights.items()}}
    if g is not None:
        leaves["gate"] = on(g)
    for t in leaves.values():
        t.requires_grad_()
    call = dict(gate=leaves.get("gate"), residual_scale=scale, post_kind=post, pre_kind=pre, eps=eps, **{k: leaves[k] for k in weights})
    result = sparse.residual_norm(leaves["residual"], leaves["y"], **call)
    out, n = result if pre else (result, None)
    assert out.dtype == stream and out.shape == residual.shape and (n is None or (n.dtype == block and n.shape == y.shape))
    with torch.no_grad():                                          # the form without statistics: the same bits
        again = sparse.residual_norm(leaves["residual"], leaves["y"], **call)
        for a, b in zip(again if pre else (again,), (out, n)):
            assert torch.equal(a, b)
    outputs, grads = ((out, n), (on(dout), on(dn))) if pre else ((out,), (on(dout),))
    got = dict(zip(leaves, torch.autograd.grad(outputs, list(leaves.values()), grads)))

    # ---- float64
    f = lambda t: None if t is None else t.double().reshape(rows, cols)  # noqa: E731
    x64, y64, h64, dout64, dn64 = f(residual), f(y), out.detach().cpu().double().reshape(rows, cols), f(dout), f(dn)
    w64 = {k: v.double() for k, v in weights.items()}
    gate64 = torch.ones(rows, cols, dtype=torch.float64) if g is None else g.double().expand(*lead, cols).reshape(rows, cols)
    spread = lambda v, kind: 1 + (oracle.statistics(v, kind, eps)[0].abs() * oracle.statistics(v, kind, eps)[1]) if kind else 1.0  # noqa: E731

    def normed(v, kind, which):
        want = oracle.norm(v, kind, w64[which + "_weight"], w64.get(which + "_bias"), eps)
        mean, r = oracle.statistics(v, kind, eps)
        size = ((v - mean).abs() * r * spread(v, kind) + 1) * w64[which + "_weight"].abs() + (w64[which + "_bias"].abs() if bias else 0)
        return want, size

    z, z_size = normed(y64, post, "post") if post else (y64, y64.abs())
    close("out", out.reshape(rows, cols), scale * x64 + gate64 * z, (scale * x64).abs() + gate64.abs() * z_size, 64)
    d, d_size = dout64, dout64.abs()
    if pre:
        want, size = normed(h64, pre, "pre")
        close("n", n.reshape(rows, cols), want, size, 64)
        dh, dw, db = oracle.norm_backward(dn64, h64, pre, w64["pre_weight"], eps)
        mean, r = oracle.statistics(h64, pre, eps)
        hat, q = (h64 - mean).abs() * r, (dn64 * w64["pre_weight"]).abs()
        s = spread(h64, pre)
        d, d_size = d + dh, d_size + r * s * (q + q.mean(-1, keepdim=True) + (1 + hat) * ((q * (1 + hat)).mean(-1, keepdim=True)))
        close("pre_weight", got["pre_weight"], dw.sum(0), (dn64.abs() * (hat + 1) * s).sum(0), 256)
        if bias:
            close("pre_bias", got["pre_bias"], db.sum(0), dn64.abs().sum(0), 256)
    close("residual", got["residual"].reshape(rows, cols), scale * d, abs(scale) * d_size, 128)
    dz, dz_size = d * gate64, d_size * gate64.abs()
    if post:
        dy, dw, db = oracle.norm_backward(dz, y64, post, w64["post_weight"], eps)
        mean, r = oracle.statistics(y64, post, eps)
        hat, q = (y64 - mean).abs() * r, dz_size * w64["post_weight"].abs()
        s = spread(y64, post)
        close("post_weight", got["post_weight"], dw.sum(0), (dz_size * (hat + 1) * s).sum(0), 256)
        if bias:
            close("post_bias", got["post_bias"], db.sum(0), dz_size.sum(0), 256)
        close("y", got["y"].reshape(rows, cols), dy, r * s * (q + q.mean(-1, keepdim=True) + (1 + hat) * (q * (1 + hat)).mean(-1, keepdim=True)), 256)
    else:
        close("y", got["y"].reshape(rows, cols), dz, dz_size, 128)
    if g is not None:
        terms, sizes = (d * z).reshape(*lead, cols), (d_size * (z_size + 1)).reshape(*lead, cols)
        shape = torch.Size((1,) * (len(lead) + 1 - g.dim()) + tuple(g.shape))
        axes = tuple(i for i, (a, b) in enumerate(zip(shape, terms.shape)) if a != b)
        want, size = (terms.sum(axes, keepdim=True), sizes.sum(axes, keepdim=True)) if axes else (terms, sizes)
        close("gate", got["gate"], want.reshape(g.shape), size.reshape(g.shape), 256)
    return leaves, out, n


SIZES = [((1,), 1), ((3,), 7), ((2, 3), 8), ((37,), 33), ((5,), 512), ((9,), 513), ((2, 150), 768), ((5,), 1024), ((6,), 1025), ((2, 13), 1601), ((3,), 2048),
         ((5,), 2056), ((4,), 4096), ((3,), 4099), ((2,), 8192), ((3,), 8200), ((2,), 16384)]


@pytest.mark.parametrize("lead,cols", SIZES)
def test_sizes(cuda, lead, cols):
    i = SIZES.index((lead, cols))
    stream, block = [(F32, F16), (BF16, BF16), (F32, BF16), (F16, F16), (F32, F32)][i % 5]
    post, pre = [("layer", "layer"), ("rms", "rms"), (None, "layer"), ("rms", None), ("layer", "rms")][i % 5]
    check(cuda, lead, cols, stream, block, post, pre, ["channel", None, "sequence", "token"][i % 4], seed=10 * i)


@pytest.mark.parametrize("post,pre,gate", list(itertools.product([None, "rms", "layer"], [None, "rms", "layer"], [None, "channel", "sequence", "token"])))
def test_kinds_and_gates(cuda, post, pre, gate):
    check(cuda, (3, 21), 200, F32, BF16, post, pre, gate, seed=77)


@pytest.mark.parametrize("stream,block,param", [(F32, F32, F32), (F32, F16, F16), (F32, BF16, BF16), (F16, F16, F32), (BF16, BF16, F32), (BF16, BF16, F16)])
def test_types_of_streams_and_parameters(cuda, stream, block, param):
    check(cuda, (4, 11), 328, stream, block, "layer", "rms", "sequence", param=param, seed=5)


@pytest.mark.parametrize("cols", [40, 77, 1600])
@pytest.mark.parametrize("bias", [True, False])
def test_strided_rows_at_any_alignment(cuda, cols, bias):
    check(cuda, (2, 9), cols, BF16, BF16, "rms", "layer", "token", bias=bias, strided=True, seed=6)
    check(cuda, (2, 9), cols, F32, F16, None, "rms", "channel", bias=bias, strided=True, seed=7)


@pytest.mark.parametrize("rows,seq", [(6000, 6000), (5000, 100), (4000, 2), (2051, 2051), (4096, 1024)])
def test_many_rows_and_groups_of_a_gate(cuda, rows, seq):
    """More rows than workgroups; gates for groups of a few rows and of many."""
    check(cuda, (rows // seq, seq), 72, F32, F16, "layer", "layer", "sequence", seed=8)


@pytest.mark.parametrize("shape", [(), (1,), (1, 1, 1), (3, 1, 1), (1, 5, 64), (3, 5, 1), (5, 64), (1, 64), (3, 1, 64), (3, 5, 64)])
def test_gates_that_broadcast(cuda, shape):
    check(cuda, (3, 5), 64, F32, F16, "rms", "rms", "given", gate_shape=shape, seed=9)


def test_large_means_keep_the_variance(cuda):
    """Values around 300 with a deviation of 1: the variance is taken from the centred values."""
    check(cuda, (7,), 1000, F32, F32, "layer", "layer", "channel", mean=300.0, scale=1.0, seed=12)


def test_no_rows(cuda):
    import sparse
    x, y, w = (torch.zeros(*s, device=cuda, requires_grad=True) for s in ((0, 4, 64), (0, 4, 64), (64,)))
    for gate in (torch.ones(64, device=cuda, requires_grad=True), torch.ones(0, 1, 64, device=cuda, requires_grad=True), torch.ones(0, 4, 64, device=cuda, requires_grad=True)):
        out, n, kept = sparse.residual_norm(x, y, gate, post_kind="rms", post_weight=w, pre_kind="layer", pre_weight=w, checkpoint=True)
        assert out.shape == n.shape == kept.decode().shape == (0, 4, 64)
        for t, g in zip((x, y, w, gate), torch.autograd.grad((out, n), (x, y, w, gate), (out.detach(), n.detach()))):
            assert g.shape == t.shape and not g.any()


def test_rows_of_zeros_infinities_and_nans_stay_in_their_rows(cuda):
    import sparse
    x = draw(20, 6, 96, dtype=F32)
    x[1], x[2, 5], x[4, 0] = 0, float("inf"), float("nan")
    w = draw(21, 96, mean=1.0)
    for kind in ("rms", "layer"):
        n = sparse.block_norm(x.to(cuda), w.to(cuda), kind=kind, eps=1e-6).cpu()
        want = oracle.norm(x, kind, w, None, 1e-6)
        assert not n[1].any()
        for r in (0, 3, 5):
            assert torch.allclose(n[r].double(), want[r], rtol=1e-5, atol=1e-6)
        assert n[2].isnan().any() and n[4].isnan().all()


def test_norm_alone_and_types(cuda):
    import sparse
    x, w, b, dn = draw(30, 4, 6, 200, dtype=F32), draw(31, 200, mean=1.0), draw(32, 200), draw(33, 4, 6, 200, dtype=F16, std=0.1)
    for kind, bias in (("rms", None), ("layer", b)):
        leaves = [t.to(cuda).requires_grad_() for t in (x, w, b) if t is not b or bias is not None]
        n = sparse.block_norm(leaves[0], leaves[1], leaves[2] if bias is not None else None, kind=kind, out_dtype=F16)
        assert n.dtype == F16
        close("n", n, oracle.norm(x, kind, w, bias, 1e-5), (x.double().abs() * 2 + 2) * (w.double().abs() + 1), 64)
        got = torch.autograd.grad(n, leaves, dn.to(cuda))
        dx, dw, db = oracle.norm_backward(dn, x, kind, w, 1e-5)
        r = oracle.statistics(x, kind, 1e-5)[1]
        close("x", got[0], dx, r * 2 * (dn.double().abs().mean() * 8 + dn.double().abs()) * 4 * (1 + x.double().abs()), 128)
        close("weight", got[1], dw.sum((0, 1)), (dn.double().abs() * (x.double().abs() + 1) * 2).sum((0, 1)), 256)
        if bias is not None:
            close("bias", got[2], db.sum((0, 1)), dn.double().abs().sum((0, 1)), 256)
    assert sparse.block_norm(x.half().to(cuda)).dtype == F16
    with pytest.raises(RuntimeError, match="not supported"):
        sparse.block_norm(x.half().to(cuda), out_dtype=F32)


def test_gradients_against_differences(cuda):
    """A directional derivative of a weighted sum of the outputs, by central differences in float32 around points where the outputs are smooth:
    differences of 2^-6 in inputs near 1 are off by their third derivative (2^-12 of the value) and by the rounding of the outputs."""
    import sparse
    torch.manual_seed(0)
    shapes = {"residual": (2, 7, 48), "y": (2, 7, 48), "gate": (2, 1, 48), "post_weight": (48,), "post_bias": (48,), "pre_weight": (48,), "pre_bias": (48,)}
    point = {k: draw(40 + i, *s, mean=0.5) for i, (k, s) in enumerate(shapes.items())}
    along = {k: draw(60 + i, *s) for i, (k, s) in enumerate(shapes.items())}
    wo, wn = draw(80, 2, 7, 48), draw(81, 2, 7, 48)

    def value(h, which):
        t = {k: (v + (h * along[k] if k == which else 0)).to(cuda) for k, v in point.items()}
        out, n = sparse.residual_norm(t.pop("residual"), t.pop("y"), post_kind="layer", pre_kind="rms", **t)
        return ((out.double() * wo.to(cuda)).sum() + (n.double() * wn.to(cuda)).sum()).item()

    leaves = {k: v.to(cuda).requires_grad_() for k, v in point.items()}
    t = dict(leaves)
    out, n = sparse.residual_norm(t.pop("residual"), t.pop("y"), post_kind="layer", pre_kind="rms", **t)
    grads = dict(zip(leaves, torch.autograd.grad((out, n), list(leaves.values()), (wo.to(cuda), wn.to(cuda)))))
    for k in shapes:
        want = (value(2.0 ** -6, k) - value(-(2.0 ** -6), k)) / 2.0 ** -5
        got = (grads[k].double().cpu() * along[k].double()).sum().item()
        scale = (grads[k].double().cpu() * along[k].double()).norm().item()
        assert abs(got - want) < 2e-2 * scale + 1e-2, (k, got, want)


def test_only_some_gradients_wanted(cuda):
    import sparse
    base = dict(post_kind="rms", pre_kind="layer")
    t = {k: draw(50 + i, *s, mean=0.5).to(cuda) for i, (k, s) in enumerate({"residual": (3, 9, 80), "y": (3, 9, 80), "gate": (80,), "post_weight": (80,),
                                                                              "pre_weight": (80,), "pre_bias": (80,)}.items())}
    go, gn = draw(58, 3, 9, 80).to(cuda), draw(59, 3, 9, 80).to(cuda)

    def grads(wanted, outputs):
        leaves = {k: v.detach().requires_grad_(k in wanted) for k, v in t.items()}
        r = dict(leaves)
        out = sparse.residual_norm(r.pop("residual"), r.pop("y"), **r, **base)
        pick = [(o, g) for o, g, use in zip(out, (go, gn), outputs) if use]
        return dict(zip(wanted, torch.autograd.grad([o for o, _ in pick], [leaves[k] for k in wanted], [g for _, g in pick], allow_unused=True)))

    full = grads(list(t), (True, True))
    for wanted in (["residual"], ["y"], ["gate"], ["pre_bias"], ["post_weight", "gate"], ["residual", "y"]):
        for k, g in grads(wanted, (True, True)).items():
            assert torch.equal(g, full[k]), (wanted, k)
    only_out, only_n = grads(list(t), (True, False)), grads(list(t), (False, True))
    assert only_out["pre_weight"] is None and torch.equal(only_n["pre_weight"], full["pre_weight"])
    assert torch.allclose(only_out["y"] + only_n["y"], full["y"], rtol=1e-4, atol=1e-4)
    assert torch.equal(only_out["residual"], go)
    with pytest.raises(RuntimeError):                              # a second derivative is refused
        x = t["residual"].detach().requires_grad_()
        (g,) = torch.autograd.grad(sparse.block_norm(x).sum(), x, create_graph=True)
        g.sum().backward()


@pytest.mark.parametrize("cols", [64, 100, 768, 2100])
def test_n_kept_in_8_bits_is_n_encoded(cuda, cols):
    import sparse
    for stream, block in ((F32, F16), (BF16, BF16), (F32, F32)):
        x, y = draw(90, 5, 3, cols, dtype=stream).to(cuda), draw(91, 5, 3, cols, dtype=block).to(cuda)
        out, n, kept = sparse.residual_norm(x, y, pre_kind="rms", checkpoint=True)
        want = sparse.checkpoint_activation(n)
        assert kept.shape == n.shape and kept.dtype == n.dtype
        assert torch.equal(kept.values.view(torch.uint8), want.values.view(torch.uint8)) and torch.equal(kept.scales, want.scales)
        n2, kept2 = sparse.block_norm(x.to(block), checkpoint=True)
        assert torch.equal(kept2.decode(), sparse.checkpoint_activation(n2).decode())


def test_modules(cuda):
    import sparse
    x, y = draw(95, 2, 5, 128).to(cuda).requires_grad_(), draw(96, 2, 5, 128).to(cuda).half().requires_grad_()
    m = sparse.ResidualNorm(128, post="rms", pre="layer", gate=0.25, residual_scale=0.5, device=cuda)
    first = sparse.BlockNorm(128, "rms", out_dtype=F16, device=cuda)
    out, n = m(x, y)
    assert torch.equal(out, sparse.residual_norm(x, y, m.gate, 0.5, post_kind="rms", post_weight=m.post_weight))
    ((out * 0.1).sum() + n.float().square().sum() + first(x).float().sum()).backward()
    assert all(p.grad is not None and p.grad.isfinite().all() for p in [x, y, *m.parameters(), *first.parameters()])
    given = torch.full((2, 1, 128), 2.0, device=cuda)
    assert torch.equal(m(x, y, gate=given)[0], sparse.residual_norm(x, y, given, 0.5, post_kind="rms", post_weight=m.post_weight))


def test_refusals(cuda):
    import sparse
    x, h = torch.zeros(4, 64, device=cuda), torch.zeros(4, 64, device=cuda, dtype=F16)
    w = torch.ones(64, device=cuda)
    for call in (lambda: sparse.residual_norm(x, h[:2]), lambda: sparse.residual_norm(h, x), lambda: sparse.residual_norm(h, h.bfloat16()),
                 lambda: sparse.residual_norm(x, h, pre_kind="batch"), lambda: sparse.residual_norm(x, h, post_weight=w), lambda: sparse.residual_norm(x, h, checkpoint=True),
                 lambda: sparse.residual_norm(x, h, torch.ones(3, 64, device=cuda)), lambda: sparse.residual_norm(x, h, torch.ones(1, 4, 64, device=cuda)),
                 lambda: sparse.residual_norm(x, h, torch.ones(64)), lambda: sparse.residual_norm(x, h, w.long()), lambda: sparse.residual_norm(x, h.to(torch.float8_e4m3fn)),
                 lambda: sparse.block_norm(x, w[:3]), lambda: sparse.block_norm(x, w.cpu()), lambda: sparse.block_norm(x, kind=None),
                 lambda: sparse.block_norm(torch.zeros(2, 16385, device=cuda)), lambda: sparse.block_norm(torch.zeros(2, 0, device=cuda)),
                 lambda: sparse.block_norm(torch.zeros((), device=cuda))):
        with pytest.raises(RuntimeError):
            call()


def test_rows_beyond_32_bits_of_elements(cuda):
    """More than 2^31 elements: the last rows are what they are by themselves, forward and backward, with a gate for every row and without."""
    import sparse
    rows, cols = 262400, 8200
    tail = {k: draw(120 + i, 5, cols, dtype=BF16).to(cuda) for i, k in enumerate(("x", "y", "gate", "go", "gn"))}
    w = draw(130, cols, mean=1.0, dtype=BF16).to(cuda)
    whole = {}
    for k, v in tail.items():
        whole[k] = torch.zeros(rows, cols, dtype=BF16, device=cuda)
        whole[k][-5:] = v
    for gated in (False, True):
        def step(t):
            x, y, g = (t[k].detach().requires_grad_() for k in ("x", "y", "gate"))
            out, n, kept = sparse.residual_norm(x, y, g if gated else None, post_kind="rms", post_weight=w, pre_kind="layer", pre_weight=w, checkpoint=True)
            grads = torch.autograd.grad((out, n), (x, y, g) if gated else (x, y), (t["go"], t["gn"]))
            return [v[-5:].clone() for v in (out.detach(), n.detach(), kept.values.view(torch.uint8), kept.scales, *grads)]
        for a, b in zip(step(whole), step(tail)):
            assert torch.equal(a, b)


def test_two_threads_on_two_streams(cuda):
    """Calls from two threads at once, each on a stream of its own."""
    import threading
    import sparse
    data = [[draw(140 + 5 * i + j, 300, 1000, dtype=BF16).to(cuda) for j in range(4)] for i in range(2)]
    w = draw(150, 1000, mean=1.0, dtype=BF16).to(cuda)

    def step(x, y, go, gn):
        leaves = [t.detach().requires_grad_() for t in (x, y, w)]
        out, n = sparse.residual_norm(leaves[0], leaves[1], post_kind="layer", post_weight=leaves[2], pre_kind="rms", pre_weight=leaves[2])
        return [out.detach(), n.detach(), *torch.autograd.grad((out, n), leaves, (go, gn))]

    want = [step(*d) for d in data]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(20):
                got = step(*data[i])
                stream.synchronize()
                if not all(torch.equal(a, b) for a, b in zip(got, want[i])):
                    wrong.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    assert not wrong and not any(t.is_alive() for t in threads)


def test_other_streams_and_replayed_graphs(cuda):
    """On a side stream, and captured (both passes): every replay gives the bits of the eager call on the inputs of the moment, with eager work between."""
    import sparse
    t = {k: draw(100 + i, *s, dtype=d, mean=0.2).to(cuda) for i, (k, s, d) in enumerate([("residual", (3, 50, 768), F32), ("y", (3, 50, 768), F16), ("gate", (3, 1, 768), F32),
                                                                                           ("post_weight", (768,), F32), ("pre_weight", (768,), F32), ("pre_bias", (768,), F32)])}
    go, gn = draw(110, 3, 50, 768).to(cuda), draw(111, 3, 50, 768, dtype=F16).to(cuda)

    def step():
        leaves = {k: v.detach().requires_grad_() for k, v in t.items()}
        r = dict(leaves)
        out, n, kept = sparse.residual_norm(r.pop("residual"), r.pop("y"), post_kind="rms", pre_kind="layer", checkpoint=True, **r)
        return [out.detach(), n.detach(), kept.decode(), *torch.autograd.grad((out, n), list(leaves.values()), (go, gn))]

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        recorded = step()
    for replay in range(3):
        for k in t:
            t[k].mul_(1.0 + 0.25 * replay)
        want = step()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(recorded, want)), replay


def test_constant_rows_of_large_values(cuda):
    """Rows of one value up to 1e12: their variance is zero, whatever rounding makes of it.  The first mean is off by 64 u |v| at most, the second one
    by 64 u of that, which r = 1 / sqrt(eps) scales."""
    import sparse
    value = 10.0 ** torch.linspace(0, 12, 400, dtype=torch.float64).view(-1, 1)
    for cols in (5, 96, 1000, 1601, 5000):
        x = value.float().expand(-1, cols).contiguous()
        x[::2] *= -1
        w, b = draw(160, cols, mean=1.0), draw(161, cols)
        leaf = x.to(cuda).requires_grad_()
        n = sparse.block_norm(leaf, w.to(cuda), b.to(cuda), kind="layer", eps=1e-5)
        assert n.isfinite().all(), cols
        off = (n.detach().cpu().double() - b.double()).abs()
        assert (off <= ((64 * U) ** 2 * value * 1e-5 ** -0.5 + 1e-6) * w.double().abs() + U * b.double().abs()).all(), cols
        assert torch.autograd.grad(n, leaf, torch.ones_like(n))[0].isfinite().all()


def test_graphs_hooks_and_changes_in_place(cuda):
    import sparse
    from torch.utils.checkpoint import checkpoint
    x, y, w = draw(170, 6, 96).to(cuda).requires_grad_(), draw(171, 6, 96).to(cuda).requires_grad_(), draw(172, 96, mean=1.0).to(cuda).requires_grad_()
    go, gn = draw(173, 6, 96).to(cuda), draw(174, 6, 96).to(cuda)
    call = lambda x, y, w: sparse.residual_norm(x, y, post_kind="rms", post_weight=w, pre_kind="layer", pre_weight=w)  # noqa: E731
    out, n = call(x, y, w)
    want = torch.autograd.grad((out, n), (x, y, w), (go, gn), retain_graph=True)
    same = lambda got: all(torch.equal(a, b) for a, b in zip(got, want))  # noqa: E731
    assert same(torch.autograd.grad((out, n), (x, y, w), (go, gn)))
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad((out, n), (x, y, w), (go, gn))
    # one output alone: as with zeros for the other one
    for one in (0, 1):
        zeros = [go, gn]
        zeros[1 - one] = torch.zeros_like(go)
        a = torch.autograd.grad(call(x, y, w)[one], (x, y, w), (go, gn)[one])
        b = torch.autograd.grad(call(x, y, w), (x, y, w), zeros)
        assert all(torch.allclose(s, t, rtol=1e-5, atol=1e-5) for s, t in zip(a, b))
    # what the backward pass reads may not change
    for i in (0, 1):
        y2 = y.detach().clone().requires_grad_()
        moved = y2 * 1
        out, n = call(x, moved, w)
        with torch.no_grad():
            (out, moved)[i].add_(1)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            torch.autograd.grad(n, w, gn)
    out = sparse.residual_norm(x, y, residual_scale=0.5)           # (reads nothing)
    out.add_(1)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(out, (x, y), go), (0.5 * go, go)))
    # hooks of the saved tensors, the forward pass made again, gradients of the outputs
    with torch.autograd.graph.save_on_cpu():
        out, n = call(x, y, w)
    assert same(torch.autograd.grad((out, n), (x, y, w), (go, gn)))
    for reentrant in (False, True):
        out, n = checkpoint(call, x, y, w, use_reentrant=reentrant)
        for t in (x, y, w):
            t.grad = None
        torch.autograd.backward((out, n), (go, gn))
        assert same((x.grad, y.grad, w.grad))
    out, n = call(x, y, w)
    out.retain_grad()
    n.register_hook(lambda g: 2 * g)
    torch.autograd.backward((out, n), (go, gn / 2))
    assert torch.equal(out.grad, go)
    with torch.inference_mode():
        assert all(torch.equal(a, b) for a, b in zip(call(x, y, w), call(x.detach(), y.detach(), w.detach())))
    out, n = call(x, y, w)
    with pytest.raises(RuntimeError, match="graph of the gradients"):
        torch.autograd.grad(n, x, gn, create_graph=True)


def test_refusals_of_what_is_no_tensor(cuda):
    import sparse
    x = torch.zeros(4, 64, device=cuda)
    for y in (None, 1.0):
        with pytest.raises(RuntimeError, match="residual_norm"):
            sparse.residual_norm(x, y, pre_kind="rms")
        with pytest.raises(RuntimeError, match="residual_norm"):
            sparse.residual_norm(x, y, x, pre_kind="rms")
    with pytest.raises(RuntimeError, match="residual_scale"):
        sparse.residual_norm(x, x, residual_scale=torch.ones((), device=cuda, requires_grad=True))
    assert torch.equal(sparse.residual_norm(x + 1, x, residual_scale=torch.tensor(0.5)), x + 0.5)


@pytest.mark.parametrize("gates,seq", [(130, 48), (300, 31)])
def test_gates_whose_rows_are_cut_into_pieces(cuda, gates, seq):
    from sparse import _native as N
    assert N.lib().tf24_block_norm_backward_workspace_bytes(gates * seq, 1152, seq) > gates * 1152 * 16
    check(cuda, (gates, seq), 1152, BF16, BF16, None, "layer", "sequence", seed=13)


@pytest.mark.parametrize("cols", [8193, 12288, 16383])
@pytest.mark.parametrize("gate", ["channel", "sequence", "token"])
def test_wide_rows(cuda, cols, gate):
    """Rows that have kernels of their own, more of them than workgroups."""
    check(cuda, (3, 171), cols, BF16, BF16, "layer", "rms", gate, seed=14)
    check(cuda, (2, 3), cols, F32, F16, "rms" if gate == "channel" else None, "layer", gate, bias=False, strided=True, seed=15)
