"""residual_norm / block_norm and their gradients at the ends of what they take: rows of one very large value, gates of 16 bits that broadcast, very many gates."""
import pytest
import torch

import oracle
from test_gpu_block_norm import check

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


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("cols", [8, 36, 50, 768, 1601, 5000, 8193, 12288])
def test_gradients_of_rows_of_one_very_large_value(cuda, cols, dtype):
    """2^110 in every column, eps 1e-12: the mean is exact (partial sums are small integers times 2^110, and cols times the float32 1 / cols rounds to 1), the
    variance 0, r = 1e6, and |mean| r is over float32's largest number.  With q = dn w the gradient is dout + r (q - mean q), nothing of which comes near that.
    The mean of q is off by 40 u of its terms' mean magnitude, q, r, the difference and the last addition by a few u each: 64 u of all of them, and
    one rounding to the type.  Weight gradients are 0: every normed value is."""
    import sparse
    eps, rows = 1e-12, 3
    large = torch.full((rows, cols), 2.0 ** 110, dtype=dtype)
    large[1] *= -1
    w, b = draw(1, cols, mean=1.0, dtype=dtype), draw(2, cols, dtype=dtype)
    dout, dn = draw(3, rows, cols, dtype=dtype), draw(4, rows, cols, dtype=dtype)
    r = eps ** -0.5

    def expected(dn, w, add):
        q = dn.double() * w.double()
        return r * (q - q.mean(-1, keepdim=True)) + add, r * (q.abs() + q.abs().mean(-1, keepdim=True)) + abs(add)

    def close(name, got, want, magnitude):
        tolerance = 64 * U * magnitude + torch.finfo(got.dtype).eps / 2 * want.abs() * 1.01
        off = (got.cpu().double() - want).abs()
        assert (off <= tolerance).all(), (name, cols, got.isnan().sum().item(), (off / tolerance).max().item())

    def leaves(*ts):
        return [t.to(cuda).requires_grad_() for t in ts]

    # before a block: by itself, and behind the addition
    x, w1, b1 = leaves(large, w, b)
    n = sparse.block_norm(x, w1, b1, eps=eps)
    assert torch.equal(n.detach().cpu(), b.expand(rows, cols))
    dx, dw, db = torch.autograd.grad(n, (x, w1, b1), dn.to(cuda))
    close("x", dx, *expected(dn, w, 0.0))
    close("bias", db, dn.double().sum(0), dn.double().abs().sum(0))
    assert not dw.any()
    x, y, w1, b1 = leaves(large, torch.zeros_like(large), w, b)
    out, n = sparse.residual_norm(x, y, pre_kind="layer", pre_weight=w1, pre_bias=b1, eps=eps)
    assert torch.equal(out.detach().cpu(), large)
    dx, dy, dw = torch.autograd.grad((out, n), (x, y, w1), (dout.to(cuda), dn.to(cuda)))
    close("residual", dx, *expected(dn, w, dout.double()))
    assert torch.equal(dx, dy) and not dw.any()
    # behind a block
    for gate in (None, torch.full((cols,), 0.5, dtype=dtype), torch.full((rows, cols), 0.5, dtype=dtype)):
        x, y, w1, b1 = leaves(draw(5, rows, cols, dtype=dtype), large, w, b)
        g = None if gate is None else gate.to(cuda)
        out = sparse.residual_norm(x, y, g, post_kind="layer", post_weight=w1, post_bias=b1, eps=eps)
        dx, dy, dw, db = torch.autograd.grad(out, (x, y, w1, b1), dout.to(cuda))
        of_z = dout.double() * (1.0 if gate is None else 0.5)
        assert torch.equal(dx.cpu(), dout) and not dw.any()
        close("y", dy, *expected(of_z, w, 0.0))
        close("post_bias", db, of_z.sum(0), of_z.abs().sum(0))


@pytest.mark.parametrize("stream", [F16, BF16])
@pytest.mark.parametrize("shape", [(), (1,), (1, 1, 1), (6, 1, 1), (1, 40, 512), (6, 40, 1), (40, 512), (1, 512), (6, 1, 512)])
def test_gates_of_16_bits_that_broadcast(cuda, shape, stream):
    """The gradient of a gate is rounded once, whatever rows and columns share it: 256 u of the sum of the magnitudes and one rounding to its type, as
    for a gate of float32."""
    check(cuda, (6, 40), 512, stream, stream, "rms", "rms", "given", gate_shape=shape, seed=9)
    check(cuda, (6, 40), 512, stream, stream, None, "layer", "given", gate_shape=shape, seed=19)


class Given:
    """Saved-tensor hooks that hand back something else than they were given: change(tensor) for tensors of `numel` elements."""

    def __init__(self, change, numel):
        self.hooks = torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: change(t) if t.numel() == numel else t)

    def __enter__(self):
        return self.hooks.__enter__()

    def __exit__(self, *args):
        return self.hooks.__exit__(*args)


def apart(t):
    """The same values, a row not next to the one before it."""
    wide = torch.full((*t.shape[:-1], t.shape[-1] + 7), 3, device=t.device).to(t.dtype)
    wide[..., :t.shape[-1]] = t
    return wide[..., :t.shape[-1]]


CHANGES = [lambda t: t.cpu(), lambda t: t[:1], lambda t: t.to(torch.float64), lambda t: t.flatten()[:1].expand(1)]


def test_saved_tensors_that_hooks_hand_back(cuda):
    """Values that lie elsewhere are taken; another shape, type or place is refused, before a kernel reads it."""
    import sparse
    rows, cols = 6, 96
    x, y, gate = (draw(i, rows, cols).to(cuda).requires_grad_() for i in (20, 21, 22))
    w = draw(23, cols, mean=1.0).to(cuda).requires_grad_()
    go, gn = draw(24, rows, cols).to(cuda), draw(25, rows, cols).to(cuda)

    def call():
        return sparse.residual_norm(x, y, gate, post_kind="rms", post_weight=w, pre_kind="layer", pre_weight=w)

    want = torch.autograd.grad(call(), (x, y, gate, w), (go, gn))
    for numel in (rows * cols, cols, 4 * rows):                    # rows; weights; statistics
        with Given(apart, numel):
            outputs = call()
        assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(outputs, (x, y, gate, w), (go, gn)), want))
        for change in CHANGES:
            with Given(change, numel):
                outputs = call()
            with pytest.raises(RuntimeError, match="saved"):
                torch.autograd.grad(outputs, (x, y, gate, w), (go, gn))
    from sparse import _native as N
    if N.torch_calls() is not None:                                # nodes that are called by themselves, past the engine's checks
        node = call()[1].grad_fn
        with torch.no_grad():
            for grads in ((go[:1], gn), (go, gn[:, :32]), (go.cpu(), gn.cpu()), (go,), ()):
                with pytest.raises((RuntimeError, TypeError), match="gradient|arguments"):       # (torch counts them)
                    node(*grads)
            assert all(torch.equal(a, b) for a, b in zip(node(go, gn), want[:3]))


def test_saved_tensors_of_the_gated_activation_that_hooks_hand_back(cuda):
    import sparse
    rows, half = 6, 96
    x, dy = draw(26, rows, 2 * half).to(cuda).requires_grad_(), draw(27, rows, half).to(cuda)
    (want,) = torch.autograd.grad(sparse.gelu_glu_checkpoint.apply(x), x, dy)
    for numel in (2 * rows * half, 2 * rows * half // 32):         # values; scales
        with Given(lambda t: apart(t.view(torch.uint8)).view(t.dtype), numel):
            out = sparse.gelu_glu_checkpoint.apply(x)
        assert torch.equal(torch.autograd.grad(out, x, dy)[0], want)
        for change in CHANGES[:2] + [lambda t: t.view(torch.int8)]:
            with Given(change, numel):
                out = sparse.gelu_glu_checkpoint.apply(x)
            with pytest.raises(RuntimeError, match="saved"):
                torch.autograd.grad(out, x, dy)


def test_sums_over_very_many_gates(cuda):
    """2^20 gates of two rows: the sums over the gates' pieces are as exact as those over few.  A sum of `count` equal terms c is count c to 256 u; in float32 in sequence
    2^15 of them in each of 32 strands would be off by 4341 u for c = 0.2."""
    import sparse
    gates, cols = 1 << 20, 8
    x, y = torch.zeros(gates, 2, cols, device=cuda, requires_grad=True), torch.ones(gates, 2, cols, device=cuda, requires_grad=True)
    gate = torch.full((gates, 1, cols), 0.1, device=cuda, requires_grad=True)
    w, b, pw, pb = (torch.full((cols,), v, device=cuda, requires_grad=True) for v in (1.0, 0.0, 1.0, 0.0))
    out, n = sparse.residual_norm(x, y, gate, post_kind="rms", post_weight=pw, post_bias=pb, pre_kind="rms", pre_weight=w, pre_bias=b, eps=0.0)
    go, gn = torch.full_like(out, 0.3), torch.full_like(n, 0.1)
    dg, dw, db, dpw, dpb = torch.autograd.grad((out, n), (gate, w, b, pw, pb), (go, gn))
    # y = 1, normed 1; out = 0.1, normed 1: no gradient passes the second norm, d = go
    c, g, s, count = (torch.tensor(v, dtype=F32).double().item() for v in (0.1, 0.1, 0.3, 2.0 * gates))
    for got, want in ((dw, count * c), (db, count * c), (dpw, count * g * s), (dpb, count * g * s)):
        assert (got.cpu().double() - want).abs().max() <= 256 * U * want, ((got.cpu().double() - want).abs().max() / want / U).item()
    assert (dg.cpu().double() - 2 * s).abs().max() <= 64 * U * 2 * s
