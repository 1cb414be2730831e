"""Activations kept in 8 bits: the format bit by bit against the oracle, the gated activation and the gradients that use it against float64."""
import pytest
import torch

import oracle

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
U = 2.0 ** -24


def draw(seed, *shape, dtype=F32, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g, dtype=torch.float64) * std * torch.exp(0.7 * torch.randn(shape[-1], generator=g, dtype=torch.float64))).to(dtype)


def same(got, want):
    got = got.detach().cpu().double()
    return got.shape == want.shape and torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(), want.nan_to_num())


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 32), (3, 7), (5, 33), (2, 64), (37, 100), (70, 768)])
def test_values_and_scales(cuda, rows, cols, dtype):
    import sparse
    x = draw(rows + cols, rows, cols, dtype=dtype)
    kept = sparse.checkpoint_activation(x.to(cuda))
    want = oracle.kept(x)
    blocks = (cols + 31) // 32
    assert kept.values.shape == (rows, 32 * blocks) and kept.scales.shape == (rows, blocks) and kept.nbytes == rows * blocks * 33
    assert kept.decode().dtype == dtype and same(kept.decode(), want)
    exponents = torch.tensor([[oracle.kept_scale(x[r, 32 * b:32 * b + 32]) for b in range(blocks)] for r in range(rows)])
    assert torch.equal(kept.scales.cpu().int() - 127, exponents.int())
    assert not kept.values.view(torch.uint8).cpu()[:, cols:].any()
    units = torch.ldexp(torch.ones(rows, blocks, dtype=torch.float64), exponents).repeat_interleave(32, 1)
    assert torch.equal((kept.values.cpu().double() * units)[:, :cols], want)
    for other in (F32, F16, BF16):
        assert torch.equal(kept.decode(other).cpu(), want.to(other)), other


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_values_at_every_edge(cuda, dtype):
    """Ties, the largest numbers, subnormal ones, zeros of either sign, infinities and NaNs, blocks without a finite number."""
    import sparse
    top = torch.finfo(dtype).max
    x = torch.zeros(12, 64, dtype=dtype)
    x[0, :16] = torch.arange(16) * 0.0625 + 1.0                     # ties of 4 bits of mantissa
    x[0, 16] = 1.75
    x[1, :16] = torch.arange(16) * 0.0625 + 1.0
    x[1, 16] = 1.8
    x[2, 0], x[2, 1], x[2, 2] = top, -top, top * 0.9375
    x[2, 33] = top
    x[3, :8] = torch.tensor([torch.finfo(dtype).smallest_normal, torch.finfo(dtype).tiny / 2, -torch.finfo(dtype).tiny / 4, 0, 0, 0, 0, 0]).to(dtype)
    x[4, 3], x[4, 4], x[4, 5] = float("inf"), 2.5, -float("inf")
    x[5, 0], x[5, 1] = float("nan"), -1.0
    x[5, 32:] = float("nan")
    x[6, 31], x[6, 32] = 100.0, 0.01
    x[7] = -0.0
    x[8, :32] = torch.logspace(-12, 0, 32).to(dtype)
    x[9, :32] = (448.0 * torch.logspace(-5, 0, 32)).to(dtype)
    if dtype != F16:
        x[10] = (torch.linspace(1, 2, 64) * 2.0 ** -120).to(dtype)
        x[11] = (torch.linspace(1, 2, 64) * 2.0 ** -110).to(dtype)
    kept = sparse.checkpoint_activation(x.to(cuda))
    assert same(kept.decode(), oracle.kept(x))
    assert kept.decode()[2].isfinite().all()
    assert torch.equal(torch.signbit(kept.decode()[7]).cpu(), torch.signbit(x[7]))


def test_every_16_bit_number(cuda):
    """All float16 and bfloat16 patterns, each alone in its block but for 1.0 (so that every magnitude meets a scale that it does not set), and alone."""
    import sparse
    every = torch.arange(-32768, 32768, dtype=torch.int32).to(torch.int16)
    for dtype in (F16, BF16):
        x = torch.zeros(65536, 32, dtype=dtype)
        x[:, 7] = every.view(dtype)
        for other in (0.0, 1.0):
            x[:, 20] = other
            got = sparse.checkpoint_activation(x.to(cuda)).decode().cpu()
            finite = x[:, 7].isfinite()
            assert torch.equal(got[finite].double(), oracle.kept_fast(x[finite])), (dtype, other)
            assert got[~finite, 7].isnan().all() and torch.equal(got[~finite, 20], x[~finite, 20])


@pytest.mark.parametrize("dtype", [F16, F32])
def test_strides_shapes_and_views(cuda, dtype):
    import sparse
    x = draw(3, 6, 5, 90, dtype=dtype).to(cuda)
    for view in (x[:, ::2], x[..., 1:78], x[..., ::3], x.transpose(0, 1), x.transpose(1, 2), x[0, 0], x[:1, :1].expand(4, 3, 90), x[:0], torch._neg_view(x)):
        got = sparse.checkpoint_activation(view)
        assert got.shape == view.shape
        assert same(got.decode().reshape(-1, view.shape[-1]), oracle.kept(view.cpu().resolve_neg().reshape(-1, view.shape[-1])))


def test_rows_beyond_32_bits_of_elements(cuda):
    """A matrix of more than 2^32 bytes and 2^31 elements: its last rows are its own."""
    import sparse
    rows, cols = 262200, 8200
    x = torch.zeros(rows, cols, dtype=F16, device=cuda)
    tail = draw(4, 3, cols, dtype=F16)
    x[-3:] = tail.to(cuda)
    kept = sparse.checkpoint_activation(x)
    out = kept.decode()
    assert same(out[-3:], oracle.kept_fast(tail)) and not out[:4].any() and not out[-200:-3].any()


# ------------------------------------------------------------------ the gated activation
def _glu_forward(x, gate):
    """The logistic form: 0.5 (1 + tanh u) loses everything below 2^-53 to its sum, for gates under -5 more than a float32 result holds."""
    return x * gate * torch.sigmoid(2 * 0.7978845608028654 * (gate + 0.044715 * gate ** 3))


def _glu_tolerance(x, gate, value, dtype, slope=False):
    """exp2, rcp and the polynomial: 16 u and 4 u of the exponent; the slope's terms add up in magnitude.  A logistic under float32's smallest
    normal number, 2^-126, is 0 (the reciprocal gives no subnormal ones), which is off by less than that times its factors: |x gate|, in
    the slope |x| (1 + |gate| (1 + 0.2 gate^2))."""
    power = 2 * 0.7978845608 * (gate.abs() + 0.044715 * gate.abs() ** 3)
    size = (1 + gate.abs() * (1 + 0.2 * gate * gate)) * x.abs() if slope else value.abs()
    factors = size if slope else (x * gate).abs()
    return U * (32 + 8 * power) * size + 2.0 ** -126 * factors + torch.finfo(dtype).eps / 2 * value.abs() * 1.01 + 2.0 ** -25 * (dtype == F16) + 1e-40


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("lead,half", [((1, 1), 1), ((2, 3), 7), ((1, 5), 32), ((3, 4), 33), ((2, 9), 200), ((7,), 1024), ((2, 3), 2049)])
def test_gated_activation(cuda, lead, half, dtype):
    import sparse
    x, dy = draw(half, *lead, 2 * half, dtype=dtype), draw(half + 1, *lead, half, dtype=dtype, std=0.1)
    leaf = x.to(cuda).requires_grad_()
    out, kept = sparse.GELUglu(checkpoint=True, output_checkpoint=True)(leaf)
    plain = sparse.gelu_glu_checkpoint.apply(leaf)
    assert torch.equal(out, plain) and torch.equal(kept.decode(), sparse.checkpoint_activation(out).decode())
    if len(lead) == 2:
        assert torch.equal(out, sparse.GELUglu()(leaf))             # the output is the one without a checkpoint
    rows = torch.Size(lead).numel()
    x64, gate64 = x.double().reshape(rows, 2, half).unbind(1)
    want = _glu_forward(x64, gate64)
    assert ((out.detach().cpu().double().reshape(rows, half) - want).abs() <= _glu_tolerance(x64, gate64, want, dtype)).all()
    for o in (out, plain):
        (dx,) = torch.autograd.grad(o, leaf, dy.to(cuda))
        kx, kg = (oracle.kept(t.contiguous()) for t in x.reshape(rows, 2, half).unbind(1))
        kx, kg = kx.requires_grad_(), kg.requires_grad_()
        want = torch.autograd.grad(_glu_forward(kx, kg), (kx, kg), dy.double().reshape(rows, half))
        got, go, kx, kg = dx.cpu().double().reshape(rows, 2, half), dy.double().reshape(rows, half), kx.detach(), kg.detach()
        assert ((got[:, 0] - want[0]).abs() <= _glu_tolerance(go, kg, want[0], dtype)).all()
        assert ((got[:, 1] - want[1]).abs() <= _glu_tolerance(go * kx, kg, want[1], dtype, slope=True)).all()


def test_gated_activation_of_views_and_empty_tensors(cuda):
    import sparse
    x = draw(5, 4, 6, 96, dtype=F16).to(cuda)
    dy = draw(6, 4, 6, 48, dtype=F16).to(cuda)
    want_in = x.clone().requires_grad_()
    want = sparse.gelu_glu_checkpoint.apply(want_in)
    (want_dx,) = torch.autograd.grad(want, want_in, dy)
    wide = torch.zeros(4, 6, 101, dtype=F16, device=cuda)
    wide[..., 2:98] = x
    for view, grad in ((wide[..., 2:98], dy), (x.transpose(1, 2).contiguous().transpose(1, 2), dy.transpose(0, 2).contiguous().transpose(0, 2)), (x, torch._neg_view(-dy))):
        leaf = view.detach().requires_grad_()
        out = sparse.gelu_glu_checkpoint.apply(leaf)
        assert torch.equal(out, want)
        assert torch.equal(torch.autograd.grad(out, leaf, grad)[0], want_dx)
    one = x[:1, :1].expand(3, 5, 96).detach().requires_grad_()     # rows that are one row in memory
    assert torch.equal(torch.autograd.grad(sparse.gelu_glu_checkpoint.apply(one).sum(), one)[0][2, 4],
                       torch.autograd.grad(sparse.gelu_glu_checkpoint.apply(want_in).sum(), want_in)[0][0, 0])
    none = x[:0].detach().requires_grad_()
    out, kept = sparse.GELUglu(True, True)(none)
    assert out.shape == (0, 6, 48) and kept.decode().shape == out.shape and torch.autograd.grad(out.sum(), none)[0].shape == none.shape


def test_gated_activation_keeps_the_signs_of_trouble(cuda):
    import sparse
    x = torch.ones(1, 1, 128, dtype=F16, device=cuda)
    x[0, 0, 3], x[0, 0, 70] = float("inf"), float("nan")
    leaf = x.requires_grad_()
    (dx,) = torch.autograd.grad(sparse.gelu_glu_checkpoint.apply(leaf).sum(), leaf)
    bad = dx[0, 0].isnan().nonzero().flatten().tolist()
    assert bad == [6, 67, 70]      # the gate's slope at x = inf, and both gradients where the gate is a NaN


def test_refusals(cuda):
    import sparse
    for call in (lambda: sparse.checkpoint_activation(torch.zeros(4, 8, device=cuda, dtype=torch.int32)), lambda: sparse.checkpoint_activation(torch.zeros((), device=cuda)),
                 lambda: sparse.checkpoint_activation(torch.zeros(4, 0, device=cuda)), lambda: sparse.gelu_glu_checkpoint.apply(torch.zeros(4, 7, device=cuda)),
                 lambda: sparse.gelu_glu_checkpoint.apply(torch.zeros(4, 8, device=cuda, dtype=torch.float64)),
                 lambda: sparse.checkpoint_activation(torch.zeros(4, 8, device=cuda)).decode(torch.float64)):
        with pytest.raises(RuntimeError):
            call()
    leaf = torch.randn(2, 2, 8, device=cuda, requires_grad=True)
    with pytest.raises(RuntimeError):                              # a second derivative is refused
        (g,) = torch.autograd.grad(sparse.gelu_glu_checkpoint.apply(leaf).sum(), leaf, create_graph=True)
        g.sum().backward()


def test_captured_and_on_another_stream(cuda):
    import sparse
    x, dy = draw(7, 3, 40, 512, dtype=BF16).to(cuda), draw(8, 3, 40, 256, dtype=BF16).to(cuda)

    def step():
        leaf = x.detach().requires_grad_()
        out, kept = sparse.GELUglu(True, True)(leaf)
        return [out.detach(), kept.decode(), sparse.checkpoint_activation(x).decode(), torch.autograd.grad(out, leaf, dy)[0]]

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
        x.mul_(1.0 + 0.5 * replay)
        want = step()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(recorded, want)), replay
