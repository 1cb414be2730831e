"""Activations kept in 8 bits: the format bit by bit against the oracle, the gated activation and the gradients that use it against float64."""
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


# ------------------------------------------------------------------ gradients of weight and bias
def check_weight_gradient(cuda, tokens, m, n, dtype, wide=False, bias=True, lead=None):
    """Sums of float32 products in float32 (an instruction adds 32 of them to its accumulator, pieces are added in order): off by less than
    (tokens / 32 + 48) u of the sum of the magnitudes, then one rounding."""
    import sparse
    x, g = draw(tokens, tokens, n, dtype=dtype), draw(m, tokens, m, dtype=dtype, std=0.1)
    shape = lead or (tokens,)
    kept = sparse.checkpoint_activation(x.to(cuda).view(*shape, n))
    dw, db = sparse.checkpoint_weight_gradient(g.to(cuda).view(*shape, m), kept, bias=bias, dtype=F32 if wide else None)
    out = F32 if wide else dtype
    assert dw.shape == (m, n) and dw.dtype == out and (db is None) == (not bias)
    g64, x64 = g.double().to(cuda), kept.decode().double().view(tokens, n)
    for got, want, size in ((dw, g64.t().contiguous() @ x64, g64.abs().t().contiguous() @ x64.abs()),) + (((db, g64.sum(0), g64.abs().sum(0)),) if bias else ()):
        tolerance = (tokens / 32 + 48) * U * size + torch.finfo(out).eps / 2 * want.abs() * 1.01 + 2.0 ** -25 * (out == F16)
        off = (got.double() - want).abs()
        assert (off <= tolerance).all(), (off / tolerance).max().item()
    again, _ = sparse.checkpoint_weight_gradient(g.to(cuda).view(*shape, m), kept, bias=False, dtype=F32 if wide else None)
    assert torch.equal(again, dw)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("tokens,m,n", [(1, 8, 1), (1, 8, 8), (2, 16, 33), (31, 200, 100), (63, 128, 128), (64, 192, 192), (65, 8, 257), (127, 264, 40), (128, 384, 193),
                                        (129, 136, 384), (300, 512, 512), (1003, 768, 520), (2047, 256, 1000), (5000, 64, 96), (4096, 1024, 1536), (1024, 4096, 4096), (1030, 4104, 4088)])
def test_weight_gradient(cuda, tokens, m, n, dtype):
    check_weight_gradient(cuda, tokens, m, n, dtype)
    check_weight_gradient(cuda, tokens, m, n, dtype, wide=True, bias=False)


@pytest.mark.parametrize("m", [1, 7, 100, 1001])
def test_weight_gradient_of_any_number_of_outputs(cuda, m):
    check_weight_gradient(cuda, 77, m, 130, BF16, lead=(7, 11))


def test_weight_gradient_of_strided_gradients(cuda):
    import sparse
    x, g = draw(1, 90, 200, dtype=BF16).to(cuda), draw(2, 90, 64, dtype=BF16).to(cuda)
    kept = sparse.checkpoint_activation(x)
    want, want_b = sparse.checkpoint_weight_gradient(g, kept, bias=True)
    wide = torch.full((90, 80), float("nan"), dtype=BF16, device=cuda)
    odd = torch.full((90, 69), float("nan"), dtype=BF16, device=cuda)
    wide[:, 8:72], odd[:, 3:67] = g, g
    for view in (wide[:, 8:72], odd[:, 3:67], g.t().contiguous().t(), torch._neg_view(-g)):
        dw, db = sparse.checkpoint_weight_gradient(view, kept, bias=True)
        assert torch.equal(dw, want) and torch.equal(db, want_b)
    ones, one = torch.ones((), dtype=BF16, device=cuda).expand(90, 64), torch.ones(90, 64, dtype=BF16, device=cuda)
    assert torch.equal(sparse.checkpoint_weight_gradient(ones, kept)[0], sparse.checkpoint_weight_gradient(one, kept)[0])
    empty = sparse.checkpoint_weight_gradient(g[:0], sparse.checkpoint_activation(x[:0]), bias=True)
    assert empty[0].shape == (64, 200) and empty[1].shape == (64,) and not empty[0].any() and not empty[1].any()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("tokens,m,n", [(64, 192, 192), (333, 264, 200), (1100, 128, 640)])
def test_weight_gradient_of_integers_is_exact(cuda, tokens, m, n, dtype):
    """Sums of products of small integers are exact in float32, in any order; each operand's rows and columns are its own, a row of one token shows
    where it goes; infinities and NaNs stay in their rows and columns."""
    import sparse
    gen = torch.Generator().manual_seed(tokens)
    x, g = (torch.randint(-4, 5, (tokens, c), generator=gen).to(dtype) for c in (n, m))
    kept = sparse.checkpoint_activation(x.to(cuda))
    assert torch.equal(kept.decode().cpu(), x)
    dw, db = sparse.checkpoint_weight_gradient(g.to(cuda), kept, bias=True, dtype=F32)
    assert torch.equal(dw.cpu().double(), g.double().t() @ x.double()) and torch.equal(db.cpu().double(), g.double().sum(0))
    x[tokens - 1, 5], g[0, 3] = float("nan"), float("inf")
    dw, db = sparse.checkpoint_weight_gradient(g.to(cuda), sparse.checkpoint_activation(x.to(cuda)), bias=True, dtype=F32)
    want = g.double().t() @ x.double()
    assert torch.equal(dw.cpu().isfinite(), want.isfinite()) and torch.equal(dw.cpu().double()[want.isfinite()], want[want.isfinite()])
    assert torch.equal(db.cpu().isfinite(), g.double().sum(0).isfinite())


def test_weight_gradient_at_every_scale(cuda):
    """Blocks of magnitudes from the smallest to the largest that a type holds, one token each: the gradient is that row."""
    import sparse
    for dtype, low, high in ((F16, -24, 15), (BF16, -126, 126)):
        exponents = torch.arange(low, high + 1)
        x = (torch.linspace(1, 1.9, 64, dtype=torch.float64)[None] * 2.0 ** exponents.double()[:, None]).to(dtype)
        g = torch.zeros(len(x), (len(x) + 7) // 8 * 8, dtype=dtype)
        g[torch.arange(len(x)), torch.arange(len(x))] = 1
        kept = sparse.checkpoint_activation(x.to(cuda))
        dw, _ = sparse.checkpoint_weight_gradient(g.to(cuda), kept, dtype=F32)
        want = kept.decode(F32)
        if dtype == BF16:                                          # (matrix instructions flush what float32 holds as subnormal)
            want = torch.where(want.abs() < 2.0 ** -126, 0, want)
        assert torch.equal(dw[:len(x)], want), dtype


@pytest.mark.parametrize("tokens,m,n", [(3000, 200, 160), (1000, 4096, 4096)])
def test_weight_gradient_without_a_workspace(cuda, tokens, m, n):
    """Through the C ABI with less scratch than the cut into pieces asks for, and none: fewer pieces, the same sums (of integers)."""
    import sparse
    from sparse import _native as N
    gen = torch.Generator().manual_seed(4)
    x, g = (torch.randint(-4, 5, (tokens, c), generator=gen).to(F16).to(cuda) for c in (n, m))
    kept = sparse.checkpoint_activation(x)
    full = N.lib().tf24_checkpoint_weight_grad_workspace_bytes(tokens, m, n)
    assert full > 0
    want = (g.double().t().contiguous() @ x.double()).float()
    for nbytes in (full, full // 2, 1000, 0):
        dw, db = torch.empty(m, n, device=cuda), torch.empty(m, device=cuda)
        ws = torch.full((max(nbytes, 1),), 255, dtype=torch.uint8, device=cuda)
        N.check(N.lib().tf24_checkpoint_weight_grad(g.data_ptr(), m, N.F16, kept.values.data_ptr(), kept.scales.data_ptr(), tokens, m, n, dw.data_ptr(), db.data_ptr(), N.F32,
                                                    ws.data_ptr() if nbytes else None, nbytes, N.stream_ptr()))
        assert torch.equal(dw, want) and torch.equal(db.double(), g.double().sum(0)), nbytes


def test_refusals(cuda):
    import sparse
    g = torch.zeros(4, 8, device=cuda, dtype=F16)
    for call in (lambda: sparse.checkpoint_activation(torch.zeros(4, 8, device=cuda, dtype=torch.int32)), lambda: sparse.checkpoint_activation(torch.zeros((), device=cuda)),
                 lambda: sparse.checkpoint_activation(torch.zeros(4, 0, device=cuda)), lambda: sparse.gelu_glu_checkpoint.apply(torch.zeros(4, 7, device=cuda)),
                 lambda: sparse.gelu_glu_checkpoint.apply(torch.zeros(4, 8, device=cuda, dtype=torch.float64)),
                 lambda: sparse.checkpoint_activation(torch.zeros(4, 8, device=cuda)).decode(torch.float64),
                 lambda: sparse.checkpoint_weight_gradient(g, sparse.checkpoint_activation(g[:3])), lambda: sparse.checkpoint_weight_gradient(g.bfloat16(), sparse.checkpoint_activation(g)),
                 lambda: sparse.checkpoint_weight_gradient(g.float(), sparse.checkpoint_activation(g.float())), lambda: sparse.checkpoint_weight_gradient(g[:, :0], sparse.checkpoint_activation(g)),
                 lambda: sparse.checkpoint_weight_gradient(g.cpu(), sparse.checkpoint_activation(g)),
                 lambda: sparse.checkpoint_weight_gradient(g, sparse.checkpoint_activation(g), dtype=BF16)):
        with pytest.raises(RuntimeError):
            call()
    leaf = torch.randn(2, 2, 8, device=cuda, requires_grad=True)
    with pytest.raises(RuntimeError):                              # a second derivative is refused
        (g,) = torch.autograd.grad(sparse.gelu_glu_checkpoint.apply(leaf).sum(), leaf, create_graph=True)
        g.sum().backward()


def test_captured_and_on_another_stream(cuda):
    import sparse
    x, dy = draw(7, 3, 400, 512, dtype=BF16).to(cuda), draw(8, 3, 400, 256, dtype=BF16).to(cuda)

    def step():
        leaf = x.detach().requires_grad_()
        out, kept = sparse.GELUglu(True, True)(leaf)
        return [out.detach(), kept.decode(), sparse.checkpoint_activation(x).decode(), torch.autograd.grad(out, leaf, dy)[0],
                *sparse.checkpoint_weight_gradient(dy, sparse.checkpoint_activation(x), bias=True)]

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


def test_a_checkpoint_that_was_changed_is_refused(cuda):
    """Before anything reads past what is kept."""
    import sparse
    x, g = draw(90, 6, 64).half().to(cuda), draw(91, 6, 32).half().to(cuda)
    for name, value in (("shape", torch.Size((7, 64))), ("shape", torch.Size((6, 96))), ("shape", torch.Size(())), ("scales", torch.zeros(6, 1, dtype=torch.uint8, device=cuda)),
                        ("values", torch.zeros(5, 64, device=cuda).to(torch.float8_e4m3fn)), ("values", torch.zeros(6, 64, device=cuda)), ("scales", torch.zeros(6, 2, dtype=torch.uint8))):
        kept = sparse.checkpoint_activation(x)
        setattr(kept, name, value)
        with pytest.raises(RuntimeError):
            kept.decode()
        with pytest.raises(RuntimeError):
            sparse.checkpoint_weight_gradient(g, kept)
