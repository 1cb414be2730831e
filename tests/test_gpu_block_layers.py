"""The layers with their inputs kept in 8 bits, and a whole block of a transformer's MLP: norm, layer, gated activation, layer, gate and residual, next norm."""
import copy

import pytest
import torch
from torch import nn

import oracle

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


@pytest.fixture(autouse=True, params=["torchcall", "python"])
def calls(request, monkeypatch):
    """Everything twice: with the module that makes ordinary calls from torch's C++ side, and with Python making all of them."""
    from sparse import _native as N
    if request.param == "python":
        monkeypatch.setattr(N, "_calls", None)
    elif N.torch_calls() is None:
        pytest.skip("_torchcall is not built for this torch")



def draw(seed, *shape, dtype=F32, std=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * std).to(dtype)


def soft_layer(cuda, d_in, d_out, seed, bias=True, **kw):
    import sparse
    layer = sparse.SoftThresholdLinear(d_in, d_out, bias=bias, device=cuda, **kw)
    with torch.no_grad():
        layer.weight.copy_(draw(seed, d_out, d_in, std=0.05))
        if bias:
            layer.bias.copy_(draw(seed + 1, d_out, std=0.1))
    layer.init_scale()
    return layer


def sparse_layer(cuda, d_in, d_out, seed, **kw):
    import sparse
    layer = sparse.SparseLinearTranspose(d_in, d_out, device=cuda, **kw)
    with torch.no_grad():
        layer.weight.copy_(draw(seed, d_out, d_in, std=0.05))
        layer.bias.copy_(draw(seed + 1, d_out, std=0.1))
    return layer


def step(layer, x, dy, dtype, **kw):
    leaf = x.detach().requires_grad_()
    torch.manual_seed(11)                                          # (MVUE24 draws from torch's generator)
    with torch.autocast("cuda", dtype=dtype):
        out = layer(leaf, **kw)
    params = [p for p in layer.parameters() if p.requires_grad]
    return out.detach(), dict(zip(["x", "weight", "bias"], torch.autograd.grad(out, [leaf, *params], dy)))


@pytest.mark.parametrize("bias", [True, False])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("lead,d_in,d_out", [((2, 150), 256, 512), ((64,), 128, 64), ((3, 700), 768, 2304), ((5,), 40, 24)])
def test_soft_threshold_layer(cuda, lead, d_in, d_out, dtype, bias):
    """Output and input gradient are those of the layer without; the weight's and the bias's are checkpoint_weight_gradient's, float32."""
    import sparse
    layer = soft_layer(cuda, d_in, d_out, 1, bias, checkpoint=True)
    plain = copy.deepcopy(layer)
    plain.checkpoint = False
    x, dy = draw(3, *lead, d_in).to(cuda), draw(4, *lead, d_out, std=0.01, dtype=dtype).to(cuda)
    out, grads = step(layer, x, dy, dtype)
    want_out, want = step(plain, x, dy, dtype)
    assert torch.equal(out, want_out) and torch.equal(grads["x"], want["x"])
    kept = sparse.checkpoint_activation(x.to(dtype))
    dw, db = sparse.checkpoint_weight_gradient(dy, kept, bias=bias, dtype=F32)
    assert torch.equal(grads["weight"], dw) and (not bias or torch.equal(grads["bias"], db))
    # (what the layer without keeps in 16 bits gives, to the rounding of x: 2^-4 of each of its elements, 2^-5 in the mean of many)
    assert (grads["weight"] - want["weight"]).norm() < 2.0 ** -4.5 * want["weight"].norm()
    for given in (step(layer, x, dy, dtype, checkpoint=kept), step(plain, x, dy, dtype, checkpoint=kept)):
        assert torch.equal(given[0], out) and all(torch.equal(given[1][k], grads[k]) for k in grads)


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("lead,d_in,d_out", [((2, 64), 256, 512), ((128,), 768, 768)])
def test_sparse_layer(cuda, lead, d_in, d_out, dtype):
    """The weight's gradient is the one of the layer without that is given the kept values; everything else is as without."""
    import sparse
    layer, plain = sparse_layer(cuda, d_in, d_out, 5, checkpoint=True), sparse_layer(cuda, d_in, d_out, 5)
    x, dy = draw(6, *lead, d_in, dtype=dtype).to(cuda), draw(7, *lead, d_out, std=0.1, dtype=F16).to(cuda)
    out, grads = step(layer, x, dy, F16)
    want_out, want = step(plain, x, dy, F16)
    kept = sparse.checkpoint_activation(x.half())
    _, of_kept = step(plain, kept.decode(), dy, F16)
    assert torch.equal(out, want_out) and torch.equal(grads["x"], want["x"]) and torch.equal(grads["bias"], want["bias"])
    assert torch.equal(grads["weight"], of_kept["weight"]) and not torch.equal(grads["weight"], want["weight"])
    given = step(plain, x, dy, F16, checkpoint=kept)
    assert torch.equal(given[0], out) and all(torch.equal(given[1][k], grads[k]) for k in grads)


def test_ordinary_calls_are_made_from_the_c_side(cuda, calls):
    """With the module, and where it is built for this torch it is there: graphs of its nodes; what it does not take is Python's, with the same result."""
    import sparse
    from sparse import _native as N
    module = N.torch_calls()
    x, y, w = draw(1, 3, 4, 64).to(cuda).requires_grad_(), draw(2, 3, 4, 64, dtype=F16).to(cuda).requires_grad_(), torch.ones(64, device=cuda, requires_grad=True)
    out, n = sparse.residual_norm(x, y, pre_kind="rms", pre_weight=w)
    strided = sparse.residual_norm(x.transpose(0, 1).contiguous().transpose(0, 1), y, pre_kind="rms", pre_weight=w)
    assert torch.equal(out, strided[0]) and torch.equal(n, strided[1])
    names = [t.grad_fn.name() for t in (out, n, strided[0], sparse.block_norm(x), sparse.gelu_glu_checkpoint.apply(x), sparse.gelu_glu_checkpoint.apply(x[..., 1:63]))]
    if module is None:
        assert not any(name in ("BlockNormBackward", "GeluGluBackward") for name in names)
    else:
        assert names[0] == names[1] == names[3] == "BlockNormBackward" != names[2] and names[4] == "GeluGluBackward" != names[5]
        assert module.checkpoint_encode(x.detach()[..., ::2]) is None and module.checkpoint_encode(x.detach()) is not None
    first = torch.autograd.grad(n.float().sum(), w, retain_graph=True)[0]
    assert torch.equal(first, torch.autograd.grad(n.float().sum(), w)[0])
    with pytest.raises(RuntimeError):                              # its tensors are gone
        torch.autograd.grad(n.float().sum(), w)
    z = draw(3, 3, 4, 64).to(cuda).requires_grad_()
    out, n = sparse.residual_norm(z, y, pre_kind="layer")
    out.detach().add_(1)                                           # what the backward pass reads was changed
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        n.float().sum().backward()


def test_what_is_held_between_the_passes(cuda):
    """A layer and an activation that keep 33/64 of their 16-bit input: what autograd saves is that, and no reference to the input."""
    import sparse
    x = draw(8, 512, 1024, dtype=BF16).to(cuda)
    layer = soft_layer(cuda, 1024, 256, 9, checkpoint=True)
    saved = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: (saved.append(t), t)[1], lambda t: t), torch.autocast("cuda", dtype=BF16):
        layer(x)                                                   # (an input that needs no gradient: nothing of the weight is saved)
        own = sum(t.numel() * t.element_size() for t in saved)
        assert own == 512 * 1024 * 33 // 32
        saved.clear()
        sparse.GELUglu(checkpoint=True)(x.view(2, 256, 1024).requires_grad_())
        assert sum(t.numel() * t.element_size() for t in saved) == 512 * 1024 * 33 // 32


def test_refusals(cuda):
    import sparse
    layer, x = soft_layer(cuda, 64, 64, 1, checkpoint=True), draw(2, 32, 64, dtype=BF16).to(cuda)
    kept = sparse.checkpoint_activation(x)
    with pytest.raises(RuntimeError, match="autocast"):
        layer(x.float(), checkpoint=kept)
    assert layer(x.float()).shape == (32, 64)                      # (without autocast nothing is kept, and nothing lost)
    with torch.autocast("cuda", dtype=BF16):
        for wrong in (sparse.checkpoint_activation(x.half()), sparse.checkpoint_activation(x[:8]), sparse.checkpoint_activation(x.view(4, 8, 64))):
            with pytest.raises(RuntimeError, match="checkpoint"):
                layer(x, checkpoint=wrong)
        leaf = x.detach().requires_grad_()
        with pytest.raises(RuntimeError, match="graph of the gradients"):
            torch.autograd.grad(layer(leaf).float().sum(), layer.weight, create_graph=True)
    sp = sparse_layer(cuda, 64, 64, 3)
    with pytest.raises(RuntimeError, match="checkpoint"):
        sp(x.half(), checkpoint=kept)
    sp.weight.mode = "dense"
    with pytest.raises(RuntimeError, match="mode"):
        sp(x.float(), checkpoint=kept)


class Block(nn.Module):
    def __init__(self, cuda, d, h, make, given, kind="rms", out_dtype=F16):
        import sparse
        super().__init__()
        self.norm = sparse.BlockNorm(d, kind, out_dtype=out_dtype, device=cuda)
        self.fc, self.proj = make(cuda, d, 2 * h, 20, checkpoint=not given), make(cuda, h, d, 22, checkpoint=not given)
        self.act = sparse.GELUglu(checkpoint=True, output_checkpoint=given)
        self.after = sparse.ResidualNorm(d, post=kind, pre=kind, gate=0.5, residual_scale=0.75, device=cuda)
        self.given = given

    def forward(self, x):
        if self.given:
            n, kept = self.norm(x, checkpoint=True)
            a, kept_a = self.act(self.fc(n, kept))
            return self.after(x, self.proj(a, kept_a))
        return self.after(x, self.proj(self.act(self.fc(self.norm(x)))))


def block_step(block, x, go, gn):
    for m in block.modules():
        if hasattr(m, "weight") and hasattr(m.weight, "cnt"):
            m.weight.cnt = 0
    leaf = x.detach().requires_grad_()
    torch.manual_seed(12)
    with torch.autocast("cuda", dtype=gn.dtype):
        out, n = block(leaf)
    params = [p for p in block.parameters() if p.requires_grad]
    return [out.detach(), n.detach(), *torch.autograd.grad((out, n), [leaf, *params], (go, gn))]


@pytest.mark.parametrize("make,dtype", [(sparse_layer, F16), (soft_layer, F16), (soft_layer, BF16)])
def test_block_with_checkpoints_handed_on_is_the_block_that_makes_its_own(cuda, make, dtype):
    x, go, gn = draw(30, 2, 64, 256).to(cuda), draw(31, 2, 64, 256, std=0.1).to(cuda), draw(32, 2, 64, 256, std=0.1, dtype=dtype).to(cuda)
    first, second = (Block(cuda, 256, 512, make, given, out_dtype=dtype) for given in (True, False))
    for a, b in zip(block_step(first, x, go, gn), block_step(second, x, go, gn)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("kind", ["rms", "layer"])
def test_block_against_float64(cuda, kind):
    """The whole block in float64, with the weights' gradients at the values that are kept of the inputs as float64 has them.  Twelve tensors are
    rounded to bfloat16 on the way there and back (n, the weights, 2 h, its halves' gradients, a, y, and the gradients of each), each by at most 2^-8
    of an element and by 2^-9 / sqrt(3) .. 2^-9 in the mean; maps in between keep relative 2-norms within the spread of their singular values (under 3
    here): 12 * 2^-9 * 3 = 0.07 of each gradient's norm.  A value that is kept in 8 bits and rounds to the other side moves by 2^-4 of itself, which a
    rounding error of 2^-9 does to one in 2^-9 / 2^-4 = 1/32 of them: 2^-4 / sqrt(32) = 0.011 in the norm."""
    d, h = 256, 384
    x, go, gn = draw(33, 2, 100, d), draw(34, 2, 100, d, std=0.1), draw(35, 2, 100, d, std=0.1, dtype=BF16)
    block = Block(cuda, d, h, soft_layer, True, kind, BF16)
    with torch.no_grad():
        for i, p in enumerate([block.norm.weight, block.after.post_weight, block.after.pre_weight]):
            p.add_(draw(36 + i, d, std=0.1).to(cuda))
    got = block_step(block, x.to(cuda), go.to(cuda), gn.to(cuda))
    names = ["out", "n", "x"] + [k for k, p in block.named_parameters() if p.requires_grad]

    p = {k: v.detach().cpu().double().requires_grad_() for k, v in block.named_parameters()}
    leaf = x.double().requires_grad_()

    class Kept(torch.autograd.Function):                           # x W^T whose weight gradient takes the kept x
        @staticmethod
        def forward(ctx, x, w):
            ctx.save_for_backward(oracle.kept_fast(x.to(BF16).reshape(-1, x.shape[-1])), w)
            return x @ w.t()

        @staticmethod
        def backward(ctx, g):
            x, w = ctx.saved_tensors
            return g @ w, g.reshape(-1, g.shape[-1]).t() @ x

    class Gated(torch.autograd.Function):
        @staticmethod
        def forward(ctx, v):
            ctx.save_for_backward(v)
            return oracle.gelu_glu_forward(v)

        @staticmethod
        def backward(ctx, g):
            (v,) = ctx.saved_tensors
            halves = v.to(BF16).reshape(-1, v.shape[-1] // 2)
            return oracle.gelu_glu_backward(g, oracle.kept_fast(halves).reshape(v.shape))

    class Thresholded(torch.autograd.Function):
        @staticmethod
        def forward(ctx, w, layer):
            return layer.get_sparse_weights().detach().cpu().double()

        @staticmethod
        def backward(ctx, g):
            return g, None

    n0 = oracle.norm(leaf, kind, p["norm.weight"], p.get("norm.bias"), 1e-5)
    a = Gated.apply(Kept.apply(n0, Thresholded.apply(p["fc.weight"], block.fc)) + p["fc.bias"])
    y = Kept.apply(a, Thresholded.apply(p["proj.weight"], block.proj)) + p["proj.bias"]
    out = 0.75 * leaf + p["after.gate"] * oracle.norm(y, kind, p["after.post_weight"], p.get("after.post_bias"), 1e-5)
    n = oracle.norm(out, kind, p["after.pre_weight"], p.get("after.pre_bias"), 1e-5)
    wanted = [leaf, *(p[k] for k in names[3:])]
    want = [out, n, *torch.autograd.grad((out, n), wanted, (go.double(), gn.double()))]
    for name, g, w in zip(names, got, want):
        w = w.detach()
        assert (g.cpu().double() - w).norm() <= (12 * 2.0 ** -9 * 3 + 0.011) * w.norm(), (name, ((g.cpu().double() - w).norm() / w.norm()).item())


def test_block_captured_and_replayed(cuda):
    """A step of the S-STE block recorded into a graph: each replay gives the eager step's bits on the inputs of the moment."""
    x, go, gn = draw(40, 2, 128, 256).to(cuda), draw(41, 2, 128, 256, std=0.1).to(cuda), draw(42, 2, 128, 256, std=0.1, dtype=BF16).to(cuda)
    block = Block(cuda, 256, 256, soft_layer, True, out_dtype=BF16)

    def one():
        leaf = x.detach().requires_grad_()
        with torch.autocast("cuda", dtype=BF16):
            out, n = block(leaf)
        params = [p for p in block.parameters() if p.requires_grad]
        return [out.detach(), n.detach(), *torch.autograd.grad((out, n), [leaf, *params], (go, gn))]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        one()                                                      # (the library's own workspaces are made outside the capture)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        recorded = one()
    for replay in range(3):
        x.mul_(1.0 + 0.25 * replay)
        go.neg_()
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in recorded]
        for a, b in zip(got, one()):
            assert torch.equal(a, b), replay


def test_no_graph_of_the_gradients_of_a_sparse_layer_that_keeps_its_input_in_8_bits(cuda):
    layer, x = sparse_layer(cuda, 64, 64, 3), draw(4, 64, 64, dtype=F16).to(cuda).requires_grad_()
    with pytest.raises(RuntimeError, match="graph of the gradients"):
        torch.autograd.grad(layer(x, checkpoint=True).float().sum(), layer.weight, create_graph=True)
