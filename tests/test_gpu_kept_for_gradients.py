"""What the operators keep in 8 bits is kept for a backward pass, and only where there will be one."""
import warnings

import pytest
import torch

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


def allocations(call):
    """(what call returns, the number of tensors that it allocates)"""
    call()                                                         # (libraries allocate workspaces the first time)
    before = torch.cuda.memory_stats()["allocation.all.allocated"]
    result = call()
    return result, torch.cuda.memory_stats()["allocation.all.allocated"] - before


def without_graph(x):
    """Ways in which a call records no graph."""
    yield "no_grad", torch.no_grad(), x.detach().requires_grad_()
    yield "inference_mode", torch.inference_mode(), x.detach().requires_grad_()
    yield "no gradient wanted", torch.enable_grad(), x.detach()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("rows,half", [(1, 1), (5, 32), (37, 200), (300, 1001)])
def test_gated_activation_without_a_graph_keeps_no_input(cuda, rows, half, dtype):
    import sparse
    x = draw(1, rows, 2 * half, dtype=dtype).to(cuda)
    out, values, scales = sparse.gelu_glu_checkpoint.apply(x.detach().requires_grad_(), True)
    for name, mode, leaf in without_graph(x):
        with mode:
            got, count = allocations(lambda: sparse.gelu_glu_checkpoint.apply(leaf))
            assert torch.equal(got, out) and not got.requires_grad and count == 1, (name, count)
            (got, v, s), count = allocations(lambda: sparse.gelu_glu_checkpoint.apply(leaf, True))
            assert torch.equal(got, out) and torch.equal(v.view(torch.uint8), values.view(torch.uint8)) and torch.equal(s, scales) and count == 3, (name, count)
            got, kept = sparse.GELUglu(checkpoint=True, output_checkpoint=True)(leaf)
            assert torch.equal(got, out) and torch.equal(kept.scales, scales)
    assert not sparse.gelu_glu_checkpoint.apply(x.detach()[None]).requires_grad
    strided = torch.zeros(rows, 2 * half + 3, dtype=dtype, device=cuda)
    strided[:, 1:-2] = x
    with torch.no_grad():
        assert torch.equal(sparse.gelu_glu_checkpoint.apply(strided[:, 1:-2]), out)


@pytest.mark.parametrize("make", ["soft threshold", "2:4"])
def test_layers_without_a_graph_keep_no_input(cuda, make):
    """As many allocations as the layer that keeps its input as it is, and the same output."""
    import sparse
    if make == "2:4":
        layer = sparse.SparseLinearTranspose(128, 256, device=cuda, checkpoint=True)
    else:
        layer = sparse.SoftThresholdLinear(128, 256, device=cuda, checkpoint=True)
        layer.init_scale()
    layer.eval()
    x = draw(3, 64, 128).to(cuda)
    with torch.autocast("cuda", dtype=F16):
        want = layer(x).detach()
        for mode in (torch.no_grad(), torch.inference_mode()):
            with mode:
                layer.checkpoint = False
                same, fewest = allocations(lambda: layer(x))
                layer.checkpoint = True
                out, count = allocations(lambda: layer(x))
                assert torch.equal(out, want) and torch.equal(same, want) and count == fewest, (mode, count, fewest)
    # with a graph it is kept
    saved = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: (saved.append(t.dtype), t)[1], lambda t: t), torch.autocast("cuda", dtype=F16):
        layer(x)
    assert torch.float8_e4m3fn in saved


@pytest.mark.parametrize("make", ["soft threshold", "2:4"])
def test_no_for_one_call(cuda, make):
    """checkpoint=False keeps the input of this call as it is, whatever the layer's own setting, True keeps it in 8 bits."""
    import sparse
    if make == "2:4":
        layer = sparse.SparseLinearTranspose(128, 256, device=cuda, checkpoint=True)
    else:
        layer = sparse.SoftThresholdLinear(128, 256, device=cuda, checkpoint=True)
        layer.init_scale()
    layer.eval()
    x = draw(4, 64, 128).to(cuda)

    def kept(**kw):
        saved = []
        with torch.autograd.graph.saved_tensors_hooks(lambda t: (saved.append(t.dtype), t)[1], lambda t: t), torch.autocast("cuda", dtype=F16):
            layer(x, **kw)
        return torch.float8_e4m3fn in saved

    assert [kept(), kept(checkpoint=False), kept(checkpoint=True)] == [True, False, True]
    layer.checkpoint = False
    assert [kept(), kept(checkpoint=False), kept(checkpoint=True)] == [False, False, True]


def test_a_layer_says_that_its_setting_has_no_effect(cuda):
    """Outside autocast, and for a transposed input, the soft-threshold layer keeps its input as it is, and says so where there will be a backward pass."""
    import sparse
    layer = sparse.SoftThresholdLinear(128, 256, device=cuda, checkpoint=True)
    layer.init_scale()
    x = draw(5, 64, 128).to(cuda)
    with pytest.warns(UserWarning, match="no effect.*autocast"):
        layer(x)
    with torch.autocast("cuda", dtype=F16), pytest.warns(UserWarning, match="no effect.*contiguous"):
        layer(draw(6, 128, 64).to(cuda).t())
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        with torch.autocast("cuda", dtype=F16):
            layer(x)
        layer(x, checkpoint=False)
        with torch.no_grad():
            layer(x)
    with pytest.raises(RuntimeError, match="autocast"):
        layer(x, checkpoint=True)
