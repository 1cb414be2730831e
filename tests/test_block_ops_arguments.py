"""What the modules around the layers take and refuse, as far as it needs no GPU."""
import warnings

import pytest
import torch


def test_a_checkpoint_off_the_gpu_is_not_decoded():
    import sparse
    kept = sparse.ActivationCheckpoint(torch.zeros(4, 64).to(torch.float8_e4m3fn), torch.zeros(4, 2, dtype=torch.uint8), (4, 64), torch.float16)
    with pytest.raises(RuntimeError, match="CUDA"):
        kept.decode()


@pytest.mark.parametrize("first", [0, 1, 0.25, torch.tensor(2)])
@pytest.mark.parametrize("dtype", [None, torch.bfloat16])
def test_first_values_of_a_learned_gate(first, dtype):
    """Whole numbers are numbers: zero and one are the usual first values."""
    import sparse
    gate = sparse.ResidualNorm(8, gate=first, dtype=dtype).gate
    assert gate.requires_grad and gate.dtype == (dtype or torch.float32) and gate.tolist() == [float(first)] * 8


def test_no_checkpoint_of_a_dense_call():
    """False is no, in mode 'dense' too; True and a checkpoint are refused there."""
    import sparse
    layer = sparse.SparseLinearTranspose(16, 8, checkpoint=True)
    layer.weight.mode = "dense"
    x = torch.randn(4, 16)
    assert torch.equal(layer(x, checkpoint=False), torch.nn.functional.linear(x, layer.weight, layer.bias))
    with pytest.raises(RuntimeError, match="mode 'sparse'"):
        layer(x, checkpoint=True)


def test_a_layer_says_that_its_setting_has_no_effect():
    import sparse
    layer = sparse.SparseLinearTranspose(16, 8, checkpoint=True)
    layer.weight.mode = "dense"
    x = torch.randn(4, 16)
    with pytest.warns(UserWarning, match="no effect.*mode 'sparse'"):
        layer(x)
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        layer(x, checkpoint=False)
        with torch.no_grad():
            layer(x)
        layer.checkpoint = False
        layer(x)
