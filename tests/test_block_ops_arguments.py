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


def test_n_that_could_not_be_read_again_is_not_kept():
    """A kept matrix has at most 2^31 units of eight columns: what decode refuses, the norm that would write it does too.  (The addresses are made up.)"""
    from sparse import _native as N
    lib, at = N.lib(), 0x7f0000001000

    def forward(rows, cols):
        return lib.tf24_block_norm_forward(at, cols, None, 0, N.BF16, N.BF16, rows, cols, None, N.F32, 0, 1, None, None, None, None, N.F32, 0, N.NORM_RMS, 1.0, 1e-5, None,
                                           at, None, at, at, None)

    def decode(rows, cols):
        return lib.tf24_checkpoint_decode(at, at, rows, cols, at, N.BF16, cols, None)

    for rows, cols in ((1 << 20, 16384), (1 << 29, 32), (1 << 29, 1)):
        assert forward(rows, cols) == decode(rows, cols) == -1 and b"too large" in lib.tf24_last_error()


def test_weight_gradient_of_a_kept_matrix_that_is_not_decoded():
    """A product whose decoded operand would be too large for that pass has the other way, and asks for room for its pieces at most."""
    from sparse import _native as N
    need = N.lib().tf24_checkpoint_weight_grad_workspace_bytes
    tokens = 1 << 21
    assert need(tokens // 4, 4096, 8192) >= tokens // 4 * 8192 * 2
    assert need(tokens, 4096, 8192) < tokens * 8192 * 2


def test_a_gate_is_a_tensor():
    import sparse
    x = torch.zeros(4, 64)
    for gate in (0.5, 1, [1.0] * 64):
        with pytest.raises(RuntimeError, match="residual_norm: gate is"):
            sparse.residual_norm(x, x, gate, pre_kind="rms")


def test_the_gated_activation_is_called_from_compiled_code(monkeypatch):
    """Without the module of torch's C++ side as well: what the compiler cannot trace it leaves to Python, whose call says here that there is no GPU."""
    import sparse
    from sparse import _native as N
    for calls in (N.torch_calls(), None):
        monkeypatch.setattr(N, "_calls", calls)
        torch._dynamo.reset()
        with pytest.raises(Exception) as raised:
            torch.compile(lambda x: sparse.gelu_glu_checkpoint.apply(x), backend="eager")(torch.zeros(2, 8))
        assert "only CUDA tensors" in str(raised.value), raised.value
