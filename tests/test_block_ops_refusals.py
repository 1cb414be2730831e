"""What the block norms and the calls that keep activations in 8 bits refuse, before anything is launched (the addresses are made up)."""
import pytest
import torch

A, B, C = 0x7f0000001000, 0x7f0000100000, 0x7f0000200000
SHAPE, DTYPE, STRIDE, ARG = -1, -2, -3, -5


@pytest.fixture(scope="module")
def lib():
    from sparse import _native
    return _native.lib()


def test_checkpoint_arguments(lib):
    from sparse import _native as N
    assert [lib.tf24_checkpoint_blocks(c) for c in (1, 32, 33, 768)] == [1, 1, 2, 24]
    encode = lambda x=A, dtype=N.F16, ld=64, rows=4, cols=64, values=B, scales=C: lib.tf24_checkpoint_encode(x, dtype, ld, rows, cols, values, scales, None)
    assert encode(rows=0) == 0 and encode(rows=0, x=None) == 0
    assert encode(dtype=N.E4M3) == DTYPE and encode(cols=0) == SHAPE and encode(rows=-1) == SHAPE and encode(rows=1 << 29) == SHAPE
    assert encode(x=None) == ARG and encode(values=None) == ARG and encode(scales=None) == ARG
    assert encode(x=A + 1) == STRIDE and encode(values=B + 8) == STRIDE and encode(ld=-64) == STRIDE
    decode = lambda values=B, scales=C, rows=4, cols=64, out=A, dtype=N.F16, ld=64: lib.tf24_checkpoint_decode(values, scales, rows, cols, out, dtype, ld, None)
    assert decode(rows=0) == 0 and decode(ld=63) == STRIDE and decode(out=None) == ARG and decode(dtype=N.I32) == DTYPE and decode(values=B + 4) == STRIDE
    assert b"aligned" in lib.tf24_last_error()


def test_glu_checkpoint_arguments(lib):
    from sparse import _native as N
    forward = lambda x=A, dtype=N.F16, ld=64, rows=4, cols=64, out=B, ld_out=32, values=C, scales=C, ov=None, os=None: lib.tf24_gelu_glu_forward_checkpoint(
        x, dtype, ld, rows, cols, out, ld_out, values, scales, ov, os, None)
    assert forward(rows=0) == 0 and forward(cols=63) == SHAPE and forward(cols=0) == SHAPE and forward(dtype=N.E4M3) == DTYPE
    assert forward(ld=63) == STRIDE and forward(ld_out=31) == STRIDE and forward(values=C + 8) == STRIDE and forward(x=A + 1) == STRIDE
    assert forward(ov=C) == ARG and forward(os=C) == ARG and forward(scales=None) == ARG
    backward = lambda go=A, ld=32, values=C, scales=C, dtype=N.F16, rows=4, cols=64, gi=B, ld_gi=64: lib.tf24_gelu_glu_backward_checkpoint(
        go, ld, values, scales, dtype, rows, cols, gi, ld_gi, None)
    assert backward(rows=0) == 0 and backward(ld=31) == STRIDE and backward(ld_gi=63) == STRIDE and backward(gi=None) == ARG and backward(cols=2 << 30) == SHAPE


def test_weight_gradient_arguments(lib):
    from sparse import _native as N

    def call(g=A, ldg=64, dtype=N.F16, values=B, scales=C, tokens=100, m=64, n=33, dw=A, db=None, out=N.F16, ws=None, ws_bytes=0):
        return lib.tf24_checkpoint_weight_grad(g, ldg, dtype, values, scales, tokens, m, n, dw, db, out, ws, ws_bytes, None)

    assert call(dtype=N.F32) == DTYPE and call(out=N.BF16) == DTYPE and call(dtype=N.BF16) == DTYPE
    assert call(tokens=0) == SHAPE and call(m=60) == SHAPE and call(m=0) == SHAPE and call(n=0) == SHAPE and call(n=(1 << 20) + 1) == SHAPE
    assert call(ldg=56) == STRIDE and call(ldg=68) == STRIDE and call(ldg=(1 << 23) + 8) == STRIDE
    assert call(g=None) == ARG and call(values=None) == ARG and call(scales=None) == ARG and call(dw=None) == ARG and call(ws_bytes=-1) == ARG
    assert call(g=A + 8) == STRIDE and call(values=B + 8) == STRIDE and call(ws=A + 8) == STRIDE and call(dw=A + 2, out=N.F32) == STRIDE
    need = lib.tf24_checkpoint_weight_grad_workspace_bytes
    assert need(0, 64, 64) == 0 and need(64, 256, 256) == 0 and need(8192, 768, 768) > 0


def test_block_norm_arguments(lib):
    from sparse import _native as N

    def forward(x=A, ld_x=64, y=B, ld_y=64, stream=N.F32, block=N.F16, rows=6, cols=64, gate=None, gate_dtype=N.F32, ld_gate=64, per_gate=1, pw=None, pb=None, w=None,
                b=None, param=N.F32, post=0, pre=N.NORM_RMS, out=C, n=C, stats=None, values=None, scales=None):
        return lib.tf24_block_norm_forward(x, ld_x, y, ld_y, stream, block, rows, cols, gate, gate_dtype, ld_gate, per_gate, pw, pb, w, b, param, post, pre, 1.0, 1e-5,
                                           out, n, stats, values, scales, None)

    assert forward(rows=0) == 0
    assert forward(stream=N.F16, block=N.BF16) == DTYPE and forward(stream=N.F16, block=N.F32) == DTYPE and forward(param=N.U8) == DTYPE
    assert forward(gate=A, gate_dtype=N.U8) == DTYPE and forward(block=N.E4M3) == DTYPE
    assert forward(cols=0) == SHAPE and forward(cols=16385) == SHAPE and forward(rows=-1) == SHAPE and forward(rows=0x7fffffff) == SHAPE
    assert forward(gate=A, per_gate=4) == SHAPE and forward(gate=A, per_gate=0) == SHAPE
    assert forward(post=3) == ARG and forward(pre=-1) == ARG
    assert forward(x=None) == ARG and forward(out=None) == ARG and forward(n=None) == ARG and forward(values=B) == ARG and forward(pre=0, values=B, scales=C) == ARG
    assert forward(y=None) == ARG and forward(y=None, out=None, pre=0) == ARG and forward(y=None, out=None, gate=A, per_gate=1) == ARG
    assert forward(ld_x=-64) == STRIDE and forward(x=A + 2) == STRIDE and forward(y=B + 1) == STRIDE and forward(w=A + 2) == STRIDE and forward(stats=A + 4) == STRIDE
    assert forward(values=B + 8, scales=C) == STRIDE

    def backward(dout=A, dn=A, h=A, y=B, stream=N.F32, block=N.F16, rows=6, cols=64, gate=None, per_gate=1, post=0, pre=N.NORM_RMS, residual=1, stats=A, gx=C, gy=C,
                 gg=None, gpw=None, gpb=None, gw=None, gb=None, ws=None, ws_bytes=0):
        return lib.tf24_block_norm_backward(dout, 64, dn, 64, h, 64, y, 64, stream, block, rows, cols, gate, N.F32, 64, per_gate, None, None, None, N.F32, post, pre,
                                            residual, 1.0, stats, gx, gy, gg, gpw, gpb, gw, gb, ws, ws_bytes, None)

    assert backward(rows=0) == SHAPE and backward(cols=20000) == SHAPE and backward(gate=A, per_gate=4) == SHAPE and backward(stream=N.BF16) == DTYPE
    assert backward(dn=None) == ARG and backward(h=None) == ARG and backward(stats=None) == ARG and backward(pre=0, dout=None) == ARG and backward(pre=0, gw=C) == ARG
    assert backward(gg=C) == ARG and backward(gpw=C) == ARG and backward(y=None, post=1) == ARG and backward(residual=0) == ARG
    assert backward(gw=C) == ARG and b"workspace" in lib.tf24_last_error()
    assert backward(gw=C, ws=A, ws_bytes=lib.tf24_block_norm_backward_workspace_bytes(6, 64, 6) - 1) == ARG
    assert backward(gw=C, ws=A + 4, ws_bytes=1 << 20) == STRIDE and backward(gx=C + 2) == STRIDE
    assert lib.tf24_block_norm_backward_workspace_bytes(0, 64, 1) == 0 and lib.tf24_block_norm_backward_workspace_bytes(6, 64, 6) % (64 * 16) == 0


def test_python_refuses_tensors_that_are_not_on_a_gpu():
    import sparse
    x = torch.zeros(4, 64)
    for call in (lambda: sparse.checkpoint_activation(x), lambda: sparse.block_norm(x), lambda: sparse.residual_norm(x, x, pre_kind="rms"),
                 lambda: sparse.gelu_glu_checkpoint.apply(x), lambda: sparse.GELUglu(checkpoint=True)(x)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


def test_python_refuses_what_does_not_fit_together():
    import sparse
    with pytest.raises(RuntimeError, match="do not hold"):
        sparse.ActivationCheckpoint(torch.zeros(4, 64).to(torch.float8_e4m3fn), torch.zeros(4, 1, dtype=torch.uint8), (4, 64), torch.float16)
    with pytest.raises(RuntimeError, match="do not hold"):
        sparse.ActivationCheckpoint(torch.zeros(4, 64).to(torch.float8_e4m3fn), torch.zeros(4, 2, dtype=torch.uint8), (4, 64), torch.float64)
    sparse.ActivationCheckpoint(torch.zeros(4, 64).to(torch.float8_e4m3fn), torch.zeros(4, 2, dtype=torch.uint8), (2, 2, 63), torch.float16)
    with pytest.raises(RuntimeError, match="kind of norm"):
        sparse.BlockNorm(8, kind="batch")
    with pytest.raises(RuntimeError, match="kind of norm"):
        sparse.ResidualNorm(8, post="batch")
    with pytest.raises(RuntimeError, match="output_checkpoint"):
        sparse.GELUglu(output_checkpoint=True)
    assert sparse.ResidualNorm(8, post="rms", pre="layer", gate=0.1).gate.tolist() == [pytest.approx(0.1)] * 8
    assert {k for k, _ in sparse.ResidualNorm(8, post="rms", pre="layer").named_parameters()} == {"post_weight", "pre_weight", "pre_bias"}


def test_calls_go_to_the_stream_of_the_tensors_device(monkeypatch):
    from contextlib import contextmanager
    from sparse import _native as N
    current, streams = [0], []

    class Tensor:
        device = "device 1"

        def get_device(self):
            return 1

    @contextmanager
    def device(d):
        assert d == "device 1"
        current[0] = 1
        yield
        current[0] = 0

    monkeypatch.setattr(torch.cuda, "current_device", lambda: current[0])
    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(N, "stream_ptr", lambda: 100 + current[0])
    N.launch(Tensor(), lambda *a: (streams.append(a), 0)[1], 7)
    current[0] = 1
    N.launch(Tensor(), lambda *a: (streams.append(a), 0)[1], 8)
    assert streams == [(7, 101), (8, 101)]


def test_rows_of_any_tensor():
    """as_rows: contiguous tensors as they are, others as a matrix of contiguous rows whose leading dimension may be 0."""
    from sparse import _native as N
    x = torch.arange(60.0).view(3, 4, 5)
    assert N.as_rows(x)[0] is x and N.as_rows(x)[1] == 5
    for view in (x[:, ::2], x[..., 1:4], x.transpose(0, 1), x.transpose(1, 2), x[:1, :1].expand(2, 3, 5), x[..., :1].expand(3, 4, 5), x[0, 0, ::2], torch._neg_view(x)):
        rows, ld = N.as_rows(view)
        flat = torch.as_strided(rows, (view.numel() // view.shape[-1], view.shape[-1]), (ld, 1))
        assert torch.equal(flat, view.resolve_neg().reshape(-1, view.shape[-1]))


def test_layers_refuse_what_is_no_checkpoint():
    from sparse.activation_checkpoint import as_checkpoint
    for given in (False, torch.zeros(4, 64), 1):
        with pytest.raises(RuntimeError, match="checkpoint"):
            as_checkpoint(torch.zeros(4, 64), given)


def test_a_gated_activation_from_before_it_could_keep_anything():
    import sparse
    old = sparse.GELUglu.__new__(sparse.GELUglu)
    old.__setstate__({k: v for k, v in sparse.GELUglu().__dict__.items() if "checkpoint" not in k})
    assert not old.checkpoint and not old.output_checkpoint
    with pytest.raises(RuntimeError, match="CUDA"):
        old(torch.zeros(1, 4, 64))


def test_more_gates_than_a_launch_has_workgroups(lib):
    from sparse import _native as N

    def backward(rows, cols, per_gate, grad_gate, ws_bytes):
        return lib.tf24_block_norm_backward(A, cols, None, 0, None, 0, A, cols, N.F16, N.F16, rows, cols, A, N.F16, cols, per_gate, None, None, None, N.F32, 0, 0, 1, 1.0,
                                            None, B, C, grad_gate, None, None, None, None, A if ws_bytes else None, ws_bytes, None)

    assert backward(1 << 24, 64, 2, None, 0) == SHAPE and b"gates" in lib.tf24_last_error()
    assert backward(1 << 22, 16384, 2, C, 1 << 62) == SHAPE and b"gates" in lib.tf24_last_error()
