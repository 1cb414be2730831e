"""What the losses of a vocabulary head refuse, before anything is launched (the addresses are made up)."""
import pytest
import torch

A, B, C, D = 0x7f0000001000, 0x7f0000100000, 0x7f0000200000, 0x7f0000300000
SHAPE, DTYPE, STRIDE, ARG = -1, -2, -3, -5
MANY = 1 << 60


@pytest.fixture(scope="module")
def lib():
    from sparse import _native
    return _native.lib()


def test_forward_arguments(lib):
    from sparse import _native as N

    def call(x=A, ldx=64, w=B, ldw=64, bias=None, bias_dtype=N.F32, dtype=N.F16, tokens=10, width=64, words=100, targets=C, indices=None, ld_i=4, logits=None, ld_l=4,
             teacher=N.F32, lse=None, entries=0, smoothing=0.0, z_loss=0.0, inv=1.0, reduction=0, loss=D, state=A, state_bytes=0, ws=B, ws_bytes=0):
        return lib.tf24_linear_loss_forward(x, ldx, w, ldw, bias, bias_dtype, dtype, tokens, width, words, targets, -100, indices, ld_i, logits, ld_l, teacher, lse, entries,
                                            smoothing, z_loss, inv, reduction, loss, state, state_bytes, ws, ws_bytes, None)

    assert call() == ARG and b"needed" in lib.tf24_last_error()    # no room
    assert call(state_bytes=MANY) == ARG and call(ws_bytes=MANY) == ARG and call(state_bytes=MANY, ws_bytes=-1) == ARG
    assert call(dtype=N.F32) == DTYPE and call(bias=A, bias_dtype=N.I8) == DTYPE
    for size in ("tokens", "width", "words"):
        assert call(**{size: 0}) == SHAPE and call(**{size: -1}) == SHAPE and call(**{size: (1 << 22) + 1}) == SHAPE
    assert call(width=(1 << 16) + 1) == SHAPE and call(tokens=1 << 22, words=1 << 22) == SHAPE
    assert call(ldx=-1) == STRIDE and call(ldw=-64) == STRIDE
    assert call(x=None) == ARG and call(w=None) == ARG and call(targets=None) == ARG and call(loss=None) == ARG and call(state=None) == ARG and call(ws=None) == ARG
    assert call(x=A + 1) == STRIDE and call(w=B + 1) == STRIDE and call(state=A + 8) == STRIDE and call(ws=B + 4) == STRIDE and call(targets=C + 4) == STRIDE
    assert call(loss=D + 2) == STRIDE and call(bias=A + 2) == STRIDE and call(bias=A + 1, bias_dtype=N.BF16) == STRIDE
    for bad in (-0.1, 1.1, float("nan")):
        assert call(smoothing=bad) == ARG
    assert call(z_loss=float("inf")) == ARG and call(inv=0.0) == ARG and call(inv=float("inf")) == ARG and call(reduction=3) == ARG
    kd = dict(targets=None, indices=C, logits=D, entries=4)
    assert call(**kd) == ARG and b"needed" in lib.tf24_last_error()
    assert call(**{**kd, "entries": 1025}) == SHAPE and call(**{**kd, "entries": -1}) == SHAPE and call(**{**kd, "targets": A}) == ARG and call(**{**kd, "logits": None}) == ARG
    assert call(**kd, smoothing=0.1) == ARG and call(**kd, z_loss=0.1) == ARG and call(**kd, teacher=N.U8) == DTYPE and call(**kd, ld_i=-4) == STRIDE
    assert call(**{**kd, "logits": D + 2}) == STRIDE and call(**kd, lse=A + 2) == STRIDE and call(indices=A) == ARG


def test_backward_arguments(lib):
    from sparse import _native as N

    def call(grad=A, x=A, w=B, bias=None, bias_dtype=N.F32, dtype=N.BF16, tokens=10, width=64, words=100, entries=0, smoothing=0.0, reduction=2, state=C, state_bytes=MANY,
             dx=D, dw=D, dw_dtype=N.BF16, db=None, ws=B, ws_bytes=0):
        return lib.tf24_linear_loss_backward(grad, x, 64, w, 64, bias, bias_dtype, dtype, tokens, width, words, entries, smoothing, 0.0, 1.0, reduction, state, state_bytes, dx, dw,
                                             dw_dtype, db, ws, ws_bytes, None)

    assert call() == ARG and b"needed" in lib.tf24_last_error()
    assert call(state_bytes=0, ws_bytes=MANY) == ARG and call(dx=None, dw=None, ws_bytes=MANY) == 0
    assert call(grad=None) == ARG and call(state=None) == ARG and call(ws=None) == ARG and call(db=D) == ARG and call(tokens=0) == SHAPE and call(dtype=N.F32) == DTYPE
    assert call(dw_dtype=N.F16) == DTYPE and call(dw=D + 2, dw_dtype=N.F32) == STRIDE and call(dx=D + 1) == STRIDE and call(grad=A + 2) == STRIDE
    assert call(bias=A, db=D + 2) == STRIDE and call(reduction=-1) == ARG


def test_sizes_of_buffers(lib):
    state, forward, backward = lib.tf24_linear_loss_state_bytes, lib.tf24_linear_loss_forward_workspace_bytes, lib.tf24_linear_loss_backward_workspace_bytes
    assert state(0, 0) == 0 and state(10, 1025) == 0 and forward(0, 64, 100, 0, 0, A, 64) == 0 and backward(10, 64, 0, 0, 0, A, 64, 1, 1, 1) == 0
    assert 192 * 4 * 5 <= state(10, 0) < state(10, 64)
    # an operand that is not in whole aligned stages is brought into them, but for few tokens; the gradient of the logits takes 2 GiB and no more
    assert forward(100, 64, 5000, 0, 0, A + 2, 64) >= forward(100, 64, 5000, 0, 0, A, 64) + 5000 * 128
    assert forward(64, 64, 5000, 0, 0, A + 2, 64) == forward(64, 64, 5000, 0, 0, A, 64)
    at_most = backward(1 << 17, 64, 1 << 17, 0, 0, A, 64, 0, 1, 0)
    assert (1 << 30) < at_most < (2 << 30) + (1 << 28) + (1 << 26)


def test_operands_off_the_gpu():
    import sparse
    x, w, t = torch.zeros(2, 8, dtype=torch.bfloat16), torch.zeros(5, 8, dtype=torch.bfloat16), torch.zeros(2, dtype=torch.long)
    with pytest.raises(RuntimeError, match="CUDA"):
        sparse.linear_cross_entropy(x, w, t)
    with pytest.raises(RuntimeError, match="CUDA"):
        sparse.VocabularyLinear(8, 5)(x.float(), indices=t[:, None], teacher_logits=torch.zeros(2, 1))
    with pytest.raises(RuntimeError, match="not a tensor"):
        sparse.linear_distillation(x, None, t, x)
    head = sparse.VocabularyLinear(8, 5, bias=True)
    assert torch.equal(head(x.float()), torch.nn.functional.linear(x.float(), head.weight, head.bias))
    for wrong in (dict(reduction="sum"), dict(indices=t), dict(teacher_logits=x)):
        with pytest.raises(RuntimeError, match="VocabularyLinear"):
            head(x, **wrong)
