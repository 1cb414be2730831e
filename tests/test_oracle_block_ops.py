"""The oracle of the block norms and of activations kept in 8 bits, against torch's own cast, norms and gradients."""
import pytest
import torch

import oracle


def test_kept_values_by_hand():
    x = torch.zeros(1, 70)
    x[0, 0], x[0, 1], x[0, 2], x[0, 3] = 1.75, 1.76, 0.001, -0.3
    x[0, 32], x[0, 33] = 1.75, 0.001
    x[0, 64], x[0, 65], x[0, 66] = float("inf"), 3.0, float("nan")
    got = oracle.kept(x)
    # 1.76 does not fit 448 * 2^-8: scale 2^-7, numbers of 4 bits of mantissa, multiples of 2^-16 at the bottom
    assert oracle.kept_scale(x[0, :32]) == -7 and oracle.kept_scale(x[0, 32:64]) == -8 and oracle.kept_scale(x[0, 64:]) == -7
    assert got[0, 0] == 1.75 and got[0, 1] == 1.75 and got[0, 3] == -0.3125
    assert got[0, 2] == 66 * 2.0 ** -16 or got[0, 2] == 64 * 2.0 ** -16
    assert got[0, 65] == 3.0 and got[0, 64].isnan() and got[0, 66].isnan() and got[0, 67] == 0
    assert oracle.kept_scale(torch.zeros(32)) == -117


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_kept_is_the_cast_of_scaled_blocks(dtype):
    g = torch.Generator().manual_seed(1)
    x = (torch.randn(20, 77, generator=g) * torch.exp(3 * torch.randn(77, generator=g))).to(dtype)
    x[1] = 0
    x[2] *= 1e-4
    x[3, 5] = torch.finfo(dtype).max
    assert torch.equal(oracle.kept(x), oracle.kept_fast(x))
    assert torch.equal(oracle.kept(x).to(dtype).double(), oracle.kept(x)) and oracle.kept(x).to(dtype).isfinite().all()
    error = (oracle.kept(x) - x.double()).abs()
    units = torch.tensor([[2.0 ** oracle.kept_scale(x[r, c // 32 * 32:c // 32 * 32 + 32]) for c in range(77)] for r in range(20)]).double()
    assert (error <= torch.maximum(x.double().abs() / 16, units * 2.0 ** -10)).all()


@pytest.mark.parametrize("kind", ["rms", "layer"])
def test_norms_and_their_gradients(kind):
    g = torch.Generator().manual_seed(2)
    v, w, b, grad = (torch.randn(*s, generator=g, dtype=torch.float64) for s in ((5, 37), (37,), (37,), (5, 37)))
    v, w, b = v.requires_grad_(), w.requires_grad_(), b.requires_grad_()
    want = torch.nn.functional.layer_norm(v, (37,), w, b, 1e-3) if kind == "layer" else torch.nn.functional.rms_norm(v, (37,), w, 1e-3) + b
    assert torch.allclose(oracle.norm(v, kind, w, b, 1e-3), want, rtol=1e-12, atol=1e-12)
    dv, dw, db = torch.autograd.grad(want, (v, w, b), grad)
    got = oracle.norm_backward(grad, v.detach(), kind, w.detach(), 1e-3)
    for a, e in zip((got[0], got[1].sum(0), got[2].sum(0)), (dv, dw, db)):
        assert torch.allclose(a, e, rtol=1e-11, atol=1e-12)
