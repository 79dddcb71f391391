"""Rotary positions under autograd."""

import pytest
import torch

from cxlsparse_b200.rotary import Rotary, frequencies
from test_gpu_rotary import close, formula

pytestmark = pytest.mark.gpu

YARN = dict(type="yarn", factor=4.0, original=4096)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("transpose", [False, True])
def test_apply_has_the_formula_s_gradient(cuda, layout, dtype, transpose):
    rotary = Rotary(64, rotary_dim=48, layout=layout, scaling=YARN)
    f, magnitude = frequencies(48, scaling=YARN)
    g = torch.Generator(device="cuda").manual_seed(0)
    q, gq = (torch.randn(33, 4, 64, generator=g, device="cuda").to(dtype) for _ in range(2))
    k, gk = (torch.randn(33, 2, 64, generator=g, device="cuda").to(dtype) for _ in range(2))
    positions = torch.randint(0, 100000, (33,), generator=g, device="cuda")
    plain = rotary.apply(q, k, positions, transpose=transpose)
    q.requires_grad_()
    k.requires_grad_()
    out = rotary.apply(q, k, positions, transpose=transpose)
    assert all(torch.equal(x, y) for x, y in zip(out, plain))
    torch.autograd.backward(out, (gq, gk))
    for x, grad in ((q, gq), (k, gk)):
        want, size = formula(grad, positions, f, magnitude, layout, not transpose)
        close(x.grad, want, size, dtype)
    # One tensor, or one that needs a gradient.
    for a, b in ((q, None), (None, k), (q, k.detach()), (q.detach(), k)):
        y = rotary.apply(a, b, positions, transpose=transpose)
        for x, out_x, grad in ((a, y[0], gq), (b, y[1], gk)):
            if x is None or not x.requires_grad:
                assert out_x is None or x is not None
                continue
            got, = torch.autograd.grad(out_x, x, grad, retain_graph=True)
            want, size = formula(grad, positions, f, magnitude, layout, not transpose)
            close(got, want, size, dtype)


def test_gradients_of_sums_parts_and_of_gradients(cuda):
    """Broadcast gradients (a sum's), an unused output, strided inputs, and the
    second derivative, which is the rotation of the gradient's gradient."""
    rotary = Rotary(64)
    positions = torch.arange(7, 20, device="cuda")
    fused = torch.randn(13, 6 * 64, device="cuda", requires_grad=True)
    rows = fused.view(13, 6, 64)
    q, k = rotary.apply(rows[:, :4], rows[:, 4:], positions)
    q.sum().backward()
    ones = torch.ones(13, 4, 64, device="cuda")
    want, _ = rotary.apply(ones, None, positions, transpose=True)
    assert torch.equal(fused.grad.view(13, 6, 64)[:, :4], want)
    assert (fused.grad.view(13, 6, 64)[:, 4:] == 0).all()
    x = torch.randn(13, 4, 64, device="cuda", requires_grad=True)
    g = torch.randn(13, 4, 64, device="cuda", requires_grad=True)
    w = torch.randn(13, 4, 64, device="cuda")
    y, _ = rotary.apply(x, None, positions)
    first, = torch.autograd.grad(y, x, g, create_graph=True)
    second, = torch.autograd.grad(first, g, w)
    assert torch.equal(second, rotary.apply(w, None, positions)[0])


def test_difference_quotient(cuda):
    """R is linear: (R(x + d) - R(x - d)) / 2 against the gradient, but for fp32
    rounding of 3328 products of unit size, each within about 1e-6."""
    rotary = Rotary(64, layout="interleaved", scaling=YARN)
    gen = torch.Generator(device="cuda").manual_seed(1)
    x, d, g = (torch.randn(13, 4, 64, generator=gen, device="cuda") for _ in range(3))
    positions = torch.randint(0, 100000, (13,), generator=gen, device="cuda")
    x.requires_grad_()
    grad, = torch.autograd.grad(rotary.apply(x, None, positions)[0], x, g)
    with torch.no_grad():
        plus, _ = rotary.apply(x + d, None, positions)
        minus, _ = rotary.apply(x - d, None, positions)
    change = (g.double() * (plus.double() - minus.double())).sum() / 2
    assert abs(change - (grad.double() * d.double()).sum()) <= 4e-3


def test_in_place_results_and_gradients(cuda):
    """``out`` is refused where a gradient would be lost; a tensor that autograd
    has saved is seen to have changed."""
    rotary = Rotary(64)
    positions = torch.arange(5, device="cuda")
    x = torch.randn(5, 2, 64, device="cuda", requires_grad=True)
    y = torch.empty(5, 2, 64, device="cuda")
    with pytest.raises(ValueError, match="gradient"):
        rotary.apply(x, None, positions, out=(y, None))
    with pytest.raises(ValueError, match="gradient"):
        rotary.apply(y, None, positions, out=(x, None))
    with torch.no_grad():
        rotary.apply(x, None, positions, out=(y, None))
    assert not rotary.apply(x.detach(), None, positions)[0].requires_grad
    w = torch.randn(5, 2, 64, device="cuda", requires_grad=True)
    product = (w * y).sum()                        # saves y
    rotary.apply(y, None, positions, out=(y, None))
    with pytest.raises(RuntimeError, match="inplace"):
        product.backward()
