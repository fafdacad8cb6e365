"""Calls of stattn.ops as torch programs make them: inside a graph of gradients, on views that torch keeps lazily."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module")
def ops():
    from stattn import ops
    return ops


@pytest.mark.parametrize("m", [3, 100])
def test_a_backward_pass_through_a_product_fails(ops, m):
    """No gradient exists: y carries the record of x and bias, so that a backward pass raises instead of leaving them out; the values
    are those of the call without a record."""
    x = torch.randn(m, 400, device=DEV)
    w = ops.mx4_quantize(torch.randn(50, 400, device=DEV))
    bias = torch.randn(50, device=DEV)
    want, q = ops.mx4_linear(x, w, bias=bias), ops.mx4_quantize(x)
    assert not want.requires_grad
    for rx, rb in ((True, False), (False, True), (True, True)):
        gx, gb = x.clone().requires_grad_(rx), bias.clone().requires_grad_(rb)
        y = ops.mx4_linear(gx, w, bias=gb)
        assert torch.equal(y.detach(), want)
        with pytest.raises(RuntimeError, match="mx4_linear has no gradient"):
            (y * 2).sum().backward()
        with torch.no_grad():
            assert not ops.mx4_linear(gx, w, bias=gb).requires_grad
        if rb:
            z = ops.mx4_matmul(q, w, bias=gb)
            assert torch.equal(z.detach(), ops.mx4_matmul(q, w, bias=bias))
            with pytest.raises(RuntimeError, match="mx4_matmul has no gradient"):
                z.sum().backward()
        assert gx.grad is None and gb.grad is None
    assert not ops.mx4_linear(x.requires_grad_(), w).detach().requires_grad


def test_a_forward_mode_tangent_is_refused(ops):
    from torch.autograd import forward_ad
    x = torch.randn(3, 64, device=DEV)
    w, bias = ops.mx4_quantize(torch.randn(5, 64, device=DEV)), torch.randn(5, device=DEV)
    q = ops.mx4_quantize(x)
    with forward_ad.dual_level():
        want = ops.mx4_linear(x, w, bias=bias)                              # a level is open, none of these is on it
        with pytest.raises(RuntimeError, match="mx4_linear has no derivative"):
            ops.mx4_linear(forward_ad.make_dual(x, torch.ones_like(x)), w)
        dual = forward_ad.make_dual(bias, torch.ones_like(bias))
        with pytest.raises(RuntimeError, match="mx4_linear has no derivative"):
            ops.mx4_linear(x, w, bias=dual)
        with pytest.raises(RuntimeError, match="mx4_matmul has no derivative"):
            ops.mx4_matmul(q, w, bias=dual)
    assert torch.equal(ops.mx4_linear(x, w, bias=bias), want)
