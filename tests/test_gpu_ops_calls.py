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
    y = ops.mx4_linear(x, w, bias=bias)                                     # x records a gradient; y may be written in place all the same
    assert y.requires_grad and not y._is_view()
    assert torch.equal(y.mul_(2).detach(), 2 * want)
    with pytest.raises(RuntimeError, match="mx4_linear has no gradient"):
        y.sum().backward()


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


def lazy(t):
    """The same numbers, their sign kept beside the memory."""
    v = torch._neg_view(-t)
    assert v.is_neg() and torch.equal(v, t)
    return v


def test_views_whose_sign_is_kept_beside_the_memory(ops):
    z = torch.randn(40, 70, 2, device=DEV)
    v = torch.view_as_complex(z).conj().imag                               # column stride 2
    assert v.is_neg()
    for axis in (0, 1):
        got, want = ops.mx4_quantize(v, axis=axis), ops.mx4_quantize(-z[:, :, 1], axis=axis)
        assert torch.equal(got.codes, want.codes) and torch.equal(got.scales, want.scales)
    x, bias = torch.randn(40, 70, device=DEV), torch.randn(30, device=DEV)
    w = ops.mx4_quantize(torch.randn(30, 70, device=DEV))
    want, q = ops.mx4_linear(x, w, bias=bias), ops.mx4_quantize(x)
    assert torch.equal(ops.mx4_linear(lazy(x), w, bias=bias), want) and torch.equal(ops.mx4_linear(x, w, bias=lazy(bias)), want)
    assert torch.equal(ops.mx4_linear(lazy(x)[3:, :], w, bias=bias), want[3:])
    assert torch.equal(ops.mx4_matmul(q, w, bias=lazy(bias)), ops.mx4_matmul(q, w, bias=bias))
    g = torch.Generator().manual_seed(1)
    t, p = (torch.softmax(3 * torch.randn(6, 3, 90, generator=g), 2).to(DEV) for _ in range(2))
    args = [torch.randint(0, 90, (6, 2), generator=g).to(DEV), t, p[:, :2].contiguous(), torch.rand(6, 2, generator=g).to(DEV), torch.rand(6, generator=g).to(DEV)]
    want = ops.verify_draft(*args)
    for i in range(1, 5):
        got = ops.verify_draft(*args[:i], lazy(args[i]), *args[i + 1:])
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), i
