"""Forward-mode derivatives of lookup_rows and its gradient: both are linear,
so the tangent of the result is the operator on the tangent."""
import pytest
import torch
import torch.autograd.forward_ad as fwad

import sdfoam_b200 as foam

pytestmark = pytest.mark.gpu


def inputs(dtype=torch.float32):
    g = torch.Generator(device="cuda").manual_seed(0)
    ids = torch.randint(-1, 45, (90,), generator=g, device="cuda").to(torch.int32).view(torch.uint32)

    def draw(*shape):
        return torch.randn(shape, generator=g, device="cuda").to(dtype)

    return ids, draw(40, 6), draw(40, 6), draw(90, 6), draw(90, 6)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("reverse", [False, True])
def test_tangents(dtype, reverse):
    """Of plain inputs and of leaves, with gradients on and off."""
    ids, table, table_t, grad, grad_t = inputs(dtype)
    ref = foam.lookup_rows(table, ids, 0.5), foam.lookup_rows(table_t, ids, 0.5)
    back = foam.lookup_rows_backward(grad, ids, 40, 0.5), foam.lookup_rows_backward(grad_t, ids, 40, 0.5)
    for mode in (torch.enable_grad, torch.no_grad):
        with fwad.dual_level(), mode():
            t = fwad.make_dual(table.clone().requires_grad_(reverse), table_t)
            got = fwad.unpack_dual(foam.lookup_rows(t, ids, 0.5))
            assert got.tangent is not None and torch.equal(got.primal, ref[0]) and torch.equal(got.tangent, ref[1])
            g = fwad.make_dual(grad.clone().requires_grad_(reverse), grad_t)
            got = fwad.unpack_dual(foam.lookup_rows_backward(g, ids, 40, 0.5))
            assert got.tangent is not None and torch.equal(got.primal, back[0]) and torch.equal(got.tangent, back[1])
            # no tangent in, none out
            assert fwad.unpack_dual(foam.lookup_rows(table, ids, 0.5)).tangent is None


def test_forward_over_reverse():
    """The tangent of a gradient, and the gradient of a tangent."""
    ids, table, table_t, w, w_t = inputs()
    leaf = table.clone().requires_grad_(True)
    with fwad.dual_level():
        dual = fwad.make_dual(w, w_t)
        (grad,) = torch.autograd.grad((foam.lookup_rows(leaf, ids, 2.0) * dual).sum(), leaf)
        got = fwad.unpack_dual(grad).tangent
        assert got is not None and torch.equal(got, foam.lookup_rows_backward(w_t, ids, 40, 2.0))
    leaf_t = table_t.clone().requires_grad_(True)
    with fwad.dual_level():
        tangent = fwad.unpack_dual(foam.lookup_rows(fwad.make_dual(table, leaf_t), ids, 2.0)).tangent
        (got,) = torch.autograd.grad((tangent * w).sum(), leaf_t)
    assert torch.equal(got, foam.lookup_rows_backward(w, ids, 40, 2.0))
