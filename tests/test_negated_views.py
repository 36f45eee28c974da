"""Views that negate as they are read: the imaginary part of a conjugate."""
import pytest
import torch

import sdfoam_b200 as foam

pytestmark = pytest.mark.gpu


def negated(*shape):
    """(a float32 view with the negative bit, its values written out)"""
    g = torch.Generator(device="cuda").manual_seed(0)
    view = torch.randn(shape, generator=g, dtype=torch.complex64, device="cuda").conj().imag
    assert view.is_neg()
    return view, view.resolve_neg().contiguous()


@pytest.mark.parametrize("shape", [(40,), (40, 7)])
def test_rows(shape):
    view, plain = (t if len(shape) == 2 else t[:, None] for t in negated(*shape))
    ids = torch.arange(39, -1, -1, device="cuda")
    assert torch.equal(foam.lookup_rows(view, ids), plain[ids])
    assert torch.equal(foam.lookup_rows_backward(view, ids, 40), plain[ids])


@pytest.mark.parametrize("shape", [(40,), (40, 7)])
def test_blocks(shape):
    view, plain = (t if len(shape) == 2 else t[:, None] for t in negated(*shape))
    for a, b in zip(foam.quantize_blocks(view), foam.quantize_blocks(plain)):
        assert torch.equal(a.float(), b.float())
    w, w_plain = negated(5, plain.shape[1])
    bias, bias_plain = negated(5)
    ref = foam.block_linear(plain, w_plain, bias_plain)
    assert torch.equal(foam.block_linear(view, w, bias), ref)
    # a vector of one element is contiguous as it is
    one, one_plain = negated(1)
    v, s = foam.quantize_blocks(plain)
    assert torch.equal(foam.block_matmul(v, s, v[:1], s[:1], one), foam.block_matmul(v, s, v[:1], s[:1], one_plain))
    # and as a gradient
    x = plain.clone().requires_grad_(True)
    wl = w_plain[:1].clone().requires_grad_(True)
    dy, dy_plain = (t[:, None] for t in negated(40))
    got = torch.autograd.grad(foam.block_linear(x, wl), (x, wl), dy)
    assert all(torch.equal(p, q) for p, q in zip(got, torch.autograd.grad(foam.block_linear(x, wl), (x, wl), dy_plain)))
