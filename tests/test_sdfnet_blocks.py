"""SDFNetwork with dtype=torch.float8_e4m3fn: its layers are block_linear."""
import math

import pytest
import torch
import torch.nn.functional as F

import sdfoam_b200 as foam
from sdfoam_b200.sdfnet import SDFNetwork, positional_encoding


def make(device, **kw):
    g = torch.Generator().manual_seed(0)
    return SDFNetwork(dtype=torch.float8_e4m3fn, init="xavier", generator=g, device=device, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("weight_norm", [True, False])
@pytest.mark.parametrize("d_hidden,n_layers,n", [(256, 8, 1000), (320, 3, 129)])
def test_forward_and_gradients_are_the_layers(weight_norm, d_hidden, n_layers, n):
    net = make("cuda", d_hidden=d_hidden, n_layers=n_layers, skip_in=(2,), d_out=1, weight_norm=weight_norm)
    x = torch.rand((n, 3), generator=torch.Generator().manual_seed(1)).cuda() * 2 - 1
    x.requires_grad_(True)
    out = net(x)
    params = dict(net.named_parameters())
    w = torch.randn_like(out)
    got = torch.autograd.grad(out, [x, *params.values()], w)

    # the same layers one by one
    enc = positional_encoding(x, 6).to(torch.bfloat16)
    h = enc
    for l in range(n_layers + 1):
        if l == 2:
            h = torch.cat([h, enc], 1) / math.sqrt(2.0)
        if weight_norm:
            v, g = params[f"lin{l}.weight_v"], params[f"lin{l}.weight_g"]
            weight = v * (g / v.norm(dim=1, keepdim=True))
        else:
            weight = params[f"lin{l}.weight"]
        h = foam.block_linear(h, weight, params[f"lin{l}.bias"])
        if l < n_layers:
            h = F.softplus(h, beta=100)
    ref = h.float()
    assert out.dtype == torch.float32 and torch.equal(out, ref)
    expected = torch.autograd.grad(ref, [x, *params.values()], w)
    for name, a, b in zip(["x", *params], got, expected):
        assert a.dtype == b.dtype and a.isfinite().all() and torch.equal(a, b), name
        assert float(a.abs().sum()) > 0, name


@pytest.mark.gpu
def test_training_steps_run():
    """A training step runs: every parameter gets a gradient of its own type."""
    net = make("cuda", d_hidden=128, n_layers=2, skip_in=())
    opt = torch.optim.Adam(net.parameters(), lr=1e-3)
    x = torch.rand((500, 3), device="cuda")
    for _ in range(3):
        opt.zero_grad()
        net.sdf(x).square().mean().backward()
        opt.step()
    assert all(p.dtype == torch.float32 and p.grad.isfinite().all() for p in net.parameters())


def test_no_second_derivative():
    net = make("cpu", d_hidden=32, n_layers=2, skip_in=())
    assert all(p.dtype == torch.float32 for p in net.parameters())
    with pytest.raises(RuntimeError, match="second derivative"):
        net.gradient(torch.rand((4, 3)))
    with pytest.raises(RuntimeError, match="CUDA"):
        net(torch.rand((4, 3)))
