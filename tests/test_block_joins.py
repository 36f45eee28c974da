"""Products of narrow tiles over long reductions: more slices than a cluster
joins, so a second launch adds them."""
import pytest
import torch

import sdfoam_b200 as foam

EPS = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
E4M3 = torch.float8_e4m3fn


def blocks(n):
    return -(-n // 128)


def widen(scales, rows, columns):
    per = 1 if scales.shape[0] == rows else 128
    return scales.double().repeat_interleave(per, 0)[:rows].repeat_interleave(128, 1)[:, :columns]


def operand(g, rows, k, per):
    x = torch.randn((rows, k), generator=g, device="cuda") * torch.exp2(
        torch.randint(-8, 7, (rows, k), generator=g, device="cuda").float())
    v = torch.zeros((rows, -(-k // 16) * 16), dtype=torch.uint8, device="cuda")
    v[:, :k] = x.clamp(-448, 448).to(E4M3).view(torch.uint8)
    s = torch.exp(torch.randn((rows if per == 1 else blocks(rows), blocks(k)), generator=g, device="cuda")) / 300
    return v[:, :k].view(E4M3), s


def check(got, ref, mag, k, dtype):
    """As in every product: 4 MMA steps of 33 terms a block, each off by at
    most a unit of 2^-23 of the magnitudes, two roundings a block for the
    scales, at most 148 slices and a bias; one rounding to the output type."""
    tol = EPS[dtype] * ref.abs() + (4 * 33 * 2 + 2 * blocks(k) + 148 + 4) * 2.0 ** -24 * mag
    if dtype == torch.float16:
        tol = tol + 2.0 ** -25
    assert got.shape == ref.shape and got.dtype == dtype
    assert ((got.double() - ref).abs() <= tol).all()


@pytest.mark.gpu
@pytest.mark.parametrize("k", [16384, 16385, 24000, 40001])
@pytest.mark.parametrize("narrow,wide", [(1, 300), (16, 200), (17, 129), (31, 1000), (49, 256), (64, 257), (64, 64)])
def test_long_reductions(narrow, wide, k):
    g = torch.Generator(device="cuda").manual_seed(narrow + k)
    for m, n in {(narrow, wide), (wide, narrow)}:
        for a_rows, b_rows in ((1, 128), (128, 1)):
            a, a_scales = operand(g, m, k, a_rows)
            b, b_scales = operand(g, n, k, b_rows)
            x, y = a.float().double() * widen(a_scales, m, k), b.float().double() * widen(b_scales, n, k)
            ref, mag = x @ y.t(), x.abs() @ y.abs().t()
            bias = torch.randn(n, generator=g, device="cuda")
            f = 2.0 ** -14  # into the range of a half
            for dtype, s in ((torch.float32, 1.0), (torch.bfloat16, 1.0), (torch.float16, f)):
                check(foam.block_matmul(a, a_scales * s, b, b_scales, out_dtype=dtype), ref * s, mag * s, k, dtype)
                got = foam.block_matmul(a, a_scales * s, b, b_scales, bias.to(dtype), dtype)
                shift = bias.to(dtype).double()
                check(got, ref * s + shift, mag * s + shift.abs(), k, dtype)
                assert torch.equal(got, foam.block_matmul(a, a_scales * s, b, b_scales, bias.to(dtype), dtype))
    foam.check_block_flags()


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", [(20000, 256, 49), (20000, 49, 256), (17000, 3, 64), (33001, 64, 16)])
def test_weight_gradient_of_a_narrow_layer(m, n, k):
    """Many rows, one width of at most 64: the weight's gradient is such a product."""
    g = torch.Generator(device="cuda").manual_seed(m + n)
    x = torch.randn((m, k), generator=g, device="cuda").to(torch.bfloat16).requires_grad_(True)
    w = (torch.randn((n, k), generator=g, device="cuda") / k ** 0.5).requires_grad_(True)
    bias = torch.randn(n, generator=g, device="cuda").requires_grad_(True)
    dy = torch.randn((m, n), generator=g, device="cuda").to(torch.bfloat16)
    foam.block_linear(x, w, bias).backward(dy)
    with torch.no_grad():
        gt, xt = (v.float().double() * widen(s, *v.shape)
                  for v, s in (foam.quantize_blocks(dy, transpose=True), foam.quantize_blocks(x, transpose=True)))
        check(w.grad, gt @ xt.t(), gt.abs() @ xt.abs().t(), m, torch.float32)
        total, mag = dy.double().sum(0), dy.double().abs().sum(0)
        assert ((bias.grad.double() - total).abs() <= 2.0 ** -24 * total.abs() + m * 2.0 ** -24 * mag).all()
