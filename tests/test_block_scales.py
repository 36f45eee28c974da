"""Products whose scales are far from one: the product of the two scales may
leave fp32 where the scaled sum does not."""
import pytest
import torch

import sdfoam_b200 as foam

E4M3 = torch.float8_e4m3fn


def blocks(n):
    return -(-n // 128)


def widen(scales, rows, columns):
    per = 1 if scales.shape[0] == rows else 128
    return scales.double().repeat_interleave(per, 0)[:rows].repeat_interleave(128, 1)[:, :columns]


def rows16(x):
    """x in e4m3, rows 16 bytes aligned."""
    v = torch.zeros((x.shape[0], -(-x.shape[1] // 16) * 16), dtype=torch.uint8, device=x.device)
    v[:, :x.shape[1]] = x.to(E4M3).view(torch.uint8)
    return v[:, :x.shape[1]].view(E4M3)


# every tile shape: the narrow ones in both orientations, one CTA, pairs, and
# reductions that are cut into slices
SIZES = [(3, 200, 300), (40, 200, 300), (200, 5, 300), (200, 30, 300), (200, 60, 300), (200, 100, 300), (19100, 250, 257),
         (1, 300, 16700), (2, 300, 16700)]


@pytest.mark.gpu
@pytest.mark.parametrize("a_rows,b_rows", [(1, 128), (1, 1), (128, 128), (128, 1)])
@pytest.mark.parametrize("exponent", [-150, -140, -127, 128, 131, 140])
@pytest.mark.parametrize("m,n,k", SIZES)
def test_product_of_scales_past_fp32(m, n, k, exponent, a_rows, b_rows):
    """Scales of 2^exponent together in every block but the first, whose are
    ordinary.  Large ones meet e4m3's smallest values in few places, small ones
    its largest (and a first block of zeros, whose sums would hide theirs); one
    row of a and one of b are zeros."""
    g = torch.Generator(device="cuda").manual_seed(m + n + exponent)

    def values(rows):
        if exponent > 0:
            x = torch.zeros((rows, k), device="cuda")
            at = torch.randint(0, k, (rows, 8), generator=g, device="cuda")
            return rows16(x.scatter_(1, at, 2.0 ** -9 * torch.randint(-1, 2, (rows, 8), generator=g, device="cuda").float()))
        return rows16(torch.randint(-448, 449, (rows, k), generator=g, device="cuda").float())

    def scales(rows, per, e):
        s = 1 + torch.rand((rows if per == 1 else blocks(rows), blocks(k)), generator=g, device="cuda")
        s[:, 1:] *= 2.0 ** e
        return s

    a, b = values(m), values(n)
    if exponent < 0:
        a.view(torch.uint8)[:, :128] = 0
    a.view(torch.uint8)[m // 2] = 0
    b.view(torch.uint8)[n // 2] = 0
    a_scales, b_scales = scales(m, a_rows, exponent // 2), scales(n, b_rows, exponent - exponent // 2)
    x, y = a.float().double() * widen(a_scales, m, k), b.float().double() * widen(b_scales, n, k)
    ref, mag = x @ y.t(), x.abs() @ y.abs().t()
    assert float(mag.max()) < 2.0 ** 127
    got = foam.block_matmul(a, a_scales, b, b_scales, out_dtype=torch.float32).double()
    # as for ordinary scales (an MMA step adds 33 terms, each off by at most a
    # unit of 2^-23 of the magnitudes, four steps a block; per block a rounding
    # of the scales' product and one of the sum; the joins of at most 148
    # slices), and half a smallest step for each rounding near zero
    adds = 4 * 33 * 2 + 2 * blocks(k) + 3 + 148
    tol = (adds + 1) * 2.0 ** -24 * mag + (2 * blocks(k) + 149) * 2.0 ** -150
    assert ((got - ref).abs() <= tol).all()
    assert (got[m // 2] == 0).all() and (got[:, n // 2] == 0).all()
    out = foam.block_matmul(a, a_scales, b, b_scales)
    # the same sums, rounded to 8 bits
    assert torch.equal(out, got.float().to(torch.bfloat16))
    foam.check_block_flags()


@pytest.mark.gpu
@pytest.mark.parametrize("a_rows,b_rows", [(1, 128), (1, 1), (128, 128), (128, 1)])
@pytest.mark.parametrize("ea,eb", [(101, -101), (-108, 107), (110, -112), (-112, 110), (120, -126), (-126, 119), (126, -140),
                                   (-149, 126)])
@pytest.mark.parametrize("m,n,k", SIZES)
def test_scales_that_cancel(m, n, k, ea, eb, a_rows, b_rows):
    """One scale so large or small that it leaves fp32 with a block's sum, the
    other bringing it back; beside columns and rows of ordinary scales, which
    give the same bits whatever stands beside them."""
    g = torch.Generator(device="cuda").manual_seed(m + n + ea)
    a, b = (rows16(torch.randint(-448, 449, (rows, k), generator=g, device="cuda").float()) for rows in (m, n))

    def scales(rows, per, e):
        s = 1 + torch.rand((rows if per == 1 else blocks(rows), blocks(k)), generator=g, device="cuda")
        far = s.clone()
        far[::3] *= 2.0 ** e
        return s, far

    (sa, far_a), (sb, far_b) = scales(m, a_rows, ea), scales(n, b_rows, eb)
    got = foam.block_matmul(a, far_a, b, far_b, out_dtype=torch.float32).double()
    x, y = a.float().double() * widen(far_a, m, k), b.float().double() * widen(far_b, n, k)
    ref, mag = x @ y.t(), x.abs() @ y.abs().t()
    tol = (4 * 33 * 2 + 2 * blocks(k) + 3 + 148 + 1) * 2.0 ** -24 * mag + (2 * blocks(k) + 149) * 2.0 ** -150
    inside = mag < 2.0 ** 127
    assert inside.any() and ((got - ref).abs() <= tol)[inside].all()
    # rows and columns whose scales are ordinary on both sides
    row = torch.arange(m, device="cuda") // a_rows % 3 != 0
    column = torch.arange(n, device="cuda") // b_rows % 3 != 0
    plain = foam.block_matmul(a, sa, b, sb, out_dtype=torch.float32).double()
    assert torch.equal(got[row][:, column], plain[row][:, column])


@pytest.mark.gpu
@pytest.mark.parametrize("m,n", [(3, 200), (200, 100), (19100, 250)])
def test_scales_of_zero_infinity_and_nan(m, n):
    """As the formula has them: zero rows, infinities and NaN in the rows whose
    scale they are."""
    a = torch.full((m, 256), 2.0, device="cuda").to(E4M3)
    b = torch.full((n, 256), 0.5, device="cuda").to(E4M3)
    sa, sb = torch.ones((m, 2), device="cuda"), torch.ones((n, 2), device="cuda")
    sa[0], sa[1, 1], sa[2, 0] = 0.0, float("inf"), float("nan")
    for per in (sb, sb[:blocks(n)]):
        got = foam.block_matmul(a, sa, b, per, out_dtype=torch.float32)
        assert (got[0] == 0).all() and (got[1] == float("inf")).all() and got[2].isnan().all()
        assert (got[3:] == 256).all()


@pytest.mark.gpu
def test_layer_of_tiny_values():
    """Rows around 2^-112 through weights around 2^-24: the layer's own scales
    multiply to 2^-151 and less, its sums are normal numbers."""
    g = torch.Generator(device="cuda").manual_seed(1)
    x = (1 + torch.rand((300, 256), generator=g, device="cuda")) * 2.0 ** -112
    w = (1 + torch.rand((64, 256), generator=g, device="cuda")) * 2.0 ** -24
    qx, qw = (v.float().double() * widen(s, *v.shape) for v, s in (foam.quantize_blocks(x), foam.quantize_blocks(w, 128)))
    ref, mag = qx @ qw.t(), qx.abs() @ qw.abs().t()
    got = foam.block_linear(x, w).double()
    assert ((got - ref).abs() <= (4 * 33 * 2 + 2 * 2 + 3 + 148 + 1) * 2.0 ** -24 * mag + (4 + 149) * 2.0 ** -150).all()
