"""The 8-bit operators (quantize_blocks, dequantize_blocks, block_matmul,
block_linear) against their definitions in 64 bits."""
import ctypes
import math

import pytest
import torch

import sdfoam_b200 as foam
from sdfoam_b200 import _lib

EPS = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
E4M3 = torch.float8_e4m3fn


def blocks(n):
    return -(-n // 128)


def widen(scales, rows, columns):
    """A scale for each element, in 64 bits."""
    per = 1 if scales.shape[0] == rows else 128
    return scales.double().repeat_interleave(per, 0)[:rows].repeat_interleave(128, 1)[:, :columns]


def largest(x, block_rows):
    """Largest finite magnitude of each block, in 64 bits."""
    m, k = x.shape
    a = torch.where(x.isfinite(), x.double().abs(), 0.0)
    p = torch.zeros((blocks(m) * 128 if block_rows == 128 else m, blocks(k) * 128), dtype=torch.float64, device=x.device)
    p[:m, :k] = a
    return p.view(p.shape[0] // block_rows, block_rows, blocks(k), 128).amax(dim=(1, 3))


def check_quantized(x, values, scales, block_rows):
    m, k = x.shape
    top = largest(x, block_rows)
    s = scales.double()
    assert values.shape == x.shape and values.dtype == E4M3 and scales.shape == top.shape
    assert torch.equal(torch.frexp(s).mantissa, torch.full_like(s, 0.5)), "a power of two"
    zero = top == 0
    assert (s[zero] == 1).all()
    s, t = s[~zero], top[~zero]
    assert (s * 448 >= t).all() and (s >= 2.0 ** -126).all()
    assert ((s / 2 * 448 < t) | (s == 2.0 ** -126)).all(), "the smallest one"
    fine = x.isfinite()
    ref = torch.where(fine, x.double() / widen(scales, m, k), float("nan"))  # exact: a power of two
    # to float32 first: exact too, unless the quotient is far below e4m3's smallest step
    ref = ref.float().to(E4M3).float()
    got = values.float()
    assert torch.equal(got.isnan(), ref.isnan())
    assert torch.equal(got[fine], ref[fine])


def product64(a, a_scales, b, b_scales):
    """(product, sum of magnitudes) in 64 bits."""
    x = a.float().double() * widen(a_scales, *a.shape)
    y = b.float().double() * widen(b_scales, *b.shape)
    return x @ y.t(), x.abs() @ y.abs().t()


def check_product(got, ref, mag, k, dtype):
    """One rounding to the output type; the products of e4m3 values are exact
    in fp32; an MMA step adds 32 of them and the sum so far, each of the 33
    terms off by at most a unit of 2^-23 of the sum of magnitudes even if the
    tensor cores truncate, four steps a block; then one multiply-add (and the
    scales' product) per block, the joins of at most 148 slices and a bias."""
    tol = EPS[dtype] * ref.abs() + (4 * 33 * 2 + blocks(k) + 3 + 148 + 1) * 2.0 ** -24 * mag
    if dtype == torch.float16:
        tol = tol + 2.0 ** -25
    assert got.shape == ref.shape and got.dtype == dtype
    off = (got.double() - ref).abs() - tol
    assert (off <= 0).all(), (off.max().item(), int((off > 0).sum()))


def operand(g, m, k, block_rows, device="cuda"):
    """Values over e4m3's whole range of magnitudes, scales of any size."""
    x = torch.randn((m, k), generator=g, device=device) * torch.exp2(
        torch.randint(-8, 7, (m, k), generator=g, device=device).float())
    rows = m if block_rows == 1 else blocks(m)
    s = torch.exp(2 * torch.randn((rows, blocks(k)), generator=g, device=device)) / 300
    v = torch.zeros((m, (k + 15) // 16 * 16), dtype=torch.uint8, device=device)
    v[:, :k] = x.clamp(-448, 448).to(E4M3).view(torch.uint8)
    return v[:, :k].view(E4M3), s


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("transpose", [False, True])
def test_quantize(dtype, block_rows, transpose):
    g = torch.Generator(device="cuda").manual_seed(1)
    for m, k in ((1, 1), (1, 4096), (3, 39), (128, 128), (130, 217), (257, 256), (1000, 49), (16, 129), (129, 16)):
        x = torch.randn((m, k), generator=g, device="cuda") * torch.exp(3 * torch.randn((m, k), generator=g, device="cuda"))
        x = x.to(dtype)
        x[m // 2] = 0  # a row of zeros
        values, scales = foam.quantize_blocks(x, block_rows, transpose)
        src = x.t() if transpose else x
        check_quantized(src, values, scales, block_rows)
        for out in (torch.float32, torch.bfloat16, torch.float16):
            back = foam.dequantize_blocks(values, scales, out)
            ref = (values.float().double() * widen(scales, *values.shape)).to(out)
            # a half beyond its range is an infinity, quantized to NaN
            assert torch.allclose(back, ref, rtol=0, atol=0, equal_nan=True)
        wide = torch.zeros((m, k + 5), dtype=dtype, device="cuda")
        wide[:, 3:3 + k] = x  # rows that no vector load may assume aligned
        for y in (wide[:, 3:3 + k], x.t().contiguous().t()):
            v, s = foam.quantize_blocks(y, block_rows, transpose)
            assert torch.equal(v.view(torch.uint8), values.view(torch.uint8)) and torch.equal(s, scales)


@pytest.mark.gpu
@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_dequantize_rows(dtype, block_rows):
    """Rows of any width, distance and start, scales of any order, and an
    output that starts at any element, with a frame that stays as it was."""
    g = torch.Generator(device="cuda").manual_seed(12)
    lib = _lib.load()
    for m, k in ((1, 1), (9000, 1), (3000, 3), (700, 5), (513, 8), (130, 217), (100, 124), (333, 132), (2, 20000), (300, 130)):
        scales = torch.randn((m if block_rows == 1 else blocks(m), blocks(k)), generator=g, device="cuda")
        for start, ld in ((0, -(-k // 16) * 16), (0, k + 5), (3, k + 16), (4, -(-k // 4) * 4 + 4), (8, -(-k // 8) * 8 + 8)):
            store = torch.randint(0, 256, (start + m * ld,), generator=g, device="cuda").to(torch.uint8)
            values = store.view(E4M3)[start:].view(m, ld)[:, :k]
            # a product of 4 and 24 significant bits: exact in 64, rounded once
            # to 32 and once to the output as the definition has it
            ref = (values.double() * widen(scales, m, k)).float().to(dtype)
            for s in (scales, scales.t().contiguous().t()):
                assert torch.allclose(foam.dequantize_blocks(values, s, dtype), ref, rtol=0, atol=0, equal_nan=True)
            frame = torch.full((m * k + 9,), 7, dtype=dtype, device="cuda")
            torch.cuda.synchronize()
            assert lib.sdfoam_block_dequantize(values.data_ptr(), ld, scales.data_ptr(), *scales.stride(), block_rows, m, k,
                                               {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}[dtype],
                                               frame[1:].data_ptr(), _lib.stream(frame.device)) == 0
            assert torch.allclose(frame[1:1 + m * k].view(m, k), ref, rtol=0, atol=0, equal_nan=True)
            assert frame[0] == 7 and (frame[1 + m * k:] == 7).all()


@pytest.mark.gpu
@pytest.mark.parametrize("block_rows", [1, 128])
def test_quantize_edges(block_rows):
    """Infinities, NaN, the smallest and largest numbers, ties, borders of the scale."""
    tiny = 2.0 ** -149
    rows = [[1.75 * 2.0 ** e] + [0.0] * 3 for e in (-140, -126, -118, -117, 0, 8, 127)]
    rows += [[1.75 * 2.0 ** e * (1 + 2.0 ** -22)] + [2.0 ** (e - 3)] * 3 for e in (-100, 0, 100)]
    rows += [[float("inf"), 1.0, -2.0, 448.0], [float("nan"), -float("inf"), float("nan"), float("inf")],
             [float("nan"), 0.0, -0.0, 3.0], [tiny, -tiny, 0.0, 3 * tiny], [3.4028235e38, 1.0, -3.4e38, 2.0 ** 120]]
    # halves between neighbours: 17/16 of a step up and down, subnormals
    rows += [[448.0, 17.0, 19.0, 2.0 ** -10], [448.0, 3 * 2.0 ** -10, 432.0, -416.0], [256.0, 1.0625, 1.1875, 464.0]]
    x = torch.tensor(rows, device="cuda")
    if block_rows == 128:
        x = torch.nn.functional.pad(x, (0, 124))  # one block of columns; rows share a scale: one row at a time
        for r in x:
            check_quantized(r[None], *foam.quantize_blocks(r[None], 128), 128)
            check_quantized(r[None].t(), *foam.quantize_blocks(r[None], 128, True), 128)
    else:
        check_quantized(x, *foam.quantize_blocks(x), 1)
        check_quantized(x.t(), *foam.quantize_blocks(x, 1, True), 1)


SIZES = [(1, 1, 1), (1, 128, 128), (1, 4096, 4096), (2, 217, 39), (7, 300, 1000), (16, 256, 256), (17, 129, 130),
         (33, 1000, 257), (64, 65, 127), (64, 64, 64), (65, 64, 128), (100, 100, 100), (128, 256, 384), (129, 257, 513),
         (300, 1, 500), (1000, 16, 256), (1000, 31, 47), (1500, 64, 2000), (2000, 217, 256), (777, 1111, 333),
         (256, 256, 20001), (5000, 3000, 128), (20000, 512, 300), (20001, 217, 300), (19100, 250, 129),
         (40000, 100, 256), (40001, 63, 257)]


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", SIZES)
def test_product(m, n, k):
    g = torch.Generator(device="cuda").manual_seed(m + n + k)
    for a_rows, b_rows in ((1, 128), (1, 1), (128, 128), (128, 1)):
        a, a_scales = operand(g, m, k, a_rows)
        b, b_scales = operand(g, n, k, b_rows)
        ref, mag = product64(a, a_scales, b, b_scales)
        bias = torch.randn(n, generator=g, device="cuda")
        for dtype in (torch.float32, torch.bfloat16, torch.float16):
            if dtype == torch.float16:  # its range is narrow: smaller scales
                f = 2.0 ** -math.ceil(math.log2(max(1.0, mag.max().item() / 3e4)))
                got = foam.block_matmul(a, a_scales * f, b, b_scales, None, dtype)
                check_product(got, ref * f, mag * f, k, dtype)
                continue
            check_product(foam.block_matmul(a, a_scales, b, b_scales, out_dtype=dtype), ref, mag, k, dtype)
            got = foam.block_matmul(a, a_scales, b, b_scales, bias.to(dtype), dtype)
            shift = bias.to(dtype).double()
            check_product(got, ref + shift, mag + shift.abs(), k, dtype)
            assert torch.equal(got, foam.block_matmul(a, a_scales, b, b_scales, bias.to(dtype), dtype))
    foam.check_block_flags()


@pytest.mark.gpu
def test_product_strides_and_empty():
    g = torch.Generator(device="cuda").manual_seed(5)
    a, a_scales = operand(g, 200, 256, 1)
    b, b_scales = operand(g, 300, 256, 128)
    ref = foam.block_matmul(a, a_scales, b, b_scales)
    wide = torch.zeros((200, 273), dtype=torch.uint8, device="cuda")
    wide[:, 1:257] = a.view(torch.uint8)
    for other in (wide[:, 1:257].view(E4M3), a.t().contiguous().t()):
        assert torch.equal(foam.block_matmul(other, a_scales, b, b_scales), ref)
    assert torch.equal(foam.block_matmul(a, a_scales.t().contiguous().t(), b, b_scales), ref)
    pad = torch.zeros((300, 512), dtype=torch.uint8, device="cuda")
    pad[:, 256:] = b.view(torch.uint8)
    assert torch.equal(foam.block_matmul(a, a_scales, pad[:, 256:].view(E4M3), b_scales), ref)
    bias = torch.randn(600, generator=g, device="cuda")[::2]
    check_product(foam.block_matmul(a, a_scales, b, b_scales, bias, torch.float32),
                  *(t + s for t, s in zip(product64(a, a_scales, b, b_scales), (bias.double(), bias.double().abs()))),
                  256, torch.float32)
    # no rows, no columns, nothing to sum over
    assert foam.block_matmul(a[:0], a_scales[:0], b, b_scales).shape == (0, 300)
    assert foam.block_matmul(a, a_scales, b[:0], b_scales[:0]).shape == (200, 0)
    got = foam.block_matmul(a[:, :0], a_scales[:, :0], b[:, :0], b_scales[:, :0], bias, torch.float32)
    assert torch.equal(got, bias.expand(200, 300))
    assert (foam.block_matmul(a[:, :0], a_scales[:, :0], b[:, :0], b_scales[:, :0]) == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("m,n", [(3, 200), (200, 200), (200, 5)])
def test_nan_stays_in_its_row(m, n):
    g = torch.Generator(device="cuda").manual_seed(6)
    x = torch.randn((m, 300), generator=g, device="cuda")
    w = torch.randn((n, 300), generator=g, device="cuda")
    clean = foam.block_matmul(*foam.quantize_blocks(x), *foam.quantize_blocks(w, 128))
    x[1, 7] = float("inf")
    got = foam.block_matmul(*foam.quantize_blocks(x), *foam.quantize_blocks(w, 128))
    assert got[1].isnan().all()
    keep = torch.arange(m, device="cuda") != 1
    assert torch.equal(got[keep], clean[keep])


@pytest.mark.gpu
def test_offsets_past_32_bits():
    m = (1 << 25) + 5
    a = torch.zeros((m, 128), dtype=torch.uint8, device="cuda").view(E4M3)
    a[-3:] = 1.0
    b = torch.ones((16, 128), device="cuda").to(E4M3)
    a_scales = torch.ones((m, 1), device="cuda")
    got = foam.block_matmul(a, a_scales, b, torch.ones((16, 1), device="cuda"))
    assert (got[-3:] == 128).all() and float(got.float().sum()) == 3 * 16 * 128
    del a, got
    x = torch.zeros((m, 128), dtype=torch.bfloat16, device="cuda")
    x[-1] = 2.0
    values, scales = foam.quantize_blocks(x)
    assert float(values[-1].float().sum()) * float(scales[-1]) == 256 and float(scales[0]) == 1.0
    assert (foam.dequantize_blocks(values, scales, torch.bfloat16)[-1] == 2).all()


def formula64(x, w, dy):
    """y, dx, dw of block_linear in 64 bits with their sums of magnitudes,
    from the values that the definition's quantizer (tested above) keeps."""
    q = lambda t, rows, turn=False: (lambda v, s: v.float().double() * widen(s, *v.shape))(
        *foam.quantize_blocks(t, rows, turn))
    qx, qw, qg, qgt, qxt = q(x, 1), q(w, 128), q(dy, 1), q(dy, 1, True), q(x, 1, True)
    return [(p @ r.t(), p.abs() @ r.abs().t()) for p, r in ((qx, qw), (qg, qw.t()), (qgt, qxt))]


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (5, 217, 39), (130, 256, 256), (1000, 64, 300), (4099, 300, 129)])
@pytest.mark.parametrize("dtype,wtype", [(torch.bfloat16, torch.float32), (torch.float32, torch.float32),
                                         (torch.float16, torch.bfloat16)])
def test_linear(m, n, k, dtype, wtype):
    g = torch.Generator(device="cuda").manual_seed(m + n)
    x = torch.randn((m, k), generator=g, device="cuda").to(dtype).requires_grad_(True)
    w = (torch.randn((n, k), generator=g, device="cuda") / math.sqrt(k)).to(wtype).requires_grad_(True)
    bias = torch.randn(n, generator=g, device="cuda").to(wtype).requires_grad_(True)
    dy = torch.randn((m, n), generator=g, device="cuda").to(dtype)
    y = foam.block_linear(x, w, bias)
    y.backward(dy)
    with torch.no_grad():
        (ry, my), (rx, mx), (rw, mw) = formula64(x, w, dy)
        b = bias.double()
        check_product(y, ry + b, my + b.abs(), k, dtype)
        check_product(x.grad, rx, mx, n, dtype)
        check_product(w.grad, rw, mw, m, wtype)
        rb, mb = dy.double().sum(0), dy.double().abs().sum(0)
        assert ((bias.grad.double() - rb).abs() <= EPS[wtype] * rb.abs() + m * 2.0 ** -24 * mb).all()
        # differences of the layer without rounding: linear, so its gradient
        # is dy w; e4m3 is off by half a step of 2^-3 relative, or of 2^-9 of
        # the scale, which is at most the block's largest / 224
        def slack(t, rows):
            s = foam.quantize_blocks(t, rows)[1]
            return t.double().abs() * 2.0 ** -4 + 2.0 ** -10 * widen(s, *t.shape)
        gd, wd = dy.double(), w.double()
        off = (gd.abs() + slack(dy, 1)) @ (wd.abs() + slack(w, 128)) - gd.abs() @ wd.abs()
        d = torch.randn((m, k), generator=g, device="cuda", dtype=torch.float64)
        diff = (((x.double() + d) @ wd.t() - x.double() @ wd.t()) * gd).sum()
        assert abs(diff - (x.grad.double() * d).sum()) <= ((off + EPS[dtype] * rx.abs() + 2.0 ** -14 * mx) * d.abs()).sum() + 1e-9


@pytest.mark.gpu
def test_linear_shapes_and_parts():
    g = torch.Generator(device="cuda").manual_seed(9)
    x = torch.randn((3, 5, 70), generator=g, device="cuda", requires_grad=True)
    w = torch.randn((40, 70), generator=g, device="cuda", requires_grad=True)
    y = foam.block_linear(x, w)
    assert y.shape == (3, 5, 40)
    flat = foam.block_linear(x.detach().reshape(15, 70), w.detach())
    assert torch.equal(y.reshape(15, 40), flat) and not flat.requires_grad
    dy = torch.randn((3, 5, 40), generator=g, device="cuda")
    gx, gw = torch.autograd.grad(foam.block_linear(x, w), (x, w), dy)
    # each gradient alone; a gradient that is broadcast; a one-dimensional x
    assert torch.equal(torch.autograd.grad(foam.block_linear(x, w.detach()), x, dy)[0], gx)
    assert torch.equal(torch.autograd.grad(foam.block_linear(x.detach(), w), w, dy)[0], gw)
    one = torch.autograd.grad(foam.block_linear(x, w).sum(), (x, w))
    two = torch.autograd.grad(foam.block_linear(x, w), (x, w), torch.ones_like(dy))
    assert all(torch.equal(p, q) for p, q in zip(one, two))
    assert foam.block_linear(x[0, 0], w).shape == (40,)
    assert foam.block_linear(x[:0], w).shape == (0, 5, 40)
    bias = torch.randn(40, generator=g, device="cuda", requires_grad=True)
    (gb,) = torch.autograd.grad(foam.block_linear(x.detach(), w.detach(), bias), bias, dy)
    assert torch.allclose(gb, dy.sum((0, 1)), rtol=1e-5, atol=1e-6)
    empty = torch.autograd.grad(foam.block_linear(x[:0], w, bias).sum(), (w, bias))
    assert all((e == 0).all() for e in empty)
    with pytest.raises(RuntimeError, match="once_differentiable|differentiable"):
        (gx2,) = torch.autograd.grad(foam.block_linear(x, w).square().sum(), x, create_graph=True)
        gx2.sum().backward()


@pytest.mark.gpu
def test_linear_over_nothing():
    """No columns to sum over, no outputs, an empty batch."""
    bias = torch.randn(4, device="cuda", requires_grad=True)
    x = torch.randn((5, 0), device="cuda", requires_grad=True)
    w = torch.randn((4, 0), device="cuda", requires_grad=True)
    y = foam.block_linear(x, w, bias)
    assert torch.equal(y, bias.expand(5, 4))
    gx, gw, gb = torch.autograd.grad(y.sum(), (x, w, bias))
    assert gx.shape == (5, 0) and gw.shape == (4, 0) and torch.equal(gb, torch.full((4,), 5.0, device="cuda"))
    x = torch.randn((5, 6), device="cuda", requires_grad=True)
    w = torch.randn((0, 6), device="cuda", requires_grad=True)
    y = foam.block_linear(x, w)
    assert y.shape == (5, 0)
    gx, gw = torch.autograd.grad(y.sum(), (x, w))
    assert (gx == 0).all() and gw.shape == (0, 6)
    for transpose in (False, True):
        v, s = foam.quantize_blocks(torch.zeros((0, 5), device="cuda"), transpose=transpose)
        assert foam.dequantize_blocks(v, s).shape == ((5, 0) if transpose else (0, 5))


@pytest.mark.gpu
def test_calls_from_several_threads_and_streams():
    import threading
    g = torch.Generator(device="cuda").manual_seed(4)
    x = torch.randn((300, 256), generator=g, device="cuda")
    w = torch.randn((200, 256), generator=g, device="cuda")
    ref = foam.block_linear(x, w)
    torch.cuda.synchronize()
    results = [None] * 4

    def work(i):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(20):
                results[i] = foam.block_linear(x, w)
        stream.synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert all(torch.equal(r, ref) for r in results)


@pytest.mark.gpu
def test_a_product_that_gave_up_is_reported():
    """The word that a kernel writes when a wait runs out, written here by the
    host: the next product and the check raise it once."""
    from sdfoam_b200 import blocks
    a, sa = foam.quantize_blocks(torch.randn((40, 128), device="cuda"))
    ref = foam.block_matmul(a, sa, a, sa)
    foam.check_block_flags()
    word = blocks._flags[a.device.index][1]
    for call in (lambda: foam.block_matmul(a, sa, a, sa), foam.check_block_flags):
        torch.cuda.synchronize()
        word[0] = 1
        with pytest.raises(RuntimeError, match="gave up waiting"):
            call()
        assert torch.equal(foam.block_matmul(a, sa, a, sa), ref)
        foam.check_block_flags()


@pytest.mark.gpu
def test_inference_keeps_nothing(monkeypatch):
    """Without gradients nothing is kept for a backward, whatever the weight
    asks for; with them, what the inputs that ask need."""
    lib = _lib.load()
    inner, kept = lib.sdfoam_block_linear_forward, []

    class Spy:
        def __getattr__(self, name):
            return getattr(lib, name)

        def sdfoam_block_linear_forward(self, *args):
            kept.append(tuple(map(bool, args[14:16])))
            return inner(*args)

    monkeypatch.setattr(_lib, "load", Spy)
    x = torch.randn((70, 200), device="cuda")
    w = torch.randn((30, 200), device="cuda", requires_grad=True)
    ref = foam.block_linear(x, w)
    assert ref.requires_grad
    with torch.no_grad():
        y = foam.block_linear(x, w)
    with torch.inference_mode():
        z = foam.block_linear(x, w)
    foam.block_linear(x.requires_grad_(), w.detach())
    assert kept == [(True, False), (False, False), (False, False), (False, True)]
    assert torch.equal(y, ref) and torch.equal(z, ref)


@pytest.mark.gpu
def test_expanded_scales():
    """One scale for all blocks, given as an expanded tensor."""
    g = torch.Generator(device="cuda").manual_seed(8)
    a, _ = operand(g, 150, 300, 1)
    b, _ = operand(g, 300, 300, 1)
    one = torch.full((1, 1), 0.25, device="cuda")
    sa, sb = one.expand(150, 3), one.expand(3, 3)
    ref, mag = product64(a, sa, b, sb)
    check_product(foam.block_matmul(a, sa, b, sb, out_dtype=torch.float32), ref, mag, 300, torch.float32)
    assert torch.equal(foam.dequantize_blocks(a, sa), a.float() * 0.25)


@pytest.mark.gpu
def test_codes_of_sites_through_a_layer():
    """Looked-up rows into an 8-bit layer, as a network over sites uses them:
    the gradient reaches the table through both."""
    g = torch.Generator(device="cuda").manual_seed(2)
    table = torch.randn((500, 96), generator=g, device="cuda", dtype=torch.float32, requires_grad=True)
    w = (torch.randn((64, 96), generator=g, device="cuda") / 10).requires_grad_(True)
    ids = torch.randint(0, 600, (1000,), generator=g, device="cuda").to(torch.int32).view(torch.uint32)
    rows = foam.lookup_rows(table, ids, 2.0)
    y = foam.block_linear(rows, w)
    dy = torch.randn_like(y)
    y.backward(dy)
    with torch.no_grad():
        named = ids.view(torch.int32).long()
        (ry, my), (rx, mx), (rw, mw) = formula64(rows, w, dy)
        check_product(y, ry, my, 96, torch.float32)
        assert (y[named >= 500] == 0).all()
        check_product(w.grad, rw, mw, 1000, torch.float32)
        keep = named < 500
        ref = torch.zeros((500, 96), dtype=torch.float64, device="cuda").index_add_(0, named[keep], rx[keep]) * 2
        mag = torch.zeros((500, 96), dtype=torch.float64, device="cuda").index_add_(0, named[keep], mx[keep]) * 2
        assert ((table.grad.double() - ref).abs() <= 2.0 ** -24 * ref.abs() + (500 + 20) * 2.0 ** -24 * mag).all()


@pytest.mark.gpu
def test_other_stream_and_graphs():
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn((1000, 256), generator=g, device="cuda").requires_grad_(True)
    w = torch.randn((256, 256), generator=g, device="cuda").requires_grad_(True)
    dy = torch.randn((1000, 256), generator=g, device="cuda")

    def step():
        y = foam.block_linear(x, w)
        return [y.detach(), *torch.autograd.grad(y, (x, w), dy)]

    ref = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(got, ref))
    # two graphs with workspaces of their own, replayed in turn
    graphs, outs = [], []
    torch.cuda.synchronize()
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        graphs.append(graph)
        outs.append(out)
    with torch.no_grad():
        x.mul_(3.0)
        dy.neg_()
    ref = step()
    for graph, out in zip(graphs * 2, outs * 2):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, ref))
    foam.check_block_flags()


def test_refusals():
    x = torch.zeros((4, 3))
    with pytest.raises(RuntimeError, match="CUDA"):
        foam.quantize_blocks(x)
    with pytest.raises(RuntimeError, match="2 dimensions"):
        foam.quantize_blocks(x[0])
    with pytest.raises(RuntimeError, match="float32, float16 or bfloat16"):
        foam.quantize_blocks(x.double())
    with pytest.raises(RuntimeError, match="1 or 128"):
        foam.quantize_blocks(x, 64)
    a, s = x.to(E4M3), torch.ones((4, 1))
    with pytest.raises(RuntimeError, match="CUDA"):
        foam.block_matmul(a, s, a, s)
    with pytest.raises(RuntimeError, match="float8_e4m3fn"):
        foam.block_matmul(x, s, a, s)
    with pytest.raises(RuntimeError, match="float32 dtype"):
        foam.block_matmul(a, s.double(), a, s)
    with pytest.raises(RuntimeError, match="must have shape"):
        foam.block_matmul(a, torch.ones((2, 1)), a, s)
    with pytest.raises(RuntimeError, match="same number of columns"):
        foam.block_matmul(a, s, a[:, :2], s)
    with pytest.raises(RuntimeError, match="out_dtype"):
        foam.block_matmul(a, s, a, s, out_dtype=torch.float64)
    with pytest.raises(RuntimeError, match="must have shape"):
        foam.dequantize_blocks(a, torch.ones((4, 2)))
    with pytest.raises(RuntimeError, match="columns"):
        foam.block_linear(x, torch.zeros((5, 4)))
    with pytest.raises(RuntimeError, match="weight must have float32"):
        foam.block_linear(x, torch.zeros((5, 3), dtype=torch.float64))
    with pytest.raises(RuntimeError, match="CUDA"):
        foam.block_linear(x, torch.zeros((5, 3)))


def test_entry_points_refuse_bad_arguments():
    from sdfoam_b200 import build
    build.build()
    lib = _lib.load()
    p = ctypes.c_void_p(4096)

    def message():
        return lib.sdfoam_last_error().decode()

    def quantize(x=p, ld=32, dtype=0, m=4, k=32, rows=1, v=p, ldv=32, s=p, t=None, ldt=0, ts=None, sums=None, st=0,
                 ws=None):
        return lib.sdfoam_block_quantize(x, ld, dtype, m, k, rows, v, ldv, s, t, ldt, ts, sums, st, ws, None)

    assert quantize(rows=2) == 1 and "block_rows" in message()
    assert quantize(dtype=3) == 2
    assert quantize(ld=31) == 1 and "apart" in message()
    assert quantize(m=1 << 31) == 1 and "too large" in message()
    assert quantize(m=(1 << 31) - 1, k=1 << 16) == 1 and "too large" in message()
    assert quantize(v=None) == 1 and quantize(s=None) == 1 and quantize(x=None) == 1
    assert quantize(ldv=40) == 1 and quantize(ldv=16) == 1 and quantize(v=ctypes.c_void_p(4100)) == 1
    assert quantize(t=p, ldt=8, ts=p) == 1 and quantize(t=p, ldt=16) == 1
    assert quantize(sums=p, ws=p) == 1 and "column_sums" in message()
    assert quantize(t=p, ldt=16, ts=p, sums=p) == 1 and quantize(t=p, ldt=16, ts=p, sums=p, ws=p, st=3) == 1
    assert quantize(m=0, x=None, v=None) == 0

    def dequantize(v=p, ldv=32, s=p, rows=1, m=4, k=32, dtype=0, out=p):
        return lib.sdfoam_block_dequantize(v, ldv, s, 1, 1, rows, m, k, dtype, out, None)

    assert dequantize(rows=0) == 1 and dequantize(dtype=5) == 2 and dequantize(ldv=31) == 1
    assert dequantize(out=None) == 1 and dequantize(out=ctypes.c_void_p(4098)) == 1

    def matmul(a=p, lda=128, sa=p, ra=1, m=300, b=p, ldb=128, sb=p, rb=128, n=256, k=128, bias=None, bt=0, out=p,
               ldo=256, ot=2, ws=p, size=1 << 30, error=p):
        return lib.sdfoam_block_matmul(a, lda, sa, 1, 1, ra, m, b, ldb, sb, 1, 1, rb, n, k, bias, bt, out, ldo, ot, ws, size, error,
                                       None)

    assert matmul(ra=3) == 1 and matmul(rb=64) == 1 and matmul(ot=3) == 2 and matmul(bias=p, bt=4) == 2
    assert matmul(a=None) == 1 and matmul(sb=None) == 1 and matmul(out=None) == 1 and matmul(error=None) == 1
    assert matmul(lda=120) == 1 and matmul(ldb=112) == 1 and matmul(a=ctypes.c_void_p(4104)) == 1
    assert "16-byte" in message()
    assert matmul(ldo=255) == 1 and matmul(out=ctypes.c_void_p(4097)) == 1
    assert matmul(n=1 << 31) == 1 and "too large" in message()
    need = lib.sdfoam_block_matmul_workspace_bytes(300, 256, 1280)
    assert need > 0 and lib.sdfoam_block_matmul_workspace_bytes(40000, 256, 256) == 0
    wide = dict(lda=1280, ldb=1280, k=1280)
    assert matmul(ws=None, **wide) == 1 and matmul(size=need - 1, **wide) == 1 and "workspace" in message()
    assert matmul(m=0) == 0 and matmul(n=0) == 0

    # the layer: m 300, n 256, k 128
    saved = lib.sdfoam_block_linear_saved_bytes(300, 256, 128, 1, 1)
    ws = lib.sdfoam_block_linear_workspace_bytes(300, 256, 128)
    assert saved > 0 and ws > 0 and lib.sdfoam_block_linear_saved_bytes(300, 256, 128, 0, 0) == 0
    assert lib.sdfoam_block_linear_workspace_bytes(1 << 31, 1, 1) == 0

    def forward(x=p, xt=2, wt=0, n=256, y=p, sv=p, svb=saved, w=p, wsb=ws, bias=None, bt=0, ldx=128):
        return lib.sdfoam_block_linear_forward(x, ldx, xt, 300, p, 128, wt, n, 128, bias, bt, y, sv, svb, 1, 1, w, wsb,
                                               p, None)

    assert forward(xt=3) == 2 and forward(wt=9) == 2 and forward(n=1 << 31) == 1
    assert forward(svb=saved - 1) == 1 and forward(sv=None) == 1 and forward(wsb=0) == 1 and forward(w=None) == 1
    assert "too small" in message()
    assert forward(x=None) == 1 and forward(ldx=100) == 1 and forward(x=ctypes.c_void_p(4097)) == 1

    def backward(dyt=2, kx=1, kw=1, sv=p, svb=saved, dx=p, dw=p, db=None, dbt=0, w=p, wsb=ws, dy=p):
        return lib.sdfoam_block_linear_backward(dy, 256, dyt, 300, 256, 128, sv, svb, kx, kw, dx, 2, dw, 0, db, dbt, w,
                                                wsb, p, None)

    assert backward(kx=0) == 1 and backward(kw=0) == 1 and "kept" in message()
    assert backward(dyt=3) == 2 and backward(svb=1) == 1 and backward(w=None) == 1
    assert backward(dy=None) == 1 and backward(db=p, dbt=3) == 1
    assert backward(dx=None, dw=None) == 0


def test_entry_points_refuse_unaligned_scales():
    """Scales, sums and the error word are read and written as 4-byte words."""
    from sdfoam_b200 import build
    build.build()
    lib = _lib.load()
    p, odd = ctypes.c_void_p(4096), ctypes.c_void_p(4098)

    def quantize(s=p, ts=p, ws=p):
        return lib.sdfoam_block_quantize(p, 32, 0, 4, 32, 1, p, 32, s, p, 16, ts, p, 0, ws, None)

    def matmul(sa=p, sb=p, error=p):
        return lib.sdfoam_block_matmul(p, 128, sa, 1, 1, 1, 300, p, 128, sb, 1, 1, 1, 256, 128, None, 0, p, 256, 2, p, 1 << 30,
                                       error, None)

    calls = [lambda: quantize(s=odd), lambda: quantize(ts=odd), lambda: quantize(ws=odd), lambda: matmul(sa=odd),
             lambda: matmul(sb=odd), lambda: matmul(error=odd),
             lambda: lib.sdfoam_block_dequantize(p, 32, odd, 1, 1, 1, 4, 32, 0, p, None)]
    for call in calls:
        assert call() == 1
        assert "4-byte aligned" in lib.sdfoam_last_error().decode()
