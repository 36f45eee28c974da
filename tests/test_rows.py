"""lookup_rows and its gradient against the same sums in 64 bits."""
import ctypes

import pytest
import torch

import sdfoam_b200 as foam
from sdfoam_b200 import _lib

EPS = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def whole(ids):
    return ids.view(torch.int32).to(torch.int64) & 0xffffffff if ids.dtype == torch.uint32 else ids.to(torch.int64)


def make_ids(values, dtype):
    """int64 values as ids of dtype (-1 becomes UINT32_MAX)."""
    if dtype == torch.uint32:
        return values.to(torch.int32).view(torch.uint32)
    return values.to(dtype)


def ref_lookup(table, ids, scale):
    i = whole(ids).reshape(-1)
    named = (i >= 0) & (i < table.shape[0])
    out = torch.zeros((i.numel(), table.shape[1]), dtype=torch.float64, device=table.device)
    out[named] = table[i[named]].double() * scale
    return out.reshape(*ids.shape, -1)


def ref_gradient(grad, ids, rows, scale):
    """(sum, sum of magnitudes) per row, in 64 bits."""
    i = whole(ids).reshape(-1)
    g = grad.reshape(i.numel(), -1).double()
    named = (i >= 0) & (i < rows)
    both = []
    for part in (g, g.abs()):
        out = torch.zeros((rows, g.shape[1]), dtype=torch.float64, device=grad.device)
        both.append(out.index_add_(0, i[named], part[named]) * scale)
    return both


def check_gradient(got, grad, ids, rows, scale, adds):
    """One rounding to the output type (twice, half a unit each: the value and
    the fp32 product by the scale) and fp32 sums: a sum of k terms in any
    order is off by at most k units of 2^-24 of the sum of magnitudes."""
    ref, mag = ref_gradient(grad, ids, rows, scale)
    assert got.shape == ref.shape and got.dtype == grad.dtype
    tol = (EPS[grad.dtype] + 2.0 ** -24) * ref.abs() + (adds + 1) * 2.0 ** -24 * mag.abs()
    if grad.dtype == torch.float16:
        tol += 2.0 ** -25  # half of the smallest step
    assert ((got.double() - ref).abs() <= tol).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("index", [torch.uint32, torch.int32, torch.int64])
@pytest.mark.parametrize("columns", [1, 2, 3, 49, 64, 217])
def test_lookup(dtype, index, columns):
    g = torch.Generator(device="cuda").manual_seed(columns)
    rows = 501
    table = torch.randn((rows, columns), generator=g, device="cuda").to(dtype)
    table[7, 0] = float("inf")
    table[8, 0] = float("nan")
    for n in (1, 33, 5000):
        v = torch.randint(-1, rows + 3, (n,), generator=g, device="cuda")
        ids = make_ids(v, index)
        got = foam.lookup_rows(table, ids)
        ref = ref_lookup(table, ids, 1.0).to(dtype)
        assert torch.equal(got.view(torch.uint8), ref.view(torch.uint8)) or torch.equal(
            torch.nan_to_num(got), torch.nan_to_num(ref))
        got = foam.lookup_rows(table, ids, 0.3)
        ref = ref_lookup(table, ids, float(torch.tensor(0.3)))
        fine = ref.isfinite()
        assert torch.equal(fine, got.isfinite())
        # the fp32 product's rounding, then the type's
        tol = (EPS[dtype] * (1 + 2.0 ** -20) + 2.0 ** -24) * ref.abs() + (2.0 ** -25 if dtype == torch.float16 else 0)
        assert ((got.double() - ref).abs()[fine] <= tol[fine]).all()


@pytest.mark.gpu
def test_lookup_shapes_and_strides():
    wide = torch.randn((100, 80), device="cuda")
    ids = torch.randint(0, 100, (4, 5, 6), device="cuda")
    for table in (wide, wide[:, 3:40], wide[:, ::2], wide.t()[:40], wide[::2], wide[:, 5:6], wide[:1]):
        i = ids % table.shape[0]
        got = foam.lookup_rows(table, i.transpose(0, 2))
        assert got.shape == (6, 5, 4, table.shape[1])
        assert torch.equal(got, table[i.transpose(0, 2)])
        # an offset start: rows that no vector load may assume aligned
        flat = torch.randn(100 * 49 + 1, device="cuda")[1:].view(100, 49)
        assert torch.equal(foam.lookup_rows(flat, ids), flat[ids])
    # site ids as a query returns them, not in the order of memory
    sites = make_ids(ids[0], torch.uint32)
    assert torch.equal(foam.lookup_rows(wide, sites.t()), wide[ids[0].t()])
    with pytest.raises(RuntimeError, match="device of table"):
        foam.lookup_rows(wide, ids.cpu())
    # nothing to look up, no columns, no rows
    assert foam.lookup_rows(wide, ids[:0]).shape == (0, 5, 6, 80)
    assert foam.lookup_rows(wide[:, :0], ids).shape == (4, 5, 6, 0)
    assert torch.equal(foam.lookup_rows(wide[:0], ids), torch.zeros((4, 5, 6, 80), device="cuda"))
    assert foam.lookup_rows(wide, torch.tensor(3, device="cuda")).shape == (80,)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("columns", [1, 2, 3, 49, 256, 700])
def test_gradient(dtype, columns):
    g = torch.Generator(device="cuda").manual_seed(columns)
    # one block sorts up to 8192 ids; more take passes of up to 9 bits, in
    # tiles of 2048 whose counts are scanned by a launch of its own past 64
    for n, rows in ((1, 1), (5, 300), (127, 5), (1000, 70000), (4097, 256), (8192, 65536), (8193, 1), (20000, 255),
                    (20000, 512), (30011, 66000), (9000, 300000), (131072, 511), (131073, 90000)):
        v = torch.randint(-2, rows + 2, (n,), generator=g, device="cuda")
        grad = torch.randn((n, columns), generator=g, device="cuda").to(dtype)
        for index in (torch.uint32, torch.int64):
            ids = make_ids(v, index)
            got = foam.lookup_rows_backward(grad, ids, rows, 0.5)
            most = int(torch.bincount(v.clamp(min=-2) + 2).max())
            check_gradient(got, grad, ids, rows, 0.5, most)


@pytest.mark.gpu
@pytest.mark.parametrize("columns", [1, 48, 49])
def test_gradient_of_hot_rows(columns):
    """One id for everything, a few ids, and runs that end on chunk borders."""
    g = torch.Generator(device="cuda").manual_seed(columns)
    n = 300001
    grad = torch.randn((n, columns), generator=g, device="cuda")
    at = torch.arange(n, device="cuda")
    for v, rows in ((torch.zeros_like(at), 1), (torch.full_like(at, 9), 1000), (at % 3 * 40, 100), (at // 32, n),
                    (at // 1024 + 5, n), (torch.full_like(at, -1), 50), (torch.where(at < n - 1, 3, 4), 6)):
        got = foam.lookup_rows_backward(grad, v, rows)
        # chunks of 4 to 128 rows, then their sums in 16 runs, then the runs
        check_gradient(got, grad, v, rows, 1.0, 128 + n // 4 // 16 + 1 + 17)
        assert torch.equal(got, foam.lookup_rows_backward(grad, v, rows)), "not the same bits"


@pytest.mark.gpu
def test_gradient_strides():
    ids = torch.randint(0, 50, (7, 11), device="cuda")
    wide = torch.randn((7, 11, 96), device="cuda")
    for grad in (wide, wide[..., 3:40], wide[..., ::2], wide.transpose(0, 1).contiguous().transpose(0, 1),
                 wide[..., :1].expand(7, 11, 33), wide[:1, :1].expand(7, 11, 96)):
        got = foam.lookup_rows_backward(grad, ids, 50)
        check_gradient(got, grad, ids, 50, 1.0, 77)
    assert foam.lookup_rows_backward(wide[..., :0], ids, 50).shape == (50, 0)
    assert torch.equal(foam.lookup_rows_backward(wide[:0], ids[:0], 50), torch.zeros((50, 96), device="cuda"))
    assert foam.lookup_rows_backward(wide, ids, 0).shape == (0, 96)


@pytest.mark.gpu
def test_autograd_and_second_derivative():
    g = torch.Generator(device="cuda").manual_seed(0)
    table = torch.randn((40, 6), generator=g, device="cuda", requires_grad=True)
    ids = make_ids(torch.randint(-1, 40, (90,), generator=g, device="cuda"), torch.uint32)
    w = torch.randn((90, 6), generator=g, device="cuda", requires_grad=True)
    rows = foam.lookup_rows(table, ids, 2.0)
    (grad,) = torch.autograd.grad((rows * w).sum(), table, create_graph=True)
    check_gradient(grad.detach(), w.detach(), ids, 40, 2.0, 90)
    # d/dw of <grad, u> is the lookup of u
    u = torch.randn((40, 6), generator=g, device="cuda")
    (back,) = torch.autograd.grad((grad * u).sum(), w)
    assert torch.equal(back, foam.lookup_rows(u, ids, 2.0))
    # against differences: the lookup is linear, so they are exact up to rounding
    d = torch.randn((40, 6), generator=g, device="cuda", dtype=torch.float64)
    lhs = ((ref_lookup(table.detach().double() + d, ids, 2.0) - ref_lookup(table.detach().double(), ids, 2.0))
           * w.detach().double()).sum()
    rhs = (grad.detach().double() * d).sum()
    assert abs(lhs - rhs) <= 90 * 2.0 ** -24 * (w.abs().double().sum() * 2 * d.abs().max())


@pytest.mark.gpu
def test_rows_of_a_query():
    """The sites that nn and farthest_neighbor return, as they return them."""
    from sdfoam_b200 import synthetic as syn
    f = syn.make_foam("tiny", num_points=4096, seed=3)
    points = torch.from_numpy(f.points).cuda()
    attributes = torch.from_numpy(f.attributes).cuda().requires_grad_(True)
    tree = foam.build_aabb_tree(points)
    sites = foam.nn(points, tree, points[:600] + 1e-4)
    rows = foam.lookup_rows(attributes, sites)
    assert torch.equal(rows, attributes.detach()[sites.view(torch.int32).long()])
    rows.sum().backward()
    count = torch.bincount(sites.view(torch.int32).long(), minlength=4096)
    assert torch.equal(attributes.grad, count[:, None].float().expand_as(attributes))


@pytest.mark.gpu
def test_other_stream_and_graph():
    table = torch.randn((3000, 49), device="cuda", requires_grad=True)
    ids = torch.randint(0, 3000, (20000,), device="cuda")
    ref = foam.lookup_rows(table, ids).detach()
    w = torch.randn_like(ref)
    ref_grad = foam.lookup_rows_backward(w, ids, 3000)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a = foam.lookup_rows(table, ids).detach()
        b = foam.lookup_rows_backward(w, ids, 3000)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(a, ref) and torch.equal(b, ref_grad)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a = foam.lookup_rows(table, ids).detach()
        b = foam.lookup_rows_backward(w, ids, 3000)
    new = torch.randint(0, 3000, (20000,), device="cuda")
    with torch.no_grad():
        ids.copy_(new)
        w.mul_(2.0)
    for _ in range(2):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(a, table.detach()[new])
        assert torch.equal(b, foam.lookup_rows_backward(w, new, 3000))


@pytest.mark.gpu
def test_offsets_past_32_bits():
    """A table and an output of more than 2^32 bytes."""
    table = torch.empty((1 << 21, 1032), dtype=torch.bfloat16, device="cuda")
    table[-5:] = torch.arange(5 * 1032, device="cuda").view(5, 1032).to(torch.bfloat16)
    ids = torch.tensor([(1 << 21) - 5, (1 << 21) - 1], device="cuda")
    assert torch.equal(foam.lookup_rows(table, ids), table[ids])
    del table
    grad = foam.lookup_rows_backward(torch.ones((2, 1032), dtype=torch.bfloat16, device="cuda"), ids, 1 << 21)
    assert float(grad[ids].float().sum()) == 2 * 1032 and float(grad.sum(dtype=torch.float64)) == 2 * 1032


def test_refusals():
    """Checked before any GPU call."""
    t, i = torch.zeros((4, 3)), torch.zeros(5, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="CUDA"):
        foam.lookup_rows(t, i)
    with pytest.raises(RuntimeError, match="2 dimensions"):
        foam.lookup_rows(t[0], i)
    with pytest.raises(RuntimeError, match="float32, float16 or bfloat16"):
        foam.lookup_rows(t.double(), i)
    with pytest.raises(RuntimeError, match="uint32, int32 or int64"):
        foam.lookup_rows(t, i.to(torch.int16))
    with pytest.raises(RuntimeError, match="columns"):
        foam.lookup_rows(torch.zeros((1, (1 << 20) + 1)), i)
    with pytest.raises(RuntimeError, match="fewer than 2\\^32 rows"):
        foam.lookup_rows(torch.zeros((1, 1)).expand(1 << 32, 1), i)
    with pytest.raises(RuntimeError, match="shape of ids"):
        foam.lookup_rows_backward(torch.zeros((4, 3)), i, 4)
    with pytest.raises(RuntimeError, match="num_rows"):
        foam.lookup_rows_backward(torch.zeros((5, 3)), i, -1)


def test_entry_points_refuse_bad_arguments():
    from sdfoam_b200 import build
    build.build()
    lib = _lib.load()
    p = ctypes.c_void_p(4096)

    def lookup(rows=4, columns=3, ld=3, dtype=0, ids=p, n=5, itype=2, table=p, out=p):
        return lib.sdfoam_lookup_rows(table, rows, columns, ld, dtype, ids, n, itype, 1.0, out, None)

    def message():
        return lib.sdfoam_last_error().decode()

    assert lookup(dtype=3) == 2 and "table type" in message()
    assert lookup(itype=3) == 2 and "id type" in message()
    assert lookup(ld=2) == 1 and "apart" in message()
    assert lookup(columns=(1 << 20) + 1, ld=1 << 21) == 1 and "columns" in message()
    assert lookup(table=None) == 1 and lookup(ids=None) == 1 and lookup(out=None) == 1
    assert lookup(table=ctypes.c_void_p(4098)) == 1 and "aligned" in message()
    assert lookup(ids=ctypes.c_void_p(4100)) == 1 and "aligned" in message()
    assert lookup(n=0, ids=None, out=None) == 0
    need = lib.sdfoam_lookup_rows_workspace_bytes(5, 4, 3)
    assert need > 0 and lib.sdfoam_lookup_rows_workspace_bytes(0, 4, 3) == 0

    def back(n=5, ws=p, size=need, grad=p, out=p, rows=4):
        return lib.sdfoam_lookup_rows_backward(grad, 3, 3, 0, p, n, 2, 1.0, out, rows, ws, size, None)

    assert back(n=1 << 31) == 1 and "2^31" in message()
    assert back(grad=None) == 1 and back(out=None) == 1
    assert back(size=need - 1) == 1 and back(ws=None) == 1 and "workspace" in message()
    assert back(ws=ctypes.c_void_p(4096 + 16)) == 1 and "256" in message()
    assert back(rows=0, out=None, ws=None, size=0) == 0
