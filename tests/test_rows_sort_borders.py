"""The row gradient at the sizes where its sort changes: 2048 ids to a tile, up
to 96 tiles without a scan of their counts."""
import pytest
import torch

import sdfoam_b200 as foam

EPS = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TILE, FEW = 2048, 96


def reference(grad, ids, rows):
    """(sum, sum of magnitudes) per row in 64 bits."""
    named = (ids >= 0) & (ids < rows)
    out = torch.zeros((2, rows, grad.shape[1]), dtype=torch.float64, device="cuda")
    for o, part in zip(out, (grad.double(), grad.double().abs())):
        o.index_add_(0, ids[named], part[named])
    return out


def adds(n, most):
    """Most fp32 additions behind one sum of `most` of n rows: rows of a chunk,
    the chunks' parts in 32 runs, the runs."""
    chunk = 4
    while chunk < 64 and chunk * 148 * 128 < n:
        chunk *= 2
    parts = -(-most // chunk) + 1
    return min(most, chunk + -(-parts // 32) + 34)


def check(grad, ids, rows, index):
    given = ids.to(torch.int32).view(torch.uint32) if index == torch.uint32 else ids.to(index)
    got = foam.lookup_rows_backward(grad, given, rows)
    ref, mag = reference(grad, ids, rows)
    most = int(torch.bincount(ids.clamp(-1, rows) + 1, minlength=2)[1:].max())
    tol = EPS[grad.dtype] * ref.abs() + (adds(ids.numel(), most) + 1) * 2.0 ** -24 * mag
    if grad.dtype == torch.float16:
        tol += 2.0 ** -25  # half of the smallest step
    assert ((got.double() - ref).abs() <= tol).all()
    assert torch.equal(got, foam.lookup_rows_backward(grad, given, rows)), "not the same bits"


# digits of 9 bits (511 rows: one pass; 150000: two), of fewer, three passes;
# FEW * TILE + 1 ids are one id in a 97th tile
@pytest.mark.gpu
@pytest.mark.parametrize("rows", [3, 511, 512, 150000, 300000])
@pytest.mark.parametrize("n", [FEW * TILE - 1, FEW * TILE, FEW * TILE + 1, 400000])
@pytest.mark.parametrize("index,dtype,columns", [(torch.uint32, torch.float32, 3), (torch.uint32, torch.bfloat16, 8),
                                                 (torch.int32, torch.float16, 5), (torch.int64, torch.float32, 4)])
def test_random_ids(n, rows, index, dtype, columns):
    g = torch.Generator(device="cuda").manual_seed(n + rows)
    ids = torch.randint(-2, rows + 2, (n,), generator=g, device="cuda")
    check(torch.randn((n, columns), generator=g, device="cuda").to(dtype), ids, rows, index)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [300001, 200000, 20000])
@pytest.mark.parametrize("columns", [1, 48, 49])
def test_hot_rows(n, columns):
    """One id for everything, few ids, and runs that end on chunk borders, with
    the additions that the chunks and runs of this size make."""
    g = torch.Generator(device="cuda").manual_seed(columns)
    grad = torch.randn((n, columns), generator=g, device="cuda")
    at = torch.arange(n, device="cuda")
    for ids, rows in ((torch.zeros_like(at), 1), (torch.full_like(at, 9), 1000), (at % 3 * 40, 100), (at // 32, n),
                      (at // 1024 + 5, n), (torch.full_like(at, -1), 50), (torch.where(at < n - 1, 3, 4), 6)):
        for index in (torch.uint32, torch.int64):
            check(grad, ids, rows, index)
