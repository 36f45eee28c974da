"""Row lookups past 2^31 rows."""
import pytest
import torch

import sdfoam_b200 as foam


@pytest.mark.gpu
@pytest.mark.parametrize("index", [torch.int32, torch.uint32, torch.int64])
@pytest.mark.parametrize("n", [40, 9000, 250000])
def test_ids_of_a_table_past_2_31_rows(index, n):
    """A negative int32 id names no row, also where the same bits as an
    unsigned number would; the other types reach the rows behind 2^31.  Ids for
    the one-block sort, for four passes without a scan and with it."""
    rows = (1 << 31) + 8
    table = torch.empty((rows, 1), dtype=torch.bfloat16, device="cuda")
    table[:8] = torch.arange(1, 9, device="cuda").view(8, 1).to(torch.bfloat16)
    table[-16:] = torch.arange(101, 117, device="cuda").view(16, 1).to(torch.bfloat16)
    low = torch.arange(n, device="cuda") % 24
    whole = torch.where(low < 8, low, low - 24 + rows)  # 0 .. 7 and the last 16 rows
    ids = whole.to(torch.int64) if index == torch.int64 else whole.to(torch.int32)
    named = torch.ones_like(whole, dtype=torch.bool)
    if index == torch.uint32:
        ids = ids.view(torch.uint32)
    if index == torch.int32:
        named = whole < 1 << 31  # the rows behind have no int32 id: their bits are negative numbers
    got = foam.lookup_rows(table, ids)
    assert torch.equal(got, torch.where(named[:, None], table[whole], 0))
    del table
    grad = foam.lookup_rows_backward(torch.ones((n, 1), dtype=torch.bfloat16, device="cuda"), ids, rows)
    count = torch.bincount(low[named], minlength=24).to(torch.bfloat16)[:, None]
    assert torch.equal(torch.cat([grad[:8], grad[-16:]]), count)
    assert not grad[8:-16].any()
