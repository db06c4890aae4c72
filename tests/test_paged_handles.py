"""Handles and workspaces of the paged cache's calls on the host: what they refuse, keep and hand on.  No GPU."""
import pytest

torch = pytest.importorskip("torch")

from homelab_b200.paged import PagedKv  # noqa: E402


def pool(pages=8, heads=2, page=16, dim=64):
    return torch.zeros(pages, heads, page, dim, dtype=torch.bfloat16), torch.zeros(pages, heads, page, dim,
                                                                                   dtype=torch.bfloat16)


def reach(table, c):
    """The entries of the table's storage that the kernels may read: row b from b * table_stride, max_pages of them."""
    rows = [c.struct.block_table + 4 * (b * c.struct.table_stride + i) for b in range(c.batch)
            for i in range(c.struct.max_pages)]
    want = [table.data_ptr() + 4 * (b * table.stride(0) + i * table.stride(1)) for b in range(table.shape[0])
            for i in range(table.shape[1])]
    return rows, want


def test_block_table_rows_that_overlap_are_refused():
    k, v = pool()
    t = torch.arange(24, dtype=torch.int32)
    for bad in (t[:8].expand(4, 8), t[None, :8].expand(2, 8), t.as_strided((3, 8), (4, 1)), t.as_strided((2, 8), (7, 1))):
        with pytest.raises(ValueError, match="overlap"):
            PagedKv(k, v, bad)


@pytest.mark.parametrize("table", [
    torch.arange(24, dtype=torch.int32).view(3, 8),
    torch.arange(48, dtype=torch.int32).view(3, 16)[:, 3:11],        # cut out of a wider one
    torch.arange(24, dtype=torch.int32).as_strided((2, 8), (8, 1)),  # rows back to back
    torch.arange(24, dtype=torch.int32).as_strided((1, 8), (0, 1)),  # one row: its stride leads nowhere
    torch.arange(8, dtype=torch.int32)[None].expand(1, 8),
    torch.arange(6, dtype=torch.int32)[:, None],                     # one page a sequence
    torch.arange(24, dtype=torch.int32).view(3, 8)[:, :1],
    torch.zeros(0, 5, dtype=torch.int32),
])
def test_block_table_rows_are_read_where_they_lie(table):
    k, v = pool()
    rows, want = reach(table, PagedKv(k, v, table))
    assert rows == want
