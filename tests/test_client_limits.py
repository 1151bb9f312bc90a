"""Limits of the client's token step that need no GPU: what a table may be, and what its values become."""
import pytest
import torch


@pytest.mark.parametrize("rows,ok", [(1 << 30, True), ((1 << 30) + 1, False), ((1 << 31) - 1, False), ((1 << 31) + 5, False)])
def test_rows_of_a_table(rows, ok):
    """The products count rows in 32 bits, rounded up to whole blocks (tensors without memory: the size alone is looked at)."""
    from fhessm import FheError
    from fhessm.client import Q4Table
    w, s = torch.empty(rows, 16, dtype=torch.uint8, device="meta"), torch.empty(rows, 1, dtype=torch.float16, device="meta")
    if ok:
        assert Q4Table(w, s, cols=32, group=32).rows == rows
    else:
        with pytest.raises(FheError, match="rows at most"):
            Q4Table(w, s, cols=32, group=32)
