"""The client's token step on the GPU at its limits: sizes that are refused, values at the ends of their types, memory that runs out,
waits that run out."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def cx():
    import fhessm
    c = fhessm.CryptoContext(logN=12, L=2, K=1, alpha=1, hw=64)
    yield c
    c.close()


@pytest.mark.parametrize("rows", [(1 << 30) + 1, (1 << 31) - 1])
def test_too_many_rows_are_refused(cx, rows):
    """At the C entries, before anything is launched: the pointers are those of one row."""
    import fhessm
    from fhessm import client
    w, s = torch.zeros(1, 16, dtype=torch.uint8, device="cuda"), torch.zeros(1, 1, device="cuda")
    x, out, ids = torch.zeros(1, 32, device="cuda"), torch.zeros(1, 32, device="cuda"), torch.zeros(1, dtype=torch.int64, device="cuda")
    table = client._Q4.pack(w.data_ptr(), s.data_ptr(), 0, rows, 32, 32, 16, 1)
    h = client._sigs()
    for rc in (h.fhe_q4_matvec(cx.h, table, x.data_ptr(), 0, 32, 1, out.data_ptr(), 0, rows, None),
               h.fhe_q4_rows(cx.h, table, ids.data_ptr(), 1, out.data_ptr(), 0, 32, None)):
        assert rc == -1 and b"FHE_Q4_MAX_ROWS" in fhessm.lib().fhe_last_error()
