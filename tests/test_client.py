"""The client's token step without a GPU: the 4-bit table's layout and its nearest values, the definition of the
choice on cases worked out by hand, and refusals that need no device."""
import ctypes as C
import os

import numpy as np
import pytest
import torch

from client_ref import pack, sample_row, table_values
from conftest import ROOT

LIB = os.path.join(ROOT, "fhe-ssm_b200", "fhessm", "libfhessm.so")


@pytest.mark.parametrize("rows,cols,group", [(1, 1, 32), (5, 31, 32), (7, 64, 32), (4, 100, 64), (3, 257, 128),
                                             (6, 48, 256)])
def test_table_layout(rows, cols, group):
    from fhessm.client import Q4Table
    rng = np.random.default_rng(1)
    q = rng.integers(0, 16, (rows, -(-cols // 32) * 32))
    s = rng.uniform(0.1, 2, (rows, -(-cols // group))).astype(np.float32)
    t = Q4Table(torch.from_numpy(pack(q)), torch.from_numpy(s), cols=cols, group=group)
    want = table_values(q, s, cols, group)
    # one product of a 4-bit whole number and a float32 scale: one rounding
    assert np.abs(t.dequantise().numpy() - want).max() <= 2.0 ** -24 * np.abs(want).max()
    assert (t.rows, t.cols, t.group) == (rows, cols, group)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_quantise_is_nearest(dtype):
    """|w - value| <= scale / 2 (rounding to the grid) + the grid's end moving with the scale's rounding."""
    from fhessm.client import Q4Table
    rng = np.random.default_rng(2)
    w = rng.normal(0, 0.02, (33, 200))
    w[5] = 0.0
    t = Q4Table.quantise(w, group=64, scale_dtype=dtype)
    s = np.repeat(t.scale.float().numpy(), 64, axis=1)[:, :200].astype(np.float64)
    unit = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}[dtype]
    err = np.abs(t.dequantise().numpy() - w)
    # w / scale is at most 7 (1 + unit): the grid ends at 7, so the end adds 7 unit scales
    assert (err <= s * (0.5 + 7 * unit) + 2.0 ** -22 * np.abs(w) + 2.0 ** -24).all()
    assert (t.dequantise()[5] == 0).all()


def test_table_refusals():
    from fhessm import FheError
    from fhessm.client import Q4Table
    w, s = torch.zeros(4, 32, dtype=torch.uint8), torch.ones(4, 2)
    Q4Table(w, s, cols=64, group=32)
    for kw, ww, ss in [(dict(cols=64, group=16), w, s), (dict(cols=64, group=48), w, s), (dict(cols=65, group=64), w, s),
                       (dict(cols=64, group=64), w, s), (dict(cols=0, group=32), w, s),
                       (dict(cols=64, group=32), w.int(), s), (dict(cols=64, group=32), w, s.double()),
                       (dict(cols=64, group=32), w, s[:3]), (dict(cols=64, group=32), w[:, ::2], s),
                       (dict(cols=64, group=32), w, torch.ones(2, 4).T), (dict(cols=64, group=32), w[0], s)]:
        with pytest.raises(FheError):
            Q4Table(ww, ss, **kw)


def test_definition_by_hand():
    """ln 1, ln 2, ln 4, ln 1 with a forbidden token between: weights 1/4, 1/2, 1, 0, 1/4 of the largest."""
    x = np.array([0.0, np.log(2), np.log(4), -np.inf, 0.0])
    pick = lambda u, t=1.0, k=0, p=1.0, mp=0.0: sample_row(x, u, t, k, p, mp)[0]
    assert [pick(u) for u in (0.0, 0.12, 0.13, 0.37, 0.38, 0.87, 0.88, 0.999)] == [0, 0, 1, 1, 2, 2, 4, 4]
    assert [pick(u, k=2) for u in (0.0, 0.32, 0.34)] == [1, 1, 2]
    assert pick(0.0, k=1) == 2 and pick(0.999, t=0.0) == 2
    # the largest alone holds 1/2: a token before which 1/2 is reached is out
    assert [pick(u, p=0.49) for u in (0.0, 0.99)] == [2, 2]
    assert [pick(u, p=0.51) for u in (0.0, 0.34)] == [1, 2]
    # of the equal tokens 0 and 4 the lower index is ranked first
    assert [pick(u, p=0.8) for u in (0.0, 0.99)] == [0, 2]
    assert [pick(u, mp=0.3) for u in (0.0, 0.99)] == [1, 2]
    assert sample_row(np.full(3, -np.inf), 0.5, 1.0, 0, 1.0, 0.0)[:2] == (-1, -np.inf)


@pytest.mark.skipif(not os.path.exists(LIB), reason="libfhessm.so not built")
def test_null_arguments_are_refused():
    import fhessm
    from fhessm import client
    h = client._sigs()
    for rc in (h.fhe_q4_matvec(None, None, None, 0, 0, 1, None, 0, 0, None),
               h.fhe_q4_rows(None, None, None, 1, None, 0, 0, None),
               h.fhe_sample(None, None, None, 0, 1, 1, 1, None, None, None, None)):
        assert rc == -1 and b"null" in fhessm.lib().fhe_last_error()


def test_c_struct_sizes():
    """The packed bytes have the header's layout (x86-64: natural alignment)."""
    from fhessm import client

    class Q4(C.Structure):
        _fields_ = [("q", C.c_void_p), ("scale", C.c_void_p), ("scale_type", C.c_int), ("rows", C.c_int), ("cols", C.c_int),
                    ("group", C.c_int), ("ldq", C.c_longlong), ("lds", C.c_longlong)]

    class Cfg(C.Structure):
        _fields_ = [("temperature", C.c_void_p), ("top_k", C.c_void_p), ("top_p", C.c_void_p), ("min_p", C.c_void_p),
                    ("temperature_all", C.c_float), ("top_k_all", C.c_int32), ("top_p_all", C.c_float),
                    ("min_p_all", C.c_float)]

    assert client._Q4.pack(1 << 40, 2, 3, 4, 5, 6, 1 << 33, 8) == bytes(Q4(1 << 40, 2, 3, 4, 5, 6, 1 << 33, 8))
    assert client._SAMPLE.pack(1, 2, 3, 4, 0.5, -6, 7.5, 8.25) == bytes(Cfg(1, 2, 3, 4, 0.5, -6, 7.5, 8.25))
