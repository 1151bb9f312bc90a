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


def random_table(rows, cols, group, seed=0, stype=torch.float16):
    from fhessm.client import Q4Table
    g = torch.Generator(device="cuda").manual_seed(seed)
    w = torch.randint(0, 256, (rows, -(-cols // 32) * 16), device="cuda", dtype=torch.uint8, generator=g)
    s = torch.rand(rows, -(-cols // group), device="cuda", generator=g) * 0.01 + 0.001
    return Q4Table(w, s.to(stype), cols=cols, group=group)


# One tile, which needs no slot twice; several tiles in every block; several ranges of columns; columns in parts.  `lost`: a block
# fills its slots long before the first of them is free again.
SHAPES = [(20, 100, 256, 64, torch.bfloat16, False), (64, 50304, 1024, 64, torch.float32, True),
          (64, 20000, 2048, 96, torch.float32, True), (17, 40000, 4096, 32, torch.float16, True),
          (64, 300, 4096, 32, torch.bfloat16, False)]


@pytest.mark.parametrize("m,rows,cols,group,xt,lost", SHAPES)
def test_a_wait_that_runs_out(cx, m, rows, cols, group, xt, lost):
    """With no tries at all, the first role that finds no free slot gives up: the call ends by itself, what is not NaN is right, a
    NaN is reported at the next sync, and the calls after it are right again."""
    from fhessm import FheError, client
    t = random_table(rows, cols, group)
    x = torch.randn(m, cols, device="cuda").to(xt)
    want = client.q4_matvec(cx, x, t)
    torch.cuda.synchronize()
    cx.sync()
    cx.set_option("q4_waits", 0)
    try:
        for _ in range(4):
            got = client.q4_matvec(cx, x, t)
            torch.cuda.synchronize()
            nan = torch.isnan(got)
            assert ((got == want) | nan).all()
            assert nan.any() or not lost
            if nan.any():
                with pytest.raises(FheError, match="wait"):
                    cx.sync()
            cx.sync()
    finally:
        cx.set_option("q4_waits", -1)
    assert torch.equal(client.q4_matvec(cx, x, t), want)
    torch.cuda.synchronize()
    cx.sync()


@pytest.mark.parametrize("m", [1, 20, 64])
@pytest.mark.parametrize("group", [1 << 20, (1 << 31) - 1024, (1 << 31) - 32])
def test_a_group_far_above_the_columns(cx, group, m):
    """One scale a row, whatever the group's size: the same product as with the next group above the columns."""
    from fhessm import client
    t = random_table(200, 1000, 1024)
    x = torch.randn(m, 1000, device="cuda")
    wide = client.Q4Table(t.weight, t.scale, cols=1000, group=group)
    want = client.q4_matvec(cx, x, t)
    # sums of the same products, rounded in another order: 1,000 roundings of 2^-24 on either side
    mag = x.abs().double() @ t.dequantise().abs().double().T
    assert ((client.q4_matvec(cx, x, wide).double() - want.double()).abs() <= 2 * 1000 * 2.0 ** -24 * mag).all()
    ids = torch.arange(200, device="cuda")
    assert torch.equal(client.q4_rows(cx, ids, wide), t.dequantise())


def trim_pool():
    """Gives the driver what its stream-ordered pool holds and nobody uses, as after earlier tests."""
    import ctypes
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    rt, pool = ctypes.CDLL("libcudart.so.12"), ctypes.c_void_p()
    assert rt.cudaDeviceGetDefaultMemPool(ctypes.byref(pool), 0) == 0
    assert rt.cudaMemPoolTrimTo(pool, ctypes.c_size_t(0)) == 0


def test_a_product_refused_for_memory(cx):
    """A workspace as large as x, of which the GPU holds one only: the call is refused, and the calls after it, torch's too, are
    served."""
    from fhessm import FheError, client
    trim_pool()
    mem = cx.memory()
    cols = 12288
    x = torch.empty(min(1 << 21, int(0.6 * mem["total"]) // (4 * cols)), cols, device="cuda")
    t = random_table(1, cols, 64)
    with pytest.raises(FheError, match="memory"):
        client.q4_matvec(cx, x, t)
    ids = torch.zeros(3, dtype=torch.int64, device="cuda")
    assert torch.equal(client.q4_rows(cx, ids, t), t.dequantise().expand(3, cols))
    assert torch.ones(5, device="cuda").sum() == 5
    few = torch.zeros(20, cols, device="cuda")
    assert (client.q4_matvec(cx, few, t) == 0).all()
    del x
    trim_pool()
