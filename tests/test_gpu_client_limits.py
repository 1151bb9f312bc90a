"""The client's token step on the GPU at its limits: sizes that are refused, values at the ends of their types, memory that runs out,
waits that run out."""
import numpy as np
import pytest
import torch

from test_gpu_client import check_product

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


@pytest.mark.parametrize("xt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("m", [1, 2, 6, 8, 18, 40])
@pytest.mark.parametrize("group", [32, 64, 128, 1024])
def test_rows_near_the_end_of_float32(cx, group, m, xt):
    """Rows of 10^37 with scales that bring the products back, beside ordinary rows: whole numbers times x alone would pass
    float32's range.  The tolerance is the products' usual one."""
    from fhessm import client
    t = random_table(200, 500, group, seed=m, stype=torch.float32)
    x = torch.randn(m, 500, device="cuda", dtype=torch.float64)
    x[::2] *= 1e37
    if m > 3:
        x[3] = 0
        x[3, 77] = torch.finfo(torch.float32).max if xt == torch.float32 else torch.finfo(xt).max
    x = x.to(xt)
    w = t.dequantise().double().cpu().numpy()
    assert np.abs(x.double().cpu().numpy()).max() * 8 > 3.4e38 / 4
    check_product(client.q4_matvec(cx, x, t), x, w, "f32")


@pytest.mark.parametrize("xt", [torch.float32, torch.bfloat16])
def test_large_values_in_some_columns_only(cx, xt):
    """Rows long enough to be taken in several blocks of columns, with their large values in the first, the last or a middle
    one, or in none."""
    from fhessm import client
    cols = 40000
    t = random_table(40, cols, 64, stype=torch.float32)
    x = torch.randn(2, 4, cols, device="cuda", dtype=torch.float64)
    x[0, 0, :50] *= 1e37
    x[0, 1, -50:] *= 1e37
    x[1, 0, 20000:20050] *= 1e37
    x[1, 2, 3::5000] *= 1e37
    w = t.dequantise().double().cpu().numpy()
    for rows in (x[0, :2], x[0, :1], x[1, :2], x[1, 2:]):
        rows = rows.to(xt).contiguous()
        check_product(client.q4_matvec(cx, rows, t), rows, w, "f32")


@pytest.mark.parametrize("xt", [torch.float32, torch.bfloat16])
def test_an_infinity_beside_large_values(cx, xt):
    from fhessm import client
    t = random_table(150, 100, 32, stype=torch.float32)
    x = torch.randn(2, 100, device="cuda")
    x[0] *= 1e37
    x[0, 40] = float("inf")
    x = x.to(xt)
    w = t.dequantise().cpu().numpy()[:, 40]
    got = client.q4_matvec(cx, x, t).cpu().numpy()
    with np.errstate(invalid="ignore"):
        want = np.where(w == 0, np.nan, np.sign(w) * np.inf)
    assert np.array_equal(got[0], want, equal_nan=True)
    check_product(torch.from_numpy(got[1:]), x[1:], t.dequantise().double().cpu().numpy(), "f32")


@pytest.mark.parametrize("m", [1, 12, 64])
def test_not_finite_in_float16(cx, m):
    """An infinity or NaN in one row stays in that row, and gives there what the sum of the products is."""
    from fhessm import client
    t = random_table(150, 100, 32)
    x = torch.randn(m, 100, device="cuda").half()
    r = m // 2
    x[r, 40] = -float("inf")
    w = t.dequantise().double().cpu().numpy()
    got = client.q4_matvec(cx, x, t).cpu().numpy()
    with np.errstate(invalid="ignore"):
        want = np.where(w[:, 40] == 0, np.nan, -np.sign(w[:, 40]) * np.inf)
    assert np.array_equal(got[r], want, equal_nan=True)
    rest = np.arange(m) != r
    if rest.any():
        check_product(torch.from_numpy(got[rest]), x[torch.from_numpy(rest).cuda()], w, "f32")
    x[r, 41] = float("nan")
    assert torch.isnan(client.q4_matvec(cx, x, t)[r]).all()


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two GPUs")
def test_the_current_device_stays():
    """A context on a GPU other than the current one: each call leaves the current one current, refused calls too."""
    import fhessm
    from fhessm import FheError, client
    from fhessm.client import Q4Table
    c = fhessm.CryptoContext(logN=12, L=2, K=1, alpha=1, hw=64, device=1)
    torch.cuda.set_device(0)
    t = random_table(64, 100, 32)
    t = Q4Table(t.weight.to("cuda:1"), t.scale.to("cuda:1"), cols=100, group=32)
    x, u = torch.randn(20, 100, device="cuda:1"), torch.rand(20, device="cuda:1")
    assert torch.cuda.current_device() == 0
    for rows in (x[:1], x):
        logits = client.q4_matvec(c, rows, t)
        assert torch.cuda.current_device() == 0
        check_product(logits, rows, t.dequantise().double().cpu().numpy(), "f32")
    token, _ = client.sample(c, logits, u, top_k=5)
    assert torch.cuda.current_device() == 0
    assert torch.equal(client.q4_rows(c, token, t), t.dequantise()[token])
    assert torch.cuda.current_device() == 0
    with pytest.raises(FheError):
        client.sample(c, logits, u, temperature=-1.0)
    assert torch.cuda.current_device() == 0
    c.close()
    torch.cuda.set_device(0)


def test_a_lost_step_is_reported(cx):
    """Lost logits pass the choice and the look-up as "nothing allowed"; the sync after the step tells."""
    from fhessm import FheError, client
    head = client.TokenHead(cx, random_table(50304, 1024, 64))
    hidden, u = torch.randn(64, 1024, device="cuda"), torch.rand(64, device="cuda")
    want, _, _ = head.step(hidden, u, top_k=50)
    torch.cuda.synchronize()
    cx.sync()
    cx.set_option("q4_waits", 0)
    try:
        tokens, _, rows = head.step(hidden, u, top_k=50)
    finally:
        cx.set_option("q4_waits", -1)
    torch.cuda.synchronize()
    assert (tokens == -1).any() and (rows[tokens == -1] == 0).all()
    with pytest.raises(FheError, match="wait"):
        cx.sync()
    tokens, _, _ = head.step(hidden, u, top_k=50)
    torch.cuda.synchronize()
    cx.sync()
    assert torch.equal(tokens, want)


def test_the_example_runs():
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    out = subprocess.run([sys.executable, os.path.join(root, "examples", "decode_loop.py"), "--ticks", "2"], timeout=300,
                         capture_output=True, text=True)
    assert out.returncode == 0, out.stderr[-2000:]
    assert out.stdout.count("mean log-probability -") == 2


@pytest.mark.parametrize("rows,whole", [(16384, 8), (1000, 18)])
@pytest.mark.parametrize("xt,pieces", [(torch.float32, 3), (torch.float16, 2), (torch.bfloat16, 1)])
def test_how_x_is_held(cx, rows, whole, xt, pieces):
    """Table rows with a single one among zeros read x out: whole while rows of x times the pieces of its type are at most `whole`,
    to 22 bits (float32) and to 2^-39 of the row's largest value above, which stands where a table row may hold zero."""
    from fhessm import client
    cols = 128
    q = torch.full((rows, cols), 8, dtype=torch.uint8, device="cuda")
    at = torch.arange(rows, device="cuda")
    q[at, at % cols] = 9
    t = client.Q4Table(q[:, 0::2] | q[:, 1::2] << 4, torch.ones(rows, 2, device="cuda"), cols=cols, group=64)
    for m in (1, whole // pieces, whole // pieces + 1, 20, 64):
        x = torch.randn(m, cols, device="cuda") * torch.exp2(torch.randint(-12, 13, (m, cols), device="cuda").float())
        if xt != torch.float16:
            x[:, 5] *= 2.0 ** 24
            x[:, 9] = 2.0 ** -30
        x = x.to(xt)
        got = client.q4_matvec(cx, x, t)[:, :cols].double()
        x = x.double()
        if m * pieces <= whole or xt == torch.float16:
            assert torch.equal(got, x)
        else:
            held = 2.0 ** -22 * x.abs() if xt == torch.float32 else 0
            assert ((got - x).abs() <= held + 2.0 ** -39 * x.abs().amax(1, keepdim=True)).all()
            assert not torch.equal(got, x)
