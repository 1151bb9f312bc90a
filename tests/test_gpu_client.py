"""The client's token step on the GPU (fhessm.client) against its definitions in float64.

Tolerances, from the definitions:
  * a product: each of its K terms and sums is rounded in float32, and a float32 row may be carried as two pieces of 11 bits;
    |error| <= (K + 8) 2^-24 sum|x w| + 2^-21 sum|x w|, plus half a unit of the output's type;
  * a table row: one float32 product of a whole number and a scale, then the output's rounding: equal bits;
  * a token: equal, decisions within 2^-20 of their limits going either way (client_ref.OPEN);
  * a log-probability: z is a rounded quotient (2^-23 |z|), the logarithm of a sum that is good to 2^-21.
"""
import numpy as np
import pytest
import torch

from client_ref import pack, sample_accepts, table_values

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
HALF_UNIT = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}


@pytest.fixture(scope="module")
def cx():
    import fhessm
    c = fhessm.CryptoContext(logN=12, L=2, K=1, alpha=1, hw=64)
    yield c
    c.close()


def make_table(rng, rows, cols, group, stype="f16", pad=0):
    """(Q4Table on the GPU, its values in float64); `pad` more bytes a row than needed, filled with noise."""
    from fhessm.client import Q4Table
    wide = -(-cols // 32) * 32
    q = rng.integers(0, 16, (rows, wide))
    s = torch.from_numpy(rng.uniform(0.001, 0.02, (rows, -(-cols // group))).astype(np.float32)).to(TYPES[stype])
    w = rng.integers(0, 256, (rows, wide // 2 + pad), dtype=np.uint8)
    w[:, :wide // 2] = pack(q)
    t = Q4Table(torch.from_numpy(w).cuda(), s.cuda(), cols=cols, group=group)
    return t, table_values(q, s.double().numpy(), cols, group)


def check_product(got, x, w, ot):
    x, got = x.double().cpu().numpy(), got.double().cpu().numpy()
    ref, mag = x @ w.T, np.abs(x) @ np.abs(w).T
    tol = ((w.shape[1] + 8) * 2.0 ** -24 + 2.0 ** -21) * mag + HALF_UNIT[ot] * np.abs(ref) + (2.0 ** -25 if ot == "f16" else 0)
    bad = np.abs(got - ref) > tol
    assert not bad.any(), (np.argwhere(bad)[:4], np.abs(got - ref)[bad][:4], tol[bad][:4])


@pytest.mark.parametrize("m,rows,cols,group,xt,st,ot", [
    (1, 1, 1, 32, "f32", "f32", "f32"), (1, 7, 33, 32, "f32", "f16", "f32"), (3, 129, 31, 32, "bf16", "f16", "f32"),
    (1, 1000, 256, 64, "f32", "bf16", "f32"), (2, 515, 1024, 64, "f16", "f16", "f16"),
    (4, 260, 1000, 32, "f32", "f32", "f32"), (5, 300, 1023, 128, "bf16", "bf16", "bf16"),
    (8, 1025, 512, 512, "f32", "f16", "f32"), (9, 257, 300, 64, "f16", "f32", "f32"),
    (16, 128, 64, 32, "f32", "f16", "f32"), (17, 127, 96, 96, "bf16", "f16", "f32"),
    (32, 640, 1024, 64, "f32", "f16", "bf16"), (33, 385, 2050, 128, "f32", "f16", "f32"),
    (48, 200, 200, 1024, "f16", "f16", "f16"), (63, 129, 999, 160, "f32", "bf16", "f32"),
    (64, 4099, 1024, 64, "f32", "f16", "f32"), (64, 300, 4096, 32, "bf16", "f16", "f32"),
    (128, 512, 48, 32, "f32", "f16", "f32"), (40, 200, 33, 32, "bf16", "f32", "f32"), (70, 513, 136, 32, "f16", "bf16", "f32"),
    (24, 50304, 1024, 32, "f32", "f16", "f32"), (64, 20000, 2048, 96, "bf16", "f16", "f32"),
    (65, 130, 320, 64, "f32", "f16", "f32"), (130, 77, 161, 32, "bf16", "f32", "f32"),
    (200, 1000, 128, 128, "f16", "f16", "f32")])
def test_matvec(cx, m, rows, cols, group, xt, st, ot):
    from fhessm import client
    rng = np.random.default_rng(m * 1000 + cols)
    t, w = make_table(rng, rows, cols, group, st)
    x = torch.from_numpy(rng.normal(0, 1, (m, cols)).astype(np.float32)).to(TYPES[xt]).cuda()
    got = client.q4_matvec(cx, x, t, dtype=TYPES[ot])
    assert got.dtype == TYPES[ot] and got.shape == (m, rows)
    check_product(got, x, w, ot)


@pytest.mark.parametrize("m", [1, 6, 40])
@pytest.mark.parametrize("xt", ["f32", "f16", "bf16"])
def test_matvec_strides(cx, m, xt):
    """Rows of x, of the output and of the table with gaps between them, none of x's or the output's aligned to more than
    one value, and noise in the table's padding."""
    from fhessm import client
    rng = np.random.default_rng(m)
    rows, cols, group = 333, 229, 64
    t, w = make_table(rng, rows, cols, group, "f16", pad=48)
    big = torch.full((m, cols + 12), float("nan"), dtype=TYPES[xt], device="cuda")
    x = big[:, 5:5 + cols]
    x.copy_(torch.from_numpy(rng.normal(0, 1, (m, cols)).astype(np.float32)))
    hold = torch.full((m, rows + 9), 7.0, device="cuda")
    out = client.q4_matvec(cx, x, t, out=hold[:, 3:3 + rows])
    check_product(out, x, w, "f32")
    assert (hold[:, :3] == 7).all() and (hold[:, 3 + rows:] == 7).all()
    scale = torch.zeros(rows, 11, dtype=t.scale.dtype, device="cuda")
    scale[:, 2:2 + t.scale.shape[1]] = t.scale
    t2 = client.Q4Table(t.weight, scale[:, 2:2 + t.scale.shape[1]], cols=cols, group=group)
    assert torch.equal(client.q4_matvec(cx, x, t2), out)


@pytest.mark.parametrize("m", [1, 7, 20])
@pytest.mark.parametrize("st", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,cols,group", [(40, 5000, 64), (2500, 1000, 32), (70, 1300, 128), (33, 4097, 32), (1300, 999, 96)])
def test_matvec_scale_rows(cx, rows, cols, group, st, m):
    """Scales whose rows start on 16-byte boundaries (contiguous or with gaps of noise) or on none: the same values."""
    from fhessm import client
    rng = np.random.default_rng(rows + m)
    t, w = make_table(rng, rows, cols, group, st)
    x = torch.from_numpy(rng.normal(0, 1, (m, cols)).astype(np.float32)).to(torch.bfloat16).cuda()
    out = client.q4_matvec(cx, x, t)
    check_product(out, x, w, "f32")
    n = t.scale.shape[1]
    for stride, at in [(-(-n // 8) * 8 + 8, 0), (-(-n // 8) * 8 + 8, 8), (n + 3 | 1, 1)]:
        big = torch.full((rows, stride + 16), float("nan"), dtype=TYPES[st], device="cuda").flatten()
        scale = big.as_strided((rows, n), (stride, 1), at)
        scale.copy_(t.scale)
        t2 = client.Q4Table(t.weight, scale, cols=cols, group=group)
        assert torch.equal(client.q4_matvec(cx, x, t2), out)


@pytest.mark.parametrize("m", [1, 5, 64])
def test_matvec_large_and_small_values(cx, m):
    """float32 rows far outside the 16-bit types' range, and rows whose values span many powers of two."""
    from fhessm import client
    rng = np.random.default_rng(m + 50)
    t, w = make_table(rng, 200, 512, 64, "f32")
    x = rng.normal(0, 1, (m, 512)) * np.exp2(rng.uniform(-12, 12, (m, 512)))
    x *= np.exp2(rng.choice([-60.0, 0.0, 60.0], (m, 1)))
    x[0] = 0.0 if m > 1 else x[0]
    x = torch.from_numpy(x.astype(np.float32)).cuda()
    check_product(client.q4_matvec(cx, x, t), x, w, "f32")


@pytest.mark.parametrize("m", [1, 12, 64])
@pytest.mark.parametrize("xt", ["f32", "bf16"])
def test_matvec_not_finite(cx, m, xt):
    """An infinity or NaN in one row stays in that row, and gives there what the sum of the products is."""
    from fhessm import client
    rng = np.random.default_rng(m + 60)
    t, w = make_table(rng, 150, 100, 32)
    x = torch.from_numpy(rng.normal(0, 1, (m, 100)).astype(np.float32)).to(TYPES[xt]).cuda()
    x[m // 2, 40] = float("inf")
    got = client.q4_matvec(cx, x, t).cpu().numpy()
    with np.errstate(invalid="ignore"):
        ref = np.where(w[:, 40] == 0, np.nan, np.sign(w[:, 40]) * np.inf)
    assert np.array_equal(got[m // 2], ref, equal_nan=True)
    rest = np.arange(m) != m // 2
    if rest.any():
        check_product(torch.from_numpy(got[rest]), x[torch.from_numpy(rest).cuda()], w, "f32")
    x[m // 2, 41] = float("nan")
    assert torch.isnan(client.q4_matvec(cx, x, t)[m // 2]).all()


def test_matvec_a_long_table(cx):
    """A table whose bytes pass 2^31: the last row's offset needs 64 bits."""
    from fhessm import client
    rows, cols = (1 << 31) // 2048 + 40, 4096
    w = torch.full((rows, cols // 2), 0x88, dtype=torch.uint8, device="cuda")     # every value 0
    rng = np.random.default_rng(7)
    q = rng.integers(0, 16, (3, cols))
    w[-3:] = torch.from_numpy(pack(q)).cuda()
    s = torch.full((rows, cols // 128), 0.01, dtype=torch.float16, device="cuda")
    t = client.Q4Table(w, s, cols=cols, group=128)
    for m in (1, 20):
        x = torch.from_numpy(rng.normal(0, 1, (m, cols)).astype(np.float32)).cuda()
        got = client.q4_matvec(cx, x, t)
        check_product(got[:, -3:], x, table_values(q, s[-3:].double().cpu().numpy(), cols, 128), "f32")
        assert (got[:, :-3] == 0).all()
    r = client.q4_rows(cx, torch.tensor([rows - 2], device="cuda"), t)
    assert torch.equal(r[0].cpu(), (torch.from_numpy(q[1]).float() - 8) * s[-1, 0].float().cpu())


@pytest.mark.parametrize("m,rows,cols,group,st,ot", [
    (1, 1, 1, 32, "f32", "f32"), (3, 10, 31, 32, "f16", "f16"), (64, 1000, 1024, 64, "f16", "f32"),
    (130, 77, 1000, 128, "bf16", "bf16"), (500, 300, 257, 32, "f32", "f16"), (9, 50, 4096, 4096, "f16", "bf16")])
def test_rows(cx, m, rows, cols, group, st, ot):
    from fhessm import client
    rng = np.random.default_rng(m + cols)
    t, _ = make_table(rng, rows, cols, group, st, pad=16)
    tokens = torch.from_numpy(rng.integers(0, rows, m)).cuda()
    if m > 5:
        tokens[2], tokens[4], tokens[5] = -1, rows, 1 << 40
    hold = torch.full((m, cols + 5), 7.0, dtype=TYPES[ot], device="cuda")
    got = client.q4_rows(cx, tokens, t, dtype=TYPES[ot], out=hold[:, 1:1 + cols])
    inside = (tokens >= 0) & (tokens < rows)
    want = t.dequantise()[tokens.clamp(0, rows - 1)] * inside.unsqueeze(1)
    assert torch.equal(got, want.to(TYPES[ot]))
    assert (hold[:, 0] == 7).all() and (hold[:, 1 + cols:] == 7).all()
    assert torch.equal(client.q4_rows(cx, tokens, t, dtype=TYPES[ot]), got)


def check_sample(cx, x, u, t=1.0, k=0, p=1.0, mp=0.0):
    from fhessm import client
    token, lp = client.sample(cx, x, u, temperature=t, top_k=k, top_p=p, min_p=mp)
    again = client.sample(cx, x, u, temperature=t, top_k=k, top_p=p, min_p=mp)
    assert torch.equal(token, again[0]) and torch.equal(lp, again[1])
    xs, us = x.double().cpu().numpy(), u.double().cpu().numpy()
    tk, lp = token.cpu().numpy(), lp.cpu().numpy()
    per = lambda v, r: float(v[r]) if torch.is_tensor(v) else float(v)
    for r in range(x.shape[0]):
        want = (xs[r], us[r], per(t, r), int(per(k, r)), per(p, r), per(mp, r))
        ok, ref = sample_accepts(*want, int(tk[r]))
        assert ok, (r, tk[r], ref, want[1:])
        if ref is not None and np.isfinite(ref):
            # z to 2^-23 of its size (at most 30), the sum to 2^-21, the result's own rounding
            assert abs(lp[r] - ref) <= 2.0 ** -23 * 32 + 2.0 ** -21 + 2.0 ** -23 * abs(ref), (r, lp[r], ref)
        elif ref is not None:
            assert lp[r] == ref
    return token


SETTINGS = [dict(), dict(t=0.7, k=50, p=0.95), dict(p=0.9), dict(mp=0.05), dict(k=3), dict(t=0.0),
            dict(t=1.3, k=400, p=0.5, mp=0.01), dict(t=0.3, p=0.999), dict(k=1000000), dict(t=5.0, k=1, p=0.1)]


@pytest.mark.parametrize("xt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,vocab", [(1, 1), (2, 2), (3, 31), (2, 33), (5, 1000), (3, 1023), (4, 5001),
                                        (2, 50277), (150, 700), (1, 140001)])
def test_sample(cx, rows, vocab, xt):
    rng = np.random.default_rng(rows * 7 + vocab)
    for n, kw in enumerate(SETTINGS if vocab < 40000 else SETTINGS[:4]):
        x = torch.from_numpy(rng.normal(0, [0.6, 2.5][n % 2], (rows, vocab)).astype(np.float32)).to(TYPES[xt]).cuda()
        u = torch.from_numpy(rng.uniform(0, 1, rows).astype(np.float32)).clamp(max=0.9999999).cuda()
        check_sample(cx, x, u, **kw)


def test_sample_settings_of_each_row(cx):
    rng = np.random.default_rng(11)
    rows, vocab = 40, 3001
    x = torch.from_numpy(rng.normal(0, 2, (rows, vocab + 6)).astype(np.float32)).cuda()[:, 3:3 + vocab]   # strided rows
    x[torch.from_numpy(rng.uniform(0, 1, (rows, vocab)) < 0.3).cuda()] = -float("inf")
    x[7] = -float("inf")
    x[9] = -float("inf")
    x[9, 17] = -3.0
    x[11, ::3] = float("nan")
    f = lambda a: torch.from_numpy(np.asarray(a, np.float32)).cuda()
    t = f(rng.uniform(0.2, 2, rows))
    t[5], t[6] = 0.0, -1.0
    k = torch.from_numpy(rng.integers(-1, 300, rows).astype(np.int32)).cuda()
    p, mp = f(rng.uniform(0.3, 1.0, rows)), f(rng.uniform(0, 0.1, rows))
    p[3] = 1.0
    token = check_sample(cx, x, f(rng.uniform(0, 0.999, rows)), t, k, p, mp)
    assert token[7] == -1 and token[9] == 17


@pytest.mark.parametrize("vocab", [40, 3266, 20000])
def test_sample_few_allowed(cx, vocab):
    """Rows that allow fewer tokens than top_k, one to thirty, spread over the whole row or all at its end."""
    rng = np.random.default_rng(vocab)
    for kw in (dict(k=50, p=0.9), dict(p=0.9), dict(k=2, p=0.99), dict(k=1500, p=0.7), dict(mp=0.3)):
        x = np.full((6, vocab), -np.inf, np.float32)
        for r in range(6):
            at = rng.choice(vocab, 1 + 5 * r, replace=False) if r % 2 else np.arange(vocab - 1 - 5 * r, vocab)
            x[r, at] = rng.normal(0, 2, len(at))
        u = torch.from_numpy(rng.uniform(0, 0.999, 6).astype(np.float32)).cuda()
        check_sample(cx, torch.from_numpy(x).cuda(), u, **kw)


@pytest.mark.parametrize("xt", ["f32", "f16"])
def test_sample_long_rows(cx, xt):
    """Rows longer than a cluster of blocks holds, and the longest that it does."""
    rng = np.random.default_rng(8)
    for vocab in (262144, 262145, 400001):
        x = torch.from_numpy(rng.normal(0, 1.5, (2, vocab)).astype(np.float32)).to(TYPES[xt]).cuda()
        u = torch.from_numpy(rng.uniform(0, 0.999, 2).astype(np.float32)).cuda()
        for kw in (dict(t=0.6, k=50, p=0.95), dict(t=0.8, p=0.9), dict(k=3000, p=0.8, mp=0.001)):
            check_sample(cx, x, u, **kw)


@pytest.mark.parametrize("vocab", [262145, 600000, 1 << 20])
def test_sample_long_rows_of_ties_and_masks(cx, vocab):
    """Rows longer than a cluster holds: all equal, a few values, only some allowed, one allowed, none allowed, and NaN."""
    rng = np.random.default_rng(vocab)
    x = np.full((6, vocab), -np.inf, np.float32)
    x[0] = 3.0
    x[1] = rng.integers(0, 4, vocab)
    some = rng.choice(vocab, 700, replace=False)
    x[2, some] = rng.normal(0, 1, 700)
    x[3, vocab - 1] = -5.0
    x[5] = rng.normal(0, 1, vocab)
    x[5, ::2] = np.nan
    x = torch.from_numpy(x).cuda()
    u = torch.from_numpy(rng.uniform(0, 0.999, 6).astype(np.float32)).cuda()
    for kw in (dict(), dict(k=1000), dict(k=40, p=0.5), dict(t=0.0), dict(p=0.3)):
        token = check_sample(cx, x, u, **kw)
        assert token[3] == vocab - 1 and token[4] == -1
    k = torch.tensor([5, 1, 701, 7, 3, 0], dtype=torch.int32, device="cuda")
    assert check_sample(cx, x, u, k=k)[0] < 5


@pytest.mark.parametrize("xt", ["f32", "bf16"])
@pytest.mark.parametrize("vocab", [6, 100, 2049, 5000, 70001])
def test_sample_ties_by_index(cx, vocab, xt):
    """All logits equal: weights are 1, so every answer is exact: kept are the first k, or the first ceil(p vocab), and the
    token is floor(u kept)."""
    from fhessm import client
    u = torch.tensor([0.0, 0.25, 0.5, 0.75, 0.984375], device="cuda")
    x = torch.full((5, vocab), -1.5, dtype=TYPES[xt], device="cuda")
    run = lambda **kw: client.sample(cx, x, u, **kw)
    for kw, kept in [({}, vocab), (dict(top_k=5), 5), (dict(top_k=vocab // 2 + 1), vocab // 2 + 1),
                     (dict(top_p=0.5), -(-vocab // 2)), (dict(top_p=0.25), -(-vocab // 4)), (dict(min_p=1.0), vocab),
                     (dict(temperature=0.0), 1), (dict(top_k=4, top_p=0.5), 2)]:
        token, lp = run(**kw)
        assert token.tolist() == [int(np.floor(v * kept)) for v in u.tolist()], kw
        assert np.abs(lp.cpu().numpy() + np.log(kept)).max() <= 2.0 ** -22 * max(1.0, np.log(kept))
    # -0 and 0 are one value
    x[:, 0::2], x[:, 1::2] = 0.0, -0.0
    assert run(top_k=2)[0].tolist() == [0, 0, 1, 1, 1]


def test_sample_extremes(cx):
    from fhessm import client
    inf = float("inf")
    x = torch.tensor([[-inf, 3.0, inf, 1.0, inf],               # infinite logits share everything
                      [3.0e38, -3.0e38, 0.0, 3.0e38, -inf],      # differences beyond float32
                      [float("nan")] * 4 + [2.0],
                      [1e-40, 0.0, -1e-40, -inf, -inf]], device="cuda")
    u = torch.tensor([0.75, 0.25, 0.9, 0.5], device="cuda")
    for t in (1.0, 1e-30, 1e30):
        token, lp = client.sample(cx, x, u, temperature=t)
        assert token[0] == 4 and token[2] == 4 and token[3] in (0, 1)
        if t < 1e29:
            assert token[1] == 0
        assert abs(lp[0].item() + np.log(2)) < 1e-6 and lp[2] == 0
    assert client.sample(cx, x, u, temperature=0.0)[0].tolist() == [2, 0, 4, 0]
    # random numbers outside [0, 1) are clamped
    token, _ = client.sample(cx, torch.zeros(3, 10, device="cuda"), torch.tensor([-1.0, 1.0, float("nan")], device="cuda"))
    assert token.tolist() == [0, 9, 0]


def test_sample_frequencies(cx):
    """Over 4096 evenly spaced random numbers each token is drawn as often as its probability says, to within one."""
    from fhessm import client
    n = 4096
    logits = torch.tensor([0.0, 1.0, 2.0, -1.0, 1.0], device="cuda")
    token, lp = client.sample(cx, logits.expand(n, 5).contiguous(), (torch.arange(n, device="cuda") + 0.5) / n)
    prob = torch.softmax(logits.double(), 0)
    assert ((torch.bincount(token, minlength=5) - n * prob).abs() <= 1).all()
    assert torch.allclose(lp.double(), prob.log()[token], atol=1e-6, rtol=0)


def test_calls_follow_the_current_stream(cx):
    """Inputs made on a side stream behind a long queue, operators on that stream: no other ordering is needed."""
    from fhessm import client
    rng = np.random.default_rng(3)
    t, w = make_table(rng, 2000, 512, 64)
    x = torch.from_numpy(rng.normal(0, 1, (16, 512)).astype(np.float32)).cuda()
    u = torch.rand(16, device="cuda")
    want = client.q4_matvec(cx, x, t)
    tok, lp = client.sample(cx, want, u, top_k=20)
    rows = client.q4_rows(cx, tok, t)
    big = torch.randn(4096, 4096, device="cuda")
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for _ in range(10):
            big = big @ big * 1e-3
        x2 = x + 0 * big[:16, :512].nan_to_num(0, 0, 0)
        got = client.q4_matvec(cx, x2, t)
        tok2, lp2 = client.sample(cx, got, u, top_k=20)
        rows2 = client.q4_rows(cx, tok2, t)
    side.synchronize()
    assert torch.equal(got, want) and torch.equal(tok, tok2) and torch.equal(lp, lp2) and torch.equal(rows, rows2)


def test_calls_on_the_context_stream_and_in_a_graph(cx):
    """The C-ABI's NULL stream is the context's own; a captured graph replays the whole step on new inputs."""
    import fhessm
    from fhessm import client
    rng = np.random.default_rng(4)
    t, w = make_table(rng, 3000, 256, 32)
    x = torch.from_numpy(rng.normal(0, 1, (8, 256)).astype(np.float32)).cuda()
    u = torch.rand(8, device="cuda")
    out = torch.empty(8, 3000, device="cuda")
    torch.cuda.synchronize()
    h = client._sigs()
    before = cx.launches()
    assert h.fhe_q4_matvec(cx.h, t.c, x.data_ptr(), 0, 256, 8, out.data_ptr(), 0, 3000, None) == 0
    cx.sync()
    assert cx.launches() > before
    assert torch.equal(out, client.q4_matvec(cx, x, t))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        logits = client.q4_matvec(cx, x, t)
        tok, lp = client.sample(cx, logits, u, temperature=0.8, top_k=40, top_p=0.9)
        rows = client.q4_rows(cx, tok, t)
    for _ in range(3):
        x.copy_(torch.from_numpy(rng.normal(0, 1, (8, 256)).astype(np.float32)))
        u.copy_(torch.rand(8))
        g.replay()
        want = client.q4_matvec(cx, x, t)
        assert torch.equal(logits, want)
        tok2, lp2 = client.sample(cx, want, u, temperature=0.8, top_k=40, top_p=0.9)
        assert torch.equal(tok, tok2) and torch.equal(lp, lp2)
        assert torch.equal(rows, client.q4_rows(cx, tok2, t))


def test_empty_calls(cx):
    from fhessm import client
    rng = np.random.default_rng(4)
    t, _ = make_table(rng, 30, 64, 32)
    assert client.q4_matvec(cx, torch.empty(0, 64, device="cuda"), t).shape == (0, 30)
    assert client.q4_rows(cx, torch.empty(0, dtype=torch.int64, device="cuda"), t).shape == (0, 64)
    token, lp = client.sample(cx, torch.empty(0, 5, device="cuda"), torch.empty(0, device="cuda"))
    assert token.shape == (0,) and lp.shape == (0,)
    none = client.Q4Table(t.weight[:0], t.scale[:0], cols=64, group=32)
    assert client.q4_matvec(cx, torch.ones(2, 64, device="cuda"), none).shape == (2, 0)
    assert (client.q4_rows(cx, torch.tensor([0, -1], device="cuda"), none) == 0).all()


def test_refusals(cx):
    from fhessm import FheError, client
    rng = np.random.default_rng(5)
    t, _ = make_table(rng, 30, 64, 32)
    x, u = torch.ones(2, 64, device="cuda"), torch.zeros(2, device="cuda")
    ids, lg = torch.zeros(2, dtype=torch.int64, device="cuda"), torch.zeros(2, 10, device="cuda")
    raw = torch.zeros(30 * 32 + 8, dtype=torch.uint8, device="cuda")[8:].view(30, 32)    # 8-byte aligned only
    for call in [lambda: client.q4_matvec(cx, x[:, :63], t), lambda: client.q4_matvec(cx, x.double(), t),
                 lambda: client.q4_matvec(cx, x.cpu(), t), lambda: client.q4_matvec(cx, x.T.contiguous().T, t),
                 lambda: client.q4_matvec(cx, x[0], t), lambda: client.q4_matvec(cx, x, t.to("cpu")),
                 lambda: client.q4_matvec(cx, x, t, dtype=torch.float64),
                 lambda: client.q4_matvec(cx, x, t, out=torch.empty(2, 31, device="cuda")),
                 lambda: client.q4_matvec(cx, x, t, out=torch.empty(2, 30)),
                 lambda: client.q4_matvec(cx, x.expand(4, 2, 64)[:, 0], t),
                 lambda: client.q4_matvec(cx, x, client.Q4Table(raw, t.scale, cols=64, group=32)),
                 lambda: client.q4_rows(cx, ids.int(), t), lambda: client.q4_rows(cx, ids.cpu(), t),
                 lambda: client.q4_rows(cx, ids.view(1, 2), t), lambda: client.q4_rows(cx, ids, t, dtype=torch.int32),
                 lambda: client.sample(cx, lg, u[:1]), lambda: client.sample(cx, lg, u.double()),
                 lambda: client.sample(cx, lg, 0.5), lambda: client.sample(cx, lg.cpu(), u),
                 lambda: client.sample(cx, lg.int(), u), lambda: client.sample(cx, lg, u, temperature=-0.5),
                 lambda: client.sample(cx, lg, u, temperature=float("nan")),
                 lambda: client.sample(cx, lg, u, top_k=-1), lambda: client.sample(cx, lg, u, top_p=0.0),
                 lambda: client.sample(cx, lg, u, top_p=1.5), lambda: client.sample(cx, lg, u, min_p=-0.1),
                 lambda: client.sample(cx, lg, u, min_p=1.5), lambda: client.sample(cx, lg, u, top_k=ids),
                 lambda: client.sample(cx, lg, u, temperature=torch.ones(3, device="cuda")),
                 lambda: client.sample(cx, torch.zeros(2, 0, device="cuda"), u),
                 lambda: client.sample(cx, torch.zeros(1, (1 << 20) + 1, device="cuda"), u[:1])]:
        with pytest.raises(FheError):
            call()
    h = client._sigs()
    many = torch.zeros((1 << 21) + 1, 32, dtype=torch.bfloat16, device="cuda")
    small, _ = make_table(rng, 1, 32, 32)
    with pytest.raises(FheError):
        client.q4_matvec(cx, many, small)
    assert (client.q4_matvec(cx, many[:1 << 21], small) == 0).all()
    host = np.zeros((2, 64), np.float32)
    out = torch.empty(2, 30, device="cuda")
    assert h.fhe_q4_matvec(cx.h, t.c, host.ctypes.data, 0, 64, 2, out.data_ptr(), 0, 30, None) == -1
    assert h.fhe_q4_matvec(cx.h, t.c, x.data_ptr(), 3, 64, 2, out.data_ptr(), 0, 30, None) == -1
    assert h.fhe_q4_matvec(cx.h, t.c, x.data_ptr(), 0, 63, 2, out.data_ptr(), 0, 30, None) == -1
    assert h.fhe_q4_matvec(cx.h, t.c, x.data_ptr(), 0, 64, 2, out.data_ptr(), 0, 29, None) == -1
    assert h.fhe_q4_matvec(cx.h, t.c, x.data_ptr(), 0, 64, -1, out.data_ptr(), 0, 30, None) == -1
    assert h.fhe_q4_matvec(cx.h, t.c, x.data_ptr() + 2, 0, 64, 1, out.data_ptr(), 0, 30, None) == -1
    assert h.fhe_q4_matvec(cx.h, t.c, None, 0, 64, 2, out.data_ptr(), 0, 30, None) == -1


def test_encrypted_decode_loop():
    """The small encrypted model decoding with a 4-bit tied table: each tick's decrypted rows go through the head, the choice
    and the look-up on the GPU, and the looked-up rows are encrypted as the next tick's input.  The tokens are the float64
    model's on the same table (its rows agree to 1e-3 rms, so tokens may differ where a decision is that close)."""
    import fhessm
    from fhessm.client import Q4Table, TokenHead
    from fhessm.model import (EncryptedModel, ModelConfig, calibrate_seeds, pack_lanes, plain_step, rel_err_rms,
                              synthetic_weights, unpack_lanes)
    cfg = ModelConfig(d=48, dff=128, n_layer=2, vocab=512, D=64, b1=8)
    w = synthetic_weights(cfg, seed=5)
    table = Q4Table.quantise(w["emb"], group=32)
    w["emb"] = table.dequantise().double().numpy()
    seeds = calibrate_seeds(cfg, w, steps=3, lanes=128)
    cx = fhessm.CryptoContext(logN=13, L=28, K=4, alpha=4, hw=192, boot_primes=14)
    cx.KeyGen(seed=9)
    cx.EvalBootstrapSetup(24.0, 59)
    m = EncryptedModel(cx, cfg, w, seeds)
    m.keygen()
    head = TokenHead(cx, table)
    lanes = 2 * cx.slots // cfg.D
    rng = np.random.default_rng(3)
    tokens = torch.from_numpy(rng.integers(0, cfg.vocab, lanes)).cuda()
    x, state = head.embed(tokens), None
    assert np.array_equal(x.double().cpu().numpy(), w["emb"][tokens.cpu().numpy()])
    for tick in range(2):
        rows = x.double().cpu().numpy()
        out = m.step(cx.Encrypt(cx.MakeCKKSPackedPlaintext(pack_lanes(rows, cfg.D, cx.slots))))
        y = unpack_lanes(cx.Decrypt(out), cfg.D, lanes, cfg.d)
        ref, state = plain_step(cfg, w, rows, state)
        u = torch.from_numpy(rng.uniform(0, 1, lanes).astype(np.float32)).cuda()
        tokens, lp, x = head.step(y, u, temperature=0.8, top_k=40, top_p=0.95)
        assert rel_err_rms(head.logits(y).double().cpu().numpy(), ref @ w["emb"].T) < 1e-3
        greedy, _, _ = head.step(y, u, temperature=0.0)
        assert np.mean(greedy.cpu().numpy() == (ref @ w["emb"].T).argmax(-1)) >= 0.98
        assert np.array_equal(x.double().cpu().numpy(), w["emb"][tokens.cpu().numpy()])
        assert torch.isfinite(lp).all() and (lp <= 0).all()
    cx.close()
