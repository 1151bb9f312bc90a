"""The choice of a token where the histogram's way leaves its short list: flat rows without ties, and a search that misses."""
import numpy as np
import pytest
import torch

from test_gpu_client import check_sample

pytestmark = pytest.mark.gpu

LIST = 2560     # tokens that a selection holds


@pytest.fixture(scope="module")
def cx():
    import fhessm
    c = fhessm.CryptoContext(logN=12, L=2, K=1, alpha=1, hw=64)
    yield c
    c.close()


def bins(e):
    """The histogram's bin of each exponential (float32): 128 an octave, from 1 down."""
    return ((0x3fffffff - e.view(np.uint32).astype(np.int64)) >> 16) - 120


def search(e, p):
    """(bin of the last token that top_p keeps, bin in which the histogram's sums, 16 bits of each e, place it)."""
    order = np.argsort(-e, kind="stable")
    weight = np.rint(e.astype(np.float64)[order] * 2.0 ** 40).astype(object)
    total = int(weight.sum())
    want = int(np.ceil(np.float64(np.float32(p)) * float(total)))
    kept = int(np.searchsorted(np.cumsum(weight.astype(np.float64)), want))
    ranked, b = e[order], bins(e[order])
    short = (ranked.view(np.uint32) & 0xffffff00).view(np.float32).astype(np.float64) * 2.0 ** 40
    lack = np.float32(total - int(short.sum())) / np.float32(total)
    guess = want - int(np.float32(want) * lack)
    return b[kept], b[min(len(b) - 1, int(np.searchsorted(np.cumsum(short), guess)))], b


@pytest.mark.parametrize("vocab,spread,t,p", [(131072, 0.6, 2.0, 0.4), (50304, 0.3, 2.0, 0.5), (65536, 0.3, 2.0, 0.5),
                                              (50304, 0.1, 1.0, 0.5), (50277, 0.1, 2.0, 0.9), (262144, 0.6, 1.3, 0.6)])
def test_flat_rows_without_ties(cx, vocab, spread, t, p):
    """The three bins around the last kept token hold more tokens than the list, all of them different."""
    rng = np.random.default_rng(vocab)
    x = rng.normal(0, spread, (2, vocab)).astype(np.float32)
    assert len(np.unique(x[0])) > 0.9 * vocab
    e = np.exp((x[0] - x[0].max()) / np.float32(t))
    at, _, b = search(e, p)
    assert (np.abs(b - at) <= 1).sum() > LIST
    u = torch.from_numpy(rng.uniform(0, 0.999, 2).astype(np.float32)).cuda()
    check_sample(cx, torch.from_numpy(x).cuda(), u, t=t, p=p)
    check_sample(cx, torch.from_numpy(x).cuda(), u, t=t, p=p, k=vocab // 2)


def test_a_search_that_misses(cx):
    """Half of the weight in tokens whose exponentials lose most in the histogram's 16 bits, half in tokens that lose nothing, and
    single tokens between them: the histogram places the last kept token ten bins too low."""
    value = lambda bits: np.uint32(bits).view(np.float32)
    near = [value(0x3f7ffff0), value(0x3f000004)]
    logs = [np.float32(np.log(np.float64(v))) for v in near]
    sparse = np.array([0.9, 0.85, 0.8, 0.75, 0.7], np.float32)
    vocab = 60006
    x = np.empty((3, vocab), np.float32)
    x[:, 0] = 0.0
    x[:, 1:30001], x[:, 30001:60001] = logs
    x[:, 60001:] = np.log(sparse.astype(np.float64))
    e = np.exp(x[0])
    top = e[:30001].astype(np.float64).sum()
    p = np.float32((top + 0.85) / e.astype(np.float64).sum())
    at, placed, b = search(e, p)
    assert at == bins(e[60001:60002])[0] and abs(placed - at) >= 2
    # the first of the single tokens, the last before it, and the first of all
    u = torch.tensor([(top + 0.5) / (top + 0.9), (top - 0.5) / (top + 0.9), 0.0], dtype=torch.float32, device="cuda")
    token = check_sample(cx, torch.from_numpy(x).cuda(), u, p=float(p))
    assert token.tolist() == [60001, 30000, 0]
