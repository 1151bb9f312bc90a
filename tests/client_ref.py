"""The client operators' definitions in numpy float64, and the inputs their tests share."""
import numpy as np

# An exponential in float32 is off by at most 2 units of 2^-23, a weight's rounding to 2^-40 of the largest by 2^-41 for each of at
# most 2^17 tokens: sums of weights agree with float64 to 2^-22 + 2^-24; decisions within four times that are open.
OPEN = 2.0 ** -20


def table_values(q, scale, cols, group):
    """q: (rows, columns) whole numbers 0..15; scale (rows, groups)."""
    return (q[:, :cols].astype(np.float64) - 8) * np.repeat(scale.astype(np.float64), group, axis=1)[:, :cols]


def pack(q):
    """Two values a byte, the even column in the low half; q's columns are a multiple of 32."""
    return (q[:, 0::2] | q[:, 1::2] << 4).astype(np.uint8)


def sample_row(x, u, t, k, p, mp, order=None):
    """(token, log-probability, mask of the kept) of one row of float64 logits holding the values of the inputs'
    type.  z is rounded as in float32, which the definition says; everything after it is float64."""
    x = np.where(np.isnan(x), -np.inf, x)
    top = x.max()
    if top == -np.inf:
        return -1, -np.inf, np.zeros(len(x), bool)
    if not t > 0:
        t, k = 1.0, 1
    with np.errstate(invalid="ignore", over="ignore"):
        x32 = x.astype(np.float32)
        z = np.where(x == top, np.float32(0), (x32 - np.float32(top)) / np.float32(t)).astype(np.float64)
    z = np.where(x == -np.inf, -np.inf, z)
    e = np.exp(z)
    if order is None:
        order = np.lexsort((np.arange(len(x)), -x))
    ranked = e[order]
    keep = np.ones(len(x), bool)
    if k > 0:
        keep[k:] = False
    if p < 1:
        before = np.concatenate([[0.0], np.cumsum(ranked)[:-1]])
        keep &= before < p * ranked[keep].sum()
        keep[0] = True
    keep &= ranked >= mp
    keep &= ranked > 0
    mask = np.zeros(len(x), bool)
    mask[order[keep]] = True
    run = np.cumsum(np.where(mask, e, 0))
    token = int(np.argmax(run > min(max(u, 0.0), np.nextafter(1.0, 0.0)) * run[-1]))
    return token, float(z[token] - np.log(run[-1])), mask


def sample_accepts(x, u, t, k, p, mp, token):
    """Whether `token` is the definition's, decisions that lie within OPEN of their limits going either way; and the
    log-probability that belongs to it (or to the nearest such decision)."""
    want, lp, _ = sample_row(x, u, t, k, p, mp)
    if token == want:
        return True, lp
    xs = np.where(np.isnan(x), -np.inf, x)
    order = np.lexsort((np.arange(len(x)), -xs))
    for dp in (0, -OPEN, OPEN):
        for dm in (0, -OPEN, OPEN):
            pp = p if p >= 1 else p * (1 + dp)
            lo, _, mask = sample_row(x, u - OPEN, t, k, pp, mp * (1 + dm), order)
            hi, lp, _ = sample_row(x, u + OPEN, t, k, pp, mp * (1 + dm), order)
            if lo <= token <= hi and mask[token]:
                return True, None
    return False, lp
