"""Log probabilities, entropy and alternatives of rows of logits in 64 bits, with
bounds on what 32-bit arithmetic may be off."""
import numpy as np

U = 2.0 ** -24


def answer(x, tokens):
    """(lp, its bound, entropy, its bound) of finite rows or rows with -infinity, x [rows, cols] float32."""
    x = x.astype(np.float64)
    top = x.max(1, keepdims=True)
    d = x - top
    e = np.exp(d)
    e[np.arange(len(x)), d.argmax(1)] = 0.0
    far = np.where(e > 0, -d, 0.0)
    rest = e.sum(1)
    slope, square = (e * far).sum(1), (e * far * far).sum(1)
    more = np.log1p(rest)
    # a term: its difference and the scaling by log2(e) each rounded, twice where parts are met, and the exponential;
    # the additions of 32 values a lane, a wave's lanes, and parts; then log1p and the last difference
    off = U * (6 * slope + 110 * rest) + 1e-37
    lp = np.take_along_axis(d, tokens.astype(np.int64), 1) - more[:, None]
    with np.errstate(invalid="ignore"):
        bound = U * (np.abs(np.take_along_axis(d, tokens.astype(np.int64), 1)) + np.abs(lp) + 6 * more[:, None]) + (
            off / (1 + rest))[:, None]
    entropy = more + slope / (1 + rest)
    # the rest's share in both, and the slope's own terms
    eb = 2 * off / (1 + rest) + off * slope / (1 + rest) ** 2 + U * ((6 * square + 114 * slope) / (1 + rest) + 8 * entropy)
    return lp, bound, entropy, eb


def order(x):
    """Ids by logit, greatest first, of equals the lowest, NaN last."""
    key = np.where(np.isnan(x), np.inf, -x.astype(np.float64))
    group = np.isnan(x).astype(int)
    return np.stack([np.lexsort((np.arange(x.shape[1]), key[r], group[r])) for r in range(len(x))])
