"""Attention with a sliding window and sinks in numpy, in 64 bits and written from
its definition (include/pk_hip.h), with a bound on what 32-bit arithmetic may be
off."""
import numpy as np

U = 2.0 ** -23              # a rounding or a truncation of a 32-bit sum


def reach(positions, left, right):
    """The window that is asked, no wider than the positions' table; None for no end."""
    if positions is None:
        return left, right
    p, center = positions[:2]
    ahead = len(p) - 1 - center
    return (center if left is None else min(left, center)), (ahead if right is None else min(right, ahead))


def attended(pos, frames, left, right, sinks):
    """Which of the frames (numbers of a stream or segment) a row at pos attends."""
    see = np.ones(len(frames), bool)
    if left is not None:
        see &= (frames >= pos - left) | (frames < sinks)
    if right is not None:
        see &= frames <= pos + right
    return see


def attend(q, first, frames, k, v, H, dk, positions=None, left=None, right=None, sinks=0):
    """Rows q [T, H * dk] at positions first on, over frames with keys and values k, v [n, G * dk]: the outputs and a
    bound, two arrays [T, H * dk]. positions is (p, center, u, w)."""
    left, right = reach(positions, left, right)
    G = k.shape[1] // dk
    out, bound = np.zeros(q.shape), np.zeros(q.shape)
    for t in range(len(q)):
        pos = first + t
        at = np.flatnonzero(attended(pos, frames, left, right, sinks))
        if not len(at):
            continue
        for h in range(H):
            c, g = slice(h * dk, (h + 1) * dk), slice(h // (H // G) * dk, (h // (H // G) + 1) * dk)
            x = q[t, c].astype(np.float64)
            kk, vv = k[at, g].astype(np.float64), v[at, g].astype(np.float64)
            y = x + (positions[2][c].astype(np.float64) if positions is not None else 0)
            s, mag, terms = kk @ y, np.abs(kk) @ np.abs(y), 3 * dk
            if positions is not None:
                dist = pos - frames[at]
                if left is not None:
                    dist = np.minimum(dist, left)
                y = x + positions[3][c].astype(np.float64)
                p = positions[0][positions[1] - dist][:, c].astype(np.float64)
                s, mag, terms = s + p @ y, mag + np.abs(p) @ np.abs(y), 6 * dk
            s, mag = s / np.sqrt(dk), mag / np.sqrt(dk)
            e = np.exp(s - s.max())
            w = e / e.sum()
            out[t, c] = w @ vv
            # a score: the additions of its terms, the inputs' sums with the biases, the scalings; the softmax: the
            # difference to the maximum and the exponential (its rescaling once more for each run of frames), then the
            # output's own terms and the division by a sum of as many
            off = ((terms + 8) * U * mag).max()
            soft = 4 * U * (np.abs(s).max() + 1) + 2 * off
            more = (3 * len(at) + 4 * (len(at) // 16 + 8)) * U
            bound[t, c] = (np.exp(soft + more) - 1) * 2 * (w @ np.abs(vv)) + 1e-37
    return out, bound
