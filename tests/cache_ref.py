"""The 4-bit cache of keys and values in numpy, in 64 bits and written from its
definition (include/pk_hip.h): what a value is kept as, where a record keeps
it, and the attention with a bound on what 32-bit arithmetic may be off."""
import numpy as np

PAGE = 64
LEVELS = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])


def record_bytes(dk):
    return PAGE * dk + 4 * PAGE


def bf16_bits(d):
    """The bfloat16 bits of float32 values that are one."""
    u = np.ascontiguousarray(d, dtype=np.float32).view(np.uint32)
    assert not (u & 0xffff).any()
    return (u >> 16).astype(np.uint16)


def scale_of(top):
    """The least bfloat16 d with 6 d >= top, or 0 where a head is kept as zeros."""
    if not (2.0 ** -121 <= top < 2.0 ** 127):
        return 0.0
    place = 2.0 ** (np.floor(np.log2(float(top) / 6.0)) - 8)
    d = np.floor(float(top) / 6.0 / place) * place          # finer than a bfloat16 by one place, at most
    while True:
        b = np.float32(d).view(np.uint32)
        if not b & 0xffff and 6.0 * float(d) >= float(top):
            return float(d)
        d += place


def codes_of(x, d):
    """The codes of x at scale d: nearest level, ties to the even code."""
    if d == 0.0:
        return np.zeros(x.shape, np.uint8)
    off = np.abs(np.abs(x.astype(np.float64))[..., None] / d - LEVELS)
    near = off == off.min(-1, keepdims=True)
    c = np.where(near, np.arange(8) % 2, 2).argmin(-1).astype(np.uint8)
    return np.where((x < 0) & (c > 0), c + 8, c).astype(np.uint8)


def kept(x, heads):
    """(values, codes, scales [rows, heads]) that x [rows, heads * dk] is kept as."""
    a = x.reshape(x.shape[0], heads, -1)
    d = np.zeros(a.shape[:2])
    codes = np.zeros(a.shape, np.uint8)
    for r in range(a.shape[0]):
        for h in range(heads):
            top = np.abs(a[r, h]).max()
            d[r, h] = scale_of(top)
            codes[r, h] = codes_of(a[r, h], d[r, h])
    v = LEVELS[codes & 7] * np.where(codes & 8, -1.0, 1.0) * d[..., None]
    return v.reshape(x.shape), codes, d


class Pool:
    """A pool's bytes [layers, pages, heads, record] on the host."""

    def __init__(self, layers, pages, heads, dk, fill=0xff):
        self.heads, self.dk = heads, dk
        self.data = np.full((layers, pages, heads, record_bytes(dk)), fill, np.uint8)

    def _value_at(self, f, c):
        g, h, w, r = f // 32, f // 16 % 2, f // 4 % 4, f % 4
        n = 4 * h + r
        return (PAGE * self.dk // 2 + 1024 * (c // 32) + 16 * (16 * w + c % 16) + 8 * (c // 16 % 2) + 4 * g + n // 2,
                4 * (n % 2))

    def write(self, layer, page, frame, k, v):
        """One frame's keys and values [heads * dk]."""
        for which, x in ((0, k), (1, v)):
            _, codes, d = kept(x[None], self.heads)
            for h in range(self.heads):
                rec = self.data[layer, page, h]
                at = PAGE * self.dk + 128 * which + 2 * frame
                rec[at:at + 2] = bf16_bits(np.float32(d[0, h])).reshape(1).view(np.uint8)
                for c in range(self.dk):
                    byte, shift = self._value_at(frame, c) if which else (frame * (self.dk // 2) + c // 2, 4 * (c % 2))
                    rec[byte] = rec[byte] & ~np.uint8(15 << shift) & 0xff | np.uint8(int(codes[0, h, c]) << shift)

    def read(self, layer, page, head):
        """The record's keys and values [64, dk] (finite only where written)."""
        rec = self.data[layer, page, head]
        f, c = np.arange(PAGE)[:, None], np.arange(self.dk)[None]
        kc = rec[f * (self.dk // 2) + c // 2] >> (4 * (c % 2)) & 15
        at, shift = self._value_at(f, c)
        vc = rec[at] >> shift & 15
        d = (rec[PAGE * self.dk:].copy().view(np.uint16).astype(np.uint32) << 16).view(np.float32).astype(np.float64)
        val = lambda x: LEVELS[x & 7] * np.where(x & 8, -1.0, 1.0)
        return val(kc) * d[:PAGE, None], val(vc) * d[PAGE:, None]


def attend(pool, layer, table, lens, row0, rows, q, H, positions=None, left=None, right=None):
    """The attention of q [rows, H * dk] in 64 bits, and a bound on how far a
    32-bit one may be off: two arrays [rows, H * dk], NaN where no stream has the
    row. positions is (p, center, u, w)."""
    G, dk = pool.heads, pool.dk
    pages = pool.data.shape[1]
    out = np.full((rows, H * dk), np.nan)
    bound = np.zeros((rows, H * dk))
    u = 2.0 ** -23            # a rounding or a truncation of a 32-bit sum
    for b, n0 in enumerate(lens):
        T = row0[b + 1] - row0[b]
        total = min(n0 + T, table.shape[1] * PAGE)
        for g in range(G):
            k, v = np.zeros((total, dk)), np.zeros((total, dk))
            there = np.zeros(total, bool)
            for pg in range(-(-total // PAGE)):
                if 0 <= table[b, pg] < pages:
                    kk, vv = pool.read(layer, table[b, pg], g)
                    e = min(total, PAGE * (pg + 1))
                    k[PAGE * pg:e], v[PAGE * pg:e] = kk[:e - PAGE * pg], vv[:e - PAGE * pg]
                    there[PAGE * pg:e] = True
            for h in range(g * (H // G), (g + 1) * (H // G)):
                cols = slice(h * dk, (h + 1) * dk)
                for t in range(T):
                    row, pos = row0[b] + t, n0 + t
                    j = np.arange(total)
                    see = there.copy()
                    lo, hi = left, right
                    if positions is not None:
                        p, center, bu, bw = positions
                        lo = center if lo is None else min(lo, center)
                        hi = len(p) - 1 - center if hi is None else min(hi, len(p) - 1 - center)
                    if lo is not None:
                        see &= j >= pos - lo
                    if hi is not None:
                        see &= j <= pos + hi
                    j = j[see]
                    if not len(j):
                        out[row, cols] = 0
                        continue
                    x = q[row, cols].astype(np.float64)
                    c = x + (positions[2][cols].astype(np.float64) if positions is not None else 0)
                    s = k[j] @ c
                    mag = np.abs(k[j]) @ np.abs(c)
                    terms = 3 * dk
                    if positions is not None:
                        y = x + positions[3][cols].astype(np.float64)
                        pr = positions[0][positions[1] - (pos - j)][:, cols].astype(np.float64)
                        s = s + pr @ y
                        mag = mag + np.abs(pr) @ np.abs(y)
                        terms = 6 * dk
                    s, mag = s / np.sqrt(dk), mag / np.sqrt(dk)
                    e = np.exp(s - s.max())
                    w = e / e.sum()
                    out[row, cols] = w @ v[j]
                    # a score: the additions of its terms, the inputs' sums with the biases, the scalings; the
                    # softmax: the difference to the maximum, the exponential (its rescaling at each page once
                    # more), then the output's own terms and the division by a sum of as many
                    off = ((terms + 8) * u * mag).max()
                    soft = 4 * u * (np.abs(s).max() + 1) + 2 * off
                    more = (3 * len(j) + 4 * (len(j) // PAGE + 8)) * u
                    bound[row, cols] = (np.exp(soft + more) - 1) * 2 * (w @ np.abs(v[j])) + 1e-37
    return out, bound
