"""The 4-bit cache of keys and values on the GPU: writes, reads and moves byte for
byte against the host model, the attention against 64 bits within the bound
that 32-bit arithmetic gives (cache_ref.attend), and a stream's life through
all of them."""
import random
import sys

import numpy as np
import pytest

import cache_ref as cr

pytestmark = pytest.mark.gpu
DKS = (32, 64, 96, 128)


def say(*a):
    print("[case]", *a, flush=True)
    sys.stdout.flush()


@pytest.fixture(scope="module")
def torch():
    import torch
    assert torch.cuda.is_available()
    return torch


class World:
    """A cache on the device and its model on the host, with some streams."""

    def __init__(self, pk, torch, lens, Ts, G, dk, seed=0, layers=1, layer=0, first=0, tail=0, spare=2, max_pages=None,
                 slack_T=0):
        self.pk, self.torch, self.layer = pk, torch, layer
        self.g = np.random.default_rng(seed)
        self.G, self.dk, self.lens, self.Ts = G, dk, list(lens), list(Ts)
        B = len(lens)
        held = [-(-(a + t) // 64) for a, t in zip(lens, Ts)]
        mp = max_pages or max(1, max(held, default=1))
        ids = self.g.permutation(sum(held) + spare)
        self.table = np.full((B, mp), -1, np.int32)
        at = 0
        for b, h in enumerate(held):
            h = min(h, mp)
            self.table[b, :h] = ids[at:at + h]
            at += h
        self.row0 = np.cumsum([first] + self.Ts).astype(np.int32)
        self.rows = int(self.row0[-1]) + tail
        self.pool = cr.Pool(layers, len(ids), G, dk)
        self.max_T = min(self.rows, max(self.Ts, default=0) + slack_T)
        self.upload()

    def dev(self, a):
        return self.torch.from_numpy(np.ascontiguousarray(a)).cuda()

    def upload(self):
        d = self.pool.data
        self.data = self.dev(d)
        self.cache = self.pk.DeviceCache(self.data, *d.shape[:3], self.dk)
        self.streams = self.pk.CacheStreams(self.dev(self.table), self.dev(np.array(self.lens, np.int32)),
                                            self.dev(self.row0), self.rows, self.max_T)

    def fill(self, upto=None, scale=1.0):
        """Random keys and values for every frame of every stream, on the host;
        frames of no stream keep bytes that are NaN as scales."""
        for b in range(len(self.lens)):
            total = self.lens[b] + self.Ts[b] if upto is None else upto[b]
            for f in range(min(total, 64 * self.table.shape[1])):
                pg = self.table[b, f // 64]
                if 0 <= pg < self.pool.data.shape[1]:
                    x = scale * self.g.standard_normal((2, self.G * self.dk))
                    self.pool.write(self.layer, pg, f % 64, *x.astype(np.float32))
        self.upload()

    def positions(self, H, back, ahead, biased=True):
        n = back + ahead + 1
        p = self.g.standard_normal((n, H * self.dk)).astype(np.float32)
        u, w = (0.3 * self.g.standard_normal((2, H * self.dk))).astype(np.float32)
        return p, back, u, w

    def attend(self, q, H, positions=None, left=None, right=None, layer=None):
        """The device's attention of q, into rows that hold a mark before."""
        torch = self.torch
        layer = self.layer if layer is None else layer
        pos = None if positions is None else (self.dev(positions[0]), positions[1], self.dev(positions[2]),
                                              self.dev(positions[3]))
        o = torch.full((self.rows, H * self.dk), 7.25, device="cuda")
        need = self.cache.attention_workspace(self.streams, H, pos, left, right)
        ws = torch.full((max(1, need),), 0xff, dtype=torch.uint8, device="cuda")
        self.cache.attention(o, layer, self.dev(q), self.streams, H, ws, pos, left, right)
        torch.cuda.synchronize()
        return o.cpu().numpy()

    def check(self, H, positions=None, left=None, right=None, qscale=1.0, q=None):
        if q is None:
            q = (qscale * self.g.standard_normal((self.rows, H * self.dk))).astype(np.float32)
        got = self.attend(q, H, positions, left, right)
        want, bound = cr.attend(self.pool, self.layer, self.table, self.lens, self.row0, self.rows, q, H, positions,
                                left, right)
        none = np.isnan(want)
        assert (got[none] == 7.25).all()            # rows of no stream: as they were
        off = np.abs(np.where(none, 0, got - np.where(none, 0, want)))
        assert np.isfinite(got).all()
        assert (off <= bound + none).all(), (off.max(), bound[off > bound].min())
        ref = np.linalg.norm(want[~none])
        assert np.linalg.norm(off[~none]) <= 1e-5 * ref + 1e-30
        return got


# ----------------------------------------------------------- write, read --

@pytest.mark.parametrize("dk", DKS)
@pytest.mark.parametrize("G", [1, 3])
def test_write_bytes(hip, torch, dk, G):
    """Streams that begin and end anywhere in a page: the bytes are the model's,
    and every byte that is not the call's keeps what it held."""
    say("write", dk, G)
    lens, Ts = [0, 1, 63, 64, 50, 0, 127, 3], [1, 2, 3, 64, 90, 0, 1, 130]
    w = World(hip, torch, lens, Ts, G, dk, seed=dk + G, layers=2, layer=1, first=2, tail=3)
    x = w.g.standard_normal((2, w.rows, G * dk)).astype(np.float32)
    x[0, 2, :5] = [0.0, -0.0, 1e-30, -1e-30, 2.0]
    x[:, 3] = 0.0
    x[0, 4, 0], x[1, 5, dk - 1], x[0, 6, 1] = np.nan, np.inf, -np.inf
    x[1, 7, 0] = 2.0 ** 127
    x[0, 8] *= np.float32(2.0 ** -124)
    w.cache.append(1, w.dev(x[0]), w.dev(x[1]), w.streams)
    ko, vo = (torch.full((w.rows, G * dk), 7.25, device="cuda") for _ in range(2))
    w.cache.read(1, ko, vo, w.streams)
    torch.cuda.synchronize()
    for b in range(len(lens)):
        for t in range(Ts[b]):
            f, r = lens[b] + t, w.row0[b] + t
            w.pool.write(1, w.table[b, f // 64], f % 64, x[0, r], x[1, r])
    assert np.array_equal(w.data.cpu().numpy(), w.pool.data)
    for got, which in ((ko, 0), (vo, 1)):
        got = got.cpu().numpy()
        want, _, _ = cr.kept(x[which], G)
        assert np.array_equal(got[2:w.row0[-1]], want[2:w.row0[-1]].astype(np.float32))
        assert (got[:2] == 7.25).all() and (got[w.row0[-1]:] == 7.25).all()


@pytest.mark.parametrize("T", [1, 2, 31, 64, 65, 200])
def test_write_in_pieces(hip, torch, T):
    """The same frames written in one call and in chunks of T: the same bytes."""
    say("pieces", T)
    G, dk, n = 2, 64, 201
    w = World(hip, torch, [0], [n], G, dk, seed=T)
    x = w.g.standard_normal((2, n, G * dk)).astype(np.float32)
    k, v = w.dev(x[0]), w.dev(x[1])
    w.cache.append(0, k, v, w.streams)
    whole = w.data.clone()
    w.data.fill_(0xff)
    length = torch.zeros(1, dtype=torch.int32, device="cuda")
    for a in range(0, n, T):
        m = min(T, n - a)
        st = hip.CacheStreams(w.streams.table, length, w.dev(np.array([0, m], np.int32)), m, m)
        w.cache.append(0, k[a:a + m], v[a:a + m], st)
        length += m
    assert torch.equal(w.data, whole)


def test_write_strides_and_holes(hip, torch):
    """Rows at strides, a table with entries outside the pool, frames past the
    table, a stream with more rows than max_T: nothing else is touched."""
    say("strides")
    G, dk = 2, 32
    w = World(hip, torch, [60, 10, 100], [80, 20, 70], G, dk, seed=3, max_pages=2)
    w.table[0, 1] = w.pool.data.shape[1]            # one past the pool
    w.table[2, 0] = -5
    w.max_T = 70
    w.upload()
    x = w.g.standard_normal((2, w.rows, G * dk + 12)).astype(np.float32)
    k, v = w.dev(x[0]), w.dev(x[1])
    w.cache.append(0, k[:, 4:4 + G * dk], v[:, 8:8 + G * dk], w.streams)
    for b in range(3):
        for t in range(min(70, w.Ts[b])):
            f, r = w.lens[b] + t, w.row0[b] + t
            if f < 128 and 0 <= w.table[b, f // 64] < w.pool.data.shape[1]:
                w.pool.write(0, w.table[b, f // 64], f % 64, x[0, r, 4:4 + G * dk], x[1, r, 8:8 + G * dk])
    assert np.array_equal(w.data.cpu().numpy(), w.pool.data)
    out = torch.full((2, w.rows, G * dk + 4), 7.25, device="cuda")
    w.cache.read(0, out[0, :, :G * dk], out[1, :, :G * dk], w.streams)
    got = out.cpu().numpy()
    assert (got[:, :, G * dk:] == 7.25).all()
    for which, cut in ((0, 4), (1, 8)):
        want, _, _ = cr.kept(x[which][:, cut:cut + G * dk], G)
        for b in range(3):
            for t in range(w.Ts[b]):
                f, r = w.lens[b] + t, w.row0[b] + t
                if t >= 70:
                    assert (got[which, r, :G * dk] == 7.25).all()
                elif f < 128 and 0 <= w.table[b, f // 64] < w.pool.data.shape[1]:
                    assert np.array_equal(got[which, r, :G * dk], want[r].astype(np.float32))
                else:
                    assert (got[which, r, :G * dk] == 0).all()


# ------------------------------------------------------------- attention --

@pytest.mark.parametrize("dk", DKS)
@pytest.mark.parametrize("H,G", [(1, 1), (4, 4), (6, 2), (3, 1)])
@pytest.mark.parametrize("with_positions", [False, True])
def test_attention(hip, torch, dk, H, G, with_positions):
    """Ragged streams from nothing to a few pages, a row gap at both ends."""
    say("attention", dk, H, G, with_positions)
    w = World(hip, torch, [0, 1, 63, 64, 130, 200, 0, 5], [1, 1, 1, 2, 17, 0, 40, 3], G, dk, seed=dk + H, first=1, tail=2)
    w.fill()
    pos = w.positions(H, 210, 60) if with_positions else None
    w.check(H, pos)


@pytest.mark.parametrize("left,right", [(0, 0), (3, 0), (None, 0), (0, None), (64, 5), (70, 63), (1 << 30, 1 << 30)])
@pytest.mark.parametrize("with_positions", [False, True])
def test_windows(hip, torch, left, right, with_positions):
    say("window", left, right, with_positions)
    w = World(hip, torch, [0, 90, 64, 150], [70, 33, 1, 2], 2, 64, seed=11)
    w.fill()
    w.check(4, w.positions(4, 160, 75) if with_positions else None, left, right)


@pytest.mark.parametrize("back,ahead", [(0, 0), (7, 0), (0, 9), (40, 3), (300, 200)])
def test_positions_table_bounds_the_window(hip, torch, back, ahead):
    """Distances that the table has no row for are not attended; rows of it
    that no frame needs may hold anything."""
    say("table", back, ahead)
    w = World(hip, torch, [100, 3], [20, 50], 2, 32, seed=12)
    w.fill()
    p, c, u, v = w.positions(2, back, ahead)
    if back >= 300:
        p[:c - 119] = np.nan
        p[c + 50:] = np.inf
    w.check(2, (p, c, u, v))


def test_single_frames(hip, torch):
    """One row a stream, many streams of every length around the pages."""
    say("single")
    lens = list(range(0, 140, 3)) + [320]
    w = World(hip, torch, lens, [1] * len(lens), 2, 128, seed=13)
    w.fill()
    w.check(2, w.positions(2, 320, 0))
    w.check(8)


@pytest.mark.parametrize("dk", DKS)
@pytest.mark.parametrize("B", [1, 5, 16, 17])
def test_single_frames_narrow(hip, torch, dk, B):
    """One row a stream and a narrow window, whose position scores are made
    where they are used (up to 16 streams, 100 distances), and on both sides
    of that."""
    say("narrow", dk, B)
    w = World(hip, torch, [(37 * b) % 150 for b in range(B)], [1] * B, 2, dk, seed=30 + B, first=1, tail=1)
    w.fill()
    for left in (0, 20, 70, 99, 100):
        w.check(2, w.positions(2, 160, 3), left, 0)
    p, c, u, v = w.positions(2, 40, 0)
    w.check(2, (p, c, u, v))
    w.table[0, :] = -1
    w.upload()
    w.check(2, (p, c, u, v))


@pytest.mark.parametrize("rows,lens,dk,H,G", [
    ([300, 240], [40, 0], 64, 2, 1),            # 540 rows: the table halved beforehand
    ([200, 320, 100, 7], [0, 3, 70, 5], 128, 1, 1),
    ([150, 20], [1300, 900], 32, 4, 2),         # many distances: 64 rows a workgroup
    ([90, 16], [1500, 10], 96, 3, 3),
])
@pytest.mark.parametrize("windowed", [False, True])
def test_many_rows_with_positions(hip, torch, rows, lens, dk, H, G, windowed):
    """The ways the position scores are made, by the call's rows and the table's
    reach."""
    say("many rows", rows, dk, H, windowed)
    w = World(hip, torch, lens, rows, G, dk, seed=40 + dk, first=3, tail=2)
    w.fill()
    far = max(a + t for a, t in zip(lens, rows))
    w.check(H, w.positions(H, far, max(rows)), *((50, 9) if windowed else (None, None)))


@pytest.mark.parametrize("qscale,pscale", [(1e-18, 1e18), (1e18, 1e-18), (1e-30, 1e30), (1e30, 1e-30)])
@pytest.mark.parametrize("T", [1, 7])
def test_position_magnitudes(hip, torch, qscale, pscale, T):
    """Queries and positions far from one and from each other: the exponents of
    their rows are put back at once."""
    say("position magnitudes", qscale, pscale, T)
    w = World(hip, torch, [100, 7], [T, T], 1, 64, seed=43)
    w.fill(scale=0.1 / qscale)              # so that neither part of a score is lost beside the other
    p, c, u, v = w.positions(1, 130, 10)
    p = (p * np.float32(pscale)).astype(np.float32)
    p[::3] *= np.float32(1e-3)
    w.check(1, (p, c, 0 * u, 0 * v), qscale=qscale)


def test_long_stream(hip, torch):
    """One row against 70 pages, and chunks against them."""
    say("long")
    for T in (1, 3, 30):
        w = World(hip, torch, [4470], [T], 1, 64, seed=14 + T)
        w.fill()
        w.check(1, w.positions(1, 4500, 30))
        w.check(4, left=2000)


@pytest.mark.parametrize("B,H,G,T,dk,pages", [
    (3, 2, 2, 1, 128, 12), (3, 2, 2, 3, 64, 22), (32, 8, 8, 1, 32, 44),     # tiles of four rows, eight waves
    (16, 8, 8, 1, 128, 33), (1, 2, 1, 2, 96, 300),                          # in splits of eight waves
    (19, 8, 8, 1, 64, 80), (12, 8, 8, 1, 32, 34),                           # in three and five splits of four
    (3, 2, 2, 20, 128, 9), (2, 2, 1, 64, 32, 31), (16, 8, 8, 17, 32, 33),   # tiles of 16 rows, eight waves
    (8, 8, 4, 9, 64, 35), (1, 1, 1, 40, 96, 120),                           # in splits
    (17, 8, 8, 16, 32, 81), (33, 8, 8, 1, 32, 40),                          # in three splits; more tiles than CUs
])
@pytest.mark.parametrize("with_positions", [False, True])
def test_pages_dealt(hip, torch, B, H, G, T, dk, pages, with_positions):
    """Each way that a tile's pages are dealt to waves and workgroups. All streams
    read one stream's pages, each with holes of its own; the last one has fewer."""
    say("dealt", B, H, G, T, dk, pages, with_positions)
    total = 64 * pages - 5
    w = World(hip, torch, [total - T] * (B - 1) + [total - T - (70 if B > 1 else 0)], [T] * B, G, dk, seed=pages)
    w.table[:] = w.table[0]
    w.fill(upto=[total] + [0] * (B - 1))
    for b in range(B):
        w.table[b, (7 * b + 3) % pages] = w.table[b, (11 * b + 1) % pages] = -1
    w.upload()
    w.check(H, w.positions(H, total, T) if with_positions else None)


@pytest.mark.parametrize("seed", range(24))
def test_any_call(hip, torch, seed):
    """Calls drawn over the documented ranges: streams, lengths, rows, heads,
    windows, holes, a table wider or narrower than the streams, the bound on a
    stream's rows above them."""
    r = random.Random(seed)
    dk, (H, G) = r.choice(DKS), r.choice([(1, 1), (2, 2), (4, 1), (6, 3), (5, 5)])
    B = r.choice([1, 2, 3, 7, 20])
    Ts = [r.choice([0, 1, 1, 2, 3, r.randint(1, 40)]) for _ in range(B)]
    if not sum(Ts):
        Ts[0] = 1
    lens = [r.choice([0, 1, 63, 64, 127, r.randint(0, 300), r.randint(0, 2500 // B)]) for _ in range(B)]
    say("any", seed, dk, H, G, lens, Ts)
    held = max(-(-(a + t) // 64) for a, t in zip(lens, Ts))
    w = World(hip, torch, lens, Ts, G, dk, seed=seed, layers=2, layer=r.randint(0, 1), first=r.randint(0, 2),
              tail=r.randint(0, 2), max_pages=held + r.randint(0, 3), slack_T=r.choice([0, 0, 5]))
    if r.random() < 0.4:
        for _ in range(r.randint(1, 4)):
            w.table[r.randrange(B), r.randrange(w.table.shape[1])] = r.choice([-1, -2 ** 31, 10 ** 6])
    w.fill(scale=r.choice([1.0, 0.01, 30.0]))
    left, right = (r.choice([None, 0, 1, 70, r.randint(0, 400)]) for _ in range(2))
    pos = None
    if r.random() < 0.6:
        far = max(a + t for a, t in zip(lens, Ts))
        pos = w.positions(H, r.choice([far, far + 9, far // 2]), r.choice([max(Ts), max(Ts) // 2, 50]))
    w.check(H, pos, left, right, qscale=r.choice([1.0, 0.1, 4.0]))


def test_rows_that_attend_nothing(hip, torch):
    """Holes in the table (given up pages, ids outside the pool, of every size):
    their frames are skipped, and a row with nothing else is zeros."""
    say("holes")
    w = World(hip, torch, [200, 64, 10, 128], [3, 2, 4, 20], 2, 64, seed=15)
    w.fill()
    w.table[0, :2] = -1
    w.table[1] = [-1, 2 ** 31 - 1, -2 ** 31, w.pool.data.shape[1]]
    w.table[2] = -7
    w.upload()
    for pos in (None, w.positions(4, 210, 20)):
        for left in (None, 5):
            got = w.check(4, pos, left)
            assert (got[3:9] == 0).all()


def test_single_dimension_precision(hip, torch):
    """A query with one dimension set scores with one term, so little is rounded:
    a score's product by its key's level is exact (8 + 8 + 8 bits), then a
    rounding each for the key's scale, the scale to powers of two and the
    exponential's argument, relative to the score; the output's few terms are
    positive. Third pieces that went missing would be 2^-16."""
    say("precision")
    dk = 64
    w = World(hip, torch, [9], [1], 1, dk, seed=16)
    w.fill(scale=1.0)
    for i in range(200):
        q = np.zeros((1, dk), np.float32)
        q[0, i % dk] = np.float32(w.g.uniform(-8, 8))
        got = w.attend(q, 1)[0]
        k, v = (a[:10] for a in w.pool.read(0, w.table[0, 0], 0))
        s = k @ q[0].astype(np.float64) / np.sqrt(dk)
        e = np.exp(s - s.max())
        want = e @ v / e.sum()
        tol = (8 + 8 * (np.abs(s).max() + 1) + 3 * 10 + 8) * 2.0 ** -24 * (e @ np.abs(v)) / e.sum()
        assert (np.abs(got - want) <= tol).all(), (np.abs(got - want) / tol).max()


@pytest.mark.parametrize("kscale,qscale", [(1e-18, 1e18), (1e18, 1e-18), (1e-30, 1e30), (3.0, 8.0)])
def test_magnitudes(hip, torch, kscale, qscale):
    """Keys and queries far from one, and peaked softmaxes."""
    say("magnitudes", kscale, qscale)
    w = World(hip, torch, [100, 7], [5, 2], 1, 128, seed=17)
    w.fill(scale=kscale)
    w.check(1, None, qscale=qscale)


@pytest.mark.parametrize("T", [1, 7])
def test_tiny_queries(hip, torch, T):
    """Queries of 1e-36 against keys of 1e35: a query is taken in pieces of 8
    bits, and pieces under 2^-126 may count as zeros, two of them at most a
    dimension. So a score (in powers of 2, as the pieces are) is off by at most
    2 x 2^-126 x sum |k|, and the softmax by the exponential of twice that."""
    say("tiny", T)
    w = World(hip, torch, [40, 7], [T, T], 1, 64, seed=44)
    w.fill(scale=1e35)
    q = (1e-36 * w.g.standard_normal((2 * T, 64))).astype(np.float32)
    got = w.attend(q, 1)
    want, bound = cr.attend(w.pool, 0, w.table, w.lens, w.row0, 2 * T, q, 1)
    most_k = max(np.abs(w.pool.read(0, pg, 0)[0][:n]).sum(1).max() for pg, n in ((w.table[0, 0], 40 + T), (w.table[1, 0], 7 + T)))
    most_v = max(np.abs(w.pool.read(0, pg, 0)[1][:n]).max() for pg, n in ((w.table[0, 0], 40 + T), (w.table[1, 0], 7 + T)))
    extra = (np.exp(2 * np.log(2) * 2 * 2.0 ** -126 * most_k) - 1) * 2 * most_v
    assert np.isfinite(got).all() and (np.abs(got - want) <= bound + extra).all()


def test_bad_values_stay_in_their_row(hip, torch):
    """A query that holds a NaN makes its own head's row NaN and no other."""
    say("nan rows")
    w = World(hip, torch, [70, 5], [20, 4], 2, 64, seed=18)
    w.fill()
    q = w.g.standard_normal((24, 4 * 64)).astype(np.float32)
    for pos in (None, w.positions(4, 100, 30)):
        clean = w.attend(q, 4, pos)
        bad = q.copy()
        bad[5, 70], bad[22, 0] = np.nan, np.inf
        got = w.attend(bad, 4, pos)
        assert np.isnan(got[5, 64:128]).all() and np.isnan(got[22, :64]).all()
        clean[5, 64:128] = clean[22, :64] = got[5, 64:128] = got[22, :64] = 0
        assert np.array_equal(clean, got)


def test_strided_and_in_place(hip, torch):
    """Queries inside wider rows, outputs into wider rows, and over the queries."""
    say("strides")
    w = World(hip, torch, [100, 30], [9, 40], 2, 64, seed=19)
    w.fill()
    H, n = 4, 49
    q = w.g.standard_normal((n, H * 64)).astype(np.float32)
    pos = w.positions(H, 140, 40)
    dpos = (w.dev(pos[0]), pos[1], w.dev(pos[2]), w.dev(pos[3]))
    want = w.attend(q, H, pos)
    ws = torch.empty(w.cache.attention_workspace(w.streams, H, dpos), dtype=torch.uint8, device="cuda")
    wide = torch.full((n, H * 64 + 20), 7.25, device="cuda")
    wide[:, 8:8 + H * 64] = w.dev(q)
    out = torch.full((n, H * 64 + 4), 7.25, device="cuda")
    w.cache.attention(out[:, :H * 64], 0, wide[:, 8:8 + H * 64], w.streams, H, ws, dpos)
    assert np.array_equal(out[:, :H * 64].cpu().numpy(), want) and (out[:, H * 64:] == 7.25).all()
    w.cache.attention(wide[:, 8:8 + H * 64], 0, wide[:, 8:8 + H * 64], w.streams, H, ws, dpos)
    assert np.array_equal(wide[:, 8:8 + H * 64].cpu().numpy(), want)
    assert (wide[:, :8] == 7.25).all() and (wide[:, 8 + H * 64:] == 7.25).all()


def test_descriptors_out_of_range(hip, torch):
    """Lengths and rows that no stream can have are cut to the call's and the
    table's bounds: the kernels' other rows are right and nothing else moves."""
    say("descriptors")
    w = World(hip, torch, [30, 20, 10], [4, 5, 6], 1, 32, seed=20, tail=4)
    w.fill(upto=[34, 26, 16])               # one frame more of stream 1, which its longer rows then attend
    q = w.g.standard_normal((w.rows, 32)).astype(np.float32)
    good = w.attend(q, 1)
    w.streams.len[0] = -9                   # as 0
    w.streams.row0[2] = 2 ** 31 - 1         # stream 1's rows to the end (max_T of them), stream 2 without any
    got = w.attend(q, 1)
    lens, row0 = [0, 20, 10], np.array([0, 4, 10, 10])
    want, bound = cr.attend(w.pool, 0, w.table, lens, row0, w.rows, q, 1)
    assert (np.abs(got[:10] - want[:10]) <= bound[:10]).all()
    assert (got[10:] == 7.25).all()
    assert not np.array_equal(good[:4], got[:4])


def test_ids_and_offsets_past_32_bits(hip, torch):
    """A pool of more than 4 GiB: its last pages."""
    say("large pool")
    G, dk, pages = 8, 128, 66000
    n = hip.cache_bytes(1, pages, G, dk)
    assert n > 1 << 32
    data = torch.zeros(n, dtype=torch.uint8, device="cuda")
    cache = hip.DeviceCache(data, 1, pages, G, dk)
    i32 = lambda *a: torch.tensor(a, dtype=torch.int32, device="cuda")
    st = hip.CacheStreams(i32([pages - 1, pages - 2]), i32(60), i32(0, 10), 10, 10)
    g = torch.Generator(device="cuda").manual_seed(1)
    k, v, q = (torch.randn(10, G * dk, device="cuda", generator=g) for _ in range(3))
    cache.append(0, k, v, st)
    small = hip.DeviceCache(torch.zeros(hip.cache_bytes(1, 2, G, dk), dtype=torch.uint8, device="cuda"), 1, 2, G, dk)
    st2 = hip.CacheStreams(i32([1, 0]), st.len, st.row0, 10, 10)
    small.append(0, k, v, st2)
    rec = G * cr.record_bytes(dk)
    assert torch.equal(data[-2 * rec:], small.data) and small.data.any()
    o, o2 = torch.empty_like(q), torch.empty_like(q)
    need = cache.attention_workspace(st, G, None)
    ws = torch.empty(max(16, need), dtype=torch.uint8, device="cuda")
    cache.attention(o, 0, q, st, G, ws)
    small.attention(o2, 0, q, st2, G, ws)
    assert torch.equal(o, o2) and torch.isfinite(o).all()
    cache.move([(pages - 1, 0)])
    assert torch.equal(data[:rec], data[-rec:])


# ------------------------------------------------------------------ move --

@pytest.mark.parametrize("dk,G,layers,n", [(32, 1, 1, 1), (128, 8, 3, 2), (96, 3, 2, 5), (64, 4, 1, 300)])
def test_move(hip, torch, dk, G, layers, n):
    say("move", dk, G, layers, n)
    pages = 2 * n + 3
    r = random.Random(n)
    g = torch.Generator(device="cuda").manual_seed(n)
    shape = (layers, pages, G, cr.record_bytes(dk))
    data = torch.randint(0, 256, shape, dtype=torch.uint8, device="cuda", generator=g)
    before = data.cpu().numpy()
    ids = r.sample(range(pages), 2 * n)
    pairs = list(zip(ids[:n], ids[n:]))
    cache = hip.DeviceCache(data, layers, pages, G, dk)
    table = torch.randint(-1, pages, (7, 11), dtype=torch.int32, device="cuda", generator=g)
    want = table.cpu().numpy()
    cache.move(pairs, table)
    to = dict(pairs)
    assert np.array_equal(table.cpu().numpy(), np.vectorize(lambda i: to.get(i, i))(want))
    after = before.copy()
    for f, t in pairs:
        after[:, t] = before[:, f]
    assert np.array_equal(data.cpu().numpy(), after)
    # to another cache, of another size; one page to several places
    other = torch.zeros(layers, pages + 5, G, cr.record_bytes(dk), dtype=torch.uint8, device="cuda")
    hip.DeviceCache(other, layers, pages + 5, G, dk).move([(0, pages + 4), (0, 1), (2, 0)], source=cache)
    got = other.cpu().numpy()
    assert np.array_equal(got[:, pages + 4], after[:, 0]) and np.array_equal(got[:, 1], after[:, 0])
    assert np.array_equal(got[:, 0], after[:, 2]) and not got[:, 2:pages + 4].any()
    cache.move([])


# ------------------------------------------------------ a stream's life --

def _segment_attention(hip, torch, q, k, v, p, u, w, T, D, H):
    """The library's whole-segment attention over the same float inputs."""
    o = torch.empty(T, D, device="cuda")
    ws = torch.empty(hip.attention_workspace(T, H), dtype=torch.uint8, device="cuda")
    hip.attention_dev(o, q, k, v, p, u, w, T, D, H, ws)
    return o


def test_whole_segment_is_the_encoders_attention(hip, torch):
    """A segment written at once and attended whole, its kept values given to the
    encoder's own attention: the same function. Both are within their 32-bit
    bounds of the same value; the bound is the cache's, twice."""
    say("segment")
    T, H, dk = 137, 2, 64
    D = H * dk
    w = World(hip, torch, [0], [T], H, dk, seed=21)
    k, v, q = (w.dev(w.g.standard_normal((T, D)).astype(np.float32)) for _ in range(3))
    p, c, u, b = w.positions(H, T - 1, T - 1)
    w.cache.append(0, k, v, w.streams)
    ko, vo = torch.empty_like(k), torch.empty_like(v)
    w.cache.read(0, ko, vo, w.streams)
    dp, du, db = w.dev(p), w.dev(u), w.dev(b)
    want = _segment_attention(hip, torch, q, ko, vo, dp, du, db, T, D, H).cpu().numpy()
    got = w.attend(q.cpu().numpy(), H, (p, c, u, b))
    w.pool.data = w.data.cpu().numpy()
    _, bound = cr.attend(w.pool, 0, w.table, w.lens, w.row0, T, q.cpu().numpy(), H, (p, c, u, b))
    assert (np.abs(got - want) <= 2 * bound).all()


def test_stream_in_chunks_is_the_segment(hip, torch):
    """Audio heard a chunk at a time, two streams side by side, one forked on the
    way and the pool compacted under them: each step's causal outputs are the
    rows of one causal pass over all the frames."""
    say("life")
    H, dk, n = 2, 64, 150
    D = H * dk
    g = torch.Generator(device="cuda").manual_seed(22)
    x = torch.randn(3, 2, n, D, device="cuda", generator=g)      # q, k, v of two streams
    p = torch.randn(n, D, device="cuda", generator=g)
    u, b = 0.1 * torch.randn(2, D, device="cuda", generator=g)
    pos = (p, n - 1, u, b)
    pages = 16
    cache = hip.DeviceCache(torch.zeros(hip.cache_bytes(1, pages, H, dk), dtype=torch.uint8, device="cuda"), 1, pages, H, dk)
    pool = hip.PagePool(pages)
    pool.alloc(2)                                                # someone else's, freed later
    table = torch.full((3, 3), -1, dtype=torch.int32, device="cuda")
    length = torch.zeros(3, dtype=torch.int32, device="cuda")
    ids, have = [[], [], []], [0, 0, 0]

    def hold(s, frames):
        while 64 * len(ids[s]) < frames:
            ids[s] += pool.alloc(1)
            table[s, len(ids[s]) - 1] = ids[s][-1]

    def step(who, T):
        """T more frames of the streams `who` ((stream, whose audio) pairs)"""
        rows = [0, 0, 0, 0]
        for s in range(3):
            rows[s + 1] = rows[s] + (T if s in dict(who) else 0)
            if s in dict(who):
                hold(s, have[s] + T)
        qkv = [torch.cat([x[i, a, have[s]:have[s] + T] for s, a in who]).contiguous() for i in range(3)]
        st = hip.CacheStreams(table, length, torch.tensor(rows, dtype=torch.int32, device="cuda"), rows[3], T)
        cache.append(0, qkv[1], qkv[2], st)
        o = torch.empty_like(qkv[0])
        ws = torch.empty(cache.attention_workspace(st, H, pos, None, 0), dtype=torch.uint8, device="cuda")
        cache.attention(o, 0, qkv[0], st, H, ws, pos, None, 0)
        for i, (s, a) in enumerate(who):
            outs[s].append(o[i * T:(i + 1) * T])
            have[s] += T
            length[s] += T

    outs = [[], [], []]
    for T in (1, 13, 1, 40, 15):                                 # 70 frames of both
        step([(0, 0), (1, 1)], T)
    ids[2] = pool.fork(cache, ids[0], have[0])
    assert ids[2][0] == ids[0][0] and ids[2][1] != ids[0][1] and pool.holders(ids[0][0]) == 2
    table[2, :2] = torch.tensor(ids[2], dtype=torch.int32)
    have[2], length[2] = have[0], have[0]
    outs[2] = list(outs[0])
    for T in (20, 1, 9):                                         # 100 of all three; the fork hears stream 1's audio
        step([(0, 0), (1, 1), (2, 1)], T)
    pool.release([0, 1])
    moved = pool.compact(cache, table)
    assert moved and pool.free_pages == pages - 5
    ids = [[i for i in row if i >= 0] for row in table.cpu().tolist()]
    assert max(map(max, ids)) == 4
    for T in (28, 22):
        step([(0, 0), (1, 1), (2, 1)], T)
    k2, v2 = (torch.cat([x[i, 0, :70], x[i, 1, 70:]]) for i in (1, 2))
    q2 = torch.cat([x[0, 0, :70], x[0, 1, 70:]])
    st = hip.CacheStreams(torch.tensor([[0, 1, 2]], dtype=torch.int32, device="cuda"),
                          torch.zeros(1, dtype=torch.int32, device="cuda"),
                          torch.tensor([0, n], dtype=torch.int32, device="cuda"), n, n)
    other = hip.DeviceCache(torch.zeros(hip.cache_bytes(1, 3, H, dk), dtype=torch.uint8, device="cuda"), 1, 3, H, dk)
    ws = torch.empty(other.attention_workspace(st, H, pos, None, 0), dtype=torch.uint8, device="cuda")
    for s, (q, k, v) in enumerate(((x[0, 0], x[1, 0], x[2, 0]), (x[0, 1], x[1, 1], x[2, 1]), (q2, k2, v2))):
        other.append(0, k.contiguous(), v.contiguous(), st)
        o = torch.empty(n, D, device="cuda")
        other.attention(o, 0, q.contiguous(), st, H, ws, pos, None, 0)
        host = cr.Pool(1, 3, H, dk)
        host.data = other.data.cpu().numpy().reshape(host.data.shape)
        _, bound = cr.attend(host, 0, np.array([[0, 1, 2]]), [0], [0, n], n, q.cpu().numpy(), H,
                             (p.cpu().numpy(), n - 1, u.cpu().numpy(), b.cpu().numpy()), None, 0)
        off = np.abs((torch.cat(outs[s]) - o).cpu().numpy())
        assert (off <= 2 * bound).all(), (s, (off / bound).max())


def test_graph_follows_the_streams(hip, torch):
    """A step captured once and replayed as the streams grow (their lengths and
    tables updated in place, the program's own work between replays) gives what
    eager steps give."""
    say("graph")
    H, dk, T, steps = 2, 64, 3, 6
    D = H * dk
    g = torch.Generator(device="cuda").manual_seed(23)
    x = torch.randn(steps, 3, 2 * T, D, device="cuda", generator=g)
    p = torch.randn(200, D, device="cuda", generator=g)
    pos = (p, 190, torch.zeros(D, device="cuda"), torch.zeros(D, device="cuda"))
    row0 = torch.tensor([0, T, 2 * T], dtype=torch.int32, device="cuda")

    def world():
        cache = hip.DeviceCache(torch.zeros(hip.cache_bytes(1, 6, H, dk), dtype=torch.uint8, device="cuda"), 1, 6, H, dk)
        table = torch.tensor([[0, 2, 4], [1, 3, 5]], dtype=torch.int32, device="cuda")
        length = torch.tensor([60, 125], dtype=torch.int32, device="cuda")
        st = hip.CacheStreams(table, length, row0, 2 * T, T)
        ws = torch.empty(cache.attention_workspace(st, H, pos), dtype=torch.uint8, device="cuda")
        return cache, st, ws, torch.empty(2 * T, D, device="cuda")

    def step(c, st, ws, o, a):
        c.append(0, a[1], a[2], st)
        c.attention(o, 0, a[0], st, H, ws, pos)

    eager = world()
    want = []
    for i in range(steps):
        step(*eager, x[i])
        eager[1].len.add_(T)
        want.append(eager[3].clone())
    c = world()
    a = x[0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(*c, a)
    c[0].data.zero_()
    for i in range(steps):
        a.copy_(x[i])
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(c[3], want[i]), i
        c[1].len.add_(T)
        (torch.randn(512, 512, device="cuda") @ torch.randn(512, 512, device="cuda")).sum().item()
    assert torch.equal(c[0].data, eager[0].data)


def test_two_streams_of_work(hip, torch):
    """Calls on two streams at once, a workspace each."""
    say("two streams")
    w = World(hip, torch, [300, 200], [4, 30], 2, 64, seed=24)
    w.fill()
    H = 4
    q = [w.dev(w.g.standard_normal((34, H * 64)).astype(np.float32)) for _ in range(2)]
    want = [w.attend(a.cpu().numpy(), H) for a in q]
    need = max(16, w.cache.attention_workspace(w.streams, H, None))
    ws = [torch.empty(need, dtype=torch.uint8, device="cuda") for _ in range(2)]
    ss = [torch.cuda.Stream() for _ in range(2)]
    o = [torch.empty_like(a) for a in q]
    torch.cuda.synchronize()
    for _ in range(20):
        for i, s in enumerate(ss):
            with torch.cuda.stream(s):
                w.cache.attention(o[i], 0, q[i], w.streams, H, ws[i])
    torch.cuda.synchronize()
    for i in range(2):
        assert np.array_equal(o[i].cpu().numpy(), want[i])


def test_same_call_same_bits(hip, torch):
    say("repeat")
    w = World(hip, torch, [700, 20, 64], [2, 50, 1], 2, 128, seed=25)
    w.fill()
    q = w.g.standard_normal((53, 256)).astype(np.float32)
    pos = w.positions(2, 720, 60)
    first = w.attend(q, 2, pos)
    for _ in range(5):
        assert np.array_equal(w.attend(q, 2, pos), first)


def test_pool_refuses_another_cache(hip, torch):
    cache = hip.DeviceCache(torch.zeros(hip.cache_bytes(1, 4, 1, 32), dtype=torch.uint8, device="cuda"), 1, 4, 1, 32)
    table = torch.zeros(1, 4, dtype=torch.int32, device="cuda")
    pool = hip.PagePool(5)
    ids = pool.alloc(2)
    for call in (lambda: pool.fork(cache, ids, 70), lambda: pool.compact(cache, table)):
        with pytest.raises(hip.PkHipError):
            call()
    assert pool.free_pages == 3 and [pool.holders(i) for i in range(5)] == [1, 1, 0, 0, 0]
    pool = hip.PagePool(4)
    ids = pool.alloc(3)
    assert pool.fork(cache, ids, 128) == ids[:2] and pool.free_pages == 1       # a page ahead of the frames is not shared
    assert pool.fork(cache, ids, 0) == []
    with pytest.raises(hip.PkHipError):
        pool.fork(cache, pool.alloc(1), 10)                                     # no page left for the copy
    assert [pool.holders(i) for i in range(4)] == [2, 2, 1, 1]


def test_wrapper_refusals(hip, torch):
    """Tensors that a kernel would misread are refused before anything runs."""
    w = World(hip, torch, [3], [4], 2, 64, seed=27)
    f = lambda *a, **k: torch.zeros(*a, device="cuda", **k)
    good, ws = f(4, 128), f(1 << 16, dtype=torch.uint8)
    for bad in (f(4, 128, dtype=torch.float16), f(4, 127), f(3, 128), f(128, 4).T, torch.zeros(4, 128), f(4, 258)[:, ::2]):
        for call in (lambda: w.cache.append(0, bad, good, w.streams), lambda: w.cache.append(0, good, bad, w.streams),
                     lambda: w.cache.read(0, good, bad, w.streams),
                     lambda: w.cache.attention(good, 0, bad, w.streams, 2, ws),
                     lambda: w.cache.attention(bad, 0, good, w.streams, 2, ws)):
            with pytest.raises(hip.PkHipError):
                call()
    b = f(128)
    for p in ((f(9, 128), 9, b, b), (f(9, 127), 4, b, b), (f(9, 256)[:, :128], 4, b, b), (f(9, 128), 4, f(64), b),
              (f(9, 128), 4, b, b.double())):
        with pytest.raises(hip.PkHipError):
            w.cache.attention(good, 0, good.clone(), w.streams, 2, ws, p)
    with pytest.raises(hip.PkHipError):
        w.cache.attention(good, 0, good.clone(), w.streams, 2, ws[:16], (f(9, 128), 4, b, b))
    with pytest.raises(hip.PkHipError):
        w.cache.move([(0, 1, 2)])
    with pytest.raises(hip.PkHipError):
        hip.DeviceCache(w.data[..., :-1], *w.pool.data.shape[:3], 64)
    with pytest.raises(hip.PkHipError):
        hip.CacheStreams(w.streams.table.long(), w.streams.len, w.streams.row0, 4, 4)
    with pytest.raises(hip.PkHipError):
        hip.CacheStreams(w.streams.table, w.streams.len, w.streams.row0[:1], 4, 4)


def test_nothing_to_do(hip, torch):
    say("empty")
    w = World(hip, torch, [10, 20], [0, 0], 2, 64, seed=26, tail=2)
    w.fill()
    q = w.g.standard_normal((2, 128)).astype(np.float32)
    assert (w.attend(q, 2) == 7.25).all()
    z = torch.zeros(0, dtype=torch.int32, device="cuda")
    st = hip.CacheStreams(z.reshape(0, 1), z, torch.zeros(1, dtype=torch.int32, device="cuda"), 0, 0)
    e = torch.empty(0, 128, device="cuda")
    assert w.cache.attention_workspace(st, 2, None) == 0


# ------------------------------------------------- rows past the table --

@pytest.mark.parametrize("lens,T,max_pages", [
    ([60, 64, 10, 0], 1, 1), ([60, 64, 63], 4, 1), ([60, 64, 0], 10, 1),
    ([128, 120, 64], 40, 2), ([0, 100], 300, 2), ([1, 64], 90, 1),
])
@pytest.mark.parametrize("with_positions", [False, True])
def test_rows_past_the_table(hip, torch, lens, T, max_pages, with_positions):
    """A stream that outgrows its table: its last rows' frames have no page, and
    the rows attend what the table holds, the first frame included."""
    say("past the table", lens, T, max_pages, with_positions)
    w = World(hip, torch, lens, [T] * len(lens), 2, 64, seed=50 + T, first=1, tail=1, max_pages=max_pages)
    w.fill()
    cap = 64 * max_pages
    for left, right in ((None, None), (None, 0), (cap - 1, None), (cap, None), (cap + 2, 0), (5, 3)):
        w.check(4 if T < 10 else 2, w.positions(4 if T < 10 else 2, max(lens) + T, T) if with_positions else None, left,
                right)
    if with_positions:                          # what the table of positions reaches, on both sides of the cap
        for back in (cap - 1, cap, cap + 1):
            w.check(2, w.positions(2, back, 2))


@pytest.mark.parametrize("seed", range(12))
def test_any_call_past_the_table(hip, torch, seed):
    """Drawn calls whose tables are narrower than some of their streams."""
    r = random.Random(1000 + seed)
    dk, (H, G) = r.choice(DKS), r.choice([(1, 1), (2, 2), (4, 1), (6, 3)])
    max_pages, B = r.choice([1, 1, 2, 3]), r.choice([1, 3, 18])
    Ts = [r.choice([1, 2, 3, r.randint(1, 70)]) for _ in range(B)]
    lens = [max(0, 64 * max_pages - r.choice([0, 1, 5, r.randint(0, 64 * max_pages)])) for _ in range(B)]
    say("any past", seed, dk, H, G, lens, Ts, max_pages)
    w = World(hip, torch, lens, Ts, G, dk, seed=seed, first=r.randint(0, 2), tail=r.randint(0, 2), max_pages=max_pages)
    w.fill()
    left, right = (r.choice([None, None, 0, 64 * max_pages, r.randint(0, 400)]) for _ in range(2))
    pos = w.positions(H, r.choice([64 * max_pages, 300, 40]), r.choice([70, 2])) if r.random() < 0.6 else None
    w.check(H, pos, left, right)


# ----------------------------------------- position scores' precision --

SHAPES = [                                      # lens, Ts, dk, the window: each way that position scores are made
    ([90], [1], 64, 70),                        # where they are used
    ([60 + b for b in range(17)], [1] * 17, 64, 70),
    ([100, 7], [3, 20], 128, None),             # 16 rows a workgroup
    ([1300, 900], [150, 20], 32, None),         # many distances, more rows a workgroup
    ([40, 0], [300, 240], 96, None),
    ([60], [1200], 32, None),                   # the table cut beforehand
]


@pytest.mark.parametrize("lens,Ts,dk,left", SHAPES, ids=str)
@pytest.mark.parametrize("wide", ["queries", "positions", "both"])
@pytest.mark.parametrize("ratio", [1e4, 1e6, 1e12])
def test_position_scores_of_wide_rows(hip, torch, lens, Ts, dk, left, wide, ratio):
    """Rows of queries and of the table that are far larger in one dimension than
    in the others, where the other factor (and the keys) have a zero: the score is
    the small dimensions', and is held as a 32-bit sum holds it."""
    say("wide rows", lens, Ts, dk, left, wide, ratio)
    w = World(hip, torch, lens, Ts, 1, dk, seed=60)
    big = 5
    std = w.g.standard_normal
    for b in range(len(lens)):
        for f in range(lens[b] + Ts[b]):
            k, v = std((2, dk)).astype(np.float32)
            k[big] = k[big + 1] = 0
            w.pool.write(0, w.table[b, f // 64], f % 64, 1e-3 * k, v)
    w.upload()
    far = max(a + t for a, t in zip(lens, Ts))
    p, c, u, b = w.positions(1, far, max(Ts))
    q = std((w.rows, dk)).astype(np.float32)
    u, b = 0 * u, (0.1 * b).astype(np.float32)
    q[:, big:big + 2], b[big:big + 2], p[:, big:big + 2] = 0, 0, 0
    if wide != "positions":                     # queries: the rest by ratio smaller, the table by as much larger
        q[:, big] = ratio * (1 + np.abs(std(w.rows)))
    if wide != "queries":
        p[:, big + 1] = ratio * (1 + np.abs(std(len(p))))
    if wide == "queries":
        q /= np.float32(ratio)
        b = (b / np.float32(ratio)).astype(np.float32)
        p = (p * np.float32(ratio)).astype(np.float32)
    elif wide == "positions":
        p /= np.float32(ratio)
        q, b = (q * np.float32(ratio)).astype(np.float32), (b * np.float32(ratio)).astype(np.float32)
        # content: keys in proportion, or the products of the larger queries would be all there is
        w.pool.data[..., 64 * dk:64 * dk + 128] = 0
        w.upload()
    w.check(1, (p, c, u, b), left, q=q)


@pytest.mark.parametrize("lens,Ts,dk,left", SHAPES, ids=str)
def test_position_scores_of_one_dimension(hip, torch, lens, Ts, dk, left):
    """Queries with one dimension set, no content scores: a position score is one
    product. Relative to it the scale to powers of two is off by three roundings
    (its factors' and its own), the scaled query by one, the product by one (two
    where pieces make it: what is left out of them, and their sum, which may cut
    where it should round), the exponential's argument by two: 10 of 2^-24 of the
    largest score at most, twice for the maximum's. Each row's largest scores are
    of one, so that what the exponentials and the output's sums add (a page's
    rescaling, n terms) is the rest."""
    say("one dimension", lens, Ts, dk, left)
    w = World(hip, torch, lens, Ts, 1, dk, seed=61)
    std = w.g.standard_normal
    for b in range(len(lens)):
        for f in range(lens[b] + Ts[b]):
            w.pool.write(0, w.table[b, f // 64], f % 64, np.zeros(dk, np.float32), std(dk).astype(np.float32))
    w.upload()
    far = max(a + t for a, t in zip(lens, Ts))
    p, c, u, b = w.positions(1, far, max(Ts))
    q = np.zeros((w.rows, dk), np.float32)
    at = np.arange(w.rows) % dk
    q[np.arange(w.rows), at] = 2 * std(w.rows) * np.sqrt(dk)
    got = w.attend(q, 1, (p, c, 0 * u, 0 * b), left)
    for s in range(len(lens)):
        total = lens[s] + Ts[s]
        v = np.concatenate([w.pool.read(0, w.table[s, i], 0)[1] for i in range(-(-total // 64))])[:total]
        for t in range(Ts[s]):
            row, pos = w.row0[s] + t, lens[s] + t
            j = np.arange(max(0, pos - left) if left is not None else 0, total)
            x = p[c - pos + j, at[row]].astype(np.float64) * float(q[row, at[row]]) / np.sqrt(dk)
            e = np.exp(x - x.max())
            want = e @ v[j] / e.sum()
            tol = (2 * 10 * (np.abs(x).max() + 1) + 2 * (3 * len(j) + 4 * (len(j) // 64 + 8))) * 2.0 ** -24
            assert (np.abs(got[row] - want) <= tol * 2 * (e @ np.abs(v[j])) / e.sum()).all(), (s, t)


@pytest.mark.parametrize("dk,H,G", [(32, 1, 1), (64, 2, 1), (96, 2, 2), (128, 1, 1)])
@pytest.mark.parametrize("left", [None, 1000])
def test_table_cut_beforehand(hip, torch, dk, H, G, left):
    """Rows and distances enough for the table's pieces to be made once, the last
    block of rows and the last run of distances in part."""
    say("cut beforehand", dk, H, G, left)
    w = World(hip, torch, [60, 3], [1201, 24], G, dk, seed=62, first=2, tail=1)
    w.fill()
    w.check(H, w.positions(H, 1270, 1201), left)


def test_step_without_streams(hip, torch):
    """A step that no stream takes part in: every call returns and nothing moves."""
    say("no streams")
    w = World(hip, torch, [10, 20], [1, 2], 2, 64, seed=63)
    w.fill()
    before = w.data.clone()
    z = torch.zeros(0, dtype=torch.int32, device="cuda")
    for rows in (0, 3):
        st = hip.CacheStreams(z.reshape(0, 1), z, torch.zeros(1, dtype=torch.int32, device="cuda"), rows, 0)
        a, o = torch.ones(rows, 128, device="cuda"), torch.full((rows, 256), 7.25, device="cuda")
        q, p, b = torch.ones(rows, 256, device="cuda"), torch.ones(9, 256, device="cuda"), torch.ones(256, device="cuda")
        w.cache.append(0, a, a, st)
        w.cache.read(0, a, a.clone(), st)
        assert w.cache.attention_workspace(st, 4, None) == 0
        w.cache.attention(o, 0, q, st, 4, None)
        ws = torch.empty(max(1, w.cache.attention_workspace(st, 4, (p, 4, b, b))), dtype=torch.uint8, device="cuda")
        w.cache.attention(o, 0, q, st, 4, ws, (p, 4, b, b))
        torch.cuda.synchronize()
        assert (a == 1).all() and (o == 7.25).all() and torch.equal(w.data, before)


@pytest.mark.parametrize("B,H,G,T,dk,pages", [
    (17, 8, 8, 2, 32, 120), (21, 8, 8, 4, 32, 119),     # tiles of four rows, in three splits from 120 pages
    (17, 8, 8, 16, 32, 100), (17, 8, 8, 5, 32, 99),     # of 16 rows, from 100
])
def test_pages_dealt_in_odd_splits(hip, torch, B, H, G, T, dk, pages):
    """On both sides of the pages from which three workgroups share a tile's. All
    streams read one stream's pages, each with a hole of its own."""
    say("odd splits", B, H, G, T, dk, pages)
    total = 64 * pages - 5
    w = World(hip, torch, [total - T] * B, [T] * B, G, dk, seed=pages)
    w.table[:] = w.table[0]
    w.fill(upto=[total] + [0] * (B - 1))
    for b in range(B):
        w.table[b, (7 * b + 3) % pages] = -1
    w.upload()
    w.check(H)


def test_graph_with_the_table_cut_beforehand(hip, torch):
    """A call of many rows captured, replayed with other queries, positions and
    lengths in the same memory and the program's own work between: each replay is
    the eager call's bits, on a stream of its own too."""
    say("graph, cut beforehand")
    w = World(hip, torch, [60, 3], [1201, 24], 1, 32, seed=64)
    w.fill()
    p, c, u, b = w.positions(1, 1270, 1201)
    pos = (w.dev(p), c, w.dev(u), w.dev(b))
    q = w.dev(w.g.standard_normal((w.rows, 32)).astype(np.float32))
    o = torch.empty_like(q)
    need = w.cache.attention_workspace(w.streams, 1, pos)
    ws = [torch.full((need,), 0xff, dtype=torch.uint8, device="cuda") for _ in range(2)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        w.cache.attention(o, 0, q, w.streams, 1, ws[0], pos)
    side, eager = torch.cuda.Stream(), torch.empty_like(q)
    for i in range(4):
        q.copy_(w.dev(w.g.standard_normal((w.rows, 32)).astype(np.float32)))
        pos[0].mul_(0.9)
        w.streams.len[0] = 60 - 7 * i
        torch.cuda.synchronize()
        graph.replay()
        with torch.cuda.stream(side):
            w.cache.attention(eager, 0, q, w.streams, 1, ws[1], pos)
        torch.cuda.synchronize()
        assert torch.equal(o, eager) and torch.isfinite(o).all(), i
        (torch.randn(512, 512, device="cuda") @ torch.randn(512, 512, device="cuda")).sum().item()
