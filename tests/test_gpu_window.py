"""Attention with a window and sinks over whole segments on the GPU, against 64
bits within the bound that 32-bit arithmetic gives (window_ref.attend)."""
import random
import sys

import numpy as np
import pytest

import window_ref as wr

pytestmark = pytest.mark.gpu
DKS = (32, 64, 96, 128)
MARK = 7.25


def say(*a):
    print("[case]", *a, flush=True)
    sys.stdout.flush()


@pytest.fixture(scope="module")
def torch():
    import torch
    assert torch.cuda.is_available()
    return torch


class Call:
    """Segments of Ts rows (`first` rows before them, `tail` behind), H heads over G."""

    def __init__(self, pk, torch, Ts, H, G, dk, seed=0, first=0, tail=0, slack_T=0):
        self.pk, self.torch, self.H, self.G, self.dk, self.Ts = pk, torch, H, G, dk, list(Ts)
        self.g = np.random.default_rng(seed)
        self.row0 = np.cumsum([first] + self.Ts).astype(np.int32)
        self.rows = int(self.row0[-1]) + tail
        self.max_T = min(self.rows, max(self.Ts, default=0) + slack_T)
        n = lambda w: self.g.standard_normal((self.rows, w)).astype(np.float32)
        self.q, self.k, self.v = 1.5 * n(H * dk), n(G * dk), n(G * dk)

    def positions(self, back, ahead):
        w = self.H * self.dk
        p = self.g.standard_normal((back + ahead + 1, w)).astype(np.float32)
        u, b = (0.3 * self.g.standard_normal((2, w))).astype(np.float32)
        return p, back, u, b

    def dev(self, a):
        return self.torch.from_numpy(np.ascontiguousarray(a)).cuda()

    def attend(self, positions=None, left=None, right=None, sinks=0, q=None, k=None, v=None):
        torch = self.torch
        pos = None if positions is None else (self.dev(positions[0]), positions[1], self.dev(positions[2]),
                                              self.dev(positions[3]))
        o = torch.full((self.rows, self.H * self.dk), MARK, device="cuda")
        q, k, v = (self.dev(own if x is None else x) for x, own in ((q, self.q), (k, self.k), (v, self.v)))
        self.pk.attention_window_dev(o, q, k, v, self.pk.Segments(self.dev(self.row0), self.rows, self.max_T), self.H,
                                     self.dk, pos, left, right, sinks)
        torch.cuda.synchronize()
        return o.cpu().numpy()

    def want(self, positions=None, left=None, right=None, sinks=0):
        out, bound = np.full((self.rows, self.H * self.dk), MARK, np.float64), np.zeros((self.rows, self.H * self.dk))
        for b, T in enumerate(self.Ts):
            r = slice(self.row0[b], self.row0[b] + T)
            out[r], bound[r] = wr.attend(self.q[r], 0, np.arange(T), self.k[r], self.v[r], self.H, self.dk, positions,
                                         left, right, sinks)
        return out, bound

    def check(self, positions=None, left=None, right=None, sinks=0):
        got = self.attend(positions, left, right, sinks)
        want, bound = self.want(positions, left, right, sinks)
        assert np.isfinite(got).all()
        off = np.abs(got - want)
        assert (off <= bound).all(), (off.max(), np.argwhere(off > bound)[:5])
        assert np.linalg.norm(off) <= 1e-5 * np.linalg.norm(want)


@pytest.mark.parametrize("dk", DKS)
@pytest.mark.parametrize("H,G", [(1, 1), (4, 2), (3, 1)])
@pytest.mark.parametrize("with_positions", [False, True])
def test_window(hip, torch, dk, H, G, with_positions):
    """Ragged segments, with rows of none before and behind them left as they were."""
    say("window", dk, H, G, with_positions)
    c = Call(hip, torch, [1, 0, 40, 100, 17], H, G, dk, seed=dk + H, first=3, tail=2)
    c.check(c.positions(30, 20) if with_positions else None, 30, 20, 3)


@pytest.mark.parametrize("left,right", [(0, 0), (1, 0), (0, 1), (None, 0), (0, None), (None, None), (15, 16), (64, 5),
                                        (33, 40)])
@pytest.mark.parametrize("sinks", [0, 1, 31, 40, 1000])
@pytest.mark.parametrize("with_positions", [False, True])
def test_reaches(hip, torch, left, right, sinks, with_positions):
    say("reach", left, right, sinks, with_positions)
    c = Call(hip, torch, [130, 77], 2, 2, 32, seed=5)
    back, ahead = 129 if left is None else left, 129 if right is None else right
    c.check(c.positions(back, ahead) if with_positions else None, left, right, sinks)


@pytest.mark.parametrize("back,ahead", [(0, 0), (7, 0), (0, 9), (40, 3), (300, 200)])
def test_positions_bound_the_window(hip, torch, back, ahead):
    """Distances that the table has no row for are not attended, but for sinks."""
    say("bounded", back, ahead)
    c = Call(hip, torch, [90, 20], 2, 1, 64, seed=6)
    for left, right, sinks in ((None, None, 0), (50, 50, 5), (None, 0, 2)):
        c.check(c.positions(back, ahead), left, right, sinks)


@pytest.mark.parametrize("T", [1, 2, 15, 16, 17, 63, 64, 65, 255, 600])
def test_lengths(hip, torch, T):
    say("length", T)
    c = Call(hip, torch, [T], 1, 1, 128, seed=T)
    c.check(c.positions(70, 13), 70, 13, 4)


@pytest.mark.parametrize("B,T,H,G,dk,left,right", [(3, 700, 4, 4, 64, 128, 128), (40, 130, 8, 2, 32, 60, 0),
                                                    (1, 2100, 2, 2, 128, 200, 30), (2, 1100, 6, 3, 96, 33, 64)])
@pytest.mark.parametrize("with_positions", [False, True])
def test_many_tiles(hip, torch, B, T, H, G, dk, left, right, with_positions):
    """Calls of many tiles, ragged, checked on rows picked over all of them."""
    say("many", B, T, H, G, dk)
    r = random.Random(B * T)
    c = Call(hip, torch, [r.randint(T // 2, T) for _ in range(B)], H, G, dk, seed=B)
    pos = c.positions(left, right) if with_positions else None
    got = c.attend(pos, left, right, 20)
    assert np.isfinite(got).all()
    for _ in range(12):
        b = r.randrange(B)
        T0, i = c.Ts[b], r.randrange(c.Ts[b])
        n = min(20, T0 - i)
        s = slice(c.row0[b], c.row0[b] + T0)
        rows = slice(c.row0[b] + i, c.row0[b] + i + n)
        want, bound = wr.attend(c.q[rows], i, np.arange(T0), c.k[s], c.v[s], H, dk, pos, left, right, 20)
        assert (np.abs(got[rows] - want) <= bound).all(), (b, i)


@pytest.mark.parametrize("dk", DKS)
@pytest.mark.parametrize("with_positions", [False, True])
@pytest.mark.parametrize("left,right,sinks", [(100, 20, 40), (33, 0, 0), (3, 70, 1), (700, 0, 5)])
def test_many_rows(hip, torch, dk, with_positions, left, right, sinks):
    """Calls of many long tiles of each width: all rows of a head around the segments' ends and some picked ones."""
    say("rows", dk, with_positions, left, right)
    r = random.Random(dk + left)
    c = Call(hip, torch, [1500, 1, 1400, 1203, 70], 8, 2, dk, seed=dk, first=1, tail=4)
    pos = c.positions(left, right) if with_positions else None
    got = c.attend(pos, left, right, sinks)
    assert (got[:1] == MARK).all() and (got[c.row0[-1]:] == MARK).all() and np.isfinite(got).all()
    for b, T in enumerate(c.Ts):
        s = slice(c.row0[b], c.row0[b] + T)
        for i in {0, max(0, T - 6), r.randrange(T), r.randrange(T), min(T - 1, 60), min(T - 1, 126)}:
            n = min(6, T - i)
            rows = slice(c.row0[b] + i, c.row0[b] + i + n)
            want, bound = wr.attend(c.q[rows], i, np.arange(T), c.k[s], c.v[s], 8, dk, pos, left, right, sinks)
            assert (np.abs(got[rows] - want) <= bound).all(), (b, i)


@pytest.mark.parametrize("dk", DKS)
@pytest.mark.parametrize("with_positions", [False, True])
def test_many_short_segments(hip, torch, dk, with_positions):
    say("short", dk, with_positions)
    r = random.Random(dk)
    c = Call(hip, torch, [r.choice([0, 1, 16, 17, 33, r.randint(1, 45)]) for _ in range(300)], 4, 2, dk, seed=dk, tail=2)
    c.check(c.positions(20, 9) if with_positions else None, 20, 9, 3)


@pytest.mark.parametrize("seed", range(16))
def test_any_call(hip, torch, seed):
    r = random.Random(seed)
    G = r.choice([1, 2, 3])
    H, dk = G * r.choice([1, 1, 2, 5]), r.choice(DKS)
    Ts = [r.choice([0, 1, r.randint(1, 40), r.randint(1, 200)]) for _ in range(r.randint(1, 6))]
    say("any", seed, Ts, H, G, dk)
    c = Call(hip, torch, Ts, H, G, dk, seed, r.randint(0, 3), r.randint(0, 3), r.choice([0, 50]))
    if not sum(Ts):
        return
    pos = c.positions(r.randint(0, 150), r.randint(0, 150)) if r.random() < 0.6 else None
    c.check(pos, r.choice([None, r.randint(0, 200)]), r.choice([None, 0, r.randint(0, 60)]),
            r.choice([0, r.randint(1, 5), r.randint(1, 300)]))


@pytest.mark.parametrize("T,H", [(120, 2), (1400, 8), (2200, 16)])
@pytest.mark.parametrize("dk", DKS)
def test_what_is_not_attended_does_not_count(hip, torch, T, H, dk):
    """NaN and infinities in keys, values and position rows reach the rows that attend them and no others."""
    say("masked", T, H, dk)
    c = Call(hip, torch, [T, 50], H, H, dk, seed=9)
    left, right, sinks = 20, 3, 2
    for pos in (None, c.positions(left, right)):
        clean = c.attend(pos, left, right, sinks)
        k, v = c.k.copy(), c.v.copy()
        rows = np.arange(c.rows)
        hit = np.zeros(c.rows, bool)
        for j, x in ((5, np.nan), (60, np.inf), (61, -np.inf), (T - 1, np.nan), (T, np.inf)):
            v[j, ::7] = x
            b = int(j >= T)
            hit |= (rows >= c.row0[b]) & (rows < c.row0[b + 1]) & wr.attended(j - c.row0[b], rows - c.row0[b], right, left, 0)
            if j - c.row0[b] < sinks:
                hit |= (rows >= c.row0[b]) & (rows < c.row0[b + 1])
        got = c.attend(pos, left, right, sinks, v=v)
        assert np.array_equal(got[~hit], clean[~hit]) and not np.isfinite(got[hit][:, ::7]).any()
        other = np.arange(got.shape[1]) % 7 != 0
        assert np.array_equal(got[:, other], clean[:, other])
        assert (got[60 - right, ::7] == np.inf).all()
        k[60, :] = np.nan
        got = c.attend(pos, left, right, sinks, k=k)
        hit = (rows >= 60 - right) & (rows <= 60 + left)
        assert np.array_equal(got[~hit], clean[~hit]) and np.isnan(got[hit]).all()


@pytest.mark.parametrize("T,H", [(120, 2), (1400, 8), (2200, 16)])
@pytest.mark.parametrize("dk", DKS)
def test_the_greatest_floats(hip, torch, T, H, dk):
    """The type's greatest and lowest values as padding, in keys and values and position rows that rows do not attend: all
    but the rows that attend them keep their bits, and the outputs of theirs that no such value takes part in."""
    say("greatest", T, H, dk)
    c = Call(hip, torch, [T, 50], H, H, dk, seed=10)
    left, right, sinks = 20, 3, 2
    for pos in (None, c.positions(left, right)):
        clean = c.attend(pos, left, right, sinks)
        for x in (np.finfo(np.float32).min, np.finfo(np.float32).max, np.float32(2.0 ** 127 * (2 - 2.0 ** -8))):
            k, v = c.k.copy(), c.v.copy()
            v[60, ::7], k[90] = x, x
            rows = np.arange(c.rows)
            of_value = (rows >= 60 - right) & (rows <= 60 + left)
            of_key = (rows >= 90 - right) & (rows <= 90 + left)
            got = c.attend(pos, left, right, sinks, k=k, v=v)
            assert np.array_equal(got[~of_value & ~of_key], clean[~of_value & ~of_key])
            other = np.arange(got.shape[1]) % 7 != 0
            assert np.array_equal(got[of_value & ~of_key][:, other], clean[of_value & ~of_key][:, other])
            assert not np.isnan(got[of_value & ~of_key]).any()


@pytest.mark.parametrize("H", [8, 480])
def test_rows_past_32_bits(hip, torch, H):
    """Rows 2^25 floats apart, the furthest past 2^33 bytes: the bits of the same rows side by side."""
    say("far rows", H)
    G, dk, step = 2, 32, 1 << 25
    c = Call(hip, torch, [78], H, G, dk, seed=23, first=1, tail=1)
    mem = torch.empty(c.rows * step, device="cuda")
    place, views = 0, []
    for x, w in ((np.full((c.rows, H * dk), MARK, np.float32), H * dk), (c.q, H * dk), (c.k, G * dk), (c.v, G * dk)):
        views.append(torch.as_strided(mem, (c.rows, w), (step, 1), place))
        views[-1].copy_(torch.from_numpy(x))
        place += w
    segments = hip.Segments(c.dev(c.row0), c.rows, c.max_T)
    for pos in (None, c.positions(30, 9)):
        at = None if pos is None else (c.dev(pos[0]), pos[1], c.dev(pos[2]), c.dev(pos[3]))
        want = c.attend(pos, 30, 9, 3)
        views[0].fill_(MARK)
        hip.attention_window_dev(*views, segments, H, dk, at, 30, 9, 3)
        assert np.array_equal(views[0].cpu().numpy(), want)


@pytest.mark.parametrize("H,G", [(2048, 1024), (3001, 1)])
@pytest.mark.parametrize("with_positions", [False, True])
def test_many_heads(hip, torch, H, G, with_positions):
    say("heads", H, G, with_positions)
    c = Call(hip, torch, [3, 2], H, G, 32, seed=24)
    c.check(c.positions(2, 1) if with_positions else None, 2, 1, 1)


def test_bad_queries_stay_in_their_row(hip, torch):
    say("nan rows")
    for Ts, H in (([50, 30], 4), ([1200, 700], 4), ([1200, 1700], 12)):
        c = Call(hip, torch, Ts, H, 2, 64, seed=18)
        for pos in (None, c.positions(40, 30)):
            clean = c.attend(pos, 40, 30, 2)
            q = c.q.copy()
            q[5, 70], q[52, 0] = np.nan, np.inf
            got = c.attend(pos, 40, 30, 2, q=q)
            assert np.isnan(got[5, 64:128]).all() and np.isnan(got[52, :64]).all()
            clean[5, 64:128] = clean[52, :64] = got[5, 64:128] = got[52, :64] = 0
            assert np.array_equal(clean, got)


@pytest.mark.parametrize("T", [40, 1500])
def test_strided_and_in_place(hip, torch, T):
    """One tensor of queries, keys and values side by side; the output over the queries."""
    say("strides", T)
    c = Call(hip, torch, [T, T // 2], 4, 4, 64, seed=21)
    w = 4 * 64
    want = c.attend(None, 50, 20, 3)
    all3 = c.dev(np.concatenate([c.q, c.k, c.v, np.full((c.rows, 4), MARK, np.float32)], 1))
    q, k, v = all3[:, :w], all3[:, w:2 * w], all3[:, 2 * w:3 * w]
    hip.attention_window_dev(q, q, k, v, hip.Segments(c.dev(c.row0), c.rows, c.max_T), 4, 64, None, 50, 20, 3)
    torch.cuda.synchronize()
    got = all3.cpu().numpy()
    assert np.array_equal(got[:, :w], want) and np.array_equal(got[:, w:2 * w], c.k)
    assert np.array_equal(got[:, 2 * w:3 * w], c.v) and (got[:, 3 * w:] == MARK).all()


@pytest.mark.parametrize("back", [0, 2])
def test_offsets_out_of_range(hip, torch, back):
    """Row offsets that fall, pass the rows or are negative: what is in range of them is attended, nothing else touched."""
    say("offsets", back)
    c = Call(hip, torch, [30, 30, 30, 30], 1, 1, 32, seed=3, tail=3)
    row0 = np.array([-5, 30, 20, 60, 1 << 30], np.int32)
    q, k, v, o = (c.dev(x) for x in (c.q, c.k, c.v, np.full_like(c.q, MARK)))
    hip.attention_window_dev(o, q, k, v, hip.Segments(c.dev(row0), c.rows, 30 - back), 1, 32, None, 10, 0)
    torch.cuda.synchronize()
    got = o.cpu().numpy()
    n = 30 - back
    want = np.full(c.q.shape, MARK)
    for r0, r1 in ((0, 30), (20, 60), (60, c.rows)):
        s = slice(r0, min(r1, r0 + n))
        T = s.stop - s.start
        if r0 != 20:                        # rows 20 to 30 are two segments', so either's
            want[s], bound = wr.attend(c.q[s], 0, np.arange(T), c.k[s], c.v[s], 1, 32, None, 10, 0)
            at = slice(s.start, 20) if r0 == 0 else s
            assert (np.abs(got[at] - want[at]) <= bound[:at.stop - at.start]).all()
    assert (got[60 + n:] == MARK).all()


def test_same_bits_two_streams_and_a_graph(hip, torch):
    """The same call gives the same bits: again, on two streams at once, captured and replayed."""
    say("streams")
    for Ts in ([90, 33], [3000, 900]):
        c = Call(hip, torch, Ts, 4, 4, 64, seed=24)
        pos = c.positions(60, 10)
        want = c.attend(pos, 60, 10, 4)
        d = [c.dev(x) for x in (c.q, c.k, c.v)]
        p = (c.dev(pos[0]), pos[1], c.dev(pos[2]), c.dev(pos[3]))
        sg = hip.Segments(c.dev(c.row0), c.rows, c.max_T)
        o = [torch.zeros_like(d[0]) for _ in range(3)]
        ss = [torch.cuda.Stream() for _ in range(2)]
        torch.cuda.synchronize()
        for _ in range(10):
            for i, s in enumerate(ss):
                with torch.cuda.stream(s):
                    hip.attention_window_dev(o[i], *d, sg, 4, 64, p, 60, 10, 4)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            hip.attention_window_dev(o[2], *d, sg, 4, 64, p, 60, 10, 4)
        for _ in range(3):
            o[2].zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert np.array_equal(o[2].cpu().numpy(), want)
            (torch.randn(256, 256, device="cuda") @ torch.randn(256, 256, device="cuda")).sum().item()
        assert all(np.array_equal(x.cpu().numpy(), want) for x in o[:2])


def test_graph_follows_the_segments(hip, torch):
    """A captured call reads the offsets of the moment."""
    say("follows")
    c = Call(hip, torch, [40, 60], 2, 2, 32, seed=2)
    d, row0 = [c.dev(x) for x in (c.q, c.k, c.v)], c.dev(c.row0)
    o = torch.zeros_like(d[0])
    sg = hip.Segments(row0, c.rows, 100)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        hip.attention_window_dev(o, *d, sg, 2, 32, None, 9, 0, 1)
    for cut in (40, 1, 99, 64):
        row0.copy_(torch.tensor([0, cut, 100], dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        c.Ts, c.row0, c.max_T = [cut, 100 - cut], np.array([0, cut, 100], np.int32), 100
        want, bound = c.want(None, 9, 0, 1)
        assert (np.abs(o.cpu().numpy() - want) <= bound).all()


def test_magnitudes(hip, torch):
    """Queries and keys of very different sizes, dimensions small beside their row's largest."""
    say("magnitudes")
    for qs, ks in ((1e-18, 1e18), (1e18, 1e-18), (1e-30, 1e30)):
        c = Call(hip, torch, [70, 1300], 2, 2, 64, seed=11)
        c.q, c.k = (c.q * np.float32(qs)).astype(np.float32), (c.k * np.float32(ks)).astype(np.float32)
        c.Ts, c.row0, c.rows, c.max_T = [70], c.row0[:2], 70, 70
        c.q, c.k, c.v = c.q[:70], c.k[:70], c.v[:70]
        c.check(None, 30, 5, 2)
        c.q[:, 0] *= np.float32(1e6)
        c.k[:, 0] = 0
        c.check(None, 30, 5, 2)


def test_whole_segment_is_the_encoders_attention(hip, torch):
    """Without an end to the window, the outputs of pk_hip_attention_dev within 32 bits."""
    say("encoder")
    T, H, dk = 200, 4, 64
    c = Call(hip, torch, [T], H, H, dk, seed=31)
    pos = c.positions(T - 1, T - 1)
    d = [c.dev(x) for x in (c.q, c.k, c.v, *pos[:1], *pos[2:])]
    o = torch.empty_like(d[0])
    ws = torch.empty(hip.attention_workspace(T, H), dtype=torch.uint8, device="cuda")
    hip.attention_dev(o, *d, T, H * dk, H, ws)
    torch.cuda.synchronize()
    _, bound = c.want(pos)
    assert (np.abs(o.cpu().numpy() - c.attend(pos)) <= 2 * bound).all()


def test_nothing_to_do(hip, torch):
    say("nothing")
    e = torch.empty(0, 64, device="cuda")
    none = torch.zeros(1, dtype=torch.int32, device="cuda")
    hip.attention_window_dev(e, e, e, e, hip.Segments(none, 0, 0), 2, 32)
    x = torch.full((3, 64), MARK, device="cuda")
    hip.attention_window_dev(x, torch.zeros_like(x), torch.zeros_like(x), torch.zeros_like(x), hip.Segments(none, 3, 3), 2, 32)
    hip.attention_window_dev(x, torch.zeros_like(x), torch.zeros_like(x), torch.zeros_like(x),
                             hip.Segments(torch.zeros(4, dtype=torch.int32, device="cuda"), 3, 3), 2, 32)
    torch.cuda.synchronize()
    assert (x == MARK).all()
