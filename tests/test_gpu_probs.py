"""Log probabilities, entropy and alternatives on the GPU against 64 bits."""
import random
import sys

import numpy as np
import pytest

import probs_ref as pr

pytestmark = pytest.mark.gpu
MARK = 7.25


def say(*a):
    print("[case]", *a, flush=True)
    sys.stdout.flush()


@pytest.fixture(scope="module")
def torch():
    import torch
    assert torch.cuda.is_available()
    return torch


def ask(pk, torch, x, tokens, k, stride=None, offset=0):
    """(lp, entropy, top, top_lp) from rows that lie `stride` apart, `offset` floats into memory that is NaN elsewhere."""
    rows, cols = x.shape
    stride = stride or cols
    host = np.full(offset + max(rows, 1) * stride + 8, np.nan, np.float32)
    host[offset:offset + rows * stride].reshape(rows, stride)[:, :cols] = x
    mem = torch.from_numpy(host).cuda()
    d = torch.as_strided(mem, (rows, cols), (stride, 1), offset)
    t = torch.from_numpy(np.ascontiguousarray(tokens, dtype=np.int32)).cuda()
    lp, entropy = torch.full(t.shape, MARK, device="cuda"), torch.full((rows,), MARK, device="cuda")
    top = torch.full((rows, k), 77, dtype=torch.int32, device="cuda") if k else None
    top_lp = torch.full((rows, k), MARK, device="cuda") if k else None
    ws = torch.full((pk.logprobs_workspace(rows, cols, k),), 0xff, dtype=torch.uint8, device="cuda")
    pk.logprobs_dev(d, t, lp, entropy, top, top_lp, ws)
    torch.cuda.synchronize()
    assert np.array_equal(mem.cpu().numpy(), host, equal_nan=True)
    return [None if y is None else y.cpu().numpy() for y in (lp, entropy, top, top_lp)]


def check(pk, torch, x, tokens, k, **where):
    lp, entropy, top, top_lp = ask(pk, torch, x, tokens, k, **where)
    want, bound, h, hb = pr.answer(x, tokens)
    same = (lp == want) | (np.abs(lp - np.where(np.isinf(want), 0, want)) <= np.where(np.isinf(want), -1, bound))
    assert same.all(), np.argwhere(~same)[:4]
    assert (np.abs(entropy - h) <= hb).all(), (np.abs(entropy - h) / hb).max()
    if k:
        ids = pr.order(x)[:, :k]
        assert np.array_equal(top, ids)
        want, bound, _, _ = pr.answer(x, ids)
        same = (top_lp == want) | (np.abs(top_lp - np.where(np.isinf(want), 0, want)) <= np.where(np.isinf(want), -1, bound))
        assert same.all()


def logits(g, rows, cols, spread=2.0, peak=12.0):
    x = spread * g.standard_normal((rows, cols))
    x[np.arange(rows), g.integers(0, cols, rows)] += peak * g.random(rows)
    return x.astype(np.float32)


COLS = (1, 2, 3, 5, 63, 64, 65, 255, 256, 257, 512, 700, 1000, 1025, 1030, 1500, 1537, 1800, 2047, 2048, 2049, 4097, 8191,
        8192, 8193, 16385, 50001)


@pytest.mark.parametrize("cols", COLS)
@pytest.mark.parametrize("rows", [1, 7])
def test_sizes(hip, torch, cols, rows):
    say("size", rows, cols)
    g = np.random.default_rng(cols)
    x = logits(g, rows, cols)
    tokens = g.integers(0, cols, (rows, 3))
    tokens[:, 0] = x.argmax(1)
    check(hip, torch, x, tokens, min(cols, 5), stride=cols + g.integers(0, 5), offset=int(g.integers(0, 4)))


@pytest.mark.parametrize("k", [0, 1, 2, 8, 20, 31, 32])
@pytest.mark.parametrize("cols", [40, 1025, 5000, 40000])
def test_alternatives(hip, torch, cols, k):
    say("top", cols, k)
    g = np.random.default_rng(k)
    check(hip, torch, logits(g, 9, cols), g.integers(0, cols, (9, 1)), k)


@pytest.mark.parametrize("cols", [5, 64, 300, 1025, 5000, 20000])
def test_ties(hip, torch, cols):
    """Equal logits, of a few values or of one, zeros of both signs among them: lowest ids first."""
    say("ties", cols)
    g = np.random.default_rng(cols)
    k = min(cols, 32)
    for x in (np.zeros((4, cols)), g.integers(-1, 2, (4, cols)), np.where(g.random((4, cols)) < 0.5, 0.0, -0.0),
              g.integers(0, 40, (4, cols)) / 8, -np.sort(-g.integers(0, 9, (4, cols)), 1), np.sort(g.integers(0, 9, (4, cols)), 1)):
        check(hip, torch, x.astype(np.float32), g.integers(0, cols, (4, 2)), k)


@pytest.mark.parametrize("cols", [4, 1025, 5000, 20000])
def test_magnitudes(hip, torch, cols):
    """Rows far from zero, wide apart, certain, and with columns masked to -infinity or the type's lowest value."""
    say("magnitudes", cols)
    g = np.random.default_rng(cols + 1)
    k = min(cols, 6)
    tokens = g.integers(0, cols, (6, 3))
    base = logits(g, 6, cols)
    check(hip, torch, base + np.float32(3e4), tokens, k)
    check(hip, torch, base - np.float32(3e4), tokens, k)
    check(hip, torch, base * np.float32(1e4), tokens, k)
    check(hip, torch, base * np.float32(1e-4), tokens, k)
    certain = base.copy()
    certain[:, 2] += 60
    tokens[:, 1] = 2
    check(hip, torch, certain, tokens, k)
    lp = ask(hip, torch, certain, tokens, 0)[0]
    if cols > 4:
        assert (lp[:, 1] < 0).all() and (lp[:, 1] > -1e-12).all()       # not rounded to a probability of 1
    for low in (-np.inf, np.finfo(np.float32).min):
        masked = np.where(g.random(base.shape) < 0.5, np.float32(low), base)
        masked[:, 0] = 1.0
        check(hip, torch, masked, tokens, min(k, 2))
        alone = np.full_like(base, low)
        alone[:, cols - 1] = -3.0
        check(hip, torch, alone, tokens, 1)


@pytest.mark.parametrize("cols", [6, 1025, 5000, 20000])
def test_rows_without_a_distribution(hip, torch, cols):
    """NaN, infinities, nothing but -infinity: NaN there, the order kept, and the rows beside them as they are."""
    say("bad rows", cols)
    g = np.random.default_rng(cols + 2)
    x = logits(g, 8, cols)
    tokens = g.integers(0, cols, (8, 2))
    clean = ask(hip, torch, x, tokens, 5)
    x[1, 3] = np.nan
    x[2, cols - 1] = np.inf
    x[3] = -np.inf
    x[4] = np.nan
    x[5, :-2] = np.nan
    x[6, 0], x[6, cols - 1] = np.inf, np.nan
    got = ask(hip, torch, x, tokens, 5)
    bad = slice(1, 7)
    assert np.isnan(got[1][bad]).all() and np.isnan(got[3][bad]).all()
    assert np.isnan(got[0][bad]).all()
    assert np.array_equal(got[2], pr.order(x)[:, :5])
    for a, b in zip(got, clean):
        assert np.array_equal(a[[0, 7]], b[[0, 7]])


def test_tokens_that_are_none(hip, torch):
    say("no tokens")
    g = np.random.default_rng(3)
    for cols in (7, 1025, 9000):
        x = logits(g, 4, cols)
        tokens = np.array([[-1, 0, cols, -2, cols - 1, 0x7fffffff, -0x80000000]] * 4)
        lp = ask(hip, torch, x, tokens, 0)[0]
        assert (lp[:, 0] == 0).all() and np.isnan(lp[:, [2, 3, 5, 6]]).all() and np.isfinite(lp[:, [1, 4]]).all()


def test_one_result_at_a_time(hip, torch):
    """Each result alone is what all together are."""
    say("alone")
    g = np.random.default_rng(4)
    for rows, cols in ((5, 1025), (3, 3000), (2, 20000)):
        x = logits(g, rows, cols)
        tokens = g.integers(0, cols, (rows, 100))
        lp, entropy, top, top_lp = ask(hip, torch, x, tokens, 7)
        d, t = torch.from_numpy(x).cuda(), torch.from_numpy(tokens.astype(np.int32)).cuda()
        ws = torch.empty(hip.logprobs_workspace(rows, cols, 7), dtype=torch.uint8, device="cuda")
        o = [torch.zeros(rows, 100, device="cuda"), torch.zeros(rows, device="cuda"),
             torch.zeros(rows, 7, dtype=torch.int32, device="cuda")]
        hip.logprobs_dev(d, t, o[0], ws=ws)
        hip.logprobs_dev(d, entropy=o[1], ws=ws)
        hip.logprobs_dev(d, top=o[2], ws=ws)
        torch.cuda.synchronize()
        for a, b in zip(o, (lp, entropy, top)):
            assert np.array_equal(a.cpu().numpy(), b)


@pytest.mark.parametrize("seed", range(12))
def test_any_call(hip, torch, seed):
    r = random.Random(seed)
    rows, cols = r.choice([1, 3, 50, 300]), int(2 ** r.uniform(0, 13.5))
    say("any", seed, rows, cols)
    g = np.random.default_rng(seed)
    x = logits(g, rows, cols, 10 ** r.uniform(-2, 1.5), r.choice([0, 20]))
    check(hip, torch, x, g.integers(0, cols, (rows, r.randint(1, 5))), r.randint(0, min(32, cols)),
          stride=cols + r.randint(0, 9), offset=r.randint(0, 5))


def test_widest(hip, torch):
    say("widest")
    g = np.random.default_rng(8)
    x = logits(g, 2, 1 << 20)
    check(hip, torch, x, np.array([[0, (1 << 20) - 1], x.argmax(1)]), 32)


def test_rows_past_32_bits(hip, torch):
    """Rows whose offset passes 2^32 bytes."""
    say("far rows")
    g = np.random.default_rng(9)
    mem = torch.zeros((1 << 30) + 4096, device="cuda")
    x = logits(g, 2, 1025)
    rows = torch.as_strided(mem, (2, 1025), (1 << 30, 1), 7)
    rows.copy_(torch.from_numpy(x))
    t = torch.tensor([[3], [9]], dtype=torch.int32, device="cuda")
    lp = torch.zeros(2, 1, device="cuda")
    hip.logprobs_dev(rows, t, lp)
    want, bound, _, _ = pr.answer(x, np.array([[3], [9]]))
    assert (np.abs(lp.cpu().numpy() - want) <= bound).all()


def test_same_bits_two_streams_and_a_graph(hip, torch):
    say("streams")
    g = np.random.default_rng(5)
    for rows, cols in ((100, 1025), (30, 30000)):
        x = logits(g, rows, cols)
        tokens = g.integers(0, cols, (rows, 2))
        want = ask(hip, torch, x, tokens, 8)
        d, t = torch.from_numpy(x).cuda(), torch.from_numpy(tokens.astype(np.int32)).cuda()
        n = hip.logprobs_workspace(rows, cols, 8)
        sets = [[torch.empty_like(t, dtype=torch.float32), torch.empty(rows, device="cuda"),
                 torch.empty(rows, 8, dtype=torch.int32, device="cuda"), torch.empty(rows, 8, device="cuda"),
                 torch.empty(n, dtype=torch.uint8, device="cuda")] for _ in range(3)]
        ss = [torch.cuda.Stream() for _ in range(2)]
        torch.cuda.synchronize()
        for _ in range(10):
            for s, o in zip(ss, sets):
                with torch.cuda.stream(s):
                    hip.logprobs_dev(d, t, *o)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            hip.logprobs_dev(d, t, *sets[2])
        for _ in range(3):
            for o in sets[2]:
                o.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert all(np.array_equal(a.cpu().numpy(), b) for a, b in zip(sets[2], want))
            (torch.randn(256, 256, device="cuda") @ torch.randn(256, 256, device="cuda")).sum().item()
        for o in sets[:2]:
            assert all(np.array_equal(a.cpu().numpy(), b) for a, b in zip(o, want))


def test_beside_the_joint(hip, torch):
    """The joint's logits: its token is the first alternative, and the durations' columns are asked as they lie."""
    say("joint")
    from libpktito_amd import synth
    dec = synth.decoder_weights(np.random.default_rng(2))
    d = hip.DeviceDecoder(dec, torch)
    d.predict(3)
    f = torch.randn(d.J, device="cuda")
    d.joint(f)
    V, n = d.V + 1, d.n_dur
    lg = d.logit[None]
    for cols, at in ((lg[:, :V], 0), (lg[:, V:V + n], 1)):
        k = min(3, cols.shape[1])
        top = torch.zeros(1, k, dtype=torch.int32, device="cuda")
        lp = torch.zeros(1, k, device="cuda")
        hip.logprobs_dev(cols, top=top, top_lp=lp)
        torch.cuda.synchronize()
        assert top[0, 0].item() == d.tok_dur[at].item()
        x = cols.cpu().numpy()
        want, bound, _, _ = pr.answer(x, pr.order(x)[:, :k])
        assert (np.abs(lp.cpu().numpy() - want) <= bound).all()
    d.release()


def test_nothing_to_do(hip, torch):
    e = torch.zeros(0, 9, device="cuda")
    hip.logprobs_dev(e, entropy=torch.zeros(0, device="cuda"))
