"""The cache's attention with a window and sinks on the GPU, against 64 bits within
the bound that 32-bit arithmetic gives, and the operators together: a plan, the
write, the attention, the joint's confidence, step after step."""
import random
import sys

import numpy as np
import pytest

import probs_ref as pr
import window_ref as wr
from test_gpu_cache import World

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


def attend(w, q, H, positions, left, right, sinks, inplace=False):
    torch = w.torch
    pos = None if positions is None else (w.dev(positions[0]), positions[1], w.dev(positions[2]), w.dev(positions[3]))
    o = torch.full((w.rows, H * w.dk), 7.25, device="cuda")
    need = w.cache.attention_workspace(w.streams, H, pos, left, right, sinks)
    ws = torch.full((max(1, need),), 0xff, dtype=torch.uint8, device="cuda")
    w.cache.attention(o, w.layer, w.dev(q), w.streams, H, ws, pos, left, right, sinks=sinks)
    torch.cuda.synchronize()
    return o.cpu().numpy()


def want(w, q, H, positions, left, right, sinks):
    out, bound = np.full(q.shape, 7.25), np.zeros(q.shape)
    for b, n0 in enumerate(w.lens):
        T = w.Ts[b]
        total = min(n0 + T, 64 * w.table.shape[1])
        k, v, frames = [np.zeros((0, w.G * w.dk))], [np.zeros((0, w.G * w.dk))], []
        for pg in range(-(-total // 64)):
            id_ = w.table[b, pg]
            if 0 <= id_ < w.pool.data.shape[1]:
                n = min(64, total - 64 * pg)
                both = [w.pool.read(w.layer, id_, g) for g in range(w.G)]
                k.append(np.concatenate([x[0][:n] for x in both], 1))
                v.append(np.concatenate([x[1][:n] for x in both], 1))
                frames += range(64 * pg, 64 * pg + n)
        r = slice(w.row0[b], w.row0[b] + T)
        out[r], bound[r] = wr.attend(q[r], n0, np.array(frames, int), np.concatenate(k), np.concatenate(v), H, w.dk,
                                     positions, left, right, sinks)
    return out, bound


def check(w, H, positions=None, left=None, right=None, sinks=0):
    q = w.g.standard_normal((w.rows, H * w.dk)).astype(np.float32)
    got = attend(w, q, H, positions, left, right, sinks)
    ref, bound = want(w, q, H, positions, left, right, sinks)
    off = np.abs(got - ref)
    assert np.isfinite(got).all() and (off <= bound).all(), (off.max(), np.argwhere(off > bound)[:4])
    assert np.linalg.norm(off) <= 1e-5 * np.linalg.norm(ref) + 1e-30


def holes(w, r, share):
    """Some pages given up."""
    w.table[w.g.random(w.table.shape) < share] = r.choice([-1, 1 << 20])


@pytest.mark.parametrize("dk", DKS)
@pytest.mark.parametrize("H,G", [(1, 1), (4, 4), (6, 2), (3, 1)])
@pytest.mark.parametrize("with_positions", [False, True])
def test_sinks(hip, torch, dk, H, G, with_positions):
    say("sinks", dk, H, G, with_positions)
    for Ts in ([1, 3, 0, 2], [20, 1, 64, 5]):
        w = World(hip, torch, [300, 0, 10, 131], Ts, G, dk, seed=dk + H, first=2, tail=3)
        w.fill()
        check(w, H, w.positions(H, 40, 3) if with_positions else None, 40, 3, 5)


@pytest.mark.parametrize("left,right", [(0, 0), (1, None), (63, 0), (64, 1), (65, 0), (200, 5), (None, 0)])
@pytest.mark.parametrize("sinks", [1, 63, 64, 65, 130, 100000])
def test_reaches(hip, torch, left, right, sinks):
    say("reach", left, right, sinks)
    for Ts in ([1, 2], [7, 30]):
        w = World(hip, torch, [270, 63], Ts, 2, 32, seed=sinks % 97)
        w.fill()
        check(w, 2, None, left, right, sinks)
        check(w, 2, w.positions(2, 400 if left is None else left, 30), left, right, sinks)


@pytest.mark.parametrize("B", [1, 3, 16, 20])
@pytest.mark.parametrize("dk", DKS)
def test_single_frames(hip, torch, B, dk):
    """A frame of each stream, a narrow window: position scores made where they are used, and beforehand."""
    say("frames", B, dk)
    r = random.Random(B)
    w = World(hip, torch, [r.choice([0, 3, 200, 700]) for _ in range(B)], [1] * B, 2, dk, seed=B)
    w.fill()
    for left in (5, 70, 200):
        check(w, 2, w.positions(2, left, 0), left, 0, 4)
        check(w, 2, None, left, 0, 70)


@pytest.mark.parametrize("seed", range(16))
def test_any_call(hip, torch, seed):
    r = random.Random(seed)
    G = r.choice([1, 2, 3])
    H, dk = G * r.choice([1, 1, 2, 4]), r.choice(DKS)
    B = r.randint(1, 5)
    lens = [r.choice([0, 64, r.randint(0, 600)]) for _ in range(B)]
    Ts = [r.choice([1, 1, r.randint(0, 9), r.randint(0, 80)]) for _ in range(B)]
    say("any", seed, lens, Ts, H, G, dk)
    if not sum(Ts):
        return
    w = World(hip, torch, lens, Ts, G, dk, seed, first=r.randint(0, 2), tail=r.randint(0, 2), slack_T=r.choice([0, 5]))
    if r.random() < 0.5:
        holes(w, r, 0.3)
    w.fill()
    pos = w.positions(H, r.randint(0, 200), r.randint(0, 90)) if r.random() < 0.6 else None
    check(w, H, pos, r.choice([None, 0, r.randint(0, 200)]), r.choice([None, 0, r.randint(0, 60)]),
          r.choice([1, r.randint(1, 70), r.randint(1, 400)]))


@pytest.mark.parametrize("B,T,pages,H,G,dk", [(1, 1, 40, 1, 1, 128), (1, 1, 70, 2, 2, 64), (3, 4, 36, 2, 1, 64),
                                              (1, 20, 40, 2, 2, 32), (2, 40, 35, 1, 1, 128)])
@pytest.mark.parametrize("with_positions", [False, True])
def test_pages_in_splits(hip, torch, B, T, pages, H, G, dk, with_positions):
    """Windows of so many pages that several workgroups share them, with sinks' pages before them."""
    say("splits", B, T, pages, H, G, dk)
    w = World(hip, torch, [64 * (pages + 8) + 5 * b for b in range(B)], [T] * B, G, dk, seed=pages)
    w.fill()
    check(w, H, w.positions(H, 64 * pages, 0) if with_positions else None, 64 * pages, 0, 150)


@pytest.mark.parametrize("with_positions", [False, True])
@pytest.mark.parametrize("T", [2, 40])
def test_rows_past_the_table(hip, torch, with_positions, T):
    """Streams that outgrew their table: rows past it attend the sinks, and what of the window it holds."""
    say("past", T)
    for left in (0, 20, 100):
        w = World(hip, torch, [120, 128, 100, 90], [T] * 4, 2, 32, seed=T, max_pages=2)
        w.fill()
        check(w, 4, w.positions(4, left, 9) if with_positions else None, left, 9, 6)


def test_table_cut_beforehand(hip, torch):
    """So many rows by distances that the positions' table is cut by a launch of its own."""
    say("cut")
    w = World(hip, torch, [3000], [900], 1, 32, seed=3)
    w.fill()
    H, left = 1, 2900
    pos = w.positions(H, left, 0)
    q = w.g.standard_normal((900, 32)).astype(np.float32)
    got = attend(w, q, H, pos, left, 0, 100)
    k, v = (np.concatenate([w.pool.read(0, p, 0)[i] for p in w.table[0]])[:3900] for i in range(2))
    for i in (0, 17, 400, 899):
        ref, bound = wr.attend(q[i:i + 1], 3000 + i, np.arange(3900), k, v, H, 32, pos, left, 0, 100)
        assert (np.abs(got[i] - ref) <= bound).all(), i


def test_no_sinks_is_the_attention_without(hip, torch):
    """Sinks that no row has behind its window change no bit."""
    say("none")
    for Ts in ([2, 1], [30, 17]):
        w = World(hip, torch, [150, 20], Ts, 2, 64, seed=5)
        w.fill()
        q = w.g.standard_normal((w.rows, 4 * 64)).astype(np.float32)
        for pos in (None, w.positions(4, 60, 5)):
            assert np.array_equal(attend(w, q, 4, pos, 60, 5, 0), w.attend(q, 4, pos, 60, 5))
        assert np.array_equal(attend(w, q, 4, None, None, 5, 9), w.attend(q, 4, None, None, 5))


def test_holes_hide_sinks(hip, torch):
    """Sinks whose page was given up are not attended, whatever its place in the pool holds."""
    say("holes")
    w = World(hip, torch, [400, 400], [1, 1], 1, 64, seed=6)
    w.table[0, 0] = -1
    w.fill()
    check(w, 2, None, 30, 0, 10)
    check(w, 2, w.positions(2, 30, 0), 30, 0, 100)
    w.table[:, :] = -1
    w.upload()
    q = w.g.standard_normal((2, 128)).astype(np.float32)
    assert (attend(w, q, 2, None, 30, 0, 10) == 0).all()


def test_steps_together(hip, torch):
    """Streams served in steps with nothing of a step on the host: a plan, the write of keys and values, the attention with
    a window and sinks, the joint's confidence, captured once and replayed, against whole segments attended in one call
    from what the cache keeps. Pages given back are used again, so the pool holds a window of each stream and no more."""
    say("together")
    B, H, dk, steps, T, left, sinks, V = 3, 2, 64, 40, 20, 100, 7, 50
    D = H * dk
    g = torch.Generator(device="cuda").manual_seed(7)
    rnd = lambda *s: torch.randn(*s, device="cuda", generator=g)
    pages = B * 5                           # the sinks' page, the window's and the one that is filled
    plan = hip.CachePlan.empty(pages, B, 40, B * T, T, True)
    cache = hip.DeviceCache(torch.zeros(hip.cache_bytes(1, pages, H, dk), dtype=torch.uint8, device="cuda"), 1, pages, H, dk)
    p = (rnd(left + T, D), left, 0.1 * rnd(D), 0.1 * rnd(D))
    ws = torch.empty(cache.attention_workspace(plan.streams, H, p, left, 0, sinks), dtype=torch.uint8, device="cuda")
    q, k, v, o, ko, vo = (torch.zeros(B * T, D, device="cuda") for _ in range(6))
    lg = torch.zeros(B * T, V, device="cuda")
    top, top_lp = torch.zeros(B * T, 3, dtype=torch.int32, device="cuda"), torch.zeros(B * T, 3, device="cuda")
    add, fresh = (torch.zeros(B, dtype=torch.int32, device="cuda") for _ in range(2))

    def step():
        plan.step(add, fresh, left, sinks)
        cache.append(0, k, v, plan.streams)
        cache.read(0, ko, vo, plan.streams)
        cache.attention(o, 0, q, plan.streams, H, ws, p, left, 0, sinks=sinks)
        lg.copy_(3 * o[:, :V])
        hip.logprobs_dev(lg, top=top, top_lp=top_lp)

    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        step()                              # what libraries keep is made before the capture; nothing is added
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    r = random.Random(8)
    kept = [[] for _ in range(B)]           # each stream's (q, kept k, kept v, o)
    whole = []

    def end(b):
        if kept[b]:
            whole.append([torch.cat(x) for x in zip(*kept[b])])
        kept[b] = []

    for n in range(steps):
        new = [int(n > 0 and r.random() < 0.05) for _ in range(B)]
        T_b = [r.randint(0, T) for _ in range(B)]
        add.copy_(torch.tensor(T_b, dtype=torch.int32))
        fresh.copy_(torch.tensor(new, dtype=torch.int32))
        for x in (q, k, v):
            x.copy_(rnd(B * T, D))
        graph.replay()
        torch.cuda.synchronize()
        row0 = plan.streams.row0.tolist()
        assert row0 == [0, T_b[0], T_b[0] + T_b[1], sum(T_b)] and plan.told.tolist()[:3] == [sum(T_b), 0, 0]
        for b in range(B):
            if new[b]:
                end(b)
            rows = slice(row0[b], row0[b + 1])
            kept[b].append([x[rows].clone() for x in (q, ko, vo, o)])
        rows = slice(0, row0[-1])
        x = lg[rows].cpu()
        ids = pr.order(x.numpy())[:, :3]        # equal ones, as single frames kept in 4 bits give: the lowest first
        lp, bound, _, _ = pr.answer(x.numpy(), ids)
        assert np.array_equal(top[rows].cpu().numpy(), ids)
        assert (np.abs(top_lp[rows].cpu().numpy() - lp) <= bound).all()
    for b in range(B):
        end(b)
    assert max(len(x[0]) for x in whole) > 64 * 4
    for qq, kk, vv, oo in whole:
        n = len(qq)
        if not n:
            continue
        row0 = torch.tensor([0, n], dtype=torch.int32, device="cuda")
        again = torch.zeros_like(oo)
        hip.attention_window_dev(again, qq, kk, vv, hip.Segments(row0, n, n), H, dk, p, left, 0, sinks)
        ref, bound = wr.attend(*(a.cpu().numpy() if torch.is_tensor(a) else a for a in (qq, 0, np.arange(n), kk, vv)), H, dk,
                               tuple(a.cpu().numpy() if torch.is_tensor(a) else a for a in p), left, 0, sinks)
        for x in (oo, again):
            assert (np.abs(x.cpu().numpy() - ref) <= bound).all()
