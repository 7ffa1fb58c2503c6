"""The plan of a step on the GPU against its host model, number for number, and
a stream's life through plan, append and attention."""
import random
import sys

import numpy as np
import pytest

import plan_ref as pr

pytestmark = pytest.mark.gpu


def say(*a):
    print("[case]", *a, flush=True)
    sys.stdout.flush()


@pytest.fixture(scope="module")
def torch():
    import torch
    assert torch.cuda.is_available()
    return torch


class Both:
    """A plan on the device and its model, stepped together."""

    def __init__(self, pk, torch, pages, B, max_pages, rows, max_T, slots=True):
        self.torch = torch
        self.model = pr.Plan(pages, B, max_pages, rows, max_T)
        self.plan = pk.CachePlan.empty(pages, B, max_pages, rows, max_T, slots)
        if slots:
            self.plan.slot.fill_(99)

    def dev(self, x):
        return None if x is None else self.torch.tensor(list(x), dtype=self.torch.int32, device="cuda")

    def step(self, add, fresh=None, left=None, sinks=0):
        m, p = self.model, self.plan
        m.step(add, fresh, left, sinks)
        p.step(self.dev(add), self.dev(fresh), left, sinks)
        self.torch.cuda.synchronize()
        host = lambda t: t.cpu().numpy()
        assert host(p.told).tolist() == m.told
        assert np.array_equal(host(p.streams.len), m.len) and np.array_equal(host(p.streams.row0), m.row0)
        assert np.array_equal(host(p.table), m.table) and np.array_equal(host(p.state), m.state)
        pool = host(p.pool)
        assert pool[0] == m.head and pool[1] == len(m.queue)
        assert [pool[2 + (m.head + i) % m.pages] for i in range(len(m.queue))] == m.queue
        if p.slot is not None:
            assert np.array_equal(host(p.slot), m.slot)


@pytest.mark.parametrize("seed", range(20))
def test_lives(hip, torch, seed):
    """Streams that come, grow, slide and go, over pools that are ample or short."""
    r = random.Random(seed)
    B = r.choice([1, 2, 7, 64, 65, 300])
    max_T = r.choice([1, 3, 64, 65, 200])
    max_pages = r.choice([1, 2, 9, 40])
    rows = max(max_T, r.choice([B * max_T, B * max_T // 2, 50]))
    pages = r.choice([1, 5, B * 3, B * max_pages])
    say("life", seed, B, max_T, max_pages, rows, pages)
    both = Both(hip, torch, pages, B, max_pages, rows, max_T)
    left = r.choice([None, 0, 1, 63, 64, 200])
    sinks = r.choice([0, 1, 64, 65])
    for _ in range(12):
        add = [r.choice([0, -1, 1, max_T, r.randint(0, 2 * max_T)]) for _ in range(B)]
        fresh = r.choice([None, [int(r.random() < 0.2) for _ in range(B)]])
        both.step(add, fresh, left, sinks)
        if r.random() < 0.2:
            left, sinks = r.choice([None, 10, 100]), r.choice([0, 3, 130])


@pytest.mark.parametrize("B", [1023, 1024, 1025, 3000])
def test_many_streams(hip, torch, B):
    """More streams than the kernel has threads: pages given back by late ones are taken by early ones."""
    say("streams", B)
    both = Both(hip, torch, 2 * B + B // 2, B, 6, 70 * B, 70)
    r = random.Random(B)
    for i in range(7):
        both.step([r.choice([0, 60, 64, 70]) for _ in range(B)], [int(b > B // 2 and i == 4) for b in range(B)], 64, 1)


def test_long_streams_end(hip, torch):
    """Tables of thousands of columns given back at once."""
    say("long")
    both = Both(hip, torch, 9000, 3, 4000, 300000, 150000)
    both.step([150000, 64 * 2500 + 5, 100])
    both.step([100000, 1, 1])
    both.step([0, 0, 9], [1, 1, 0])
    both.step([3, 70, 9])
    assert both.model.told[3] > 8900


def test_sums_past_32_bits(hip, torch):
    say("sums")
    both = Both(hip, torch, 10, 5, 4, 100, 90)
    both.step([0x7fffffff] * 5)
    assert both.model.told[:2] == [100, 0x7fffffff]


def test_numbers_that_no_call_leaves(hip, torch):
    """State, pool and table of any numbers: results in range, and nothing outside of the arrays written."""
    say("any numbers")
    r = np.random.default_rng(1)
    B, max_pages, pages, rows = 70, 5, 30, 120
    for trial in range(6):
        big = lambda *shape: r.choice([-(1 << 31), -1, 0, 3, 29, 30, 200, 320, 321, (1 << 31) - 1], shape).astype(np.int32)
        sizes = dict(table=B * max_pages, state=2 * B, pool=2 + pages, slot=rows)
        whole = torch.from_numpy(big(sum(sizes.values()) + 5 * 64)).cuda()
        parts, at, marks = {}, 64, [(0, 64)]
        for name, n in sizes.items():
            parts[name] = whole[at:at + n]
            marks.append((at + n, at + n + 64))
            at += n + 64
        before = whole.cpu().numpy().copy()
        plan = hip.CachePlan(parts["table"].view(B, max_pages), parts["state"].view(B, 2), parts["pool"], rows, 40,
                             parts["slot"])
        for _ in range(3):
            plan.step(torch.from_numpy(big(B)).cuda(), torch.from_numpy(big(B)).cuda() if trial % 2 else None, 10, 70)
        torch.cuda.synchronize()
        after = whole.cpu().numpy()
        for a, b in marks:
            b = min(b, len(after))
            assert np.array_equal(before[a:b], after[a:b])
        row0, length = plan.streams.row0.cpu().numpy(), plan.streams.len.cpu().numpy()
        assert (np.diff(row0) >= 0).all() and row0[0] == 0 and row0[-1] <= rows and (np.diff(row0) <= 40).all()
        assert (length >= 0).all() and (length + np.diff(row0) <= 64 * max_pages).all()
        pool, slot = parts["pool"].cpu().numpy(), parts["slot"].cpu().numpy()
        assert 0 <= pool[0] < pages and 0 <= pool[1] <= pages and (slot >= -1).all() and (slot < 64 * pages).all()


def test_no_streams_and_no_rows(hip, torch):
    say("none")
    both = Both(hip, torch, 4, 0, 3, 5, 5)
    both.step([])
    assert both.model.slot.tolist() == [-1] * 5
    both = Both(hip, torch, 4, 2, 3, 0, 0)
    both.step([3, 1])
    both.step([0, 1], [1, 1], 5, 1)


def test_graph_of_steps(hip, torch):
    """A plan captured once and replayed does what steps do, `add` and `fresh` changed in place."""
    say("graph")
    B = 9
    both = Both(hip, torch, 30, B, 20, 100, 30)
    add, fresh = (torch.zeros(B, dtype=torch.int32, device="cuda") for _ in range(2))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        both.plan.step(add, fresh, 100, 5)
    step = both.plan.step
    both.plan.step = lambda a, f, left, sinks: (add.copy_(a), fresh.copy_(f), graph.replay())
    r = random.Random(4)
    for _ in range(15):
        both.step([r.randint(0, 30) for _ in range(B)], [int(r.random() < 0.1) for _ in range(B)], 100, 5)
        (torch.randn(256, 256, device="cuda") @ torch.randn(256, 256, device="cuda")).sum().item()
    both.plan.step = step
    both.step([1] * B, [0] * B, 100, 5)


def test_two_plans_on_two_streams(hip, torch):
    say("two streams")
    ss = [torch.cuda.Stream() for _ in range(2)]
    plans = [hip.CachePlan.empty(50, 20, 10, 400, 20, True) for _ in range(2)]
    adds = [torch.full((20,), n, dtype=torch.int32, device="cuda") for n in (20, 7)]
    models = [pr.Plan(50, 20, 10, 400, 20) for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(6):
        for s, p, a, m in zip(ss, plans, adds, models):
            with torch.cuda.stream(s):
                p.step(a, None, 30, 2)
            m.step(a.tolist(), None, 30, 2)
    torch.cuda.synchronize()
    for p, m in zip(plans, models):
        assert np.array_equal(p.table.cpu().numpy(), m.table) and p.told.tolist() == m.told
        assert np.array_equal(p.slot.cpu().numpy(), m.slot)
