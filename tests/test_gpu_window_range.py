"""Attention with a window and sinks over the whole range of floats: the greatest
and the lowest ones, infinities, the smallest, in rows that attend them, against 64
bits (window_ref.attend). Calls of few tiles and of so many that keys and values
are cut into pieces."""
import sys

import numpy as np
import pytest

import window_ref as wr
from test_gpu_window import Call

pytestmark = pytest.mark.gpu
DKS = (32, 64, 96, 128)
FEW, MANY = (120, 2), (2200, 16)
F32 = np.finfo(np.float32)


def say(*a):
    print("[case]", *a, flush=True)
    sys.stdout.flush()


@pytest.fixture(scope="module")
def torch():
    import torch
    assert torch.cuda.is_available()
    return torch


def want(c, rows, positions, left, right, sinks, without=()):
    """The outputs of rows of the first segment and their bound, as if the frames `without` were not there."""
    frames = np.setdiff1d(np.arange(c.Ts[0]), without)
    out = [wr.attend(c.q[i:i + 1], i, frames, c.k[frames], c.v[frames], c.H, c.dk, positions, left, right, sinks)
           for i in rows]
    return np.concatenate([x[0] for x in out]), np.concatenate([x[1] for x in out])


def near(got, ref, bound):
    off = np.abs(got - ref)
    assert np.isfinite(got).all() and (off <= bound).all(), (got[off > bound][:4], ref[off > bound][:4], off.max())


@pytest.mark.parametrize("T,H", [FEW, MANY])
@pytest.mark.parametrize("dk", DKS)
@pytest.mark.parametrize("with_positions", [False, True])
@pytest.mark.parametrize("lowest", [F32.min, -np.inf, np.float32(-(2.0 ** 127) * (2 - 2.0 ** -8))])
def test_a_dimension_as_a_mask(hip, torch, T, H, dk, with_positions, lowest):
    """Frames masked by a key of the type's lowest value (or an infinity) where queries are 1: weight 0, and rows that
    attend them as if they were not there; one row attends nothing else and is not asked for."""
    say("mask", T, H, dk, with_positions, lowest)
    c = Call(hip, torch, [T, 50], H, H, dk, seed=dk)
    left, right, sinks = 20, 3, 2
    pos = c.positions(left, right) if with_positions else None
    at = np.arange(H) * dk + 5
    c.q[:, at] = 1.0
    masked = np.array([1, 60, 61, 62, 77, T - 2])
    c.k[np.ix_(masked, at)] = lowest
    got = c.attend(pos, left, right, sinks)
    rows = [0, 1, 30, 58, 59, 60, 61, 62, 70, 77, 79, 82, 83, 97, T - 20, T - 2, T - 1]
    near(got[rows], *want(c, rows, pos, left, right, sinks, masked))


@pytest.mark.parametrize("T,H", [FEW, MANY])
@pytest.mark.parametrize("dk", DKS)
@pytest.mark.parametrize("with_positions", [False, True])
@pytest.mark.parametrize("small,great", [(2.0 ** -126, F32.max), (1e-30, 1e30), (1e-18, 1e18), (1e30, 1e-30), (1e18, 1e-18),
                                         (F32.max / 4, 2.0 ** -125), (2.0 ** 49, 2.0 ** -50)])
def test_small_queries_great_keys(hip, torch, T, H, dk, with_positions, small, great):
    """A dimension whose queries are as small as its keys are great, and the other way round: scores of both signs."""
    say("scales", T, H, dk, with_positions, small, great)
    c = Call(hip, torch, [T, 50], H, H, dk, seed=dk)
    left, right, sinks = 20, 3, 2
    pos = c.positions(left, right) if with_positions else None
    at = np.arange(H) * dk + 5
    if pos:
        pos[2][at] = pos[3][at] = 0         # the smallest queries stay as small with their biases
        pos[0][:, at] = 0
    sign = np.where(c.g.random((c.rows, H)) < 0.5, -1, 1)
    q = (1 + 0.5 * c.g.random((c.rows, H))) * (small if small < 1 else small / 2)
    k = sign * (0.5 + 0.5 * c.g.random((c.rows, H))) * great
    c.q[:, at], c.k[:, at] = q.astype(np.float32), k.astype(np.float32)
    got = c.attend(pos, left, right, sinks)
    rows = [0, 1, 30, 59, 60, 77, 100, T - 2, T - 1]
    near(got[rows], *want(c, rows, pos, left, right, sinks))


def great(c, dims, ceiling):
    """Values up to the type's greatest in some dimensions of each head; scores that rise by 7.8 powers of two from one 16
    frames to the next, so sums of weights are far over what they are to the greatest score."""
    d = np.arange(c.H) * c.dk
    c.k[:, d + 9] = (7.8 * np.log(2) * (np.arange(c.rows) // 16 % 2))[:, None]
    c.q[:, d + 9] = np.sqrt(c.dk)
    sign = np.where(c.g.random((c.rows, c.H)) < 0.5, -1, 1)
    for n, x in zip(dims, (ceiling, ceiling * sign, ceiling * (2 * c.g.random((c.rows, c.H)) - 1),
                           np.where(np.arange(c.rows)[:, None] == 60, ceiling, 1.0))):
        c.v[:, d + n] = np.broadcast_to(x, (c.rows, c.H)).astype(np.float32)


@pytest.mark.parametrize("T,H", [FEW, MANY])
@pytest.mark.parametrize("dk", DKS)
@pytest.mark.parametrize("with_positions", [False, True])
@pytest.mark.parametrize("ceiling", [1e30, 1e34, 1e36, float(F32.max)])
def test_great_values(hip, torch, T, H, dk, with_positions, ceiling):
    """Outputs that floats hold, of sums that they do not: the other dimensions keep their bits."""
    say("great", T, H, dk, with_positions, ceiling)
    c = Call(hip, torch, [T, 50], H, H, dk, seed=dk)
    left, right, sinks = 70, 33, 2
    pos = c.positions(left, right) if with_positions else None
    dims = (0, 7, dk // 2 + 1, dk - 1)
    great(c, dims, 1.0)
    clean = c.attend(pos, left, right, sinks)
    c.g = np.random.default_rng(7)
    great(c, dims, ceiling)
    got = c.attend(pos, left, right, sinks)
    other = np.setdiff1d(np.arange(H * dk), (np.arange(H)[:, None] * dk + np.array(dims)).ravel())
    assert np.array_equal(got[:, other], clean[:, other])
    rows = [0, 1, 15, 16, 30, 59, 60, 77, 100, T - 40, T - 2, T - 1]
    near(got[rows], *want(c, rows, pos, left, right, sinks))


@pytest.mark.parametrize("T,H", [FEW, MANY])
@pytest.mark.parametrize("with_positions", [False, True])
def test_great_values_in_place(hip, torch, T, H, with_positions):
    """The same with the output over the queries, which the rows made again still need."""
    say("great in place", T, H, with_positions)
    c = Call(hip, torch, [T, 50], H, H, 64, seed=3)
    pos = c.positions(70, 33) if with_positions else None
    great(c, (0, 7, 33, 63), float(F32.max))
    expected = c.attend(pos, 70, 33, 2)
    q, k, v = c.dev(c.q), c.dev(c.k), c.dev(c.v)
    at = None if pos is None else (c.dev(pos[0]), pos[1], c.dev(pos[2]), c.dev(pos[3]))
    hip.attention_window_dev(q, q, k, v, hip.Segments(c.dev(c.row0), c.rows, c.max_T), H, 64, at, 70, 33, 2)
    torch.cuda.synchronize()
    assert np.isfinite(expected).all() and np.array_equal(q.cpu().numpy(), expected)


@pytest.mark.parametrize("T,H", [FEW, MANY])
@pytest.mark.parametrize("dk", DKS)
@pytest.mark.parametrize("with_positions", [False, True])
def test_scores_that_are_no_floats(hip, torch, T, H, dk, with_positions):
    """Rows all of whose scores are under the type's lowest are the softmax of them all the same, the value of the frame
    that is far over the others; rows all of whose scores are -infinity are 0."""
    say("no floats", T, H, dk, with_positions)
    c = Call(hip, torch, [T, 50], H, H, dk, seed=dk)
    left, right, sinks = 20, 3, 2
    pos = c.positions(left, right) if with_positions else None
    at = np.arange(H) * dk + 5
    c.q[30:34, at], c.q[70:72, at] = 1e38, 1.0
    c.k[:, at] = np.float32(-1e20) * np.arange(1, c.rows + 1, dtype=np.float32)[:, None]
    got = c.attend(pos, left, right, sinks)
    assert (got[30:34] == c.v[0]).all()
    c.k[np.ix_([0, 1, *range(70 - left, 72 + right)], at)] = -np.inf
    got = c.attend(pos, left, right, sinks)
    assert (got[70:72] == 0).all()


@pytest.mark.parametrize("T,H", [FEW, MANY])
@pytest.mark.parametrize("dk", DKS)
@pytest.mark.parametrize("with_positions", [False, True])
@pytest.mark.parametrize("size", [1e-24, 1e-30, 1e-33, 1e-36, 2.0 ** -125])
def test_small_values(hip, torch, T, H, dk, with_positions, size):
    """Values that keep the bits of 32 however small they are, and those of dimensions small beside others."""
    say("small", T, H, dk, with_positions, size)
    c = Call(hip, torch, [T, 50], H, H, dk, seed=dk)
    left, right, sinks = 20, 3, 2
    pos = c.positions(left, right) if with_positions else None
    c.v *= np.float32(size)
    c.v[:, 4::9] *= np.float32(1e20)
    got = c.attend(pos, left, right, sinks)
    rows = [0, 1, 30, 59, 60, 77, 100, T - 2, T - 1]
    ref, bound = want(c, rows, pos, left, right, sinks)
    # the model's bound has 1e-37 for what ends at 2^-126: here a product or a sum of the 26 that is rounded at 2^-149, and
    # as many times that again by the weights of up to 2^8 and their sum
    near(got[rows], ref, bound - 1e-37 + 64 * 2.0 ** -149)


@pytest.mark.parametrize("dk", [64, 128])
@pytest.mark.parametrize("kind", ["content", "content, great", "places, great"])
def test_two_streams_and_a_graph(hip, torch, dk, kind):
    """Calls of many tiles give the same bits on two streams at once, captured and replayed: without positions, and with
    values whose rows are made again."""
    say("streams", dk, kind)
    H = 4
    c = Call(hip, torch, [3001, 700, 1, 5100], H, H, dk, seed=24)
    pos = c.positions(60, 10) if "places" in kind else None
    if "great" in kind:
        c.v[1000:1100, ::7], c.v[20, 3] = 1e38, np.nan
    want_ = c.attend(pos, 60, 10, 4)
    d = [c.dev(x) for x in (c.q, c.k, c.v)]
    p = None if pos is None else (c.dev(pos[0]), pos[1], c.dev(pos[2]), c.dev(pos[3]))
    sg = hip.Segments(c.dev(c.row0), c.rows, c.max_T)
    o = [torch.zeros_like(d[0]) for _ in range(3)]
    ss = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(5):
        for i, s in enumerate(ss):
            with torch.cuda.stream(s):
                hip.attention_window_dev(o[i], *d, sg, H, dk, p, 60, 10, 4)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        hip.attention_window_dev(o[2], *d, sg, H, dk, p, 60, 10, 4)
    same = lambda x: np.array_equal(x.cpu().numpy(), want_, equal_nan=True)
    for _ in range(3):
        o[2].zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert same(o[2])
        (torch.randn(256, 256, device="cuda") @ torch.randn(256, 256, device="cuda")).sum().item()
    assert all(same(x) for x in o[:2])
    assert np.isfinite(want_).all() == (kind == "content")


@pytest.mark.parametrize("T,H", [FEW, MANY])
@pytest.mark.parametrize("dk", DKS)
@pytest.mark.parametrize("with_positions", [False, True])
@pytest.mark.parametrize("span", [100, 45])
def test_any_magnitudes(hip, torch, T, H, dk, with_positions, span):
    """Each dimension of queries, and against it of keys and positions, and of values at a power of two of its own."""
    say("any magnitudes", T, H, dk, with_positions, span)
    c = Call(hip, torch, [T, 50], H, H, dk, seed=span)
    left, right, sinks = 25, 6, 3
    e = np.float32(2.0) ** c.g.integers(-span, span + 1, H * dk).astype(np.float32)
    f = np.float32(2.0) ** c.g.integers(-110, 111, H * dk).astype(np.float32)
    c.q, c.k, c.v = c.q * e, c.k / e, c.v * f
    pos = None
    if with_positions:
        p, center, u, w = c.positions(left, right)
        pos = (p / e, center, u * e, w * e)
    got = c.attend(pos, left, right, sinks)
    rows = [0, 1, 30, 59, 60, 77, 100, T - 2, T - 1]
    ref, bound = want(c, rows, pos, left, right, sinks)
    near(got[rows], ref, bound - 1e-37 + 64 * 2.0 ** -149)
