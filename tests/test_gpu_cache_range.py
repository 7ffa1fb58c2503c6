"""The cache's attention with the greatest floats in its positions, against 64 bits
(window_ref.attend)."""
import sys

import numpy as np
import pytest

import window_ref as wr
from test_gpu_cache import World
from test_gpu_sinks import attend

pytestmark = pytest.mark.gpu
F32 = np.finfo(np.float32)


def say(*a):
    print("[case]", *a, flush=True)
    sys.stdout.flush()


@pytest.fixture(scope="module")
def torch():
    import torch
    assert torch.cuda.is_available()
    return torch


@pytest.mark.parametrize("B,T,left,dk", [(B, T, 70, dk) for B, T in ((2, 1), (20, 1), (3, 7), (3, 90)) for dk in (32, 64, 96, 128)]
                         + [(1, 1300, 2000, 32)])        # the last one's table is cut beforehand
@pytest.mark.parametrize("sinks", [0, 5])
@pytest.mark.parametrize("lowest", [F32.min, np.float32(-(2.0 ** 127) * (2 - 2.0 ** -8))])
def test_a_dimension_of_positions_as_a_mask(hip, torch, B, T, left, dk, sinks, lowest):
    """Distances masked by a position of the type's lowest value where queries are 1, whether its scores are made beforehand
    or where they are used: weight 0, rows as if those frames were not there."""
    say("positions mask", B, T, dk, sinks, lowest)
    G, H, right = 2, 2, 4
    w = World(hip, torch, [100 + 7 * b for b in range(B)], [T] * B, G, dk, seed=dk)
    w.fill()
    p, center, u, b_ = w.positions(H, left, right)
    at = np.arange(H) * dk + 5
    u[at] = b_[at] = 0
    masked = np.array([1, 2, 33, left - 1])             # frames behind the row by these
    p[np.ix_(center - masked, at)] = lowest
    q = w.g.standard_normal((w.rows, H * dk)).astype(np.float32)
    q[:, at] = 1.0
    got = attend(w, q, H, (p, center, u, b_), left, right, sinks)
    for s, t in {(0, 0), (B - 1, T - 1), (B // 2, T // 2)}:
        pos, total = w.lens[s] + t, w.lens[s] + T
        both = [np.concatenate([np.concatenate(w.pool.read(w.layer, w.table[s, pg], g), 1)
                                for pg in range(-(-total // 64))])[:total] for g in range(G)]
        k, v = (np.concatenate([x[:, n * dk:(n + 1) * dk] for x in both], 1) for n in (0, 1))
        frames = np.setdiff1d(np.arange(total), pos - masked)
        row = w.row0[s] + t
        ref, bound = wr.attend(q[row:row + 1], pos, frames, k[frames], v[frames], H, dk, (p, center, u, b_), left, right, sinks)
        off = np.abs(got[row:row + 1] - ref)
        assert np.isfinite(got[row]).all() and (off <= bound).all(), (s, t, off.max())
