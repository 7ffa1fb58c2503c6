"""The 4-bit cache of keys and values without a GPU: the layout's arithmetic (the
header the kernels take every address and bound from, compiled for the host),
the pool of pages, and what the entries refuse."""
import ctypes
import os
import random
import subprocess
import sys

import numpy as np
import pytest

import cache_ref as cr

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DKS = (32, 64, 96, 128)


@pytest.fixture(scope="module")
def layout(tmp_path_factory):
    so = str(tmp_path_factory.mktemp("layout") / "layout.so")
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-ffp-contract=off", "-shared", "-fPIC",
                    "-fsanitize=undefined", "-fno-sanitize-recover=all", "-I",
                    os.path.join(ROOT, "libpktito_amd", "csrc"), os.path.join(ROOT, "tests", "cache_layout_host.cpp"),
                    "-o", so], check=True)
    l = ctypes.CDLL(so)
    f, u, i = ctypes.c_float, ctypes.c_uint32, ctypes.c_int32
    for name, res, args in (("t_scale", u, [f]), ("t_code", u, [f, f]), ("t_level", f, [u]), ("t_record", u, [u]),
                            ("t_key_at", u, [u, u]), ("t_value_dword", u, [u] * 4), ("t_frame_of", u, [u] * 3),
                            ("t_key_scale_at", u, [u, u]), ("t_value_scale_at", u, [u, u]),
                            ("t_page_ok", ctypes.c_int, [i, u]), ("t_tile_pages", u, [u, i, i]), ("t_place_stride", u, [u]),
                            ("t_place_pad", u, []),
                            ("t_lo", i, [i, i]), ("t_hi", i, [i, i, i]),
                            ("t_span", None, [u, u, u, i, i, i, ctypes.POINTER(i)])):
        getattr(l, name).restype, getattr(l, name).argtypes = res, args
    return l


def test_scale_is_the_least_that_holds(layout):
    g = np.random.default_rng(1)
    tops = np.concatenate([g.standard_normal(3000).astype(np.float32), np.float32(2.0) ** g.uniform(-121, 126.9, 3000),
                           [2.0 ** -121, np.nextafter(np.float32(2.0 ** 127), np.float32(0)), 6.0, 1.5, 0.75,
                            np.nextafter(np.float32(6), np.float32(7))]]).astype(np.float32)
    for top in np.abs(tops):
        got = layout.t_scale(float(top))
        want = cr.scale_of(float(top))
        assert np.uint32(got << 16).view(np.float32) == np.float32(want), top
        if want:
            assert 6 * want >= top > 6 * float(np.uint32((got - 1) << 16).view(np.float32))
    for top in (0.0, np.nextafter(np.float32(2.0 ** -121), np.float32(0)), 2.0 ** 127, 3.4e38, np.inf, np.nan):
        assert layout.t_scale(float(top)) == 0


def test_code_is_the_nearest_level(layout):
    g = np.random.default_rng(2)
    for _ in range(40):
        d = cr.scale_of(float(np.float32(abs(g.standard_normal()) * 10.0 ** g.uniform(-30, 30))))
        mid = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0]) * d
        x = np.concatenate([g.uniform(-6, 6, 200) * d, mid, -mid, cr.LEVELS * d, [0.0, -0.0]]).astype(np.float32)
        x = np.concatenate([x, np.nextafter(x, np.float32(np.inf)), np.nextafter(x, np.float32(-np.inf))])
        x = x[np.abs(x) <= 6 * d]
        want = cr.codes_of(x, d)
        got = np.array([layout.t_code(float(v), d) for v in x], np.uint8)
        assert np.array_equal(got, want)
    for c in range(16):
        assert layout.t_level(c) == cr.LEVELS[c & 7] * (-1 if c & 8 else 1)


@pytest.mark.parametrize("dk", DKS)
def test_record_holds_each_value_once(layout, dk):
    """Every nibble of a record belongs to one (which, frame, dimension), every
    scale to one frame; nothing lies outside the record; dwords are aligned."""
    n = layout.t_record(dk)
    assert n == cr.record_bytes(dk) and n % 16 == 0
    used = np.zeros(2 * n, int)
    for f in range(64):
        for c in range(dk):
            used[2 * (layout.t_key_at(dk, f) + c // 2) + c % 2] += 1
        for at in (layout.t_key_scale_at(dk, f), layout.t_value_scale_at(dk, f)):
            assert at % 2 == 0
            used[2 * at:2 * at + 4] += 1
    pool = cr.Pool(1, 1, 1, dk)
    for c in range(dk):
        for g in range(2):
            for w in range(4):
                at = layout.t_value_dword(dk, c, g, w)
                assert at % 4 == 0
                for i in range(8):
                    used[2 * (at + i // 2) + i % 2] += 1
                    byte, shift = pool._value_at(layout.t_frame_of(g, w, i), c)
                    assert (byte, shift) == (at + i // 2, 4 * (i % 2))
    assert (used == 1).all()


def test_spans_stay_in_bounds(layout):
    """Whatever the arrays hold: rows in the call, frames in the table, and a
    tile's pages and position scores where they are counted."""
    r = random.Random(3)
    odd = [0, 1, -1, 2 ** 31 - 1, -2 ** 31, 63, 64, 65, 1000]
    out = (ctypes.c_int32 * 4)()
    for _ in range(20000):
        max_pages = r.choice([1, 2, 3, 100, 1 << 24])
        rows = r.choice([0, 1, 5, 300, 1 << 22])
        max_T = r.randint(0, rows)
        pick = lambda: r.choice(odd) if r.random() < 0.3 else r.randint(0, 400)
        layout.t_span(max_pages, rows, max_T, pick(), pick(), pick(), out)
        r0, T, ln, total = out
        assert 0 <= r0 and 0 <= T <= max_T and r0 + T <= rows
        assert 0 <= ln <= total <= 64 * max_pages and total <= ln + T
        left, right = min(r.choice(odd[:1] + odd[5:]), 64 * max_pages - 1), min(r.choice([0, 3, 1000]), max(0, max_T - 1))
        if T == 0:
            continue
        t0 = r.randint(0, T - 1)
        t1 = min(T - 1, t0 + r.randint(0, 15))
        j0, j1 = layout.t_lo(ln + t0, left), layout.t_hi(ln + t1, right, total)
        for pg in {j0 // 64, max(j0 // 64, j1 // 64)}:
            if 64 * pg > j1:
                continue
            assert 0 <= pg < max_pages
            assert pg - j0 // 64 < layout.t_tile_pages(max_pages, left, right), (left, right, j0, j1)
            for pos in (ln + t0, ln + t1):
                first = layout.t_place_pad() + 64 * pg - (pos - left)
                assert 0 <= first and first + 64 <= layout.t_place_stride(left + right + 1), (pos, left, right, pg)
    for id, pages, ok in ((0, 1, 1), (1, 1, 0), (-1, 5, 0), (-2 ** 31, 5, 0), (4, 5, 1), (2 ** 31 - 1, 1 << 30, 0)):
        assert bool(layout.t_page_ok(id, pages)) == bool(ok)


# ------------------------------------------------------------------ pool --

def test_pool_counts_holders():
    import libpktito_amd as pk
    p = pk.PagePool(130)
    assert p.free_pages == 130
    a = p.alloc(3)
    assert a == [0, 1, 2] and p.free_pages == 127
    p.share([1, 1])
    assert [p.holders(i) for i in (0, 1, 2, 3, -1, 130)] == [1, 3, 1, 0, 0, 0]
    p.release([1, 0, 1])
    assert p.free_pages == 128 and p.holders(1) == 1 and p.alloc(1) == [0]
    with pytest.raises(pk.PkHipError) as e:
        p.alloc(128)
    assert e.value.code == pk.PK_HIP_ENOMEM and p.free_pages == 127
    for bad in ([3], [-1], [130], [2, 2]):
        with pytest.raises(pk.PkHipError) as e:
            p.release(bad)
        assert e.value.code == pk.PK_HIP_EINVAL
        assert [p.holders(i) for i in (0, 1, 2)] == [1, 1, 1]
    with pytest.raises(pk.PkHipError):
        p.share([0, 7])
    assert p.holders(0) == 1
    p.share([2])
    p.release([2, 2])                   # both holders in one call: free once
    assert p.free_pages == 128
    with pytest.raises(pk.PkHipError):
        pk.PagePool(0)


def test_pool_against_a_model():
    import libpktito_amd as pk
    r = random.Random(4)
    for pages in (1, 63, 64, 200):
        p, model = pk.PagePool(pages), {}
        for _ in range(400):
            what = r.random()
            free = [i for i in range(pages) if i not in model]
            if what < 0.4:
                n = r.randint(0, 5)
                if n <= len(free):
                    assert p.alloc(n) == free[:n]
                    model.update({i: 1 for i in free[:n]})
                else:
                    with pytest.raises(pk.PkHipError):
                        p.alloc(n)
            elif what < 0.6 and model:
                ids = r.choices(sorted(model), k=r.randint(1, 3))
                p.share(ids)
                for i in ids:
                    model[i] += 1
            elif what < 0.9 and model:
                i = r.choice(sorted(model))
                p.release([i])
                model[i] -= 1
                model = {k: v for k, v in model.items() if v}
            else:
                cap = r.choice([0, 1, 2, pages])
                pairs = (ctypes.c_int32 * (2 * pages + 2))()
                n = ctypes.c_uint32()
                assert pk.lib().pk_hip_pool_compact(p.handle, pairs, cap, ctypes.byref(n)) == 0
                moves = [(pairs[2 * i], pairs[2 * i + 1]) for i in range(n.value)]
                want = sum(i >= len(model) for i in model)
                assert len(moves) == min(cap, want)
                assert len({t for _, t in moves} | {f for f, _ in moves}) == 2 * len(moves)
                for f, t in moves:
                    assert f in model and t not in model and t < f
                    model[t] = model.pop(f)
                if cap == pages:
                    assert sorted(model) == list(range(len(model)))
            assert p.free_pages == pages - len(model)
            assert [p.holders(i) for i in range(pages)] == [model.get(i, 0) for i in range(pages)]


class _Moves:
    """Stands for a cache: keeps the pairs that the pool would have moved."""
    def __init__(self, pages):
        self.st, self.pairs, self.device = type("St", (), {"pages": pages}), [], 0

    def move(self, pairs, table=None, source=None, stream=None):
        self.pairs += pairs


def test_compact_refuses_before_it_moves():
    """A limit under 0 (which an unsigned count would take for all pages, more
    than the pairs' array holds) and a table that cannot follow leave the pool
    as it was."""
    import torch
    import libpktito_amd as pk
    p, cache = pk.PagePool(8), _Moves(8)
    p.release(p.alloc(5)[:3])
    for table, most in ((None, -1), (None, -(1 << 32)), (torch.zeros(2, 4, dtype=torch.int32), None),
                        (torch.zeros(2, 4, dtype=torch.int64), None)):
        with pytest.raises(pk.PkHipError) as e:
            p.compact(cache, table, most)
        assert e.value.code == pk.PK_HIP_EINVAL
        assert [p.holders(i) for i in range(8)] == [0, 0, 0, 1, 1, 0, 0, 0] and not cache.pairs
    assert p.compact(cache, None, 0) == [] and p.compact(cache, None, 1) == [(4, 0)] == cache.pairs
    assert p.compact(cache, None) == [(3, 1)] and [p.holders(i) for i in range(4)] == [1, 1, 0, 0]


def test_fork_takes_what_a_stream_has():
    """Frames that the pages do not hold, and pages that nobody holds, are
    refused with nothing taken; holes stay holes."""
    import libpktito_amd as pk
    p, cache = pk.PagePool(8), _Moves(8)
    ids = p.alloc(3)
    for pages, frames in ((ids, -1), (ids, 3 * 64 + 1), ([], 1), ([5], 64), ([5], 10), (ids + [5], 200), (ids + [5], 256)):
        with pytest.raises(pk.PkHipError) as e:
            p.fork(cache, pages, frames)
        assert e.value.code == pk.PK_HIP_EINVAL and not cache.pairs
        assert p.free_pages == 5 and [p.holders(i) for i in range(4)] == [1, 1, 1, 0]
    assert p.fork(cache, [-1, 1, 2], 140) == [-1, 1, 3] and cache.pairs == [(2, 3)]
    assert [p.holders(i) for i in range(4)] == [1, 2, 1, 1]
    assert p.fork(cache, [0, 8], 100) == [0, 8] and p.fork(cache, [-1], 64) == [-1] and cache.pairs == [(2, 3)]
    assert [p.holders(i) for i in range(4)] == [2, 2, 1, 1] and p.free_pages == 4


# -------------------------------------------------------------- refusals --

def _calls(pk, **change):
    """Each entry's return for a call that is in order but for `change` (all have
    one, so nothing is launched: the pointers stand for device memory)."""
    v = dict(data=4096, layers=2, pages=8, heads=4, dk=64, table=4096, len=4096, row0=4096, B=2, max_pages=4, rows=5,
             max_T=3, layer=1, k=4096, ks=256, v=4096, vs=256, o=4096, os=512, q=8192, qs=512, H=8, p=4096, bu=4096,
             bw=4096, n=9, center=4, ws=4096, ws_bytes=1 << 40)
    v.update(change)
    c = pk.Cache(v["data"], v["layers"], v["pages"], v["heads"], v["dk"])
    st = pk.Streams(v["table"], v["len"], v["row0"], v["B"], v["max_pages"], v["rows"], v["max_T"])
    pos = pk.Positions(v["p"], v["bu"], v["bw"], v["n"], v["center"])
    l, r = pk.lib(), ctypes.byref
    return {
        "append": lambda: l.pk_hip_cache_append_dev(r(c), v["layer"], v["k"], v["ks"], v["v"], v["vs"], r(st), None),
        "read": lambda: l.pk_hip_cache_read_dev(r(c), v["layer"], v["k"], v["ks"], v["v"], v["vs"], r(st), None),
        "attention": lambda: l.pk_hip_attention_cache_dev(v["o"], v["os"], v["q"], v["qs"], r(c), v["layer"], r(st),
                                                          v["H"], r(pos), 10, 10, v["ws"], v["ws_bytes"], None),
    }


BOTH = ("append", "read")
ALL = BOTH + ("attention",)


@pytest.mark.parametrize("entries,change", [
    (ALL, {"data": None}), (ALL, {"data": 4100}), (ALL, {"layers": 0}), (ALL, {"pages": 0}), (ALL, {"heads": 0}),
    (ALL, {"dk": 48}), (ALL, {"dk": 0}), (ALL, {"dk": 160}), (ALL, {"dk": 256}), (ALL, {"pages": 1 << 31}),
    (ALL, {"layer": 2}), (ALL, {"table": None}), (ALL, {"len": None}), (ALL, {"row0": None}), (ALL, {"max_pages": 0}),
    (ALL, {"max_pages": (1 << 24) + 1}), (ALL, {"B": 65536}), (ALL, {"rows": (1 << 22) + 1}), (ALL, {"max_T": 6}),
    (BOTH, {"k": None}), (BOTH, {"v": None}), (BOTH, {"k": 4104}), (BOTH, {"v": 4100}), (BOTH, {"ks": 252}),
    (BOTH, {"vs": 0}), (BOTH, {"ks": 258}), (BOTH, {"vs": 257}),
    (("attention",), {"o": None}), (("attention",), {"q": None}), (("attention",), {"o": 4104}),
    (("attention",), {"q": 4104}), (("attention",), {"os": 508}), (("attention",), {"qs": 508}),
    (("attention",), {"qs": 514}), (("attention",), {"H": 0}), (("attention",), {"H": 6}),
    (("attention",), {"p": None}), (("attention",), {"bu": None}), (("attention",), {"bw": None}),
    (("attention",), {"p": 4104}), (("attention",), {"center": 9}), (("attention",), {"n": 0, "center": 0}),
    (("attention",), {"ws": None}), (("attention",), {"ws": 4104}), (("attention",), {"ws_bytes": 100}),
    (("attention",), {"q": 4096, "qs": 516}),
    (("attention",), {"B": 65535, "rows": 1 << 21, "max_T": 1 << 21}),      # more workgroups than a launch holds
], ids=lambda v: "-".join(f"{k}={x}" for k, x in v.items()) if isinstance(v, dict) else "")
def test_refusals(entries, change):
    import libpktito_amd as pk
    calls = _calls(pk, **change)
    for e in entries:
        assert calls[e]() == pk.PK_HIP_EINVAL, e
        assert pk.lib().pk_hip_last_error()


@pytest.mark.parametrize("pairs,change", [
    ([(0, 8)], {}), ([(8, 0)], {}), ([(-1, 0)], {}), ([(0, -1)], {}),
    ([(0, 1), (2, 1)], {}),                     # copied to twice
    ([(0, 1), (1, 2)], {}), ([(3, 3)], {}),     # copied from and to
    ([(0, 1), (0, 2)], {"table": 4096}),        # moves to two places
    ([(i, 4) for i in range(9)], {}),           # more pairs than pages
    ([(0, 1)], {"dst": dict(dk=32)}), ([(0, 1)], {"dst": dict(heads=2)}), ([(0, 1)], {"dst": dict(layers=1)}),
    ([(0, 1)], {"dst": dict(pages=4)}),         # one memory, two sizes
    ([(0, 1)], {"dst": dict(data=8192)}),       # memories that overlap
    ([(0, 1)], {"dst": dict(data=1 << 30), "table": 4096}),
])
def test_move_refusals(pairs, change):
    import libpktito_amd as pk
    base = dict(data=4096, layers=2, pages=8, heads=4, dk=64)
    src = pk.Cache(**base)
    dst = pk.Cache(**(base | change.get("dst", {})))
    flat = np.array(pairs, np.int32).reshape(-1)
    assert pk.lib().pk_hip_cache_move_dev(ctypes.byref(dst), ctypes.byref(src), flat.ctypes.data, len(pairs),
                                          change.get("table"), 16, None) == pk.PK_HIP_EINVAL
    assert pk.lib().pk_hip_last_error()


def test_sizes():
    import libpktito_amd as pk
    for dk in DKS:
        assert pk.cache_bytes(3, 5, 7, dk) == 3 * 5 * 7 * cr.record_bytes(dk)
    for bad in ((0, 1, 1, 64), (1, 0, 1, 64), (1, 1, 0, 64), (1, 1, 1, 16), (1, 1, 1025, 64)):
        assert pk.cache_bytes(*bad) == 0


def test_sizes_past_what_a_size_holds():
    """Products that pass 64 bits are no size (41361 x 2^30 x 1024 x 8448 would
    come out as a smaller one), and a cache of them is refused."""
    import libpktito_amd as pk
    assert pk.cache_bytes(24, 1 << 20, 8, 128) == 24 * (1 << 20) * 8 * cr.record_bytes(128)
    for big in ((41361, 1 << 30, 1024, 128), (65535, 1 << 30, 1024, 32), (65535, (1 << 30) - 1, 1023, 96)):
        n = big[0] * big[1] * big[2] * cr.record_bytes(big[3])
        assert n > 2 ** 64 and pk.cache_bytes(*big) == 0
        calls = _calls(pk, layers=big[0], pages=big[1], heads=big[2], dk=big[3], H=big[2], ks=1 << 20, vs=1 << 20,
                       os=1 << 20, qs=1 << 20)
        for e in ALL:
            assert calls[e]() == pk.PK_HIP_EINVAL, e


def test_host_tensors_are_refused():
    import torch
    import libpktito_amd as pk
    z = torch.zeros(2, 4, dtype=torch.int32)
    with pytest.raises(pk.PkHipError, match="device tensor"):
        pk.CacheStreams(z, z[0, :2], z[0, :3], 4, 2)
    with pytest.raises(pk.PkHipError, match="device tensor"):
        pk.DeviceCache(torch.zeros(1 << 20, dtype=torch.uint8), 1, 1, 1, 64)


class _Device:
    """Stands for a device tensor in calls that are refused before one is read."""
    is_cuda = True

    def __init__(self, dtype, *shape, dense=True, device=0):
        self.dtype, self.shape, self.dense, self.device = dtype, shape, dense, f"cuda:{device}"
        self.get_device = lambda: device

    def numel(self):
        return int(np.prod(self.shape))

    def dim(self):
        return len(self.shape)

    def is_contiguous(self):
        return self.dense

    def stride(self):
        return self.shape[1], 1

    def data_ptr(self):
        return 4096


def _wrapped(pk, torch):
    i32 = lambda *s: _Device(torch.int32, *s)
    return (pk.DeviceCache(_Device(torch.uint8, pk.cache_bytes(2, 8, 4, 64)), 2, 8, 4, 64),
            pk.CacheStreams(i32(2, 4), i32(2), i32(3), 5, 3))


@pytest.mark.parametrize("past", [-1, -(1 << 32), 1 << 32, (1 << 32) + 1])
def test_numbers_past_32_bits_are_refused(monkeypatch, past):
    """A number whose last 32 bits would do is not taken for those."""
    import torch
    import libpktito_amd as pk
    monkeypatch.setattr(pk, "_device", lambda: 0)
    cache, st = _wrapped(pk, torch)
    f = lambda n: _Device(torch.float32, 5, n)
    kv, q, ws, b = f(256), f(512), _Device(torch.uint8, 1 << 24), _Device(torch.float32, 512)
    at = lambda center: (_Device(torch.float32, 9, 512), center, b, b)
    i32 = lambda *s: _Device(torch.int32, *s)
    pool = pk.PagePool(8)
    pool.alloc(2)
    for call in (lambda: cache.append(past, kv, kv, st), lambda: cache.read(past, kv, kv, st),
                 lambda: cache.attention(q, past, q, st, 8, ws), lambda: cache.attention(q, 0, q, st, 8, ws, left=past),
                 lambda: cache.attention(q, 0, q, st, 8, ws, right=past), lambda: cache.attention(q, 0, q, st, 8, ws, at(past)),
                 lambda: cache.attention_workspace(st, 8, None, past), lambda: cache.attention_workspace(st, 8, None, 1, past),
                 lambda: cache.attention_workspace(st, past, None), lambda: cache.attention_workspace(st, past, at(4)),
                 lambda: cache.move([(0, past)], stream=0), lambda: cache.move([(past, 0)], stream=0),
                 lambda: pk.CacheStreams(i32(2, 4), i32(2), i32(3), past, 3),
                 lambda: pk.CacheStreams(i32(2, 4), i32(2), i32(3), 5, past),
                 lambda: pk.DeviceCache(_Device(torch.uint8, 1 << 40), past, 8, 4, 64),
                 lambda: pk.DeviceCache(_Device(torch.uint8, 1 << 40), 2, past, 4, 64),
                 lambda: pk.DeviceCache(_Device(torch.uint8, 1 << 40), 2, 8, past, 64),
                 lambda: pool.alloc(past), lambda: pool.share([past]), lambda: pool.release([0, past]),
                 lambda: pk.PagePool(past)):
        with pytest.raises(pk.PkHipError) as e:
            call()
        assert e.value.code == pk.PK_HIP_EINVAL
    assert pool.holders(past) == 0 and pool.holders(0) == 1 and pool.free_pages == 6


@pytest.mark.parametrize("B,max_T,heads,ok", [(65535, 1 << 21, 4, False), (65535, 2, 1024, True), (65535, 66, 1024, True),
                                              (65535, 450, 1024, False), (2048, 1 << 20, 8, False), (2048, 1 << 20, 7, True)])
def test_launches_past_what_is_run(B, max_T, heads, ok):
    """Pages of all streams and heads, 2^28 at most. The calls that are in order
    end at a null k, which is looked at after."""
    import libpktito_amd as pk
    assert ((max_T + 62) // 64 + 1) * B * heads <= 1 << 28 if ok else True
    calls = _calls(pk, B=B, rows=1 << 21, max_T=max_T, heads=heads, ks=1 << 18, vs=1 << 18, k=None)
    for e in BOTH:
        assert calls[e]() == pk.PK_HIP_EINVAL
        assert (b"launch holds" in pk.lib().pk_hip_last_error()) == (not ok)


def test_workspaces_that_are_none_are_refused():
    import torch
    import libpktito_amd as pk
    cache, st = _wrapped(pk, torch)
    q = _Device(torch.float32, 5, 512)
    for ws in (torch.zeros(1 << 20, dtype=torch.uint8), _Device(torch.float32, 1 << 20),
               _Device(torch.uint8, 1 << 20, dense=False)):
        with pytest.raises(pk.PkHipError) as e:
            cache.attention(q, 0, q, st, 8, ws, stream=0)
        assert e.value.code == pk.PK_HIP_EINVAL and ("ws" in str(e.value))


def test_other_devices_are_refused(monkeypatch):
    """Tensors on another device than the cache's, and a current device that is
    another (where the launch would go)."""
    import torch
    import libpktito_amd as pk
    cache, st = _wrapped(pk, torch)
    other = pk.DeviceCache(_Device(torch.uint8, pk.cache_bytes(2, 8, 4, 64), device=1), 2, 8, 4, 64)
    f = lambda *s, device=0: _Device(torch.float32, *s, device=device)
    i32 = lambda *s, device=0: _Device(torch.int32, *s, device=device)
    kv, q, b, ws = f(5, 256), f(5, 512), f(512), _Device(torch.uint8, 1 << 24)
    kv1, q1, b1, ws1 = f(5, 256, device=1), f(5, 512, device=1), f(512, device=1), _Device(torch.uint8, 1 << 24, device=1)
    st1 = pk.CacheStreams(i32(2, 4, device=1), i32(2, device=1), i32(3, device=1), 5, 3)
    p = f(9, 512)

    def refused(*calls):
        for call in calls:
            with pytest.raises(pk.PkHipError) as e:
                call()
            assert e.value.code == pk.PK_HIP_EINVAL

    monkeypatch.setattr(pk, "_device", lambda: 0)
    refused(lambda: pk.CacheStreams(i32(2, 4), i32(2, device=1), i32(3), 5, 3),
            lambda: pk.CacheStreams(i32(2, 4), i32(2), i32(3, device=1), 5, 3),
            lambda: cache.append(0, kv1, kv, st, 0), lambda: cache.append(0, kv, kv1, st, 0),
            lambda: cache.append(0, kv, kv, st1, 0), lambda: cache.read(0, kv, kv1, st, 0),
            lambda: cache.read(0, kv, kv, st1, 0), lambda: cache.attention(q1, 0, q, st, 8, ws, stream=0),
            lambda: cache.attention(q, 0, q1, st, 8, ws, stream=0), lambda: cache.attention(q, 0, q, st1, 8, ws, stream=0),
            lambda: cache.attention(q, 0, q, st, 8, ws1, stream=0),
            lambda: cache.attention(q, 0, q, st, 8, ws, (f(9, 512, device=1), 4, b, b), stream=0),
            lambda: cache.attention(q, 0, q, st, 8, ws, (p, 4, b1, b), stream=0),
            lambda: cache.attention(q, 0, q, st, 8, ws, (p, 4, b, b1), stream=0),
            lambda: cache.move([(0, 1)], i32(2, 4, device=1), stream=0), lambda: cache.move([(0, 1)], None, other, 0),
            lambda: pk.PagePool(8).compact(cache, i32(2, 4, device=1)))
    monkeypatch.setattr(pk, "_device", lambda: 1)
    refused(lambda: cache.append(0, kv, kv, st, 0), lambda: cache.read(0, kv, kv, st, 0),
            lambda: cache.attention(q, 0, q, st, 8, ws, stream=0), lambda: cache.move([(0, 1)], stream=0))


def test_reference_round_trip():
    """The host model of a pool keeps what its own quantizer gives."""
    g = np.random.default_rng(5)
    for dk in DKS:
        pool = cr.Pool(1, 2, 2, dk)
        x = g.standard_normal((64, 2, 2 * dk)).astype(np.float32)
        for f in range(64):
            pool.write(0, 1, f, x[f, 0], x[f, 1])
        for h in range(2):
            for which in range(2):
                want, _, _ = cr.kept(x[:, which], 2)
                got = pool.read(0, 1, h)[which]
                assert np.array_equal(got, want[:, h * dk:(h + 1) * dk])


def test_windows_reach_the_first_frame(layout):
    """Streams that outgrow their tables, up to the largest: the widest window has
    frame 0 in it for every row, the narrower ones theirs, and the distances
    between a block's rows and the frames are right (the build stops at sums that
    pass 32 bits)."""
    i, u = ctypes.c_int32, ctypes.c_uint32
    layout.t_most_left.restype, layout.t_most_left.argtypes = i, [u, u]
    layout.t_places.restype, layout.t_places.argtypes = None, [u, u, u, i, i, i, i, i, i, ctypes.POINTER(i)]
    r, out = random.Random(6), (i * 6)()
    for _ in range(20000):
        max_pages = r.choice([1, 2, 100, 1 << 24])
        cap = 64 * max_pages
        T = r.choice([1, 4, 300, 1 << 21])
        n = r.choice([0, cap, cap - 1, max(0, cap - T), r.randint(0, cap)])
        most = layout.t_most_left(max_pages, T)
        t0 = r.choice([0, T - 1, r.randint(0, T - 1)])
        t1 = r.randint(t0, T - 1)
        left = r.choice([most, min(most, cap), cap - 1, r.randint(0, most)])
        layout.t_places(max_pages, T, T, 0, T, n, t0, t1 + 1, left, out)
        _, rows, ln, total, lo, hi = out
        assert (rows, ln, total) == (T, n, min(n + T, cap))
        assert layout.t_lo(ln + t1, most) == 0 and layout.t_lo(ln + t1, left) == max(0, ln + t1 - left)
        assert lo == left - (ln + t1) and hi == left + total - 1 - (ln + t0)


class _Fails(_Moves):
    """Stands for a cache that refuses every move (its device is not the current
    one), or the launch of one."""
    def __init__(self, pages, where):
        super().__init__(pages)
        self.where = where

    def move(self, pairs, table=None, source=None, stream=None):
        if pairs or self.where == "device":
            raise RuntimeError(self.where)


@pytest.mark.parametrize("where", ["device", "launch"])
@pytest.mark.parametrize("most", [None, 1])
def test_compact_that_fails_leaves_the_pool(where, most):
    """Pages whose copy is refused stay their streams': the counts are as they were
    and the next pages given out are others."""
    import libpktito_amd as pk
    p = pk.PagePool(200)
    held = p.alloc(150)
    p.share([149, 149, 100])
    p.release([i for i in held if i not in (100, 130, 149, 3)])
    before = [p.holders(i) for i in range(200)]
    with pytest.raises(RuntimeError):
        p.compact(_Fails(200, where), None, most)
    assert [p.holders(i) for i in range(200)] == before and p.free_pages == 196
    assert p.alloc(5) == [0, 1, 2, 4, 5]


def test_compact_on_another_device_leaves_the_pool(monkeypatch):
    """The current device is another than the cache's: refused with nothing moved."""
    import torch
    import libpktito_amd as pk
    cache, _ = _wrapped(pk, torch)
    monkeypatch.setattr(pk, "_device", lambda: 1)
    p = pk.PagePool(8)
    p.release(p.alloc(5)[:3])
    with pytest.raises(pk.PkHipError) as e:
        p.compact(cache, _Device(torch.int32, 2, 4))
    assert e.value.code == pk.PK_HIP_EINVAL
    assert [p.holders(i) for i in range(8)] == [0, 0, 0, 1, 1, 0, 0, 0] and p.alloc(1) == [0]


def test_pool_restore():
    """A compaction undone: all of it or its last pairs, in any state of the other
    pages; refused, with nothing changed, where it is not undone so."""
    import libpktito_amd as pk
    l = pk.lib()
    r = random.Random(7)

    def restore(p, pairs):
        flat = (ctypes.c_int32 * max(1, 2 * len(pairs)))(*[i for pair in pairs for i in pair])
        return l.pk_hip_pool_restore(p.handle, flat, len(pairs))

    for pages in (1, 5, 64, 130):
        for _ in range(60):
            p = pk.PagePool(pages)
            held = p.alloc(r.randint(0, pages))
            p.share(r.choices(held, k=3) if held else [])
            for i in held:
                if r.random() < 0.5:
                    p.release([i] * p.holders(i))
            counts = lambda: [p.holders(i) for i in range(pages)]
            before, free = counts(), p.free_pages
            pairs = (ctypes.c_int32 * (2 * pages))()
            n = ctypes.c_uint32()
            assert l.pk_hip_pool_compact(p.handle, pairs, pages, ctypes.byref(n)) == 0
            moves = [(pairs[2 * i], pairs[2 * i + 1]) for i in range(n.value)]
            after = counts()
            if moves:
                f, t = moves[0]
                for bad in ([(f, f)], [(t, f)], [(f, pages)], [(pages, t)], [(-1, t)], moves + [(f, t)], moves[:1] * 2):
                    assert restore(p, bad) == pk.PK_HIP_EINVAL and counts() == after and p.free_pages == free
            assert restore(p, []) == pk.PK_HIP_OK and counts() == after
            assert restore(p, moves) == pk.PK_HIP_OK and counts() == before and p.free_pages == free
            if free:                            # the lowest free page is found again
                assert p.alloc(1) == [before.index(0)]
    p = pk.PagePool(4)
    p.release([p.alloc(3)[0]])
    pairs, n = (ctypes.c_int32 * 8)(), ctypes.c_uint32()
    l.pk_hip_pool_compact(p.handle, pairs, 4, ctypes.byref(n))
    assert n.value == 1 and p.alloc(1) == [pairs[0]]        # given out since
    assert restore(p, [(pairs[0], pairs[1])]) == pk.PK_HIP_EINVAL and p.free_pages == 1
    assert l.pk_hip_pool_restore(None, pairs, 1) == pk.PK_HIP_EINVAL
    assert l.pk_hip_pool_restore(p.handle, None, 1) == pk.PK_HIP_EINVAL


def test_move_takes_memory_for_its_pairs():
    """One page of the largest pool: the host memory that the checks take goes by
    the pairs, not by the pool (a child process with 256 MB to spare, no device)."""
    child = """
import ctypes, resource, sys
sys.path.insert(0, sys.argv[1])
import libpktito_amd as pk
l = pk.lib()
c = pk.Cache(4096, 1, 1 << 30, 1, 32)
pairs = (ctypes.c_int32 * 4)((1 << 30) - 1, 5, 7, 6)
used = int(open("/proc/self/statm").read().split()[0]) * resource.getpagesize()
resource.setrlimit(resource.RLIMIT_AS, (used + (256 << 20),) * 2)
for n in (0, 1, 2):
    e = l.pk_hip_cache_move_dev(ctypes.byref(c), ctypes.byref(c), pairs, n, None, 0, None)
    print(e, l.pk_hip_last_error().decode())
    assert e == pk.PK_HIP_ENODEV
"""
    r = subprocess.run([sys.executable, "-c", child, ROOT], env=os.environ | {"PKTITO_HIP_DISABLE": "1"},
                       capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stdout + r.stderr


def test_move_checks_many_pairs():
    """Pairs in any order, some thousand of them: what is refused is found wherever
    it is, and nothing else is."""
    import libpktito_amd as pk
    r = random.Random(8)
    n = 3000
    c = pk.Cache(4096, 1, 2 * n, 1, 32)
    ids = r.sample(range(2 * n), 2 * n)

    def move(pairs, table=None):
        flat = (ctypes.c_int32 * (2 * len(pairs)))(*[i for pair in pairs for i in pair])
        return pk.lib().pk_hip_cache_move_dev(ctypes.byref(c), ctypes.byref(c), flat, len(pairs), table, 16, None)

    good = list(zip(ids[:n], ids[n:]))
    for i, j in (r.sample(range(n), 2) for _ in range(20)):
        for bad, table in (((good[j][0], good[i][1]), None), ((good[i][1], good[j][1]), None),
                           ((good[j][0], good[j][0]), None), ((good[i][0], good[j][1]), 4096)):
            pairs = good[:j] + [bad] + good[j + 1:]
            assert move(pairs, table) == pk.PK_HIP_EINVAL, (i, j, bad)


def test_pairs_that_are_none_are_refused(monkeypatch):
    """Each of them two pages, not all of them together."""
    import torch
    import libpktito_amd as pk
    monkeypatch.setattr(pk, "_device", lambda: 0)
    cache, _ = _wrapped(pk, torch)
    for pairs in ([(1,), (2, 3, 4)], [(0, 1, 2, 3), ()], [(0,), (1,)], [(0, 1), (2,), (3, 4, 5)]):
        with pytest.raises(pk.PkHipError) as e:
            cache.move(pairs, stream=0)
        assert e.value.code == pk.PK_HIP_EINVAL and "pairs" in str(e.value)


def test_sizes_that_no_call_takes_are_refused_at_once():
    """Sizes that have no number of bytes, whatever memory is given with them."""
    import torch
    import libpktito_amd as pk
    big = _Device(torch.uint8, 1 << 40)
    for sizes in ((2, 8, 4, 48), (2, 8, 4, 0), (0, 8, 4, 64), (2, 0, 4, 64), (2, 8, 0, 64), (2, 8, 1025, 64)):
        with pytest.raises(pk.PkHipError) as e:
            pk.DeviceCache(big, *sizes)
        assert e.value.code == pk.PK_HIP_EINVAL


@pytest.mark.parametrize("rows", [0, 5])
def test_steps_without_streams(rows):
    """No streams: their table and lengths are empty, which torch gives no address,
    and there is nothing to do (or no device to do it on)."""
    import libpktito_amd as pk
    none = {} if rows else dict(k=None, v=None, o=None, q=None)
    calls = _calls(pk, B=0, table=None, len=None, rows=rows, max_T=0, **none)
    for e in ALL:
        assert calls[e]() in (pk.PK_HIP_OK, pk.PK_HIP_ENODEV), (e, pk.lib().pk_hip_last_error())
    calls = _calls(pk, B=0, table=None, len=None, row0=None, rows=rows, max_T=0, **none)
    for e in ALL:
        assert calls[e]() == pk.PK_HIP_EINVAL


@pytest.mark.parametrize("max_pages,T", [(1 << 24, 1), (1 << 24, 5), ((1 << 24) - 2, 5), (1 << 24, 0)])
def test_widest_tables(max_pages, T):
    """Every frame of the widest table may be attended without positions. The calls
    end at an output that is not aligned, which is looked at after the window."""
    import libpktito_amd as pk
    r = ctypes.byref
    c, st = pk.Cache(4096, 2, 8, 4, 64), pk.Streams(4096, 4096, 4096, 2, max_pages, 5, T)
    for left, right in ((pk.UNLIMITED, pk.UNLIMITED), (64 * max_pages, 0), (1 << 30, 3)):
        assert pk.lib().pk_hip_attention_cache_dev(4100, 512, 8192, 512, r(c), 1, r(st), 8, None, left, right, 4096, 1 << 40,
                                                   None) == pk.PK_HIP_EINVAL
        assert b"aligned" in pk.lib().pk_hip_last_error(), pk.lib().pk_hip_last_error()
@pytest.mark.parametrize("H,n", [
    (32768, (1 << 26) - 160),                   # 2^64 bytes of scores: none would be left
    (32768, (1 << 26) - 144),                   # and 2^38 more
    (65532, 0xffffffff), (4, 0xffffffff),       # the widest tables; the last one's scores would pass 2^48 bytes only
])
def test_workspaces_past_what_a_size_holds(H, n):
    """Position scores whose bytes pass what a size holds have no workspace, and a
    call of them is refused, not run in the one that the last bits give."""
    import libpktito_amd as pk
    rows, r = 1 << 21, ctypes.byref
    c = pk.Cache(4096, 2, 8, 4, 32)
    st = pk.Streams(4096, 4096, 4096, 1, 1 << 24, rows, 1)
    for center in {min(n - 1, (1 << 30) - 1), n - 1}:
        pos = pk.Positions(4096, 4096, 4096, n, center)
        args = (r(st), H, r(pos), pk.UNLIMITED, 0)
        assert pk.lib().pk_hip_attention_cache_workspace(r(c), *args) == 0
        assert pk.lib().pk_hip_attention_cache_dev(4096, H * 32, 8192, H * 32, r(c), 1, *args, 4096, 1 << 62,
                                                   None) == pk.PK_HIP_EINVAL
        assert b"workspace" in pk.lib().pk_hip_last_error()
    # the largest position table that 288 GB hold beside its queries is taken: 2^31 of its numbers
    st.rows, pos = 64, pk.Positions(4096, 4096, 4096, 1 << 24, (1 << 24) - 1)
    assert pk.lib().pk_hip_attention_cache_workspace(r(c), r(st), 4, r(pos), pk.UNLIMITED, 0) >= 64 * 4 * 4 << 24


def test_how_far_kept_values_are_off(layout):
    """Half a level's step of a scale that is up to 2^-7 over a sixth of the head's
    largest magnitude: a sixth of that and 2^-7 more, a twenty-fourth so up to two
    levels. Tops just over a bfloat16's six-fold come near it."""
    g = np.random.default_rng(9)
    most = 0.0
    for _ in range(3000):
        top = np.float32(6.0 * (1 + 2.0 ** -20)) if g.random() < 0.1 else np.float32(abs(g.standard_normal()) + 0.1)
        d = float(np.uint32(layout.t_scale(float(top)) << 16).view(np.float32))
        for x in (np.float32(v) for v in (g.uniform(-1, 1) * float(top), 5 * d, 1.25 * d, float(top))):
            if abs(x) > top:
                continue
            off = abs(layout.t_level(layout.t_code(float(x), d)) * d - float(x)) / float(top)
            assert off <= (1 + 2.0 ** -7) / (24 if abs(x) <= 2 * d else 6)
            most = max(most, off)
    assert most > 1 / 6
