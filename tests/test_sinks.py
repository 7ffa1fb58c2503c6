"""The cache's attention with sinks without a device: what it refuses, its sizes,
and the pages that hold sinks before a window."""
import ctypes
import os

import pytest

from test_cache import layout  # noqa: F401


@pytest.fixture(scope="module")
def pk():
    import libpktito_amd as pk
    if not os.path.exists(pk.LIB_PATH):
        from libpktito_amd import build
        build.build()
    return pk


def call(pk, entry, **change):
    a = dict(o=4096, os=512, q=8192, qs=512, layer=1, H=4, left=9, right=2, sinks=5, ws=1 << 20, ws_bytes=1 << 30,
             pages=5, max_pages=8, B=2, rows=6, max_T=3, dk=128, heads=2) | change
    c = pk.Cache(16, 2, a["pages"], a["heads"], a["dk"])
    st = pk.Streams(16, 16, 16, a["B"], a["max_pages"], a["rows"], a["max_T"])
    pos = pk.Positions(16, 16, 16, a.get("n", 40), 12) if "n" in a else None
    r = lambda x: None if x is None else ctypes.byref(x)
    l = pk.lib()
    args = (r(st), a["H"], r(pos), a["left"], a["right"])
    if entry == "need":
        return l.pk_hip_attention_sinks_workspace(r(c), *args, a["sinks"])
    if entry == "need without":
        return l.pk_hip_attention_cache_workspace(r(c), *args)
    code = l.pk_hip_attention_sinks_dev(a["o"], a["os"], a["q"], a["qs"], r(c), a["layer"], *args, a["sinks"], a["ws"],
                                        a["ws_bytes"], None)
    return code, l.pk_hip_last_error().decode()


@pytest.mark.parametrize("change", [
    dict(o=None), dict(q=4), dict(os=510), dict(layer=2), dict(H=3), dict(H=0), dict(dk=48), dict(pages=0), dict(max_pages=0),
    dict(rows=2), dict(n=12), dict(q=4096, qs=516), dict(n=40, rows=1 << 21, B=9, max_T=3, ws_bytes=100),
    dict(B=65535, rows=1 << 21, max_T=1 << 21),
], ids=str)
def test_refusals(pk, change):
    code, why = call(pk, "", **change)
    assert code == pk.PK_HIP_EINVAL and why.startswith("attention_sinks_dev: "), (code, why)


@pytest.mark.parametrize("change", [dict(), dict(n=40), dict(sinks=0), dict(sinks=0xffffffff), dict(left=0xffffffff)], ids=str)
def test_calls_that_are_taken(pk, change):
    import torch
    if torch.cuda.is_available():
        pytest.skip("would run on addresses that are none")
    code, why = call(pk, "", **change)
    assert code == pk.PK_HIP_ENODEV, (code, why)


def test_workspaces(pk):
    """Without sinks, or with a window that nothing is behind, the workspace is that of the attention without; sinks of many
    pages may make it share a tile's pages among workgroups."""
    for n in ({}, dict(n=40)):
        assert call(pk, "need", sinks=0, **n) == call(pk, "need without", **n)
    far = dict(left=0xffffffff, max_pages=4000, B=1, rows=1, max_T=1)
    assert call(pk, "need", sinks=64 * 300, **far) == call(pk, "need without", **far) > 0
    wide = dict(B=1, rows=1, max_T=1, max_pages=4000)
    assert call(pk, "need", sinks=0, **wide) == call(pk, "need without", **wide) == 0
    assert call(pk, "need", sinks=64 * 300, **wide) > 0


def test_wrapper_refuses_sinks_past_32_bits(pk, monkeypatch):
    import torch
    from test_window import Tensor
    monkeypatch.setattr(pk, "_device", lambda: 0)
    i = torch.int32
    st = pk.CacheStreams(Tensor(i, 2, 4), Tensor(i, 2), Tensor(i, 3), 6, 3)
    cache = pk.DeviceCache(Tensor(torch.uint8, pk.cache_bytes(1, 4, 2, 64)), 1, 4, 2, 64)
    x = Tensor(torch.float32, 6, 128)
    for bad in (-1, 1 << 32):
        with pytest.raises(pk.PkHipError) as e:
            cache.attention(x, 0, x, st, 2, None, sinks=bad, stream=0)
        assert "sinks" in str(e.value)
        with pytest.raises(pk.PkHipError):
            cache.attention_workspace(st, 2, None, sinks=bad)


def test_pages_before_a_window(layout):  # noqa: F811
    """The first pages that hold a sink that some row attends, and that the window does not begin in or before."""
    import itertools
    for sinks, p0, j1 in itertools.product((0, 1, 63, 64, 65, 128, 1000), (0, 1, 2, 5), (-1, 0, 62, 63, 64, 300)):
        held = {j // 64 for j in range(min(sinks, j1 + 1)) if j // 64 < p0}
        assert layout.t_far_pages(sinks, p0, j1) == len(held), (sinks, p0, j1)
