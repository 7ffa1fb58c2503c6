"""The plan of a step without a device: what it refuses, and its model on a life
that is followed by hand."""
import ctypes
import os

import numpy as np
import pytest

import plan_ref as pr


@pytest.fixture(scope="module")
def pk():
    import libpktito_amd as pk
    if not os.path.exists(pk.LIB_PATH):
        from libpktito_amd import build
        build.build()
    return pk


def call(pk, **change):
    a = dict(table=4096, len=8192, row0=12288, state=16384, pool=20480, slot=24576, told=28672, B=3, max_pages=5, rows=10,
             max_T=4, pages=7, add=32768, fresh=36864, left=9, sinks=2) | change
    p = pk.Plan(*(a[n] for n in ("table", "len", "row0", "state", "pool", "slot", "told", "B", "max_pages", "rows", "max_T",
                                 "pages")))
    l = pk.lib()
    code = l.pk_hip_cache_plan_dev(None if change.get("none") else ctypes.byref(p), a["add"], a["fresh"], a["left"],
                                   a["sinks"], None)
    return code, l.pk_hip_last_error().decode()


@pytest.mark.parametrize("change", [
    dict(none=True), dict(table=None), dict(len=None), dict(row0=None), dict(state=None), dict(pool=None), dict(told=None),
    dict(add=None), dict(add=32770), dict(fresh=1), dict(table=4097), dict(len=2), dict(row0=3), dict(state=5), dict(pool=6),
    dict(slot=7), dict(told=9), dict(max_pages=0), dict(max_pages=(1 << 24) + 1), dict(pages=0), dict(pages=(1 << 24) + 1),
    dict(B=65536), dict(rows=(1 << 21) + 1), dict(max_T=11),
    dict(B=256, max_pages=1 << 24), dict(B=129, max_pages=1 << 24), dict(B=257, max_pages=16711935),
], ids=str)
def test_refusals(pk, change):
    code, why = call(pk, **change)
    assert code == pk.PK_HIP_EINVAL and why.startswith("cache_plan_dev: "), (code, why)


@pytest.mark.parametrize("change", [
    dict(), dict(fresh=None), dict(slot=None), dict(left=0xffffffff, sinks=0xffffffff), dict(rows=0, max_T=0),
    dict(B=0, table=None, len=None, state=None, add=None), dict(B=128, max_pages=1 << 24),
], ids=str)
def test_calls_that_are_taken(pk, change):
    import torch
    if torch.cuda.is_available():
        pytest.skip("would run on addresses that are none")
    code, why = call(pk, **change)
    assert code == pk.PK_HIP_ENODEV, (code, why)


def test_wrapper_refusals(pk, monkeypatch):
    import torch
    from test_window import Tensor
    i = torch.int32
    device = [0]
    monkeypatch.setattr(pk, "_device", lambda: device[0])
    real = torch.zeros

    def zeros(n, dtype=None, device=None):
        return Tensor(dtype, n)
    monkeypatch.setattr(torch, "zeros", zeros)
    fine = dict(table=Tensor(i, 3, 5), state=Tensor(i, 3, 2), pool=Tensor(i, 9), rows=10, max_T=4, slot=Tensor(i, 10))
    plan = pk.CachePlan(**fine)
    assert (plan.st.B, plan.st.max_pages, plan.st.pages, plan.st.rows, plan.st.max_T) == (3, 5, 7, 10, 4)
    for change in (dict(table=Tensor(i, 3)), dict(table=Tensor(torch.int64, 3, 5)), dict(table=Tensor(i, 3, 5, dense=False)),
                   dict(table=real(3, 5, dtype=i)), dict(state=Tensor(i, 2, 2)), dict(state=Tensor(i, 3, 2, device=1)),
                   dict(pool=Tensor(i, 2)), dict(pool=Tensor(i, 3, 3)), dict(slot=Tensor(i, 9)), dict(slot=Tensor(torch.int64, 10)),
                   dict(rows=1 << 32), dict(max_T=-1)):
        with pytest.raises(pk.PkHipError) as e:
            pk.CachePlan(**(fine | change))
        assert e.value.code == pk.PK_HIP_EINVAL, change
    for args in ((Tensor(i, 2),), (Tensor(torch.int64, 3),), (real(3, dtype=i),), (Tensor(i, 3, device=1),),
                 (Tensor(i, 3, dense=False),), (Tensor(i, 3), Tensor(i, 4)), (Tensor(i, 3), None, -1),
                 (Tensor(i, 3), None, 1 << 32), (Tensor(i, 3), None, None, -1)):
        with pytest.raises(pk.PkHipError) as e:
            plan.step(*args, stream=0)
        assert e.value.code == pk.PK_HIP_EINVAL, args
    device[0] = 1
    with pytest.raises(pk.PkHipError):
        plan.step(Tensor(i, 3), stream=0)


def test_model_by_hand():
    """Two streams over four pages: taken in order, given back behind the window but the sinks' page, queued behind the
    free ones; a full pool leaves holes; a stream that begins anew gives all back first."""
    p = pr.Plan(4, 2, 8, 300, 200)
    p.step([100, 1], left=64, sinks=3)
    assert p.table[0, :2].tolist() == [0, 1] and p.table[1, 0] == 2 and p.told == [101, 0, 0, 1]
    assert p.slot[99] == 64 + 35 and p.slot[100] == 128 and p.slot[101] == -1
    p.step([64, 0], left=64, sinks=3)            # frame 100 on: frames 36 on are in reach
    assert p.table[0, :3].tolist() == [0, 1, 3] and p.told == [64, 0, 0, 0]
    p.step([64, 64], left=36, sinks=3)           # frame 164: 128 on in reach, column 1 given back and taken at once
    assert p.table[0, :4].tolist() == [0, -1, 3, 1] and p.table[1, :2].tolist() == [2, -1] and p.told == [128, 0, 1, 0]
    p.step([0, 5], [0, 1], left=None)
    assert p.table[1, :2].tolist() == [2, -1] and p.len.tolist() == [228, 0] and p.told == [5, 0, 0, 0]
    p.step([500, -3])
    assert p.told == [200, 300, 3, 0] and p.state[0, 0] == 428
    p.step([500, 0])
    assert p.told == [84, 416, 1, 0] and p.state[0, 0] == 512
