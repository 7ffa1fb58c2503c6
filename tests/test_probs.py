"""Log probabilities without a device: refusals and sizes."""
import os

import pytest


@pytest.fixture(scope="module")
def pk():
    import libpktito_amd as pk
    if not os.path.exists(pk.LIB_PATH):
        from libpktito_amd import build
        build.build()
    return pk


X, T, L, E, P, Q, W = (0x10000000 * i for i in range(1, 8))


def call(pk, **change):
    a = dict(x=X, xs=1040, rows=10, cols=1025, tokens=T, m=2, lp=L, entropy=E, k=4, top=P, top_lp=Q, ws=W, ws_bytes=1 << 30)
    a |= change
    l = pk.lib()
    return l.pk_hip_logprobs_dev(*a.values(), None), l.pk_hip_last_error().decode()


@pytest.mark.parametrize("change", [
    dict(cols=0), dict(cols=(1 << 20) + 1, xs=1 << 21), dict(k=33), dict(cols=3, k=4), dict(rows=(1 << 21) + 1),
    dict(rows=1 << 21, cols=1 << 16, xs=1 << 16), dict(m=65536), dict(tokens=None), dict(lp=None), dict(m=0),
    dict(m=0, tokens=None), dict(m=0, lp=None), dict(top=None), dict(k=0), dict(k=0, top=None),
    dict(m=0, tokens=None, lp=None, entropy=None, k=0, top=None, top_lp=None), dict(x=None), dict(x=X + 2), dict(xs=1024),
    dict(tokens=T + 1), dict(lp=L + 2), dict(entropy=E + 3), dict(top=P + 1), dict(top_lp=Q + 2),
    dict(lp=X), dict(entropy=X + 4 * 1024), dict(top=T), dict(top_lp=T + 76), dict(top_lp=P), dict(entropy=L + 76),
    dict(top=X + 4 * 1040 * 9 + 4 * 1024), dict(cols=9000, xs=9000, ws=None), dict(cols=9000, xs=9000, ws_bytes=100),
    dict(cols=9000, xs=9000, ws=W + 8),
], ids=str)
def test_refusals(pk, change):
    code, why = call(pk, **change)
    assert code == pk.PK_HIP_EINVAL and why.startswith("logprobs_dev: "), (code, why)


@pytest.mark.parametrize("change", [
    dict(), dict(x=X + 4, xs=1025), dict(m=0, tokens=None, lp=None), dict(entropy=None), dict(k=0, top=None, top_lp=None),
    dict(top_lp=None), dict(rows=0, x=None), dict(rows=0, x=None, tokens=None, lp=None, entropy=None, top=None, top_lp=None), dict(rows=1, xs=0), dict(cols=8192, xs=8192, ws=None, ws_bytes=0),
    dict(cols=9000, xs=9000), dict(cols=5, xs=1040, x=X + 4100, entropy=None, k=5),
    dict(cols=5, xs=1040, entropy=X + 4 * 1040 * 9 + 20), dict(cols=32, k=32, xs=40),
], ids=str)
def test_calls_that_are_taken(pk, change):
    import torch
    if torch.cuda.is_available():
        pytest.skip("would run on addresses that are none")
    code, why = call(pk, **change)
    assert code == pk.PK_HIP_ENODEV, (code, why)


def test_workspaces(pk):
    need = pk.logprobs_workspace
    assert need(100, 8192, 20) == 0 and need(0, 1, 0) == 0
    assert need(10, 8193, 0) >= 10 * 2 * 20 and need(10, 8193, 32) > need(10, 8193, 1)
    assert need(10, 0, 0) == need(10, 5, 6) == need(10, (1 << 20) + 1, 1) == need(1 << 21, 1 << 16, 1) == 0
    assert need(10, 9000, 33) == 0
    for bad in ((-1, 5, 1), (1, 1 << 32, 1), (1, 5, -1)):
        with pytest.raises(pk.PkHipError):
            need(*bad)


def test_wrapper_refusals(pk, monkeypatch):
    import torch
    from test_window import Tensor
    device = [0]
    monkeypatch.setattr(pk, "_device", lambda: device[0])
    f, i = torch.float32, torch.int32
    fine = dict(x=Tensor(f, 6, 9), tokens=Tensor(i, 6, 2), lp=Tensor(f, 6, 2), entropy=Tensor(f, 6), top=Tensor(i, 6, 3),
                top_lp=Tensor(f, 6, 3), ws=Tensor(torch.uint8, 64))
    for change in (dict(x=Tensor(f, 54)), dict(x=Tensor(f, 6, 9, strides=(1, 6))), dict(x=Tensor(torch.float16, 6, 9)),
                   dict(x=torch.zeros(6, 9)), dict(tokens=Tensor(torch.int64, 6, 2)), dict(tokens=Tensor(i, 6)),
                   dict(tokens=Tensor(i, 5, 2)), dict(tokens=None), dict(lp=None), dict(lp=Tensor(f, 6, 3)),
                   dict(lp=Tensor(f, 6, 2, dense=False)), dict(lp=Tensor(f, 6, 2, device=1)), dict(entropy=Tensor(f, 6, 1)),
                   dict(top=Tensor(i, 6)), dict(top=None), dict(top=Tensor(torch.int64, 6, 3)), dict(top_lp=Tensor(f, 6, 2)),
                   dict(ws=Tensor(f, 64)), dict(ws=Tensor(torch.uint8, 64, dense=False)), dict(ws=torch.zeros(4, dtype=torch.uint8))):
        with pytest.raises(pk.PkHipError) as e:
            pk.logprobs_dev(**(fine | change), stream=0)
        assert e.value.code == pk.PK_HIP_EINVAL, change
    device[0] = 1
    with pytest.raises(pk.PkHipError) as e:
        pk.logprobs_dev(**fine, stream=0)
    assert "device" in str(e.value)
