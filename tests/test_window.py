"""Attention with a window over whole segments without a device: what it refuses,
before anything is opened, and its 64-bit model."""
import ctypes
import os

import numpy as np
import pytest

import window_ref as wr


@pytest.fixture(scope="module")
def pk():
    import libpktito_amd as pk
    if not os.path.exists(pk.LIB_PATH):
        from libpktito_amd import build
        build.build()
    return pk


A, B_, C, D, E, F = (0x1000000 * i for i in range(1, 7))


def call(pk, **change):
    """The entry's answer to a call that is fine but for `change` (addresses that nothing reads before a refusal)."""
    a = dict(o=A, os=256, q=B_, qs=256, k=C, ks=128, v=D, vs=128, row0=E, B=2, rows=10, max_T=6, H=4, G=2, dk=64, p=None,
             u=F, w=F + 4096, n=9, center=5, left=3, right=1, sinks=2) | change
    sg = pk.SegmentRows(a["row0"], a["B"], a["rows"], a["max_T"])
    pos = None if a["p"] is None else ctypes.byref(pk.Positions(a["p"], a["u"], a["w"], a["n"], a["center"]))
    l = pk.lib()
    code = l.pk_hip_attention_window_dev(a["o"], a["os"], a["q"], a["qs"], a["k"], a["ks"], a["v"], a["vs"],
                                         None if change.get("none") else ctypes.byref(sg), a["H"], a["G"], a["dk"], pos,
                                         a["left"], a["right"], a["sinks"], None)
    return code, l.pk_hip_last_error().decode()


@pytest.mark.parametrize("change", [
    dict(none=True), dict(row0=None), dict(B=65536), dict(rows=(1 << 21) + 1), dict(max_T=11),
    dict(dk=16), dict(dk=48), dict(dk=160), dict(dk=0), dict(H=0), dict(H=3), dict(H=65536), dict(G=0), dict(G=1025, H=1025),
    dict(B=60000, rows=1 << 20, max_T=1 << 20),
    dict(o=None), dict(q=None), dict(k=None), dict(v=None), dict(o=A + 4), dict(q=B_ + 8), dict(k=C + 4), dict(v=D + 12),
    dict(os=255), dict(qs=257), dict(ks=126), dict(vs=127), dict(os=252), dict(ks=124), dict(ks=(1 << 25) + 4),
    dict(vs=1 << 26),
    dict(p=F + 8192, u=None), dict(p=F + 8192, w=None), dict(p=F + 8196), dict(p=F + 8192, center=9), dict(p=F + 8192, n=0),
    dict(o=B_, os=260), dict(o=B_ + 1024), dict(o=C), dict(o=D + 4 * 128 * 9), dict(k=A + 4 * 256 * 9),
    dict(os=512, qs=512, q=A + 4 * 252), dict(os=512, ks=512, k=A + 4 * 388), dict(os=508, qs=508, q=A + 4 * 256),
    dict(p=A - 4 * 256 * 9 + 16), dict(p=F + 8192, u=A), dict(p=F + 8192, w=A + 16),
], ids=str)
def test_refusals(pk, change):
    code, why = call(pk, **change)
    assert code == pk.PK_HIP_EINVAL and why.startswith("attention_window_dev: "), (code, why)


@pytest.mark.parametrize("change", [
    dict(), dict(o=B_), dict(p=F + 8192), dict(p=F + 8192, left=0xffffffff, right=0xffffffff, sinks=0xffffffff),
    dict(rows=1, max_T=1, os=0, qs=0, ks=0, vs=0), dict(k=B_, ks=256), dict(k=C, v=C), dict(rows=0, max_T=0, o=None, q=None),
    dict(os=512, qs=512, ks=512, vs=512, q=A, k=A + 4 * 256, v=A + 4 * 384), dict(os=512, qs=512, q=A + 4 * 256),
    dict(os=512, qs=512, q=A - 4 * 256), dict(k=A + 4 * 256 * 10, ks=256, os=256), dict(v=A - 4 * (128 * 9 + 128)),
], ids=str)
def test_calls_that_are_taken(pk, change, monkeypatch):
    """Without a device these get as far as opening it."""
    import torch
    if torch.cuda.is_available():
        pytest.skip("would run on addresses that are none")
    code, why = call(pk, **change)
    assert code == pk.PK_HIP_ENODEV, (code, why)


class Tensor:
    """What a wrapper looks at of a device tensor."""

    def __init__(self, dtype, *shape, device=0, strides=None, dense=True):
        self.dtype, self.shape, self.device, self.dense = dtype, shape, f"cuda:{device}", dense
        self.is_cuda, self.index = True, device
        self.strides = strides or tuple(int(np.prod(shape[i + 1:])) for i in range(len(shape)))

    def get_device(self):
        return self.index

    def dim(self):
        return len(self.shape)

    def numel(self):
        return int(np.prod(self.shape))

    def is_contiguous(self):
        return self.dense

    def stride(self, i=None):
        return self.strides if i is None else self.strides[i]

    def data_ptr(self):
        return 16


def test_wrapper_refusals(pk, monkeypatch):
    import torch
    monkeypatch.setattr(pk, "_device", lambda: 0)
    f, i = torch.float32, torch.int32

    def refused(**change):
        x = lambda n, w, name: change.get(name, Tensor(f, n, w))
        with pytest.raises(pk.PkHipError) as e:
            sg = pk.Segments(change.get("row0", Tensor(i, 3)), change.get("rows", 10), change.get("max_T", 5))
            pk.attention_window_dev(x(10, 128, "o"), x(10, 128, "q"), x(10, 64, "k"), x(10, 64, "v"), sg,
                                    change.get("H", 4), change.get("dk", 32), change.get("positions"),
                                    change.get("left"), change.get("right"), change.get("sinks", 0), 0)
        assert e.value.code == pk.PK_HIP_EINVAL
        return str(e.value)

    assert "row0" in refused(row0=torch.zeros(3, dtype=i))
    assert "row0" in refused(row0=Tensor(torch.int64, 3))
    assert "row0" in refused(row0=Tensor(i, 3, dense=False))
    assert "row0" in refused(row0=Tensor(i, 3, 1))
    for name in "oqkv":
        w = 128 if name in "oq" else 64
        assert name in refused(**{name: Tensor(torch.float16, 10, w)})
        assert name in refused(**{name: Tensor(f, 10, w, device=1)})
        assert name in refused(**{name: Tensor(f, 9, w)})
        assert name in refused(**{name: Tensor(f, 10, w, strides=(1, 10))})
        assert name in refused(**{name: torch.zeros(10, w)})
    assert "k" in refused(k=Tensor(f, 10, 65))
    assert "device" in refused(row0=Tensor(i, 3, device=1))
    for name in ("left", "right", "sinks", "rows", "max_T", "H"):
        assert name in refused(**{name: 1 << 32}) and name in refused(**{name: -1})
    p, b = Tensor(f, 9, 128), Tensor(f, 128)
    assert "positions" in refused(positions=(Tensor(f, 9, 127), 5, b, b))
    assert "p:" in refused(positions=(Tensor(torch.float16, 9, 128), 5, b, b))
    assert "bias_u" in refused(positions=(p, 5, Tensor(f, 128, device=1), b))
    assert "positions" in refused(positions=(p, 5, b, Tensor(f, 64)))
    assert "center" in refused(positions=(p, 9, b, b))


def test_model_of_a_window():
    """The 64-bit model on a case whose answer is known: equal scores, so means of the attended values."""
    T, dk = 9, 32
    v = np.arange(T, dtype=np.float64)[:, None] * np.ones((1, dk))
    out, _ = wr.attend(np.zeros((T, dk)), 0, np.arange(T), np.ones((T, dk)), v, 1, dk, None, 2, 1, 1)
    for t in range(T):
        seen = [j for j in range(T) if j <= t + 1 and (j >= t - 2 or j < 1)]
        assert np.allclose(out[t], np.mean(seen))
