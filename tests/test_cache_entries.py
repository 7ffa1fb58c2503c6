"""Which entry point the cache's Python attention calls: refusals name it."""
import os

import pytest

from test_window import Tensor


@pytest.fixture(scope="module")
def pk():
    import libpktito_amd as pk
    if not os.path.exists(pk.LIB_PATH):
        from libpktito_amd import build
        build.build()
    return pk


@pytest.mark.parametrize("sinks,entry", [(None, "attention_cache"), (0, "attention_cache"), (3, "attention_sinks")])
def test_refusals_name_the_entry_that_was_asked(pk, monkeypatch, sinks, entry):
    import torch
    monkeypatch.setattr(pk, "_device", lambda: 0)
    i = torch.int32
    streams = pk.CacheStreams(Tensor(i, 2, 4), Tensor(i, 2), Tensor(i, 3), 6, 3)
    cache = pk.DeviceCache(Tensor(torch.uint8, pk.cache_bytes(1, 4, 2, 64)), 1, 4, 2, 64)
    x = Tensor(torch.float32, 6, 128)
    more = {} if sinks is None else dict(sinks=sinks)
    with pytest.raises(pk.PkHipError) as e:
        cache.attention(x, 5, x, streams, 2, None, left=9, stream=0, **more)
    assert e.value.code == pk.PK_HIP_EINVAL and f": {entry}_dev: layer 5 of 1" in str(e.value)
    assert cache.attention_workspace(streams, 3, None, 9, **more) == 0
    assert pk.lib().pk_hip_last_error().decode().startswith(f"{entry}_workspace: ")
