"""Lists from the host reach a page pool without a copy that waits (no GPU: the library's
calls are recorded)."""
import types

import pytest
import torch


def test_lists_travel_in_the_launch(monkeypatch):
    from hetero_kvcache_optimizer_b200 import _lib as L
    from hetero_kvcache_optimizer_b200 import kvstore as kv
    from hetero_kvcache_optimizer_b200.memory.page_pool import PagePool
    import contextlib
    seen = []

    def put(values, n, dst, stream):
        seen.append(list(values)[:n])
        return 0
    monkeypatch.setattr(L, "load", lambda: types.SimpleNamespace(hkv_put_i32=put))
    monkeypatch.setattr(kv, "launch_on", lambda *a: contextlib.nullcontext())
    monkeypatch.setattr(kv, "raw_stream", lambda d: 0)
    pool = PagePool.__new__(PagePool)
    pool.store = types.SimpleNamespace(batch=3, pool=torch.zeros(1))
    pool.refs = torch.zeros(1, dtype=torch.int32)
    for x in ([2, -1, 0], (2, -1, 0), torch.tensor([2, -1, 0]), torch.tensor([2, -1, 0], dtype=torch.int32)):
        out = pool._per_sequence(x, "parents")
        assert out.shape == (3,) and out.dtype == torch.int32
    assert seen == [[2, -1, 0]] * 4
    for bad in ([0, 1], [0, 1, 2, 3], [0, 0, 2**31], torch.zeros(3), torch.zeros(1, 3, dtype=torch.int32)):
        with pytest.raises(ValueError):
            pool._per_sequence(bad, "parents")
    assert len(seen) == 4


def test_refusals():
    from hetero_kvcache_optimizer_b200.csrc import build
    build.build()
    from hetero_kvcache_optimizer_b200 import _lib as L
    import ctypes
    v = (ctypes.c_int32 * 4)()
    lib = L.load()
    assert lib.hkv_put_i32(v, 0, None, None) == L.HKV_OK
    for args in ((v, -1, 1 << 20), (None, 4, 1 << 20), (v, 4, None), (v, 4, (1 << 20) + 2)):
        assert lib.hkv_put_i32(*args, None) == L.HKV_ERR_ARG
