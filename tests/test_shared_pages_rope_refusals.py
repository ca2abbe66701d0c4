"""What norm_rope, the page operations and decode_shared refuse, without a GPU: every
bad argument is answered before anything is launched (the addresses are never read)."""
import ctypes

import pytest
import torch

FAKE = 1 << 20  # a 16-byte aligned address


@pytest.fixture(scope="module")
def L():
    from hetero_kvcache_optimizer_b200.csrc import build
    build.build()
    from hetero_kvcache_optimizer_b200 import _lib
    _lib.load()
    return _lib


def rows(L, data=FAKE, sb=4096, sh=128, st=1024, heads=8):
    return L.HkvRows(data, sb, sh, st, heads, 0)


def norm_rope(L, q="default", k=None, q_out="default", k_out=None, **kw):
    a = dict(dtype=1, B=2, T=3, D=128, qw=0, kw=0, wdt=0, eps=1e-6, pos=FAKE, bits=32, psb=3, pst=1, table=FAKE, ts=128,
             max_pos=64, rot=128, adjacent=0)
    a.update(kw)
    q, q_out = (rows(L) if x == "default" else x for x in (q, q_out))
    return L.load().hkv_norm_rope(q, k, q_out, k_out, a["dtype"], a["B"], a["T"], a["D"], a["qw"], a["kw"], a["wdt"], a["eps"],
                                  a["pos"], a["bits"], a["psb"], a["pst"], a["table"], a["ts"], a["max_pos"], a["rot"],
                                  a["adjacent"], None)


def test_norm_rope(L):
    assert norm_rope(L, T=0) == L.HKV_OK  # nothing to do, nothing launched
    for bad in (dict(q=None, q_out=None), dict(q_out=None), dict(k=rows(L)), dict(B=0), dict(T=-1), dict(dtype=2), dict(dtype=7),
                dict(rot=0), dict(rot=3), dict(rot=130), dict(max_pos=0), dict(ts=64), dict(pos=0), dict(bits=16),
                dict(eps=-1.0), dict(eps=float("nan")), dict(eps=float("inf")), dict(qw=FAKE, wdt=3), dict(table=0, rot=2),
                dict(q=rows(L, data=0)), dict(q=rows(L, heads=0)), dict(q_out=rows(L, heads=4)), dict(q_out=rows(L, sh=0)),
                dict(q_out=rows(L, st=0)), dict(q_out=rows(L, sb=0)), dict(q=rows(L, data=FAKE + 1))):
        assert norm_rope(L, **bad) == L.HKV_ERR_ARG, bad
    assert norm_rope(L, D=64) == L.HKV_ERR_UNSUPPORTED
    assert norm_rope(L, B=1 << 20, T=1 << 10) == L.HKV_ERR_UNSUPPORTED


def store(L, **kw):
    s = L.HkvInt4Store()
    s.pages, s.page_stride, s.format, s.group, s.page_tokens, s.max_pages = FAKE, 128 * 168, 0, 32, 128, 4
    s.page_table, s.lengths, s.len, s.num_pages = FAKE, FAKE, 512, 64
    for k, v in kw.items():
        setattr(s, k, v)
    return s


def test_pages(L):
    lib, R = L.load(), ctypes.byref
    ok = store(L)
    need = lib.hkv_pages_workspace_bytes(R(ok), 3, 2)
    assert need == 4 * (7 * 3 * 2 * 4 + 3 + 4 + 64)
    for bad in (dict(page_table=None), dict(lengths=None), dict(num_pages=0), dict(pages=None), dict(page_stride=100), dict(group=48)):
        s = store(L, **bad)
        assert lib.hkv_pages_workspace_bytes(R(s), 3, 2) == 0
        assert lib.hkv_pages_fork(R(s), 3, 2, FAKE, FAKE, FAKE, need, None) != L.HKV_OK
        assert lib.hkv_pages_reserve(R(s), 3, 2, FAKE, 1, None, FAKE, need, None) != L.HKV_OK
        assert lib.hkv_pages_compact(R(s), 3, 2, R(ok), FAKE, FAKE, need, None) != L.HKV_OK
    assert lib.hkv_pages_fork(R(ok), 3, 2, None, FAKE, FAKE, need, None) == L.HKV_ERR_ARG
    assert lib.hkv_pages_fork(R(ok), 3, 2, FAKE, None, FAKE, need, None) == L.HKV_ERR_ARG
    assert lib.hkv_pages_fork(R(ok), 3, 2, FAKE, FAKE, FAKE, need - 4, None) == L.HKV_ERR_CAPACITY
    assert lib.hkv_pages_fork(R(ok), 3, 2, FAKE, FAKE, None, need, None) == L.HKV_ERR_CAPACITY
    assert lib.hkv_pages_fork(R(ok), 0, 2, FAKE, FAKE, FAKE, need, None) == L.HKV_ERR_ARG
    assert lib.hkv_pages_reserve(R(ok), 3, 2, FAKE, -1, None, FAKE, need, None) == L.HKV_ERR_ARG
    assert lib.hkv_pages_reserve(R(ok), 3, 2, FAKE, 0, None, FAKE, need, None) == L.HKV_OK
    assert lib.hkv_pages_reserve(R(ok), 3, 2, FAKE, 513, None, FAKE, need, None) == L.HKV_ERR_CAPACITY
    far = dict(pages=1 << 30, page_table=1 << 29, lengths=1 << 28)
    for bad in (dict(), dict(far, format=1, page_stride=128 * 160), dict(far, group=64), dict(far, page_tokens=256, page_stride=256 * 168),
                dict(far, max_pages=3), dict(far, pages=FAKE + 128 * 168), dict(far, lengths=FAKE)):
        assert lib.hkv_pages_compact(R(ok), 3, 2, R(store(L, **bad)), FAKE, FAKE, need, None) == L.HKV_ERR_ARG, bad


def shared(L, starts=(0, 2, 4), lens=(100, 200), B=4, Hq=8, Hkv=2, D=128, dense=None, prefix=None, scale=0.1, dt=0, odt=2, ws=None):
    lib, R = L.load(), ctypes.byref
    pf = prefix or store(L)
    st, ln = (ctypes.c_int32 * len(starts))(*starts), (ctypes.c_int32 * len(lens))(*lens)
    d = R(dense) if dense is not None else None
    need = lib.hkv_decode_shared_workspace_bytes(R(pf), st, ln, len(starts) - 1, None, d, B, Hq, Hkv, D, 0)
    rc = lib.hkv_decode_shared(FAKE, dt, Hq * D, D, R(pf), st, ln, len(starts) - 1, None, d, B, Hq, Hkv, D, scale, 0,
                               FAKE if ws is None else ws, max(need, 1) - 1, FAKE, odt, Hq * D, D, None)
    return need, rc


def test_decode_shared(L):
    need, rc = shared(L)
    assert need > 262144 and rc == L.HKV_ERR_CAPACITY  # one byte short of the workspace
    for bad in (dict(starts=(0, 3, 2)), dict(starts=(-1, 2, 4)), dict(starts=(0, 2, 5)), dict(Hq=7), dict(B=0),
                dict(prefix=store(L, page_tokens=100)), dict(prefix=store(L, pages=None))):
        need, rc = shared(L, **bad)
        assert need == 0 and rc == L.HKV_ERR_ARG, bad
    for bad in (dict(scale=0.0), dict(scale=float("nan")), dict(dt=2), dict(odt=3)):
        assert shared(L, **bad)[1] == L.HKV_ERR_ARG, bad
    assert shared(L, D=64) == (0, L.HKV_ERR_UNSUPPORTED)
    n = 513
    assert shared(L, starts=tuple(range(n + 1)), lens=(1,) * n, B=n)[1] == L.HKV_ERR_UNSUPPORTED
    dense = L.HkvDenseKV()
    dense.k = dense.v = FAKE
    dense.dtype, dense.capacity, dense.stride_b, dense.stride_h, dense.stride_t, dense.len = 0, 8, 2048, 1024, 128, 8
    assert shared(L, dense=dense)[0] > 262144
    assert shared(L, Hq=32, dense=dense) == (0, L.HKV_ERR_UNSUPPORTED)  # 16 query heads per KV head beside a dense segment
    assert shared(L, Hq=32)[0] > 0


def test_python_layer_without_a_gpu(L):
    from hetero_kvcache_optimizer_b200 import kvstore as kv
    from hetero_kvcache_optimizer_b200.memory.page_pool import PagePool
    q = torch.zeros(2, 4, 3, 128, dtype=torch.float16)
    with pytest.raises(RuntimeError, match="CUDA"):
        kv.norm_rope(q, None, torch.zeros(2, 3, dtype=torch.int32), kv.rope_table(8, device="cpu"))
    with pytest.raises(TypeError):
        kv.norm_rope(q.float(), None)
    pool = torch.zeros(8, kv.page_bytes("ref", 32, 128), dtype=torch.uint8)
    lens = torch.zeros(2, dtype=torch.int32)
    table = torch.full((4, 2), -1, dtype=torch.int32)
    st = kv.Int4KVStore.wrap(pool, table, lens, 2, page_tokens=128)
    assert (st.batch, st.kv_heads, st.max_pages, st.capacity, st.num_pages, st.paged) == (2, 2, 2, 256, 8, True)
    s = st.struct(b0=1)
    assert s.page_table == table.data_ptr() + 2 * 2 * 4 and s.lengths == lens.data_ptr() + 4
    plain = kv.Int4KVStore.wrap(pool, None, lens, 2, page_tokens=128)
    assert plain.max_pages == 2 and not plain.paged
    for bad in ((pool[:, 1:], table, lens), (pool, table[:3], lens), (pool, table.long(), lens), (pool, table, lens.long()),
                (pool[:7], None, lens), (pool.float(), table, lens), (pool, table[:, :0], lens)):
        with pytest.raises(ValueError):
            kv.Int4KVStore.wrap(*bad, 2, page_tokens=128)
    with pytest.raises(RuntimeError, match="CUDA"):
        PagePool(st)
    sp = kv.SharedPrefix(st, [0, 2, 5])
    with pytest.raises(ValueError):
        sp.set_lengths([1])
    with pytest.raises(RuntimeError, match="CUDA"):
        kv.decode_shared(q[:, :, 0], sp)
    with pytest.raises(ValueError):
        kv.rope_table(0, device="cpu")
    t = kv.rope_table(200000, 128, base=1e6, device="cpu")
    i = 37
    ang = 199999.0 * 1e6 ** (-2.0 * i / 128)
    # the angle in 64 bits is off by 2e5 * 2^-53, the table entry by half a step of fp32
    assert abs(t[199999, i].item() - torch.cos(torch.tensor(ang, dtype=torch.float64)).item()) < 2.0 ** -24
    assert abs(t[199999, 64 + i].item() - torch.sin(torch.tensor(ang, dtype=torch.float64)).item()) < 2.0 ** -24
