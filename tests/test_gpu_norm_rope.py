"""norm_rope (norm of query and key heads + position rotation) against the
formula in 64 bits.

Tolerance per value: the last rounding is half a step of the type, eps / 2
relative. Before it, in fp32 (u = 2^-24): the sum of 128 squares carries at most
12 roundings (8 in a lane, 4 between lanes), halved by the root; rsqrt 4 u (2
units in the last place); mean, + eps and two products 4 u; the rotation 2
products and a sum: under 16 u of |a| + |b|, the pair's coordinates. f16 values
below 2^-14 have steps of 2^-24: half of one is added."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


@pytest.fixture(scope="module")
def kv():
    from hetero_kvcache_optimizer_b200 import kvstore
    return kvstore


@pytest.fixture(scope="module")
def L():
    from hetero_kvcache_optimizer_b200 import _lib
    _lib.device_error(clear=True)
    return _lib


def expected(x, pos, table, w, eps, adjacent):
    """(y, bound) in 64 bits of x [B, H, T, 128], pos [B, T]."""
    y = x.double()
    if w is not None:
        y = y / torch.sqrt(y.square().mean(-1, keepdim=True) + eps) * w.double()
    out, mag = y.clone(), y.abs()
    if table is not None:
        r = table.shape[1] // 2
        cs = table.double()[pos.long()][:, None]
        c, s = cs[..., :r], cs[..., r:]
        i0 = torch.arange(r, device=x.device) * (2 if adjacent else 1)
        i1 = i0 + (1 if adjacent else r)
        a, b = y[..., i0], y[..., i1]
        out[..., i0], out[..., i1] = a * c - b * s, b * c + a * s
        mag[..., i0] = mag[..., i1] = a.abs() + b.abs()
    tol = out.abs() * torch.finfo(x.dtype).eps / 2 * (1 + 2.0 ** -8) + mag * 16 * 2.0 ** -24
    return out, tol + (2.0 ** -25 if x.dtype == F16 else 0)


def check(got, want):
    out, tol = want
    over = (got.double() - out).abs() - tol
    assert bool((over <= 0).all()), f"{int((over > 0).sum())} values off, worst by {over.max().item():.3e}"


def inputs(seed, B, H, T, dtype, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(B, H, T, 128, generator=g, device="cuda") * scale).to(dtype)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("rot,adjacent", [(128, False), (64, False), (16, False), (2, False), (90, False), (126, False),
                                          (128, True), (64, True), (2, True), (90, True), (0, False)])
@pytest.mark.parametrize("B,Hq,Hkv,T", [(1, 1, 1, 1), (3, 7, 2, 5), (2, 32, 8, 131)])
def test_matches_formula(kv, L, dtype, rot, adjacent, B, Hq, Hkv, T):
    q, k = inputs(1, B, Hq, T, dtype, 3.0), inputs(2, B, Hkv, T, dtype, 0.1)
    table = kv.rope_table(4096, rot, base=1e6) if rot else None
    pos = torch.randint(0, 4096, (B, T), dtype=torch.int32, device="cuda")
    qw, kw = (1 + 0.3 * torch.randn(2, 128, device="cuda")).to(dtype)
    for w0, w1 in ((qw, kw), (None, None), (None, kw)):
        qo, ko = kv.norm_rope(q, k, pos, table, w0, w1, eps=1e-5, adjacent=adjacent)
        check(qo, expected(q, pos, table, w0, 1e-5, adjacent))
        check(ko, expected(k, pos, table, w1, 1e-5, adjacent))
    assert L.device_error() == 0


def test_many_rows_take_the_wide_split(kv):
    """More rows than 64 warps of every SM hold: eight heads a warp, odd head counts."""
    q, k = inputs(1, 2, 9, 1501, BF16), inputs(2, 2, 3, 1501, BF16)
    w = (1 + 0.3 * torch.randn(128, device="cuda")).float()
    pos = torch.arange(1501, device="cuda").expand(2, -1)
    for rot, adjacent in ((128, False), (44, False), (60, True)):
        table = kv.rope_table(1501, rot)
        qo, ko = kv.norm_rope(q, k, pos, table, w, w, adjacent=adjacent)
        check(qo, expected(q, pos, table, w, 1e-6, adjacent))
        check(ko, expected(k, pos, table, w, 1e-6, adjacent))


@pytest.mark.parametrize("T", [5, 1501])
@pytest.mark.parametrize("rot,adjacent", [(128, False), (96, False), (64, False), (44, False), (64, True)])
def test_tables_and_weights_that_are_slices(kv, rot, adjacent, T):
    q, k = inputs(3, 2, 9, T, F16), inputs(4, 2, 8, T, F16)
    wide = torch.zeros(T, rot + 9, device="cuda")
    w3 = 1 + 0.3 * torch.randn(3 * 128 + 1, device="cuda")
    pos = torch.arange(T, device="cuda").expand(2, -1)
    for off in (0, 1, 4):  # table rows of odd strides, from odd addresses
        table = wide[:, off:off + rot]
        table.copy_(kv.rope_table(T, rot))
        for w in (w3[:128], w3[1:129].to(BF16), w3.to(F16)[1:129]):
            qo, ko = kv.norm_rope(q, k, pos, table, w, w, adjacent=adjacent)
            check(qo, expected(q, pos, table, w, 1e-6, adjacent))
            check(ko, expected(k, pos, table, w, 1e-6, adjacent))


@pytest.mark.parametrize("rot,adjacent", [(128, False), (20, False), (128, True)])
def test_strided_in_place_and_unaligned(kv, rot, adjacent):
    B, T, Hq, Hkv = 2, 37, 6, 2
    table = kv.rope_table(64, rot)
    pos = torch.arange(T, device="cuda", dtype=torch.int32) + 3
    w = (1 + 0.3 * torch.randn(128, device="cuda")).to(F16)
    for shift in (0, 1):  # rows 16-byte aligned, or not
        flat = inputs(5, 1, 1, B * T * (Hq + 2 * Hkv) + 1, F16).reshape(-1)
        packed = flat[shift:shift + B * T * (Hq + 2 * Hkv) * 128].view(B, T, Hq + 2 * Hkv, 128)
        q, k = packed[:, :, :Hq].transpose(1, 2), packed[:, :, Hq:Hq + Hkv].transpose(1, 2)
        v0 = packed[:, :, Hq + Hkv:].clone()
        p2 = pos.expand(B, T)
        want = expected(q.clone(), p2, table, w, 1e-6, adjacent), expected(k.clone(), p2, table, None, 1e-6, adjacent)
        qo, ko = kv.norm_rope(q, k, pos, table, w, None, adjacent=adjacent, q_out=q, k_out=k)
        assert qo.data_ptr() == q.data_ptr()
        check(q, want[0])
        check(k, want[1])
        assert torch.equal(packed[:, :, Hq + Hkv:], v0)  # the values beside them are left alone


def test_single_tokens_and_one_side(kv):
    q, k = inputs(1, 5, 8, 1, BF16), inputs(2, 5, 2, 1, BF16)
    table = kv.rope_table(200000, 128)
    pos = torch.tensor([0, 1, 131071, 7, 199999], device="cuda")
    qo, ko = kv.norm_rope(q[:, :, 0], k[:, :, 0], pos, table)
    check(qo[:, :, None], expected(q, pos[:, None], table, None, 0, False))
    check(ko[:, :, None], expected(k, pos[:, None], table, None, 0, False))
    a, none = kv.norm_rope(q, None, pos[:, None], table)
    assert none is None and torch.equal(a[:, :, 0], qo)
    none, b = kv.norm_rope(None, k, pos[:, None], table)
    assert none is None and torch.equal(b[:, :, 0], ko)
    # a broadcast input (every head the same vector)
    one = q[:, :1].expand(5, 8, 1, 128)
    c, _ = kv.norm_rope(one, None, pos[:, None], table)
    assert torch.equal(c[:, 3], c[:, 0]) and torch.equal(c[:, 0], a[:, 0])


def test_padding_and_positions_behind_the_table(kv, L):
    q, k = inputs(1, 2, 4, 6, F16), inputs(2, 2, 1, 6, F16)
    table = kv.rope_table(100, 64)
    pos = torch.tensor([[0, 1, 2, 3, -1, -7], [5, 99, 4, -2, 98, 97]], device="cuda", dtype=torch.int32)
    qo, ko = torch.full_like(q, 7.0), torch.full_like(k, 7.0)
    L.device_error(clear=True)
    kv.norm_rope(q, k, pos, table, q_out=qo, k_out=ko)
    assert L.device_error() == 0
    pad = (pos < 0)[:, None, :, None]
    assert bool((qo.masked_select(pad) == 7).all()) and bool((ko.masked_select(pad) == 7).all())
    want, tol = expected(q, pos.clamp_min(0), table, None, 0, False)
    check(torch.where(pad, want.to(F16), qo), (want, tol))
    pos[1, 1] = 100
    qo.fill_(7.0)
    kv.norm_rope(q, k, pos, table, q_out=qo, k_out=ko)
    assert L.device_error() == L.DEVERR_BAD_POSITION
    assert bool((qo[1, :, 1] == 7).all()) and L.device_error() == 0


def test_infinities_stay_in_their_row(kv):
    q = inputs(1, 1, 2, 4, F16)
    q[0, 0, 1, 3] = float("inf")
    q[0, 0, 2, 100] = float("inf")
    q[0, 1, 3, 64] = float("nan")
    table = kv.rope_table(16, 64)
    pos = torch.arange(4, device="cuda")
    a, _ = kv.norm_rope(q, None, pos, table)
    y, _ = expected(q, pos[None], table, None, 0, False)
    assert torch.equal(torch.isfinite(a), torch.isfinite(y))  # dims that are not turned pass through
    assert a[0, 0, 2, 100] == float("inf")


def test_empty(kv):
    q, k = torch.empty(2, 4, 0, 128, dtype=F16, device="cuda"), torch.empty(2, 1, 0, 128, dtype=F16, device="cuda")
    qo, ko = kv.norm_rope(q, k, torch.empty(2, 0, dtype=torch.int32, device="cuda"), kv.rope_table(8))
    assert qo.shape == q.shape and ko.shape == k.shape


def test_refusals(kv):
    q, k, pos, table = inputs(1, 2, 4, 3, F16), inputs(2, 2, 2, 3, F16), torch.zeros(2, 3, dtype=torch.int32, device="cuda"), kv.rope_table(8)
    for bad in (dict(q=None, k=None), dict(k=k.bfloat16()), dict(k=k[:1]), dict(k=k[:, :, :2]), dict(table=table.half()),
                dict(positions=pos.float()), dict(positions=pos[:, :2]), dict(positions=None), dict(q=q[..., :64], k=None),
                dict(q_weight=torch.ones(64, device="cuda")), dict(q_out=q[:, :2]), dict(k=None, k_out=k),
                dict(q=q.transpose(2, 3).contiguous().transpose(2, 3), k=None)):
        args = {**dict(q=q, k=k, positions=pos, table=table), **bad}
        with pytest.raises((ValueError, TypeError)):
            kv.norm_rope(**args)
    with pytest.raises(TypeError):
        kv.norm_rope(q.float(), k.float(), pos, table)
    from hetero_kvcache_optimizer_b200 import _lib
    with pytest.raises(_lib.HkvError):  # heads written onto each other
        kv.norm_rope(q, None, pos, table, q_out=torch.empty(2, 1, 3, 128, dtype=F16, device="cuda").expand(2, 4, 3, 128))
    with pytest.raises(_lib.HkvError):
        kv.norm_rope(q, None, pos, table[:, :3])


def test_captured_and_on_another_stream(kv):
    q, k = inputs(1, 4, 8, 1, BF16), inputs(2, 4, 2, 1, BF16)
    table = kv.rope_table(64, 128)
    pos = torch.zeros(4, 1, dtype=torch.int32, device="cuda")
    qo, ko = torch.empty_like(q), torch.empty_like(k)
    kv.norm_rope(q, k, pos, table, q_out=qo, k_out=ko)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        kv.norm_rope(q, k, pos, table, q_out=qo, k_out=ko)
        pos += 1
    for step in range(3):
        q.copy_(inputs(10 + step, 4, 8, 1, BF16))
        g.replay()
        check(qo, expected(q, torch.full((4, 1), step, device="cuda"), table, None, 0, False))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    a, b = kv.norm_rope(q, k, pos, table, stream=s)
    s.synchronize()
    check(a, expected(q, pos, table, None, 0, False))
    check(b, expected(k, pos, table, None, 0, False))
