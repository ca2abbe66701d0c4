"""decode_shared (decode attention over shared INT4 prefixes) against attention in
64 bits over the dequantised tokens.

Tolerance: max |out - ref| <= 2e-3 ||ref||_2 per row, the bound that every
attention test here holds, plus the output's own rounding. What it has to cover:
V rounded to f16 as it is dequantised (at most 2^-11 relative, with the ref
format's f32 scale rounded to f16 too at most 2^-10), P rounded to f16 (2^-11),
and scores off by K's rounding: each of 128 products by up to 2^-11 (2^-10) with
random signs, 2^-12.3 of sqrt(sum (q k)^2) sm_scale in the mean, about 3e-4 for
N(0, 1) data and 1e-3 with the outlier channels; errors of p that every token has
at random average out like the output itself. A row's values are 1 / 11.3 of its
norm, so 2e-3 of the norm is 2e-2 of a value: over ten times the sum of these.
A row of one token carries V's rounding alone: 2^-10 |v| < 1e-3 ||ref||."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def kv():
    from hetero_kvcache_optimizer_b200 import kvstore
    return kvstore


@pytest.fixture(scope="module")
def L():
    from hetero_kvcache_optimizer_b200 import _lib
    _lib.device_error(clear=True)
    return _lib


def randn(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")


def filled(kv, seed, lens, H, fmt, group, P, paged=False, k=None, extra=0):
    """A store with lens[b] random tokens per sequence (pages of a paged one
    shuffled, the rest of the pool random bytes) and its K, V in fp32."""
    B, T = len(lens), max(max(lens), 1)
    cap = -(-T // P) * P + extra * P
    src = kv.Int4KVStore(B, H, cap, fmt=fmt, group=group, page_tokens=P)
    src.pool.random_(0, 256, generator=torch.Generator(device="cuda").manual_seed(seed))
    if k is None:
        k = randn(seed + 1, B, H, T, 128)
        k[..., 3::41] *= 10
    v = randn(seed + 2, B, H, T, 128)
    store = src
    if paged:
        n = src.pool.shape[0]
        perm = torch.randperm(n + 3, generator=torch.Generator().manual_seed(seed))[:n].to(torch.int32)
        pool = torch.empty(n + 3, src.page_bytes, dtype=torch.uint8, device="cuda").random_(0, 256)
        store = kv.Int4KVStore.wrap(pool, perm.cuda().view(B * H, -1), torch.zeros(B, dtype=torch.int32, device="cuda"), H,
                                    fmt=fmt, group=group, page_tokens=P)
    for s in {id(src): src, id(store): store}.values():
        for b, m in enumerate(lens):  # tokens behind the length keep their random bytes
            if m:
                one = kv.Int4KVStore.wrap(s.pool, s.page_table[b * H:(b + 1) * H] if s.paged else
                                          torch.arange(b * H * s.max_pages, (b + 1) * H * s.max_pages, dtype=torch.int32, device="cuda").view(H, -1),
                                          s.lengths[b:b + 1], H, fmt=fmt, group=group, page_tokens=P)
                kv.quantize_pack_kv(k[b:b + 1, :, :m].to(F16), v[b:b + 1, :, :m].to(F16), one)
        s.set_lengths(torch.tensor(lens, dtype=torch.int32, device="cuda"))
    return store, kv.dequantize_pack(src, 0, 0, cap, dtype=F32), kv.dequantize_pack(src, 1, 0, cap, dtype=F32)


def reference(q, starts, parts, dense, scale):
    """parts: (k, v, lens) of the prefixes and of the body (or None); 64 bits."""
    B, Hq, D = q.shape
    pk, pv, pn = parts[0]
    H = pk.shape[1]
    G = Hq // H
    out = torch.zeros(B, Hq, D, dtype=torch.float64, device="cuda")
    for b in range(B):
        ks, vs = [], []
        g = next((i for i in range(len(pn)) if starts[i] <= b < starts[i + 1]), None)
        if g is not None:
            ks.append(pk[g, :, :pn[g]]), vs.append(pv[g, :, :pn[g]])
        if parts[1] is not None:
            k, v, n = parts[1]
            ks.append(k[b, :, :n[b]]), vs.append(v[b, :, :n[b]])
        if dense is not None:
            n = int(dense.lengths[b])
            ks.append(dense.k[b, :, :n]), vs.append(dense.v[b, :, :n])
        if sum(x.shape[1] for x in ks):
            k, v = torch.cat([x.double() for x in ks], 1), torch.cat([x.double() for x in vs], 1)
            p = torch.softmax(q[b].double().view(H, G, D) @ k.transpose(1, 2) * scale, -1)
            out[b] = (p @ v).view(Hq, D)
    return out


def check(out, ref):
    norm = ref.norm(dim=-1, keepdim=True)
    tol = 2e-3 * norm + ref.abs() * torch.finfo(out.dtype).eps / 2
    over = (out.double() - ref).abs() - tol
    assert bool((over <= 0).all()), f"worst row {((out.double() - ref).abs().amax(-1) / norm[..., 0]).max().item():.2e} of its norm"


def make_dense(kv, seed, B, H, cap, lens, dtype):
    if cap == 0:
        return None
    d = kv.DenseKV(B, H, cap, dtype=dtype, k=randn(seed, B, H, cap, 128).to(dtype), v=randn(seed + 1, B, H, cap, 128).to(dtype))
    d.lengths.copy_(torch.tensor(lens, dtype=torch.int32))
    d.len_hint = max(lens)
    return d


CASES = [
    # starts, prefix lens, body lens (or None), dense lens (or None), H, G
    ([0, 1], [1], None, None, 1, 1),
    ([0, 1], [128], None, None, 2, 4),
    ([0, 2], [129], None, [5, 1], 1, 8),
    ([0, 4], [1000], [100, 0, 1, 129], [96, 96, 0, 7], 4, 7),
    ([0, 5], [3000], None, [9] * 5, 2, 3),
    ([0, 8], [2500], [300] * 8, [64] * 8, 8, 4),
    ([0, 13], [700], None, [33] * 13, 2, 5),
    ([0, 33], [1300], [0] * 33, [17] * 33, 1, 4),
    ([0, 40], [900], None, [3] * 40, 2, 7),
    ([0, 3, 3, 4, 9], [0, 77, 383, 2049], [10, 0, 500, 3, 0, 0, 1, 2, 3], [1, 2, 0, 0, 5, 6, 7, 8, 9], 2, 4),
    ([1, 3, 6], [511, 640], None, [4] * 8, 2, 2),
]


@pytest.mark.parametrize("fmt,group,P,paged", [("fp16min", 32, 256, True), ("ref", 32, 128, False), ("ref", 64, 128, True),
                                               ("fp16min", 128, 384, False), ("fp16min", 64, 128, True), ("ref", 128, 256, True)])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_matches_reference(kv, L, case, fmt, group, P, paged):
    starts, plens, blens, dlens, H, G = CASES[case]
    B = max(starts[-1], len(dlens or []), len(blens or []))
    dtype = BF16 if (case + group) % 2 else F16
    prefix, pk, pv = filled(kv, 10 * case, plens, H, fmt, group, P, paged)
    body = filled(kv, 10 * case + 5, blens, H, fmt, group, P, paged) if blens else None
    dense = make_dense(kv, 7, B, H, max(dlens), dlens, dtype) if dlens else None
    q = randn(3, B, H * G, 128).to(dtype)
    ref = reference(q, starts, ((pk, pv, plens), (body[1], body[2], blens) if body else None), dense, 128 ** -0.5)
    shared = kv.SharedPrefix(prefix, starts)
    out = kv.decode_shared(q, shared, body[0] if body else None, dense, out_dtype=dtype)
    assert L.device_error() == 0
    check(out, ref)
    again = kv.decode_shared(q, shared, body[0] if body else None, dense, out_dtype=dtype)
    assert torch.equal(out, again)  # sums are taken in one order


def test_rows_of_every_width(kv, L):
    """1 to 300 rows per KV head: each product width, partly filled tiles, several row tiles."""
    prefix, pk, pv = filled(kv, 1, [1500], 1, "fp16min", 32, 256)
    for B, G in ((1, 1), (3, 5), (2, 8), (17, 1), (4, 8), (11, 3), (8, 8), (13, 5), (16, 8), (43, 3), (75, 4)):
        q = randn(B, B, G, 128).to(F16)
        out = kv.decode_shared(q, kv.SharedPrefix(prefix, [0, B]))
        check(out, reference(q, [0, B], ((pk, pv, [1500]), None), None, 128 ** -0.5))
    assert L.device_error() == 0


@pytest.mark.parametrize("B,G", [(2, 4), (8, 4), (16, 4), (32, 4)])
def test_maxima_that_keep_moving(kv, L, B, G):
    """Scores that grow along the prefix (every tile moves the max), that fall, and
    one far above the rest."""
    T = 128 * 9 + 5
    base = randn(1, 1, 1, 1, 128)
    ramp = torch.linspace(0, 6, T, device="cuda").view(1, 1, T, 1)
    for k in (base * ramp, base * ramp.flip(2), base * (torch.arange(T, device="cuda") == 777).view(1, 1, T, 1) * 8.0):
        k = k + 0.05 * randn(2, 1, 1, T, 128)
        prefix, pk, pv = filled(kv, 1, [T], 1, "fp16min", 32, 256, k=k)
        q = (base[:, 0] * 1.5 * (1 - 2.0 * (torch.arange(B * G, device="cuda") % 3 == 0)).view(B, G, 1) + 0.1 * randn(5, B, G, 128)).to(F16)
        out = kv.decode_shared(q, kv.SharedPrefix(prefix, [0, B]))
        # scores of up to 100: f16 K is off by 2^-11 of each product, the sum of |q k| sm_scale is <= 100 as well,
        # so p by up to 2 * 100 * 2^-11 / sqrt(128) (random signs, 3 sigma: x 3 / 1.7) = 1.5e-2 relative
        ref = reference(q, [0, B], ((pk, pv, [T]), None), None, 128 ** -0.5)
        err = (out.double() - ref).abs().amax(-1) / ref.norm(dim=-1)
        assert err.max().item() < 1.5e-2, err.max().item()
    assert L.device_error() == 0


def test_few_ctas_make_long_pieces(kv, L):
    """One to nine CTAs: many tiles and units per CTA (the ring and the barriers' phases go round)."""
    prefix, pk, pv = filled(kv, 1, [2000, 0, 1111], 2, "ref", 32, 128, True)
    starts = [0, 7, 9, 12]
    q = randn(3, 12, 8, 128).to(F16)
    ref = reference(q, starts, ((pk, pv, [2000, 0, 1111]), None), None, 128 ** -0.5)
    for ctas in (1, 2, 5, 9, 300):
        check(kv.decode_shared(q, kv.SharedPrefix(prefix, starts), ctas=ctas), ref)
    assert L.device_error() == 0


def test_strides_types_and_no_prefix(kv, L):
    prefix, pk, pv = filled(kv, 1, [300], 2, "ref", 32, 128)
    dense = make_dense(kv, 5, 3, 2, 50, [50, 3, 0], F16)
    for dtype in (F16, BF16):
        q = randn(3, 3, 9, 3 * 128).to(dtype)[:, :8, 128:256]  # rows 384 apart
        out = torch.zeros(3, 8, 2, 128, dtype=F32, device="cuda")[:, :, 1]
        got = kv.decode_shared(q, kv.SharedPrefix(prefix, [0, 2]), None, dense if dtype == F16 else None, out=out, sm_scale=0.05)
        assert got.data_ptr() == out.data_ptr()
        ref = reference(q, [0, 2], ((pk, pv, [300]), None), dense if dtype == F16 else None, 0.05)
        check(got, ref)
        assert bool((got[2] == 0).all())  # no prefix, nothing of its own
    four = kv.decode_shared(q[:, :, None], kv.SharedPrefix(prefix, [0, 2]))
    assert four.shape == (3, 8, 1, 128)
    assert L.device_error() == 0


def test_many_query_heads(kv, L):
    """More than 8 query heads per KV head: in groups beside a dense segment, at once without one."""
    prefix, pk, pv = filled(kv, 1, [400], 1, "fp16min", 32, 128)
    dense = make_dense(kv, 5, 2, 1, 20, [20, 11], F16)
    q = randn(3, 2, 20, 128).to(F16)
    for d in (dense, None):
        check(kv.decode_shared(q, kv.SharedPrefix(prefix, [0, 2]), None, d),
              reference(q, [0, 2], ((pk, pv, [400]), None), d, 128 ** -0.5))
    assert L.device_error() == 0


def test_missing_pages_count_as_hidden(kv, L):
    prefix, pk, pv = filled(kv, 1, [700], 1, "ref", 32, 128, True)
    q = randn(3, 4, 4, 128).to(F16)
    prefix.page_table[0, 2] = -1
    prefix.page_table[0, 4] = 1000
    out = kv.decode_shared(q, kv.SharedPrefix(prefix, [0, 4]))
    assert L.device_error() == L.DEVERR_BAD_PAGE
    keep = [t for t in range(700) if t // 128 not in (2, 4)]
    check(out, reference(q, [0, 4], ((pk[:, :, keep], pv[:, :, keep], [len(keep)]), None), None, 128 ** -0.5))
    prefix.page_table.fill_(-1)
    out = kv.decode_shared(q, kv.SharedPrefix(prefix, [0, 4]))
    assert L.device_error() == L.DEVERR_BAD_PAGE and bool((out == 0).all())


def test_graphs_streams_and_growing_prefix(kv, L):
    """Two graphs over one prefix replayed side by side, lengths that grow between replays."""
    prefix, pk, pv = filled(kv, 1, [900], 2, "fp16min", 32, 128, True, extra=0)
    shared = kv.SharedPrefix(prefix, [0, 6])
    qs = [randn(i, 6, 8, 128).to(BF16) for i in (1, 2)]
    dense = make_dense(kv, 5, 6, 2, 40, [40, 1, 2, 3, 4, 5], BF16)
    outs = [kv.decode_shared(q, shared, None, dense) for q in qs]
    graphs = []
    for q, o in zip(qs, outs):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            kv.decode_shared(q, shared, None, dense, out=o)
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in graphs]
    for n in (900, 1, 0, 513):
        prefix.lengths.fill_(n)
        refs = [reference(q, [0, 6], ((pk, pv, [n]), None), dense, 128 ** -0.5) for q in qs]
        torch.cuda.synchronize()
        for _ in range(5):
            for g, s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    g.replay()
        torch.cuda.synchronize()
        for o, r in zip(outs, refs):
            check(o, r)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    o = kv.decode_shared(qs[0], shared, None, dense, stream=s)
    s.synchronize()
    check(o, refs[0])
    assert L.device_error() == 0


def test_refusals(kv, L):
    prefix, _, _ = filled(kv, 1, [10, 20], 2, "ref", 32, 128)
    q = randn(3, 4, 8, 128).to(F16)
    for starts in ([0, 4], [0, 3, 2], [-1, 2, 4], [0, 1, 2, 3]):
        with pytest.raises(ValueError):
            kv.SharedPrefix(prefix, starts)
    sp = kv.SharedPrefix(prefix, [0, 2, 4])
    for bad in (dict(q=q[:3]), dict(q=q[0]), dict(q=q, dense=kv.DenseKV(3, 2, 8)), dict(q=q, store=kv.Int4KVStore(4, 1, 128)),
                dict(q=q, out=torch.empty(4, 8, 64, device="cuda"))):
        with pytest.raises(ValueError):
            kv.decode_shared(prefix=sp, **bad)
    with pytest.raises(RuntimeError):
        kv.decode_shared(q[:, :7], sp)
    with pytest.raises(L.HkvError):
        kv.decode_shared(q.float(), sp)
    with pytest.raises(L.HkvError):
        kv.decode_shared(q, sp, sm_scale=0.0)
