"""decode_shared by output type: f16 and f32 outputs from exact codes at every number of
rows, bf16 outputs through the wide products (more than 16 rows), whose edges are looked at
here in that type. Tolerances of the wide form as in test_gpu_shared.py (2e-3 of a row's
norm) plus half a step of bf16."""
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


def prefix_of(kv, k, v, lens, fmt="fp16min", group=32, P=128):
    """Prefixes of the first lens[i] tokens of k, v [N, H, T, 128], and both as dequantised."""
    N, H, T, _ = k.shape
    st = kv.Int4KVStore(N, H, T, fmt=fmt, group=group, page_tokens=P)
    st.pool.random_(0, 256, generator=torch.Generator(device="cuda").manual_seed(1))
    kv.quantize_pack_kv(k.to(F16), v.to(F16), st)
    st.set_lengths(torch.tensor(lens, dtype=torch.int32, device="cuda"))
    return st, kv.dequantize_pack(st, 0, 0, T, dtype=F32), kv.dequantize_pack(st, 1, 0, T, dtype=F32)


def reference(q, starts, k, v, lens, scale=128 ** -0.5):
    B, Hq, D = q.shape
    H = k.shape[1]
    out = torch.zeros(B, Hq, D, dtype=torch.float64, device="cuda")
    for g in range(len(lens)):
        if lens[g]:
            a, b = starts[g], starts[g + 1]
            x = q[a:b].double().view(b - a, H, Hq // H, D)
            p = torch.softmax(torch.einsum("bhgd,htd->bhgt", x, k[g, :, :lens[g]].double()) * scale, -1)
            out[a:b] = torch.einsum("bhgt,htd->bhgd", p, v[g, :, :lens[g]].double()).reshape(b - a, Hq, D)
    return out


def check(out, ref, part=2e-3):
    tol = part * ref.norm(dim=-1, keepdim=True) + ref.abs() * torch.finfo(out.dtype).eps / 2
    over = (out.double() - ref).abs() - tol
    assert bool((over <= 0).all()), over.max().item()


@pytest.mark.parametrize("rows", [3, 16, 17, 40, 100, 300])
@pytest.mark.parametrize("dtype", [F16, F32])
def test_codes_are_exact_at_every_width(kv, L, rows, dtype):
    """ref, group 32, N(0, 1): the only errors are the fp32 sums of (1024 + n) q, a step of
    2^-10 at most for each of 8 products a score, times a scale below 0.4 and 128^-0.5: below
    2.8e-4 of a weight if all went one way, random over tokens like the output itself, so
    below that part of the output's norm; and P times scale in two f16, 2^-22."""
    T = 1000
    st, k, v = prefix_of(kv, randn(1, 1, 2, T, 128), randn(2, 1, 2, T, 128), [T], fmt="ref")
    q = randn(rows, rows, 2, 128).to(F16)
    out = kv.decode_shared(q, kv.SharedPrefix(st, [0, rows]), out_dtype=dtype).double()
    ref = reference(q, [0, rows], k, v, [T])
    err = ((out - ref).abs() - ref.abs() * (torch.finfo(dtype).eps / 2)).clamp_min(0)  # beyond the output's own rounding
    assert (err.norm(dim=-1) / ref.norm(dim=-1)).max().item() < 2.8e-4
    assert L.device_error() == 0


@pytest.mark.parametrize("fmt,group", [("fp16min", 32), ("fp16min", 128), ("ref", 64)])
def test_wide_products_of_every_width(kv, L, fmt, group):
    k, v = randn(1, 1, 1, 1500, 128), randn(2, 1, 1, 1500, 128)
    k[..., 3::41] *= 10
    st, k, v = prefix_of(kv, k, v, [1500], fmt, group)
    for B, G in ((17, 1), (4, 8), (11, 3), (8, 8), (13, 5), (16, 8), (43, 3), (75, 4)):
        q = randn(B, B, G, 128).to(BF16)
        out = kv.decode_shared(q, kv.SharedPrefix(st, [0, B]), out_dtype=BF16)
        check(out, reference(q, [0, B], k, v, [1500]))
        assert torch.equal(out, kv.decode_shared(q, kv.SharedPrefix(st, [0, B]), out_dtype=BF16))
    assert L.device_error() == 0


@pytest.mark.parametrize("rows", [32, 64, 128])
def test_wide_maxima_that_keep_moving(kv, L, rows):
    """Scores of up to 100 along the prefix: f16 K is off by 2^-11 of each product, the sum of
    |q k| sm_scale is <= 100 as well, so p by up to 2 * 100 * 2^-11 / sqrt(128) (random signs,
    3 sigma: x 3 / 1.7) = 1.5e-2 relative."""
    T = 128 * 9 + 5
    base = randn(1, 1, 1, 1, 128)
    ramp = torch.linspace(0, 6, T, device="cuda").view(1, 1, T, 1)
    for k in (base * ramp, base * ramp.flip(2), base * (torch.arange(T, device="cuda") == 777).view(1, 1, T, 1) * 8.0):
        st, kd, vd = prefix_of(kv, k + 0.05 * randn(2, 1, 1, T, 128), randn(3, 1, 1, T, 128), [T])
        sign = 1 - 2.0 * (torch.arange(rows, device="cuda") % 3 == 0)
        q = (base[:, 0] * 1.5 * sign.view(rows, 1, 1) + 0.1 * randn(5, rows, 1, 128)).to(F16)
        out = kv.decode_shared(q, kv.SharedPrefix(st, [0, rows]), out_dtype=BF16)
        check(out, reference(q, [0, rows], kd, vd, [T]), 1.5e-2)
    assert L.device_error() == 0


def test_wide_few_ctas_ragged_groups_and_missing_pages(kv, L):
    lens, starts = [2000, 0, 1111], [0, 7, 9, 12]
    st, k, v = prefix_of(kv, randn(1, 3, 2, 2000, 128), randn(2, 3, 2, 2000, 128), lens, "ref")
    q = randn(3, 12, 16, 128).to(F16)
    ref = reference(q, starts, k, v, lens)
    for ctas in (1, 2, 5, 9, 300):
        check(kv.decode_shared(q, kv.SharedPrefix(st, starts), ctas=ctas, out_dtype=BF16), ref)
    assert L.device_error() == 0
    table = torch.arange(st.pool.shape[0], dtype=torch.int32, device="cuda").view(6, -1)
    table[:, 2], table[:, 4] = -1, 10**6
    paged = kv.Int4KVStore.wrap(st.pool, table, st.lengths, 2, page_tokens=128)
    out = kv.decode_shared(q, kv.SharedPrefix(paged, starts), out_dtype=BF16)
    assert L.device_error() == L.DEVERR_BAD_PAGE
    keep = [t for t in range(2000) if t // 128 not in (2, 4)]
    check(out, reference(q, starts, k[:, :, keep], v[:, :, keep], [2000 - 256, 0, 1111 - 256]))
    table.fill_(-1)
    out = kv.decode_shared(q, kv.SharedPrefix(paged, starts), out_dtype=BF16)
    assert L.device_error() == L.DEVERR_BAD_PAGE and bool((out == 0).all())


def test_output_types_share_a_workspace(kv, L):
    """Calls of either form in turn on one stream, eager and captured, beside a dense segment."""
    st, k, v = prefix_of(kv, randn(1, 1, 2, 900, 128), randn(2, 1, 2, 900, 128), [900])
    shared = kv.SharedPrefix(st, [0, 9])
    q = randn(4, 9, 8, 128).to(BF16)
    dense = kv.DenseKV(9, 2, 40, dtype=BF16, k=randn(5, 9, 2, 40, 128).to(BF16), v=randn(6, 9, 2, 40, 128).to(BF16))
    dense.set_lengths(40)
    first = {t: kv.decode_shared(q, shared, None, dense, out_dtype=t) for t in (BF16, F32, F16)}
    kc = torch.cat([k.expand(9, -1, -1, -1).double(), dense.k.double()], 2)
    vc = torch.cat([v.expand(9, -1, -1, -1).double(), dense.v.double()], 2)
    ref = reference(q, list(range(10)), kc, vc, [940] * 9)
    outs = {t: torch.zeros_like(o) for t, o in first.items()}
    graphs = []
    for t, o in outs.items():
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            kv.decode_shared(q, shared, None, dense, out=o)
        graphs.append(g)
    for _ in range(3):
        for g in graphs:
            g.replay()
        for t, o in first.items():
            assert torch.equal(kv.decode_shared(q, shared, None, dense, out_dtype=t), o)
    torch.cuda.synchronize()
    for t, o in outs.items():
        assert torch.equal(o, first[t])
        check(o, ref)
    assert L.device_error() == 0
