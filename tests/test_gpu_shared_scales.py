"""The ref format's f32 scales enter a shared prefix's scores and values unrounded.

Two kinds of tokens with the same codes: scales just below and just above the middle
between two neighbouring f16 numbers, 2^-10 of them apart. Their scores differ by next to
nothing, but rounded to f16 the scales would differ by 2^-10, and at scores of 20 the two
kinds' weights by 20 * 2^-10 = 2 %, which their values (+1 and -1) turn into an output of
1e-2. What is left is the rounding of each key element, code times scale, to f16: for each
code at most 2^-11, 2^-11 / sqrt(3) rms; over the codes 1 .. 15 alike, weighted with the
code, 2^-11 / sqrt(3) sqrt(sum c^2) / sum c = 8.3e-5 of the score, 1.7e-3 of a weight,
1.2e-3 of the output (half the difference of two). Three of those, and the weights' own
f16, the same for all tokens of a kind and so at most 2^-11 of the output: 4e-3."""
import pytest
import torch

pytestmark = pytest.mark.gpu
F16 = torch.float16


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows", [4, 20, 40, 100])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_scales_between_two_f16_numbers(rows, group, dtype):
    from hetero_kvcache_optimizer_b200 import _lib, kvstore as kv
    _lib.device_error(clear=True)
    T, ng = 256, 128 // group
    up = torch.arange(T, device="cuda") % 2 == 1
    store = kv.Int4KVStore(1, 1, T, fmt="ref", group=group)
    scale = 0.25 * (1 + 2.0 ** -11 * (1 + 2.0 ** -6 * (2 * up.double() - 1)))
    codes = (torch.arange(128, device="cuda") % 15 + 1).to(torch.uint8).expand(1, 1, T, 128)
    zero = torch.zeros(T * ng, dtype=torch.uint8, device="cuda")
    kv.repack_ref(codes, scale.float().repeat_interleave(ng), zero, group, store, 0)
    # values: +1 or -1 by kind in the first half of the dims, 1 in the second
    v = torch.ones(T, 128, device="cuda")
    v[~up, :64] = -1
    kv.repack_ref((v > 0).to(torch.uint8).view(1, 1, T, 128) * 2, torch.ones(T * ng, device="cuda"), zero + 1, group, store, 1)
    store.set_lengths(T)
    want_score = 20.0
    x = codes[0, 0, 0].double().sum().item() * 0.25
    q = torch.full((rows, 1, 128), want_score / x, device="cuda").to(F16)
    out = kv.decode_shared(q, kv.SharedPrefix(store, [0, rows]), sm_scale=1.0, out_dtype=dtype).double()
    s = (q[0, 0].double() * codes[0, 0].double()).sum(-1) * scale
    p = torch.softmax(s, 0)
    ref = (p[:, None] * v.double()).sum(0)
    assert ref[:64].abs().max() < 1e-3 and (ref[64:] - 1).abs().max() < 1e-9
    over = (out - ref).abs() - ref.abs() * torch.finfo(dtype).eps / 2
    assert over.max().item() < 4e-3
    assert _lib.device_error() == 0


@pytest.mark.parametrize("rows", [1, 9, 16])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_one_token_returns_its_value(rows, group):
    """One token: P = 1, so the output is code times scale. With at most 16 rows the codes
    are exact and P times the scale is two f16. The second is a multiple of 2^-24 at
    the finest and 2^-11 of the first at most, so what is left is 2^-25 or 2^-22 of the
    scale, whichever is more; that times code - zero, and fp32: 2^-21 + 2^-21."""
    from hetero_kvcache_optimizer_b200 import kvstore as kv
    ng = 128 // group
    gen = torch.Generator(device="cuda").manual_seed(rows)
    store = kv.Int4KVStore(1, 1, 128, fmt="ref", group=group, page_tokens=128)
    codes = torch.randint(0, 16, (1, 1, 1, 128), generator=gen, device="cuda").to(torch.uint8)
    scale = 0.01 + torch.rand(ng, generator=gen, device="cuda")
    zero = torch.randint(0, 16, (ng,), generator=gen, device="cuda").to(torch.uint8)
    for role in (0, 1):
        kv.repack_ref(codes, scale, zero, group, store, role)
    store.set_lengths(1)
    q = torch.randn(rows, 1, 128, generator=gen, device="cuda").to(F16)
    out = kv.decode_shared(q, kv.SharedPrefix(store, [0, rows])).double()
    n = codes[0, 0, 0].view(ng, group).double() - zero.double()[:, None]
    ref = (n * scale.double()[:, None]).view(128)
    assert ((out - ref).abs() - 2.0 ** -20 * ref.abs() - 2.0 ** -25 * n.abs().view(128)).max().item() <= 0


@pytest.mark.parametrize("rows", [2, 16, 40])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_codes_and_mins_cancel(rows, group):
    """fp16min values that are zero as 15 scale + min: the codes' products and the mins' are
    both 15 scale P and cancel if both see the same P. Left are fp32 sums (four steps of
    2^-23 on either side: 2^-20 of 15 scale) and what the second f16 of scale times P cannot
    hold, 2^-25 a token times its code, over a sum of P of at least 1."""
    from hetero_kvcache_optimizer_b200 import kvstore as kv
    T, ng = 20, 128 // group
    gen = torch.Generator(device="cuda").manual_seed(group + rows)
    scale = torch.randint(40, 128, (T, ng), generator=gen, device="cuda").double() * 2.0 ** -8
    v = torch.zeros(T, ng, group, dtype=torch.float64, device="cuda")
    v[:, :, 0] = -15 * scale  # exact in f16: 15 * 127 < 2^11
    k = torch.randn(T, 128, generator=gen, device="cuda")
    store = kv.Int4KVStore(1, 1, 128, fmt="fp16min", group=group, page_tokens=128)
    kv.quantize_pack_kv(k.to(F16).view(1, 1, T, 128), v.to(F16).view(1, 1, T, 128), store)
    store.set_lengths(T)
    back = kv.dequantize_pack(store, 1, 0, T, dtype=torch.float32)[0, 0].view(T, ng, group)
    assert bool((back[:, :, 1:] == 0).all()) and bool((back.double() == v).all())
    q = torch.randn(rows, 1, 128, generator=gen, device="cuda").to(F16)
    out = kv.decode_shared(q, kv.SharedPrefix(store, [0, rows])).view(rows, ng, group)
    bound = 15 * (scale.max().item() * 2.0 ** -20 + T * 2.0 ** -25)
    assert out[:, :, 1:].abs().max().item() <= bound
