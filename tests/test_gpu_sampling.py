"""Several sequences from one prompt through the decoder: a shared INT4 prefix, raw
queries and keys normed and rotated on the way in, bodies in page pools, forks in
the middle, eager and captured. Every step's output against 64-bit attention over
what the caches hold (dequantised) with queries rotated by the formula; tolerance
as in test_gpu_shared.py (2e-3 of a row's norm, fp32 outputs) plus the rounding of
the rotated query to its 16-bit type: 2^-9 (bf16) relative, by which every score is
off by at most 2^-9 of it, with random signs over 128 products 2^-9 / 11.3 of scores
below 16: under 3e-3 of p, random over tokens like p's own rounding."""
import pytest
import torch

pytestmark = pytest.mark.gpu
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def rotated(x, pos, table, w, eps=1e-6):
    y = x.double()
    if w is not None:
        y = y / torch.sqrt(y.square().mean(-1, keepdim=True) + eps) * w.double()
    r = table.shape[1] // 2
    c, s = table.double()[pos.long()][:, None].split(r, -1)
    a, b = y[..., :r], y[..., r:2 * r]
    return torch.cat((a * c - b * s, b * c + a * s, y[..., 2 * r:]), -1)


class Run:
    L, B, H, G, T = 2, 6, 2, 4, 700

    def __init__(self, fmt, prefix=True, seed=0):
        from hetero_kvcache_optimizer_b200 import kvstore as kv
        from hetero_kvcache_optimizer_b200.decode_engine import TieredKVDecoder
        self.kv, self.gen = kv, torch.Generator(device="cuda").manual_seed(seed)
        self.dec = TieredKVDecoder(self.L, self.B, self.H * self.G, self.H, sink=2, recent=6, body_capacity=1024, fmt=fmt,
                                   page_tokens=128, kv_dtype=BF16, out_dtype=F32, num_pages=60)
        self.starts = [0, 3, self.B]
        self.prefix = []
        for _ in range(self.L):
            st = kv.Int4KVStore(2, self.H, self.T, fmt=fmt, page_tokens=256)
            kv.prefill(st, self.randn(2, self.H, self.T, 128).to(F16), self.randn(2, self.H, self.T, 128).to(F16))
            st.set_lengths(torch.tensor([self.T, 301]))
            self.prefix.append(kv.SharedPrefix(st, self.starts))
        if prefix:
            self.dec.attach_prefix(self.prefix)
        self.table = kv.rope_table(2048, 128, base=1e6)
        self.qw, self.kw = ([(1 + 0.2 * self.randn(128)).to(BF16) for _ in range(self.L)] for _ in range(2))
        self.dec.set_rotary(self.table, self.qw, self.kw)
        for st in self.dec.stores:
            st.set_lengths(0)

    def randn(self, *shape):
        return torch.randn(*shape, generator=self.gen, device="cuda")

    def inputs(self):
        return (self.randn(self.L, self.B, self.H * self.G, 128).to(BF16), self.randn(self.L, self.B, self.H, 128).to(BF16),
                self.randn(self.L, self.B, self.H, 128).to(BF16))

    def check(self, out, q, pos):
        kv, dec = self.kv, self.dec
        for l in range(self.L):
            qr = rotated(q[l], pos, self.table, self.qw[l]).view(self.B, self.H, self.G, 128)
            st, d = dec.stores[l], dec.dense[l]
            n = st.lengths.tolist()
            most = max(max(n), 1)
            sides = []
            for role, dense in ((0, d.k), (1, d.v)):
                body = kv.dequantize_pack(st, role, 0, most, dtype=F32)
                pre = kv.dequantize_pack(self.prefix[l].store, role, 0, self.T, dtype=F32)
                sides.append([torch.cat(([pre[int(b >= 3), :, :(self.T, 301)[int(b >= 3)]].double()] if dec.prefixes else [])
                                        + [body[b, :, :n[b]].double(), dense[b, :, :int(d.lengths[b])].double()], 1) for b in range(self.B)])
            for b in range(self.B):
                p = torch.softmax(qr[b] @ sides[0][b].transpose(1, 2) * 128 ** -0.5, -1)
                ref = (p @ sides[1][b]).reshape(self.H * self.G, 128)
                err = (out[l, b].double() - ref).abs().amax(-1) / ref.norm(dim=-1)
                assert err.max().item() < 2e-3, (l, b, err.max().item())


@pytest.mark.parametrize("fmt", ["fp16min", "ref"])
def test_samples_fork_and_go_on(fmt):
    from hetero_kvcache_optimizer_b200 import _lib
    _lib.device_error(clear=True)
    run = Run(fmt)
    pos = torch.full((run.B,), 700, dtype=torch.int32, device="cuda")
    for step in range(140):  # the ring fills after 8, then tokens move into the body, past a page
        if step % 50 == 0:
            run.dec.reserve(50)
        if step in (5, 60, 133):
            parents = [[0, 0, 1, 3, 3, 5], [2, 1, 0, 5, 4, 4], [0, 0, 0, 3, 3, 3]][(5, 60, 133).index(step)]
            keys = [st.lengths.clone() for st in run.dec.stores]
            run.dec.fork(parents)
            assert all(torch.equal(st.lengths, k[torch.tensor(parents, device="cuda")]) for st, k in zip(run.dec.stores, keys))
            run.dec.reserve(50)
            q, k, v = run.inputs()
            for x in (q, k, v):  # the same token for all: the same result for those with one parent
                x.copy_(x[:, :1].expand_as(x))
            out = run.dec.step(q, k, v, positions=pos)
            for b in range(run.B):
                for c in range(b):
                    if parents[b] == parents[c]:
                        assert torch.equal(out[:, b], out[:, c])
        else:
            q, k, v = run.inputs()
            out = run.dec.step(q, k, v, positions=pos)
        if step in (0, 5, 7, 8, 9, 59, 60, 61, 133, 136, 139):
            run.check(out, q, pos)
        pos += 1
    assert _lib.device_error() == 0


def test_captured_step():
    from hetero_kvcache_optimizer_b200 import _lib
    _lib.device_error(clear=True)
    run = Run("fp16min", seed=3)
    run.dec.reserve(300)
    for _ in range(9):
        q, k, v = run.inputs()
        run.dec.step(q, k, v, positions=torch.zeros(run.B, dtype=torch.int32, device="cuda"))
    run.dec.capture(64, positions=torch.full((run.B,), 900))
    qs, ks, vs, out = run.dec.static_buffers
    for step in range(4):
        q, k, v = run.inputs()
        qs.copy_(q), ks.copy_(k), vs.copy_(v)
        run.dec.replay()
        run.check(out, q, torch.full((run.B,), 900 + step, device="cuda"))
        assert run.dec.positions.tolist() == [901 + step] * run.B
    with pytest.raises(RuntimeError):
        run.dec.capture_host()
    assert _lib.device_error() == 0


def test_without_prefix_the_fused_step_takes_raw_queries():
    from hetero_kvcache_optimizer_b200 import _lib
    _lib.device_error(clear=True)
    run = Run("fp16min", prefix=False, seed=5)
    assert run.dec.launches_per_layer == 1
    run.dec.reserve(64)
    for step in range(20):
        q, k, v = run.inputs()
        pos = torch.full((run.B,), step, dtype=torch.int64, device="cuda")
        out = run.dec.step(q, k, v, positions=pos)
    run.check(out, q, pos)
    assert _lib.device_error() == 0


def test_refusals():
    run = Run("ref")
    from hetero_kvcache_optimizer_b200.decode_engine import TieredKVDecoder
    plain = TieredKVDecoder(1, 2, 4, 1, sink=2, recent=4, body_capacity=128)
    for call in (lambda: plain.fork([0, 0]), lambda: plain.reserve(1),
                 lambda: plain.step(*(torch.zeros(1, 2, h, 128, dtype=F16, device="cuda") for h in (4, 1, 1)),
                                    positions=torch.zeros(2, dtype=torch.int32, device="cuda"))):
        with pytest.raises(RuntimeError):
            call()
    for bad in (run.prefix[:1], [run.prefix[0]] * 3):
        with pytest.raises(ValueError):
            run.dec.attach_prefix(bad)
    with pytest.raises(ValueError):
        plain.attach_prefix(run.prefix[:1])
    with pytest.raises(ValueError):
        run.dec.set_rotary(run.table, run.qw[:1])
    with pytest.raises(ValueError):
        run.dec.fork([0, 0, 0, 0, 0, -2])


def test_parents_on_the_device_and_emptied_sequences():
    from hetero_kvcache_optimizer_b200 import _lib
    _lib.device_error(clear=True)
    run = Run("fp16min", seed=7)
    run.dec.reserve(200)
    pos = torch.arange(run.B, dtype=torch.int64, device="cuda")
    for _ in range(20):
        q, k, v = run.inputs()
        run.dec.step(q, k, v, positions=pos)
    for parents in (torch.tensor([4, -1, 4, 0, -1, 0], device="cuda"), [-1, 2, 2, 3, 3, -1]):
        run.dec.fork(parents)
        run.dec.reserve(200)
        gone = [b for b in range(run.B) if int(parents[b]) < 0]
        for st, d in zip(run.dec.stores, run.dec.dense):
            assert all(st.lengths[b] == 0 and d.lengths[b] == 0 for b in gone)
        for _ in range(11):
            q, k, v = run.inputs()
            out = run.dec.step(q, k, v, positions=pos)
        run.check(out, q, pos)
    assert _lib.device_error() == 0


def test_prefill_after_a_fork_writes_no_shared_page():
    from hetero_kvcache_optimizer_b200 import _lib
    _lib.device_error(clear=True)
    run = Run("ref", seed=8)
    n = 2 + 6 + 300
    pos = torch.full((run.B,), 3, dtype=torch.int32, device="cuda")
    for again in range(2):
        for l in range(run.L):
            run.dec.prefill_layer(l, run.randn(run.B, run.H, n, 128).to(BF16), run.randn(run.B, run.H, n, 128).to(BF16))
        for st in run.dec.stores:
            t = st.page_table[st.page_table >= 0]
            assert t.numel() == run.B * run.H * 3 and t.unique().numel() == t.numel()
        run.dec.reserve(20)
        q, k, v = run.inputs()
        run.check(run.dec.step(q, k, v, positions=pos), q, pos)
        run.dec.fork([0, 0, 0, 1, 1, 1])
    run.dec.set_state(200)
    for st in run.dec.stores:
        t = st.page_table[st.page_table >= 0]
        assert t.numel() == run.B * run.H * 2 and t.unique().numel() == t.numel()
    assert _lib.device_error() == 0


def test_attention_alone_sees_the_prefix_and_a_stale_graph_is_dropped():
    from hetero_kvcache_optimizer_b200 import _lib
    _lib.device_error(clear=True)
    run = Run("fp16min", prefix=False, seed=9)
    run.dec.reserve(64)
    pos = torch.zeros(run.B, dtype=torch.int32, device="cuda")
    for _ in range(12):
        q, k, v = run.inputs()
        run.dec.step(q, k, v, positions=pos)
    run.dec.capture(4, positions=pos)
    run.dec.attach_prefix(run.prefix)
    with pytest.raises(RuntimeError):
        run.dec.replay()
    q = run.inputs()[0]
    out = torch.empty(run.L, run.B, run.H * run.G, 128, device="cuda")
    ready = torch.stack([run.kv.norm_rope(q[l], None, pos, run.table, run.qw[l])[0] for l in range(run.L)])
    run.dec.decode_only(ready, out)
    run.check(out, q, pos)
    assert _lib.device_error() == 0
