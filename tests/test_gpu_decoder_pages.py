"""TieredKVDecoder over page pools: steps, forks and reserves back to back."""
import pytest
import torch

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def decoder(layers, **kw):
    from hetero_kvcache_optimizer_b200.decode_engine import TieredKVDecoder
    return TieredKVDecoder(layers, 3, 8, 2, sink=2, recent=6, body_capacity=1024, fmt="fp16min", page_tokens=128,
                           kv_dtype=BF16, num_pages=40, **kw)


@pytest.mark.parametrize("layers", [2, 3])
@pytest.mark.parametrize("ctas", [2, 0])
def test_early_layers_see_what_the_pool_calls_and_the_last_step_wrote(layers, ctas):
    """Fused steps without positions (no launch between the layers), with pool calls just
    before them and few CTAs (room for the next grid beside a running one), give the same
    bits as steps that wait for everything before them."""
    from hetero_kvcache_optimizer_b200 import _lib
    _lib.device_error(clear=True)
    runs = []
    for early in (None, False):
        gen = torch.Generator(device="cuda").manual_seed(5)
        dec = decoder(layers, ctas=ctas, early=early)
        for l in range(layers):
            k, v = (torch.randn(3, 2, 8 + 300, 128, generator=gen, device="cuda").to(BF16) for _ in range(2))
            dec.prefill_layer(l, k, v)
        dec.reserve(128)
        outs = []
        for step in range(24):
            q = torch.randn(layers, 3, 8, 128, generator=gen, device="cuda").to(BF16)
            k, v = (torch.randn(layers, 3, 2, 128, generator=gen, device="cuda").to(BF16) for _ in range(2))
            if step % 6 == 3:
                dec.fork([[0, 0, 2], [1, 1, 0], [2, 0, 1], [0, 1, 2]][step // 6])
                dec.reserve(128)
            elif step % 6 == 5:
                dec.pools[layers - 1].reserve(128)
            outs.append(dec.step(q, k, v))
        torch.cuda.synchronize()
        runs.append((outs, [(s.lengths.clone(), s.page_table.clone(), d.k.clone(), d.ring_head.clone())
                            for s, d in zip(dec.stores, dec.dense)]))
    for a, b in zip(runs[0][0], runs[1][0]):
        assert torch.equal(a, b)
    for a, b in zip(runs[0][1], runs[1][1]):
        assert all(torch.equal(x, y) for x, y in zip(a, b))
    assert _lib.device_error() == 0


def test_a_captured_step_goes_on_from_its_parents_positions():
    """Sequences at different positions, forked between replays: the same caches and
    outputs as eager steps that are given the parents' positions."""
    from hetero_kvcache_optimizer_b200 import _lib, kvstore as kv
    _lib.device_error(clear=True)
    runs = []
    for captured in (True, False):
        gen = torch.Generator(device="cuda").manual_seed(6)
        dec = decoder(2)
        table = kv.rope_table(1024, 128)
        dec.set_rotary(table)
        pos = torch.tensor([5, 300, 77], dtype=torch.int32, device="cuda")
        dec.reserve(128)
        if captured:
            dec.capture(20, positions=pos)
        outs = []
        for step in range(9):
            q = torch.randn(2, 3, 8, 128, generator=gen, device="cuda").to(BF16)
            k, v = (torch.randn(2, 3, 2, 128, generator=gen, device="cuda").to(BF16) for _ in range(2))
            if step in (3, 6):
                parents = [1, 0, 1] if step == 3 else [2, -1, 0]
                dec.fork(parents)
                pos = torch.where(torch.tensor(parents, device="cuda") < 0, 0, pos[torch.tensor(parents, device="cuda").clamp(min=0)])
                dec.reserve(128)
            if captured:
                for buf, x in zip(dec.static_buffers, (q, k, v)):
                    buf.copy_(x)
                dec.replay()
                outs.append(dec.static_buffers[3].clone())
            else:
                outs.append(dec.step(q, k, v, positions=pos, len_hint=20))
            pos = pos + 1
            if captured:
                assert dec.positions.tolist() == pos.tolist()
        runs.append(outs + [d.k.clone() for d in dec.dense])
    assert all(torch.equal(a, b) for a, b in zip(*runs))
    assert _lib.device_error() == 0


def test_host_steps_after_a_second_capture():
    """The host buffers of the first capture still serve as plain inputs; their graph is gone."""
    runs = []
    for again in (False, True):
        gen = torch.Generator(device="cuda").manual_seed(8)
        dec = decoder(2)
        for l in range(2):
            dec.prefill_layer(l, *(torch.randn(3, 2, 8 + 200, 128, generator=gen, device="cuda").to(BF16) for _ in range(2)))
        dec.reserve(128)
        dec.capture(8)
        dec.capture_host()
        bufs = dec.host_buffers
        if again:
            dec.capture(8)
            assert dec.host_buffers is None
        outs = []
        for _ in range(3):
            for b, n in zip(bufs, (8, 2, 2)):
                b.copy_(torch.randn(2, 3, n, 128, generator=gen, device="cuda"))
            torch.cuda.synchronize()
            dec.step_host(*bufs)
            torch.cuda.synchronize()
            outs.append(bufs[3].clone())
        runs.append(outs)
    assert all(torch.equal(a, b) for a, b in zip(*runs))


def test_a_padded_batch_stays_padded_in_a_captured_step():
    """A sequence of negative position pads the batch at every replay; the others go on
    as eager steps with the same positions do."""
    from hetero_kvcache_optimizer_b200 import _lib, kvstore as kv
    _lib.device_error(clear=True)
    runs = []
    for captured in (True, False):
        gen = torch.Generator(device="cuda").manual_seed(9)
        dec = decoder(2)
        dec.set_rotary(kv.rope_table(64, 128))
        dec.reserve(128)
        pos = torch.tensor([5, -3, 40], dtype=torch.int32, device="cuda")
        if captured:
            dec.capture(12, positions=pos)
        outs = []
        for step in range(12):
            q = torch.randn(2, 3, 8, 128, generator=gen, device="cuda").to(BF16)
            k, v = (torch.randn(2, 3, 2, 128, generator=gen, device="cuda").to(BF16) for _ in range(2))
            if captured:
                for buf, x in zip(dec.static_buffers, (q, k, v)):
                    buf.copy_(x)
                dec.replay()
                outs.append(dec.static_buffers[3][:, [0, 2]])
            else:
                outs.append(dec.step(q, k, v, positions=pos, len_hint=12)[:, [0, 2]])
            pos = torch.where(pos < 0, pos, pos + 1)
            if captured:
                assert dec.positions.tolist() == pos.tolist()
        runs.append(outs)
    assert all(torch.equal(a, b) for a, b in zip(*runs))
    assert _lib.device_error() == 0
