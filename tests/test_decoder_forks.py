"""What TieredKVDecoder keeps beside the caches when sequences fork, are rotated and share
prefixes: host logic, on the CPU with page pools that only record their calls (no kernel runs)."""
import pytest
import torch


class Pool:
    def __init__(self, batch):
        self.batch, self.calls = batch, []

    def _per_sequence(self, x, name):
        return x if isinstance(x, torch.Tensor) else torch.tensor(list(x), dtype=torch.int32)

    def fork(self, parents, stream=None):
        self.calls.append(("fork", parents.tolist()))

    def reserve(self, tokens, tokens_of=None, stream=None):
        self.calls.append(("reserve", tokens))


class Reached(Exception):
    """The step got as far as its first launch."""


@pytest.fixture
def dec(monkeypatch):
    from hetero_kvcache_optimizer_b200 import kvstore as kv
    from hetero_kvcache_optimizer_b200.csrc import build
    from hetero_kvcache_optimizer_b200.decode_engine import TieredKVDecoder
    build.build()
    d = TieredKVDecoder(2, 6, 4, 2, sink=2, recent=4, body_capacity=256, page_tokens=128, device="cpu")
    d.pools = [Pool(6) for _ in range(2)]

    def launch(*a, **k):
        raise Reached
    for name in ("append_kv", "decode_append", "decode", "decode_shared", "norm_rope"):
        monkeypatch.setattr(kv, name, launch)
    return d


def prefixes(starts, layers=2):
    from hetero_kvcache_optimizer_b200 import kvstore as kv
    return [kv.SharedPrefix(kv.Int4KVStore(len(starts) - 1, 2, 256, page_tokens=128, device="cpu"), starts) for _ in range(layers)]


def step(d):
    q, k = torch.zeros(2, 6, 4, 128, dtype=torch.float16), torch.zeros(2, 6, 2, 128, dtype=torch.float16)
    with pytest.raises(Reached):
        d.step(q, k, k)


def refused(d):
    q, k = torch.zeros(2, 6, 4, 128, dtype=torch.float16), torch.zeros(2, 6, 2, 128, dtype=torch.float16)

    class Graph:
        def replay(self):
            raise AssertionError("a graph over a mixed context was replayed")
    d.graph = d.host_graph = Graph()
    d._host = (q, k, k, q)
    for call in (lambda: d.step(q, k, k), lambda: d.decode_only(q, q), d.replay, lambda: d.step_host(q, k, k, q)):
        with pytest.raises(RuntimeError, match="prefix group"):
            call()


def test_a_fork_across_prefix_groups_is_not_attended_to(dec):
    dec.attach_prefix(prefixes([0, 3, 5]))  # sequence 5 has no prefix
    for parents in ([0, 0, 1, 3, 3, 5], [2, 2, 2, 4, -1, 5], [-1] * 6, torch.tensor([1, 1, 1, 4, 4, -1])):
        dec.fork(parents)
        step(dec)
    for parents in ([0, 1, 3, 3, 4, 5], [0, 1, 2, 3, 4, 0], [0, 1, 2, 5, 4, 5], torch.tensor([4, 1, 2, 3, 4, 5])):
        dec.attach_prefix(prefixes([0, 3, 5]))
        dec.fork(parents)
        refused(dec)


def test_what_makes_a_mixed_sequence_whole_again(dec):
    def mix():
        dec.attach_prefix(prefixes([0, 3, 6]))
        dec.fork([0, 1, 3, 3, 4, 5])  # sequence 2 follows group 1
        refused(dec)
    mix()
    dec.fork([2, 1, 1, 3, 4, 5])  # handed on within the group
    refused(dec)
    dec.fork([1, 1, 1, 3, 4, 5])
    step(dec)
    mix()
    dec.fork([0, 1, -1, 3, 4, 2])  # emptied; and back in its own group
    step(dec)
    mix()
    dec.attach_prefix(prefixes([0, 2, 6]))  # the batch is cut elsewhere now
    step(dec)
    mix()
    dec.attach_prefix(None)
    step(dec)
    mix()
    dec.fused_append = False
    dec.set_state(0)
    step(dec)
    dec.fork([3] * 6)
    dec.prefill_layer(0, *(torch.zeros(6, 2, 3, 128),) * 2)
    step(dec)


def test_layers_may_be_cut_into_different_groups(dec):
    dec.attach_prefix(prefixes([0, 3, 6], 1) + prefixes([0, 6], 1))
    dec.fork([2, 1, 0, 5, 4, 3])
    step(dec)
    dec.fork([0, 1, 2, 0, 4, 5])
    refused(dec)


def test_positions_of_a_captured_step_follow_the_fork(dec):
    dec.positions = torch.tensor([7, 20, 300, 4, 50, 6], dtype=torch.int32)
    address = dec.positions.data_ptr()
    dec.fork([2, 0, -1, 5, 5, 3])
    assert dec.positions.tolist() == [300, 7, 0, 6, 6, 4]
    dec.fork(torch.tensor([1, 1, 1, -1, 0, 9], dtype=torch.int32))
    assert dec.positions.tolist() == [7, 7, 7, 0, 300, 0]
    assert dec.positions.data_ptr() == address  # the graph's own buffer


def test_another_rotation_drops_the_step_captured_with_the_old_one(dec):
    class Graph:
        def replay(self):
            pass
    dec.graph, dec.positions = Graph(), None  # captured without positions: holds no table
    dec.set_rotary(torch.zeros(8, 128))
    dec.replay()
    dec.positions = torch.zeros(6, dtype=torch.int32)
    dec.set_rotary(torch.zeros(16, 128))
    with pytest.raises(RuntimeError, match="captured"):
        dec.replay()
    dec._static = (torch.zeros(1),) * 4  # still a step that takes raw queries: not for the host's
    with pytest.raises(RuntimeError, match="rotated"):
        dec.capture_host()


def test_a_new_capture_drops_the_steps_over_the_buffers_it_replaces(dec, monkeypatch):
    def stream(*a, **k):
        raise Reached
    monkeypatch.setattr(torch.cuda, "Stream", stream)
    dec.graph = dec.host_graph = dec._host = object()
    with pytest.raises(Reached):
        dec.capture(4)
    assert dec.graph is None and dec.host_graph is None and dec.host_buffers is None
