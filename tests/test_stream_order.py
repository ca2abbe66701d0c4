"""What the wrappers copy on the way in is copied on the stream that the call is given,
behind the work already queued there (on the CPU: the calls' order; on the GPU: a query
written late on that stream)."""
import pytest
import torch


def test_the_copy_of_strided_queries_is_inside_the_streams_context(monkeypatch):
    from hetero_kvcache_optimizer_b200.csrc import build
    build.build()
    from hetero_kvcache_optimizer_b200 import kvstore as kv

    class Entered(Exception):
        pass

    def launch_on(device, stream=None):
        raise Entered

    def contiguous(self, *a, **k):
        raise AssertionError("copied before the stream's context")
    monkeypatch.setattr(kv, "_require_cuda", lambda *t: None)
    monkeypatch.setattr(kv, "launch_on", launch_on)
    prefix = kv.SharedPrefix(kv.Int4KVStore(1, 1, 128, page_tokens=128, device="cpu"), [0, 2])
    q = torch.zeros(2, 128, 4, dtype=torch.float16).transpose(1, 2)
    monkeypatch.setattr(torch.Tensor, "contiguous", contiguous)
    with pytest.raises(Entered):
        kv.decode_shared(q, prefix)


@pytest.mark.gpu
def test_strided_queries_written_late_on_another_stream():
    from hetero_kvcache_optimizer_b200 import kvstore as kv
    gen = torch.Generator(device="cuda").manual_seed(1)
    st = kv.Int4KVStore(1, 2, 512)
    kv.prefill(st, *(torch.randn(1, 2, 400, 128, generator=gen, device="cuda").to(torch.float16) for _ in range(2)))
    prefix = kv.SharedPrefix(st, [0, 3])
    new = torch.randn(3, 128, 8, generator=gen, device="cuda").to(torch.float16)
    want = kv.decode_shared(new.transpose(1, 2).contiguous(), prefix)
    late = torch.zeros_like(new)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        torch.cuda._sleep(20_000_000)  # about 10 ms
        late.copy_(new)
    out = kv.decode_shared(late.transpose(1, 2), prefix, stream=s)
    s.synchronize()
    assert torch.equal(out, want)
