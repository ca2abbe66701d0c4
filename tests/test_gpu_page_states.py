"""PagePool calls on states that a long life of forks alone does not reach: sequences cut
back while others still use the pages, tables and lengths that the caller built, full rows.
Ids, counts and bytes are equal to what the text of each call says."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
P = 128


@pytest.fixture(scope="module")
def kv():
    from hetero_kvcache_optimizer_b200 import kvstore
    return kvstore


@pytest.fixture(scope="module")
def PagePool():
    from hetero_kvcache_optimizer_b200.memory.page_pool import PagePool
    return PagePool


@pytest.fixture(scope="module")
def L():
    from hetero_kvcache_optimizer_b200 import _lib
    _lib.device_error(clear=True)
    return _lib


def pool_of(kv, PagePool, table, lengths, H, pages, fill=None, fmt="ref", group=128):
    """A pool over a table [B * H][max_pages] and lengths of the caller's own."""
    nbytes = kv.page_bytes(fmt, group, P)
    data = (torch.full((pages, nbytes), fill, dtype=torch.uint8, device="cuda") if fill is not None
            else torch.randint(0, 256, (pages, nbytes), dtype=torch.uint8, device="cuda", generator=torch.Generator(device="cuda").manual_seed(pages)))
    return PagePool(kv.Int4KVStore.wrap(data, torch.tensor(table, dtype=torch.int32, device="cuda"),
                                        torch.tensor(lengths, dtype=torch.int32, device="cuda"), H, fmt=fmt, group=group, page_tokens=P))


@pytest.mark.parametrize("lengths", [(0, 300, 150), (129, 384, 1), (128, 127, 384), (384, 0, 0), (0, 0, 0), (1, 0, 129)])
@pytest.mark.parametrize("wide", [False, True])
def test_compact_copies_a_page_that_any_sequence_uses(kv, PagePool, L, lengths, wide):
    """Three sequences of two heads that share pages and stand at different lengths; with
    `wide` rows the table takes several CTAs to rank and sharers lie in different ones."""
    H, maxp = 2, 6 if not wide else 3000
    rows = np.full((6, maxp), -1, np.int64)
    rows[:, :3] = [[4, 9, 2], [7, 0, 12], [4, 9, 2], [7, 0, 13], [4, 3, 2], [7, 11, 13]]
    src = pool_of(kv, PagePool, rows.tolist(), lengths, H, 16)
    into = pool_of(kv, PagePool, np.full((6, maxp), -1).tolist(), [5, 5, 5], H, 16, fill=9)
    before = src.store.pool.cpu().numpy().copy()
    src.compact(into)
    assert L.device_error() == 0
    rank, used = {}, set()
    for u in range(6):
        for i in range(3):
            rank.setdefault(rows[u, i], len(rank))
            if i * P < lengths[u // H]:
                used.add(rows[u, i])
    want = np.full_like(before, 9)
    for page in used:
        want[rank[page]] = before[page]
    table = np.full((6, maxp), -1)
    table[:, :3] = np.vectorize(rank.get)(rows[:, :3])
    assert np.array_equal(into.store.page_table.cpu().numpy(), table)
    assert np.array_equal(into.store.pool.cpu().numpy(), want)
    assert np.array_equal(src.store.pool.cpu().numpy(), before)
    assert into.store.lengths.tolist() == list(lengths)
    refs = np.zeros(16, np.int64)
    np.add.at(refs, table[table >= 0], 1)
    assert into.refs.tolist() == refs.tolist()


@pytest.mark.parametrize("held,tokens,short", [(10, 502, False), (10, 503, True), (10, 512, True), (0, 512, False), (1, 512, True),
                                               (128, 384, False), (128, 385, True), (512, 1, True), (511, 1, False), (600, 1, True)])
@pytest.mark.parametrize("lowered", [False, True])
def test_reserve_beyond_a_rows_end_is_flagged(kv, PagePool, L, held, tokens, short, lowered):
    """Rows of 4 pages: the entries that exist get pages, and what does not fit sets
    DEVERR_CAPACITY, however far behind the row's end it lies."""
    n = min(4, -(-held // P))
    table = [list(range(n)) + [-1] * (4 - n), [-1] * 4]
    pool = pool_of(kv, PagePool, table, [held, 0], 1, 12)
    if lowered:
        pool.reserve(512, torch.tensor([tokens, 0]))
    else:
        pool.reserve(tokens)
    assert L.device_error() == (L.DEVERR_CAPACITY if short else 0)
    full = min(4, -(-(held + tokens) // P))
    got = pool.store.page_table.tolist()
    assert got[0] == list(range(full)) + [-1] * (4 - full)
    assert (sum(x >= 0 for x in got[1]) == (0 if lowered else -(-tokens // P)))
    assert pool.refs.tolist() == [int(i < sum(x >= 0 for r in got for x in r)) for i in range(12)]


def test_lists_from_the_host_do_not_wait_and_are_captured(kv, PagePool, L):
    """free, fork and reserve with plain lists (and tensors on the host): queued behind a
    busy stream without waiting for it, captured with their values, the same state after."""
    table = [[0, 1, -1, -1], [2, 3, 4, -1], [5, -1, -1, -1]]

    def calls(pool):
        pool.fork([1, 0, 0])
        pool.reserve(200, torch.tensor([1, 200, 100]))
        pool.free([2])
        pool.fork(torch.tensor([0, 1, 1]))
    plain, queued, graphed = (pool_of(kv, PagePool, table, [250, 300, 7], 1, 24) for _ in range(3))
    calls(plain)
    torch.cuda.synchronize()
    done = torch.cuda.Event()
    torch.cuda._sleep(400_000_000)  # about 0.2 s
    calls(queued)
    done.record()
    assert not done.query()
    s, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        calls(graphed)
    torch.cuda.synchronize()
    assert graphed.store.lengths.tolist() == [250, 300, 7]
    torch.empty(1 << 20, device="cuda").fill_(1)  # whatever memory the calls' temporaries had
    g.replay()
    torch.cuda.synchronize()
    for pool in (queued, graphed):
        for a, b in ((pool.refs, plain.refs), (pool.store.page_table, plain.store.page_table), (pool.store.lengths, plain.store.lengths),
                     (pool.store.pool, plain.store.pool)):
            assert torch.equal(a, b)
    assert L.device_error() == 0


@pytest.mark.parametrize("n", [1, 255, 960, 961, 4000])
def test_many_values_from_the_host(L, n):
    import ctypes
    dst = torch.full((n + 1,), 7, dtype=torch.int32, device="cuda")
    values = [(i * 2654435761) % 2**32 - 2**31 for i in range(n)]
    host = (ctypes.c_int32 * n)(*values)
    L.check(L.load().hkv_put_i32(host, n, dst.data_ptr(), torch.cuda.current_stream().cuda_stream), "hkv_put_i32")
    ctypes.memset(host, 0, 4 * n)  # read before the call returned
    assert dst.tolist() == values + [7]


def test_lists_of_another_length_or_range_are_refused(kv, PagePool):
    pool = pool_of(kv, PagePool, [[0], [1]], [5, 5], 1, 4)
    for bad in ([0], [0, 1, 2], [0, 2**31], [-2**31 - 1, 0], torch.tensor([0, 2**40])):
        with pytest.raises(ValueError):
            pool.fork(bad)
        with pytest.raises(ValueError):
            pool.reserve(1, bad)


def test_wide_integers_on_the_device_are_not_cut_down(kv, PagePool, L):
    """Parents beyond 32 bits are outside the batch like any other, and counts beyond them
    lower nothing."""
    pool = pool_of(kv, PagePool, [[0, -1, -1], [1, -1, -1], [2, -1, -1]], [100, 90, 80], 1, 12)
    pool.reserve(200, torch.tensor([2**32, -2**32, 2**33 + 5], device="cuda"))
    assert L.device_error() == 0
    assert pool.store.page_table.tolist() == [[0, 3, 4], [1, -1, -1], [2, 5, 6]]
    pool.fork(torch.tensor([2**32, 1, -2**32 + 2], device="cuda"))
    assert L.device_error() == L.DEVERR_BAD_PAGE
    assert pool.store.lengths.tolist() == [0, 90, 0]
    assert pool.store.page_table.tolist() == [[-1] * 3, [1, -1, -1], [-1] * 3]
