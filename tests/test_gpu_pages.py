"""PagePool (fork, reserve, free, compact) against a model in Python: page ids,
counts and bytes have to be equal, whatever the order of the threads."""
import random

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


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


class Model:
    """The state of a pool on the host, and what each call does to it."""

    def __init__(self, B, H, maxp, pages, P, fmt, group, kv):
        self.B, self.H, self.maxp, self.pages, self.P = B, H, maxp, pages, P
        self.bytes = kv.page_bytes(fmt, group, P)
        self.table = np.full((B, H, maxp), -1, np.int64)
        self.lengths = np.zeros(B, np.int64)
        self.refs = np.zeros(pages, np.int64)
        self.pool = np.random.RandomState(1).randint(0, 256, (pages, self.bytes)).astype(np.uint8)

    def take(self):
        free = np.flatnonzero(self.refs == 0)
        if not len(free):
            return -1
        self.refs[free[0]] = 1
        return int(free[0])

    def count(self, extra=None):
        self.refs[:] = 0 if extra is None else extra
        np.add.at(self.refs, self.table[self.table >= 0], 1)

    def reserve(self, tokens):
        short = False
        for b in range(self.B):
            for h in range(self.H):
                first, end = self.lengths[b] // self.P, -(-(self.lengths[b] + tokens[b]) // self.P)
                for i in range(first, end):
                    if i >= self.maxp:
                        short = True
                    elif self.table[b, h, i] < 0:
                        self.table[b, h, i] = self.take()
                        short |= self.table[b, h, i] < 0
        return short

    def fork(self, parents, owned=None):
        old, lens = self.table.copy(), self.lengths.copy()
        wants, short = [], False
        for b, a in enumerate(parents):
            self.table[b] = -1
            self.lengths[b] = lens[a] if a >= 0 else 0
            if a < 0:
                continue
            if a not in parents[:b]:
                self.table[b] = old[a]
                continue
            full = lens[a] // self.P
            self.table[b, :, :full] = old[a, :, :full]
            if lens[a] % self.P:
                wants += [(b, h, full, old[a, h, full], lens[a] % self.P) for h in range(self.H) if old[a, h, full] >= 0]
        self.count(owned)
        for b, h, i, src, rest in wants:
            page = self.take()
            self.table[b, h, i] = page
            if page < 0:
                short = True
                continue
            n = -(-rest // 128) * (self.bytes * 128 // self.P)
            self.pool[page, :n] = self.pool[src, :n]
        return short

    def upload(self, kv, PagePool, fmt, group, refs=None):
        s = kv.Int4KVStore.wrap(torch.from_numpy(self.pool).cuda(), torch.from_numpy(self.table.reshape(-1, self.maxp)).int().cuda(),
                                torch.from_numpy(self.lengths).int().cuda(), self.H, fmt=fmt, group=group, page_tokens=self.P)
        return PagePool(s, refs)

    def same(self, pool):
        torch.cuda.synchronize()
        st = pool.store
        assert np.array_equal(st.lengths.cpu().numpy(), self.lengths)
        assert np.array_equal(st.page_table.cpu().numpy().reshape(self.table.shape), self.table)
        assert np.array_equal(pool.refs.cpu().numpy(), self.refs)
        assert np.array_equal(st.pool.cpu().numpy(), self.pool)


@pytest.mark.parametrize("fmt,group,P", [("ref", 128, 128), ("fp16min", 32, 256), ("ref", 32, 640)])
@pytest.mark.parametrize("B,H", [(1, 1), (5, 2), (9, 3)])
def test_a_long_life(kv, PagePool, L, fmt, group, P, B, H):
    """Growth, forks, beam reorders and frees in a random order, the pool checked whole after each."""
    rng = random.Random(17 * B + P)
    m = Model(B, H, 6, B * H * 6 + 5, P, fmt, group, kv)
    pool = m.upload(kv, PagePool, fmt, group)
    for step in range(30):
        what = rng.choice(["grow", "grow", "fork", "reorder", "free"])
        if what == "grow":
            room = [rng.choice([0, 1, P // 2, P, 2 * P + 1]) for _ in range(B)]
            room = [min(r, 6 * P - int(n)) for r, n in zip(room, m.lengths)]
            m.reserve(room)
            pool.reserve(2 * P + 1, torch.tensor(room))
            m.lengths += room
            pool.store.lengths += torch.tensor(room, dtype=torch.int32, device="cuda")
        elif what == "fork":
            a = rng.randrange(B)
            par = [a if rng.random() < 0.5 else b for b in range(B)]
            m.fork(par)
            pool.fork(par)
        elif what == "reorder":
            par = [rng.randrange(-1, B) for _ in range(B)]
            m.fork(par)
            pool.fork(torch.tensor(par, dtype=torch.int32, device="cuda"))
        else:
            gone = [b for b in range(B) if rng.random() < 0.3]
            m.fork([-1 if b in gone else b for b in range(B)])
            pool.free(gone)
        m.same(pool)
        assert pool.free_pages() == int((m.refs == 0).sum())
    assert L.device_error() == 0


@pytest.mark.parametrize("B,H,pages", [(3, 2, 40), (64, 8, 9001)])
def test_fork_of_full_and_part_pages(kv, PagePool, L, B, H, pages):
    """Lengths at and beside the page border, more pages than one round of the ranking."""
    P = 256
    for n in (1, P - 1, P, P + 1, 3 * P - 128, 4 * P):
        m = Model(B, H, 4, pages, P, "ref", 128, kv)
        ids = np.random.RandomState(n).permutation(pages)
        k = -(-n // P)
        m.table[0, :, :k] = ids[:H * k].reshape(H, k)
        m.lengths[0] = n
        # pages that another owner holds are never handed out
        owned = (np.random.RandomState(n + 1).rand(pages) < 0.5).astype(np.int64) * (pages > 100)
        m.count(owned)
        pool = m.upload(kv, PagePool, "ref", 128, torch.from_numpy(m.refs).int().cuda())
        m.fork([0] * B, owned)
        pool.fork([0] * B)
        m.same(pool)
        pool.fork([0] * B)  # the copies are given back and taken again
        m.same(pool)
    assert L.device_error() == 0


def test_no_pages_left(kv, PagePool, L):
    m = Model(4, 2, 3, 9, 128, "ref", 128, kv)
    m.reserve([130, 0, 0, 0])
    m.lengths[0] = 130
    pool = m.upload(kv, PagePool, "ref", 128)
    assert m.fork([0, 0, 0, 0])  # five free pages for six copies
    pool.fork([0, 0, 0, 0])
    assert L.device_error() == L.DEVERR_CAPACITY
    m.same(pool)
    assert m.reserve([1, 127, 300, 0])  # none free, and one row too short
    pool.reserve(300, torch.tensor([1, 127, 300, 0]))
    assert L.device_error() == L.DEVERR_CAPACITY
    m.same(pool)
    pool.free([1, 2, 3])
    m.fork([0, -1, -1, -1])
    m.same(pool)
    assert L.device_error() == 0


def test_bad_ids_are_flagged_and_skipped(kv, PagePool, L):
    m = Model(2, 1, 3, 8, 128, "ref", 128, kv)
    m.reserve([200, 0])
    m.lengths[0] = 200
    pool = m.upload(kv, PagePool, "ref", 128)
    pool.fork([0, 5])  # no such sequence
    assert L.device_error() == L.DEVERR_BAD_PAGE
    m.fork([0, -1])
    m.same(pool)
    pool.store.page_table[0, 0] = 99  # an id outside the pool
    pool.fork([0, 0])
    assert L.device_error() == L.DEVERR_BAD_PAGE
    assert pool.store.page_table.tolist() == [[-1, 1, -1], [-1, 2, -1]]


@pytest.mark.parametrize("fmt,group,P", [("ref", 64, 128), ("fp16min", 32, 384)])
@pytest.mark.parametrize("B,H", [(1, 1), (6, 2), (33, 8)])
def test_compact(kv, PagePool, L, fmt, group, P, B, H):
    rng = np.random.RandomState(B)
    lens = [int(rng.randint(0, 7 * P)) if b % 4 else 3 * P for b in range(B)]
    m = Model(B, H, 8, B * H * 9, P, fmt, group, kv)
    m.refs[::3] = 1  # scattered
    m.reserve(lens)
    m.lengths[:] = lens
    m.count()
    m.fork([b if b % 3 else max(0, b - 2) for b in range(B)])
    pool = m.upload(kv, PagePool, fmt, group)
    pool.reserve(P)  # pages behind the length: they move, their bytes do not
    m.reserve([P] * B)
    m.same(pool)
    live, new = {}, np.full((B * H, 10), -1, np.int64)
    flat = m.table.reshape(B * H, 8)
    into = Model(B, H, 10, len(set(flat[flat >= 0])) + 2, P, fmt, group, kv)
    into.pool[:] = 9
    for u in range(B * H):
        for i in range(8):
            page = flat[u, i]
            if page >= 0:
                if page not in live:
                    live[page] = len(live)
                    if i * P < m.lengths[u // H]:
                        into.pool[live[page]] = m.pool[page]
                new[u, i] = live[page]
    into.table, into.lengths = new.reshape(B, H, 10), m.lengths
    start = Model(B, H, 10, into.pages, P, fmt, group, kv)
    start.pool[:] = 9
    start.table[:] = 0
    to = start.upload(kv, PagePool, fmt, group)
    into.count()
    for _ in range(2):
        pool.compact(to)
        into.same(to)
        m.same(pool)
    assert L.device_error() == 0
    small = Model(B, H, 8, max(1, len(live) - 1), P, fmt, group, kv).upload(kv, PagePool, fmt, group)
    pool.compact(small)
    assert L.device_error() == (L.DEVERR_CAPACITY if len(live) > 1 else 0)
    t = small.store.page_table.cpu().numpy()
    assert np.array_equal(t, np.where(new[:, :8] < max(1, len(live) - 1), new[:, :8], -1))


def test_refusals(kv, PagePool):
    plain = kv.Int4KVStore(2, 2, 256)
    with pytest.raises(ValueError):
        PagePool(plain)
    pool = PagePool(kv.Int4KVStore(2, 2, 512, num_pages=8))
    for bad in ([0], [0, 1, 2], torch.zeros(2), torch.zeros(1, 2, dtype=torch.int32)):
        with pytest.raises(ValueError):
            pool.fork(bad)
    with pytest.raises(ValueError):
        pool.free([2])
    with pytest.raises(ValueError):
        PagePool(pool.store, torch.zeros(7, dtype=torch.int32, device="cuda"))
    from hetero_kvcache_optimizer_b200 import _lib
    for tokens in (-1, 513):
        with pytest.raises(_lib.HkvError):
            pool.reserve(tokens)
    with pytest.raises(ValueError):
        pool.compact(PagePool(kv.Int4KVStore(2, 2, 512, num_pages=8, group=64)))
    with pytest.raises(_lib.HkvError):  # into itself
        pool.compact(pool)
    with pytest.raises(_lib.HkvError):  # rows too short
        pool.compact(PagePool(kv.Int4KVStore(2, 2, 256, num_pages=8)))
    with pytest.raises(ValueError):
        kv.Int4KVStore.wrap(pool.store.pool[:, :-1], None, pool.store.lengths, 2)
    with pytest.raises(ValueError):
        kv.Int4KVStore.wrap(pool.store.pool, pool.store.page_table[:2], pool.store.lengths, 2)


def test_captured_steps_replay(kv, PagePool, L):
    """A step that reserves, and a beam reorder, each captured once and replayed."""
    m = Model(3, 2, 5, 40, 128, "fp16min", 64, kv)
    m.reserve([100, 150, 1])
    m.lengths[:] = [100, 150, 1]
    pool = m.upload(kv, PagePool, "fp16min", 64)
    par = torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")
    keep = {k: v.clone() for k, v in (("t", pool.store.page_table), ("l", pool.store.lengths), ("r", pool.refs))}
    s = torch.cuda.Stream()
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1, stream=s):
        pool.reserve(40)
        pool.store.lengths += 40
    with torch.cuda.graph(g2, stream=s):
        pool.fork(par)
    torch.cuda.synchronize()
    assert torch.equal(keep["t"], pool.store.page_table) and torch.equal(keep["r"], pool.refs)
    for step, p in enumerate([[0, 0, 1], [2, 1, 1], [1, -1, 1], [0, 0, 0]]):
        g1.replay()
        m.reserve([40] * 3)
        m.lengths += 40
        m.same(pool)
        par.copy_(torch.tensor(p, dtype=torch.int32))
        g2.replay()
        m.fork(p)
        m.same(pool)
    assert L.device_error() == 0
