"""norm_rope in place is row by row: the same memory under other strides is refused before
anything is launched (no GPU: the addresses are never read)."""
import pytest

FAKE = 1 << 20


@pytest.fixture(scope="module")
def L():
    from hetero_kvcache_optimizer_b200.csrc import build
    build.build()
    from hetero_kvcache_optimizer_b200 import _lib
    _lib.load()
    return _lib


def call(L, x, y, B, T):
    return L.load().hkv_norm_rope(x, None, y, None, 1, B, T, 128, 0, 0, 0, 1e-6, 0, 32, 0, 0, 0, 0, 0, 0, 0, None)


@pytest.mark.parametrize("strides", [(4096, 512, 128), (8192, 128, 1024), (4096, 128, 2048)])
def test_other_strides_over_the_same_memory(L, strides):
    x = L.HkvRows(FAKE, 4096, 128, 1024, 8, 0)
    assert call(L, x, L.HkvRows(FAKE, *strides, 8, 0), 2, 4) == L.HKV_ERR_ARG


def test_strides_of_single_rows_do_not_matter(L):
    x = L.HkvRows(FAKE, 4096, 128, 1024, 8, 0)
    assert call(L, x, L.HkvRows(FAKE, 1, 128, 1, 8, 0), 1, 0) == L.HKV_OK  # no tokens: nothing is launched
    one = L.HkvRows(FAKE, 4096, 128, 1024, 1, 0)
    assert call(L, one, L.HkvRows(FAKE, 5, 7, 9, 1, 0), 1, 0) == L.HKV_OK
