"""PagedKVCache.extend: blocks for several requests' next tokens, on the host."""
import numpy as np
import pytest

from rngd_pd_amd.engines.paged_cache import PagedKVCache
from tests import _chunk_ref as ref


@pytest.fixture
def cache():
    return PagedKVCache(n_layers=1, num_blocks=20, n_kv_heads=1, head_dim=32, device="cpu", seed=2)


def test_tables_and_ids_make_the_requests_tables(cache):
    cache.allocate("a", 40)                             # three blocks, 33 tokens in use
    a = cache.blocks("a")
    tables, free = cache.extend([("a", 33, 30), ("b", 0, 17), ("c", 0, 0)])
    assert tables.dtype == np.int32 and tables.shape == (3, 4)
    assert tables[0].tolist() == a + [-1] and (tables[1:] == -1).all()
    got, *_ = ref.chunk_map([33, 0, 0], [30, 17, 0], tables, free.tolist(), 47)
    assert cache.blocks("a") == got[0].tolist() and cache.blocks("a")[:3] == a
    assert cache.blocks("b") == got[1, :2].tolist() and cache.blocks("c") == []
    assert cache.alloc.free_blocks() == 20 - 6
    # Blocks that are there already are taken again, in order.
    tables, free = cache.extend([("b", 3, 20), ("a", 16, 1)])
    assert free.tolist() == cache.blocks("b")[1:] + cache.blocks("a")[1:2]
    assert tables[0, 0] == cache.blocks("b")[0] and cache.alloc.free_blocks() == 20 - 6


def test_refusals_change_nothing(cache):
    cache.allocate("a", 40)
    cache.fork("a", ["b"], 32)
    before = (cache.blocks("a"), cache.blocks("b"), cache.alloc.free_blocks())
    for bad in ([("a", 49, 1)], [("a", 30, 1)], [("a", 40, 1), ("a", 41, 1)], [("x", 1, 4)],
                [("a", -1, 1)], [("a", 40, -1)]):
        with pytest.raises(ValueError):
            cache.extend(bad)
    with pytest.raises(MemoryError):
        cache.extend([("a", 40, 16), ("x", 0, 400)])
    assert before == (cache.blocks("a"), cache.blocks("b"), cache.alloc.free_blocks())
    assert "x" not in cache._tables
    cache.extend([("a", 32, 9), ("b", 32, 1)])          # behind what they share
    cache.drop_before("a", 48)
    with pytest.raises(ValueError, match="dropped"):
        cache.extend([("a", 40, 20)])
