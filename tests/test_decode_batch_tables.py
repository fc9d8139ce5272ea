"""The block tables that BatchDecodeAttention keeps between steps follow what the
cache does in between (host logic on a CPU cache)."""
import pytest

from rngd_pd_amd.engines import paged_cache as pc
from rngd_pd_amd.engines.decode_batch import BatchDecodeAttention


@pytest.fixture
def engine(monkeypatch):
    def copy(k, v, src, dst, stream=None):
        k[:, list(dst)], v[:, list(dst)] = k[:, list(src)], v[:, list(src)]
    monkeypatch.setattr(pc._pages, "copy_blocks", copy)
    cache = pc.PagedKVCache(n_layers=1, num_blocks=16, n_kv_heads=1, head_dim=32, device="cpu")
    eng = BatchDecodeAttention(cache, n_q_heads=1)
    for r, n in (("gone", 40), ("a", 20), ("b", 5)):
        cache.allocate(r, n)
        eng.admit_loaded(r, n)
    return eng


def _check(eng, ids):
    tables, ctx, _ = eng.prepare(ids)
    for row, r in zip(tables.tolist(), ids):
        blocks = eng.cache.blocks(r)
        assert row[:len(blocks)] == blocks and set(row[len(blocks):]) <= {-1}
    assert ctx.tolist() == [eng.positions[r] + 1 for r in ids]
    return tables


def test_compact_between_steps(engine):
    ids = ["a", "b"]
    engine.retire("gone")
    before = _check(engine, ids)
    assert engine.cache.compact() == 3
    after = _check(engine, ids)
    assert before.tolist() != after.tolist()
    free = set(engine.cache.alloc._free)
    assert not free & {b for row in after.tolist() for b in row}


def test_request_replaced_at_the_cache(engine):
    ids = ["a", "b"]
    _check(engine, ids)
    engine.cache.free("a")                              # the same name, the same length, other blocks
    engine.cache.allocate("c", 1)
    engine.cache.allocate("a", 21)
    _check(engine, ids)
    engine.cache.free("a")
    engine.cache.allocate("d", 1)
    engine.cache.fork("gone", ["a"], 20)
    _check(engine, ids)


def test_blocks_dropped_at_the_cache(engine):
    ids = ["gone", "b"]
    _check(engine, ids)
    assert engine.cache.drop_before("gone", 16) == 1
    assert _check(engine, ids)[0, 0] == -1


def test_table_is_kept_while_nothing_changes(engine):
    ids = ["a", "b"]
    first = _check(engine, ids)
    engine.cache.allocate("later", 30)                  # of no concern to these two
    engine.advance(ids)
    assert _check(engine, ids) is first
    assert engine.cache.compact() == 0
    assert _check(engine, ids) is first
