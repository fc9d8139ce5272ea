"""Forked, trimmed and compacted block tables of the paged cache: host logic, with
the copies done on a CPU cache by plain indexing."""
import numpy as np
import pytest
import torch

from rngd_pd_amd.engines import paged_cache as pc


@pytest.fixture
def cache(monkeypatch):
    log = []

    def copy(k, v, src, dst, stream=None):
        src, dst = list(src), list(dst)
        assert len(set(dst)) == len(dst) and not set(src) & set(dst)
        k[:, dst], v[:, dst] = k[:, src], v[:, src]
        log.append((src, dst))
    monkeypatch.setattr(pc._pages, "copy_blocks", copy)
    c = pc.PagedKVCache(n_layers=2, num_blocks=24, n_kv_heads=1, head_dim=32, device="cpu", seed=1)
    c.k.normal_()
    c.v.normal_()
    c.log = log
    return c


def _content(c, req, n):
    """The first n tokens of a request, K as rows."""
    b = c.blocks(req)[:-(-n // 16)]
    k = pc.k_block_rows(c.k[:, b]).permute(0, 1, 3, 2, 4).reshape(2, -1, 1, 32)[:, :n]
    v = c.v[:, b].permute(0, 1, 4, 2, 3).reshape(2, -1, 1, 32)[:, :n]
    return torch.cat([k, v], -1)


def test_fork_shares_full_blocks_and_copies_the_last(cache):
    cache.allocate("a", 40)
    want = _content(cache, "a", 37)
    cache.fork("a", ["b", "c"], 37)
    a, b, c = (cache.blocks(r) for r in "abc")
    assert b[:2] == a[:2] == c[:2] and len({a[2], b[2], c[2]}) == 3
    assert cache.log == [([a[2], a[2]], [b[2], c[2]])]
    assert torch.equal(_content(cache, "b", 37), want) and torch.equal(_content(cache, "c", 37), want)
    assert cache.alloc.free_blocks() == 24 - 5
    cache.ensure("b", 70)
    cache.free("a")
    assert cache.alloc.free_blocks() == 24 - 6          # b holds 5, c one of its own
    assert torch.equal(_content(cache, "b", 37), want)
    cache.free("b")
    assert torch.equal(_content(cache, "c", 37), want) and cache.alloc.free_blocks() == 24 - 3
    cache.free("c")
    assert cache.alloc.free_blocks() == 24 and not cache._shared
    assert sorted(cache.alloc.allocate(24)) == list(range(24))


def test_fork_edges(cache):
    cache.allocate("a", 32)
    cache.fork("a", ["b"], 32)                          # whole blocks: nothing is copied
    cache.fork("b", ["c"], 0)
    assert cache.log == [] and cache.blocks("b") == cache.blocks("a") and cache.blocks("c") == []
    cache.fork("b", [], 20)
    assert cache.log == []
    with pytest.raises(KeyError):
        cache.fork("a", ["b"], 16)
    with pytest.raises(KeyError):
        cache.fork("a", ["x", "x"], 16)
    with pytest.raises(KeyError):
        cache.fork("nobody", ["x"], 1)
    for n in (33, -1):
        with pytest.raises(ValueError):
            cache.fork("a", ["x"], n)
    cache.allocate("big", 22 * 16)
    with pytest.raises(MemoryError):
        cache.fork("a", ["x"], 17)
    assert "x" not in cache._tables and cache.alloc.free_blocks() == 0
    cache.free("big")
    cache.free("a")
    cache.free("b")
    assert cache.alloc.free_blocks() == 24


def test_frames_refuse_shared_and_dropped_blocks(cache):
    cache.allocate("a", 48)
    cache.fork("a", ["b"], 40)
    with pytest.raises(ValueError, match="shares"):
        cache.write_frame("b", None, 20, 64)
    cache.drop_before("a", 16)
    with pytest.raises(ValueError, match="dropped"):
        cache.read_frame("a", 20, 64)
    with pytest.raises(ValueError, match="dropped"):
        cache.write_frame("a", None, 1, 64)


def test_drop_before_keeps_sinks_and_the_window(cache):
    cache.allocate("a", 100)                            # blocks 0..6
    b = cache.blocks("a")
    assert cache.drop_before("a", 15) == 0
    assert cache.drop_before("a", 50, keep=4) == 2      # tokens 16..47; block 0 holds the sinks
    assert cache.blocks("a") == [b[0], -1, -1] + b[3:]
    assert cache.table("a").tolist() == [b[0], -1, -1] + b[3:]
    assert cache.alloc.free_blocks() == 24 - 5
    assert cache.drop_before("a", 50, keep=4) == 0      # again: nothing left
    assert cache.drop_before("a", -7, keep=-3) == 0
    assert cache.drop_before("a", 64, keep=16) == 1
    cache.ensure("a", 130)
    assert len(cache.blocks("a")) == 9
    cache.fork("a", ["f"], 100)                         # dropped entries stay dropped
    assert cache.blocks("f")[:6] == [b[0], -1, -1, -1, b[4], b[5]]
    assert cache.drop_before("a", 96, keep=0) == 3      # two of them shared with f
    cache.free("a")
    assert cache.alloc.free_blocks() == 24 - 4
    cache.free("f")
    assert sorted(cache.alloc.allocate(24)) == list(range(24))
    with pytest.raises(KeyError):
        cache.drop_before("a", 10)


def test_views_refuse_shared_and_dropped_blocks(cache):
    """A view's blocks are written by a transport: nobody else may hold them."""
    cache.allocate("a", 40)
    cache.view("a", 40, 48)
    cache.fork("a", ["b"], 32)
    with pytest.raises(ValueError, match="shares"):
        cache.view("a", 40, 48)
    cache.free("b")
    cache.drop_before("a", 16)
    with pytest.raises(ValueError, match="dropped"):
        cache.view("a", 40, 48)


def test_fork_of_a_dropped_last_block_is_refused(cache):
    cache.allocate("a", 48)
    cache.drop_before("a", 48)
    with pytest.raises(ValueError, match="dropped"):
        cache.fork("a", ["b"], 40)


def test_compact(cache):
    rng = np.random.default_rng(0)
    for i in range(10):
        cache.allocate(i, int(rng.integers(1, 33)))
    for i in (1, 3, 4, 8):
        cache.free(i)
    cache.fork(0, ["f"], 1)
    cache.fork(2, ["g"], 16)
    want = {r: _content(cache, r, 1) for r in cache._tables}
    shared = sum(cache._shared.values())
    held = {b for t in cache._tables.values() for b in t}
    cache.table(0)
    moved = cache.compact()
    now = {b for t in cache._tables.values() for b in t}
    assert now == set(range(len(held))) and moved == len(held - now) > 0
    assert sum(cache._shared.values()) == shared
    for r, x in want.items():
        assert torch.equal(_content(cache, r, 1), x)
    assert cache.table(0).tolist() == cache.blocks(0)
    assert cache.compact() == 0
    assert cache.alloc.allocate(2) == [len(held), len(held) + 1]
    for r in list(cache._tables):
        cache.free(r)
    assert cache.alloc.free_blocks() == 24 - 2


def test_compact_leaves_blocks_that_no_table_holds(cache):
    loose = cache.alloc.allocate(3)                     # a caller's own
    cache.allocate("a", 50)
    cache.compact()
    assert not set(loose) & set(cache.blocks("a"))
    assert sorted(cache.blocks("a")) == sorted(set(range(24)) - set(loose))[:4]
