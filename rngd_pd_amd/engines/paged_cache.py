"""Paged decode-side KV cache and its block allocator.

Replaces the reference's per-stream S-wide lanes ([nl, B, NKV, HD, S] /
[nl, B, NKV, S, HD], engines/decode_batch.py:305-330) with fixed 16-token
blocks shared by every request: a request holds ceil(tokens/16) blocks in any
order, listed in its block table (the same table for every layer). Capacity
is then set by HBM, not by a compiled S.

Layout (bf16): K [L, num_blocks, Hkv, 16, D] and V [L, num_blocks, Hkv, D, 16]
(dim rows, contiguous tokens). A K block holds its 16 tokens x D dims as
16-byte units of 8 dims of one token, tiled in the order the decode-attention
QK tiles read them (k_block_index); V is already in the order the PV tiles
read. k_block_rows / k_block_tiled convert K blocks to and from token rows.

Requests may share blocks: fork gives new requests the full blocks of a prefix
(counted; the partly filled one is copied), and a block returns to the pool with
its last holder. drop_before returns the blocks that a sliding window has left
behind (their table entries become -1, which attention under that window does not
read), compact moves what is held to the lowest ids.
"""
import threading

import numpy as np
import torch

from ..kernels import handoff as _h
from ..kernels import pages as _pages

BLOCK = 16


def k_block_index(head_dim, device=None):
    """int64 [16, head_dim]: position of (token slot, dim) inside one K block.

    Unit (16 bytes, 8 dims) of slot s and dims d0..d0+7 is
    ((t * head_dim/32 + d0/32) * 4 + (d0/8) % 4) * 8 + j8 with t = bit 2 of s
    and j8 = (s // 8) * 4 + s % 4 -- the order of rngdpd.h's paged cache."""
    if head_dim % 32:
        raise ValueError(f"head_dim {head_dim} is not a multiple of 32")
    s = torch.arange(BLOCK, device=device).view(BLOCK, 1)
    d = torch.arange(head_dim, device=device).view(1, head_dim)
    unit = ((((s >> 2) & 1) * (head_dim // 32) + d // 32) * 4 + (d // 8) % 4) * 8 \
        + (s >> 3) * 4 + (s & 3)
    return unit * 8 + d % 8


def k_block_rows(blocks):
    """K blocks [..., 16, D] in cache order -> token rows [..., 16, D]."""
    D = blocks.shape[-1]
    flat = blocks.reshape(*blocks.shape[:-2], BLOCK * D)
    return flat[..., k_block_index(D, blocks.device)]


def k_block_tiled(rows):
    """Token rows [..., 16, D] -> K blocks [..., 16, D] in cache order."""
    D = rows.shape[-1]
    out = torch.empty(*rows.shape[:-2], BLOCK * D, dtype=rows.dtype, device=rows.device)
    out[..., k_block_index(D, rows.device).reshape(-1)] = rows.reshape(*rows.shape[:-2], BLOCK * D)
    return out.view(rows.shape)


class BlockAllocator:
    """Free list of block ids. ``seed`` shuffles the initial order (a permuted
    block table, as the handoff workloads use)."""

    def __init__(self, num_blocks, seed=None):
        ids = np.arange(num_blocks, dtype=np.int64)
        if seed is not None:
            ids = np.random.default_rng(seed).permutation(num_blocks)
        self._free = [int(i) for i in ids[::-1]]
        self.num_blocks = num_blocks
        self._lock = threading.Lock()

    def free_blocks(self):
        return len(self._free)

    def allocate(self, n):
        with self._lock:
            if n > len(self._free):
                raise MemoryError(f"paged cache exhausted: need {n} blocks, {len(self._free)} free")
            return [self._free.pop() for _ in range(n)]

    def release(self, blocks):
        with self._lock:
            self._free.extend(reversed(list(blocks)))

    def repack(self, plan):
        """Calls ``plan`` on the free ids in increasing order, for the ids that
        become free in exchange for as many of them, the lowest; returns what it
        returned. Low ids are handed out first from then on."""
        with self._lock:
            free = sorted(self._free)
            freed = plan(free)
            self._free = sorted(free[len(freed):] + list(freed), reverse=True)
            return freed


class PagedKVCache:
    """One paged K/V cache for all layers plus per-request block tables."""

    def __init__(self, n_layers, num_blocks, n_kv_heads=8, head_dim=128, device="cuda",
                 seed=None, dtype=torch.bfloat16):
        self.n_layers, self.num_blocks = n_layers, num_blocks
        self.n_kv_heads, self.head_dim = n_kv_heads, head_dim
        self.device = torch.device(device)
        self.k = torch.zeros((n_layers, num_blocks, n_kv_heads, BLOCK, head_dim), dtype=dtype,
                             device=self.device)
        self.v = torch.zeros((n_layers, num_blocks, n_kv_heads, head_dim, BLOCK), dtype=dtype,
                             device=self.device)
        self.alloc = BlockAllocator(num_blocks, seed)
        self._tables = {}          # req_id -> [block ids]
        self._dev_tables = {}      # req_id -> device int32 tensor
        self._shared = {}          # block -> holders beyond the first
        # Raised whenever an entry of a table is replaced or a table goes; tables that
        # only grow keep it. What is kept from tables holds for one generation.
        self.generation = 0
        self._lock = threading.Lock()

    # -- block tables ---------------------------------------------------------
    def allocate(self, req_id, n_tokens):
        """Blocks for the first ``n_tokens`` tokens of a new request."""
        need = (n_tokens + BLOCK - 1) // BLOCK
        with self._lock:
            if req_id in self._tables:
                raise KeyError(f"request {req_id!r} already holds blocks")
            self._tables[req_id] = self.alloc.allocate(need)
            self._dev_tables.pop(req_id, None)
        return self.table(req_id)

    def ensure(self, req_id, n_tokens):
        """Grow the request's table to cover ``n_tokens`` tokens (decode growth)."""
        need = (n_tokens + BLOCK - 1) // BLOCK
        with self._lock:
            have = self._tables.setdefault(req_id, [])
            if need > len(have):
                have.extend(self.alloc.allocate(need - len(have)))
                self._dev_tables.pop(req_id, None)

    def extend(self, chunks):
        """Blocks for the next tokens of several requests, as chunk_map takes them:
        ``chunks`` holds (req_id, tokens in the cache before, new ones) of different
        requests, one without tokens and blocks being a new request. Returns (tables,
        free): host int32 [R, max_blocks] with the entries of the tokens that are there
        (the others -1), and the ids that the new tokens' entries take, request after
        request. Nothing changes if the blocks do not suffice."""
        chunks = [(r, int(past), int(n)) for r, past, n in chunks]
        if len({r for r, _, _ in chunks}) != len(chunks):
            raise ValueError("a request comes twice")
        with self._lock:
            grow = []
            for r, past, n in chunks:
                have = self._tables.get(r, [])
                if past < 0 or n < 0 or len(have) * BLOCK < past:
                    raise ValueError(f"{r!r} holds {len(have)} blocks, fewer than {past} tokens, "
                                     f"or its {n} new ones are negative")
                # The blocks that are written: the partly filled one and those behind it.
                last = -(-(past + n) // BLOCK)
                written = have[past // BLOCK:last] if n else []
                if any(b < 0 for b in written):
                    raise ValueError(f"{r!r} has dropped blocks of tokens {past} to {past + n - 1}")
                if any(b in self._shared for b in written):
                    raise ValueError(f"{r!r} shares blocks of tokens {past} to {past + n - 1}")
                grow.append(max(0, last - len(have)))
            ids = self.alloc.allocate(sum(grow))
            tables = np.full((len(chunks), max([1] + [-(-(p + n) // BLOCK) for _, p, n in chunks])),
                             -1, np.int32)
            free, at = [], 0
            for i, ((r, past, n), g) in enumerate(zip(chunks, grow)):
                have = self._tables.setdefault(r, [])
                have.extend(ids[at:at + g])
                at += g
                if g:
                    self._dev_tables.pop(r, None)
                held = -(-past // BLOCK)
                tables[i, :held] = have[:held]
                free += have[held:-(-(past + n) // BLOCK)]
        return tables, np.asarray(free, np.int32)

    def free(self, req_id):
        with self._lock:
            if req_id in self._tables:
                self.generation += 1
            blocks = self._tables.pop(req_id, [])
            self._dev_tables.pop(req_id, None)
            self.alloc.release(self._let_go(blocks))

    def _let_go(self, blocks):
        """Those of a holder's blocks that nobody else holds; the others lose it."""
        last = []
        for b in blocks:
            more = self._shared.get(b, 0)
            if more > 1:
                self._shared[b] = more - 1
            elif more:
                del self._shared[b]
            elif b >= 0:
                last.append(b)
        return last

    # -- sharing and moving blocks ----------------------------------------------
    def fork(self, req_id, new_ids, num_tokens, stream=None):
        """New requests ``new_ids`` that start with the first ``num_tokens`` tokens
        of ``req_id``: its full blocks are shared, a partly filled one is copied
        to a block of each (one launch, on ``stream`` or the current one, ordered
        after what was written there). Shared blocks are not written again: a
        request's later tokens go to blocks of its own (ensure)."""
        new_ids = list(new_ids)
        full, part = divmod(num_tokens, BLOCK)
        with self._lock:
            have = self._tables[req_id]
            if num_tokens < 0 or len(have) < full + (part > 0):
                raise ValueError(f"{req_id!r} holds {len(have)} blocks, fewer than {num_tokens} tokens")
            if part and have[full] < 0:
                raise ValueError(f"{req_id!r} has dropped the block of token {num_tokens - 1}")
            if len(set(new_ids)) != len(new_ids) or any(r in self._tables for r in new_ids):
                raise KeyError(f"{new_ids} are not all new, different requests")
            own = self.alloc.allocate(len(new_ids)) if part else []
            try:
                if own:
                    _pages.copy_blocks(self.k, self.v, [have[full]] * len(own), own, stream=stream)
            except BaseException:
                self.alloc.release(own)
                raise
            for i, r in enumerate(new_ids):
                self._tables[r] = have[:full] + own[i:i + 1]
                self._dev_tables.pop(r, None)
            for b in have[:full]:
                if b >= 0 and new_ids:
                    self._shared[b] = self._shared.get(b, 0) + len(new_ids)

    def drop_before(self, req_id, num_tokens, keep=0):
        """Return the request's blocks that hold only tokens from ``keep`` on and
        before ``num_tokens`` (behind a sliding window, beside its sinks) to the
        pool; their table entries become -1. How many there were. No step that
        still reads them may be queued where another stream could fill them."""
        with self._lock:
            have = self._tables[req_id]
            gone = [j for j in range(-(-max(keep, 0) // BLOCK), min(num_tokens // BLOCK, len(have)))
                    if have[j] >= 0]
            if gone:
                self.generation += 1
                free = self._let_go([have[j] for j in gone])
                for j in gone:
                    have[j] = -1
                self._dev_tables.pop(req_id, None)
                self.alloc.release(free)
            return len(gone)

    def compact(self, stream=None):
        """Move held blocks onto the lowest free ids until no free id lies below a
        held one's; returns how many moved. Tables change: device tables and
        graphs made before are stale (BatchDecodeAttention.prepare makes its own
        anew), and no other stream may be using the cache."""
        with self._lock:
            moved = {}

            def plan(free):
                held = sorted({b for t in self._tables.values() for b in t if b >= 0})
                while len(moved) < len(free) and held and held[-1] > free[len(moved)]:
                    moved[held.pop()] = free[len(moved)]
                if moved:
                    _pages.copy_blocks(self.k, self.v, list(moved), list(moved.values()),
                                       stream=stream)
                return list(moved)
            self.alloc.repack(plan)
            if not moved:
                return 0
            self.generation += 1
            for t in self._tables.values():
                t[:] = [moved.get(b, b) for b in t]
            self._shared = {moved.get(b, b): n for b, n in self._shared.items()}
            self._dev_tables.clear()
            return len(moved)

    def blocks(self, req_id):
        return list(self._tables[req_id])

    def table(self, req_id):
        """Device int32 block table of the request."""
        with self._lock:
            t = self._dev_tables.get(req_id)
            if t is None:
                t = torch.tensor(self._tables[req_id] or [0], dtype=torch.int32, device=self.device)
                self._dev_tables[req_id] = t
            return t

    def batch_tables(self, req_ids, max_blocks=None):
        """[B, max_blocks] device int32 tables (unused entries -1)."""
        rows = [self._tables[r] for r in req_ids]
        width = max_blocks or max(1, max(len(r) for r in rows))
        arr = np.full((len(rows), width), -1, np.int32)
        for i, r in enumerate(rows):
            arr[i, :len(r)] = r
        return torch.from_numpy(arr).to(self.device)

    # -- frames in and out ----------------------------------------------------
    def write_frame(self, req_id, frame, num_tokens, S, stream=None):
        """Scatter tokens 0..num_tokens-1 of a transport frame [L, 2, Hkv*D*S]."""
        self._whole(req_id, num_tokens, write=True)
        _h.scatter_paged(frame, self.table(req_id), num_tokens, S, self.k, self.v, stream=stream)

    def read_frame(self, req_id, num_tokens, S, frame=None, stream=None):
        """The request's S-wide transport frame (zero for t >= num_tokens)."""
        self._whole(req_id, num_tokens)
        return _h.gather_paged(self.k, self.v, self.table(req_id), num_tokens, S, frame=frame,
                               stream=stream)

    def _whole(self, req_id, num_tokens, write=False):
        """Refuses a frame of blocks that were dropped, or to be written over
        blocks that others hold."""
        blocks = self._tables[req_id][:-(-num_tokens // BLOCK)]
        if -1 in blocks:
            raise ValueError(f"{req_id!r} has dropped blocks of its first {num_tokens} tokens")
        if write and self._shared and any(b in self._shared for b in blocks):
            raise ValueError(f"{req_id!r} shares blocks of its first {num_tokens} tokens")

    def view(self, req_id, num_tokens, S):
        """What the connector's decode side registers for one request."""
        return PagedRequestView(self, req_id, num_tokens, S)


class PagedRequestView:
    """One request's slice of a PagedKVCache, as registered with the connector."""

    def __init__(self, cache, req_id, num_tokens, S):
        self.cache, self.req_id = cache, req_id
        self.num_tokens, self.S = num_tokens, S
        if req_id not in cache._tables:
            cache.allocate(req_id, num_tokens)
        else:
            cache._whole(req_id, num_tokens, write=True)

    @property
    def table(self):
        return self.cache.table(self.req_id)
