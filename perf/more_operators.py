"""More operators whose speed counts, as cases that can be timed one by one
against their plain forms (perf/operators.py has the earlier ones).

Five operators that take several requests' next tokens (pieces of prompts, a
draft's tokens, single ones) through a layer over the paged cache of 16-token
blocks, its projections in 8 bits:

  map        from the requests' lengths: their block tables grown from a list of
             free blocks, and every token's position and cache slot;
  write      RoPE at those positions, K and V into those slots;
  attention  of every new token over all that its request has in the cache;
  norm       RMSNorm with the residual's addition, out in 8 bits (e4m3) with a
             scale for each 128 columns of a row;
  linear     the product of such rows with weights of 8 bits that have a scale
             for each block of 128 x 128.

Where ``own`` is false run() computes the plain form in elementary torch
operations; where it is true it calls the framework. listed() gives the named
cases, draw(rng) another one of the same ranges, prepare(case, seed) what a
program holds before the call, work(case) the bytes and operations a pass cannot
do without, exact(case, seed) the result in 64 bits. The shapes are
Llama-3.1-8B's (hidden 4096, 32 query and 8 KV heads of 128, inner width 14336)
and others of the kind.
"""
import math
import random

import numpy as np
import torch

own = False

BF16 = torch.bfloat16
FP8 = torch.float8_e4m3fn
HEAD = 128
BLOCK = 16
GROUP = 128                 # columns per scale
EPS = 1e-5
TOP = 448.0                 # the largest e4m3 value
LEAST = 2.0 ** -100         # a group's largest value counts as at least this


# ---- cases ------------------------------------------------------------------
def listed():
    return [
        # The decode batch of 64, each request one token further.
        {"name": "map_64_single", "kind": "map", "R": 64, "new_lo": 1, "new_hi": 1, "past_hi": 16000,
         "width": 1024, "spare": 0, "len_seed": 0},
        # A prefill step: pieces of 48 prompts, in a launch sized for 16384 tokens.
        {"name": "map_48_chunks", "kind": "map", "R": 48, "new_lo": 1, "new_hi": 500,
         "past_hi": 4000, "width": 512, "spare": 1000, "len_seed": 1},
        # The single tokens of 16 streams.
        {"name": "write_16", "kind": "write", "N": 16, "hq": 32, "hkv": 8, "pos_hi": 16000,
         "unplaced": 0, "len_seed": 0},
        # The largest step's tokens, padding behind them.
        {"name": "write_8192", "kind": "write", "N": 8192, "hq": 32, "hkv": 8, "pos_hi": 40000,
         "unplaced": 37, "len_seed": 1},
        # Eight streams whose draft of four tokens is verified beside the last one.
        {"name": "attend_verify", "kind": "attention", "R": 8, "singles": 0, "new_lo": 5,
         "new_hi": 5, "past_lo": 500, "past_hi": 4000, "window": 0, "sinks": 0, "hq": 32, "hkv": 8,
         "len_seed": 2},
        # A user's next turn of 470 tokens on a conversation of 4000.
        {"name": "attend_turn_470", "kind": "attention", "R": 1, "singles": 0, "new_lo": 470,
         "new_hi": 470, "past_lo": 4000, "past_hi": 4000, "window": 0, "sinks": 0, "hq": 32,
         "hkv": 8, "len_seed": 0},
        # 31 streams' single tokens beside a piece of a prompt, as a step with both has them.
        {"name": "attend_mixed_32", "kind": "attention", "R": 32, "singles": 31, "new_lo": 2000,
         "new_hi": 2000, "past_lo": 500, "past_hi": 12000, "window": 0, "sinks": 0, "hq": 32,
         "hkv": 8, "len_seed": 3},
        # The last piece of a long document.
        {"name": "attend_long_4096", "kind": "attention", "R": 1, "singles": 0, "new_lo": 4096,
         "new_hi": 4096, "past_lo": 28000, "past_hi": 28000, "window": 0, "sinks": 0, "hq": 32,
         "hkv": 8, "len_seed": 0},
        # Before the projections of 16 streams' single tokens.
        {"name": "norm_16", "kind": "norm", "T": 16, "H": 4096, "add": True},
        # Of the largest step's tokens.
        {"name": "norm_8192", "kind": "norm", "T": 8192, "H": 4096, "add": True},
        # gate|up for 16 streams' single tokens: the weights' bytes.
        {"name": "linear_16", "kind": "linear", "T": 16, "N": 28672, "K": 4096},
        # gate|up for the largest step's tokens: the products.
        {"name": "linear_8192", "kind": "linear", "T": 8192, "N": 28672, "K": 4096},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["map", "write", "attention", "attention", "attention", "norm", "linear",
                       "linear", "linear"])
    hq, hkv = rng.choice([(32, 8), (32, 8), (64, 8), (16, 2), (8, 8), (28, 4), (40, 8), (32, 2)])
    seed = rng.randrange(1 << 20)
    if kind == "map":
        R = _log_int(rng, 1, 256)
        lo = rng.choice([0, 1, 1])
        return {"kind": kind, "R": R, "new_lo": lo, "new_hi": _log_int(rng, 1, 16384 // R),
                "past_hi": _log_int(rng, 1, 16000), "width": 2048, "spare": rng.randint(0, 300),
                "len_seed": seed}
    if kind == "write":
        N = _log_int(rng, 1, 8192)
        return {"kind": kind, "N": N, "hq": hq, "hkv": hkv, "pos_hi": _log_int(rng, 1, 1000000),
                "unplaced": rng.randint(0, N // 8), "len_seed": seed}
    if kind == "attention":
        R = _log_int(rng, 1, 64)
        singles = rng.choice([0, 0, R // 2, R - 1, R])
        new = 1 if singles == R else _log_int(rng, 1, 4096 // (R - singles))
        past = _log_int(rng, 1, min(28000, 400000 // R))
        if new * (past + new) * hq > 4096 * 28000 * 32 // max(1, R - singles):
            past = 4000
        window = _log_int(rng, 16, 4096) if rng.random() < 0.25 else 0
        return {"kind": kind, "R": R, "singles": singles, "new_lo": rng.randint(1, new),
                "new_hi": new, "past_lo": rng.randint(0, past), "past_hi": past, "window": window,
                "sinks": rng.choice([0, 4, 33]) if window else 0, "hq": hq, "hkv": hkv,
                "len_seed": seed}
    if kind == "norm":
        return {"kind": kind, "T": _log_int(rng, 1, 8192), "H": GROUP * rng.randint(1, 64),
                "add": rng.random() < 0.7}
    N, K = rng.choice([(6144, 4096), (4096, 4096), (28672, 4096), (4096, 14336),
                       (8 * _log_int(rng, 1, 2048), GROUP * _log_int(rng, 1, 64)),
                       (8 * _log_int(rng, 1, 2048), GROUP * _log_int(rng, 1, 64))])
    return {"kind": kind, "T": _log_int(rng, 1, 8192), "N": N, "K": K}


# ---- inputs -----------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _normal(gen, *shape, std=1.0):
    return torch.empty(shape, dtype=BF16, device="cuda").normal_(0.0, std, generator=gen)


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _k_place(D):
    """int64 [16, D]: where a K block keeps (slot, dim) among its 16 D values."""
    s = torch.arange(BLOCK, device="cuda").view(BLOCK, 1)
    d = torch.arange(D, device="cuda").view(1, D)
    unit = ((((s >> 2) & 1) * (D // 32) + d // 32) * 4 + (d // 8) % 4) * 8 + (s >> 3) * 4 + (s & 3)
    return unit * 8 + d % 8


def _blocks(n):
    return -(-n // BLOCK)


def _map_lengths(case):
    rng = random.Random(case["len_seed"])
    return [(rng.randint(0, case["past_hi"]), rng.randint(case["new_lo"], case["new_hi"]))
            for _ in range(case["R"])]


def _prepare_map(case, seed):
    lens, R, W = _map_lengths(case), case["R"], case["width"]
    held = [_blocks(p) for p, _ in lens]
    need = sum(_blocks(p + n) for p, n in lens) - sum(held)
    nb = sum(held) + need + 7
    ids = np.random.default_rng(seed).permutation(nb).astype(np.int32)
    tables, at = np.full((R, W), -1, np.int32), 0
    for r, h in enumerate(held):
        tables[r, :h] = ids[at:at + h]
        at += h
    return {"past": _int32([p for p, _ in lens]), "new": _int32([n for _, n in lens]),
            "tables": torch.from_numpy(tables).cuda(), "free": torch.from_numpy(ids[at:]).cuda(),
            "max_tokens": sum(n for _, n in lens) + case["spare"]}


def _inv_freq():
    return torch.tensor([500000.0 ** (-2 * i / HEAD) for i in range(HEAD // 2)], device="cuda")


def _prepare_write(case, seed):
    gen, N, rng = _gen(seed), case["N"], np.random.default_rng(seed)
    nb = _blocks(N) + 3
    # Runs of tokens in blocks of any order, as requests' tables give them.
    slots = (rng.permutation(nb)[:, None] * BLOCK + np.arange(BLOCK)).reshape(-1)[:N]
    slots = np.roll(slots, 5).astype(np.int32)
    if case["unplaced"]:
        slots[N - case["unplaced"]:] = -1
    first = random.Random(case["len_seed"]).randint(0, case["pos_hi"])
    return {"qkv": _normal(gen, N, (case["hq"] + 2 * case["hkv"]) * HEAD), "inv": _inv_freq(),
            "positions": torch.arange(first, first + N, dtype=torch.int32, device="cuda"),
            "slots": torch.from_numpy(slots).cuda(),
            "k": _normal(gen, nb, case["hkv"], BLOCK, HEAD),
            "v": _normal(gen, nb, case["hkv"], HEAD, BLOCK)}


def _chunk_lengths(case):
    """(tokens in the cache before, new ones) of each request."""
    rng = random.Random(case["len_seed"])
    return [(rng.randint(case["past_lo"], case["past_hi"]),
             1 if r < case["singles"] else rng.randint(case["new_lo"], case["new_hi"]))
            for r in range(case["R"])]


def _prepare_attention(case, seed):
    gen, lens, hkv = _gen(seed), _chunk_lengths(case), case["hkv"]
    width = max(_blocks(p + n) for p, n in lens)
    sink_blocks = _blocks(case["sinks"])
    held = []
    for p, n in lens:
        # Under a window the blocks behind it were given back.
        first = max(0, p + 1 - case["window"]) // BLOCK if case["window"] else 0
        last = _blocks(p + n)
        held.append(sorted(set(range(min(sink_blocks, last))) | set(range(first, last))))
    nb = sum(len(h) for h in held) + 5
    ids = np.random.default_rng(seed).permutation(nb).astype(np.int32)
    tables, at = np.full((case["R"], width), -1, np.int32), 0
    for r, h in enumerate(held):
        tables[r, h] = ids[at:at + len(h)]
        at += len(h)
    starts = np.concatenate([[0], np.cumsum([n for _, n in lens])])
    return {"q": _normal(gen, int(starts[-1]), case["hq"], HEAD),
            "k": _normal(gen, nb, hkv, BLOCK, HEAD), "v": _normal(gen, nb, hkv, HEAD, BLOCK),
            "tables": torch.from_numpy(tables).cuda(), "starts": _int32(starts.tolist()),
            "ctx": _int32([p + n for p, n in lens]), "lens": lens}


def _prepare_norm(case, seed):
    gen, T, H = _gen(seed), case["T"], case["H"]
    return {"x": _normal(gen, T, H, std=2.0), "add": _normal(gen, T, H),
            "weight": _normal(gen, H, std=0.3) + 1, "sum": torch.empty((T, H), dtype=BF16, device="cuda")}


def _prepare_linear(case, seed):
    gen, T, N, K = _gen(seed), case["T"], case["N"], case["K"]
    x, xs = _to_8_bits(_normal(gen, T, K).float())
    n = -(-N // GROUP)
    w = torch.zeros((n * GROUP, K), dtype=BF16, device="cuda")
    w[:N] = _normal(gen, N, K, std=0.02)
    blocks = w.float().view(n, GROUP, K // GROUP, GROUP)
    ws = blocks.abs().amax((1, 3)).clamp(min=LEAST) / TOP
    w = (blocks / ws[:, None, :, None]).to(FP8).view(n * GROUP, K)[:N].contiguous()
    # A group's scales of all rows lie together, as the norm leaves them.
    return {"x": x, "xs": xs.t().contiguous().t(), "w": w, "ws": ws}


# ---- the plain forms -----------------------------------------------------------
def _plain_map(st):
    past, new, tables, free = st["past"].long(), st["new"].long(), st["tables"], st["free"]
    R, W = tables.shape
    held = (past + BLOCK - 1) // BLOCK
    ctx = past + new
    need = (ctx + BLOCK - 1) // BLOCK - held
    first = need.cumsum(0) - need
    i = torch.arange(W, device="cuda") - held[:, None]
    src = first[:, None] + i
    ids = torch.where(src < free.numel(), free[src.clamp(0, free.numel() - 1)], -1)
    tables.copy_(torch.where((i >= 0) & (i < need[:, None]), ids, tables))
    ends = new.cumsum(0)
    j = torch.arange(st["max_tokens"], device="cuda")
    row = (j[:, None] >= ends).sum(1)
    real, row = row < R, row.clamp(max=R - 1)
    pos = past[row] + j - (ends - new)[row]
    block = tables[row, (pos // BLOCK).clamp(0, W - 1)].long()
    slots = torch.where(block >= 0, block * BLOCK + pos % BLOCK, -1)
    starts = torch.cat([ends.new_zeros(1), ends])
    return {"tables": tables, "starts": starts.int(), "ctx": ctx.int(),
            "positions": torch.where(real, pos, -1).int(),
            "slots": torch.where(real, slots, -1).int(), "taken": need.sum().view(1).int()}


def _plain_write(st):
    case, N = st["case"], st["case"]["N"]
    hq, hkv, ck, cv, slots = case["hq"], case["hkv"], st["k"], st["v"], st["slots"].long()
    x = st["qkv"].float().view(N, hq + 2 * hkv, HEAD)
    # 64 bits: 32 lose the angles of far positions.
    angle = st["positions"].double()[:, None] * st["inv"].double()
    c, s = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    a, b = x[:, :hq + hkv, :HEAD // 2], x[:, :hq + hkv, HEAD // 2:]
    y = torch.cat([a * c - b * s, b * c + a * s], -1).to(BF16)
    v = x[:, hq + hkv:].to(BF16)
    at = (slots >= 0).nonzero()[:, 0]
    blk, slot, heads = slots[at] // BLOCK, slots[at] % BLOCK, torch.arange(hkv, device="cuda")
    flat = ck.view(ck.shape[0], hkv, BLOCK * HEAD)
    flat[blk[:, None, None], heads[:, None], _k_place(HEAD)[slot][:, None, :]] = y[at, hq:]
    cv[blk[:, None, None], heads[:, None], torch.arange(HEAD, device="cuda"),
       slot[:, None, None]] = v[at]
    return {"q": y[:, :hq], "k": ck, "v": cv}


def _plain_attention(st):
    q, ck, cv, case = st["q"], st["k"], st["v"], st["case"]
    N, hq, D = q.shape
    nb, H = ck.shape[:2]
    G, place = hq // H, _k_place(D)
    window = case["window"] or 1 << 30
    out, at = torch.empty_like(q), 0
    for r, (past, n) in enumerate(st["lens"]):
        ctx = past + n
        ids = st["tables"][r, :_blocks(ctx)].long()
        there = (ids >= 0).repeat_interleave(BLOCK)[:ctx]
        ids = ids.clamp(min=0)
        k = ck[ids].view(-1, H, BLOCK * D)[..., place.view(-1)].view(-1, H, BLOCK, D)
        k = k.permute(1, 3, 0, 2).reshape(H, D, -1)[..., :ctx].float()
        v = cv[ids].permute(1, 0, 3, 2).reshape(H, -1, D)[:, :ctx].float()
        t, p = torch.arange(ctx, device="cuda"), torch.arange(past, ctx, device="cuda")[:, None]
        seen = (t <= p) & ((t > p - window) | (t < case["sinks"])) & there
        qr = q[at:at + n].float().view(n, H, G, D).permute(1, 2, 0, 3)       # [H, G, n, D]
        # Heads together as far as their scores fit.
        step = max(1, min(H, (1 << 29) // (G * n * ctx)))
        for h in range(0, H, step):
            e = min(h + step, H)
            s = torch.matmul(qr[h:e].reshape(e - h, G * n, D), k[h:e].contiguous())
            s = (s * (1.0 / math.sqrt(D))).view(e - h, G, n, ctx).masked_fill_(~seen, float("-inf"))
            top = s.amax(-1, keepdim=True)
            w = torch.exp(s - torch.where(top == float("-inf"), 0.0, top))
            del s
            total = w.sum(-1, keepdim=True)
            o = torch.matmul(w.view(e - h, G * n, ctx), v[h:e].contiguous()).view(e - h, G, n, D)
            o = torch.where(total > 0, o / total, 0.0)
            out[at:at + n].view(n, H, G, D)[:, h:e] = o.permute(2, 0, 1, 3).to(BF16)
        at += n
    return out


def _to_8_bits(y):
    """(values, scales [rows, groups]) of float32 rows, a scale for each 128 columns."""
    groups = y.view(y.shape[0], -1, GROUP)
    scales = groups.abs().amax(-1).clamp(min=LEAST) / TOP
    return (groups / scales[..., None]).to(FP8).view(y.shape), scales


def _plain_norm(st):
    x = st["x"].float()
    if st["case"]["add"]:
        st["sum"].copy_(x + st["add"].float())
        x = st["sum"].float()
    y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * st["weight"].float()
    values, scales = _to_8_bits(y)
    out = {"values": values, "scales": scales}
    return {**out, "sum": st["sum"]} if st["case"]["add"] else out


def _plain_linear(st):
    N, K = st["w"].shape
    scale = st["ws"].repeat_interleave(GROUP, 0)[:N].repeat_interleave(GROUP, 1)
    w = st["w"].float() * scale
    x = st["x"].float() * st["xs"].repeat_interleave(GROUP, 1)
    return torch.matmul(x, w.t()).to(BF16)


# ---- the framework's calls -------------------------------------------------------
def _own_map(st):
    from rngd_pd_amd import kernels
    m = kernels.chunk_map(st["past"], st["new"], st["tables"], st["free"], st["max_tokens"])
    return {"tables": st["tables"], "starts": m.starts, "ctx": m.ctx_lens,
            "positions": m.positions, "slots": m.slots, "taken": m.taken}


def _own_write(st):
    from rngd_pd_amd import kernels
    q = kernels.rope_cache_write(st["qkv"], st["inv"], st["positions"], st["slots"], st["k"],
                                 st["v"], st["case"]["hq"])
    return {"q": q, "k": st["k"], "v": st["v"]}


def _own_attention(st):
    from rngd_pd_amd import kernels
    case = st["case"]
    span = {"window": case["window"], "sinks": case["sinks"]} if case["window"] else {}
    return kernels.chunk_attention(st["q"], st["k"], st["v"], st["tables"], st["starts"], st["ctx"],
                                   max(n for _, n in st["lens"]), max(p + n for p, n in st["lens"]),
                                   scale=1.0 / math.sqrt(HEAD), **span)


def _own_norm(st):
    from rngd_pd_amd import kernels
    if not st["case"]["add"]:
        values, scales = kernels.rmsnorm_fp8(st["x"], st["weight"], EPS)
        return {"values": values, "scales": scales}
    values, scales = kernels.rmsnorm_fp8(st["x"], st["weight"], EPS, add=st["add"],
                                         sum_out=st["sum"])
    return {"values": values, "scales": scales, "sum": st["sum"]}


def _own_linear(st):
    from rngd_pd_amd import kernels
    return kernels.linear_fp8(st["x"], st["xs"], st["w"], st["ws"])


# ---- the results in 64 bits --------------------------------------------------------
def _exact_map(case, seed):
    st = _prepare_map(case, seed)
    tables, free = st["tables"].cpu().numpy(), st["free"].tolist()
    starts, ctx, positions, slots, taken = [0], [], [], [], 0
    for r, (past, n) in enumerate(zip(st["past"].tolist(), st["new"].tolist())):
        for t in range(past, past + n):
            if t % BLOCK == 0:
                tables[r, t // BLOCK] = free[taken] if taken < len(free) else -1
                taken += 1
            block = int(tables[r, t // BLOCK])
            positions.append(t)
            slots.append(block * BLOCK + t % BLOCK if block >= 0 else -1)
        starts.append(len(positions))
        ctx.append(past + n)
    pad = [-1] * (st["max_tokens"] - len(positions))
    return {"tables": torch.from_numpy(tables), "starts": torch.tensor(starts, dtype=torch.int32),
            "ctx": torch.tensor(ctx, dtype=torch.int32),
            "positions": torch.tensor(positions + pad, dtype=torch.int32),
            "slots": torch.tensor(slots + pad, dtype=torch.int32),
            "taken": torch.tensor([taken], dtype=torch.int32)}


def _exact_write(case, seed):
    st = _prepare_write(case, seed)
    hq, hkv, N = case["hq"], case["hkv"], case["N"]
    z = st["qkv"].double().view(N, -1, 2, HEAD // 2)
    turn = torch.polar(torch.ones((N, HEAD // 2), dtype=torch.float64, device="cuda"),
                       st["positions"].double()[:, None] * st["inv"].double())
    y = torch.complex(z[:, :hq + hkv, 0].contiguous(), z[:, :hq + hkv, 1].contiguous()) * turn[:, None]
    y = torch.stack([y.real, y.imag], 2).view(N, hq + hkv, HEAD)
    k, v = st["k"].double().view(-1, hkv, BLOCK * HEAD), st["v"].double()
    place = _k_place(HEAD)
    n = N - case["unplaced"]
    blk, slot = (st["slots"][:n].long() // BLOCK), (st["slots"][:n].long() % BLOCK)
    for i in range(BLOCK):
        rows = (slot == i).nonzero()[:, 0]
        b = blk[rows]
        part = k[b]
        part[..., place[i]] = y[rows, hq:]
        k[b] = part
        v[b, :, :, i] = z[rows, hq + hkv:].reshape(-1, hkv, HEAD)
    return {"q": y[:, :hq], "k": k.view(st["k"].shape), "v": v}


def _exact_attention(case, seed):
    if work(case)["flops"] > 3e12:
        return None
    st = _prepare_attention(case, seed)
    H, G = case["hkv"], case["hq"] // case["hkv"]
    place, out, at = _k_place(HEAD), torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda"), 0
    tables = st["tables"].tolist()
    for r, (past, n) in enumerate(st["lens"]):
        # The blocks that are there, one after another, and their tokens' positions.
        have = [(j, b) for j, b in enumerate(tables[r][:_blocks(past + n)]) if b >= 0]
        ids = torch.tensor([b for _, b in have], device="cuda")
        t = (torch.tensor([j for j, _ in have], device="cuda")[:, None] * BLOCK
             + torch.arange(BLOCK, device="cuda")).view(-1)
        ago = torch.arange(past, past + n, device="cuda")[:, None] - t
        hidden = ago < 0
        if case["window"]:
            hidden = hidden | ((ago >= case["window"]) & (t >= case["sinks"]))
        for h in range(H):
            k = st["k"][ids, h].view(len(have), -1)[:, place].reshape(-1, HEAD).double()
            v = st["v"][ids, h].transpose(1, 2).reshape(-1, HEAD).double()
            for g in range(h * G, (h + 1) * G):
                s = st["q"][at:at + n, g].double() @ k.t().contiguous() / math.sqrt(HEAD)
                s.masked_fill_(hidden, -math.inf)
                out[at:at + n, g] = torch.softmax(s, -1) @ v
        at += n
    return out


def _exact_norm(case, seed):
    st = _prepare_norm(case, seed)
    x = st["x"].double()
    total = x + st["add"].double()
    if case["add"]:
        x = total.to(BF16).double()         # the norm is that of the sum as it is kept
    y = x / torch.sqrt(x.square().mean(-1, keepdim=True) + EPS) * st["weight"].double()
    groups = y.unflatten(-1, (-1, GROUP))
    scales = groups.abs().amax(-1).clamp(min=LEAST) / TOP
    # The scaled values before their rounding to 8 bits.
    out = {"values": (groups / scales[..., None]).flatten(-2), "scales": scales}
    return {**out, "sum": total} if case["add"] else out


def _exact_linear(case, seed):
    st = _prepare_linear(case, seed)
    T, N, K = case["T"], case["N"], case["K"]
    out = torch.empty((T, N), dtype=torch.float64, device="cuda")
    x = (st["x"].double().view(T, -1, GROUP) * st["xs"].double()[..., None]).view(T, K)
    for b in range(-(-N // GROUP)):
        rows = slice(b * GROUP, min(N, (b + 1) * GROUP))
        w = st["w"][rows].double().unflatten(1, (-1, GROUP)) * st["ws"][b].double()[:, None]
        out[:, rows] = x @ w.flatten(1).t().contiguous()
    return out


# ---- what the measuring program calls ---------------------------------------------
_PREPARE = {"map": _prepare_map, "write": _prepare_write, "attention": _prepare_attention,
            "norm": _prepare_norm, "linear": _prepare_linear}
_PLAIN = {"map": _plain_map, "write": _plain_write, "attention": _plain_attention,
          "norm": _plain_norm, "linear": _plain_linear}
_OWN = {"map": _own_map, "write": _own_write, "attention": _own_attention, "norm": _own_norm,
        "linear": _own_linear}
_EXACT = {"map": _exact_map, "write": _exact_write, "attention": _exact_attention,
          "norm": _exact_norm, "linear": _exact_linear}


def prepare(case, seed):
    st = _PREPARE[case["kind"]](case, seed)
    st["case"] = case
    return st


def run(state):
    return (_OWN if own else _PLAIN)[state["case"]["kind"]](state)


def _pairs(past, n, window, sinks):
    """How many (query, token) pairs n new tokens after ``past`` see."""
    if not window:
        return n * past + n * (n + 1) // 2
    total = 0
    for p in range(past, past + n):
        near = min(p + 1, window)
        total += near + min(sinks, p + 1 - near)
    return total


def _span(past, n, window, sinks):
    """How many tokens some of them see."""
    first = max(0, past + 1 - window) if window else 0
    return past + n - first + min(sinks, first)


def work(case):
    kind = case["kind"]
    if kind == "map":
        lens = _map_lengths(case)
        tokens = sum(n for _, n in lens) + case["spare"]
        grown = sum(_blocks(p + n) - _blocks(p) for p, n in lens)
        # Lengths, starts and contexts; a block's id per token's block; positions and slots.
        return {"bytes": 16 * case["R"] + 8 * grown + 8 * tokens + 4 * (tokens // BLOCK + case["R"]),
                "flops": 0}
    if kind == "write":
        heads, placed = case["hq"] + 2 * case["hkv"], case["N"] - case["unplaced"]
        return {"bytes": 2 * HEAD * (case["N"] * (heads + case["hq"]) + placed * 2 * case["hkv"])
                + 8 * case["N"], "flops": 3 * case["N"] * (case["hq"] + case["hkv"]) * HEAD}
    if kind == "attention":
        lens, span = _chunk_lengths(case), (case["window"], case["sinks"])
        pairs = sum(_pairs(p, n, *span) for p, n in lens)
        tokens = sum(_span(p, n, *span) for p, n in lens)
        return {"bytes": tokens * case["hkv"] * HEAD * 4 + sum(n for _, n in lens) * case["hq"] * HEAD * 4,
                "flops": 4 * pairs * case["hq"] * HEAD}
    if kind == "norm":
        T, H = case["T"], case["H"]
        return {"bytes": T * H * (7 if case["add"] else 3) + 4 * T * H // GROUP + 2 * H,
                "flops": 5 * T * H}
    T, N, K = case["T"], case["N"], case["K"]
    scales = 4 * (T + -(-N // GROUP)) * (K // GROUP)
    return {"bytes": T * K + N * K + 2 * T * N + scales, "flops": 2 * T * N * K}


def exact(case, seed):
    return _EXACT[case["kind"]](case, seed)
