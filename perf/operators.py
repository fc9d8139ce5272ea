"""Operators whose speed counts, as cases that can be timed one by one against
their plain forms.

Five operators of a server that keeps its KV in a paged cache (16-token blocks,
K tiled and V dim-major as rngd_pd_amd.engines.paged_cache lays them out):

  decode   attention of one new token per stream over a sliding window and the
           first few tokens (sinks), with or without the token's cache write;
  prompt   the same mask over all tokens of a prompt;
  copy     whole blocks copied inside the cache, all layers of K and V (a fork's
           last block, a compaction);
  select   beam search's n best of beams x vocabulary, from logits and the
           beams' scores;
  reorder  the cache following the selection: block tables shared with the
           parent beam, the partly filled block copied.

Where ``own`` is false run() computes the plain form in elementary torch
operations; where it is true it calls the framework. listed() gives the named
cases, draw(rng) another one of the same ranges, prepare(case, seed) what a
program holds before the call, work(case) the bytes and operations a pass cannot
do without, exact(case, seed) the result in 64 bits. The shapes are
Llama-3.1-8B's (32 layers, 32 query and 8 KV heads of 128, vocabulary 128256)
and other groupings of heads.
"""
import math
import random

import numpy as np
import torch

own = False

BF16 = torch.bfloat16
HEAD = 128
BLOCK = 16
VOCAB = 128256


# ---- cases ------------------------------------------------------------------
def listed():
    return [
        # One chat stream just past its window: the step's latency.
        {"name": "window_decode_b1", "kind": "decode", "B": 1, "lo": 700, "hi": 700, "window": 512,
         "sinks": 4, "hq": 32, "hkv": 8, "append": True, "dropped": False, "len_seed": 0},
        # The serving batch of 16 with ragged contexts, some inside the window yet.
        {"name": "window_decode_b16", "kind": "decode", "B": 16, "lo": 500, "hi": 9000,
         "window": 1024, "sinks": 4, "hq": 32, "hkv": 8, "append": True, "dropped": False,
         "len_seed": 1},
        # Long-running streams whose blocks behind the window were freed.
        {"name": "window_decode_b48", "kind": "decode", "B": 48, "lo": 20000, "hi": 200000,
         "window": 4096, "sinks": 16, "hq": 64, "hkv": 8, "append": False, "dropped": True,
         "len_seed": 2},
        # A request of the length the handoff was benchmarked on, short window.
        {"name": "window_prompt_470", "kind": "prompt", "T": 470, "window": 128, "sinks": 4,
         "hq": 32, "hkv": 8},
        # A long document.
        {"name": "window_prompt_8000", "kind": "prompt", "T": 8000, "window": 1024, "sinks": 4,
         "hq": 32, "hkv": 8},
        # A fork into three beams: the prompt's last block, once for each.
        {"name": "copy_blocks_3", "kind": "copy", "n": 3, "layers": 32, "hkv": 8},
        # A compaction of a cache with scattered free blocks.
        {"name": "copy_blocks_512", "kind": "copy", "n": 512, "layers": 32, "hkv": 8},
        # One request of four beams, twice as many candidates kept for those that end.
        {"name": "beam_select_r1", "kind": "select", "R": 1, "K": 4, "V": VOCAB, "n": 8,
         "f32": False, "eos": True, "masked": False},
        # The decoder's widest batch, 64 rows, as 16 requests of four beams.
        {"name": "beam_select_r16", "kind": "select", "R": 16, "K": 4, "V": VOCAB, "n": 4,
         "f32": False, "eos": True, "masked": False},
        # An offline batch with 32-bit logits under a grammar's mask.
        {"name": "beam_select_r32_f32", "kind": "select", "R": 32, "K": 8, "V": VOCAB, "n": 16,
         "f32": True, "eos": False, "masked": True},
        # The states of those four beams, and of the 64 rows.
        {"name": "beam_reorder_r1", "kind": "reorder", "R": 1, "K": 4, "lo": 603, "hi": 603,
         "layers": 32, "hkv": 8, "len_seed": 0},
        {"name": "beam_reorder_r16", "kind": "reorder", "R": 16, "K": 4, "lo": 100, "hi": 4000,
         "layers": 32, "hkv": 8, "len_seed": 3},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["decode", "decode", "decode", "prompt", "prompt", "copy", "select",
                       "select", "reorder"])
    heads = rng.choice([(32, 8), (32, 8), (64, 8), (16, 2), (8, 8), (28, 4), (24, 8), (40, 8)])
    if kind == "decode":
        B = _log_int(rng, 1, 48)
        window = _log_int(rng, 1, 4096)
        dropped = rng.random() < 0.5
        hi = _log_int(rng, 1, 200000 if dropped else min(32768, 262144 // B))
        return {"kind": kind, "B": B, "lo": rng.randint(1, hi), "hi": hi, "window": window,
                "sinks": rng.choice([0, 1, 4, 4, 16, 33, 64]), "hq": heads[0], "hkv": heads[1],
                "append": rng.random() < 0.7, "dropped": dropped,
                "len_seed": rng.randrange(1 << 20)}
    if kind == "prompt":
        T = _log_int(rng, 1, 8000)
        return {"kind": kind, "T": T, "window": _log_int(rng, 1, 1024 if T > 4000 else 2048),
                "sinks": rng.choice([0, 1, 4, 4, 16, 33, 64]), "hq": min(heads[0], 32),
                "hkv": heads[1]}
    if kind == "copy":
        return {"kind": kind, "n": _log_int(rng, 1, 512), "layers": rng.choice([8, 16, 32]),
                "hkv": rng.choice([1, 2, 4, 8])}
    if kind == "select":
        K = rng.randint(1, 16)
        R = _log_int(rng, 1, 256 // K)
        return {"kind": kind, "R": R, "K": K, "V": _log_int(rng, 1000, VOCAB),
                "n": rng.choice([K, K, 2 * K, rng.randint(1, 32)]), "f32": rng.random() < 0.4,
                "eos": rng.random() < 0.5, "masked": rng.random() < 0.3}
    K = rng.randint(2, 16)
    hi = _log_int(rng, 1, 4000)
    return {"kind": kind, "R": _log_int(rng, 1, 64 // K), "K": K, "lo": rng.randint(1, hi),
            "hi": hi, "layers": rng.choice([8, 16, 32]), "hkv": rng.choice([1, 2, 4, 8]),
            "len_seed": rng.randrange(1 << 20)}


# ---- inputs -----------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _normal(gen, *shape, std=1.0):
    return torch.empty(shape, dtype=BF16, device="cuda").normal_(0.0, std, generator=gen)


def _lengths(case, n):
    rng = random.Random(case["len_seed"])
    return [rng.randint(case["lo"], case["hi"]) for _ in range(n)]


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _k_place(D):
    """int64 [16, D]: where a K block keeps (slot, dim) among its 16 D values."""
    s = torch.arange(BLOCK, device="cuda").view(BLOCK, 1)
    d = torch.arange(D, device="cuda").view(1, D)
    unit = ((((s >> 2) & 1) * (D // 32) + d // 32) * 4 + (d // 8) % 4) * 8 + (s >> 3) * 4 + (s & 3)
    return unit * 8 + d % 8


def _prepare_decode(case, seed):
    gen, B, hq, hkv = _gen(seed), case["B"], case["hq"], case["hkv"]
    ctx = _lengths(case, B)
    width = -(-max(ctx) // BLOCK)
    sink_blocks = -(-case["sinks"] // BLOCK)
    held = []
    for c in ctx:
        first = max(0, c - case["window"]) // BLOCK if case["dropped"] else 0
        last = -(-c // BLOCK)
        held.append(sorted(set(range(min(sink_blocks, last))) | set(range(first, last))))
    nb = sum(len(h) for h in held) + 5
    ids = np.random.default_rng(seed).permutation(nb).astype(np.int32)
    tables, at = np.full((B, width), -1, np.int32), 0
    for b, h in enumerate(held):
        tables[b, h] = ids[at:at + len(h)]
        at += len(h)
    return {"q": _normal(gen, B, hq, HEAD), "k_new": _normal(gen, B, hkv, HEAD),
            "v_new": _normal(gen, B, hkv, HEAD), "k": _normal(gen, nb, hkv, BLOCK, HEAD),
            "v": _normal(gen, nb, hkv, HEAD, BLOCK), "tables": torch.from_numpy(tables).cuda(),
            "ctx": _int32(ctx), "max_ctx": max(ctx)}


def _prepare_prompt(case, seed):
    gen, T = _gen(seed), case["T"]
    # q, k and v as a projection leaves them: columns of one tensor.
    qkv = _normal(gen, T, case["hq"] + 2 * case["hkv"], HEAD)
    q, k, v = qkv.split([case["hq"], case["hkv"], case["hkv"]], 1)
    return {"q": q, "k": k, "v": v}


def _cache(gen, layers, nb, hkv):
    return {"k": _normal(gen, layers, nb, hkv, BLOCK, HEAD),
            "v": _normal(gen, layers, nb, hkv, HEAD, BLOCK)}


def _prepare_copy(case, seed):
    n = case["n"]
    nb = 2 * n + 3
    ids = np.random.default_rng(seed).permutation(nb).astype(np.int32)
    # A fork reads one block several times; a compaction moves each once.
    src = ids[n:2 * n] if n > 16 else np.repeat(ids[n:n + 1], n)
    return {**_cache(_gen(seed), case["layers"], nb, case["hkv"]), "src": src, "dst": ids[:n]}


def _prepare_select(case, seed):
    gen, R, K, V = _gen(seed), case["R"], case["K"], case["V"]
    x = torch.empty((R * K, V), device="cuda").normal_(0.0, 2.5, generator=gen)
    if case["masked"]:
        x.masked_fill_(torch.rand((R * K, V), generator=gen, device="cuda") < 0.9, float("-inf"))
    scores = -20.0 * torch.rand((R, K), generator=gen, device="cuda")
    last = torch.randint(0, V, (R, K), generator=gen, device="cuda", dtype=torch.int32)
    eos = V // 3
    last[torch.rand((R, K), generator=gen, device="cuda") < 0.25] = eos
    return {"logits": x if case["f32"] else x.to(BF16), "scores": scores, "last": last, "eos": eos}


def _parents(case):
    """Half of the beams (rounded up) go on, each into two places or one."""
    rng, K = random.Random(case["len_seed"] + 1), case["K"]
    rows = []
    for _ in range(case["R"]):
        rows.append([i % (-(-K // 2)) for i in range(K)])
        rng.shuffle(rows[-1])
    return rows


def _prepare_reorder(case, seed):
    gen, R, K = _gen(seed), case["R"], case["K"]
    ctx = _lengths(case, R)
    width = max(ctx) // BLOCK + 3
    nb = R * K * 3 + 37
    rng = np.random.default_rng(seed)
    # Filled blocks may be anyone's; those from the partly filled one on are the beam's own.
    tables = rng.integers(0, nb, (R, K, width)).astype(np.int32)
    own_ids = rng.permutation(nb)[:R * K * 3].astype(np.int32).reshape(R, K, 3)
    for r, c in enumerate(ctx):
        n = min(3, width - c // BLOCK)
        tables[r, :, c // BLOCK:] = -1
        tables[r, :, c // BLOCK:c // BLOCK + n] = own_ids[r, :, :n]
    return {**_cache(gen, case["layers"], nb, case["hkv"]),
            "tables": torch.from_numpy(tables.reshape(R * K, width)).cuda(),
            "parents": _int32(_parents(case)), "ctx": _int32([c for c in ctx for _ in range(K)])}


# ---- the plain forms -----------------------------------------------------------
def _plain_decode(st):
    q, ck, cv, tables, ctx = st["q"], st["k"], st["v"], st["tables"], st["ctx"].long()
    window, sinks = st["case"]["window"], st["case"]["sinks"]
    B, hq, D = q.shape
    nb, H = ck.shape[:2]
    place, heads = _k_place(D), torch.arange(H, device="cuda")
    flat = ck.view(nb, H, BLOCK * D)
    if st["case"]["append"]:
        blk = tables.gather(1, ((ctx - 1) // BLOCK)[:, None])[:, 0].long()
        slot = (ctx - 1) % BLOCK
        flat[blk[:, None, None], heads[:, None], place[slot][:, None, :]] = st["k_new"]
        cv[blk[:, None, None], heads[:, None], torch.arange(D, device="cuda"),
           slot[:, None, None]] = st["v_new"]
    # The tokens each stream sees: the sinks, then the window's (those not among the sinks).
    window = min(window, st["max_ctx"])
    i = torch.arange(sinks + window, device="cuda")
    pos = torch.where(i < sinks, i, (ctx[:, None] - window) + i - sinks)
    seen = torch.where(i < sinks, pos < ctx[:, None], pos >= sinks)
    pos = pos.clamp(0, tables.shape[1] * BLOCK - 1)
    blk = tables.gather(1, pos // BLOCK).long()
    seen = seen & (blk >= 0) & (blk < nb)
    blk, slot = blk.clamp(0, nb - 1), pos % BLOCK
    k = flat[blk[:, :, None, None], heads[:, None], place[slot][:, :, None, :]].float()
    v = cv[blk[:, :, None], heads, :, slot[:, :, None]].float()              # [B, n, H, D]
    s = torch.matmul(q.float().view(B, H, hq // H, D), k.permute(0, 2, 3, 1).contiguous())
    s = (s * (1.0 / math.sqrt(D))).masked_fill(~seen[:, None, None, :], float("-inf"))
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top == float("-inf"), 0.0, top))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p, v.permute(0, 2, 1, 3).contiguous())
    out = torch.where(total > 0, o / total, 0.0).view(B, hq, D).to(BF16)
    return {"out": out, "k": ck, "v": cv} if st["case"]["append"] else {"out": out}


def _plain_prompt(st):
    q, k, v = st["q"].float(), st["k"].float(), st["v"].float()
    T, hq, D = q.shape
    H = k.shape[1]
    qg = q.view(T, H, hq // H, D).permute(1, 2, 0, 3).reshape(H, -1, D).contiguous()
    s = torch.matmul(qg, k.permute(1, 2, 0).contiguous()).view(H, hq // H, T, T)
    i = torch.arange(T, device="cuda")
    seen = (i <= i[:, None]) & ((i > i[:, None] - st["case"]["window"]) | (i < st["case"]["sinks"]))
    s = (s * (1.0 / math.sqrt(D))).masked_fill(~seen, float("-inf"))
    p = torch.exp(s - s.amax(-1, keepdim=True))
    o = torch.matmul((p / p.sum(-1, keepdim=True)).view(H, -1, T),
                     v.permute(1, 0, 2).contiguous())
    return o.view(H, hq // H, T, D).permute(2, 0, 1, 3).reshape(T, hq, D).to(BF16)


def _plain_copy(st):
    src, dst = (torch.from_numpy(st[n]).cuda().long() for n in ("src", "dst"))
    st["k"][:, dst] = st["k"][:, src]
    st["v"][:, dst] = st["v"][:, src]
    return {"k": st["k"], "v": st["v"]}


def _plain_select(st):
    scores, case = st["scores"].double(), st["case"]
    R, K = scores.shape
    n, V = case["n"], st["logits"].shape[1]
    x = st["logits"].float().view(R, K, V) + 0.0                             # -0 is 0
    # 64 bits: totals of different beams may lie closer than 32 bits can tell.
    wide = x.double()
    top = wide.amax(-1, keepdim=True)
    lse = top[..., 0] + torch.log(torch.exp(wide - top).sum(-1))
    # A beam's n best by logit, the lowest token first among equals, as one integer key.
    bits = x.view(torch.int32)
    code = torch.where(bits < 0, bits ^ 0x7fffffff, bits).long()
    token = torch.arange(V, device="cuda")
    best = ((code << 32) + (0xffffffff - token)).topk(min(n, V), -1).values
    tokens = 0xffffffff - (best & 0xffffffff)
    totals = scores[..., None] + (wide.gather(-1, tokens) - lse[..., None])
    alive = torch.isfinite(lse) & torch.isfinite(scores)
    totals = torch.where(alive[..., None], totals, float("-inf"))
    if case["eos"]:
        ended = (st["last"] == st["eos"])[..., None]
        first = torch.arange(tokens.shape[-1], device="cuda") == 0
        totals = torch.where(ended, torch.where(first, scores[..., None], float("-inf")), totals)
        tokens = torch.where(ended, st["eos"], tokens)
    beams = torch.arange(K, device="cuda")[:, None].expand(K, tokens.shape[-1]).reshape(-1)
    order = torch.sort(totals.view(R, -1), dim=-1, descending=True, stable=True)
    pick = order.indices[:, :n]
    got = order.values[:, :n]
    none = got == float("-inf")
    return {"tokens": torch.where(none, -1, tokens.view(R, -1).gather(1, pick)).int(),
            "parents": torch.where(none, -1, beams[pick]).int(), "scores": got.float()}


def _plain_reorder(st):
    case, parents, ctx = st["case"], st["parents"].long(), st["ctx"].long()
    R, K = parents.shape
    rows = st["tables"].view(R, K, -1)
    W = rows.shape[2]
    full = (ctx.view(R, K)[:, :1] // BLOCK)[:, :, None]
    old = rows.gather(1, parents[:, :, None].expand(R, K, W))
    last = full.clamp(max=W - 1).expand(R, K, 1)
    dst, src = rows.gather(2, last)[..., 0].long(), old.gather(2, last)[..., 0].long()
    part = (ctx.view(R, K) % BLOCK > 0)
    src = torch.where(part, src, dst).view(-1)
    dst = dst.view(-1)
    rows.copy_(torch.where(torch.arange(W, device="cuda") < full, old, rows))
    st["k"][:, dst] = st["k"][:, src]
    st["v"][:, dst] = st["v"][:, src]
    return {"tables": st["tables"], "k": st["k"], "v": st["v"]}


# ---- the framework's calls -------------------------------------------------------
def _own_decode(st):
    from rngd_pd_amd import kernels
    case, scale = st["case"], 1.0 / math.sqrt(HEAD)
    span = {"window": case["window"], "sinks": case["sinks"]}
    if not case["append"]:
        return {"out": kernels.decode_attention(st["q"], st["k"], st["v"], st["tables"], st["ctx"],
                                                st["max_ctx"], scale=scale, **span)}
    out = kernels.decode_attention_append(st["q"], st["k_new"], st["v_new"], st["k"], st["v"],
                                          st["tables"], st["ctx"], st["max_ctx"], scale=scale,
                                          **span)
    return {"out": out, "k": st["k"], "v": st["v"]}


def _own_prompt(st):
    from rngd_pd_amd import kernels
    return kernels.prefill_attention(st["q"], st["k"], st["v"], scale=1.0 / math.sqrt(HEAD),
                                     window=st["case"]["window"], sinks=st["case"]["sinks"])


def _own_copy(st):
    from rngd_pd_amd import kernels
    kernels.copy_blocks(st["k"], st["v"], st["src"], st["dst"])
    return {"k": st["k"], "v": st["v"]}


def _own_select(st):
    from rngd_pd_amd import kernels
    end = {"eos": st["eos"], "last_tokens": st["last"]} if st["case"]["eos"] else {}
    tokens, parents, scores = kernels.beam_select(st["logits"], st["scores"], st["case"]["n"],
                                                  **end)
    return {"tokens": tokens, "parents": parents, "scores": scores}


def _own_reorder(st):
    from rngd_pd_amd import kernels
    kernels.beam_reorder(st["parents"], st["ctx"], st["tables"], st["k"], st["v"])
    return {"tables": st["tables"], "k": st["k"], "v": st["v"]}


# ---- the results in 64 bits --------------------------------------------------------
def _visible(p, window, sinks):
    """Sorted positions that a query at position p sees."""
    first = max(0, p - window + 1)
    return list(range(min(sinks, first, p + 1))) + list(range(first, p + 1))


def _exact_decode(case, seed):
    st = _prepare_decode(case, seed)
    q, k, v = st["q"].double(), st["k"], st["v"]
    H, G = case["hkv"], case["hq"] // case["hkv"]
    place, ctx, tables = _k_place(HEAD), st["ctx"].tolist(), st["tables"].cpu().numpy()
    out = torch.zeros_like(q)
    for b, c in enumerate(ctx):
        pos = np.asarray(_visible(c - 1, case["window"], case["sinks"]))
        blocks, where = np.unique(pos // BLOCK, return_inverse=True)
        ids = torch.from_numpy(tables[b, blocks].astype(np.int64)).cuda()
        where, slot = torch.from_numpy(where).cuda(), torch.from_numpy(pos % BLOCK).cuda()
        kb = k[ids].reshape(len(blocks), H, -1)[..., place].double()         # [n, H, 16, D]
        vb = v[ids].double().transpose(2, 3)                                 # [n, H, 16, D]
        ks, vs = kb[where, :, slot], vb[where, :, slot]                      # [t, H, D]
        if case["append"]:
            ks[-1], vs[-1] = st["k_new"][b].double(), st["v_new"][b].double()
        for h in range(H):
            w = torch.softmax(q[b, h * G:(h + 1) * G] @ ks[:, h].t().contiguous()
                              / math.sqrt(HEAD), -1)
            out[b, h * G:(h + 1) * G] = w @ vs[:, h].contiguous()
    if not case["append"]:
        return {"out": out}
    for b, c in enumerate(ctx):
        blk, slot = int(tables[b, (c - 1) // BLOCK]), (c - 1) % BLOCK
        k[blk].view(H, -1)[:, place[slot]] = st["k_new"][b]
        v[blk, :, :, slot] = st["v_new"][b]
    return {"out": out, "k": k, "v": v}


def _exact_prompt(case, seed):
    st = _prepare_prompt(case, seed)
    q, k, v = st["q"].double(), st["k"].double(), st["v"].double()
    T, G = case["T"], case["hq"] // case["hkv"]
    t, out = torch.arange(T, device="cuda"), torch.zeros_like(q)
    ago = t[:, None] - t
    hidden = (ago < 0) | ((ago >= case["window"]) & (t >= case["sinks"]))
    for h in range(case["hq"]):
        s = q[:, h].contiguous() @ k[:, h // G].t().contiguous() / math.sqrt(HEAD)
        out[:, h] = torch.softmax(s.masked_fill(hidden, -math.inf), -1) @ v[:, h // G].contiguous()
    return out


def _exact_copy(case, seed):
    st = _prepare_copy(case, seed)
    k, v = st["k"].clone(), st["v"].clone()
    for s, d in zip(st["src"].tolist(), st["dst"].tolist()):
        k[:, d], v[:, d] = st["k"][:, s], st["v"][:, s]
    return {"k": k, "v": v}


def _exact_select(case, seed):
    st = _prepare_select(case, seed)
    R, K, V, n = case["R"], case["K"], case["V"], case["n"]
    tokens = torch.full((R, n), -1, dtype=torch.int32, device="cuda")
    parents, out = tokens.clone(), torch.full((R, n), -math.inf, dtype=torch.float64, device="cuda")
    for r in range(R):
        total = st["scores"][r].double()[:, None] + torch.log_softmax(
            st["logits"][r * K:(r + 1) * K].double(), -1)
        if case["eos"]:
            done = st["last"][r] == st["eos"]
            total[done] = -math.inf
            total[done, st["eos"]] = st["scores"][r].double()[done]
        total, at = torch.sort(total.view(-1), descending=True, stable=True)
        m = min(n, int((total > -math.inf).sum()))
        tokens[r, :m], parents[r, :m], out[r, :m] = at[:m] % V, at[:m] // V, total[:m]
    return {"tokens": tokens, "parents": parents, "scores": out}


def _exact_reorder(case, seed):
    st = _prepare_reorder(case, seed)
    R, K = case["R"], case["K"]
    k, v, tables = st["k"].clone(), st["v"].clone(), st["tables"].clone()
    old, ctx = st["tables"].tolist(), st["ctx"].tolist()
    for r, row in enumerate(st["parents"].tolist()):
        full, rest = divmod(ctx[r * K], BLOCK)
        for j, p in enumerate(row):
            tables[r * K + j, :full] = st["tables"][r * K + p, :full]
            if rest:
                d, s = old[r * K + j][full], old[r * K + p][full]
                k[:, d], v[:, d] = st["k"][:, s], st["v"][:, s]
    return {"tables": tables, "k": k, "v": v}


# ---- what the measuring program calls ---------------------------------------------
_PREPARE = {"decode": _prepare_decode, "prompt": _prepare_prompt, "copy": _prepare_copy,
            "select": _prepare_select, "reorder": _prepare_reorder}
_PLAIN = {"decode": _plain_decode, "prompt": _plain_prompt, "copy": _plain_copy,
          "select": _plain_select, "reorder": _plain_reorder}
_OWN = {"decode": _own_decode, "prompt": _own_prompt, "copy": _own_copy, "select": _own_select,
        "reorder": _own_reorder}
_EXACT = {"decode": _exact_decode, "prompt": _exact_prompt, "copy": _exact_copy,
          "select": _exact_select, "reorder": _exact_reorder}


def prepare(case, seed):
    st = _PREPARE[case["kind"]](case, seed)
    st["case"] = case
    return st


def run(state):
    return (_OWN if own else _PLAIN)[state["case"]["kind"]](state)


def _seen(p, window, sinks):
    """How many tokens a query at position p sees."""
    near = min(p + 1, window)
    return near + min(sinks, p + 1 - near)


def work(case):
    kind = case["kind"]
    if kind == "decode":
        seen = sum(_seen(c - 1, case["window"], case["sinks"]) for c in _lengths(case, case["B"]))
        io = case["B"] * (2 * case["hq"] + (4 * case["hkv"] if case["append"] else 0)) * HEAD * 2
        return {"bytes": seen * case["hkv"] * HEAD * 4 + io,
                "flops": 4 * seen * case["hq"] * HEAD}
    if kind == "prompt":
        seen = sum(_seen(p, case["window"], case["sinks"]) for p in range(case["T"]))
        return {"bytes": case["T"] * (2 * case["hq"] + 2 * case["hkv"]) * HEAD * 2,
                "flops": 4 * seen * case["hq"] * HEAD}
    if kind == "select":
        rows = case["R"] * case["K"] * case["V"]
        return {"bytes": rows * (4 if case["f32"] else 2) + 12 * case["R"] * case["n"],
                "flops": 4 * rows}
    block = case["layers"] * 2 * case["hkv"] * BLOCK * HEAD * 2
    if kind == "copy":
        return {"bytes": block * (case["n"] + (case["n"] if case["n"] > 16 else 1)), "flops": 0}
    total = 0
    for row, c in zip(_parents(case), _lengths(case, case["R"])):
        moved = [p for k, p in enumerate(row) if p != k]
        total += block * (len(moved) + len(set(moved))) if c % BLOCK else 0
        total += 8 * len(moved) * (c // BLOCK)
    return {"bytes": total, "flops": 0}


def exact(case, seed):
    return _EXACT[case["kind"]](case, seed)
