"""Performance cases of serving with sliding windows and 8-bit block caches: the page bookkeeping of a
step on the GPU, the write of its keys and values into pages of e4m3 values with one scale per page and
KV head, attention over such pages, and attention with a sliding window and a few first tokens (sinks)
over caches of every kind.

A step of a serving batch runs them in this order. `reserve_pages_` gives every sequence the pages for
its new positions and makes the step's positions, slots and query offsets, `store_kv_` writes the new
rows, `paged_attention_` or `window_attention_` reads the cache, and `release_pages_` takes back what
the step did not keep.

`run` with `own` false is the plain form in elementary torch operations; with `own` true it makes
the calls of tileinfer_hip.
"""
from __future__ import annotations

import math
import os
import random
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
E4M3 = torch.float8_e4m3fn


def _ti():
    path = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "tileinfer.jl_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import tileinfer_hip
    return tileinfer_hip


# ---- cases ----------------------------------------------------------------------------------

def _pages(name=None, **kw):
    # ctx / new: positions that each sequence holds and gets; the step is taken back whole afterwards
    c = dict(op="pages", page=64, seqs=1, ctx_min=0, ctx=0, new_min=1, new=1, lens=1)
    c.update(kw)
    return c if name is None else dict(c, name=name)


def _write(name=None, **kw):
    c = dict(op="write", dtype="bf16", kv_heads=8, head_dim=128, page=64, seqs=1, ctx_min=0, ctx=0, new_min=1, new=1, lens=1)
    c.update(kw)
    return c if name is None else dict(c, name=name)


def _attend(name=None, **kw):
    # window 0: every key up to the query's own; else the last `window` and the first `sinks` ones
    c = dict(op="attend", dtype="bf16", kv="dense", heads=32, kv_heads=8, head_dim=128, page=64, seqs=1, ctx_min=0, ctx=0,
             new_min=1, new=1, window=0, sinks=0, lens=1)
    c.update(kw)
    return c if name is None else dict(c, name=name)


def listed():
    return [
        # eight drafted tokens for each chat of a serving batch, none of them kept: pages given and taken back
        _pages("pages_drafts_b32", seqs=32, ctx_min=1000, ctx=8191, new_min=8, new=8),
        # a batch of requests comes and goes: prompts of up to 4096 tokens in 16-token pages
        _pages("pages_prompts_b256", page=16, seqs=256, new_min=100, new=4096),
        # one new row for each chat of a serving batch
        _write("write_token_b32", seqs=32, ctx_min=1023, ctx=8191),
        # a long prompt into empty pages of 16 tokens
        _write("write_prompt_8192", page=16, new_min=8192, new=8192),
        # a serving batch on an 8-bit block cache, one token each
        _attend("fp8_decode_b32", kv="fp8", page=16, seqs=32, ctx_min=4095, ctx=4095),
        # a chunk of a long document on an 8-bit block cache
        _attend("fp8_chunk_1500_on_3000", kv="fp8", ctx_min=3000, ctx=3000, new_min=1500, new=1500),
        # one long chat of a sliding-window model, one token: the smallest attention call
        _attend("window_token", ctx_min=32767, ctx=32767, window=1024, sinks=4),
        # a serving batch of such chats, of very different lengths
        _attend("window_ragged_b32", page=16, seqs=32, ctx_min=100, ctx=32767, window=4096, sinks=4),
        # the same on an INT8 cache with fewer chats
        _attend("window_int8_b8", kv="int8", page=16, seqs=8, ctx_min=8000, ctx=32767, window=8192),
        # drafted blocks of 16 tokens are verified on an 8-bit block cache
        _attend("window_fp8_verify_b16", kv="fp8", seqs=16, ctx_min=4096, ctx=16383, new_min=16, new=16, window=4096, sinks=4),
        # a Float32 model's chunk
        _attend("window_fp32_chunk_512", dtype="fp32", heads=16, page=16, ctx_min=2000, ctx=2000, new_min=512, new=512, window=512),
        # a long prompt of a sliding-window model: the largest call
        _attend("window_prompt_8192", new_min=8192, new=8192, window=2048, sinks=4),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / (3 if case.get("dtype") == "fp32" else 50))


def draw(rng):
    most = max(_cost(c) for c in listed())
    heads, kv_heads = rng.choice([(32, 8), (32, 8), (16, 8), (24, 8), (32, 4), (64, 8), (8, 8)])
    while True:
        op = rng.choice(["pages", "write", "attend", "attend", "attend"])
        lens, page = rng.randrange(1 << 30), rng.choice([16, 64, 64, 32])
        step = rng.choice(["token", "token", "block", "prompt", "chunk"])
        if step == "token":
            seqs, ctx, new = _log(rng, 1, 128), _log(rng, 1, 32768), 1
        elif step == "block":
            seqs, ctx, new = _log(rng, 1, 64), _log(rng, 1, 16384), rng.randint(2, 16)
        elif step == "prompt":
            seqs, ctx, new = _log(rng, 1, 16), 0, _log(rng, 17, 8192)
        else:
            seqs, ctx, new = rng.choice([1, 1, 2, 4]), _log(rng, 1, 16384), _log(rng, 17, 2048)
        ctx_min = rng.randint(ctx // 4, ctx) if rng.random() < 0.7 else ctx
        new_min = rng.randint(max(1, new // 4), new) if step in ("prompt", "chunk") else new
        shape = dict(page=page, seqs=seqs, ctx_min=ctx_min, ctx=ctx, new_min=new_min, new=new, lens=lens)
        if op == "pages":
            c = _pages(**shape)
        elif op == "write":
            c = _write(dtype=rng.choice(["bf16", "bf16", "fp32"]), kv_heads=kv_heads, head_dim=rng.choice([128, 128, 64]), **shape)
        else:
            dtype, kv = rng.choice([("bf16", "dense")] * 3 + [("bf16", "fp8")] * 4 + [("bf16", "int8"), ("fp32", "dense")])
            window = 0 if kv == "fp8" and rng.random() < 0.5 else _log(rng, 32, 8192)
            c = _attend(dtype=dtype, kv=kv, heads=heads, kv_heads=kv_heads, head_dim=rng.choice([128, 128, 64]), window=window,
                        sinks=rng.choice([0, 0, 4, 4, rng.randint(1, 100)]) if window else 0, **shape)
            keys = max(_union(c, *l) for l in _lengths(c))
            if c["seqs"] * c["heads"] * c["new"] * keys > 1 << 31 or c["seqs"] * keys * kv_heads > 1 << 22:
                continue
        if _cost(c) <= most and sum(_held(c)) * page <= 1 << 20:
            return c


def _lengths(case):
    """Cached and new positions of each sequence."""
    r = random.Random(case["lens"])
    return [(r.randint(case["ctx_min"], case["ctx"]), r.randint(case["new_min"], case["new"])) for _ in range(case["seqs"])]


def _held(case):
    return [-(-(c + n) // case["page"]) for c, n in _lengths(case)]


def _first(case, c):
    """The first position of the window of the query at position c."""
    return max(0, c - case["window"] + 1) if case["window"] else 0


def _union(case, c, n):
    """Keys that any of a sequence's queries sees."""
    lo = _first(case, c)
    return c + n - lo + min(lo, case["sinks"])


def _seen(case, c, n):
    """Visible (query, key) pairs of a sequence."""
    total = 0
    for p in range(c, c + n):
        lo = _first(case, p)
        total += p + 1 - lo + min(lo, case["sinks"])
    return total


def work(case):
    lens, P = _lengths(case), case["page"]
    tokens = sum(n for _, n in lens)
    if case["op"] == "pages":
        # a count, a length and an offset per sequence; a position and a slot per token; a table entry and
        # a place of the stack per page, in both directions
        fresh = sum(-(-(c + n) // P) - -(-c // P) for c, n in lens)
        return {"bytes": 16.0 * len(lens) + 8.0 * tokens + 16.0 * fresh, "flops": float(tokens)}
    Hk, D = case["kv_heads"], case["head_dim"]
    size = DTYPES[case["dtype"]].itemsize
    if case["op"] == "write":
        # rows in, e4m3 rows and the scales of the touched pages out
        touched = sum((c + n - 1) // P - c // P + 1 for c, n in lens)
        return {"bytes": 2.0 * tokens * Hk * D * (size + 1) + 2.0 * touched * Hk * 4, "flops": 2.0 * tokens * Hk * D}
    row = {"dense": D * size, "int8": D + 4, "fp8": D + 4 / P}[case["kv"]]
    return {"bytes": 2.0 * Hk * row * sum(_union(case, c, n) for c, n in lens) + 2.0 * tokens * case["heads"] * D * size,
            "flops": 4.0 * D * case["heads"] * sum(_seen(case, c, n) for c, n in lens)}


# ---- inputs ---------------------------------------------------------------------------------

def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _flat(lists):
    return [x for l in lists for x in l]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(case=case, lens=_lengths(case))
    (_prepare_pages if case["op"] == "pages" else _prepare_step)(s, case, g)
    if own:
        _handles(s)
    return s


def _prepare_pages(s, case, g):
    """A pool whose sequences hold their cached positions, in pages in no order; the step's counts."""
    P, lens = case["page"], s["lens"]
    held, after = [-(-c // P) for c, _ in lens], _held(case)
    pages = sum(after) + 8
    ids = torch.randperm(pages, generator=g, device="cuda").to(torch.int32) + 1
    width, used = max(after), sum(held)
    at = torch.arange(width, device="cuda")
    first = torch.tensor([sum(held[:b]) for b in range(len(held))], device="cuda")
    s["tables"] = torch.where(at < torch.tensor(held, device="cuda")[:, None], ids[torch.clamp(first[:, None] + at, max=pages - 1)], 0).to(torch.int32).contiguous()
    s["free"] = torch.zeros(pages, dtype=torch.int32, device="cuda")
    s["free"][:pages - used] = ids[used:]
    s["free_count"] = _i32([pages - used])
    s["lengths"], s["before"] = (_i32([c for c, _ in lens]) for _ in range(2))
    s["counts"] = _i32([n for _, n in lens])
    tokens = sum(n for _, n in lens)
    s["positions"], s["slots"] = (torch.zeros(tokens, dtype=torch.int32, device="cuda") for _ in range(2))
    s["starts"] = torch.zeros(len(lens) + 1, dtype=torch.int32, device="cuda")
    s["short"] = torch.zeros(1, dtype=torch.int32, device="cuda")


def _prepare_step(s, case, g):
    """Block tables (1-based ids in no order; 0 for pages that no query sees, which a window gave back), the
    step's positions, offsets and slots, and the pools."""
    P, D, Hk, T, lens = case["page"], case["head_dim"], case["kv_heads"], DTYPES[case["dtype"]], s["lens"]
    window, sinks = case.get("window", 0), case.get("sinks", 0)
    per = _held(case)
    kept = []
    for (c, n), w in zip(lens, per):
        lo = max(0, c - window + 1) // P if window else 0
        kept.append([i for i in range(w) if i >= lo or i * P < sinks])
    pages = sum(len(k) for k in kept)
    ids = (torch.randperm(pages, generator=g, device="cuda") + 1).to(torch.int32)
    tables = torch.zeros((len(lens), max(per)), dtype=torch.int32, device="cuda")
    rows = torch.tensor(_flat([b] * len(k) for b, k in enumerate(kept)), device="cuda")
    tables[rows, torch.tensor(_flat(kept), device="cuda")] = ids
    counts = [n for _, n in lens]
    s.update(block_tables=tables, max_new=max(counts), tokens=sum(counts), pages=pages,
             positions=_i32(_flat(range(c, c + n) for c, n in lens)), starts=_i32([sum(counts[:b]) for b in range(len(counts) + 1)]))
    kv = case.get("kv", "fp8")
    if kv == "fp8":
        held = torch.randn((2, pages, Hk, P, D), generator=g, device="cuda", dtype=torch.bfloat16) * 64
        s["layer_q"] = held.to(E4M3).view(torch.uint8)
        # values of variance about 1, blocks that new rows make grow now and then
        s["layer_scale"] = _power(torch.randint(-8, -5, (2, pages, Hk), generator=g, device="cuda"))
    elif kv == "int8":
        s["layer_q"] = torch.empty((2, pages, Hk, P, D), dtype=torch.int8, device="cuda").random_(-127, 128, generator=g)
        s["layer_scale"] = torch.rand((2, pages, Hk, P), generator=g, device="cuda") * 0.02 + 0.005
        half = torch.rand(D // 2, generator=g, device="cuda") + 0.5
        s["smooth"] = torch.cat([half, half])
    else:
        s["k_pages"] = torch.randn((pages, Hk, P, D), generator=g, device="cuda", dtype=T)
        s["v_pages"] = torch.randn((pages, Hk, P, D), generator=g, device="cuda", dtype=T)
    if case["op"] == "attend":
        s["q"] = torch.randn((s["tokens"], case["heads"], D), generator=g, device="cuda", dtype=T)
        s["out"] = torch.zeros_like(s["q"])
        return
    # rows of unlike sizes, as layers give them
    for name in ("k", "v"):
        size = torch.exp(0.3 * torch.randn((s["tokens"], Hk, 1), generator=g, device="cuda"))
        s[name] = (torch.randn((s["tokens"], Hk, D), generator=g, device="cuda") * size).to(T)
    seq = torch.tensor(_flat([b] * n for b, n in enumerate(counts)), device="cuda")
    pos = s["positions"].long()
    page = tables[seq, pos // P].long() - 1
    s["slots"] = (page * P + pos % P + 1).to(torch.int32)
    # the pages that the step writes to, as a host's bookkeeping knows them, and each token's among them
    s["touched"], s["touched_of"] = torch.unique(page, return_inverse=True)


def _handles(s):
    """What a program of the framework keeps between steps: the cache's objects and workspaces."""
    ti, case = _ti(), s["case"]
    s["be"] = be = ti.HipBackend()
    if case["op"] == "pages":
        s["pool"] = ti.PagePool(s["free"], s["free_count"], s["tables"], s["lengths"], case["page"])
        return
    if "k_pages" in s:
        s["kc"], s["vc"] = s["k_pages"], s["v_pages"]
    elif "smooth" in s:
        s["kc"] = ti.Int8Pages(s["layer_q"], s["layer_scale"], s["smooth"], 0)
        s["vc"] = ti.Int8Pages(s["layer_q"], s["layer_scale"], torch.ones_like(s["smooth"]), 1)
    else:
        s["kc"], s["vc"] = (ti.Fp8Pages(s["layer_q"], s["layer_scale"], h) for h in (0, 1))
    if case["op"] == "attend":
        B, n = case["seqs"], s["max_new"]
        if case["window"]:
            s["workspace"] = ti.window_attention_workspace(be, s["q"], s["kc"], case["window"], case["sinks"], B, n)
        else:
            s["workspace"] = ti.attention_workspace(be, s["q"], s["kc"], B, n)


# ---- one pass -------------------------------------------------------------------------------

def run(s):
    op = s["case"]["op"]
    if own:
        return _own(s, op)
    return {"pages": _plain_pages, "write": _plain_write, "attend": _plain_attend}[op](s)


def _own(s, op):
    ti, be, case = _ti(), s["be"], s["case"]
    if op == "pages":
        ti.reserve_pages_(be, s["pool"], s["counts"], s["positions"], s["slots"], s["starts"], s["short"])
        ti.release_pages_(be, s["pool"], s["before"])
        return _books(s)
    if op == "write":
        ti.store_kv_(be, s["kc"], s["vc"], s["k"], s["v"], s["slots"])
        return s["layer_q"].view(E4M3), s["layer_scale"]
    scale = 1 / math.sqrt(case["head_dim"])
    if case["window"]:
        return ti.window_attention_(be, s["out"], s["workspace"], s["q"], s["kc"], s["vc"], s["block_tables"], s["positions"], scale,
                                    case["window"], case["sinks"], s["starts"], s["max_new"])
    return ti.paged_attention_(be, s["out"], s["workspace"], s["q"], s["kc"], s["vc"], s["block_tables"], s["positions"], scale, True,
                               s["starts"], s["max_new"])


def _books(s):
    return {k: s[k] for k in ("positions", "slots", "starts", "short", "tables", "lengths", "free", "free_count")}


def _power(e):
    """2^e as a float, for whole e in [-126, 127]."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _plain_pages(s):
    """Pages leave the stack in order of sequence and position, and come back in the opposite order."""
    P, tables, lengths, free = s["case"]["page"], s["tables"], s["lengths"], s["free"]
    at = torch.arange(tables.shape[1], device="cuda")
    # the step's positions: offsets, the sequence of each token, its place
    counts, old, have = s["counts"].long(), lengths.long(), s["free_count"].long()
    ends = torch.cumsum(counts, 0)
    held = (old + P - 1) // P
    need = (old + counts + P - 1) // P - held
    before = torch.cumsum(need, 0) - need
    total = need.sum()
    ok = total <= have
    s["short"].copy_(torch.clamp(total - have, min=0))
    place = at - held[:, None]
    new = (place >= 0) & (place < need[:, None]) & ok
    from_top = torch.clamp(have - 1 - before[:, None] - place, 0, free.numel() - 1)
    tables.copy_(torch.where(new, free[from_top], tables))
    lengths.add_(torch.where(ok, s["counts"], 0))
    s["free_count"].sub_(torch.where(ok, total, 0).to(torch.int32))
    s["starts"][1:] = torch.where(ok, ends, 0)
    token = torch.arange(s["positions"].numel(), device="cuda")
    seq = torch.clamp(torch.searchsorted(ends, token, right=True), max=len(counts) - 1)
    valid = (token < ends[-1]) & ok
    pos = old[seq] + token - (ends - counts)[seq]
    slot = (tables[seq, pos // P].long() - 1) * P + pos % P + 1
    s["positions"].copy_(torch.where(valid, pos, 0))
    s["slots"].copy_(torch.where(valid, slot, 0))
    # taken back: the pages past those that the kept positions need
    stay = (s["before"].long() + P - 1) // P
    gone = (at >= stay[:, None]) & (tables > 0)
    rank = torch.cumsum(gone.flatten(), 0)
    have = s["free_count"].long()
    to = torch.where(gone.flatten(), have + rank[-1] - rank, free.numel())
    grown = torch.cat([free, free[:1]])
    grown[to] = tables.flatten()
    free.copy_(grown[:-1])
    s["free_count"].add_(rank[-1].to(torch.int32))
    tables.masked_fill_(gone, 0)
    lengths.copy_(s["before"])
    return _books(s)


def _plain_write(s):
    P, idx, off = s["case"]["page"], s["touched_of"], ((s["slots"].long() - 1) % s["case"]["page"])
    U, Hk = len(s["touched"]), s["case"]["kv_heads"]
    fresh = torch.zeros(U, device="cuda").index_reduce_(0, idx, (off == 0).float(), "amax")[:, None] > 0
    for half, rows in ((0, s["k"]), (1, s["v"])):
        x = rows.float()
        most = torch.zeros((U, Hk), device="cuda").index_reduce_(0, idx, x.abs().amax(2), "amax")
        # the least e with most <= 448 2^e = 0.875 2^(e + 9)
        f, e = torch.frexp(most)
        e = torch.where(f <= 0.875, e - 9, e - 8)
        need = _power(torch.clamp(torch.where(most > 0, e, -120), -120, 120))
        old = s["layer_scale"][half][s["touched"]]
        new = torch.where(fresh, need, torch.maximum(old, need))
        held = s["layer_q"][half][s["touched"]].view(E4M3).float() * torch.where(fresh, 1.0, old / new)[..., None, None]
        held = held.to(E4M3).view(torch.uint8)
        held[idx, :, off] = (x / new[idx][..., None]).to(E4M3).view(torch.uint8)
        s["layer_q"][half][s["touched"]] = held
        s["layer_scale"][half][s["touched"]] = new
    return s["layer_q"].view(E4M3), s["layer_scale"]


def _plain_attend(s):
    case, P = s["case"], s["case"]["page"]
    Hq, Hk, D, W, S = case["heads"], case["kv_heads"], case["head_dim"], case["window"], case["sinks"]
    B, n, G = case["seqs"], s["max_new"], Hq // Hk
    starts = s["starts"].long()
    count = starts[1:] - starts[:-1]
    start = s["positions"].long()[starts[:-1]]
    # the keys that any query of a sequence sees: sinks before the first window, then up to the last position
    lo = torch.clamp(start - W + 1, min=0) if W else torch.zeros_like(start)
    extra = torch.clamp(lo, max=S)
    most = max(_union(case, *l) for l in s["lens"])
    at = torch.arange(most, device="cuda")[None]
    key = torch.where(at < extra[:, None], at, at - extra[:, None] + lo[:, None])
    real = key < (start + count)[:, None]
    key = torch.minimum(key, (start + count - 1)[:, None])
    page = torch.clamp(torch.gather(s["block_tables"].long(), 1, key // P) - 1, min=0)
    k, v = _values(s, 0, page, key % P), _values(s, 1, page, key % P)             # [B][keys][Hk][D]
    token = torch.clamp(starts[:-1, None] + torch.arange(n, device="cuda"), max=s["tokens"] - 1)
    q = s["q"][token].float()                                                       # [B][n][Hq][D]
    pos = start[:, None] + torch.arange(n, device="cuda")
    see = (key[:, None] <= pos[..., None]) & real[:, None]
    if W:
        see &= (key[:, None] > pos[..., None] - W) | (key[:, None] < S)
    rows = q.reshape(B, n, Hk, G, D).permute(0, 2, 3, 1, 4).reshape(B, Hk, G * n, D)
    score = torch.matmul(rows, k.permute(0, 2, 3, 1).contiguous()).view(B, Hk, G, n, most)
    score.mul_(1 / math.sqrt(D)).masked_fill_(~see[:, None, None], -math.inf)
    # rows past a sequence's own tokens see its last keys too; they are not kept
    score.sub_(torch.clamp(score.amax(4, keepdim=True), min=-1e30)).exp_()
    total = score.sum(4, keepdim=True).clamp_(min=1e-30)
    out = torch.matmul(score.view(B, Hk, G * n, most), v.permute(0, 2, 1, 3).contiguous()).view(B, Hk, G, n, D) / total
    out = out.permute(0, 3, 1, 2, 4).reshape(B * n, Hq, D)
    seq = torch.searchsorted(starts[1:].contiguous(), torch.arange(s["tokens"], device="cuda"), right=True)
    return out[seq * n + torch.arange(s["tokens"], device="cuda") - starts[seq]].to(s["q"].dtype)


def _values(s, half, page, off):
    """The cache's keys (half 0) or values at (page, offset): [..][Hk][D] in 32 bits."""
    if "k_pages" in s:
        return (s["k_pages"], s["v_pages"])[half][page, :, off].float()
    if "smooth" in s:
        x = s["layer_q"][half][page, :, off].float() * s["layer_scale"][half][page, :, off][..., None]
        return x * s["smooth"] if half == 0 else x
    return s["layer_q"][half][page, :, off].view(E4M3).float() * s["layer_scale"][half][page][..., None]


# ---- the same from the definitions, in 64 bits ----------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return {"pages": _exact_pages, "write": _exact_write, "attend": _exact_attend}[case["op"]](s, case)


def _exact_pages(s, case):
    """The stack and tables as lists, page by page."""
    P = case["page"]
    free = s["free"].tolist()
    count = int(s["free_count"])
    tables = s["tables"].tolist()
    positions, slots, starts = [], [], [0]
    taken = []
    for b, (c, n) in enumerate(s["lens"]):
        for p in range(c, c + n):
            if p % P == 0:
                count -= 1
                tables[b][p // P] = free[count]
                taken.append((b, p // P))
            positions.append(p)
            slots.append((tables[b][p // P] - 1) * P + p % P + 1)
        starts.append(len(slots))
    for b, i in reversed(taken):
        free[count] = tables[b][i]
        count += 1
        tables[b][i] = 0
    return {"positions": _i32(positions), "slots": _i32(slots), "starts": _i32(starts), "short": _i32([0]), "tables": _i32(tables),
            "lengths": s["before"], "free": _i32(free), "free_count": _i32([count])}


def _nearest(x):
    """The e4m3 value nearest to x (ties to the even one), for |x| <= 448, in 64 bits."""
    step = torch.pow(2.0, torch.clamp(torch.floor(torch.log2(torch.clamp(x.abs(), min=2.0 ** -20))), min=-6) - 3)
    return torch.round(x / step) * step


def _exact_write(s, case):
    """Block by block: the step's least power of two, the held rows made smaller, the new rows rounded."""
    P, slots = case["page"], s["slots"].long() - 1
    q, scale = s["layer_q"].clone().view(E4M3).double(), s["layer_scale"].double()
    order = torch.argsort(s["touched_of"], stable=True)
    sizes = torch.bincount(s["touched_of"], minlength=len(s["touched"])).tolist()
    at = 0
    for page, n in zip(s["touched"].tolist(), sizes):
        tokens = order[at:at + n]
        at += n
        off = slots[tokens] % P
        begins = bool((off == 0).any())
        for half, rows in ((0, s["k"]), (1, s["v"])):
            x = rows[tokens].double()                                                # [n][Hk][D]
            most = x.abs().amax((0, 2))
            need = torch.pow(2.0, torch.ceil(torch.log2(most / 448)))
            need = torch.where(need / 2 * 448 >= most, need / 2, torch.where(need * 448 < most, need * 2, need))
            new = need if begins else torch.maximum(need, scale[half, page])
            if not begins:
                q[half, page] = _nearest(q[half, page] * (scale[half, page] / new)[:, None, None])
            q[half, page, :, off] = _nearest(x / new[None, :, None]).permute(1, 0, 2)
            scale[half, page] = new
    return q, scale


def _exact_attend(s, case):
    P, Hk, D, W = case["page"], case["kv_heads"], case["head_dim"], case["window"]
    G = case["heads"] // Hk
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    at = 0
    for b, (c, n) in enumerate(s["lens"]):
        lo = _first(case, c)
        key = torch.cat([torch.arange(min(lo, case["sinks"]), device="cuda"), torch.arange(lo, c + n, device="cuda")])
        page, off = s["block_tables"][b].long()[key // P] - 1, key % P
        for h in range(Hk):
            k, v = (_row(s, half, page, h, off) for half in (0, 1))
            for t in range(0, n, 512):
                m = min(512, n - t)
                rows = s["q"][at + t:at + t + m, h * G:(h + 1) * G].double().reshape(m * G, D)
                score = (rows @ k.T).reshape(m, G, -1) / math.sqrt(D)
                p = torch.arange(c + t, c + t + m, device="cuda")[:, None]
                hidden = key > p
                if W:
                    hidden |= (key <= p - W) & (key >= case["sinks"])
                weight = torch.softmax(score.masked_fill(hidden[:, None], -math.inf), 2)
                out[at + t:at + t + m, h * G:(h + 1) * G] = (weight.reshape(m * G, -1) @ v).reshape(m, G, D)
        at += n
    return out


def _row(s, half, page, h, off):
    if "k_pages" in s:
        return (s["k_pages"], s["v_pages"])[half][page, h, off].double()
    if "smooth" in s:
        x = s["layer_q"][half][page, h, off].double() * s["layer_scale"][half][page, h, off].double()[:, None]
        return x * s["smooth"].double() if half == 0 else x
    return s["layer_q"][half][page, h, off].view(E4M3).double() * s["layer_scale"][half][page, h].double()[:, None]
