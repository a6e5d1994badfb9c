"""Performance cases of the long-context and speculative operators: bounds of the keys of each
cache page, the pages that a query keeps by them, attention over those pages alone, and the
verification of drafted tokens.

A step of a long chat runs them in this order. `update_key_bounds_` refreshes the bounds of
the pages that the step's new keys went to, `select_pages_` scores every page of a sequence by
the largest product that a key inside the bounds could have with the query and keeps the best,
`sparse_attention_` attends to the kept pages, and `verify_draft_` turns the target's and the
drafter's probabilities into accepted tokens.

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


def _ti():
    path = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "tileinfer.jl_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import tileinfer_hip
    return tileinfer_hip


# ---- cases ----------------------------------------------------------------------------------

def _bounds(name=None, **kw):
    # cached positions per sequence between ctx_min and ctx, new ones between new_min and new
    c = dict(op="bounds", dtype="bf16", kv="dense", kv_heads=8, head_dim=128, page=64, seqs=1, ctx_min=0, ctx=0, new_min=1,
             new=1, lens=1)
    c.update(kw)
    return c if name is None else dict(c, name=name)


def _select(name=None, **kw):
    # keep: pages per query token and KV head, the first `sinks` and the last `window` among them
    c = dict(op="select", dtype="bf16", heads=32, kv_heads=8, head_dim=128, page=64, seqs=1, ctx_min=0, ctx=0, new_min=1,
             new=1, keep=64, sinks=1, window=2, causal=True, lens=1)
    c.update(kw)
    return c if name is None else dict(c, name=name)


def _attend(name=None, **kw):
    # tables of `keep` pages per query token and KV head; one token shares most pages with the last
    c = dict(op="attend", dtype="bf16", kv="dense", heads=32, kv_heads=8, head_dim=128, page=64, seqs=1, ctx_min=0, ctx=0,
             new=1, keep=64, lens=1)
    c.update(kw)
    return c if name is None else dict(c, name=name)


def _verify(name=None, **kw):
    c = dict(op="verify", dtype="fp32", seqs=1, drafted_min=4, drafted=4, vocab=32000, greedy=False, noise=0.5, lens=1)
    c.update(kw)
    return c if name is None else dict(c, name=name)


def listed():
    return [
        # one token of each chat of a serving batch: the pages that the tokens went to
        _bounds("bounds_b32", seqs=32, ctx_min=1023, ctx=8191),
        # prompts of a batch, 16-token pages
        _bounds("bounds_prompts_b8", page=16, seqs=8, new_min=300, new=4000),
        # a chunk of a long document on an INT8 cache
        _bounds("bounds_chunk_int8", kv="int8", page=64, ctx_min=30001, ctx=30001, new_min=4096, new=4096),
        # one chat with a long context, one token: the pages of each KV head
        _select("select_token_32k", ctx_min=32767, ctx=32767),
        # a serving batch of long and short contexts, 16-token pages
        _select("select_ragged_b32", page=16, seqs=32, ctx_min=2000, ctx=32767, keep=128, window=8),
        # a chunk of a long document, each token with pages of its own
        _select("select_chunk_512_on_64k", ctx_min=65536, ctx=65536, new_min=512, new=512),
        # one chat, one token over 4096 of its 32768 positions
        _attend("attend_token_32k", ctx_min=32767, ctx=32767),
        # a serving batch: the ordinary call
        _attend("attend_b32_32k", seqs=32, ctx_min=20000, ctx=32767),
        # drafted blocks of 16 tokens on an INT8 cache of 16-token pages
        _attend("attend_verify_int8_b8", kv="int8", page=16, seqs=8, ctx_min=8000, ctx=16383, new=16, keep=128),
        # a chunk of a document, each token over pages of its own
        _attend("attend_chunk_512", ctx_min=30000, ctx=30000, new=512, keep=32),
        # one chat, four drafted tokens, a small vocabulary: the smallest call
        _verify("verify_b1"),
        # a serving batch of eight drafted tokens and a large vocabulary
        _verify("verify_b64", seqs=64, drafted_min=2, drafted=8, vocab=151936),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 50)


def draw(rng):
    most = max(_cost(c) for c in listed())
    heads, kv_heads = rng.choice([(32, 8), (32, 8), (16, 8), (24, 8), (32, 4), (64, 8), (8, 8)])
    while True:
        op = rng.choice(["bounds", "select", "attend", "verify"])
        lens = rng.randrange(1 << 30)
        if op == "verify":
            drafted = rng.randint(1, 16)
            c = _verify(seqs=_log(rng, 1, 128), drafted=drafted, drafted_min=rng.randint(0, drafted), vocab=_log(rng, 1000, 160000),
                        dtype=rng.choice(["fp32", "fp32", "bf16"]), greedy=rng.random() < 0.25, noise=rng.choice([0.2, 0.5, 1.0]),
                        lens=lens)
            if _cost(c) <= most:
                return c
            continue
        dtype, kv = rng.choice([("bf16", "dense")] * 5 + [("bf16", "int8")] * 3 + [("fp32", "dense")])
        shape = dict(dtype=dtype, kv_heads=kv_heads, head_dim=rng.choice([128, 128, 128, 64]), page=rng.choice([16, 64, 64, 32]),
                     lens=lens)
        step = rng.choice(["token", "token", "block", "chunk"])
        if step == "token":
            seqs, ctx, new = _log(rng, 1, 64), _log(rng, 500, 65536), 1
        elif step == "block":
            seqs, ctx, new = _log(rng, 1, 16), _log(rng, 500, 32768), rng.randint(2, 16)
        else:
            seqs, ctx, new = 1, _log(rng, 500, 65536), _log(rng, 17, 512)
        ctx_min = rng.randint(ctx // 4, ctx) if rng.random() < 0.7 else ctx
        keep = max(4, min(_log(rng, 256, 4096) // shape["page"], 256))
        if op == "bounds":
            if step == "chunk":
                seqs, new = rng.randint(1, 8), _log(rng, 17, 4096)
            c = _bounds(kv=kv, seqs=seqs, ctx_min=ctx_min, ctx=ctx, new_min=rng.randint(max(1, new // 4), new), new=new, **shape)
        elif op == "select":
            window = rng.randint(1, max(1, keep // 8))
            c = _select(heads=heads, seqs=seqs, ctx_min=ctx_min, ctx=ctx, new_min=rng.randint(max(1, new // 2), new), new=new,
                        keep=keep, sinks=rng.randint(0, 2), window=window, causal=rng.random() < 0.8, **shape)
        else:
            c = _attend(kv=kv, heads=heads, seqs=seqs, ctx_min=ctx_min, ctx=ctx, new=new, keep=keep, **shape)
        if _cost(c) <= most and sum(_pages(c)) * c["page"] * c["kv_heads"] * c["head_dim"] < 3 << 29:
            return c


def _lengths(case):
    """Cached and new positions of each sequence."""
    r = random.Random(case["lens"])
    lo = case.get("new_min", case["new"])
    return [(r.randint(case["ctx_min"], case["ctx"]), r.randint(lo, case["new"])) for _ in range(case["seqs"])]


def _drafted(case):
    r = random.Random(case["lens"])
    return [r.randint(case["drafted_min"], case["drafted"]) for _ in range(case["seqs"])]


def _pages(case):
    return [-(-(c + n) // case["page"]) for c, n in _lengths(case)]


def _key_bytes(case):
    return case["head_dim"] + 4 if case["kv"] == "int8" else case["head_dim"] * DTYPES[case["dtype"]].itemsize


def work(case):
    op = case["op"]
    if op == "verify":
        # the acceptance reads one value per drafted token; the token after it needs the row of the
        # target's probabilities and, where a draft was rejected, the drafter's
        rows = 1 if case["greedy"] else 2
        n = sum(_drafted(case))
        size = DTYPES[case["dtype"]].itemsize
        return {"bytes": case["seqs"] * (rows * case["vocab"] * size + 4 * (case["drafted"] + 2)) + n * (8 + 2 * size),
                "flops": case["seqs"] * case["vocab"] * 3.0}
    Hk, D, P = case["kv_heads"], case["head_dim"], case["page"]
    lens = _lengths(case)
    if op == "bounds":
        # the keys of the touched pages (those before the step that share its first page too), and the bounds
        keys = sum(n + c % P for c, n in lens)
        pages = sum((c + n - 1) // P - c // P + 1 for c, n in lens)
        return {"bytes": Hk * (keys * _key_bytes(case) + pages * (2 * D + 4)), "flops": Hk * keys * 2.0 * D}
    G, size = case["heads"] // Hk, DTYPES[case["dtype"]].itemsize
    tokens = sum(n for _, n in lens)
    if op == "select":
        seen = sum(min(c + (t if case["causal"] else n - 1), c + n - 1) // P + 1 for c, n in lens for t in range(n))
        return {"bytes": sum(_pages(case)) * Hk * (2 * D + 4) + tokens * (case["heads"] * D * size + Hk * 4 * (case["keep"] + 1)),
                "flops": Hk * G * 2.0 * D * 2 * seen}
    # a page that several tokens of a sequence keep is read once: about a tenth of the sequence's
    # pages beside those of one token (see _pick)
    keys = sum(min(case["keep"] * P, c + t + 1) for c, n in lens for t in range(n))
    read = sum(min(n * case["keep"] * P, case["keep"] * P + (c + n) // 10 if n > 1 else c + n, c + n) for c, n in lens)
    return {"bytes": 2 * Hk * read * _key_bytes(case) + tokens * (2 * case["heads"] * D * size + Hk * 4 * (case["keep"] + 1)),
            "flops": 4.0 * D * case["heads"] * keys}


# ---- inputs ---------------------------------------------------------------------------------

def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _batch(case, g):
    """Block tables (1-based page ids, in no order, zero-padded), positions and query offsets."""
    lens, per = _lengths(case), _pages(case)
    pages, width = sum(per), max(per)
    ids = (torch.randperm(pages, generator=g, device="cuda") + 1).to(torch.int32)
    first = torch.tensor([sum(per[:b]) for b in range(len(per))], device="cuda")
    at = torch.arange(width, device="cuda")
    held = at[None] < torch.tensor(per, device="cuda")[:, None]
    tables = torch.where(held, ids[torch.clamp(first[:, None] + at, max=pages - 1)], 0).to(torch.int32).contiguous()
    counts = [n for _, n in lens]
    return dict(block_tables=tables, pages=pages, lens=lens, counts=counts, max_new=max(counts),
                positions=_i32([c + t for c, n in lens for t in range(n)]),
                starts=_i32([sum(counts[:b]) for b in range(len(counts) + 1)]))


def _pools(case, pages, g):
    T, P, D, Hk = DTYPES[case["dtype"]], case["page"], case["head_dim"], case["kv_heads"]
    if case["kv"] == "int8":
        q = torch.empty((2, pages, Hk, P, D), dtype=torch.int8, device="cuda").random_(-127, 128, generator=g)
        s = torch.rand((2, pages, Hk, P), generator=g, device="cuda") * 0.02 + 0.01
        half = torch.rand(D // 2, generator=g, device="cuda") + 0.5
        return dict(layer_q=q, layer_scale=s, smooth=torch.cat([half, half]))
    k = torch.randn((pages, Hk, P, D), generator=g, device="cuda", dtype=T)
    v = torch.randn((pages, Hk, P, D), generator=g, device="cuda", dtype=T)
    return dict(k_pages=k, v_pages=v)


def _pick(case, b, g):
    """Tables of kept pages as a selection leaves them: the first and the last page and others in
    order of position, most of them shared by the tokens of a sequence; and their lengths."""
    P, Hk, keep, lens = case["page"], case["kv_heads"], case["keep"], b["lens"]
    counts = torch.tensor(b["counts"], device="cuda")
    seq = torch.repeat_interleave(torch.arange(len(lens), device="cuda"), counts, output_size=sum(b["counts"]))
    pos = b["positions"].long()
    width = b["block_tables"].shape[1]
    liked = torch.rand((len(lens), Hk, width), generator=g, device="cuda")
    own_part = torch.rand((len(seq), Hk, width), generator=g, device="cuda")
    rank = liked[seq] + 0.1 * own_part
    at = torch.arange(width, device="cuda")
    seen = (pos // P + 1)[:, None, None]
    rank = torch.where((at == 0) | (at == seen - 1), 10.0, rank)
    rank = torch.where(at < seen, rank, -1.0)
    kept = torch.clamp(seen[..., 0], max=keep)
    top = torch.topk(rank, min(keep, width), dim=2).indices
    order = torch.arange(top.shape[2], device="cuda")
    top = torch.sort(torch.where(order < kept[..., None], top, 1 << 30), dim=2).values
    ids = torch.gather(b["block_tables"][seq][:, None].expand(-1, Hk, -1), 2, torch.clamp(top, max=width - 1))
    tables = torch.zeros((len(seq), Hk, keep), dtype=torch.int32, device="cuda")
    tables[:, :, :top.shape[2]] = torch.where(top < 1 << 30, ids, 0)
    lengths = ((kept - 1) * P + (pos % P + 1)[:, None]).expand(-1, Hk).to(torch.int32).contiguous()
    return tables, lengths


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(case=case)
    if case["op"] == "verify":
        B, N, V = case["seqs"], case["drafted"], case["vocab"]
        logits = torch.randn((B, N + 1, V), generator=g, device="cuda") * 3
        s["target"] = torch.softmax(logits, 2).to(DTYPES[case["dtype"]])
        near = torch.softmax(logits[:, :N] + case["noise"] * torch.randn((B, N, V), generator=g, device="cuda"), 2)
        if case["greedy"]:      # a drafter that gives its most likely token and no probabilities
            s["draft"], s["drafted"] = None, near.argmax(2).to(torch.int32)
        else:
            s["draft"] = near.to(DTYPES[case["dtype"]])
            s["drafted"] = torch.multinomial(near.reshape(B * N, V), 1, generator=g).reshape(B, N).to(torch.int32)
        s["uniforms"] = torch.rand((B, N + 1), generator=g, device="cuda")
        s["counts"] = _i32(_drafted(case))
        s["accepted"] = torch.zeros(B, dtype=torch.int32, device="cuda")
        s["tokens"] = torch.zeros((B, N + 1), dtype=torch.int32, device="cuda")
    else:
        b = _batch(case, g)
        s.update(b)
        D, Hk, T = case["head_dim"], case["kv_heads"], DTYPES[case["dtype"]]
        tokens = len(b["positions"])
        if case["op"] in ("bounds", "attend"):
            s.update(_pools(case, b["pages"], g))
        if case["op"] in ("bounds", "select"):
            # bounds of pages as random keys about a page's own mean leave them
            mid = torch.randn((b["pages"], Hk, 1, D), generator=g, device="cuda") * 25
            out = torch.rand((b["pages"], Hk, 2, D), generator=g, device="cuda") * 40 + 20
            sign = torch.tensor([1.0, -1.0], device="cuda")[:, None]
            s["bounds"] = torch.clamp(torch.round(mid + sign * out), -127, 127).to(torch.int8)
            s["scale"] = _power(torch.randint(-6, -4, (b["pages"], Hk), generator=g, device="cuda"))
        if case["op"] == "bounds":
            touched = [(i, p) for i, (c, n) in enumerate(b["lens"]) for p in range(c // case["page"], (c + n - 1) // case["page"] + 1)]
            s["touched_seq"], s["touched_page"] = (torch.tensor(x, device="cuda") for x in zip(*touched))
        else:
            s["q"] = torch.randn((tokens, case["heads"], D), generator=g, device="cuda", dtype=T)
            if case["op"] == "select":
                s["tables"] = torch.zeros((tokens, Hk, case["keep"]), dtype=torch.int32, device="cuda")
                s["lengths"] = torch.zeros((tokens, Hk), dtype=torch.int32, device="cuda")
            else:
                s["tables"], s["lengths"] = _pick(case, b, g)
                s["out"] = torch.zeros_like(s["q"])
    if own:
        _handles(s)
    return s


def _handles(s):
    """What a program of the framework keeps between steps: the cache's objects and workspaces."""
    ti, case = _ti(), s["case"]
    s["be"] = be = ti.HipBackend()
    if "layer_q" in s:
        D = s["smooth"].numel()
        s["k"] = ti.Int8Pages(s["layer_q"], s["layer_scale"], s["smooth"], 0)
        s["v"] = ti.Int8Pages(s["layer_q"], s["layer_scale"], torch.ones(D, device="cuda"), 1)
    elif "k_pages" in s:
        s["k"], s["v"] = s["k_pages"], s["v_pages"]
    if "bounds" in s:
        s["kb"] = ti.KeyBounds(s["bounds"], s["scale"], case["page"])
    if case["op"] == "select":
        s["workspace"] = ti.select_pages_workspace(be, s["q"], s["kb"], s["block_tables"])
    elif case["op"] == "attend":
        s["workspace"] = ti.sparse_attention_workspace(be, s["q"], s["k"], s["tables"], s["max_new"])
    elif case["op"] == "verify":
        s["workspace"] = ti.verify_draft_workspace(be, s["target"])


# ---- one pass -------------------------------------------------------------------------------

def run(s):
    op = s["case"]["op"]
    if own:
        return _own(s, op)
    return {"bounds": _plain_bounds, "select": _plain_select, "attend": _plain_attend, "verify": _plain_verify}[op](s)


def _own(s, op):
    ti, be, case = _ti(), s["be"], s["case"]
    if op == "bounds":
        ti.update_key_bounds_(be, s["kb"], s["k"], s["v"], s["block_tables"], s["positions"], s["starts"], s["max_new"])
        return s["bounds"], s["scale"]
    if op == "select":
        ti.select_pages_(be, s["tables"], s["lengths"], s["workspace"], s["q"], s["kb"], s["block_tables"], s["positions"],
                         case["sinks"], case["window"], case["causal"], s["starts"], s["max_new"])
        return s["tables"], s["lengths"]
    if op == "attend":
        return ti.sparse_attention_(be, s["out"], s["workspace"], s["q"], s["k"], s["v"], s["tables"], s["lengths"],
                                    1 / math.sqrt(case["head_dim"]), s["starts"], s["max_new"])
    ti.verify_draft_(be, s["accepted"], s["tokens"], s["workspace"], s["drafted"], s["target"], s["draft"], s["uniforms"], s["counts"])
    return s["accepted"], s["tokens"]


def _exponent(a):
    """The least e in [-126, 127] with a <= 127 2^e (a >= 0 and finite)."""
    f, x = torch.frexp(a)
    e = torch.where(f <= 127 / 128, x - 7, x - 6)
    return torch.clamp(torch.where(a > 0, e, -126), min=-126)


def _power(e):
    """2^e as a float, for whole e in [-126, 127]."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _plain_bounds(s):
    """Largest and smallest key element of each touched page, rounded outward to whole multiples of
    the page's power of two (whole numbers and powers of two: no rounding in 32 bits)."""
    P, seq, page = s["case"]["page"], s["touched_seq"], s["touched_page"]
    ids = (s["block_tables"][seq, page] - 1).long()
    starts = s["starts"].long()
    count = starts[1:] - starts[:-1]
    length = s["positions"].long()[starts[:-1]] + count
    valid = page[:, None] * P + torch.arange(P, device="cuda") < length[seq][:, None]
    valid = valid[:, None, :, None]
    if "layer_q" in s:
        k = s["layer_q"][0][ids].float() * s["layer_scale"][0][ids][..., None] * s["smooth"]
    else:
        k = s["k_pages"][ids].float()
    hi = torch.where(valid, k, -math.inf).amax(2)
    lo = torch.where(valid, k, math.inf).amin(2)
    e = _exponent(torch.maximum(hi.abs(), lo.abs()).amax(2))
    back = _power(-e)[..., None]
    s["bounds"][ids] = torch.stack([torch.ceil(hi * back), torch.floor(lo * back)], 2).to(torch.int8)
    s["scale"][ids] = _power(e)
    return s["bounds"], s["scale"]


def _sequences(s):
    """The sequence, the first position of its step and the step's tokens, for each token."""
    starts = s["starts"].long()
    tokens = torch.arange(s["positions"].numel(), device="cuda")
    seq = (tokens[:, None] >= starts[None, 1:]).sum(1)
    first = starts[seq]
    start = s["positions"].long()[first]
    return seq, start, tokens - first, starts[seq + 1] - first


def _plain_select(s):
    """Products of whole numbers below 2^22, summed exactly in 32 bits whatever the order."""
    case, q = s["case"], s["q"].float()
    T, Hq, D = q.shape
    Hk, P, keep = case["kv_heads"], case["page"], case["keep"]
    e = _exponent(q.abs().amax(2, keepdim=True))
    whole = torch.round(q * _power(-e))
    both = torch.cat([torch.clamp(whole, min=0), torch.clamp(whole, max=0)], 2).reshape(T, Hk, Hq // Hk, 2 * D)
    seq, start, at, count = _sequences(s)
    ids = torch.clamp(s["block_tables"].long() - 1, min=0)
    page = s["bounds"][ids].float()[seq]                                    # [T][width][Hk][2][D]
    width = page.shape[1]
    page = page.permute(0, 2, 3, 4, 1).reshape(T, Hk, 2 * D, width)
    score = (torch.matmul(both, page) * _power(e).reshape(T, Hk, Hq // Hk, 1)).amax(2)
    score = score * s["scale"][ids].permute(0, 2, 1)[seq]
    last = start + (at if case["causal"] else count - 1)
    seen = torch.clamp(last // P + 1, max=width)[:, None, None]
    index = torch.arange(width, device="cuda")
    kind = torch.where(index >= seen, 2, torch.where((index < case["sinks"]) | (index >= seen - case["window"]), 0, 1))
    by_score = torch.sort(score, dim=2, descending=True, stable=True).indices
    by_kind = torch.sort(torch.gather(kind.expand_as(score), 2, by_score), dim=2, stable=True).indices
    best = torch.gather(by_score, 2, by_kind)[..., :keep]
    kept = torch.clamp(seen, max=keep)
    order = torch.arange(best.shape[2], device="cuda")
    best = torch.sort(torch.where(order < kept, best, width), dim=2).values
    found = torch.gather(s["block_tables"][seq][:, None].expand(-1, Hk, -1), 2, torch.clamp(best, max=width - 1))
    tables = torch.zeros((T, Hk, keep), dtype=torch.int32, device="cuda")
    tables[:, :, :best.shape[2]] = torch.where(best < width, found, 0)
    lengths = (kept[..., 0] - 1) * P + (last + 1 - (seen[:, 0, 0] - 1) * P)[:, None]
    return tables, lengths.expand(-1, Hk).to(torch.int32).contiguous()


def _plain_attend(s):
    case, q = s["case"], s["q"].float()
    T, Hq, D = q.shape
    Hk, P, keep = case["kv_heads"], case["page"], case["keep"]
    ids, head = torch.clamp(s["tables"].long() - 1, min=0), torch.arange(Hk, device="cuda")[None, :, None]
    if "layer_q" in s:
        k = s["layer_q"][0][ids, head].float() * s["layer_scale"][0][ids, head][..., None] * s["smooth"]
        v = s["layer_q"][1][ids, head].float() * s["layer_scale"][1][ids, head][..., None]
    else:
        k, v = s["k_pages"][ids, head].float(), s["v_pages"][ids, head].float()
    k, v = k.reshape(T, Hk, keep * P, D), v.reshape(T, Hk, keep * P, D)
    score = torch.matmul(q.reshape(T, Hk, Hq // Hk, D), k.transpose(2, 3)) * (1 / math.sqrt(D))
    seen = torch.arange(keep * P, device="cuda") < s["lengths"][..., None, None]
    score = torch.where(seen, score, -math.inf)
    weight = torch.exp(score - score.amax(3, keepdim=True))
    out = torch.matmul(weight, v) / weight.sum(3, keepdim=True)
    return out.reshape(T, Hq, D).to(s["q"].dtype)


def _plain_verify(s):
    """Probabilities are summed in 64 bits: the drawn token sits between two partial sums."""
    p, x, u, count = s["target"], s["drafted"].long(), s["uniforms"].double(), s["counts"].long()
    B, N = x.shape
    at = torch.arange(N, device="cuda")
    likely = torch.gather(p[:, :N], 2, x[..., None])[..., 0].double()
    given = 1.0 if s["draft"] is None else torch.gather(s["draft"], 2, x[..., None])[..., 0].double()
    ok = (u[:, :N] * given < likely) & (at < count[:, None])
    accepted = torch.cumprod(ok.long(), 1).sum(1)
    rows = torch.arange(B, device="cuda")
    weight = p[rows, accepted].double()
    below = torch.clamp(accepted, max=N - 1)
    rejected = (accepted < count)[:, None]
    if s["draft"] is None:
        gone = rejected & (torch.arange(weight.shape[1], device="cuda") == x[rows, below][:, None])
        weight = torch.where(gone, 0.0, weight)
    else:
        weight = torch.where(rejected, torch.clamp(weight - s["draft"][rows, below].double(), min=0), weight)
    total = torch.cumsum(weight, 1)
    hit = (total > u[:, N:] * total[:, -1:]) & (weight > 0)
    token = hit.to(torch.int8).argmax(1)
    index = torch.arange(N + 1, device="cuda")
    drafted = torch.cat([x, x[:, :1]], 1)
    tokens = torch.where(index < accepted[:, None], drafted, torch.where(index == accepted[:, None], token[:, None], -1))
    return accepted.to(torch.int32), tokens.to(torch.int32)


# ---- the same from the definitions, in 64 bits ----------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return {"bounds": _exact_bounds, "select": _exact_select, "attend": _exact_attend, "verify": _exact_verify}[case["op"]](s, case)


def _least_power(a):
    """The least power of two, from 2^-126 on, that 127 times it is no less than a."""
    p = torch.pow(2.0, torch.ceil(torch.log2(torch.clamp(a, min=2.0 ** -140) / 127)))
    p = torch.where(p / 2 * 127 >= a, p / 2, torch.where(p * 127 < a, p * 2, p))
    return torch.clamp(p, min=2.0 ** -126)


def _exact_bounds(s, case):
    P, bounds, scale = case["page"], s["bounds"].clone(), s["scale"].clone()
    tables = s["block_tables"].tolist()
    for b, (c, n) in enumerate(s["lens"]):
        for p in range(c // P, (c + n - 1) // P + 1):
            i, held = tables[b][p] - 1, min(P, c + n - p * P)
            if case["kv"] == "int8":
                k = s["layer_q"][0, i, :, :held].double() * s["layer_scale"][0, i, :, :held, None].double() * s["smooth"].double()
            else:
                k = s["k_pages"][i, :, :held].double()
            step = _least_power(k.abs().flatten(1).amax(1))
            bounds[i, :, 0] = torch.ceil(k.amax(1) / step[:, None]).to(torch.int8)
            bounds[i, :, 1] = torch.floor(k.amin(1) / step[:, None]).to(torch.int8)
            scale[i] = step.float()
    return bounds, scale


def _exact_select(s, case):
    Hk, P, keep, D = case["kv_heads"], case["page"], case["keep"], case["head_dim"]
    G = case["heads"] // Hk
    q = s["q"].double()
    step = _least_power(q.abs().amax(2))
    whole = torch.round(q / step[..., None])
    tables = torch.zeros_like(s["tables"])
    lengths = torch.zeros_like(s["lengths"])
    t0 = 0
    for b, (c, n) in enumerate(s["lens"]):
        ids = s["block_tables"][b].long()
        ids = ids[ids > 0] - 1
        top = s["bounds"][ids].double()                                     # [pages][Hk][2][D]
        for t in range(n):
            last = c + (t if case["causal"] else n - 1)
            seen = min(last // P + 1, len(ids))
            w = whole[t0 + t].reshape(1, Hk, G, D)
            for_hi, for_lo = torch.where(w > 0, w, 0.0), torch.where(w < 0, w, 0.0)
            dots = (for_hi * top[:seen, :, None, 0]).sum(3) + (for_lo * top[:seen, :, None, 1]).sum(3)
            score = (dots * step[t0 + t].reshape(1, Hk, G)).amax(2) * s["scale"][ids[:seen]].double()
            forced = torch.zeros(seen, dtype=torch.bool, device="cuda")
            forced[:case["sinks"]] = True
            forced[max(0, seen - case["window"]):] = True
            score[forced] = math.inf
            kept = min(keep, seen)
            chosen = torch.sort(torch.argsort(-score, dim=0, stable=True)[:kept], dim=0).values
            tables[t0 + t, :, :kept] = (ids[chosen] + 1).t().to(torch.int32)
            lengths[t0 + t] = (kept - 1) * P + last + 1 - (seen - 1) * P
        t0 += n
    return tables, lengths


def _exact_attend(s, case):
    Hk, P, D = case["kv_heads"], case["page"], case["head_dim"]
    G = case["heads"] // Hk
    out, lengths = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda"), s["lengths"].tolist()
    for t in range(s["q"].shape[0]):
        for h in range(Hk):
            at = torch.arange(lengths[t][h], device="cuda")
            page = s["tables"][t, h].long()[at // P] - 1
            if case["kv"] == "int8":
                k = s["layer_q"][0, page, h, at % P].double() * s["layer_scale"][0, page, h, at % P, None].double() * s["smooth"].double()
                v = s["layer_q"][1, page, h, at % P].double() * s["layer_scale"][1, page, h, at % P, None].double()
            else:
                k, v = s["k_pages"][page, h, at % P].double(), s["v_pages"][page, h, at % P].double()
            rows = s["q"][t, h * G:(h + 1) * G].double()
            score = (rows[:, None] * k).sum(2) / math.sqrt(D)
            weight = torch.exp(score - score.max(1, keepdim=True).values)
            weight = weight / weight.sum(1, keepdim=True)
            out[t, h * G:(h + 1) * G] = (weight[:, :, None] * v).sum(1)
    return out


def _exact_verify(s, case):
    counts = s["counts"].tolist()
    accepted, tokens = torch.zeros_like(s["accepted"]), torch.full_like(s["tokens"], -1)
    for b, n in enumerate(counts):
        a = 0
        while a < n:
            x = int(s["drafted"][b, a])
            given = 1.0 if s["draft"] is None else float(s["draft"][b, a, x])
            if not float(s["uniforms"][b, a]) * given < float(s["target"][b, a, x]):
                break
            tokens[b, a] = x
            a += 1
        w = s["target"][b, a].double()
        if a < n:
            if s["draft"] is None:
                w[int(s["drafted"][b, a])] = 0.0
            else:
                w = torch.relu(w - s["draft"][b, a].double())
        goal = float(s["uniforms"][b, -1]) * float(w.sum())
        held = torch.nonzero(w)[:, 0]
        below = int((torch.cumsum(w[held], 0) <= goal).sum())
        accepted[b], tokens[b, a] = a, held[min(below, len(held) - 1)].to(torch.int32)
    return accepted, tokens
