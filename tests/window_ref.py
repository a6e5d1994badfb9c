"""Definitions in 64 bits of the 8-bit block cache, of attention with a sliding window and of the page bookkeeping
of a step, and caches to run them on. numpy on the CPU; nothing of the kernels."""
from __future__ import annotations

import math

import numpy as np
import torch

import tileinfer_hip as ti

BE = None


def i32(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")


# ---- e4m3 ---------------------------------------------------------------------------------------

def _value(code):
    e, m = code >> 3 & 15, code & 7
    return math.ldexp(m, -9) if e == 0 else math.ldexp(8 + m, e - 10)


E4M3 = np.array([_value(c) for c in range(127)])           # 0 .. 448, in order of their codes


def decode(codes):
    """Values of e4m3 codes (uint8)."""
    c = np.asarray(codes).astype(np.int64)
    v = np.where((c & 127) == 127, np.nan, E4M3[np.minimum(c & 127, 126)])
    return np.where(c & 128, -v, v)


def encode(x):
    """Codes of the nearest e4m3 values, ties to even codes, |x| <= 448; NaN where x is not finite."""
    x = np.asarray(x, np.float64)
    a = np.where(np.isfinite(x), np.abs(x), 0.0)
    hi = np.clip(np.searchsorted(E4M3, a), 1, 126)
    lo = hi - 1
    dl, dh = a - E4M3[lo], E4M3[hi] - a
    code = np.where(dl < dh, lo, np.where(dh < dl, hi, np.where(lo % 2 == 0, lo, hi)))
    code = code + np.where(np.signbit(x), 128, 0)
    return np.where(np.isfinite(x), code, 127).astype(np.uint8)


def least_scale(most):
    e = -120
    while e < 120 and most > 448 * 2.0 ** e:
        e += 1
    return 2.0 ** e


def store(q, scale, k, v, slots):
    """store_kv_ on numpy arrays: q [2][pages][H][P][D] uint8, scale [2][pages][H]; k, v [n][H][D]; in place."""
    _, pages, H, P, _ = q.shape
    by_page = {}
    for i, s in enumerate(slots):
        if 1 <= s <= pages * P:
            by_page.setdefault((int(s) - 1) // P, {})[(int(s) - 1) % P] = i
    for page, rows in by_page.items():
        offs, toks = list(rows), list(rows.values())
        for half, x in ((0, k), (1, v)):
            for h in range(H):
                new = x[toks, h].astype(np.float64)
                fine = np.abs(new[np.isfinite(new)])
                need = least_scale(fine.max() if fine.size else 0.0)
                old = float(scale[half, page, h])
                fresh = 0 in rows or not (0 < old < math.inf)
                now = need if fresh else max(old, need)
                if not fresh and now > old:
                    held = [o for o in range(P) if o not in rows]
                    q[half, page, h, held] = encode(decode(q[half, page, h, held]) * (old / now))
                q[half, page, h, offs] = encode(new / now)
                scale[half, page, h] = now


# ---- caches -------------------------------------------------------------------------------------

class Layer:
    """A layer's pools of a kind, garbage (NaN where the kind has it) everywhere but in the rows that are put there."""

    def __init__(self, kv, D, H, P, pages, seed=0):
        self.kv, self.D, self.H, self.P, self.pages = kv, D, H, P, pages
        self.g = np.random.Generator(np.random.PCG64(seed))
        shape = (pages, H, P, D)
        self.k, self.v = np.full(shape, np.nan), np.full(shape, np.nan)      # what the rows stand for
        if kv == "int8":
            self.q = self.g.integers(-127, 128, (2, *shape)).astype(np.int8)
            self.scale = np.full((2, pages, H, P), np.nan, np.float32)
            # powers of two: queries times them are exact
            half = 2.0 ** self.g.integers(-1, 2, D // 2)
            self.smooth = np.concatenate([half, half]).astype(np.float32)
        elif kv == "fp8":
            self.q = np.full((2, *shape), 127, np.uint8)
            self.scale = np.full((2, pages, H), np.nan, np.float32)

    def fill(self, page, off):
        """Random rows at (0-based page, offset), arrays of equal length."""
        page, off = np.asarray(page, np.int64), np.asarray(off, np.int64)
        n, H, D = len(page), self.H, self.D
        heads = np.arange(H)[None]
        at = (page[:, None], heads, off[:, None])
        for half, x in ((0, self.k), (1, self.v)):
            if self.kv == "int8":
                s = (self.g.random((n, H)) * 0.02 + 0.005).astype(np.float32)
                self.scale[(half,) + at] = s
                x[at] = self.q[(half,) + at].astype(np.float64) * s[..., None].astype(np.float64) * (self.smooth if half == 0 else 1.0)
            elif self.kv == "fp8":
                for p in np.unique(page):
                    fresh = ~np.isfinite(self.scale[half, p])
                    self.scale[half, p, fresh] = 2.0 ** self.g.integers(-8, -5, int(fresh.sum()))
                codes = encode(np.clip(self.g.standard_normal((n, H, D)) * 64, -448, 448))
                self.q[(half,) + at] = codes
                x[at] = decode(codes) * self.scale[half, page][..., None].astype(np.float64)
            else:
                r = torch.from_numpy(self.g.standard_normal((n, H, D)).astype(np.float32))
                x[at] = (r.bfloat16() if self.kv == "bf16" else r).double().numpy()

    def put(self, half, page, head, off, value):
        """One row of one head, all its elements the same (dense and fp8, which holds what is not finite as NaN)."""
        (self.k, self.v)[half][page, head, off] = np.nan if self.kv == "fp8" and not math.isfinite(value) else value
        if self.kv == "fp8":
            self.q[half, page, head, off] = encode(np.full(self.D, value) / float(self.scale[half, page, head]))

    def device(self):
        """(k_pages, v_pages) as the ops take them."""
        if self.kv == "int8":
            q, s = torch.from_numpy(self.q).cuda(), torch.from_numpy(self.scale).cuda()
            sm = torch.from_numpy(self.smooth).cuda()
            return ti.Int8Pages(q, s, sm, 0), ti.Int8Pages(q, s, torch.ones_like(sm), 1)
        if self.kv == "fp8":
            q, s = torch.from_numpy(self.q).cuda(), torch.from_numpy(self.scale).cuda()
            return ti.Fp8Pages(q, s, 0), ti.Fp8Pages(q, s, 1)
        T = torch.bfloat16 if self.kv == "bf16" else torch.float32
        return torch.from_numpy(self.k).to(T).cuda(), torch.from_numpy(self.v).to(T).cuda()


class Step:
    """A step of sequences (cached, new) over a Layer whose only rows are those that a query may see; pages that hold
    none of them have table entry 0."""

    def __init__(self, kv, lens, window=0, sinks=0, D=128, H=2, G=4, P=16, seed=0, dtype=None, spare=3):
        self.lens, self.window, self.sinks, self.H, self.G, self.D, self.P = lens, window, sinks, H, G, D, P
        rows, kept = [], []
        for c, n in lens:
            lo = max(0, c - window + 1) if window else 0
            seen = [i for i in range(c + n) if i >= lo or i < sinks] if n else []
            rows.append(seen)
            kept.append(sorted({i // P for i in seen}))
        total = sum(map(len, kept))
        self.layer = Layer(kv, D, H, P, total + spare, seed)
        g = self.layer.g
        ids = g.permutation(total + spare)[:total] + 1
        width = max([-(-(c + n) // P) for c, n in lens] + [1])
        self.tables = np.zeros((len(lens), width), np.int32)
        at = 0
        for b, k in enumerate(kept):
            self.tables[b, k] = ids[at:at + len(k)]
            at += len(k)
        self.rows = rows
        for b, seen in enumerate(rows):
            if seen:
                s = np.asarray(seen)
                self.layer.fill(self.tables[b][s // P] - 1, s % P)
        self.T = dtype or (torch.float32 if kv == "fp32" else torch.bfloat16)
        self.tokens = sum(n for _, n in lens)
        self.q = torch.from_numpy(g.standard_normal((max(self.tokens, 1), H * G, D)).astype(np.float32)).to(self.T)
        self.starts = np.concatenate([[0], np.cumsum([n for _, n in lens])]).astype(np.int32)
        self.positions = np.array([p for c, n in lens for p in range(c, c + n)] or [0], np.int32)
        self.most = max([n for _, n in lens] + [1])
        self.scale = 1 / math.sqrt(D)

    def args(self):
        return i32(self.tables), i32(self.positions), i32(self.starts)

    def want(self, causal=True):
        """(outputs, sums of weight times |value|) in 64 bits, from the rows that each query sees alone."""
        P, G = self.P, self.G
        q = self.q.double().numpy()
        out, size = np.zeros(q.shape), np.zeros(q.shape)
        at = 0
        for b, (c, n) in enumerate(self.lens):
            for t in range(n):
                p = c + t
                last = p if causal else c + n - 1
                i = np.arange(last + 1)
                if self.window:
                    i = i[(i > p - self.window) | (i < self.sinks)]
                page, off = self.tables[b][i // P].astype(np.int64) - 1, i % P
                for h in range(self.H):
                    k, v = self.layer.k[page, h, off], self.layer.v[page, h, off]
                    s = q[at, h * G:(h + 1) * G] @ k.T * self.scale
                    w = np.exp(s - s.max(1, keepdims=True))
                    w /= w.sum(1, keepdims=True)
                    out[at, h * G:(h + 1) * G] = w @ v
                    size[at, h * G:(h + 1) * G] = w @ np.abs(v)
                at += 1
        return out, size


def tolerance(T, want, size):
    """Largest error of an output. bf16: weights are rounded to bf16 (at most 2^-8 of each, so 2^-8 of the sum of
    weight times |value|), the output once more (2^-8 of it); scores, exponentials and sums in 32 bits are within
    2^-12 of the same sum. Float32: scores of 128 products of about 1 are off by at most 130 * 2^-24 of the sum of their
    magnitudes (about 8 after scaling), sums and exponentials by less: 1e-4 of the sum."""
    if T == torch.bfloat16:
        return (2.0 ** -8 + 2.0 ** -12) * size + 2.0 ** -8 * np.abs(want) + 1e-30
    return 1e-4 * size + 1e-30


def check(got, want, size, T):
    got = got.double().cpu().numpy()
    assert np.isfinite(got).all()
    over = np.abs(got - want) - tolerance(T, want, size)
    assert over.max() <= 0, f"off by {np.abs(got - want).max():.3g} at {np.unravel_index(over.argmax(), over.shape)}"
