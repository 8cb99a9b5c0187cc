"""A paged cache with its sequences on the host, for the tests of the paged
entry points: rows in the pools' own types, what they stand for in float64,
and the definitions of append, read and attention over them."""
import numpy as np

F32, BF16, I8 = 0, 0x200, 0x201
NAMES = {F32: "f32", BF16: "bf16", I8: "i8"}


def to_bf16(x):
    """float32 -> bf16 bit patterns, nearest even (NaN stays NaN)"""
    u = np.ascontiguousarray(x, np.float32).view(np.uint32)
    r = ((u + np.uint32(0x7FFF) + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), r)


def from_bf16(u):
    return (np.asarray(u, np.uint16).astype(np.uint32) << 16).view(np.float32)


def enc(x, t):
    return np.ascontiguousarray(x, np.float32) if t == F32 else to_bf16(x)


def dec(a, t):
    return np.asarray(a, np.float32) if t == F32 else from_bf16(a)


def itemsize(t):
    return {F32: 4, BF16: 2, I8: 1}[t]


def np_type(t):
    return {F32: np.float32, BF16: np.uint16, I8: np.int8}[t]


def quantise(y):
    """(codes, scales) of float32 rows by the definition, in float64"""
    y = np.asarray(y, np.float32)
    bad = ~np.isfinite(y).all(-1)
    with np.errstate(all="ignore"):
        d = (np.abs(y).max(-1).astype(np.float64) / 127).astype(np.float32)
        d = np.where(bad, np.float32(np.nan), d)
        c = np.rint(y.astype(np.float64) / d.astype(np.float64)[..., None])
        c = np.where((d > 0)[..., None], np.clip(c, -127, 127), 0)
    return c.astype(np.int8), d


def rotate(x, cs):
    """x [..., hd] float32 by cs [..., hd / 2, 2]: every product and sum rounded"""
    e, o, c, s = x[..., 0::2], x[..., 1::2], cs[..., 0], cs[..., 1]
    y = np.empty_like(x)
    y[..., 0::2], y[..., 1::2] = e * c - o * s, e * s + o * c
    return y


def rope_table(n, hd, theta=500000.0):
    f = (1.0 / theta ** (np.arange(0, hd, 2) / hd)).astype(np.float32)
    a = (np.arange(n, dtype=np.float32)[:, None] * f).astype(np.float64)
    return np.ascontiguousarray(np.stack([np.cos(a), np.sin(a)], -1), np.float32)


class World:
    """Pools, page table and lengths.  hist: positions before the new tokens
    (-1: idle slot), new: tokens of the call.  Rows of no position hold NaN (the
    scale, for int8), pages lie anywhere, unused table entries are bad numbers.
    holes: (sequence, page index) whose table entry is a bad number too."""

    def __init__(self, seed, hist, new, nkv, hd, cache, page, holes=(), pad=0, scale=1.0):
        r = self.r = np.random.default_rng(seed)
        self.hist, self.new, self.nkv, self.hd, self.cache, self.page = list(hist), list(new), nkv, hd, cache, page
        self.lens = [h + n if h >= 0 else 0 for h, n in zip(hist, new)]
        need = [-(-n // page) for n in self.lens]
        self.n_pages, self.stride = sum(need) + 2, max(need + [1]) + 1
        self.max_len = max(self.lens + [1])
        free = list(r.permutation(self.n_pages))
        bad = [-1, self.n_pages, 2 ** 31 - 1, -2 ** 31]
        self.table = r.choice(bad, (len(hist), self.stride)).astype(np.int64)
        for s, n in enumerate(need):
            for i in range(n):
                p = free.pop()
                if (s, i) not in holes:
                    self.table[s, i] = p
        shape = (self.n_pages, nkv, page, hd)
        self.pools = []
        for _ in range(2):
            x = r.standard_normal(shape).astype(np.float32) * np.float32(scale)
            live = np.zeros((self.n_pages, page), bool)
            for s, n in enumerate(self.lens):
                for i in range(need[s]):
                    if self.table[s, i] in range(self.n_pages):
                        live[self.table[s, i], :max(0, min(page, n - i * page))] = True
            x[~np.broadcast_to(live[:, None], shape[:3])] = np.nan
            self.pools.append((*quantise(x),) if cache == I8 else (enc(x, cache), None))
        self.first = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        self.rows = int(self.first[-1]) + pad
        # (sequence, position) of every packed row; position -1: idle
        self.at = [(s, h + i if h >= 0 else -1) for s, (h, n) in enumerate(zip(hist, new)) for i in range(n)]

    def slot(self, s, p):
        """(page, slot) of a position, or None"""
        if p < 0 or p >= self.max_len or p // self.page >= self.stride:
            return None
        g = int(self.table[s, p // self.page])
        return (g, p % self.page) if 0 <= g < self.n_pages else None

    def values(self, which, page, slot):
        codes, d = self.pools[which]
        v = codes[page, :, slot]
        return v.astype(np.float32) * d[page, :, slot, None] if self.cache == I8 else dec(v, self.cache)

    def upload(self, ctx, H, with_first=True):
        b = self.buf = {}
        for n, (codes, d) in zip("kv", self.pools):
            b[n] = ctx.upload(codes)
            b[n + "s"] = ctx.upload(d) if d is not None else None
        b["table"], b["pos"] = ctx.upload(self.table.astype(np.int32)), ctx.upload(np.array(self.hist, np.int32))
        b["first"] = ctx.upload(self.first) if with_first else None
        p = lambda k: b[k].ptr if b[k] is not None else None  # noqa: E731
        self.pages = H.GqPages(p("k"), p("v"), p("ks"), p("vs"), self.cache, self.n_pages, self.page, self.nkv, self.hd)
        self.batch = H.GqBatch(p("table"), p("pos"), p("first"), len(self.hist), self.stride, self.rows, self.max_len)
        return self

    def free(self):
        for b in self.buf.values():
            if b is not None:
                b.free()

    def download(self, which):
        n = "kv"[which]
        codes = self.buf[n].download(np_type(self.cache)).reshape(self.pools[which][0].shape)
        d = self.buf[n + "s"]
        return codes, None if d is None else d.download(np.float32).reshape(self.pools[which][1].shape)

    # ---- definitions, in float64 ----
    def attention(self, q, row):
        """(out, sum p |v| / sum p, largest sum |q k| / sqrt(hd)) of packed row
        `row`, q [heads, hd]"""
        s, p = self.at[row]
        G, hd = q.shape[0] // self.nkv, self.hd
        seen = [x for x in (self.slot(s, i) for i in range(p + 1)) if x is not None]
        out, mag = np.zeros(q.shape), np.zeros(q.shape)
        if not seen:
            return out, mag, 0.0
        pg, sl = np.array(seen).T
        k, v = ((c[pg, :, sl].astype(np.float32) * d[pg, :, sl, None] if self.cache == I8 else dec(c[pg, :, sl], self.cache)).astype(np.float64)
                for c, d in self.pools)
        if self.cache == I8:  # the values are code * scale, not its rounding
            k, v = (c[pg, :, sl].astype(np.float64) * d[pg, :, sl, None].astype(np.float64) for c, d in self.pools)
        top = 0.0
        for h in range(q.shape[0]):
            z = k[:, h // G] @ q[h] / np.sqrt(hd)
            top = max(top, float((np.abs(k[:, h // G]) @ np.abs(q[h])).max() / np.sqrt(hd)))
            w = np.exp(z - z.max())
            out[h], mag[h] = w @ v[:, h // G] / w.sum(), w @ np.abs(v[:, h // G]) / w.sum()
        return out, mag, top
