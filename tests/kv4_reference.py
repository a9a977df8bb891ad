"""The paged 4-bit K/V cache in NumPy: quantiser (the f32 operations one by one, so that codes and
parameters are the kernels' bit for bit), page bytes, and attention in 64 bits."""
from dataclasses import dataclass

import numpy as np

LIMIT = np.float32(32640.0)


def half_towards(values, up):
    """The fp16 neighbour of f32 values on their upper / lower side (themselves where exact)."""
    h = values.astype(np.float16)
    wrong = h.astype(np.float32) < values if up else h.astype(np.float32) > values
    return np.where(wrong, np.nextafter(h, np.float16(np.inf if up else -np.inf)), h)


def quantised(x, group):
    """f32 rows [..., D] -> codes [..., D] uint8, steps and minima [..., D/g] fp16."""
    x = np.asarray(x, dtype=np.float32).reshape(*x.shape[:-1], -1, group)
    with np.errstate(invalid="ignore"):
        bad = ~(np.abs(x).max(-1) <= LIMIT)
    x = np.where(bad[..., None], np.float32(0), x)
    low, high = x.min(-1), x.max(-1)
    minimum = half_towards(low, False) + np.float16(0)   # a zero is held as +0
    base = minimum.astype(np.float32)
    step = half_towards((high - base) / np.float32(15), True)
    wide = np.where(step == 0, np.float32(1), step.astype(np.float32))
    codes = np.clip(np.rint((x - base[..., None]) / wide[..., None]), 0, 15).astype(np.uint8)
    step = np.where(bad, np.float16(np.nan), step)
    minimum = np.where(bad, np.float16(0), minimum)
    return codes.reshape(*codes.shape[:-2], -1), step, minimum


def turned(x, cos, sin, rotary, layout):
    """f32 rows [rows, heads, D], angles [rows, >= rotary/2]: products rounded, then joined."""
    x = np.array(x, dtype=np.float32)
    j = np.arange(rotary // 2)
    first, second = (j, j + rotary // 2) if layout == 0 else (2 * j, 2 * j + 1)
    c, s = (t[:, None, :rotary // 2].astype(np.float32) for t in (cos, sin))
    a, b = x[..., first], x[..., second]
    with np.errstate(invalid="ignore"):
        x[..., first], x[..., second] = a * c - b * s, b * c + a * s
    return x


@dataclass
class Layout:
    kv_heads: int
    depth: int
    group: int
    page_rows: int

    def __post_init__(self):
        p, d, g = self.page_rows, self.depth, self.depth // self.group
        self.key = np.dtype([("codes", "u1", (p, 4, d // 32, 4)), ("params", "<f2", (p, g, 2)),
                             ("vcodes", "u1", (p // 4, d // 8, 4, 4)),
                             ("vparams", "<f2", (p // 4, g, 2, 4))])
        self.page_bytes = self.key.itemsize * self.kv_heads

    def pages(self, raw):
        """[pages, page_bytes] bytes as records [pages, kv_heads] (a view)."""
        return raw.reshape(-1, self.page_bytes).view(self.key).reshape(-1, self.kv_heads)

    def write(self, raw, page, row, head, k, v):
        """One row: (codes, steps, minima) of a head's key and value."""
        block = self.pages(raw)[page:page + 1, head]
        codes, step, minimum = k
        for word in range(self.depth // 8):
            e = codes[8 * word:8 * word + 8].astype(np.uint32)
            value = sum(int(e[2 * i]) << (4 * i) | int(e[2 * i + 1]) << (16 + 4 * i) for i in range(4))
            block["codes"][0, row, word % 4, word // 4] = list(value.to_bytes(4, "little"))
        block["params"][0, row, :, 0], block["params"][0, row, :, 1] = step, minimum
        codes, step, minimum = v
        for word in range(self.depth // 8):
            e = codes[8 * word:8 * word + 8]
            block["vcodes"][0, row // 4, word, row % 4] = e[0::2] | e[1::2] << 4
        block["vparams"][0, row // 4, :, 0, row % 4] = step
        block["vparams"][0, row // 4, :, 1, row % 4] = minimum

    def values(self, raw, page_ids):
        """f64 keys and values [kv_heads, pages * P, D] of the pages in order."""
        with np.errstate(invalid="ignore"):
            return self._values(raw, page_ids)

    def _values(self, raw, page_ids):
        b = self.pages(raw)[np.asarray(page_ids, dtype=np.int64)]
        n, h = b.shape
        nib = np.stack([b["codes"] & 15, b["codes"] >> 4], -1).reshape(n, h, self.page_rows, 4, -1, 8)
        order = np.array([(e % 2) * 4 + e // 2 for e in range(8)])
        k = nib[..., order].swapaxes(3, 4).reshape(n, h, self.page_rows, self.depth).astype(np.float64)
        par = np.repeat(b["params"].astype(np.float64), self.group, axis=3)
        k = k * par[..., 0] + par[..., 1]
        nib = np.stack([b["vcodes"] & 15, b["vcodes"] >> 4], -1).reshape(n, h, self.page_rows // 4, -1, 4, 8)
        v = nib.swapaxes(3, 4).reshape(n, h, self.page_rows, self.depth).astype(np.float64)
        par = b["vparams"].astype(np.float64).transpose(0, 1, 2, 5, 3, 4).reshape(n, h, self.page_rows, -1, 2)
        par = np.repeat(par, self.group, axis=3)
        v = v * par[..., 0] + par[..., 1]
        return (x.transpose(1, 0, 2, 3).reshape(h, n * self.page_rows, self.depth) for x in (k, v))


@dataclass
class Step:
    """A step's rows over a cache: rows and columns of each sequence, and their pages."""
    layout: Layout
    rows: list
    lens: list
    pages: int
    table: np.ndarray

    @classmethod
    def make(cls, layout, rows, lens, rng, spare=2, extra=1):
        """Pages dealt in random order; table entries past a sequence are no pages at all."""
        need = [-(-n // layout.page_rows) for n in lens]
        pages = sum(need) + spare
        order, at = rng.permutation(pages), 0
        table = np.full((len(lens), max(need + [0]) + extra), 0x7fffffff, dtype=np.int32)
        for i, n in enumerate(need):
            table[i, :n] = order[at:at + n]
            at += n
        return cls(layout, list(rows), list(lens), pages, table)

    @property
    def cu(self):
        return np.concatenate([[0], np.cumsum(self.rows)]).astype(np.int32)

    @property
    def total(self):
        return int(sum(self.rows))

    def shape(self):
        lay = self.layout
        return dict(nseq=len(self.rows), max_query=max(self.rows + [0]), total_rows=self.total,
                    kv_heads=lay.kv_heads, depth=lay.depth, group=lay.group,
                    page_rows=lay.page_rows, pages=self.pages, table_stride=self.table.shape[1])

    def columns_of(self, i):
        """(page, row in it) of each column of sequence i."""
        c = np.arange(self.lens[i])
        return self.table[i, c // self.layout.page_rows], c % self.layout.page_rows

    def random_cache(self, rng, spread=1.0, poison=True):
        """Quantised normal rows in every column; NaN parameters and full codes everywhere else."""
        lay = self.layout
        raw = np.full((self.pages, lay.page_bytes), 0xff if poison else 0, dtype=np.uint8)
        records = lay.pages(raw)
        shape = (self.pages, lay.kv_heads, lay.page_rows, lay.depth)
        channel = np.exp(0.5 * rng.normal(size=(lay.kv_heads, 1, lay.depth)))
        full = raw.copy()
        target = lay.pages(full)
        k = quantised((rng.normal(size=shape) * channel * spread).astype(np.float32), lay.group)
        v = quantised((rng.normal(size=shape) * spread).astype(np.float32), lay.group)
        pack_all(lay, target, k, v)
        used = np.zeros((self.pages, lay.page_rows), dtype=bool)
        for i in range(len(self.lens)):
            page, row = self.columns_of(i)
            used[page, row] = True
        p, r = np.nonzero(used)
        for name in ("codes", "params"):
            records[name][p, :, r] = target[name][p, :, r]
        records["vcodes"][p, :, r // 4, :, r % 4] = target["vcodes"][p, :, r // 4, :, r % 4]
        records["vparams"][p, :, r // 4, :, :, r % 4] = target["vparams"][p, :, r // 4, :, :, r % 4]
        return raw

    def attention(self, raw, q, half_scale, window=0):
        """(out f64 [total, H, D], the largest sum_d |q k| scale^2 of a row and column, max |v|)."""
        out = np.zeros(q.shape, dtype=np.float64)
        share = q.shape[1] // self.layout.kv_heads
        reach, top, cu = 0.0, 0.0, self.cu
        for i, n in enumerate(self.rows):
            if not n:
                continue
            c = self.lens[i]
            need = -(-c // self.layout.page_rows)
            k, v = (x[:, :c] for x in self.layout.values(raw, self.table[i, :need]))
            x = q[cu[i]:cu[i + 1]].astype(np.float64).transpose(1, 0, 2)   # [H, n, D]
            kk, vv = np.repeat(k, share, axis=0), np.repeat(v, share, axis=0)
            s = np.matmul(x, kk.swapaxes(1, 2)) * half_scale ** 2
            reach = max(reach, (np.matmul(np.abs(x), np.abs(kk).swapaxes(1, 2)).max()) * half_scale ** 2)
            top = max(top, np.abs(v).max())
            far = np.arange(c - n, c)[:, None] - np.arange(c)
            s = np.where((far >= 0) & (far < (window or c + 1)), s, -np.inf)
            p = np.exp(s - s.max(-1, keepdims=True))
            o = np.matmul(p / p.sum(-1, keepdims=True), vv)
            out[cu[i]:cu[i + 1]] = o.transpose(1, 0, 2)
        return out, reach, top


def attention_by_row(step, raw, q, half_scale, window=0, values=np.float64):
    """(out f64 [total, H, D] of values rounded to the given type; by how much, at most, it may be moved by the errors of
    f32 scores [total, H, 1]; their size [total, H]; max |v|).

    A score is sum q (step * code + minimum) half_scale^2 from products that are exact or known to 2^-22, so its error is
    counted against m = sum |q| (step * code + |minimum|) half_scale^2: at most 3 D/16 matrix products and 16 other
    operations come in a row, each rounds by 2^-23 of what it holds at most: e = (3 D/16 + 16) 2^-23 m, m the row's
    largest.  Every weight is then off by a factor within exp(+-2 e), and all of them together, normalised, move by
    exp(2 e) - 1; where one column holds nearly all the weight, by twice what the others can have with their scores 2 e
    nearer.  An output moves by that times the largest value."""
    lay, out = step.layout, np.zeros(q.shape, dtype=np.float64)
    moved, size, top, cu = np.zeros((*q.shape[:2], 1)), np.zeros(q.shape[:2]), 0.0, step.cu
    share, spans = q.shape[1] // lay.kv_heads, raw.copy()
    minima = lay.pages(spans)["params"][..., 1]
    minima[...] = np.abs(minima)
    for i, n in enumerate(step.rows):
        if not n:
            continue
        c = step.lens[i]
        ids = step.table[i, :-(-c // lay.page_rows)]
        k, v = (np.repeat(x[:, :c], share, axis=0) for x in lay.values(raw, ids))
        span, _ = (np.repeat(x[:, :c], share, axis=0) for x in lay.values(spans, ids))
        v = v.astype(values).astype(np.float64)
        x = q[cu[i]:cu[i + 1]].astype(np.float64).transpose(1, 0, 2)
        far = np.arange(c - n, c)[:, None] - np.arange(c)
        seen = (far >= 0) & (far < (window or c + 1))
        s = np.where(seen, np.matmul(x, k.swapaxes(1, 2)) * half_scale ** 2, -np.inf)
        m = np.where(seen, np.matmul(np.abs(x), span.swapaxes(1, 2)) * half_scale ** 2, 0.0).max(-1, keepdims=True)
        e, most = (3 * lay.depth / 16 + 16) * 2.0**-23 * m, s.max(-1, keepdims=True)
        with np.errstate(over="ignore"):
            p = np.exp(s - most)
            others = np.exp(np.minimum(0.0, s - most + 2 * e)).sum(-1, keepdims=True) - 1.0
            moves = np.minimum(np.expm1(2 * e), 2 * others) * np.abs(v).max((1, 2), keepdims=True)
        rows, top = slice(cu[i], cu[i + 1]), max(top, np.abs(v).max())
        out[rows] = np.matmul(p / p.sum(-1, keepdims=True), v).transpose(1, 0, 2)
        moved[rows], size[rows] = moves.transpose(1, 0, 2), m[..., 0].T
    return out, moved, size, top


def pack_all(lay, records, k, v):
    """Codes and parameters of [pages, Hkv, P, D] keys and values into page records."""
    codes, step, minimum = k
    c = codes.reshape(*codes.shape[:-1], -1, 4, 4, 2)            # step, column, i, parity
    c = c.transpose(0, 1, 2, 4, 3, 6, 5).reshape(*codes.shape[:-1], 4, -1, 8)
    records["codes"] = c[..., 0::2] | c[..., 1::2] << 4
    records["params"] = np.stack([step, minimum], -1)
    codes, step, minimum = v
    c = codes.reshape(*codes.shape[:2], lay.page_rows // 4, 4, lay.depth // 8, 8).swapaxes(3, 4)
    records["vcodes"] = c[..., 0::2] | c[..., 1::2] << 4
    p = np.stack([step, minimum], -1)                            # pages, Hkv, P, g, 2
    p = p.reshape(*p.shape[:2], lay.page_rows // 4, 4, -1, 2)
    records["vparams"] = p.transpose(0, 1, 2, 4, 5, 3)
