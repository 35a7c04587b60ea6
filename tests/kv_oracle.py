"""A paged key-value cache in numpy, and attention over it in 64 bits, for the tests of the C ABI's.

Tolerances count roundings.  A score is a dot product of `dim` exact products (f16 times f16, or times an e4m3 code, has at most 22
bits) added in f32: dim steps of 2^-23 of the sum of their magnitudes, should the matrix unit cut off instead of rounding.  Scale and the
logarithm's base cost 2^-22 of the score more, the exponential 2^-22 of the weight.  So a weight is off by a factor of 1 + d,

    d = scale * dim * 2^-23 * max_t sum |q k_t| + 2^-22 max_t |score_t| + 2^-21,

its difference to the largest score included twice over.  The sums over n tokens, the running sum's rescalings among them, cost n + 16
steps of 2^-23.  Weights that enter the products in f16 are off by 2^-11 of themselves, or 2^-25 of the largest where they are
subnormal; as two f16 terms by 2^-21, and 2^-25.  All of it counts relative to sum p |v| / sum p; then the result is rounded to f16."""
import numpy as np

import tensorwarp_amd as T


def e4m3_table():
    t = np.zeros(256, np.float64)
    for c in range(256):
        e, m = (c >> 3) & 15, c & 7
        v = np.nan if e == 15 and m == 7 else m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10)
        t[c] = -v if c & 128 else v
    return t


E4M3 = e4m3_table()


def half_step_f16(x):
    """Half a step of f16 at x, or more where x is on a border."""
    return np.maximum(2.0 ** -11 * np.abs(x), 2.0 ** -25)


def attend(q, k, v, seen, scale, weight_step):
    """q [heads, dim], k, v [heads, tokens, dim], seen [tokens]: (result [heads, dim], how far an f16 result may be off)."""
    heads, dim = q.shape
    if not seen.any():
        return np.zeros((heads, dim)), np.zeros((heads, dim))
    k, v = k[:, seen], v[:, seen]
    with np.errstate(invalid="ignore", over="ignore"):
        products = k * q[:, None, :]
        s = products.sum(2) * scale
        top = s.max(1, keepdims=True)
        p = np.exp(s - top)
        total = p.sum(1)[:, None]
        out = (p[:, :, None] * v).sum(1) / total
        d = scale * dim * 2.0 ** -23 * np.abs(products).sum(2).max(1) + 2.0 ** -22 * np.abs(s).max(1) + 2.0 ** -21
        n = k.shape[1]
        relative = (2 * d + (n + 16) * 2.0 ** -23 + weight_step)[:, None]
        tol = (p[:, :, None] * np.abs(v)).sum(1) / total * relative + 2.0 ** -25 * np.abs(v).sum(1) / total
    return out, tol * (1 + 2.0 ** -11) + half_step_f16(out)


class Pool:
    """Pages of keys and values on the host (f16 bits or e4m3 codes) and, by upload(), on the device.  Pages that no token fills hold NaN."""

    def __init__(self, rng, pages, kv_heads, page_tokens, dim, cache="f16", scales=True):
        self.rng, self.shape, self.cache, self.page = rng, (pages, kv_heads, page_tokens, dim), cache, page_tokens
        garbage = (0x7E00, np.uint16) if cache == "f16" else (0x7F, np.uint8)
        self.bits = {name: np.full(self.shape, *garbage) for name in "kv"}
        self.scales = {name: (rng.uniform(0.01, 0.04, kv_heads).astype(np.float32) if cache == "e4m3" and scales else None) for name in "kv"}
        self.free = list(rng.permutation(pages))

    def values(self, name):
        if self.cache == "f16":
            return self.bits[name].view(np.float16).astype(np.float64)
        v = E4M3[self.bits[name]]
        return v if self.scales[name] is None else v * self.scales[name].astype(np.float64)[None, :, None, None]

    def fill(self, lengths, width=None, spread=1.0):
        """Sequences of these lengths in random pages: their table."""
        width = max([1] + [-(-n // self.page) for n in lengths]) if width is None else width
        table = np.full((len(lengths), width), -1, np.int32)
        for s, n in enumerate(lengths):
            for i in range(-(-n // self.page)):
                table[s, i] = self.free.pop()
                here = min(self.page, n - i * self.page)
                for name in "kv":
                    x = spread * self.rng.standard_normal((self.shape[1], here, self.shape[3]))
                    if self.cache == "f16":
                        self.bits[name][table[s, i], :, :here] = x.astype(np.float16).view(np.uint16)
                    else:
                        codes = self.rng.integers(0, 127, x.shape).astype(np.uint8)
                        codes = np.where(codes > 0x70, codes - 0x40, codes) | (x > 0).astype(np.uint8) << 7   # (few of the largest)
                        self.bits[name][table[s, i], :, :here] = codes
        return table

    def tokens(self, name, row, count):
        """[kv_heads, count, dim] of a table's row; absent pages are NaN."""
        out = np.full((self.shape[1], count, self.shape[3]), np.nan)
        at = np.flatnonzero(self.present(row, count))
        places = np.asarray(row)[at // self.page], slice(None), at % self.page
        bits = self.bits[name][places]
        values = bits.view(np.float16).astype(np.float64) if self.cache == "f16" else E4M3[bits]
        if self.scales[name] is not None:
            values = values * self.scales[name].astype(np.float64)[:, None]
        out[:, at] = values.transpose(1, 0, 2)
        return out

    def present(self, row, count):
        at = np.arange(count) // self.page
        pages = np.concatenate([np.asarray(row, np.int64), [-1]])[np.minimum(at, len(row))]
        return (pages >= 0) & (pages < self.shape[0])

    def upload(self, dev):
        self.dev = {name: T.GpuTensor.from_host(dev, self.bits[name], "f16" if self.cache == "f16" else "u8") for name in "kv"}
        of = {name: None if self.scales[name] is None else T.GpuTensor.from_host(dev, self.scales[name]) for name in "kv"}
        return T.KvCache(self.dev["k"], self.dev["v"], self.page, self.shape[1], self.shape[3], k_scales=of["k"], v_scales=of["v"])

    def download(self):
        for name in "kv":
            self.bits[name] = self.dev[name].to_host().reshape(self.shape)


def attend_rows(pool, table, lengths, new, q, scale, window, weight_step):
    """q [rows, q_heads, dim]: (results, tolerances, which rows belong to a sequence) of packed rows, new[s] of sequence s in turn."""
    rows, heads, dim = q.shape
    group = heads // pool.shape[1]
    out, tol = np.zeros(q.shape), np.zeros(q.shape)
    row = 0
    for s, (n, length) in enumerate(zip(new, lengths)):
        length = max(length, 0)
        k, v = (np.repeat(pool.tokens(name, table[s], length), group, axis=0) for name in "kv")
        there, at = pool.present(table[s], length), np.arange(length)
        for i in range(n):
            position = length - n + i
            seen = there & (at <= position) & ((at > position - window) if window else True)
            out[row], tol[row] = attend(q[row].astype(np.float64), k, v, seen, scale, weight_step)
            row += 1
    return out, tol, row


DECODE_STEP, PROMPT_STEP = 2.0 ** -21, 2.0 ** -11


def check(got, want, tol):
    got = got.astype(np.float64)
    assert np.array_equal(np.isnan(got), np.isnan(want)), (np.isnan(got).sum(), np.isnan(want).sum())
    there = np.isfinite(want)
    assert np.array_equal(got[~there & ~np.isnan(want)], want[~there & ~np.isnan(want)])
    off = np.abs(got - want)[there] / np.maximum(tol[there], 1e-300)
    bad = np.where(np.abs(got - want)[there] == 0, 0.0, off)
    assert bad.size == 0 or bad.max() <= 1.0, (bad.max(), (bad > 1).sum(), bad.size)
