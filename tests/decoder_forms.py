"""The decoder operators' definitions in float64 numpy, with a bound on the
kernels' error per element where results are rounded.  Rows, pages and batches
as include/ipus.h describes them; nothing here calls the library."""
from __future__ import annotations

import numpy as np

HALF_STEP = {np.float16: 2.0 ** -11, np.float32: 2.0 ** -24}
SMALLEST = {np.float16: 2.0 ** -25, np.float32: 2.0 ** -150}  # half the smallest subnormal step


def rotate(x, positions, frequencies, magnitude, rotary_width, interleaved):
    """x [rows, heads, width] turned, and the bound on the kernel's error before
    its last rounding: sin and cos within 3 * 2^-24 (the reduced angle's
    rounding, the series' last operations, the magnitude's product), each
    product and the sum rounded once in fp32, and the angle's 52 bits."""
    out, bound = x.copy(), np.zeros_like(x)
    r = rotary_width
    if r == 0:
        return out, bound
    angle = positions.astype(np.float64)[:, None] * frequencies.astype(np.float64)[None, :]
    c, s = (magnitude * f(angle)[:, None, :] for f in (np.cos, np.sin))
    i = np.arange(r // 2)
    ia, ib = (2 * i, 2 * i + 1) if interleaved else (i, i + r // 2)
    a, b = x[..., ia], x[..., ib]
    out[..., ia], out[..., ib] = a * c - b * s, b * c + a * s
    far = np.abs(angle)[:, None, :] * 2.0 ** -51
    e = (np.abs(a) + np.abs(b)) * abs(magnitude) * (5 * 2.0 ** -24 + far)
    bound[..., ia] = bound[..., ib] = e
    return out, bound


def norm(x, weight, epsilon):
    """x [rows, heads, width]; the bound: a sum of `width` squares in fp32 in
    any order (halved by the root), the root, the division and two products."""
    width = x.shape[-1]
    y = x / np.sqrt(np.mean(x * x, axis=-1, keepdims=True) + epsilon) * weight
    return y, np.abs(y) * (width / 2 + 8) * 2.0 ** -24


def norm_rotate(x, weight, epsilon, positions, frequencies, magnitude, rotary_width, interleaved):
    y, e = norm(x, weight, epsilon)
    out, bound = rotate(y, positions, frequencies, magnitude, rotary_width, interleaved)
    # The norm's error passes the rotation: both elements of a pair.
    through, _ = rotate(np.zeros_like(e), positions, frequencies, magnitude, 0, False)
    r = rotary_width
    through = e.copy()
    if r:
        i = np.arange(r // 2)
        ia, ib = (2 * i, 2 * i + 1) if interleaved else (i, i + r // 2)
        both = (e[..., ia] + e[..., ib]) * abs(magnitude)
        through[..., ia] = through[..., ib] = both
    return out, bound + through


def rounded(want, bound, dtype):
    """The bound with the result's rounding to `dtype`."""
    return bound + (np.abs(want) + bound) * HALF_STEP[dtype] + SMALLEST[dtype]


class Batch:
    """A ragged batch over a paged cache, as arrays and as plain lists."""

    def __init__(self, rng, rows, lengths, page_rows, pad_rows=0, spare_columns=1, shared=0):
        self.n, self.k, self.page_rows = list(rows), list(lengths), page_rows
        self.shared = shared
        need = [(k + page_rows - 1) // page_rows for k in self.k]
        self.columns = max(need + [0]) + spare_columns
        common = shared // page_rows
        self.pages = common + sum(max(0, x - common) for x in need) + 2
        free = list(rng.permutation(self.pages))
        prefix = [free.pop() for _ in range(common)]
        self.table = np.full((len(self.k), self.columns), -1, np.int32)
        for s, x in enumerate(need):
            mine = (prefix + [free.pop() for _ in range(max(0, x - common))])[:x]
            self.table[s, :x] = mine
        self.offsets = np.concatenate([[0], np.cumsum(self.n)]).astype(np.int32)
        self.lengths = np.array(self.k, np.int32)
        self.rows = int(self.offsets[-1]) + pad_rows

    def sequences(self):
        return len(self.n)

    def places(self, s):
        """(position, page, row in page) of every allocated key of sequence s."""
        p = np.arange(self.k[s])
        table = np.where(p < self.shared, self.table[0][np.minimum(p // self.page_rows, self.columns - 1)],
                         self.table[s][np.minimum(p // self.page_rows, self.columns - 1)])
        table = np.where(p // self.page_rows < self.columns, table, -1)
        return p, table, p % self.page_rows


def attention(batch, query, cache, key_heads, causal, scale, fp16_probabilities=True):
    """query [rows, heads, width] and cache [pages, 2, key heads, page rows, width]
    in float64.  Output, the bound before the last rounding, and which rows belong
    to a sequence."""
    rows, heads, width = query.shape
    out, bound = np.zeros_like(query), np.zeros_like(query)
    inside = np.zeros(rows, bool)
    for s in range(batch.sequences()):
        first, n = int(batch.offsets[s]), batch.n[s]
        inside[first:first + n] = True
        p, page, row = batch.places(s)
        good = (page >= 0) & (page < batch.pages)
        p, page, row = p[good], page[good], row[good]
        if n == 0 or len(p) == 0:
            continue
        for h in range(heads):
            kh = h // (heads // key_heads)
            k, v = cache[page, 0, kh, row], cache[page, 1, kh, row]
            q = query[first:first + n, h]
            x = (q @ k.T) * scale
            # fp32 sums of `width` exact products, the scale and the
            # exponential in fp32 (about 2^-22 of the exponent each)
            dx = (np.abs(q) @ np.abs(k).T) * scale * (width + 4) * 2.0 ** -24 + np.abs(x) * 2.0 ** -21
            if causal:
                position = batch.k[s] - n + np.arange(n)
                ok = p[None, :] <= position[:, None]
            else:
                ok = np.ones((n, len(p)), bool)
            x, dx = np.where(ok, x, -np.inf), np.where(ok, dx, 0.0)
            top = x.max(axis=1, keepdims=True)
            w = np.where(ok, np.exp(x - np.where(np.isfinite(top), top, 0.0)), 0.0)
            total = w.sum(axis=1, keepdims=True)
            w = np.where(total > 0, w / np.where(total > 0, total, 1.0), 0.0)
            w = np.where(np.isnan(x).any(axis=1, keepdims=True), np.nan, w)  # a NaN score that the row reads
            at = slice(first, first + n)
            if np.all(np.isfinite(v)):
                out[at, h] = w @ v
            else:  # a row's own keys alone: 0 times another's infinity is not there
                for r in range(n):
                    out[first + r, h] = w[r, ok[r]] @ v[ok[r]]
                v = np.where(np.isfinite(v), v, 0.0)
            # Probabilities rounded to fp16, and their sum of unrounded ones;
            # probabilities below fp16's normal range lose 2^-25 each against
            # a largest of 2^-8 at least; fp32 accumulation.
            step = 2 * 2.0 ** -11 if fp16_probabilities else 0.0
            tiny = 2.0 ** -17 if fp16_probabilities else 0.0
            delta = 2.0 * dx.max(axis=1, keepdims=True)
            bound[at, h] = ((step + delta + len(p) * 2.0 ** -23) * (w @ np.abs(v))
                            + tiny * (ok @ np.abs(v)) / np.maximum(total, 1.0))
    return out, bound, inside


def close_weights(rng, batch, heads, key_heads, width):
    """Query and cache whose outputs nearly cancel, fp16: keys of nearly equal weights by
    twos whose values are each other's negatives, so that the output's rounding does
    not hide what the weights lost.  Rows outside the sequences' keys are NaN."""
    q = (0.05 * rng.standard_normal((batch.rows, heads, width))).astype(np.float16)
    cache = np.full((batch.pages, 2, key_heads, batch.page_rows, width), np.nan, np.float16)
    for s in range(batch.sequences()):
        p, page, row = batch.places(s)
        cache[page, 0, :, row] = rng.standard_normal((len(p), key_heads, width)).astype(np.float16)
        v = (1 + rng.random(((len(p) + 1) // 2, key_heads, width))).astype(np.float16)
        cache[page, 1, :, row] = np.stack([v, -v], axis=1).reshape(-1, key_heads, width)[:len(p)]
    return q, cache


def weighed(batch, query, cache, key_heads, scale, weights):
    """Not causal: (output, bound before the last rounding) in float64, the weights as
    `weights` leaves the probabilities: "exact", "two halves" or "one half".

    The bound of exact and two halves: fp32 scores (`width` products, the scale, the
    exponential) as in `attention`; the sums of n products and n probabilities in
    fp32; two halves hold a probability, at most 1, within 2^-22 of itself and 2^-25
    (the second's subnormal step)."""
    rows, heads, width = query.shape
    out, bound = np.zeros(query.shape), np.zeros(query.shape)
    q64 = query.astype(np.float64)
    for s in range(batch.sequences()):
        at = slice(int(batch.offsets[s]), int(batch.offsets[s]) + batch.n[s])
        _, page, row = batch.places(s)
        for h in range(heads):
            k, v = (cache[page, i, h // (heads // key_heads), row].astype(np.float64) for i in (0, 1))
            x = (q64[at, h] @ k.T) * scale
            dx = (np.abs(q64[at, h]) @ np.abs(k).T) * scale * (width + 4) * 2.0 ** -24 + np.abs(x) * 2.0 ** -21
            p = np.exp(x - x.max(axis=1, keepdims=True))
            total = p.sum(axis=1, keepdims=True)
            if weights != "exact":
                high = p.astype(np.float16).astype(np.float64)
                low = (p - high).astype(np.float16).astype(np.float64) if weights == "two halves" else 0.0
                out[at, h] = (high + low) @ v / total
            else:
                out[at, h] = p @ v / total
            step, tiny = (2.0 ** -22, 2.0 ** -25) if weights != "exact" else (0.0, 0.0)
            size = (p @ np.abs(v)) / total
            bound[at, h] = ((step + 2.0 * dx.max(axis=1, keepdims=True) + len(page) * 2.0 ** -23) * size
                            + tiny * np.abs(v).sum(axis=0) / total)
    return out, bound
