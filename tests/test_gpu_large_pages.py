"""Pages of 65536 rows: of just below 2^32 bytes, which the tile kernels address, and of
2^32, which the general kernel does."""
from __future__ import annotations

import numpy as np
import pytest

from decoder_forms import HALF_STEP, rotate, rounded
from test_gpu_pages import halves

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [[1, 2], [3, 70]])
@pytest.mark.parametrize("heads", [63, 64])
def test_pages_of_4_gib(ipus, ctx, heads, rows):
    """The last new rows of two sequences that end with their pages, zeros before them."""
    width, page_rows, pages, sequences = 256, 65536, 3, 2
    assert (2 * heads * page_rows * width * 2 >= 1 << 32) == (heads == 64)
    cache = ctx.alloc(pages * 2 * heads * page_rows * width * 2)
    ctx.memset(cache, 0)
    total, lengths = sum(rows), [page_rows, page_rows + 40]
    table = np.array([[2, -1], [0, 1]], np.int32)
    offsets = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
    keys, values, q = (halves(ipus, (total, heads, width), t) for t in (1, 2, 3))
    f, _ = ipus.rotary_frequencies(width)
    bufs = [ctx.upload(a) for a in (keys, values, f, table, offsets, np.array(lengths, np.int32), q)]
    dk, dv, df, dt, do, dl, dq = bufs
    ctx.launch("ipu_stack_append_pages_f16", cache, [dk, dv, df, dt, do, dl],
               [sequences, total, heads, width, heads * width, heads * width, width, 0, 0, pages, page_rows, 2])
    out = ctx.alloc(q.nbytes)
    ctx.launch("ipu_stack_attention_pages_f16", out, [dq, cache, dt, do, dl],
               [sequences, total, max(rows), heads, heads, width, heads * width, pages, page_rows, 2, 1, 0])
    got = out.download(np.float16).reshape(q.shape).astype(np.float64)
    row_bytes = width * 2
    for s in range(sequences):
        for i in range(rows[s]):
            t, p = int(offsets[s]) + i, lengths[s] - rows[s] + i
            page, at = int(table[s][p // page_rows]), p % page_rows
            turned, e = rotate(keys[t].astype(np.float64)[None], np.array([p]), f, 1.0, width, False)
            e = rounded(turned, e, np.float16)
            for h in (0, 1, heads - 1):
                place = cache.ptr + ((page * 2 * heads + h) * page_rows + at) * row_bytes
                k = ipus.DeviceBuffer(ctx, place, row_bytes).download(np.float16).astype(np.float64)
                v = ipus.DeviceBuffer(ctx, place + heads * page_rows * row_bytes, row_bytes).download(np.float16)
                assert np.all(np.abs(k - turned[0, h]) <= e[0, h])
                assert np.array_equal(v, values[t, h])
    for s in range(sequences):
        at = slice(int(offsets[s]), int(offsets[s + 1]))
        position = lengths[s] - rows[s] + np.arange(rows[s])
        k64 = rotate(keys[at].astype(np.float64), position, f, 1.0, width, False)[0]
        for h in range(heads):
            k, v, x = k64[:, h], values[at, h].astype(np.float64), q[at, h].astype(np.float64)
            score = (x @ k.T) * width ** -0.5
            # fp32 scores of keys within half a step of k64
            dx = ((width + 4) * 2.0 ** -24 + 2 * HALF_STEP[np.float16]) * (np.abs(x) @ np.abs(k).T) * width ** -0.5
            dx += np.abs(score) * 2.0 ** -21
            ok = np.tril(np.ones_like(score, bool))
            top = np.maximum(np.where(ok, score, -np.inf).max(axis=1, keepdims=True), 0.0)
            w = np.where(ok, np.exp(score - top), 0.0)
            # Every other key scores 0 and its value is 0.
            total_w = w.sum(axis=1, keepdims=True) + (position[:, None] - np.arange(rows[s])[:, None]) * np.exp(-top)
            want = (w / total_w) @ v
            # Probabilities of fp16, at least 2^-17 of the largest each (tests of the many-row
            # kernel), and fp32 sums over as many keys.
            bound = ((2 * HALF_STEP[np.float16] + 2 * np.where(ok, dx, 0.0).max() + page_rows * 2.0 ** -23)
                     * ((w / total_w) @ np.abs(v)) + 2.0 ** -17 * (ok @ np.abs(v)) / total_w)
            assert np.all(np.abs(got[at, h] - want) <= rounded(want, bound, np.float16)), (s, h)
    for x in bufs + [out, cache]:
        x.free()
