"""How many bits of the probabilities reach the output of paged attention: two fp16 values
(22 bits) with up to 16 queries of a key head on the matrix units, and up to 32 at 97 to 128
columns; fp32 in the general kernel."""
from __future__ import annotations

import struct

import numpy as np
import pytest

from decoder_forms import Batch, close_weights, rounded, weighed


def bits(x):
    return struct.unpack("<I", struct.pack("<f", x))[0]


CASES = [
    # sequences' rows, keys, query heads, key heads, width, page_rows, weights
    ([1] * 5, [8, 2, 16, 30, 12], 16, 4, 128, 16, "two halves"),
    ([2, 1, 4], [10, 24, 6], 4, 1, 64, 8, "two halves"),
    ([1] * 3, [8, 14, 20], 4, 4, 32, 4, "two halves"),
    ([3, 1], [12, 26], 10, 2, 72, 16, "two halves"),
    ([1, 2], [8, 18], 8, 2, 96, 16, "two halves"),
    ([1] * 4, [8, 6, 22, 4], 5, 1, 192, 32, "two halves"),
    ([1] * 4, [10, 4, 12, 28], 16, 2, 256, 16, "two halves"),
    ([1] * 320, [6, 8, 10, 12] * 80, 8, 4, 64, 8, "two halves"),  # a wave for each
    # 17 to 32 queries, in pages of which few make a long table.
    ([3, 1, 2], [14, 6, 30], 16, 2, 128, 4096, "two halves"),
    ([2], [24], 28, 2, 104, 8192, "two halves"),
    ([1] * 5, [8, 2, 16, 30, 12], 4, 2, 65, 16, "exact"),
    ([2, 1], [10, 24], 4, 1, 500, 8, "exact"),
]


def make(rows, keys, heads, key_heads, width, page_rows):
    rng = np.random.default_rng(width + heads)
    b = Batch(rng, rows, keys, page_rows)
    return b, *close_weights(rng, b, heads, key_heads, width)


@pytest.mark.parametrize("rows,keys,heads,key_heads,width,page_rows,weights", CASES)
def test_the_bound_holds_for_two_halves_and_not_for_one(rows, keys, heads, key_heads, width, page_rows, weights):
    """The oracle with its probabilities rounded stands outside of the bound."""
    b, q, cache = make(rows, keys, heads, key_heads, width, page_rows)
    want, bound = weighed(b, q, cache, key_heads, width ** -0.5, "exact")
    halves, wide = weighed(b, q, cache, key_heads, width ** -0.5, "two halves")
    assert np.all(np.abs(halves - want) <= wide)
    lost, _ = weighed(b, q, cache, key_heads, width ** -0.5, "one half")
    bound = rounded(want, wide if weights == "two halves" else bound, np.float16)
    assert np.mean(np.abs(lost.astype(np.float16).astype(np.float64) - want) > bound) > 0.2


@pytest.mark.gpu
@pytest.mark.parametrize("rows,keys,heads,key_heads,width,page_rows,weights", CASES)
def test_probabilities(ipus, ctx, rows, keys, heads, key_heads, width, page_rows, weights):
    b, q, cache = make(rows, keys, heads, key_heads, width, page_rows)
    bufs = [ctx.upload(a) for a in (q, cache, b.table, b.offsets, b.lengths)]
    out = ctx.alloc(q.nbytes)
    ctx.launch("ipu_stack_attention_pages_f16", out, bufs,
               [b.sequences(), b.rows, max(b.n), heads, key_heads, width, heads * width, b.pages, b.page_rows,
                b.columns, 0, 0])
    got = out.download(np.float16).reshape(q.shape).astype(np.float64)
    want, bound = weighed(b, q, cache, key_heads, width ** -0.5, "exact")
    if weights == "two halves":
        _, bound = weighed(b, q, cache, key_heads, width ** -0.5, weights)
    assert np.all(np.abs(got - want) <= rounded(want, bound, np.float16))
    for x in bufs + [out]:
        x.free()
