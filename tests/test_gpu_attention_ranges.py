"""Paged attention at the ends of fp16's range: scores that fp32 holds in steps of
more than one, and values whose mean must not pass the largest."""
from __future__ import annotations

import math
import struct

import numpy as np
import pytest

from decoder_forms import Batch
from test_gpu_pages import attention_symbol, upload_batch

pytestmark = pytest.mark.gpu


def bits(x):
    return struct.unpack("<I", struct.pack("<f", x))[0]


# rows, lengths, query heads, key heads, width, page_rows, table columns to spare, shared
KERNELS = {
    "one tile": ([1] * 3, [300, 64, 5], 8, 2, 128, 16, 1, 0),
    "one tile in parts": ([1], [2100], 8, 1, 64, 16, 1, 0),
    "two tiles": ([3, 1, 2], [300, 64, 500], 16, 2, 128, 16, 400, 0),
    "two tiles, 64 columns": ([2], [450], 12, 1, 64, 64, 400, 0),
    "blocks": ([100, 40], [300, 60], 8, 2, 128, 64, 1, 0),
    "split blocks": ([40], [2000], 4, 1, 64, 16, 200, 0),
    "blocks, 256 columns": ([70], [400], 4, 2, 256, 16, 1, 0),
    "shared": ([1] * 300, [1030] * 300, 16, 4, 64, 16, 1, 1000),
    "general": ([2, 1], [300, 31], 2, 1, 65, 16, 1, 0),
}


def run(ipus, ctx, b, q, cache, heads, key_heads, width, causal, scale):
    bufs = [ctx.upload(q), ctx.upload(cache)] + upload_batch(ctx, b)
    out = ctx.alloc(q.nbytes)
    ctx.launch(attention_symbol(b), out, bufs,
               [b.sequences(), b.rows, max(b.n), heads, key_heads, width, heads * width, b.pages, b.page_rows,
                b.columns, int(causal), bits(scale)] + ([b.shared] if b.shared else []))
    got = out.download(np.float16).reshape(q.shape).astype(np.float64)
    for x in bufs + [out]:
        x.free()
    return got


@pytest.mark.parametrize("kernel", sorted(KERNELS))
@pytest.mark.parametrize("size", [5000.0, 20000.0, -60000.0])
def test_scores_past_fp32s_whole_steps(ipus, ctx, kernel, size):
    """Every second key scores the same, up to 2^36 in log2 units, the others far less:
    a row's output is the mean of the former's values."""
    rows, lengths, heads, key_heads, width, page_rows, spare, shared = KERNELS[kernel]
    b = Batch(np.random.default_rng(51), rows, lengths, page_rows, 0, spare, shared)
    q = np.full((b.rows, heads, width), size, np.float16)
    cache = np.full((b.pages, 2, key_heads, page_rows, width), np.nan, np.float16)
    values = ipus.synth_f16(max(lengths) * width, 94, 1, ipus.NORMAL, 1.0).view(np.float16).reshape(-1, width)
    low, high = (abs(size) * x for x in ((0.5, 1.0) if size > 0 else (1.0, 0.5)))
    for s in range(b.sequences()):
        p, page, row = b.places(s)
        for h in range(key_heads):
            cache[page, 0, h, row] = np.where(p % 2 == 0, high, low)[:, None]
            cache[page, 1, h, row] = values[p]
    got = run(ipus, ctx, b, q, cache, heads, key_heads, width, True, width ** -0.5)
    sums = np.cumsum(values.astype(np.float64)[::2], axis=0)
    sizes = np.cumsum(np.abs(values.astype(np.float64))[::2], axis=0)
    for s in range(b.sequences()):
        for i in range(b.n[s]):
            n = (b.k[s] - b.n[s] + i) // 2 + 1  # even keys up to the row's position
            want, weight = sums[n - 1] / n, sizes[n - 1] / n
            # Equal weights: the sums over n keys in fp32, the division, the output's rounding.
            bound = weight * (2 * n + 8) * 2.0 ** -24
            bound += (np.abs(want) + bound) * 2.0 ** -11 + 2.0 ** -25
            at = int(b.offsets[s]) + i
            assert np.all(np.abs(got[at] - want) <= bound), (s, i)


@pytest.mark.parametrize("kernel", sorted(KERNELS))
def test_equal_values_come_out_as_they_are(ipus, ctx, kernel):
    """Every 32nd key of weight 1, the others of a weight just past the middle of two fp16
    values: where the sum of the weights is not the one that the values meet, the largest fp16
    value becomes infinity."""
    rows, lengths, heads, key_heads, width, page_rows, spare, shared = KERNELS[kernel]
    b = Batch(np.random.default_rng(52), rows, lengths, page_rows, 0, spare, shared)
    q = np.zeros((b.rows, heads, width), np.float16)
    q[..., 0], q[..., 1] = 1.0, 2.0 ** -10
    score = math.log(0.5 + 1.05 * 2.0 ** -12)  # its weight rounds up by nearly 2^-11
    coarse = float(np.float16(score))
    cache = np.full((b.pages, 2, key_heads, page_rows, width), np.nan, np.float16)
    for s in range(b.sequences()):
        p, page, row = b.places(s)
        for h in range(key_heads):
            cache[page, :, h, row] = 0.0
            cache[page, 0, h, row, 0] = np.where(p % 32 == 0, 0.0, coarse)
            cache[page, 0, h, row, 1] = np.where(p % 32 == 0, 0.0, (score - coarse) * 2.0 ** 10)
            cache[page, 1, h, row] = 65504.0
    got = run(ipus, ctx, b, q, cache, heads, key_heads, width, False, 1.0)
    # Up to 2100 keys, summed by lanes and waves: within 2^-13, a quarter of a step.
    assert np.all(got == 65504.0)
