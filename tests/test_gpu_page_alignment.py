"""Paged operators at addresses and strides of no alignment but the elements', and at
those that just allow the widest accesses."""
from __future__ import annotations

import numpy as np
import pytest

from decoder_forms import Batch, attention, rounded
from test_gpu_pages import append64, append_scalars, attention_scalars, halves, upload_batch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [[1, 2, 1], [60, 1, 9]])
@pytest.mark.parametrize("width", [128, 72])
@pytest.mark.parametrize("shift,stride", [((8, 0, 0), 8), ((1, 0, 0), 0), ((0, 1, 0), 0), ((0, 0, 1), 0),
                                          ((0, 0, 0), 4), ((4, 4, 4), 1), ((0, 0, 4), 0)])
def test_attention_alignment(ipus, ctx, rows, width, shift, stride):
    """Query, cache and output `shift` elements into their buffers, query rows `stride`
    elements further apart than their heads fill."""
    heads, key_heads = 4, 2
    b = Batch(np.random.default_rng(71), rows, [k + 40 for k in rows], 16, 1)
    pitch = heads * width + stride
    cache = halves(ipus, (b.pages, 2, key_heads, 16, width), 1)
    flat = halves(ipus, (b.rows * pitch + 8,), 2)
    q = flat[:b.rows * pitch].reshape(b.rows, pitch)[:, :heads * width].reshape(b.rows, heads, width)
    at = [ctx.upload(np.concatenate([np.zeros(n, np.float16), x.ravel()])) for n, x in zip(shift, (flat, cache))]
    out = ctx.upload(np.full(q.size + 16, 7.0, np.float16))
    batch = upload_batch(ctx, b)
    ctx.launch("ipu_stack_attention_pages_f16", out.ptr + 2 * shift[2],
               [at[0].ptr + 2 * shift[0], at[1].ptr + 2 * shift[1]] + batch,
               attention_scalars(b, heads, key_heads, width, 1, pitch=pitch))
    raw = out.download(np.float16)
    got = raw[shift[2]:shift[2] + q.size].reshape(q.shape).astype(np.float64)
    want, bound, inside = attention(b, q.astype(np.float64), cache.astype(np.float64), key_heads, 1, width ** -0.5)
    assert np.all(np.abs(got - want)[inside] <= rounded(want, bound, np.float16)[inside])
    assert np.all(got[~inside] == 7.0)
    assert np.all(raw[:shift[2]] == 7.0) and np.all(raw[shift[2] + q.size:] == 7.0)
    for x in at + batch + [out]:
        x.free()


@pytest.mark.parametrize("width,rotary_width", [(128, 128), (72, 32), (64, 0)])
@pytest.mark.parametrize("shift", [(0, 0, 0), (1, 0, 0), (0, 2, 0), (0, 0, 4), (4, 4, 4)])
@pytest.mark.parametrize("strides", [(0, 0), (1, 0), (8, 2)])
def test_append_alignment(ipus, ctx, width, rotary_width, shift, strides):
    heads = 3
    b = Batch(np.random.default_rng(72), [5, 0, 1], [20, 7, 33], 8, 1)
    pitches = [heads * width + x for x in strides]
    flat = [halves(ipus, (b.rows * p + 8,), 2 + i) for i, p in enumerate(pitches)]
    keys, values = (x[:b.rows * p].reshape(b.rows, p)[:, :heads * width].reshape(b.rows, heads, width)
                    for x, p in zip(flat, pitches))
    cache = halves(ipus, (b.pages, 2, heads, 8, width), 1)
    f, _ = ipus.rotary_frequencies(max(2, rotary_width))
    src = [ctx.upload(np.concatenate([np.zeros(n, np.float16), x])) for n, x in zip(shift, flat)]
    out = ctx.upload(np.concatenate([np.full(shift[2], 7.0, np.float16), cache.ravel(), np.full(8, 7.0, np.float16)]))
    rest = [ctx.upload(f)] + upload_batch(ctx, b)
    ctx.launch("ipu_stack_append_pages_f16", out.ptr + 2 * shift[2],
               [s.ptr + 2 * n for s, n in zip(src, shift)] + rest,
               append_scalars(b, heads, width, rotary_width, 1, 0.0, pitches))
    raw = out.download(np.float16)
    got = raw[shift[2]:shift[2] + cache.size].reshape(cache.shape).astype(np.float64)
    want, bound = append64(b, cache, keys, values, f[:rotary_width // 2], 1.0, rotary_width, 1)
    assert np.all(np.abs(got - want) <= bound)
    assert np.all(raw[:shift[2]] == 7.0) and np.all(raw[shift[2] + cache.size:] == 7.0)
    for x in src + rest + [out]:
        x.free()
