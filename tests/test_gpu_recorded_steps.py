"""A decoder's step recorded once and replayed as offsets, lengths, tables and inputs
change, on a stream of its own beside the context's launches."""
from __future__ import annotations

import struct

import numpy as np
import pytest

from decoder_forms import Batch, attention, norm_rotate, rounded
from test_gpu_caller_capture import Recording
from test_gpu_pages import attention_scalars, attention_symbol, halves, upload_batch

pytestmark = pytest.mark.gpu


def bits(x):
    return struct.unpack("<I", struct.pack("<f", x))[0]


@pytest.mark.parametrize("query,heads,width", [(8, 2, 128), (4, 4, 72), (3, 1, 65)])
def test_steps_of_other_lengths(ipus, ctx, query, heads, width):
    """Norm and rotation in place, append, attention: rows that begin, end and
    move to other sequences between the replays of one graph."""
    page_rows, columns, rows, total, epsilon = 16, 200, 45, query + 2 * heads, 1e-6
    steps = [([40, 1, 0], [40, 900, 0]), ([1, 1, 1], [41, 901, 1]), ([0, 3, 42], [41, 904, 43]),
             ([1, 0, 1], [3000, 904, 44]), ([0, 0, 0], [41, 904, 44])]
    rng = np.random.default_rng(61)
    pages = 300
    table = np.full((3, columns), -1, np.int32)
    free = list(rng.permutation(pages))
    for s, n in enumerate((190, 60, 4)):
        table[s, :n] = [free.pop() for _ in range(n)]
    cache = halves(ipus, (pages, 2, heads, page_rows, width), 1)
    weights = [(1 + 0.1 * halves(ipus, (width,), t).astype(np.float32)).astype(np.float16) for t in (2, 3)]
    f, _ = ipus.rotary_frequencies(width // 2 * 2)
    dcache, dw, df = ctx.upload(cache), [ctx.upload(w) for w in weights], ctx.upload(f)
    dx, dp = ctx.alloc(rows * total * width * 2), ctx.alloc(rows * 4)
    batch = [ctx.upload(table), ctx.alloc(16), ctx.alloc(12)]
    out = ctx.alloc(rows * query * width * 2)
    pitch = total * width
    noise = [ctx.upload(halves(ipus, (70, query, width), 4)), ctx.alloc(70 * query * width * 2)]
    other = upload_batch(ctx, Batch(np.random.default_rng(62), [70], [2000], page_rows))
    recording = Recording(ipus, ctx)
    with recording:
        ctx.launch("ipu_stack_norm_rotary_f16", dx, [dx, *dw, dp, df],
                   [rows, query, heads, width, width // 2 * 2, 0, pitch, pitch, bits(epsilon), 0])
        ctx.launch("ipu_stack_append_pages_f16", dcache,
                   [dx.ptr + query * width * 2, dx.ptr + (query + heads) * width * 2, df] + batch,
                   [3, rows, heads, width, pitch, pitch, 0, 0, 0, pages, page_rows, columns])
        ctx.launch("ipu_stack_attention_pages_f16", out, [dx, dcache] + batch,
                   [3, rows, 42, query, heads, width, pitch, pages, page_rows, columns, 1, 0])
    eps = float(np.float32(epsilon))
    for step, (n, k) in enumerate(steps):
        offsets = np.concatenate([[0], np.cumsum(n)]).astype(np.int32)
        x = halves(ipus, (rows, total, width), 7 + step)
        position = np.zeros(rows, np.int32)
        for s in range(3):
            position[offsets[s]:offsets[s + 1]] = k[s] - n[s] + np.arange(n[s])
        for buf, a in ((dx, x), (dp, position), (batch[1], offsets), (batch[2], np.array(k, np.int32)),
                       (out, np.full((rows, query, width), 7.0, np.float16))):
            ctx.write(buf, a)
        ctx.sync()
        recording.replay()
        ctx.launch("ipu_stack_attention_pages_f16", noise[1], [noise[0], dcache] + other,
                   [1, 70, 70, query, heads, width, query * width, pages, page_rows, 126, 1, 0])
        recording.sync()
        ctx.sync()
        turned = dx.download(np.float16).reshape(x.shape)
        per_head = np.stack([weights[0]] * query + [weights[1]] * heads).astype(np.float64)
        want, bound = norm_rotate(x[:, :query + heads].astype(np.float64), per_head, eps, position, f, 1.0,
                                  width // 2 * 2, 0)
        assert np.all(np.abs(turned[:, :query + heads].astype(np.float64) - want)
                      <= rounded(want, bound, np.float16))
        for s in range(3):
            at = slice(int(offsets[s]), int(offsets[s + 1]))
            page, row = table[s][position[at] // page_rows], position[at] % page_rows
            cache[page, 0, :, row] = turned[at, query:query + heads]
            cache[page, 1, :, row] = turned[at, query + heads:]
        assert np.array_equal(dcache.download(np.float16).reshape(cache.shape), cache)
        b = Batch(np.random.default_rng(1), n, k, page_rows)
        b.table, b.columns, b.pages, b.offsets = table, columns, pages, offsets
        want, bound, inside = attention(b, turned[:, :query].astype(np.float64), cache.astype(np.float64), heads,
                                        1, width ** -0.5)
        inside[sum(n):] = False
        got = out.download(np.float16).reshape(rows, query, width).astype(np.float64)
        assert np.all(np.abs(got - want)[inside] <= rounded(want, bound, np.float16)[inside])
        assert np.all(got[~inside] == 7.0)
    recording.close()
    for buf in [dcache, df, dx, dp, out] + dw + batch + noise + other:
        buf.free()


def test_recorded_shared_prefix(ipus, ctx):
    """Eager launches read the prefix once, in a launch of its own and the context's
    workspace; the recorded one does without, beside them."""
    heads, key_heads, width = 16, 4, 64
    b = Batch(np.random.default_rng(63), [1] * 300, [1003 + i % 40 for i in range(300)], 16, 2, shared=1000)
    cache = halves(ipus, (b.pages, 2, key_heads, 16, width), 1)
    q = halves(ipus, (b.rows, heads, width), 2)
    ins = [ctx.upload(q), ctx.upload(cache)] + upload_batch(ctx, b)
    outs = [ctx.alloc(q.nbytes) for _ in range(2)]
    scalars = attention_scalars(b, heads, key_heads, width, 1)
    recording = Recording(ipus, ctx)
    with recording:
        ctx.launch(attention_symbol(b), outs[0], ins, scalars)
    want, bound, inside = attention(b, q.astype(np.float64), cache.astype(np.float64), key_heads, 1, width ** -0.5)
    bound = rounded(want, bound, np.float16)
    for _ in range(3):
        for out in outs:
            ctx.write(out, np.full(q.shape, 7.0, np.float16))
        ctx.sync()
        for _ in range(4):
            recording.replay()
            ctx.launch(attention_symbol(b), outs[1], ins, scalars)
        recording.sync()
        ctx.sync()
        for out in outs:
            got = out.download(np.float16).reshape(q.shape).astype(np.float64)
            assert np.all(np.abs(got - want)[inside] <= bound[inside])
            assert np.all(got[~inside] == 7.0)
    recording.close()
    for buf in ins + outs:
        buf.free()
