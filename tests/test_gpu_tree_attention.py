"""Attention of trees of drafted tokens over the paged cache, against float64."""
from __future__ import annotations

import numpy as np
import pytest

from decoder_forms import Batch, attention, rounded
from step_forms import tree, tree_attention, words
from test_gpu_caller_capture import Recording
from test_gpu_pages import attention_scalars, bits, halves, upload_batch

pytestmark = pytest.mark.gpu


def scalars_of(b, heads, key_heads, width, count, max_rows=None, scale=0.0, pitch=None):
    s = attention_scalars(b, heads, key_heads, width, 0, max_rows, scale, pitch)
    s[10] = count
    return s


def check(ipus, ctx, b, masks, heads, key_heads, width, max_rows=None, scale=0.0, change=None, count=None):
    cache = halves(ipus, (b.pages, 2, key_heads, b.page_rows, width), 1)
    q = halves(ipus, (b.rows, heads, width), 2)
    if change:
        change(cache, q)
    count = count or max(1, (max(b.n) + 31) // 32)
    bufs = [ctx.upload(q), ctx.upload(cache)] + upload_batch(ctx, b) + [ctx.upload(words(masks, count))]
    out = ctx.upload(np.full(q.size + 8, 7.0, np.float16))
    launch = ("ipu_stack_attention_tree_pages_f16", out, bufs, scalars_of(b, heads, key_heads, width, count, max_rows, scale))
    ctx.launch(*launch)
    raw = out.download(np.float16)
    read = [m & (1 << 32 * count) - 1 for m in masks]
    with np.errstate(invalid="ignore", over="ignore"):
        want, bound, inside = tree_attention(b, read, q.astype(np.float64), cache.astype(np.float64), key_heads,
                                             scale or width ** -0.5)
    got = raw[:q.size].reshape(q.shape).astype(np.float64)
    assert np.all(got[~inside] == 7.0) and np.all(raw[q.size:] == 7.0)
    bound = rounded(want, bound, np.float16)
    assert np.all((np.abs(got - want) <= bound)[inside])
    ctx.launch(*launch)  # once more: the same bits
    assert np.array_equal(out.download(np.float16), raw)
    for x in bufs + [out]:
        x.free()
    return got


def masks_of(rng, b, unused=0.0):
    masks = [m for n in b.n for m in tree(rng, n, unused)]
    return masks + [~0 & 0xffffffff] * (b.rows - len(masks))


SHAPES = [
    # rows, lengths, query heads, key heads, width, page_rows, pad
    ([1], [1], 1, 1, 8, 1, 0),
    ([8, 5, 1, 8], [300, 5, 64, 1000], 16, 16, 64, 16, 0),
    ([4] * 5, [4, 36, 67, 4100, 129], 32, 8, 128, 64, 2),
    ([4, 2, 0, 1], [2000, 3, 7, 64], 16, 4, 96, 8, 0),
    ([8, 8], [700, 40], 16, 8, 128, 16, 0),
    ([5, 3], [3000, 90], 12, 2, 96, 32, 1),
    ([7, 4], [70, 2700], 16, 4, 64, 16, 0),
    ([3, 6], [3000, 7], 10, 2, 32, 4, 0),
    ([13, 16], [700, 16], 3, 3, 256, 16, 0),
    ([9, 2], [9, 1200], 2, 2, 192, 128, 0),
    ([64, 33, 1], [500, 33, 900], 8, 2, 128, 64, 3),
    ([99, 50], [3000, 60], 4, 4, 72, 32, 5),
    ([65, 31, 32], [65, 95, 2100], 2, 2, 96, 16, 0),
    ([200, 129], [1300, 129], 4, 1, 64, 16, 0),
    ([40, 20], [1000, 30], 2, 1, 256, 16, 1),
    ([70], [400], 3, 3, 32, 8, 0),
    ([100], [333], 2, 1, 192, 4, 0),
    ([64, 2, 1, 70], [2100, 90, 700, 2600], 16, 16, 64, 16, 0),
    ([6, 40], [50, 90], 3, 1, 65, 2, 1),
    ([10], [37], 2, 2, 520, 16, 0),
    ([3] * 220, [3 + i % 90 for i in range(220)], 16, 4, 128, 16, 1),
    ([2, 5, 1] * 90, [40 + i % 20 for i in range(270)], 8, 8, 64, 8, 0),
    # Parts of the keys by all lengths: of up to 64 sequences and more, of more than those are
    # planned for, beside short ones, and a second round of workgroups.
    ([20, 33, 40, 9] * 5, [60, 1500, 3300, 9, 800] * 4, 4, 1, 64, 16, 1),
    ([20, 33, 40] * 30, [60, 1500, 33, 2300, 800] * 18, 2, 1, 32, 16, 0),
    ([40, 18] * 150, [300, 90, 1300] * 100, 1, 1, 32, 64, 0),
    ([130, 40, 0, 300], [2500, 40, 0, 1400], 4, 4, 96, 32, 0),
    ([40] * 9, [1100 + 300 * i for i in range(9)], 2, 2, 256, 16, 0),
]


@pytest.mark.parametrize("rows,lengths,heads,key_heads,width,page_rows,pad", SHAPES)
@pytest.mark.parametrize("unused", [0.0, 0.3])
def test_trees(ipus, ctx, rows, lengths, heads, key_heads, width, page_rows, pad, unused):
    rng = np.random.default_rng(width)
    b = Batch(rng, rows, lengths, page_rows, pad)
    check(ipus, ctx, b, masks_of(rng, b, unused), heads, key_heads, width)


@pytest.mark.parametrize("rows,lengths", [([5, 9], [90, 300]), ([70, 40], [120, 2500])])
@pytest.mark.parametrize("width", [128, 96, 65])
def test_masks_of_any_bits(ipus, ctx, rows, lengths, width):
    """Masks that are no trees (later rows, none, all), wider or narrower than the rows."""
    rng = np.random.default_rng(11)
    b = Batch(rng, rows, lengths, 16)
    masks = [int.from_bytes(rng.bytes(16), "little") for _ in range(b.rows)]
    masks[1], masks[-2] = 0, (1 << 128) - 1
    for count in (1, 2, 3, 4):
        check(ipus, ctx, b, masks, 4, 2, width, count=count)


def test_a_chain_is_causal(ipus, ctx):
    """Every row reading all before it: what the causal operator computes, bit for bit where
    the reference points of the probabilities are the same.  Those of the kernel for many
    queries may be others (a wave's unused queries keep their keys masked in a tree's every
    block, in a causal one's last alone, and a block with such a query sets them anew): both
    are then within the bound of the exact result, and of each other within twice that."""
    rng = np.random.default_rng(12)
    for rows, lengths, heads, key_heads, width in (([4, 1, 3], [70, 9, 2000], 16, 4, 128), ([90, 64], [90, 700], 4, 2, 64),
                                                   ([3, 20], [5, 60], 2, 1, 65)):
        b = Batch(rng, rows, lengths, 16, 1)
        cache, q = halves(ipus, (b.pages, 2, key_heads, 16, width), 1), halves(ipus, (b.rows, heads, width), 2)
        bufs = [ctx.upload(q), ctx.upload(cache)] + upload_batch(ctx, b)
        mask = ctx.upload(words([(2 << i) - 1 for n in rows for i in range(n)] + [0], 3))
        outs = [ctx.upload(np.zeros(q.size, np.float16)) for _ in range(2)]
        ctx.launch("ipu_stack_attention_pages_f16", outs[0], bufs, attention_scalars(b, heads, key_heads, width, 1))
        ctx.launch("ipu_stack_attention_tree_pages_f16", outs[1], bufs + [mask], scalars_of(b, heads, key_heads, width, 3))
        first, second = (o.download(np.float16).reshape(q.shape) for o in outs)
        if max(rows) * heads // key_heads <= 32:
            assert np.array_equal(first, second)
        want, bound, inside = attention(b, q.astype(np.float64), cache.astype(np.float64), key_heads, 1, width ** -0.5)
        apart = np.abs(first.astype(np.float64) - second.astype(np.float64))
        assert np.all((apart <= 2 * rounded(want, bound, np.float16))[inside])
        for x in bufs + outs + [mask]:
            x.free()


@pytest.mark.parametrize("rows,width", [([3, 4], 128), ([3, 4], 64), ([3, 4], 96), ([3, 4], 65), ([60, 70], 128), ([60, 70], 256)])
def test_rows_that_read_nothing(ipus, ctx, rows, width):
    """No prefix and an empty mask: zeros."""
    rng = np.random.default_rng(13)
    b = Batch(rng, rows, [rows[0], rows[1] + 20], 16)
    masks = masks_of(rng, b)
    masks[1] = 0
    got = check(ipus, ctx, b, masks, 4, 2, width)
    assert np.all(got[1] == 0.0)


@pytest.mark.parametrize("max_rows", [0, 1, 9, 1000])
def test_any_row_hint(ipus, ctx, max_rows):
    rng = np.random.default_rng(14)
    b = Batch(rng, [70, 1, 9], [300, 400, 9], 16)
    check(ipus, ctx, b, masks_of(rng, b), 8, 2, 128, max_rows)


@pytest.mark.parametrize("rows", [[4, 4, 4, 4], [70, 1, 20, 40]])
@pytest.mark.parametrize("width", [128, 65])
def test_without_a_place(ipus, ctx, rows, width):
    """Keys on no page, lengths past the table, more rows than keys: row j's key stands at
    position lengths - rows + j still."""
    rng = np.random.default_rng(15)
    b = Batch(rng, rows, [100, 90, 80, 60], 16, 2)
    b.table[0, 1] = -7
    b.table[1, :] = b.pages
    b.lengths[2] = b.columns * b.page_rows + 3
    b.k[2] = int(b.lengths[2])
    b.lengths[3] = b.n[3] - 1
    b.k[3] = b.n[3] - 1
    check(ipus, ctx, b, masks_of(rng, b, 0.1), 4, 2, width)


@pytest.mark.parametrize("rows,lengths,width,heads", [
    ([5, 3], [75, 130], 128, 4), ([5, 3], [75, 130], 64, 4), ([5, 3], [75, 130], 65, 4), ([40, 70], [75, 2000], 128, 4),
    ([40, 70], [75, 2000], 96, 4), ([40, 50], [75, 130], 256, 2), ([6, 3], [3000, 130], 96, 8), ([7, 3], [3000, 130], 64, 8),
    ([7, 3], [3000, 130], 128, 8), ([9, 4], [90, 60], 192, 2)])
def test_values_that_a_row_may_not_read(ipus, ctx, rows, lengths, width, heads):
    """Infinite and NaN keys and values of other branches, and behind the end, reach no row
    that does not read them; those that are read make their column non-finite."""
    rng = np.random.default_rng(16)
    b = Batch(rng, rows, lengths, 16)
    masks = masks_of(rng, b)
    bad = {}
    for s, n in enumerate(rows):  # one drafted row of each sequence: read by its subtree alone
        bad[s] = n // 2

    def spoil(cache, q):
        used = np.zeros((b.pages, 16), bool)
        for s in range(b.sequences()):
            _, page, row = b.places(s)
            used[page, row] = True
        cache[:, 0].transpose(0, 2, 1, 3)[~used] = np.nan
        cache[:, 1].transpose(0, 2, 1, 3)[~used] = np.inf
        for s, j in bad.items():
            p = b.k[s] - b.n[s] + j
            cache[b.table[s, p // 16], 1, :, p % 16, 3] = np.inf
            cache[b.table[s, p // 16], 1, :, p % 16, 5] = np.nan

    count = (max(rows) + 31) // 32
    cache, q = halves(ipus, (b.pages, 2, 2, 16, width), 1), halves(ipus, (b.rows, heads, width), 2)
    spoil(cache, q)
    bufs = [ctx.upload(q), ctx.upload(cache)] + upload_batch(ctx, b) + [ctx.upload(words(masks, count))]
    out = ctx.upload(np.zeros(q.size, np.float16))
    ctx.launch("ipu_stack_attention_tree_pages_f16", out, bufs, scalars_of(b, heads, 2, width, count))
    got = out.download(np.float16).reshape(q.shape).astype(np.float64)
    with np.errstate(invalid="ignore"):
        want, bound, _ = tree_attention(b, masks, q.astype(np.float64), cache.astype(np.float64), 2, width ** -0.5)
    bound = rounded(want, bound, np.float16)
    finite = np.isfinite(want)
    assert np.any(~finite) and np.all(finite[:, :, :3]) and np.array_equal(np.isnan(got), np.isnan(want))
    assert np.array_equal(np.isinf(got), np.isinf(want))
    assert np.all((np.abs(got - want) <= bound)[finite])
    for x in bufs + [out]:
        x.free()


def test_queries_of_a_fused_projection_and_scale(ipus, ctx):
    rng = np.random.default_rng(17)
    heads, key_heads, width, pitch = 8, 2, 64, 1000
    for rows, lengths in (([3, 2], [70, 300]), ([60, 64], [60, 700])):
        b = Batch(rng, rows, lengths, 32)
        masks = masks_of(rng, b)
        cache, x = halves(ipus, (b.pages, 2, key_heads, 32, width), 1), halves(ipus, (b.rows, pitch), 3)
        q = x[:, :heads * width].reshape(b.rows, heads, width)
        bufs = [ctx.upload(x), ctx.upload(cache)] + upload_batch(ctx, b) + [ctx.upload(words(masks, 2))]
        out = ctx.alloc(q.size * 2)
        ctx.launch("ipu_stack_attention_tree_pages_f16", out, bufs, scalars_of(b, heads, key_heads, width, 2, scale=0.21, pitch=pitch))
        got = out.download(np.float16).reshape(q.shape).astype(np.float64)
        want, bound, _ = tree_attention(b, masks, q.astype(np.float64), cache.astype(np.float64), key_heads,
                                        float(np.float32(0.21)))
        assert np.all(np.abs(got - want) <= rounded(want, bound, np.float16))
        for buf in bufs + [out]:
            buf.free()


def test_recorded(ipus, ctx):
    """One recorded launch, trees, lengths and masks that change between the replays, beside
    the context's own launches."""
    heads, key_heads, width, rows, columns, pages = 8, 2, 128, 50, 160, 400
    rng = np.random.default_rng(18)
    table = rng.permutation(pages)[:2 * columns].reshape(2, columns).astype(np.int32)
    cache = halves(ipus, (pages, 2, key_heads, 16, width), 1)
    q = halves(ipus, (rows, heads, width), 2)
    dq, dcache, dtable = ctx.upload(q), ctx.upload(cache), ctx.upload(table)
    offsets, lengths, mask, out, own = ctx.alloc(12), ctx.alloc(8), ctx.alloc(rows * 8), ctx.alloc(q.nbytes), ctx.alloc(q.nbytes)
    scalars = [2, rows, 40, heads, key_heads, width, heads * width, pages, 16, columns, 2, 0]
    bufs = [dq, dcache, dtable, offsets, lengths, mask]
    recording = Recording(ipus, ctx)
    with recording:
        ctx.launch("ipu_stack_attention_tree_pages_f16", out, bufs, scalars)
    for n, k in (([5, 3], [2000, 60]), ([40, 10], [41, 2500]), ([0, 40], [9, 40]), ([1, 1], [2500, 1])):
        b = Batch(np.random.default_rng(1), n, k, 16)
        b.table, b.columns, b.pages, b.rows = table, columns, pages, rows
        masks = masks_of(rng, b, 0.1)
        for buf, a in ((offsets, b.offsets), (lengths, b.lengths), (mask, words(masks, 2)),
                       (out, np.full(q.shape, 7.0, np.float16)), (own, np.full(q.shape, 7.0, np.float16))):
            ctx.write(buf, a)
        ctx.sync()
        recording.replay()
        ctx.launch("ipu_stack_attention_tree_pages_f16", own, bufs, scalars)
        recording.sync()
        ctx.sync()
        want, bound, inside = tree_attention(b, masks, q.astype(np.float64), cache.astype(np.float64), key_heads, width ** -0.5)
        bound = rounded(want, bound, np.float16)
        for o in (out, own):
            got = o.download(np.float16).reshape(q.shape).astype(np.float64)
            assert np.all((np.abs(got - want) <= bound)[inside]) and np.all(got[~inside] == 7.0)
    recording.close()
    for buf in bufs + [out, own]:
        buf.free()
