"""The paged cache: appends and the attention that reads it, against float64,
alone and as a decoder runs them one after the other."""
from __future__ import annotations

import struct

import numpy as np
import pytest

from decoder_forms import Batch, attention, norm_rotate, rotate, rounded
from test_gpu_caller_capture import Recording

pytestmark = pytest.mark.gpu


def bits(x):
    return struct.unpack("<I", struct.pack("<f", x))[0]


def halves(ipus, shape, tensor, scale=1.0, seed=93):
    return ipus.synth_f16(int(np.prod(shape)), seed, tensor, ipus.NORMAL, scale).view(np.float16).reshape(shape)


def append_scalars(b, heads, width, rotary_width, interleaved, magnitude=0.0, pitches=None):
    pitches = pitches or (heads * width, heads * width)
    return [b.sequences(), b.rows, heads, width, *pitches, rotary_width, interleaved,
            bits(magnitude) if magnitude else 0, b.pages, b.page_rows, b.columns]


def attention_scalars(b, heads, key_heads, width, causal, max_rows=None, scale=0.0, pitch=None):
    s = [b.sequences(), b.rows, max(b.n) if max_rows is None else max_rows, heads, key_heads, width,
         pitch or heads * width, b.pages, b.page_rows, b.columns, int(causal), bits(scale) if scale else 0]
    return s + ([b.shared] if b.shared else [])


def attention_symbol(b):
    return "ipu_stack_attention_shared_pages_f16" if b.shared else "ipu_stack_attention_pages_f16"


def upload_batch(ctx, b):
    return [ctx.upload(a) for a in (b.table, b.offsets, b.lengths)]


def append64(b, cache, keys, values, f, magnitude, rotary_width, interleaved):
    """The cache after the append, and the bound (0 where bits are copied)."""
    want, bound = cache.astype(np.float64), np.zeros(cache.shape)
    written = np.zeros(cache.shape, bool)
    for s in range(b.sequences()):
        first, n = int(b.offsets[s]), b.n[s]
        position = b.k[s] - n + np.arange(n)
        keep = position >= 0
        position = position[keep]
        t = first + np.arange(n)[keep]
        column = position // b.page_rows
        inside = column < b.columns
        page = np.where(inside, b.table[s][np.minimum(column, b.columns - 1)], -1)
        good = (page >= 0) & (page < b.pages)
        t, page, row, position = t[good], page[good], (position % b.page_rows)[good], position[good]
        turned, e = rotate(keys[t].astype(np.float64), position, f, magnitude, rotary_width, interleaved)
        e[..., :rotary_width] = rounded(turned, e, np.float16)[..., :rotary_width]
        want[page, 0, :, row], bound[page, 0, :, row] = turned, e
        want[page, 1, :, row] = values[t]
    return want, bound


@pytest.mark.parametrize("rows,lengths,heads,width,rotary_width,interleaved,page_rows,pad", [
    ([1], [1], 1, 2, 2, 0, 1, 0),
    ([1] * 5, [1, 7, 16, 17, 300], 8, 128, 128, 0, 16, 3),
    ([3, 0, 40, 1], [3, 0, 77, 5], 4, 64, 32, 1, 8, 0),
    ([130, 257], [500, 257], 2, 72, 72, 0, 64, 11),
    ([5, 2], [5, 9], 3, 65, 10, 1, 4, 1),
    ([4, 3], [4, 12], 2, 80, 0, 0, 32, 0),
    ([9], [2000], 1, 2048, 2048, 0, 16, 0),
    ([1] * 70 + [0] * 5 + [2] * 60, [9] * 70 + [0] * 5 + [33] * 60, 2, 96, 24, 0, 16, 0),
    ([1] * 4200, [3] * 4200, 1, 32, 32, 1, 2, 2),
    ([300] * 130, [311] * 130, 1, 8, 4, 0, 16, 5),
    ([700] * 9, [900] * 9, 3, 40, 20, 0, 64, 1),
])
def test_append(ipus, ctx, rows, lengths, heads, width, rotary_width, interleaved, page_rows, pad):
    b = Batch(np.random.default_rng(width), rows, lengths, page_rows, pad)
    cache = halves(ipus, (b.pages, 2, heads, page_rows, width), 1)
    keys, values = (halves(ipus, (b.rows, heads, width), t) for t in (2, 3))
    f, _ = ipus.rotary_frequencies(max(2, rotary_width))
    bufs = [ctx.upload(a) for a in (keys, values, f)] + upload_batch(ctx, b)
    out = ctx.upload(cache)
    ctx.launch("ipu_stack_append_pages_f16", out, bufs,
               append_scalars(b, heads, width, rotary_width, interleaved, 1.5))
    got = out.download(np.float16).reshape(cache.shape).astype(np.float64)
    want, bound = append64(b, cache, keys, values, f[:rotary_width // 2], 1.5, rotary_width, interleaved)
    assert np.all(np.abs(got - want) <= bound)
    for x in bufs + [out]:
        x.free()


def test_append_from_a_fused_projection(ipus, ctx):
    """Keys and values read from the rows of one wider buffer."""
    heads, query, width = 4, 8, 64
    b = Batch(np.random.default_rng(3), [2, 30], [40, 31], 16)
    pitch = (query + 2 * heads) * width
    x = halves(ipus, (b.rows, pitch), 4)
    cache = halves(ipus, (b.pages, 2, heads, 16, width), 1)
    f, _ = ipus.rotary_frequencies(width)
    src, out = ctx.upload(x), ctx.upload(cache)
    rest = [ctx.upload(f)] + upload_batch(ctx, b)
    ctx.launch("ipu_stack_append_pages_f16", out,
               [src.ptr + query * width * 2, src.ptr + (query + heads) * width * 2] + rest,
               append_scalars(b, heads, width, width, 0, 0.0, (pitch, pitch)))
    part = x.reshape(b.rows, query + 2 * heads, width)
    want, bound = append64(b, cache, part[:, query:query + heads], part[:, query + heads:], f, 1.0, width, 0)
    got = out.download(np.float16).reshape(cache.shape).astype(np.float64)
    assert np.all(np.abs(got - want) <= bound)
    for buf in [src, out] + rest:
        buf.free()


def spoil(b):
    """Entries and lengths that have no place: a page below 0, one past the
    cache, a length past the table, rows before position 0."""
    b.table[0, 1] = -7
    b.table[1, 0] = b.pages
    b.lengths[2] = b.columns * b.page_rows + 5
    b.k[2] = int(b.lengths[2])
    b.lengths[3] = b.n[3] - 2
    b.k[3] = b.n[3] - 2
    return b


def test_append_without_a_place(ipus, ctx):
    heads, width, page_rows = 2, 64, 8
    b = spoil(Batch(np.random.default_rng(5), [20, 5, 9, 6], [30, 12, 24, 20], page_rows, 4))
    cache = halves(ipus, (b.pages, 2, heads, page_rows, width), 1)
    keys, values = (halves(ipus, (b.rows, heads, width), t) for t in (2, 3))
    f, _ = ipus.rotary_frequencies(width)
    bufs = [ctx.upload(a) for a in (keys, values, f)] + upload_batch(ctx, b)
    out = ctx.upload(cache)
    ctx.launch("ipu_stack_append_pages_f16", out, bufs, append_scalars(b, heads, width, width, 0))
    got = out.download(np.float16).reshape(cache.shape).astype(np.float64)
    want, bound = append64(b, cache, keys, values, f, 1.0, width, 0)
    assert np.all(np.abs(got - want) <= bound)
    for x in bufs + [out]:
        x.free()


def check_attention(ipus, ctx, b, heads, key_heads, width, causal, max_rows=None, scale=0.0, seed=93,
                    change=None, q_scale=1.0):
    cache = halves(ipus, (b.pages, 2, key_heads, b.page_rows, width), 1, seed=seed)
    q = halves(ipus, (b.rows, heads, width), 2, q_scale, seed=seed)
    if change:
        change(cache, q)
    bufs = [ctx.upload(q), ctx.upload(cache)] + upload_batch(ctx, b)
    out = ctx.upload(np.full(q.size + 8, 7.0, np.float16))
    scalars = attention_scalars(b, heads, key_heads, width, causal, max_rows, scale)
    ctx.launch(attention_symbol(b), out, bufs, scalars)
    raw = out.download(np.float16)
    with np.errstate(invalid="ignore", over="ignore"):
        want, bound, inside = attention(b, q.astype(np.float64), cache.astype(np.float64), key_heads,
                                        causal, scale or width ** -0.5)
    got = raw[:q.size].reshape(q.shape).astype(np.float64)
    assert np.all(got[~inside] == 7.0) and np.all(raw[q.size:] == 7.0)
    bound = rounded(want, bound, np.float16)
    assert np.all(np.abs(got - want)[inside] <= bound[inside])
    # Once more: the same bits.
    ctx.launch(attention_symbol(b), out, bufs, scalars)
    assert np.array_equal(out.download(np.float16), raw)
    for x in bufs + [out]:
        x.free()
    return got


DECODE = [
    # rows, lengths, query heads, key heads, width, page_rows, pad
    ([1], [1], 1, 1, 8, 1, 0),
    ([1] * 4, [1, 15, 16, 700], 16, 16, 64, 16, 0),
    ([1] * 3, [4099, 31, 129], 32, 8, 128, 64, 2),
    ([1] * 6, [33, 0, 1000, 64, 127, 2], 14, 2, 80, 8, 0),
    ([2, 1, 3], [2, 300, 900], 8, 1, 96, 32, 0),
    ([5, 0, 1], [5, 77, 2100], 12, 12, 72, 128, 1),
    ([1] * 2, [1500, 3], 16, 1, 256, 16, 0),
    ([1] * 2, [600, 61], 24, 1, 192, 4, 0),
    ([1] * 130, [17 + 3 * i for i in range(130)], 4, 4, 32, 16, 0),
    ([1] * 2, [90, 5], 3, 1, 65, 2, 0),
    ([2], [40], 2, 1, 1000, 16, 0),
    ([3, 4], [50, 10], 6, 3, 40, 16, 0),
    # 17 to 32 queries of a key head: short tables, and long ones (two tiles).
    ([3, 1, 0, 2], [300, 40, 0, 65], 16, 2, 128, 16, 1),
    ([3, 1, 0, 2], [300, 4000, 0, 65], 16, 2, 128, 16, 1),
    ([2, 2], [2700, 31], 14, 1, 96, 64, 0),
    ([4], [5000], 6, 1, 64, 128, 0),
    ([2] * 3, [2600, 1, 100], 28, 2, 32, 8, 2),
]


@pytest.mark.parametrize("rows,lengths,heads,key_heads,width,page_rows,pad", DECODE)
@pytest.mark.parametrize("causal", [0, 1])
def test_attention_decode(ipus, ctx, rows, lengths, heads, key_heads, width, page_rows, pad, causal):
    b = Batch(np.random.default_rng(width), rows, lengths, page_rows, pad)
    check_attention(ipus, ctx, b, heads, key_heads, width, causal)


CHUNKS = [
    ([64], [64], 1, 1, 64, 16, 0),
    ([100, 1, 300], [100, 500, 1000], 8, 2, 128, 64, 3),
    ([33, 129], [700, 129], 4, 4, 72, 8, 0),
    ([257], [300], 7, 1, 96, 32, 0),
    ([40, 0, 17], [2000, 0, 17], 4, 1, 256, 128, 0),
    ([200], [333], 3, 3, 32, 16, 0),
    ([130, 65], [131, 1000], 2, 2, 192, 4, 0),
    ([20, 30], [20, 90], 4, 2, 65, 8, 0),
    ([90], [1], 16, 8, 128, 16, 0),
]


@pytest.mark.parametrize("rows,lengths,heads,key_heads,width,page_rows,pad", CHUNKS)
@pytest.mark.parametrize("causal", [0, 1])
def test_attention_chunks(ipus, ctx, rows, lengths, heads, key_heads, width, page_rows, pad, causal):
    b = Batch(np.random.default_rng(width), rows, lengths, page_rows, pad)
    check_attention(ipus, ctx, b, heads, key_heads, width, causal)


SPLIT = [
    # blocks of queries whose keys are cut, up to 16 times, beside ones that are not
    ([70], [4100], 4, 1, 64, 16, 0),
    ([64, 64], [3000, 90], 4, 4, 128, 64, 0),
    ([33, 1, 40, 1], [1100, 2500, 64, 9], 2, 2, 96, 8, 2),
    ([60, 60], [1025, 1024], 2, 1, 128, 32, 0),
    ([40], [513], 3, 3, 256, 16, 0),
    ([129], [2200], 1, 1, 192, 128, 1),
    ([200], [5000], 5, 1, 32, 16, 0),
    ([100, 1, 3, 1], [150, 2700, 40, 1], 8, 2, 128, 64, 0),
    ([30, 1, 0, 2], [2600, 3000, 5, 2], 16, 16, 72, 16, 3),
    ([1, 90, 17], [5000, 91, 2000], 8, 8, 256, 128, 0),
]


@pytest.mark.parametrize("rows,lengths,heads,key_heads,width,page_rows,pad", SPLIT)
@pytest.mark.parametrize("causal", [0, 1])
def test_attention_with_split_keys(ipus, ctx, rows, lengths, heads, key_heads, width, page_rows, pad, causal):
    b = Batch(np.random.default_rng(width), rows, lengths, page_rows, pad)
    check_attention(ipus, ctx, b, heads, key_heads, width, causal)


MANY = [
    # sequences (their rows in turn), lengths from, to, query heads, key heads, width, page_rows
    (220, [1], 65, 96, 16, 4, 128, 16),
    (330, [1], 0, 64, 2, 2, 64, 8),
    (160, [2], 40, 64, 64, 4, 96, 32),
    (100, [1], 8, 30, 8, 8, 256, 16),
    (100, [1, 0], 90, 90, 16, 16, 192, 64),
    (1100, [1], 1, 6, 8, 8, 32, 2),
    (260, [3, 2, 5], 33, 60, 8, 4, 72, 4),
]


@pytest.mark.parametrize("sequences,rows,low,high,heads,key_heads,width,page_rows", MANY)
@pytest.mark.parametrize("causal", [0, 1])
def test_attention_of_many_short_sequences(ipus, ctx, sequences, rows, low, high, heads, key_heads, width, page_rows,
                                           causal):
    rng = np.random.default_rng(sequences)
    n = [rows[s % len(rows)] for s in range(sequences)]
    lengths = [int(x) for x in rng.integers(low, high + 1, sequences)]
    b = Batch(rng, n, lengths, page_rows, 3)
    check_attention(ipus, ctx, b, heads, key_heads, width, causal)

    def spoilt(cache, q):  # the last row's own value, which the rows before it may not read
        for s in range(0, sequences, 7):
            _, page, row = b.places(s)
            if len(page) and b.n[s] > 1:
                cache[page[-1], 1, 0, row[-1], 1] = np.nan

    if causal and max(rows) > 1:
        cache = halves(ipus, (b.pages, 2, key_heads, page_rows, width), 1)
        q = halves(ipus, (b.rows, heads, width), 2)
        spoilt(cache, q)
        bufs = [ctx.upload(q), ctx.upload(cache)] + upload_batch(ctx, b)
        out = ctx.upload(np.zeros(q.shape, np.float16))
        ctx.launch("ipu_stack_attention_pages_f16", out, bufs, attention_scalars(b, heads, key_heads, width, 1))
        got = out.download(np.float16).reshape(q.shape).astype(np.float64)
        with np.errstate(invalid="ignore"):
            want, bound, inside = attention(b, q.astype(np.float64), cache.astype(np.float64), key_heads, 1,
                                            width ** -0.5)
        bad = np.isnan(want)
        assert np.any(bad) and np.array_equal(np.isnan(got)[inside], bad[inside])
        good = inside[:, None, None] & ~bad
        assert np.all(np.abs(got - want)[good] <= rounded(want, bound, np.float16)[good])
        for x in bufs + [out]:
            x.free()


@pytest.mark.parametrize("max_rows", [0, 1, 7, 1000])
def test_attention_is_whole_for_any_row_hint(ipus, ctx, max_rows):
    b = Batch(np.random.default_rng(2), [70, 1, 9], [300, 400, 9], 16)
    check_attention(ipus, ctx, b, 8, 2, 128, 1, max_rows)


@pytest.mark.parametrize("rows", [[1, 1, 1, 1], [70, 1, 20, 40]])
@pytest.mark.parametrize("width", [128, 65])
def test_attention_without_a_place(ipus, ctx, rows, width):
    """Keys on pages outside the cache or past the table carry no weight; rows
    before position 0 read nothing."""
    b = Batch(np.random.default_rng(6), rows, [100, 90, 80, 60], 16, 2)
    b.table[0, 1] = -7
    b.table[1, :] = b.pages
    b.lengths[2] = b.columns * b.page_rows + 5
    b.k[2] = int(b.lengths[2])
    b.lengths[3] = b.n[3] - 1
    b.k[3] = b.n[3] - 1
    for causal in (0, 1):
        check_attention(ipus, ctx, b, 4, 2, width, causal)


@pytest.mark.parametrize("rows,width", [([1, 1], 128), ([1, 1], 65), ([40, 40], 128), ([1, 1], 256)])
def test_attention_non_finite(ipus, ctx, rows, width):
    """NaN and infinities behind a sequence's end and beyond a row's position are
    never read into a result; keys whose scores are -inf carry no weight, a NaN
    key makes the rows that read it NaN, and no others."""
    b = Batch(np.random.default_rng(8), rows, [75, 130], 16)

    def rest(cache, q):
        # Everything but the keys in use.
        used = np.zeros((b.pages, 16), bool)
        for s in range(2):
            _, page, row = b.places(s)
            used[page, row] = True
        dead = ~used
        cache[:, 0].transpose(0, 2, 1, 3)[dead] = np.nan
        cache[:, 1].transpose(0, 2, 1, 3)[dead] = np.inf

    check_attention(ipus, ctx, b, 4, 2, width, 1, change=rest)

    def minus_infinity(cache, q):
        rest(cache, q)
        q[:, :, 0] = 1.0
        for s in range(2):
            _, page, row = b.places(s)
            cache[page[:20], 0, :, row[:20], 0] = -np.inf

    check_attention(ipus, ctx, b, 4, 2, width, 0, change=minus_infinity)
    # One NaN key of sequence 1.
    cache = halves(ipus, (b.pages, 2, 2, 16, width), 1)
    q = halves(ipus, (b.rows, 4, width), 2)
    _, page, row = b.places(1)
    cache[page[70], 0, 0, row[70], 3] = np.nan
    bufs = [ctx.upload(q), ctx.upload(cache)] + upload_batch(ctx, b)
    out = ctx.alloc(q.nbytes)
    ctx.launch("ipu_stack_attention_pages_f16", out, bufs, attention_scalars(b, 4, 2, width, 0))
    got = out.download(np.float16).reshape(q.shape)
    first = b.n[0]
    assert np.all(np.isnan(got[first:, :2])) and not np.any(np.isnan(got[first:, 2:]))
    assert not np.any(np.isnan(got[:first]))
    for x in bufs + [out]:
        x.free()


@pytest.mark.parametrize("rows,lengths,heads,key_heads,width,page_rows,shared", [
    ([3, 5], [100, 40], 4, 2, 128, 16, 0),        # few rows, one and two query tiles
    ([8, 1], [700, 900], 8, 2, 64, 16, 0),
    ([5], [37], 4, 4, 96, 8, 0),
    ([4], [90], 1, 1, 256, 64, 0),
    ([70, 200], [300, 200], 4, 2, 128, 64, 0),    # blocks
    ([90, 1], [1500, 30], 2, 2, 72, 16, 0),       # split keys
    ([65], [80], 2, 1, 192, 16, 0),
    ([40], [40], 8, 1, 32, 1, 0),
    ([3, 4], [50, 60], 2, 1, 65, 16, 0),          # the general kernel
    ([6, 3, 2], [40, 44, 100], 4, 1, 128, 16, 42),
    ([2] * 300, [1003] * 150 + [1001] * 150, 16, 4, 64, 16, 1002),  # prefix in its own launch
])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_values_that_rows_may_not_read(ipus, ctx, rows, lengths, heads, key_heads, width, page_rows, shared, bad):
    """A non-finite value at a sequence's last position reaches the rows that read it,
    in its column, and none before them."""
    b = Batch(np.random.default_rng(14), rows, lengths, page_rows, shared=shared)
    for c in range((shared + page_rows - 1) // page_rows):
        if b.table[0, c] < 0:
            b.table[0, c] = b.pages - 1
    cache = halves(ipus, (b.pages, 2, key_heads, page_rows, width), 1)
    for s in range(b.sequences()):
        p, page, row = b.places(s)
        cache[page[-1], 1, 0, row[-1], 5] = bad
        cache[page[-1], 0, key_heads - 1, row[-1], 3] = np.nan
    q = halves(ipus, (b.rows, heads, width), 2)
    bufs = [ctx.upload(q), ctx.upload(cache)] + upload_batch(ctx, b)
    out = ctx.alloc(q.nbytes)
    ctx.launch(attention_symbol(b), out, bufs, attention_scalars(b, heads, key_heads, width, 1))
    got = out.download(np.float16).reshape(q.shape).astype(np.float64)
    with np.errstate(invalid="ignore"):
        want, bound, _ = attention(b, q.astype(np.float64), cache.astype(np.float64), key_heads, 1, width ** -0.5)
        bound = rounded(want, bound, np.float16)
    fine = np.isfinite(want)
    assert 0 < np.sum(fine) < fine.size
    assert np.array_equal(np.isfinite(got), fine)
    assert np.all(np.abs(got[fine] - want[fine]) <= bound[fine])
    for x in bufs + [out]:
        x.free()


@pytest.mark.parametrize("q_scale", [0.0, 30.0])
def test_attention_score_ranges(ipus, ctx, q_scale):
    """Equal scores, and scores whose softmax is nearly one key."""
    for rows, lengths in (([1, 1], [900, 33]), ([50], [200])):
        b = Batch(np.random.default_rng(9), rows, lengths, 16)
        check_attention(ipus, ctx, b, 4, 4, 128, 1, q_scale=q_scale)


SHARED = [
    # rows, lengths, heads, key heads, width, page_rows, shared
    ([1] * 4, [300, 260, 257, 900], 8, 2, 128, 16, 256),
    ([1] * 9, [1100 + i for i in range(9)], 16, 4, 64, 64, 1000),   # ends inside a page
    ([1] * 40, [2050 + i for i in range(40)], 4, 4, 128, 16, 2048),
    ([3, 1, 2], [700, 650, 644], 14, 2, 80, 32, 640),
    ([1, 1], [50, 300], 4, 1, 256, 16, 288),                         # shorter than the prefix
    ([60, 1], [400, 300], 4, 2, 128, 16, 256),
    ([1, 1], [100, 90], 2, 1, 65, 16, 64),
    ([5, 0, 4], [131, 0, 130], 16, 16, 72, 8, 128),                  # rows inside the prefix
]


@pytest.mark.parametrize("rows,lengths,heads,key_heads,width,page_rows,shared", SHARED)
def test_attention_shared(ipus, ctx, rows, lengths, heads, key_heads, width, page_rows, shared):
    b = Batch(np.random.default_rng(shared), rows, lengths, page_rows, 1, shared=shared)
    # The first sequence's table holds the whole prefix; the others' entries for
    # it are not read.
    for c in range((shared + page_rows - 1) // page_rows):
        if b.table[0, c] < 0:
            b.table[0, c] = b.pages - 1
    b.table[1:, :shared // page_rows] = -3
    for causal in (0, 1):
        check_attention(ipus, ctx, b, heads, key_heads, width, causal)


ONCE = [
    # As above, large enough that the shared keys get a launch of their own (160 MB saved).
    (300, 1, 1003, 16, 4, 64, 16, 1000),
    (180, 3, 700, 8, 8, 80, 32, 640),
    (260, 1, 1500, 4, 1, 256, 64, 1455),
    (100, 2, 3300, 12, 4, 128, 8, 3296),
    (500, 1, 300, 64, 32, 32, 16, 288),
    # Many with few keys of their own: a wave takes a segment and joins its parts.
    (600, 1, 1003, 16, 4, 64, 16, 1000),
    (400, 2, 700, 64, 4, 96, 32, 690),
    (400, 1, 900, 8, 8, 128, 16, 890),
    (300, 1, 600, 12, 12, 72, 8, 590),
]


@pytest.mark.parametrize("sequences,rows,keys,heads,key_heads,width,page_rows,shared", ONCE)
@pytest.mark.parametrize("causal", [0, 1])
def test_attention_shared_read_once(ipus, ctx, sequences, rows, keys, heads, key_heads, width, page_rows,
                                    shared, causal):
    rng = np.random.default_rng(shared)
    n = rng.integers(0, rows + 1, sequences)
    k = rng.integers(shared - 20, keys + 40, sequences)  # some shorter than the prefix
    k[0] = keys
    n[0], k[3], n[3] = rows, 0, rows
    b = Batch(rng, n, k, page_rows, 3, shared=shared)
    b.table[1:, :shared // page_rows] = -3
    if causal and width == 128:
        b.table[0, 7] = b.pages  # shared keys without a page
    check_attention(ipus, ctx, b, heads, key_heads, width, causal)


def test_positions_past_32_bits(ipus, ctx):
    """A cache and rows of more than 2^32 elements."""
    heads, width, page_rows, pages = 8, 128, 256, 9000
    page_bytes = 2 * heads * page_rows * width * 2
    assert pages * page_bytes // 2 > 1 << 32
    cache = ctx.alloc(pages * page_bytes)
    ctx.memset(cache, 0)
    b = Batch(np.random.default_rng(1), [300, 7], [300, 500], page_rows)
    b.table[:] = np.where(b.table >= 0, b.table + 8990, -1)
    b.pages = pages
    keys, values = (halves(ipus, (b.rows, heads, width), t) for t in (2, 3))
    f, _ = ipus.rotary_frequencies(width)
    batch = upload_batch(ctx, b)
    bufs = [ctx.upload(a) for a in (keys, values, f)] + batch
    ctx.launch("ipu_stack_append_pages_f16", cache, bufs, append_scalars(b, heads, width, width, 0))
    low, high = 8990, 9000
    tail = ipus.DeviceBuffer(ctx, cache.ptr + low * page_bytes, (high - low) * page_bytes)
    host = np.zeros((high - low, 2, heads, page_rows, width), np.float16)
    got = tail.download(np.float16).reshape(host.shape)
    shifted = Batch(np.random.default_rng(1), [300, 7], [300, 500], page_rows)
    want, bound = append64(shifted, host, keys, values, f, 1.0, width, 0)
    assert np.all(np.abs(got.astype(np.float64) - want) <= bound)
    for rows, lengths in (([300, 7], [300, 500]), ([1, 1], [300, 500])):
        a = Batch(np.random.default_rng(1), rows, lengths, page_rows)
        view = Batch(np.random.default_rng(1), rows, lengths, page_rows)
        a.table, a.pages = b.table, pages
        q = halves(ipus, (a.rows, 16, width), 4)
        ins = [ctx.upload(q), cache] + upload_batch(ctx, a)
        out = ctx.alloc(q.nbytes)
        ctx.launch("ipu_stack_attention_pages_f16", out, ins, attention_scalars(a, 16, heads, width, 1))
        view.table = shifted.table
        want, bound, _ = attention(view, q.astype(np.float64), got.astype(np.float64), heads, 1, width ** -0.5)
        result = out.download(np.float16).reshape(q.shape).astype(np.float64)
        assert np.all(np.abs(result - want) <= rounded(want, bound, np.float16))
        for x in [ins[0], out] + ins[2:]:
            x.free()
    # Rotary rows 2^31 elements apart, in the same buffer: the third starts at 2^32.
    stride, rows = 1 << 31, 3
    x = halves(ipus, (rows, width), 5)
    views = [ipus.DeviceBuffer(ctx, cache.ptr + r * stride * 2, width * 2) for r in range(rows)]
    for r in range(rows):
        ctx.write(views[r], x[r])
    position = np.array([5, 6, 7], np.int32)
    dp = ctx.upload(position)
    ctx.launch("ipu_stack_rotary_f16", cache, [cache, dp, bufs[2]],
               [rows, 1, width, width, 0, stride, width, stride, width, 0])
    want, bound = rotate(x.astype(np.float64)[:, None], position, f, 1.0, width, False)
    turned = np.stack([v.download(np.float16) for v in views]).astype(np.float64)[:, None]
    assert np.all(np.abs(turned - want) <= rounded(want, bound, np.float16))
    for x in bufs + [cache, dp]:
        x.free()


def test_recorded_launches(ipus, ctx):
    """A caller's graph of a decoder step, replayed on a stream of its own beside the
    context's launches: what it records uses no memory of the context."""
    query, heads, width, page_rows = 8, 2, 128, 16
    rows, lengths = [1] * 5 + [40], [3000, 17, 900, 1, 333, 700]
    b = Batch(np.random.default_rng(21), rows, lengths, page_rows, 1)
    start = halves(ipus, (b.pages, 2, heads, page_rows, width), 1)
    q, keys, values = (halves(ipus, (b.rows, h, width), t) for h, t in ((query, 2), (heads, 3), (heads, 4)))
    f, _ = ipus.rotary_frequencies(width)
    position = np.zeros(b.rows, np.int32)
    for s in range(b.sequences()):
        position[b.offsets[s]:b.offsets[s + 1]] = b.k[s] - b.n[s] + np.arange(b.n[s])
    dq, dk, dv, df, dp = (ctx.upload(a) for a in (q, keys, values, f, position))
    batch = upload_batch(ctx, b)
    sets = [(ctx.upload(start), ctx.alloc(q.nbytes), ctx.upload(np.full(q.shape, 7.0, np.float16)))
            for _ in range(2)]
    pitch = query * width

    def launch(cache, turned, out):
        ctx.launch("ipu_stack_rotary_f16", turned, [dq, dp, df],
                   [b.rows, query, width, width, 0, pitch, width, pitch, width, 0])
        ctx.launch("ipu_stack_append_pages_f16", cache, [dk, dv, df] + batch,
                   append_scalars(b, heads, width, width, 0))
        ctx.launch("ipu_stack_attention_pages_f16", out, [turned, cache] + batch,
                   attention_scalars(b, query, heads, width, 1))

    def check(cache, turned, out):
        got_cache = cache.download(np.float16).reshape(start.shape)
        want, bound = append64(b, start, keys, values, f, 1.0, width, 0)
        assert np.all(np.abs(got_cache.astype(np.float64) - want) <= bound)
        got_q = turned.download(np.float16).reshape(q.shape)
        want, bound, inside = attention(b, got_q.astype(np.float64), got_cache.astype(np.float64), heads, 1,
                                        width ** -0.5)
        got = out.download(np.float16).reshape(q.shape).astype(np.float64)
        assert np.all(np.abs(got - want)[inside] <= rounded(want, bound, np.float16)[inside])
        assert np.all(got[~inside] == 7.0)

    recording = Recording(ipus, ctx)
    with recording:
        launch(*sets[0])
    for _ in range(4):
        for cache, turned, out in sets:
            ctx.write(cache, start)
            ctx.memset(turned, 0xFF)
            ctx.write(out, np.full(q.shape, 7.0, np.float16))
        ctx.sync()
        recording.replay()
        launch(*sets[1])
        recording.replay()
        ctx.sync()
        recording.sync()
        check(*sets[0])
        check(*sets[1])
    recording.close()
    for x in [dq, dk, dv, df, dp] + batch + [y for group in sets for y in group]:
        x.free()


def test_two_contexts_at_once(ipus, ctx):
    """Launches of two contexts on one device run side by side, each with its own
    workspace."""
    other = ipus.Context(0)
    b = Batch(np.random.default_rng(31), [1] * 3 + [50], [2500, 1300, 800, 600], 16)
    cache = halves(ipus, (b.pages, 2, 2, 16, 128), 1)
    runs = []
    for c, t in ((ctx, 2), (other, 3)):
        q = halves(ipus, (b.rows, 8, 128), t)
        ins = [c.upload(q), c.upload(cache)] + upload_batch(c, b)
        runs.append((c, q, ins, c.alloc(q.nbytes)))
    for _ in range(20):
        for c, q, ins, out in runs:
            c.launch("ipu_stack_attention_pages_f16", out, ins, attention_scalars(b, 8, 2, 128, 1))
    for c, q, ins, out in runs:
        want, bound, _ = attention(b, q.astype(np.float64), cache.astype(np.float64), 2, 1, 128 ** -0.5)
        got = out.download(np.float16).reshape(q.shape).astype(np.float64)
        assert np.all(np.abs(got - want) <= rounded(want, bound, np.float16))
        for x in ins + [out]:
            x.free()
    other.close()


def test_decoder_steps(ipus, ctx):
    """What a decoder does per layer, two prompts and then four tokens: norm and
    turn the queries and keys of the fused projection in place, append, attend."""
    query, heads, width, page_rows, epsilon = 8, 2, 64, 16, 1e-6
    total = query + 2 * heads
    f, _ = ipus.rotary_frequencies(width)
    weights = [(1 + 0.1 * halves(ipus, (width,), t).astype(np.float32)).astype(np.float16) for t in (5, 6)]
    steps = [([37, 5], [37, 5])] + [([1, 1], [38 + i, 6 + i]) for i in range(4)]
    whole = Batch(np.random.default_rng(12), steps[-1][0], steps[-1][1], page_rows)
    cache = np.zeros((whole.pages, 2, heads, page_rows, width), np.float16)
    dcache, dw, df = ctx.upload(cache), [ctx.upload(w) for w in weights], ctx.upload(f)
    eps = float(np.float32(epsilon))
    for step, (rows, lengths) in enumerate(steps):
        b = Batch(np.random.default_rng(12), rows, lengths, page_rows)
        b.table, b.columns, b.pages = whole.table, whole.columns, whole.pages
        x = halves(ipus, (b.rows, total, width), 7 + step)
        position = np.concatenate([k - n + np.arange(n) for n, k in zip(rows, lengths)]).astype(np.int32)
        dx, dp = ctx.upload(x), ctx.upload(position)
        batch = upload_batch(ctx, b)
        out = ctx.alloc(b.rows * query * width * 2)
        pitch = total * width
        ctx.launch("ipu_stack_norm_rotary_f16", dx, [dx, *dw, dp, df],
                   [b.rows, query, heads, width, width, 0, pitch, pitch, bits(epsilon), 0])
        ctx.launch("ipu_stack_append_pages_f16", dcache,
                   [dx.ptr + query * width * 2, dx.ptr + (query + heads) * width * 2, df] + batch,
                   append_scalars(b, heads, width, 0, 0, 0.0, (pitch, pitch)))
        ctx.launch("ipu_stack_attention_pages_f16", out, [dx, dcache] + batch,
                   attention_scalars(b, query, heads, width, 1, pitch=pitch))
        # Each kernel against float64 of its own inputs.
        turned = dx.download(np.float16).reshape(x.shape)
        per_head = np.stack([weights[0]] * query + [weights[1]] * heads).astype(np.float64)
        want, bound = norm_rotate(x[:, :query + heads].astype(np.float64), per_head, eps, position, f, 1.0,
                                  width, 0)
        assert np.all(np.abs(turned[:, :query + heads].astype(np.float64) - want)
                      <= rounded(want, bound, np.float16))
        for s in range(2):
            at = slice(int(b.offsets[s]), int(b.offsets[s + 1]))
            p = position[at]
            page, row = b.table[s][p // page_rows], p % page_rows
            cache[page, 0, :, row] = turned[at, query:query + heads]
            cache[page, 1, :, row] = turned[at, query + heads:]
        got_cache = dcache.download(np.float16).reshape(cache.shape)
        assert np.array_equal(got_cache, cache)
        want, bound, _ = attention(b, turned[:, :query].astype(np.float64), cache.astype(np.float64), heads,
                                   1, width ** -0.5)
        got = out.download(np.float16).reshape(b.rows, query, width).astype(np.float64)
        assert np.all(np.abs(got - want) <= rounded(want, bound, np.float16))
        for buf in [dx, dp, out] + batch:
            buf.free()
    for buf in [dcache, df] + dw:
        buf.free()


def test_refusals(ipus, ctx):
    buf = ctx.alloc(4096)
    for at in range(5):  # odd addresses: fp16 by 1, int32 by 2
        inputs = [buf.ptr] * 5
        inputs[at] += 1 if at < 2 else 2
        with pytest.raises(ipus.IpusError) as e:
            ctx.launch("ipu_stack_attention_pages_f16", buf.ptr + 2048, inputs,
                       [1, 1, 1, 1, 1, 8, 8, 1, 1, 1, 0, 0])
        assert e.value.status == ipus.ERROR_INVALID_ARGUMENT
    for at in range(6):
        inputs = [buf.ptr] * 6
        inputs[at] += 1 if at < 2 else 2
        with pytest.raises(ipus.IpusError) as e:
            ctx.launch("ipu_stack_append_pages_f16", buf.ptr + 2048, inputs,
                       [1, 1, 1, 8, 8, 8, 0, 0, 0, 1, 1, 1])
        assert e.value.status == ipus.ERROR_INVALID_ARGUMENT
    # No rows or no sequences: nothing to do.
    ctx.launch("ipu_stack_attention_pages_f16", buf, [buf] * 5, [1, 0, 1, 1, 1, 8, 8, 1, 1, 1, 0, 0])
    ctx.launch("ipu_stack_append_pages_f16", buf, [buf] * 6, [0, 5, 1, 8, 8, 8, 0, 0, 0, 1, 1, 1])
    buf.free()
