"""Page tables, slot maps and the removal of rejected drafts on the device, against
their definitions."""
from __future__ import annotations

import numpy as np
import pytest

from decoder_forms import Batch
from step_forms import fit_tables, keep_rows, slot_maps, table_state, tree, words
from test_gpu_caller_capture import Recording

pytestmark = pytest.mark.gpu


def launch_tables(ctx, state, source, lengths, previous, pages, page_rows, columns):
    count = len(lengths)
    ints = [ctx.upload(np.array(a, np.int32)) for a in (state, list(source) or [0], list(lengths) or [0])]
    size = 2 + pages + count * (1 + columns)
    out = ctx.upload(np.full(size + 3, 77, np.int32))
    ctx.launch("ipu_stack_page_tables", out, ints, [count, previous, pages, page_rows, columns])
    got = out.download(np.int32)
    for b in ints + [out]:
        b.free()
    assert np.all(got[size:] == 77)
    return got[:size]


@pytest.mark.parametrize("sequences,columns,page_rows,pages", [
    (1, 1, 1, 1), (1, 700, 16, 900), (5, 9, 8, 30), (64, 40, 16, 2000), (600, 3, 1, 900), (70, 1100, 4, 30000),
    (1500, 20, 64, 20000), (4096, 5, 16, 9000), (3, 0, 16, 5), (33, 17, 65536, 300)])
def test_tables_over_many_steps(ctx, sequences, columns, page_rows, pages):
    """Requests begin, grow, shrink, end, change places and run out of pages."""
    rng = np.random.default_rng(sequences)
    free, rows = [int(p) for p in rng.permutation(pages)], []
    state = table_state(free, rows, pages, columns)
    for step in range(7):
        count = int(rng.integers(max(1, sequences // 2), sequences + 1))
        if step == 5:
            count = 0  # all end
        previous = len(rows)
        source = [int(p) for p in rng.permutation(max(previous, count))[:count]]
        # Some begin, one names a row that another goes on with, some are no row.
        source = [p if p < previous and rng.random() < 0.8 else int(rng.integers(-2, previous + 2)) for p in source]
        most = columns * page_rows
        lengths = [int(rng.integers(-1, most + most // 8 + 2)) for _ in range(count)]
        if step == 3 and count:
            lengths = [int(rng.integers(0, most // 4 + 1)) for _ in range(count)]
        got = launch_tables(ctx, state, source, lengths, previous, pages, page_rows, columns)
        free, rows, missing = fit_tables(free, rows, source, lengths, page_rows, columns)
        state = table_state(free, rows, pages, columns, missing)
        assert np.array_equal(got, state), step


def test_tables_of_the_most_sequences(ctx):
    """4096 rows before and after, in another order."""
    rng = np.random.default_rng(10)
    pages, columns, page_rows, count = 20000, 6, 8, 4096
    free, rows = [int(p) for p in rng.permutation(pages)], []
    state = table_state(free, rows, pages, columns)
    for step in range(3):
        previous = len(rows)
        source = [int(p) for p in rng.permutation(count)] if step else [-1] * count
        lengths = [int(x) for x in rng.integers(0, 45, count)]
        got = launch_tables(ctx, state, source, lengths, previous, pages, page_rows, columns)
        free, rows, missing = fit_tables(free, rows, source, lengths, page_rows, columns)
        state = table_state(free, rows, pages, columns, missing)
        assert np.array_equal(got, state)


def test_tables_of_any_content(ctx):
    """A state that the operator did not write: what comes out is bounded, and what lies
    behind it untouched (no values are promised)."""
    rng = np.random.default_rng(4)
    for _ in range(6):
        state = rng.integers(-2 ** 31, 2 ** 31, 2 + 50 + 9 * 8).astype(np.int32)
        got = launch_tables(ctx, state, rng.integers(-2 ** 31, 2 ** 31, 12), rng.integers(-2 ** 31, 2 ** 31, 12), 9, 50, 16, 7)
        assert 0 <= got[0] <= 50 and np.all((got[52:64] >= 0) & (got[52:64] <= 7))


def launch_slots(ctx, counts, lengths, table, rows, page_rows, pages, mask=None):
    mask = np.zeros((1, 0), np.uint32) if mask is None else mask
    bufs = [ctx.upload(np.array(a, np.int32)) for a in (list(counts) or [0], list(lengths) or [0])]
    bufs += [ctx.upload(table if table.size else np.zeros(1, np.int32)), ctx.upload(mask if mask.size else np.zeros(1, np.uint32))]
    size = len(counts) + 1 + 2 * rows
    out = ctx.upload(np.full(size + 3, 77, np.int32))
    ctx.launch("ipu_stack_slot_maps", out, bufs, [len(counts), rows, pages, page_rows, table.shape[1], mask.shape[1]])
    got = out.download(np.int32)
    for b in bufs + [out]:
        b.free()
    assert np.all(got[size:] == 77)
    return got[:size]


@pytest.mark.parametrize("rows,lengths,page_rows,pad", [
    ([1], [1], 1, 0), ([1] * 64, list(range(1, 65)), 16, 0), ([3, 0, 40, 1], [3, 9, 77, 50], 8, 5),
    ([700, 1, 513], [900, 700, 513], 64, 0), ([1] * 513, [7] * 513, 4, 1), ([0, 0], [5, 0], 16, 3),
    ([2, 0, 1] * 700, [40, 3, 19] * 700, 16, 17), ([], [], 16, 4), ([], [], 16, 0), ([5000], [5000], 128, 0)])
def test_slots(ctx, rows, lengths, page_rows, pad):
    b = Batch(np.random.default_rng(5), rows, lengths, page_rows, pad)
    got = launch_slots(ctx, rows, lengths, b.table, b.rows, page_rows, b.pages)
    assert np.array_equal(got, slot_maps(rows, lengths, b.table, b.rows, page_rows, b.pages))


@pytest.mark.parametrize("rows,lengths,pad,extra", [
    ([1, 8, 3], [10, 8, 300], 0, 0), ([33, 64, 1, 0, 31], [100, 64, 9, 4, 31], 6, 0), ([5, 5], [9, 70], 0, 2),
    ([200, 100], [333, 100], 0, 0), ([40] * 300, [64] * 300, 1, 0)])
def test_slots_of_trees(ctx, rows, lengths, pad, extra):
    """Positions by depth; masks wider than the trees, rows of no mask, bits past the rows."""
    rng = np.random.default_rng(6)
    b = Batch(rng, rows, lengths, 16, pad)
    masks = [m for n in rows for m in tree(rng, n, 0.1)] + [5] * pad
    count = (max(rows) + 31) // 32 + extra
    masks = [m | 1 << 32 * count - 1 if i % 7 == 0 and rows[0] < 32 * count else m for i, m in enumerate(masks)]
    got = launch_slots(ctx, rows, lengths, b.table, b.rows, 16, b.pages, words(masks, count))
    assert np.array_equal(got, slot_maps(rows, lengths, b.table, b.rows, 16, b.pages, masks))


def test_slots_without_a_place(ctx):
    """Rows before position 0, past the table or the rows, entries that are no page, counts
    below 0, a mask narrower than the rows."""
    rng = np.random.default_rng(7)
    counts, lengths = [6, -4, 3, 9, 50], [4, 3, 300, 30, 60]
    table = rng.permutation(50)[:25].reshape(5, 5).astype(np.int32)
    table[3, 1], table[3, 0], table[4, 2] = -1, 50, 2 ** 31 - 1
    rows = 40  # the last sequence's rows are cut off
    got = launch_slots(ctx, counts, lengths, table, rows, 8, 50)
    assert np.array_equal(got, slot_maps(counts, lengths, table, rows, 8, 50))
    masks = [int(x) for x in rng.integers(0, 2 ** 32, rows)]
    got = launch_slots(ctx, counts, lengths, table, rows, 8, 50, words(masks, 1))
    assert np.array_equal(got, slot_maps(counts, lengths, table, rows, 8, 50, masks))


def random_paths(rng, rows, columns):
    path, counts = np.full((len(rows), max(columns, 1)), -1, np.int32), []
    for s, n in enumerate(rows):
        count = int(rng.integers(0, min(n, columns) + 1))
        path[s, :count] = np.sort(rng.permutation(n)[:count])
        counts.append(count)
    return path, np.array(counts, np.int32)


def check_keep(ctx, b, layers, heads, width, path, counts, offset=0):
    shape = (layers, b.pages, 2, heads, b.page_rows, width)
    size = int(np.prod(shape))
    caches = np.arange(size, dtype=np.uint32).astype(np.uint16)  # bits of any kind, NaN among them
    raw = np.concatenate([np.full(offset, 9, np.uint16), caches, np.full(8, 9, np.uint16)])
    out = ctx.upload(raw)
    bufs = [ctx.upload(a) for a in (b.table, b.offsets, b.lengths, path, counts)]
    ctx.launch("ipu_stack_keep_pages_f16", out.ptr + 2 * offset, bufs,
               [b.sequences(), b.rows, layers, heads, width, b.pages, b.page_rows, b.columns, path.shape[1]])
    got = out.download(np.uint16)
    want = keep_rows(caches.reshape(shape), b, path, counts)
    assert np.array_equal(got[offset:offset + size], want.ravel())
    assert np.all(got[:offset] == 9) and np.all(got[offset + size:] == 9)
    for x in bufs + [out]:
        x.free()


@pytest.mark.parametrize("rows,lengths,layers,heads,width,page_rows,columns", [
    ([1], [1], 1, 1, 1, 1, 1), ([8] * 8, [8 + 9 * i for i in range(8)], 1, 8, 128, 16, 4),
    ([64, 1, 0, 33], [100, 1, 40, 33], 3, 2, 72, 8, 12), ([200, 65], [300, 65], 2, 1, 64, 64, 200),
    ([5, 9], [20, 9], 4, 3, 65, 4, 5), ([16] * 40, [50] * 40, 2, 16, 256, 16, 16),
    ([12, 30], [40, 50], 5, 2, 6, 2, 7), ([9], [12], 2, 3, 12, 16, 9), ([7], [9], 300, 1, 8, 4, 6)])
def test_keep(ctx, rows, lengths, layers, heads, width, page_rows, columns):
    rng = np.random.default_rng(len(rows) + width)
    b = Batch(rng, rows, lengths, page_rows, 1)
    for _ in range(2):
        check_keep(ctx, b, layers, heads, width, *random_paths(rng, rows, columns))


@pytest.mark.parametrize("offset,width", [(1, 64), (2, 64), (4, 64), (8, 64), (3, 20)])
def test_keep_of_any_alignment(ctx, offset, width):
    rng = np.random.default_rng(offset)
    b = Batch(rng, [20, 7], [33, 70], 8)
    check_keep(ctx, b, 2, 3, width, *random_paths(rng, [20, 7], 9), offset=offset)


def test_keep_of_paths_that_end_early(ctx):
    """The same row twice, rows out of order, no rows of the sequence, counts past the
    path, more rows than keys, and pages that are none."""
    rng = np.random.default_rng(8)
    b = Batch(rng, [9, 9, 9, 9, 9, 100, 9], [30, 30, 30, 30, 5, 120, 40], 4, 2)
    path = np.full((7, 80), -1, np.int32)
    path[0, :4] = [2, 2, 5, 6]
    path[1, :4] = [1, 4, 3, 8]
    path[2, :4] = [-1, 3, 4, 5]
    path[3, :4] = [3, 8, 9, 10]
    path[4, :4] = [1, 5, 6, 8]        # positions before 0
    path[5, :80] = np.arange(80) + 20  # two groups
    path[6, :3] = [2, 6, 8]
    b.table[6, 8] = -1
    b.table[0, 6] = b.pages
    check_keep(ctx, b, 2, 2, 16, path, np.array([4, 4, 4, 100, 4, 80, 3], np.int32))
    check_keep(ctx, b, 1, 1, 8, path, np.array([2 ** 31 - 1, -5, 0, -2 ** 31, 2, 65, 1], np.int32))


def test_recorded(ipus, ctx):
    """Tables and maps of a step recorded once: lengths, counts and states that change
    between the replays, two states in turn."""
    pages, page_rows, columns, count, rows = 300, 8, 20, 6, 64
    rng = np.random.default_rng(9)
    free, held = [int(p) for p in rng.permutation(pages)], [[] for _ in range(count)]
    size = 2 + pages + count * (1 + columns)
    states = [ctx.upload(table_state(free, held, pages, columns)), ctx.alloc(4 * size)]
    source, lengths, counts = (ctx.upload(np.arange(count, dtype=np.int32)) for _ in range(3))
    mask = ctx.upload(np.zeros(1, np.uint32))
    maps = [ctx.alloc(4 * (count + 1 + 2 * rows)) for _ in range(2)]
    recording = Recording(ipus, ctx)
    with recording:
        for i in (0, 1):
            ctx.launch("ipu_stack_page_tables", states[1 - i], [states[i], source, lengths],
                       [count, count, pages, page_rows, columns])
            ctx.launch("ipu_stack_slot_maps", maps[i],
                       [counts, lengths, states[1 - i].ptr + 4 * (2 + pages + count), mask],
                       [count, rows, pages, page_rows, columns, 0])
    length = np.zeros(count, np.int64)
    for step in range(5):
        n = rng.integers(0, 11, count)
        length = np.where(rng.random(count) < 0.2, n, length + n)
        src = np.where(length == n, -1, np.arange(count))
        for buf, a in ((source, src), (lengths, length), (counts, n)):
            ctx.write(buf, a.astype(np.int32))
        ctx.sync()
        recording.replay()
        recording.sync()
        for i in (0, 1):  # the second time nothing changes but the new ones' pages
            free, held, missing = fit_tables(free, held, list(src), list(length), page_rows, columns)
            state = table_state(free, held, pages, columns, missing)
            if i == 1:
                assert np.array_equal(states[0].download(np.int32), state)
            table = state[2 + pages + count:].reshape(count, columns)
            assert np.array_equal(maps[i].download(np.int32), slot_maps(n, length, table, rows, page_rows, pages))
    recording.close()
    for b in states + [source, lengths, counts, mask] + maps:
        b.free()
