"""Operators of a drafted step at calls that the other tests leave out: layouts, sizes at
which a kernel takes another of its ways, steps that are cut off."""
from __future__ import annotations

import numpy as np
import pytest

from decoder_forms import Batch
from step_forms import fit_tables, slot_maps, table_state, tree, within, words
from test_gpu_logits import TYPES, Step
from test_gpu_page_maps import launch_slots, launch_tables
from test_gpu_tree_attention import check as check_trees, masks_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", sorted(TYPES))
@pytest.mark.parametrize("rows", [[1] * 30, [9, 11] * 40])
def test_logits_between_the_rows_of_their_input(ctx, kind, rows):
    """Input and output rows in turn in one buffer: no two of them meet."""
    dtype, columns = TYPES[kind], 28673
    step = Step(np.random.default_rng(1), rows, columns, 100, 10)
    x = np.full((step.rows, 2, columns), 5.0, dtype)
    x[:, 0] = (3 * np.random.default_rng(2).standard_normal((step.rows, columns))).astype(dtype)
    buffer = ctx.upload(x)
    bufs, scalars = step.upload(ctx)
    ctx.launch("ipu_stack_adjust_logits_" + kind, buffer.ptr + columns * x.itemsize, [buffer] + bufs,
               [len(step.n), step.rows, columns, 2 * columns, 2 * columns] + scalars)
    got = buffer.download(dtype).reshape(x.shape)
    want, bound, inside = step.exact(x[:, 0])
    assert np.all(inside) and np.array_equal(got[:, 0], x[:, 0]) and np.all(within(got[:, 1], want, bound, dtype))
    for b in bufs + [buffer]:
        b.free()


@pytest.mark.parametrize("kind", sorted(TYPES))
def test_biases_before_penalties(ctx, kind):
    """A launch with the biases alone, then one with the penalties alone, in place."""
    dtype, columns = TYPES[kind], 5001
    step = Step(np.random.default_rng(5), [3, 1, 6], columns, 200, 400, allowed=False)
    x = (3 * np.random.default_rng(6).standard_normal((step.rows, columns))).astype(dtype)
    penalties, logits = step.penalties, ctx.upload(x)
    for penal in (False, True):
        step.penalties = penalties if penal else np.tile(np.array([1, 0, 0], np.float32), (3, 1))
        if penal:
            step.bias_offsets = np.zeros(4, np.int32)
            step.bias_tokens, step.bias_values = step.bias_tokens[:0], step.bias_values[:0]
        bufs, scalars = step.upload(ctx)
        assert (scalars[2] == 0) == penal
        ctx.launch("ipu_stack_adjust_logits_" + kind, logits, [logits] + bufs,
                   [3, step.rows, columns, columns, columns] + scalars)
        got = logits.download(dtype).reshape(x.shape)
        want, bound, inside = step.exact(x)
        assert np.all(inside) and np.all(within(got, want, bound, dtype)) and np.any(got != x)
        x = got  # what the next launch begins with
        for b in bufs:
            b.free()
    logits.free()


@pytest.mark.parametrize("trees", [False, True])
def test_slots_of_a_step_that_is_cut_off(ctx, trees):
    """Fewer rows than the counts' sum: with lengths less the rows cut off, the rows that are
    left stand where they stand in the whole step."""
    rng = np.random.default_rng(3)
    counts, lengths = [40, 3, 0, 70, 5], [90, 60, 7, 70, 200]
    b = Batch(rng, counts, lengths, 16)
    masks = [m for n in counts for m in tree(rng, n, 0.1)]
    count, sequences = 3 if trees else 0, len(counts)
    whole = launch_slots(ctx, counts, lengths, b.table, b.rows, 16, b.pages, words(masks, count))
    for rows in (0, 1, 39, 40, 42, 43, 44, 112, 113, 117):
        left = [int(min(rows, end) - min(rows, end - n)) for n, end in zip(counts, np.cumsum(counts))]
        shorter = [length - n + m for length, n, m in zip(lengths, counts, left)]
        got = launch_slots(ctx, counts, shorter, b.table, rows, 16, b.pages, words(masks[:rows], count))
        assert list(got[:sequences + 1]) == [0] + list(np.cumsum(left))
        for part in (0, 1):  # positions, slots
            here, there = sequences + 1 + part * rows, sequences + 1 + part * b.rows
            assert np.array_equal(got[here:here + rows], whole[there:there + rows])
        assert np.array_equal(got, slot_maps(counts, shorter, b.table, rows, 16, b.pages, masks if trees else None))


@pytest.mark.parametrize("sequences,columns,page_rows,pages", [(300, 1200, 4, 400000), (4096, 70, 16, 290000), (2, 200000, 1, 270000)])
def test_tables_of_more_words_than_threads(ctx, sequences, columns, page_rows, pages):
    """More entries and more free pages than the largest grid has threads (2^18): requests
    begin, grow, shrink, end and change places."""
    assert sequences * columns > 1 << 18 and pages > 1 << 18
    rng = np.random.default_rng(columns)
    free, rows = [int(p) for p in rng.permutation(pages)], []
    state = table_state(free, rows, pages, columns)
    most = columns * page_rows
    for step in range(6):
        previous = len(rows)
        count = sequences if step < 2 else int(rng.integers(max(1, sequences // 2), sequences + 1))
        source = [int(p) for p in rng.permutation(max(previous, count))[:count]]
        # Some begin, and one names a row that another goes on with.
        source = [p if p < previous and rng.random() < 0.8 else int(rng.integers(-2, previous + 2)) for p in source]
        # Few pages at first, so that most stay free, then as many as there are.
        lengths = [int(rng.integers(0, most // (8 if step % 3 == 0 else 1) + 1)) for _ in range(count)]
        got = launch_tables(ctx, state, source, lengths, previous, pages, page_rows, columns)
        free, rows, missing = fit_tables(free, rows, source, lengths, page_rows, columns)
        state = table_state(free, rows, pages, columns, missing)
        assert np.array_equal(got, state), step


@pytest.mark.parametrize("rows,lengths,heads,width", [
    ([2] * 130, [40 + 9 * (37 * i % 130) for i in range(130)], 16, 128),      # one tile of 16 queries
    ([20, 3] * 65, [100 + 18 * (37 * i % 130) for i in range(130)], 16, 64),  # two, tiles of 64 keys
    ([3] * 150, [20 + 7 * (41 * i % 150) for i in range(150)], 14, 192)])
def test_trees_cut_anywhere(ipus, ctx, rows, lengths, heads, width):
    """More segments (sequence and key head) than workgroups, the longest of more than 32 tiles of
    keys: all of their tiles are one line, cut into equal chunks wherever the cuts fall, through
    the tiles that hold a tree's own keys too."""
    rng = np.random.default_rng(width)
    b = Batch(rng, rows, lengths, 16, 1)
    check_trees(ipus, ctx, b, masks_of(rng, b, 0.3), heads, heads, width)


def test_long_trees_cut_anywhere(ipus, ctx):
    """Chunks shorter than a segment, so that its parts are those of three and more workgroups: 200
    tiles of keys and more for each.  The sequences read the same pages, in other orders."""
    rng = np.random.default_rng(4)
    lengths = [34000 + 2001 * (7 * i % 10) for i in range(10)]
    b = Batch(rng, [3] * 10, [max(lengths)] + [3] * 9, 64)
    pages = b.table[0, :-(-max(lengths) // 64)].copy()
    for s, length in enumerate(lengths):
        b.table[s, :len(pages)] = rng.permutation(pages)
    b.k, b.lengths = lengths, np.array(lengths, np.int32)
    assert sum(-(-x // 64) for x in lengths) * 16 >= 200 * 512
    check_trees(ipus, ctx, b, masks_of(rng, b, 0.3), 16, 16, 32)
