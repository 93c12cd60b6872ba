"""Penalties, biases and masks on logits, against float64."""
from __future__ import annotations

import numpy as np
import pytest

from step_forms import adjust_logits, tree, within, words
from test_gpu_caller_capture import Recording

pytestmark = pytest.mark.gpu

TYPES = {"f16": np.float16, "f32": np.float32}


class Step:
    """A step's rows and everything that changes their logits, at random."""

    def __init__(self, rng, rows, columns, history=0, biases=0, masks=True, allowed=True, pad=0, twice=False):
        self.n, self.columns = list(rows), columns
        self.offsets = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
        self.rows, count = int(self.offsets[-1]) + pad, len(rows)
        few = min(columns, 30)  # tokens repeat

        def tokens(shape):
            any_token, some = rng.integers(0, columns, shape), rng.integers(0, few, shape)
            return np.where(rng.random(shape) < 0.5, any_token, some).astype(np.int32)
        self.tokens = tokens(self.rows)
        self.masks = [m for n in rows for m in tree(rng, n, 0.1)] + [7] * pad if masks else None
        self.words = max(1, (max(rows + [0]) + 31) // 32) if masks else 0
        self.history = tokens((count, history))
        total = rng.integers(0, history + 1, count)
        self.counts = np.stack([(total * rng.random(count)).astype(np.int64), total], axis=1).astype(np.int32)
        self.penalties = np.stack([rng.uniform(0.8, 1.4, count), rng.uniform(-0.5, 1, count), rng.uniform(-0.5, 1, count)],
                                  axis=1).astype(np.float32)
        each = rng.integers(0, biases + 1, count) if biases else np.zeros(count, int)
        self.bias_offsets = np.concatenate([[0], np.cumsum(each)]).astype(np.int32)
        entries = int(self.bias_offsets[-1])
        if twice:  # the last entry of a token holds
            self.bias_tokens = rng.integers(0, few, entries).astype(np.int32)
        else:
            self.bias_tokens = (np.concatenate([rng.permutation(columns)[:e] for e in each] + [np.zeros(0)])).astype(np.int32)
        self.bias_values = rng.uniform(-9, 9, entries).astype(np.float32)
        self.allowed = None
        if allowed:
            share = rng.choice([0.0, 0.02, 0.5, 1.0], self.rows)
            self.allowed = rng.random((self.rows, columns)) < share[:, None]

    def allowed_words(self, extra=0):
        if self.allowed is None:
            return np.zeros((1, 0), np.uint32)
        count = (self.columns + 31) // 32 + extra
        padded = np.ones((self.rows, 32 * count), bool)  # bits past the columns are not read
        padded[:, :self.columns] = self.allowed
        return np.packbits(padded, axis=1, bitorder="little").view(np.uint32)

    def upload(self, ctx, extra=0):
        """The inputs behind the logits, and the scalars behind the strides."""
        mask = words(self.masks, self.words) if self.masks is not None else np.zeros(1, np.uint32)
        biases = np.stack([self.bias_tokens, self.bias_values.view(np.int32)], axis=1)
        allowed = self.allowed_words(extra)
        arrays = [self.offsets, self.tokens, mask, self.history, self.counts, self.penalties, self.bias_offsets,
                  biases, allowed]
        bufs = [ctx.upload(np.ascontiguousarray(a) if a.size else np.zeros(1, np.int32)) for a in arrays]
        return bufs, [self.words, self.history.shape[1], len(biases), allowed.shape[1]]

    def exact(self, x):
        return adjust_logits(x.astype(np.float64), self.offsets, self.tokens, self.masks, self.history, self.counts,
                             self.penalties, self.bias_offsets, (self.bias_tokens, self.bias_values), self.allowed)


def check(ctx, step, kind, strides=None, extra=0, offset=0, in_place=False, change=None, seed=1):
    dtype = TYPES[kind]
    rng = np.random.default_rng(seed)
    columns = step.columns
    a, b = strides or (columns, columns)
    x = np.full((step.rows, a), 9.0, dtype)
    x[:, :columns] = (3 * rng.standard_normal((step.rows, columns))).astype(dtype)
    if change:
        change(x)
    front = np.full(offset, 5.0, dtype)
    source = ctx.upload(np.concatenate([front, x.ravel()]))
    blank = np.concatenate([front, np.full(step.rows * b + 8, 5.0, dtype)])
    out = source if in_place else ctx.upload(blank)
    bufs, scalars = step.upload(ctx, extra)
    size = x.itemsize
    ctx.launch("ipu_stack_adjust_logits_" + kind, out.ptr + size * offset, [source.ptr + size * offset] + bufs,
               [len(step.n), step.rows, columns, a, b] + scalars)
    raw = out.download(dtype)
    want, bound, inside = step.exact(x[:, :columns])
    got = raw[offset:offset + step.rows * b].reshape(step.rows, b)
    assert np.all(within(got[:, :columns], want, bound, dtype)[inside])
    before = x if in_place else blank[offset:offset + step.rows * b].reshape(step.rows, b)
    assert np.array_equal(got[~inside], before[~inside], equal_nan=True) and np.array_equal(got[:, columns:], before[:, columns:])
    assert np.all(raw[:offset] == 5.0) and (in_place or np.all(raw[offset + step.rows * b:] == 5.0))
    for buf in bufs + ([source] if in_place else [source, out]):
        buf.free()
    return got[:, :columns]


@pytest.mark.parametrize("kind", sorted(TYPES))
@pytest.mark.parametrize("rows,columns,history,biases,masks,allowed,pad", [
    ([1], 1, 0, 0, False, False, 0), ([1] * 3, 7, 5, 2, False, True, 0), ([1] * 40, 1000, 300, 20, False, False, 2),
    ([4, 0, 9, 1], 5003, 1000, 50, True, True, 3), ([2, 3], 4096, 0, 0, True, False, 0), ([2, 3], 4097, 64, 0, False, False, 1),
    ([33, 70], 999, 100, 300, True, True, 0), ([16] * 8, 32000, 2000, 100, True, True, 0), ([1, 2], 131072, 9000, 400, True, True, 0),
    ([3] * 100, 257, 50, 9, False, True, 4), ([2], 70001, 70000, 0, False, True, 0), ([5, 1], 12289, 20, 0, True, True, 0),
    ([64] * 5, 8192, 500, 30, True, False, 0), ([200], 300, 40, 10, True, True, 0)])
def test_logits(ctx, kind, rows, columns, history, biases, masks, allowed, pad):
    rng = np.random.default_rng(columns)
    check(ctx, Step(rng, rows, columns, history, biases, masks, allowed, pad), kind)


# Enough rows for several per workgroup: of few and of many sequences, some without rows, of one
# of more rows than a workgroup has threads; with lists and without.
@pytest.mark.parametrize("kind,rows,columns,history,biases,masks,allowed", [
    ("f16", [64, 0, 70, 100, 3] * 3, 30000, 2000, 200, True, True), ("f32", [64, 70, 100, 3] * 3, 30001, 2000, 0, True, False),
    ("f32", [9, 0, 11] * 33, 28673, 300, 40, True, True), ("f16", [9, 8, 1] * 40, 28680, 0, 0, False, False),
    ("f32", [700, 3], 28700, 100, 20, False, True), ("f16", [650, 3], 28700, 5000, 100, True, True),
    ("f16", [33] * 250, 4100, 20, 3, True, False), ("f32", [33] * 125, 4097, 0, 300, True, True),
    ("f16", [40] * 52, 12288, 12000, 3000, True, False)])
def test_several_rows_per_workgroup(ctx, kind, rows, columns, history, biases, masks, allowed):
    rng = np.random.default_rng(columns)
    step = Step(rng, rows, columns, history, biases, masks, allowed, 2)
    for s in range(0, len(rows), 5):
        step.penalties[s] = [1.0, 0.0, 0.0]  # none
    check(ctx, step, kind)


@pytest.mark.parametrize("kind", sorted(TYPES))
def test_several_rows_in_place_of_any_content(ctx, kind):
    """As below, in place, with strides, and logits that are not finite."""
    rng = np.random.default_rng(27)
    step = Step(rng, [90, 7, 60], 60001, 60, 50, True, True, twice=True)
    step.history[:, ::7] = [[-1], [60001], [2 ** 31 - 1]]
    step.tokens[::5] = -2 ** 31
    step.bias_tokens[::4] = 60001
    step.counts[:] = [[5, 90], [-1, 60], [2 ** 31 - 1, 30]]
    step.words = 2
    step.masks = [m & (1 << 64) - 1 for m in step.masks]
    step.allowed[3] = False

    def change(x):
        x[:, 5], x[:, 6], x[:, 40], x[:, 41] = np.nan, np.inf, -np.inf, np.finfo(x.dtype).min
    check(ctx, step, kind, strides=(60005, 60005), offset=1, in_place=True, change=change)


@pytest.mark.parametrize("kind", sorted(TYPES))
@pytest.mark.parametrize("strides,extra,offset,in_place", [
    ((1001, 1001), 0, 0, True), ((1008, 1001), 3, 0, False), ((1003, 1020), 0, 1, False), ((1024, 1024), 0, 3, True),
    ((1005, 2000), 1, 8, False)])
def test_strides_and_alignment(ctx, kind, strides, extra, offset, in_place):
    rng = np.random.default_rng(21)
    check(ctx, Step(rng, [3, 1, 5], 1001, 100, 20, True, True, 2), kind, strides, extra, offset, in_place)


@pytest.mark.parametrize("kind", sorted(TYPES))
def test_the_last_bias_of_a_token_holds(ctx, kind):
    rng = np.random.default_rng(22)
    check(ctx, Step(rng, [2, 3, 1], 500, 40, 200, True, False, twice=True), kind)


@pytest.mark.parametrize("kind", sorted(TYPES))
def test_non_finite_logits(ctx, kind):
    """NaN and infinities stay as they are, but where the mask forbids the token; a type's
    lowest value, and a row that allows nothing."""
    rng = np.random.default_rng(23)
    step = Step(rng, [2, 4], 600, 50, 10, True, True)
    step.allowed[0], step.allowed[1] = False, True

    def change(x):
        x[:, 5], x[:, 6], x[:, 40], x[:, 41] = np.nan, np.inf, -np.inf, np.finfo(x.dtype).min
        x[1, :20] = np.nan
    got = check(ctx, step, kind, change=change)
    assert np.all(np.isneginf(got[0]))


@pytest.mark.parametrize("kind", sorted(TYPES))
def test_tokens_and_lists_of_any_content(ctx, kind):
    """Tokens outside the vocabulary count for nothing; counts and offsets past their arrays
    are cut off; masks narrower than the rows."""
    rng = np.random.default_rng(24)
    step = Step(rng, [40, 3], 700, 60, 12, True, False)
    step.history[:, ::7] = [[-1], [700]]
    step.tokens[::5] = 2 ** 31 - 1
    step.tokens[1::9] = -2 ** 31
    step.bias_tokens[::4] = -5
    step.counts[0] = [2 ** 31 - 1, 2 ** 31 - 1]
    step.counts[1] = [-7, -7]
    step.words = 1
    step.masks = [m & 0xffffffff for m in step.masks]
    check(ctx, step, kind)
    step.counts[0] = [90, 30]
    step.counts[1] = [-7, 100]
    check(ctx, step, kind)


def test_many_rows_and_long_histories(ctx):
    """Rows of one sequence that share a long history, with paths of their own; uses beyond
    2^16 of one token."""
    rng = np.random.default_rng(25)
    step = Step(rng, [64, 20], 20000, 140000, 50, True, True)
    step.history[0, :] = np.where(rng.random(140000) < 0.7, 11, step.history[0])
    step.counts[:] = [[100, 140000], [70000, 139999]]
    step.penalties[0] = [1.1, 1e-4, 0.5]
    check(ctx, step, "f32")
    check(ctx, step, "f16")


def test_recorded(ipus, ctx):
    """One recorded launch as rows, histories and masks change between the replays."""
    columns, rows = 3001, 12
    rng = np.random.default_rng(26)
    steps = [Step(np.random.default_rng(t), n, columns, 80, 0, True, True, rows - sum(n)) for t, n in
             enumerate(([4, 8, 0], [1, 1, 1], [0, 0, 12], [12, 0, 0], [3, 3, 3]))]
    for s in steps:
        s.words = 1
    first, scalars = steps[0].upload(ctx)
    x = rng.standard_normal((rows, columns)).astype(np.float32)
    source, out = ctx.upload(x), ctx.alloc(x.nbytes)
    recording = Recording(ipus, ctx)
    with recording:
        ctx.launch("ipu_stack_adjust_logits_f32", out, [source] + first, [3, rows, columns, columns, columns] + scalars)
    for step in steps:
        for buf, a in ((first[0], step.offsets), (first[1], step.tokens), (first[2], words(step.masks, 1)),
                       (first[3], step.history), (first[4], step.counts), (first[5], step.penalties),
                       (first[8], step.allowed_words()), (out, np.full_like(x, 5.0))):
            ctx.write(buf, a)
        ctx.sync()
        recording.replay()
        recording.sync()
        want, bound, inside = step.exact(x)
        got = out.download(np.float32).reshape(x.shape)
        assert np.all(within(got, want, bound, np.float32)[inside]) and np.all(got[~inside] == 5.0)
    recording.close()
    for buf in first + [source, out]:
        buf.free()
