"""Operators of a drafted step at calls that the other tests leave out: layouts, sizes at
which a kernel takes another of its ways, steps that are cut off."""
from __future__ import annotations

import numpy as np
import pytest

from step_forms import within
from test_gpu_logits import TYPES, Step

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
