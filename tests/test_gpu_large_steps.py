"""The operators of a drafted step where offsets pass 32 bits: caches of pages of 4 GiB,
logits whose rows lie 2^31 elements apart, slots up to 2^31 - 1."""
from __future__ import annotations

import numpy as np
import pytest

from step_forms import within, words
from test_gpu_logits import Step
from test_gpu_pages import halves

pytestmark = pytest.mark.gpu


def view(ipus, ctx, base, element, count):
    return ipus.DeviceBuffer(ctx, base.ptr + 2 * element, 2 * count)


@pytest.mark.parametrize("heads", [63, 64])
def test_pages_of_4_gib(ipus, ctx, heads):
    """Drafts across a page's end in two layers; those accepted move together, and a chain
    attends as causal rows do."""
    width, page_rows, pages, layers = 256, 65536, 2, 2
    page = 2 * heads * page_rows * width
    assert (page * 2 >= 1 << 32) == (heads == 64)
    caches = ctx.alloc(layers * pages * page * 2)
    ctx.memset(caches, 0)
    n, length, table = 6, page_rows + 3, np.array([[1, 0]], np.int32)

    def place(layer, position, which, head):
        return ((layer * pages + int(table[0, position // page_rows])) * page
                + ((which * heads + head) * page_rows + position % page_rows) * width)
    rows = halves(ipus, (layers, n, 2, heads, width), 1)
    for layer in range(layers):
        for i in range(n):
            for which in (0, 1):
                for head in range(heads):
                    ctx.write(view(ipus, ctx, caches, place(layer, length - n + i, which, head), width),
                              rows[layer, i, which, head])
    bufs = [ctx.upload(a) for a in (table, np.array([0, n], np.int32), np.array([length], np.int32))]
    q = halves(ipus, (n, heads, width), 2)
    dq, mask = ctx.upload(q), ctx.upload(words([(2 << i) - 1 for i in range(n)], 1))
    outs = [ctx.alloc(q.nbytes) for _ in range(2)]
    scalars = [1, n, n, heads, heads, width, heads * width, pages, page_rows, 2, 1, 0]
    layer_bytes = pages * page * 2
    ctx.launch("ipu_stack_attention_pages_f16", outs[0], [dq, caches.ptr + layer_bytes] + bufs, scalars)
    ctx.launch("ipu_stack_attention_tree_pages_f16", outs[1], [dq, caches.ptr + layer_bytes] + bufs + [mask], scalars)
    first, second = (o.download(np.float16) for o in outs)
    assert np.all(np.isfinite(first.astype(np.float32))) and np.array_equal(first, second)
    path = ctx.upload(np.array([[1, 2, 5]], np.int32))
    counts = ctx.upload(np.array([3], np.int32))
    ctx.launch("ipu_stack_keep_pages_f16", caches, bufs + [path, counts], [1, n, layers, heads, width, pages, page_rows, 2, 3])
    ctx.sync()
    for layer in range(layers):
        for i, j in enumerate((1, 2, 5, 3, 4, 5)):
            for which in (0, 1):
                for head in (0, 1, heads - 1):
                    got = view(ipus, ctx, caches, place(layer, length - n + i, which, head), width).download(np.float16)
                    assert np.array_equal(got, rows[layer, j, which, head]), (layer, i, which, head)
        for head in (0, heads - 1):  # the row before
            assert not np.any(view(ipus, ctx, caches, place(layer, length - n - 1, 1, head), width).download(np.float16))
    for b in bufs + [dq, mask, path, counts, caches] + outs:
        b.free()


@pytest.mark.parametrize("rows", [[3], [2, 1]])
def test_logits_rows_2_31_elements_apart(ipus, ctx, rows):
    columns, stride = 9000, (1 << 31) + 8
    step = Step(np.random.default_rng(3), rows, columns, 50, 10, True, True)
    x = (3 * np.random.default_rng(4).standard_normal((3, columns))).astype(np.float16)
    data = ctx.alloc(2 * (2 * stride + columns))
    for r in range(3):
        ctx.write(view(ipus, ctx, data, r * stride, columns), x[r])
    bufs, scalars = step.upload(ctx)
    ctx.launch("ipu_stack_adjust_logits_f16", data, [data] + bufs, [len(rows), 3, columns, stride, stride] + scalars)
    ctx.sync()
    want, bound, _ = step.exact(x)
    got = np.stack([view(ipus, ctx, data, r * stride, columns).download(np.float16) for r in range(3)])
    assert np.all(within(got, want, bound, np.float16))
    for b in bufs + [data]:
        b.free()


def test_slots_up_to_2_31(ctx):
    table = np.array([[32767, 0, 16384]], np.int32)
    bufs = [ctx.upload(np.array(a, np.int32)) for a in ([4], [65537], table, [0])]
    out = ctx.alloc(4 * (2 + 8))
    ctx.launch("ipu_stack_slot_maps", out, bufs, [1, 4, 32768, 65536, 3, 0])
    got = out.download(np.int32)
    assert list(got) == [0, 4, 65533, 65534, 65535, 65536, 2 ** 31 - 3, 2 ** 31 - 2, 2 ** 31 - 1, 0]
    for b in bufs + [out]:
        b.free()
