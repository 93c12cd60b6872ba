"""Rotary positions and the norms of query and key heads with them, against
float64."""
from __future__ import annotations

import struct

import numpy as np
import pytest

from decoder_forms import norm_rotate, rotate, rounded

pytestmark = pytest.mark.gpu


def bits(x):
    return struct.unpack("<I", struct.pack("<f", x))[0]


def values(ipus, count, tensor, dtype, scale=1.0, seed=91):
    if dtype == np.float32:
        return ipus.synth_f32(count, seed, tensor, ipus.NORMAL, scale)
    return ipus.synth_f16(count, seed, tensor, ipus.NORMAL, scale).view(np.float16)


def symbol(base, dtype):
    return f"ipu_stack_{base}_{'f32' if dtype == np.float32 else 'f16'}"


SHAPES = [
    # rows, heads, width, rotary_width: one row; several rows per workgroup;
    # part of the head; widths whose chunks are 8, 4, 2 and 1 elements; more
    # units than a wave; an odd width's copied end; nothing turned.
    (1, 1, 2, 2), (1, 16, 128, 128), (5, 3, 128, 64), (4100, 2, 64, 64), (1100, 12, 72, 72),
    (33, 5, 72, 18), (7, 40, 80, 40), (9, 2, 96, 24), (3, 2, 2048, 2048), (2, 3, 1000, 500),
    (6, 4, 65, 10), (6, 3, 67, 6), (3, 300, 32, 32), (2050, 17, 32, 16), (3, 2, 24, 0),
    # Many rows per workgroup: up to 32, and the most that the rows leave.
    (40000, 1, 16, 8),
    (33000, 3, 32, 32),
    (2600, 5, 72, 72),
    (5003, 33, 64, 16),
]


@pytest.mark.parametrize("rows,heads,width,rotary_width", SHAPES)
@pytest.mark.parametrize("interleaved", [0, 1])
@pytest.mark.parametrize("dtype", [np.float16, np.float32])
def test_rotary(ipus, ctx, rows, heads, width, rotary_width, interleaved, dtype):
    x = values(ipus, rows * heads * width, 1, dtype)
    rng = np.random.default_rng(rows + width)
    positions = rng.integers(-5, 1 << 20, rows).astype(np.int32)
    f = ipus.rotary_frequencies(max(rotary_width, 2))[0]
    magnitude = 1.25
    bufs = [ctx.upload(a) for a in (x, positions, f)]
    out = ctx.upload(np.full(x.size + 16, 7.0, dtype))
    pitch = heads * width
    ctx.launch(symbol("rotary", dtype), out, bufs,
               [rows, heads, width, rotary_width, interleaved, pitch, width, pitch, width, bits(magnitude)])
    raw = out.download(dtype)
    got = raw[:x.size].reshape(rows, heads, width).astype(np.float64)
    want, bound = rotate(x.astype(np.float64).reshape(rows, heads, width), positions,
                         f[:rotary_width // 2], magnitude, rotary_width, interleaved)
    assert np.all(np.abs(got - want) <= rounded(want, bound, dtype))
    # What is not turned is copied, and nothing is written behind the rows.
    assert np.array_equal(raw[:x.size].reshape(rows, heads, width)[..., rotary_width:],
                          x.reshape(rows, heads, width)[..., rotary_width:])
    assert np.all(raw[x.size:] == 7.0)
    # In place: the same bits.
    ctx.launch(symbol("rotary", dtype), bufs[0], bufs,
               [rows, heads, width, rotary_width, interleaved, pitch, width, pitch, width, bits(magnitude)])
    assert np.array_equal(bufs[0].download(dtype), raw[:x.size])
    for b in bufs + [out]:
        b.free()


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("width,offset", [(128, 0), (128, 1), (64, 4), (80, 2)])
def test_rotary_strides(ipus, ctx, dtype, width, offset):
    """Token-major rows of a wider buffer into head-major streams, at an offset
    that leaves less alignment than the widths do."""
    rows, heads, pitch = 37, 6, 6 * width + 2 * offset + 8
    x = values(ipus, rows * pitch + 64, 2, dtype)
    positions = np.arange(100, 100 + rows, dtype=np.int32)
    f, _ = ipus.rotary_frequencies(width, scaling=ipus.ROTARY_LINEAR, factor=4.0)
    bufs = [ctx.upload(a) for a in (x, positions, f)]
    out = ctx.upload(np.full(heads * rows * width + 8, 7.0, dtype))
    size = x.itemsize
    ctx.launch(symbol("rotary", dtype), out, [bufs[0].ptr + offset * size, bufs[1], bufs[2]],
               [rows, heads, width, width, 0, pitch, width, width, rows * width, 0])
    raw = out.download(dtype)
    got = raw[:heads * rows * width].reshape(heads, rows, width).astype(np.float64)
    source = x[offset:offset + rows * pitch].reshape(rows, pitch)[:, :heads * width]
    want, bound = rotate(source.astype(np.float64).reshape(rows, heads, width), positions, f, 1.0, width, False)
    bound = rounded(want, bound, dtype)
    assert np.all(np.abs(got - want.transpose(1, 0, 2)) <= bound.transpose(1, 0, 2))
    assert np.all(raw[-8:] == 7.0)
    for b in bufs + [out]:
        b.free()


@pytest.mark.parametrize("rows,heads,width,rotary_width", SHAPES)
@pytest.mark.parametrize("interleaved", [0, 1])
@pytest.mark.parametrize("dtype", [np.float16, np.float32])
def test_norm_rotary(ipus, ctx, rows, heads, width, rotary_width, interleaved, dtype):
    """Query heads and key heads with weights of their own, value heads left
    out, into rows of another stride; then in place."""
    query, key, extra = heads - heads // 3, heads // 3, 2
    pitch, out_pitch = (heads + extra) * width, heads * width + 8
    x = values(ipus, rows * pitch, 3, dtype, 2.0)
    weights = [(1 + 0.2 * values(ipus, width, t, np.float32)).astype(dtype) for t in (4, 5)]
    positions = np.random.default_rng(rows).integers(0, 1 << 17, rows).astype(np.int32)
    f, _ = ipus.rotary_frequencies(max(rotary_width, 2))
    epsilon = 1e-5
    bufs = [ctx.upload(a) for a in (x, *weights, positions, f)]
    out = ctx.upload(np.full(rows * out_pitch, 7.0, dtype))
    scalars = [rows, query, key, width, rotary_width, interleaved, pitch, out_pitch, bits(epsilon), 0]
    ctx.launch(symbol("norm_rotary", dtype), out, bufs, scalars)
    raw = out.download(dtype).reshape(rows, out_pitch)
    full = x.reshape(rows, heads + extra, width)
    eps = float(np.float32(epsilon))
    per_head = np.stack([weights[0]] * query + [weights[1]] * key).astype(np.float64)
    want, bound = norm_rotate(full[:, :heads].astype(np.float64), per_head, eps, positions,
                              f[:rotary_width // 2], 1.0, rotary_width, interleaved)
    got = raw[:, :heads * width].reshape(rows, heads, width)
    assert np.all(np.abs(got.astype(np.float64) - want) <= rounded(want, bound, dtype))
    assert np.all(raw[:, heads * width:] == 7.0)
    scalars[7] = pitch
    ctx.launch(symbol("norm_rotary", dtype), bufs[0], bufs, scalars)
    after = bufs[0].download(dtype).reshape(rows, heads + extra, width)
    assert np.array_equal(after[:, :heads], got)
    assert np.array_equal(after[:, heads:], full[:, heads:])
    for b in bufs + [out]:
        b.free()


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("width", [128, 2048, 65])
@pytest.mark.parametrize("query,key", [(3, 0), (0, 3)])
def test_norm_rotary_of_one_group(ipus, ctx, dtype, width, query, key):
    """The weight of the group without heads is anything but null, at any address."""
    rows, heads = 5, 3
    x = values(ipus, rows * heads * width, 6, dtype)
    w = (1 + 0.2 * values(ipus, width, 7, np.float32)).astype(dtype)
    f, _ = ipus.rotary_frequencies(64)
    bufs = [ctx.upload(a) for a in (x, w, np.arange(rows, dtype=np.int32), f)]
    other = ctx.upload(np.full(2 * width + 8, np.nan, dtype))
    got = []
    for unused in (bufs[1].ptr, other.ptr + 1):
        out = ctx.alloc(x.nbytes)
        weights = [bufs[1], unused] if query else [unused, bufs[1]]
        ctx.launch(symbol("norm_rotary", dtype), out, [bufs[0], *weights, *bufs[2:]],
                   [rows, query, key, width, 64, 0, heads * width, heads * width, bits(1e-6), 0])
        got.append(out.download(np.uint8))
        out.free()
    assert np.array_equal(got[0], got[1])
    want, bound = norm_rotate(x.astype(np.float64).reshape(rows, heads, width), w.astype(np.float64),
                              float(np.float32(1e-6)), np.arange(rows), f, 1.0, 64, False)
    result = got[1].view(dtype).astype(np.float64).reshape(want.shape)
    assert np.all(np.abs(result - want) <= rounded(want, bound, dtype))
    for b in bufs + [other]:
        b.free()


@pytest.mark.parametrize("size", [1e37, 1e25, 2.0 ** 64, 1e-15, 1e-20, 1e-37])
@pytest.mark.parametrize("heads,width,rotary_width", [(5, 128, 128), (3, 65, 10), (2, 2048, 64), (40, 64, 0)])
@pytest.mark.parametrize("epsilon", [0.0, 1e-6])
def test_norm_of_fp32_values_whose_squares_are_not_fp32(ipus, ctx, size, heads, width, rotary_width, epsilon):
    rows = 4
    x = (values(ipus, rows * heads * width, 8, np.float32).astype(np.float64) * size).astype(np.float32)
    w = 1 + 0.2 * values(ipus, width, 9, np.float32)
    positions = np.arange(rows, dtype=np.int32) * 1000
    f, _ = ipus.rotary_frequencies(max(rotary_width, 2))
    bufs = [ctx.upload(a) for a in (x, w, w, positions, f)]
    out = ctx.alloc(x.nbytes)
    ctx.launch("ipu_stack_norm_rotary_f32", out, bufs,
               [rows, heads, 0, width, rotary_width, 0, heads * width, heads * width, bits(epsilon), 0])
    got = out.download(np.float32).astype(np.float64).reshape(rows, heads, width)
    want, bound = norm_rotate(x.astype(np.float64).reshape(rows, heads, width), w.astype(np.float64),
                              float(np.float32(epsilon)), positions, f[:rotary_width // 2], 1.0, rotary_width, False)
    assert np.all(np.abs(got - want) <= rounded(want, bound, np.float32))
    for b in bufs + [out]:
        b.free()


def test_norm_of_zeros_and_large_values(ipus, ctx):
    """A head of zeros stays zero, one at fp16's end does not overflow."""
    width = 128
    x = np.zeros((3, 1, width), np.float16)
    x[1] = 65504.0
    x[2, 0, 5] = 2.0 ** -24
    w = np.ones(width, np.float16)
    f, _ = ipus.rotary_frequencies(width)
    positions = np.zeros(3, np.int32)
    bufs = [ctx.upload(a) for a in (x, w, w, positions, f)]
    out = ctx.alloc(x.nbytes)
    ctx.launch("ipu_stack_norm_rotary_f16", out, bufs, [3, 1, 0, width, width, 0, width, width, bits(1e-6), 0])
    got = out.download(np.float16).reshape(3, width)
    assert np.all(got[0] == 0) and np.all(got[1] == 1)
    want = 2.0 ** -24 / np.sqrt(2.0 ** -48 / width + float(np.float32(1e-6)))
    assert abs(float(got[2, 5]) - want) <= want * 2.0 ** -10
    for b in bufs + [out]:
        b.free()


def test_rotary_refuses_in_place_with_other_strides(ipus, ctx):
    x = ctx.alloc(4 * 128 * 2)
    p = ctx.alloc(64)
    for scalars in ([2, 2, 64, 64, 0, 128, 64, 256, 64, 0], [2, 1, 64, 64, 0, 64, 64, 64, 128, 0]):
        with pytest.raises(ipus.IpusError) as e:
            ctx.launch("ipu_stack_rotary_f16", x, [x, p, p], scalars)
        assert e.value.status == ipus.ERROR_INVALID_ARGUMENT
    # fp32 elements and int32 positions at odd addresses
    for out, inputs in ((x.ptr + 2, [x, p, p]), (x, [x.ptr + 2, p, p]), (x, [x.ptr + 256, p.ptr + 2, p])):
        with pytest.raises(ipus.IpusError) as e:
            ctx.launch("ipu_stack_rotary_f32", out, inputs, [1, 1, 32, 32, 0, 32, 32, 32, 32, 0])
        assert e.value.status == ipus.ERROR_INVALID_ARGUMENT
    x.free()
    p.free()
