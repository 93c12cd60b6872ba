"""Frequencies of the rotary kernels, and what the decoder operators refuse
before any device work (CPU)."""
from __future__ import annotations

import math
import struct

import numpy as np
import pytest


def bits(x):
    return struct.unpack("<I", struct.pack("<f", x))[0]


@pytest.mark.parametrize("r", [2, 6, 64, 72, 128])
@pytest.mark.parametrize("scaling", ["PLAIN", "LINEAR", "BASE", "BANDED"])
def test_frequencies(ipus, r, scaling):
    if scaling == "BASE" and r == 2:
        pytest.skip("one frequency has no base")
    base, factor, trained = 10000.0, 8.0, 4096.0
    got, magnitude = ipus.rotary_frequencies(r, base, getattr(ipus, "ROTARY_" + scaling), factor, trained)
    want = []
    for i in range(r // 2):
        b = base * factor ** (r / (r - 2)) if scaling == "BASE" else base
        f = b ** (-2.0 * i / r)
        if scaling == "LINEAR":
            f /= factor
        if scaling == "BANDED":
            keep = min(max((trained * f / (2 * math.pi) - 1.0) / 31.0, 0.0), 1.0)
            f = f * keep + f / factor * (1.0 - keep)
        want.append(f)
    # 64-bit powers, one rounding to fp32.
    assert np.all(np.abs(got - np.array(want)) <= np.array(want) * (2.0 ** -24 + 2.0 ** -40))
    expect = 0.1 * math.log(factor) + 1.0 if scaling == "BANDED" else 1.0
    assert abs(magnitude - expect) <= expect * 2.0 ** -23
    if scaling == "BASE":  # the fastest stays, the slowest is divided by the factor
        assert got[0] == 1.0
        plain, _ = ipus.rotary_frequencies(r)
        assert abs(got[-1] * factor / plain[-1] - 1.0) < 1e-6


@pytest.mark.parametrize("arguments", [
    dict(rotary_width=0), dict(rotary_width=7), dict(rotary_width=8, base=0.0),
    dict(rotary_width=8, base=math.inf), dict(rotary_width=8, scaling=4), dict(rotary_width=8, scaling=-1),
    dict(rotary_width=8, scaling=1, factor=0.0), dict(rotary_width=8, scaling=1, factor=math.nan),
    dict(rotary_width=2, scaling=2, factor=2.0), dict(rotary_width=8, scaling=3, factor=2.0),
    dict(rotary_width=8, scaling=3, factor=2.0, trained_rows=64.0, slow_turns=2.0, fast_turns=2.0),
])
def test_frequencies_refuse(ipus, arguments):
    with pytest.raises(ipus.IpusError) as e:
        ipus.rotary_frequencies(**arguments)
    assert e.value.status == ipus.ERROR_INVALID_ARGUMENT


@pytest.mark.parametrize("rotary_width", [-2, -1, -(2 ** 32) + 8, 2 ** 32, 2 ** 32 + 8])
def test_frequencies_refuse_widths_past_32_bits(ipus, rotary_width):
    """They would wrap to a width that the array was not made for."""
    with pytest.raises(ipus.IpusError) as e:
        ipus.rotary_frequencies(rotary_width)
    assert e.value.status == ipus.ERROR_INVALID_ARGUMENT and str(rotary_width) in e.value.message


@pytest.mark.parametrize("arguments", [
    dict(rotary_width=64, base=1e-300), dict(rotary_width=64, scaling=1, factor=1e-300),
    dict(rotary_width=4, base=1e200, scaling=2, factor=1e200), dict(rotary_width=4, base=1e-200, scaling=2, factor=1e-200),
    dict(rotary_width=64, scaling=3, factor=1e-300, trained_rows=4096.0),
])
def test_frequencies_that_are_not_finite_are_refused(ipus, arguments):
    """Each turns some pair by an angle that is not a number."""
    with pytest.raises(ipus.IpusError) as e:
        ipus.rotary_frequencies(**arguments)
    assert e.value.status == ipus.ERROR_INVALID_ARGUMENT


def test_frequencies_null(ipus):
    assert ipus._lib().ipus_rotary_frequencies(None, None, 8, 10000.0, 0, 1.0, 0.0, 0.0, 0.0) == \
        ipus.ERROR_INVALID_ARGUMENT


GOOD = {
    "ipu_stack_rotary_f16": (3, [4, 2, 64, 32, 0, 128, 64, 128, 64, 0]),
    "ipu_stack_norm_rotary_f16": (5, [4, 2, 1, 64, 32, 1, 192, 192, bits(1e-6), 0]),
    "ipu_stack_append_pages_f16": (6, [2, 8, 2, 64, 128, 128, 64, 0, 0, 10, 16, 4]),
    "ipu_stack_attention_pages_f16": (5, [2, 8, 4, 8, 2, 64, 512, 10, 16, 4, 1, 0]),
    "ipu_stack_attention_shared_pages_f16": (5, [2, 8, 4, 8, 2, 64, 512, 10, 16, 4, 1, 0, 48]),
}
GOOD["ipu_stack_rotary_f32"] = GOOD["ipu_stack_rotary_f16"]
GOOD["ipu_stack_norm_rotary_f32"] = GOOD["ipu_stack_norm_rotary_f16"]

# symbol -> (scalar, value, status)
BAD = {
    "ipu_stack_rotary_f16": [
        ("width", 0, -1), ("width", 4096, -3), ("rotary_width", 31, -1), ("rotary_width", 66, -1),
        ("interleaved", 2, -1), ("output_row_stride", 127, -1), ("output_head_stride", 63, -1),
        ("output_row_stride", 0, -1), ("magnitude_bits", bits(math.inf), -1),
        ("magnitude_bits", bits(math.nan), -1), ("rows", 1 << 31, -1), ("heads", 1 << 31, -1)],
    "ipu_stack_norm_rotary_f16": [
        ("width", 0, -1), ("width", 2050, -3), ("rotary_width", 3, -1), ("interleaved", 2, -1),
        ("output_row_stride", 191, -1), ("epsilon_bits", bits(-1.0), -1),
        ("epsilon_bits", bits(math.nan), -1), ("magnitude_bits", bits(-math.inf), -1),
        ("rows", 1 << 31, -1), ("key_heads", 0xffffffff, -1)],
    "ipu_stack_append_pages_f16": [
        ("width", 0, -1), ("width", 2050, -3), ("rotary_width", 66, -1), ("rotary_width", 1, -1),
        ("interleaved", 2, -1), ("key_heads", 0, -1), ("key_heads", 40000, -1), ("page_rows", 0, -1),
        ("page_rows", 24, -1), ("page_rows", 1 << 17, -1), ("rows", 1 << 31, -1),
        ("magnitude_bits", bits(math.nan), -1)],
    "ipu_stack_attention_pages_f16": [
        ("query_heads", 0, -1), ("query_heads", 7, -1), ("query_heads", 1 << 16, -1),
        ("key_heads", 0, -1), ("key_heads", 3, -1), ("width", 0, -1), ("width", 1025, -3),
        ("page_rows", 0, -1), ("page_rows", 48, -1), ("causal", 2, -1),
        ("scale_bits", bits(-1.0), -1), ("scale_bits", bits(math.inf), -1),
        ("scale_bits", bits(math.nan), -1), ("rows", 1 << 31, -1)],
}
BAD["ipu_stack_rotary_f32"] = BAD["ipu_stack_rotary_f16"]
BAD["ipu_stack_norm_rotary_f32"] = BAD["ipu_stack_norm_rotary_f16"]
BAD["ipu_stack_attention_shared_pages_f16"] = BAD["ipu_stack_attention_pages_f16"]


@pytest.mark.parametrize("symbol", sorted(GOOD))
def test_scalars(ipus, symbol):
    inputs, scalars = GOOD[symbol]
    names = ipus.kernel_abi(symbol).scalar_names
    assert len(names) == len(scalars)
    ipus.validate_kernel_run(symbol, inputs, scalars)
    for bad_inputs in (inputs - 1, inputs + 1):
        with pytest.raises(ipus.KernelAbiError) as e:
            ipus.validate_kernel_run(symbol, bad_inputs, scalars)
        assert e.value.status == ipus.ERROR_POINTER_ARITY
    with pytest.raises(ipus.IpusError):
        ipus.validate_kernel_run(symbol, inputs, scalars[:-1])
    for name, value, status in BAD[symbol]:
        changed = list(scalars)
        changed[names.index(name)] = value
        with pytest.raises(ipus.IpusError) as e:
            ipus.validate_kernel_run(symbol, inputs, changed)
        assert e.value.status == status, (name, value)


def test_head_major_outputs_are_accepted(ipus):
    """[heads][rows][width], and one row or head with any stride of that axis."""
    for scalars in ([4, 2, 64, 32, 0, 0, 0, 64, 256, 0], [1, 2, 64, 32, 0, 0, 0, 0, 64, 0],
                    [4, 1, 64, 32, 0, 0, 0, 64, 0, 0], [0, 2, 64, 32, 0, 0, 0, 0, 0, 0]):
        ipus.validate_kernel_run("ipu_stack_rotary_f16", 3, scalars)
    with pytest.raises(ipus.IpusError):
        ipus.validate_kernel_run("ipu_stack_rotary_f16", 3, [4, 2, 64, 32, 0, 0, 0, 64, 255, 0])


@pytest.mark.parametrize("symbol", ["ipu_stack_append_pages_f16", "ipu_stack_attention_pages_f16",
                                    "ipu_stack_attention_shared_pages_f16"])
def test_sequences_past_31_bits_are_refused(ipus, symbol):
    """Sequence numbers that steps of 64 in 32 bits would pass without end."""
    inputs, scalars = GOOD[symbol]
    for sequences, good in ((0x7fffffff, True), (0x80000000, False), (0xffffffff, False)):
        changed = [sequences] + scalars[1:]
        if good:
            ipus.validate_kernel_run(symbol, inputs, changed)
            continue
        with pytest.raises(ipus.IpusError) as e:
            ipus.validate_kernel_run(symbol, inputs, changed)
        assert e.value.status == ipus.ERROR_INVALID_ARGUMENT


@pytest.mark.parametrize("symbol", ["ipu_stack_attention_pages_f16", "ipu_stack_attention_shared_pages_f16"])
def test_scales_past_fp32_are_refused(ipus, symbol):
    """65504^2 * width * scale * log2(e), the largest score, is a finite fp32 value."""
    inputs, scalars = GOOD[symbol]
    names = ipus.kernel_abi(symbol).scalar_names
    for width in (8, 64, 1024):
        largest = np.finfo(np.float32).max / (65504.0 ** 2 * width * math.log2(math.e))
        for scale, good in ((2.0 ** -149, True), (largest * 0.999, True), (largest * 1.001, False), (3e38, False)):
            changed = list(scalars)
            changed[names.index("width")], changed[names.index("scale_bits")] = width, bits(scale)
            if good:
                ipus.validate_kernel_run(symbol, inputs, changed)
                continue
            with pytest.raises(ipus.IpusError) as e:
                ipus.validate_kernel_run(symbol, inputs, changed)
            assert e.value.status == ipus.ERROR_INVALID_ARGUMENT
