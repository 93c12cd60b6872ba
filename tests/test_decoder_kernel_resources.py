"""Register, scratch, occupancy and LDS budgets of the decoder kernels, from the
compiler's resource remarks (no GPU needed)."""
from __future__ import annotations

import os
import re

import pytest

from test_kernel_resources import BUILD, matching, parse

SOURCES = ("k_rotary", "k_attention_pages", "k_attention_blocks")


@pytest.fixture(scope="module")
def kernels():
    out = {}
    for s in SOURCES:
        path = os.path.join(BUILD, f"{s}.resources")
        if not os.path.exists(path):
            pytest.skip("library not built by the package Makefile (no resource remarks)")
        got = parse(open(path).read())
        assert got, f"{s}.resources holds no kernel"
        out.update(got)
    return out


def test_no_scratch_memory(kernels):
    for name, f in kernels.items():
        assert int(f["ScratchSize [bytes/lane]"]) == 0, (name, f)
        assert f.get("Dynamic Stack", "False") == "False", name


def test_decode_kernels_fit_their_workgroups_per_cu(kernels):
    # Two workgroups per CU; one for more than 128 columns, and two tiles of queries at 128.
    for name, f in matching(kernels, "attention_pages_decode_kernel").items():
        columns, tiles = map(int, re.search(r"decode_kernelILi(\d+)ELi(\d+)E", name).groups())
        per_cu = 1 if columns > 128 or (columns == 128 and tiles == 2) else 2
        assert int(f["Occupancy [waves/SIMD]"]) >= per_cu, (name, f)
        assert per_cu * int(f["LDS Size [bytes/block]"]) <= 163840, (name, f)


def test_block_kernels_fit_two_workgroups_per_cu(kernels):
    for name, f in matching(kernels, "attention_blocks_kernel").items():
        assert int(f["Occupancy [waves/SIMD]"]) >= 2, (name, f)
        assert 2 * int(f["LDS Size [bytes/block]"]) <= 163840, (name, f)


def test_rotary_kernels_hide_their_loads(kernels):
    for fragment in ("rotary_kernel", "append_kernel"):
        for name, f in matching(kernels, fragment).items():
            assert int(f["Occupancy [waves/SIMD]"]) >= 5, (name, f)
            assert int(f["AGPRs"]) == 0 and int(f["VGPRs Spill"]) == 0, (name, f)


def test_scalar_registers_parked_in_vector_lanes(kernels):
    """They are moved around a segment's or a block's start, a lane each: as many as there are
    now, some in reserve."""
    for fragment, most in (("attention_pages_decode_kernel", None), ("attention_blocks_kernel", 80),
                           ("attention_pages_general_kernel", 60), ("rotary_kernel", 0), ("append_kernel", 0)):
        for name, f in matching(kernels, fragment).items():
            budget = most if most is not None else 280 if "ELb1E" in name else 100
            assert int(f["SGPRs Spill"]) <= budget, (name, f)
