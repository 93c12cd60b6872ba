"""Register, scratch, occupancy and LDS budgets of the kernels around a step with drafted
tokens, from the compiler's resource remarks (no GPU needed; those of the tree attention
are the decoder kernels')."""
from __future__ import annotations

import os

import pytest

from test_kernel_resources import BUILD, matching, parse


@pytest.fixture(scope="module")
def kernels():
    out = {}
    for s in ("k_page_maps", "k_logits"):
        path = os.path.join(BUILD, f"{s}.resources")
        if not os.path.exists(path):
            pytest.skip("library not built by the package Makefile (no resource remarks)")
        got = parse(open(path).read())
        assert got, f"{s}.resources holds no kernel"
        out.update(got)
    return out


def test_no_spills(kernels):
    for name, f in kernels.items():
        assert int(f["ScratchSize [bytes/lane]"]) == 0 and int(f["VGPRs Spill"]) == 0, (name, f)
        assert f.get("Dynamic Stack", "False") == "False", name


@pytest.mark.parametrize("fragment,lds", [
    # Four workgroups of 512 threads per CU hide each other's start.
    ("adjust_row_kernel", 32768), ("adjust_rows_kernel", 40960), ("page_tables_kernel", 1024), ("slot_maps_kernel", 4096),
    ("keep_pages_kernel", 2048)])
def test_full_occupancy(kernels, fragment, lds):
    found = matching(kernels, fragment)
    assert found
    for name, f in found.items():
        assert int(f["Occupancy [waves/SIMD]"]) == 8 and int(f["LDS Size [bytes/block]"]) <= lds, (name, f)
        assert int(f["SGPRs Spill"]) <= 40, (name, f)
