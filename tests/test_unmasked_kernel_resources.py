"""Registers of the paged attention's kernels that take no tree's mask (causal rows, whole sequences,
shared keys): what the masks need is not to change them (no GPU needed)."""
from __future__ import annotations

import os

import pytest

from test_kernel_resources import BUILD, matching, parse


@pytest.mark.parametrize("source,fragment,registers", [
    # <width, columns loaded, query tiles, shared keys, tree>
    ("k_attention_blocks", "attention_blocks_kernelILi128ELi128ELi2ELb0ELb0E", 239),
    ("k_attention_blocks", "attention_blocks_kernelILi128ELi96ELi2ELb0ELb0E", 207),
    ("k_attention_blocks", "attention_blocks_kernelILi64ELi64ELi2ELb0ELb0E", 169),
    ("k_attention_blocks", "attention_blocks_kernelILi64ELi32ELi2ELb0ELb0E", 136),
    ("k_attention_blocks", "attention_blocks_kernelILi128ELi128ELi2ELb1ELb0E", 240),
    ("k_attention_blocks", "attention_blocks_kernelILi128ELi96ELi2ELb1ELb0E", 205),
    # <width, query tiles, shared keys, tree>
    ("k_attention_pages", "attention_pages_decode_kernelILi96ELi2ELb0ELb0E", 231),
    ("k_attention_pages", "attention_pages_decode_kernelILi64ELi2ELb0ELb0E", 233),
    ("k_attention_pages", "attention_pages_decode_kernelILi32ELi2ELb0ELb0E", 176),
    ("k_attention_pages", "attention_pages_decode_kernelILi96ELi2ELb1ELb0E", 238)])
def test_registers(source, fragment, registers):
    path = os.path.join(BUILD, source + ".resources")
    if not os.path.exists(path):
        pytest.skip("library not built by the package Makefile (no resource remarks)")
    found = matching(parse(open(path).read()), fragment)
    assert len(found) == 1
    for name, f in found.items():
        assert int(f["VGPRs"]) <= registers and int(f["VGPRs Spill"]) == 0, (name, f)
