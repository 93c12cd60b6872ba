"""What the operators of a drafted step refuse before any device work, the tree masks'
arithmetic for any content, and the launches' grids (CPU)."""
from __future__ import annotations

import os
import shutil
import struct
import subprocess

import numpy as np
import pytest

from host_programs import run_program
from step_forms import fit_tables, table_state

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def bits(x):
    return struct.unpack("<I", struct.pack("<f", x))[0]


GOOD = {
    "ipu_stack_page_tables": (3, [4, 3, 100, 16, 8]),
    "ipu_stack_slot_maps": (4, [4, 9, 100, 16, 8, 1]),
    "ipu_stack_attention_tree_pages_f16": (6, [2, 8, 4, 8, 2, 64, 512, 10, 16, 4, 1, 0]),
    "ipu_stack_keep_pages_f16": (5, [2, 8, 3, 2, 64, 10, 16, 4, 5]),
    "ipu_stack_adjust_logits_f16": (10, [2, 8, 1001, 1001, 1008, 1, 50, 7, 32]),
}
GOOD["ipu_stack_adjust_logits_f32"] = GOOD["ipu_stack_adjust_logits_f16"]

# symbol -> (scalar, value, status)
BAD = {
    "ipu_stack_page_tables": [
        ("sequences", 4097, -3), ("previous_sequences", 4097, -3), ("sequences", 1 << 31, -1),
        ("page_rows", 0, -1), ("page_rows", 24, -1), ("page_rows", 1 << 17, -1), ("pages", 1 << 31, -1),
        ("table_columns", 1 << 30, -1), ("table_columns", 0xffffffff, -1)],
    "ipu_stack_slot_maps": [
        ("sequences", 1 << 31, -1), ("rows", 1 << 31, -1), ("page_rows", 3, -1), ("page_rows", 0, -1),
        ("pages", (1 << 27) + 1, -1), ("pages", 0xffffffff, -1)],
    "ipu_stack_attention_tree_pages_f16": [
        ("mask_words", 0, -1), ("query_heads", 0, -1), ("query_heads", 7, -1), ("width", 0, -1), ("width", 1025, -3),
        ("page_rows", 12, -1), ("key_heads", 0, -1), ("rows", 1 << 31, -1), ("sequences", 1 << 31, -1),
        ("scale_bits", bits(-1.0), -1), ("scale_bits", bits(float("nan")), -1), ("scale_bits", bits(1e30), -1)],
    "ipu_stack_keep_pages_f16": [
        ("sequences", 1 << 31, -1), ("rows", 1 << 31, -1), ("key_heads", 0, -1), ("key_heads", 40000, -1),
        ("width", 0, -1), ("page_rows", 5, -1)],
    "ipu_stack_adjust_logits_f16": [
        ("sequences", 1 << 31, -1), ("rows", 1 << 31, -1), ("columns", 0, -1), ("columns", 1 << 31, -1),
        ("input_row_stride", 1000, -1), ("output_row_stride", 1000, -1), ("allowed_words", 31, -1),
        ("allowed_words", 1, -1), ("bias_entries", 1 << 31, -1)],
}
BAD["ipu_stack_adjust_logits_f32"] = BAD["ipu_stack_adjust_logits_f16"]


@pytest.mark.parametrize("symbol", sorted(GOOD))
def test_refusals(ipus, symbol):
    inputs, scalars = GOOD[symbol]
    info = ipus.kernel_abi(symbol)
    assert info.input_count == inputs and len(info.scalar_names) == len(scalars)

    def run(values, count=inputs):
        array = (ipus.ctypes.c_uint32 * len(values))(*values)
        return ipus._lib().ipus_validate_kernel_run(symbol.encode(), count, array, len(values))
    assert run(scalars) == 0
    assert run(scalars, inputs + 1) == ipus.ERROR_POINTER_ARITY
    assert run(scalars[:-1]) == ipus.ERROR_INVALID_ARGUMENT
    for name, value, status in BAD[symbol]:
        changed = list(scalars)
        changed[info.scalar_names.index(name)] = value
        assert run(changed) == status, (name, value)
    # None of what is optional.
    if "logits" in symbol:
        assert run(scalars[:5] + [0, 0, 0, 0]) == 0


MASKS = r"""
#include <limits.h>
#include <stdio.h>
#include <stdlib.h>
#include <vector>
#include "page_lookup.h"
using namespace ipus;
int main() {
  int failures = 0;
  srand(7);
  for (int round = 0; round < 200000; ++round) {
    const uint32_t words = rand() % 5;
    // Exactly as large as it says: a read past an end is seen by the sanitizer.
    std::vector<uint32_t> mask(words);
    for (uint32_t& w : mask) w = (uint32_t)rand() << 16 ^ (uint32_t)rand() ^ (rand() % 3 ? 0 : ~0u);
    std::vector<int> offsets = {rand() % 4 ? rand() % 9 : -3, rand() % 200}, lengths = {rand() % 400 - 20};
    if (rand() % 50 == 0) offsets = {INT_MIN, INT_MAX};
    if (rand() % 50 == 0) lengths = {rand() % 2 ? INT_MIN : INT_MAX};
    PagedBatch b{nullptr, offsets.data(), lengths.data(), 1, 4, 10, 16, 4, 0, 0};
    const uint32_t rows = rand() % 200;
    const TreeRows t = tree_rows(b, 0, rows, words);
    const int64_t n = offsets[1] > offsets[0] ? (int64_t)offsets[1] - offsets[0] : 0;
    if (t.bits > 32 * words || t.bits > rows || t.base != (int64_t)lengths[0] - n) ++failures;
    const uint32_t key = rand() % 3 ? (uint32_t)(rand() % 500) : (uint32_t)rand() * 2u;
    const uint64_t x = tree_window(mask.data(), t, key);
    for (int i = 0; i < 64; ++i) {
      const int64_t j = (int64_t)key + i - t.base;
      const bool want = j < 0 || (j < (int64_t)t.bits && (mask[j / 32] >> j % 32 & 1));
      if (want != (bool)(x >> i & 1)) ++failures;
    }
  }
  printf("%d failures\n", failures);
  return failures != 0;
}
"""


def test_masks_hold_for_any_content(tmp_path):
    compiler = shutil.which("g++") or shutil.which("c++")
    if compiler is None:
        pytest.skip("no host compiler")
    (tmp_path / "masks.cpp").write_text(MASKS)
    subprocess.run([compiler, "-std=c++20", "-g", "-O1", "-fsanitize=address,undefined",
                    "-I", os.path.join(ROOT, "ipu-stack_amd", "csrc"),
                    "-o", str(tmp_path / "masks"), str(tmp_path / "masks.cpp")], check=True)
    done = subprocess.run([str(tmp_path / "masks")], capture_output=True, text=True)
    assert done.returncode == 0, done.stdout + done.stderr


GRIDS = r"""
#include <algorithm>
#include "host_runtime.h"
static char memory[1 << 16] __attribute__((aligned(256)));
static ipus_context* ctx;
static int run(const char* symbol, const void* out, std::vector<const void*> in, std::vector<uint32_t> s) {
  entries.clear();
  return ipus_launch(ctx, symbol, (void*)out, in.data(), (int)in.size(), s.data(), (int)s.size());
}
int main() {
  CHECK(ipus_context_create(0, &ctx) == 0);
  const char* m = memory;
  const uint64_t threads = 1ull << 32;
  // Page tables: the new state apart from the previous one.
  const char* n = m + 4096;
  auto tables = [&](const char* out, const char* previous, uint32_t before, const char* source, const char* lengths) {
    return run("ipu_stack_page_tables", out, {previous, source, lengths}, {2, before, 27, 16, 10});
  };
  CHECK(tables(m, m + 4 * 51, 2, n, n) == 0 && entries.size() == 1);
  CHECK(tables(m + 4 * 29, m, 0, n, n) == 0 && tables(m, n, 2, m + 4 * 51, m + 4 * 51) == 0);
  CHECK(tables(m, n, 2, m + 4 * 51, n + 2) == IPUS_ERROR_INVALID_ARGUMENT);
  CHECK(tables(m, m + 4 * 50, 2, n, n) == IPUS_ERROR_INVALID_ARGUMENT && tables(m + 4 * 50, m, 2, n, n) == IPUS_ERROR_INVALID_ARGUMENT);
  CHECK(tables(m, m, 2, n, n) == IPUS_ERROR_INVALID_ARGUMENT && tables(m + 2, n, 2, n, n) == IPUS_ERROR_INVALID_ARGUMENT);
  CHECK(tables(m, n, 2, m + 4 * 50, n) == IPUS_ERROR_INVALID_ARGUMENT && tables(m, n, 2, n, m) == IPUS_ERROR_INVALID_ARGUMENT);
  CHECK(tables(m + 4, n, 2, n, m) == IPUS_ERROR_INVALID_ARGUMENT && tables(m + 8, n, 2, n, m) == 0);
  // Slot maps likewise: 3 + 1 + 2 x 5 words.
  for (int input = 0; input < 4; ++input) {
    std::vector<const void*> in = {n, n, n, n};
    in[input] = m + 4 * 13;
    CHECK(run("ipu_stack_slot_maps", m, in, {3, 5, 10, 16, 4, 1}) == IPUS_ERROR_INVALID_ARGUMENT);
    in[input] = m + 4 * 14;
    CHECK(run("ipu_stack_slot_maps", m, in, {3, 5, 10, 16, 4, 1}) == 0);
  }
  CHECK(run("ipu_stack_slot_maps", m, {n, n, n, m}, {3, 5, 10, 16, 4, 0}) == 0);  // a mask that is not read
  for (uint32_t sequences : {0u, 1u, 4096u})
    for (uint32_t columns : {0u, 1u, 2048u, 500000u})
      for (uint32_t pages : {0u, 3u, 0x7fffffffu}) {
        CHECK(run("ipu_stack_page_tables", m, {(const void*)(1ull << 40), m - 65536, m - 65536}, {sequences, 4096, pages, 1, columns}) == 0);
        CHECK(entries.size() == 1 && entries[0].grid.x >= 1 && (uint64_t)entries[0].grid.x * entries[0].block.x < threads);
        CHECK(entries[0].shared == 8 * (sequences + 4096) && entries[0].shared <= 65536);
      }
  // Slot maps: a thread per row, one workgroup at least (for the offsets).
  first_words = 1;
  for (uint32_t rows : {0u, 1u, 512u, 513u, 1u << 30, 0x7fffffffu}) {
    CHECK(run("ipu_stack_slot_maps", m, {m - 4096, m - 4096, m - 4096, m}, {3, rows, 10, 16, 4, 0}) == 0);
    uint64_t next = 0;
    for (const Entry& e : entries) {
      CHECK(e.words[0] == next && (uint64_t)e.grid.x * e.block.x < threads);
      next += e.grid.x;
    }
    CHECK(next >= 1 && next * 512 >= rows);
  }
  // Accepted rows: all columns of all heads of all sequences and layers.
  for (uint32_t sequences : {1u, 70000u, 0x7fffffffu})
    for (uint32_t width : {1u, 8u, 72u, 2048u})
      for (uint32_t heads : {1u, 8u, 32767u}) {
        const int status = run("ipu_stack_keep_pages_f16", m, {m, m, m, m, m}, {sequences, 5, 40, heads, width, 10, 16, 4, 3});
        uint64_t next = 0;
        for (const Entry& e : entries) {
          CHECK(e.words[0] == next && (uint64_t)e.grid.x * e.block.x < threads && e.grid.z == 40);
          CHECK((uint64_t)e.grid.y * 256 >= 2ull * heads * (width % 8 ? width : width / 8) && e.grid.y <= 65535);
          next += e.grid.x;
        }
        CHECK(status == 0 && next == sequences);
      }
  CHECK(run("ipu_stack_keep_pages_f16", m, {m, m, m, m, m}, {1, 5, 65536, 1, 8, 10, 16, 4, 3}) == IPUS_ERROR_UNAVAILABLE);
  CHECK(run("ipu_stack_keep_pages_f16", m + 1, {m, m, m, m, m}, {1, 5, 1, 1, 8, 10, 16, 4, 3}) == IPUS_ERROR_INVALID_ARGUMENT);
  for (int zero : {0, 1, 2, 8}) {
    std::vector<uint32_t> s = {1, 5, 1, 1, 8, 10, 16, 4, 3};
    s[zero] = 0;
    CHECK(run("ipu_stack_keep_pages_f16", m, {m, m, m, m, m}, s) == 0 && entries.empty());
  }
  // Logits: all rows; in place only with one stride.
  std::vector<const void*> in(10, m);
  CHECK(run("ipu_stack_adjust_logits_f16", m, in, {3, 70, 100, 100, 104, 0, 0, 0, 0}) == IPUS_ERROR_INVALID_ARGUMENT);
  CHECK(run("ipu_stack_adjust_logits_f16", m, in, {3, 70, 100, 104, 104, 0, 0, 0, 0}) == 0 && entries.size() == 1);
  CHECK(run("ipu_stack_adjust_logits_f32", m + 2, in, {3, 70, 100, 100, 100, 0, 0, 0, 0}) == IPUS_ERROR_INVALID_ARGUMENT);
  CHECK(run("ipu_stack_adjust_logits_f16", m + 2, in, {3, 70, 100, 100, 100, 0, 0, 0, 0}) == 0);
  CHECK(run("ipu_stack_adjust_logits_f16", m, in, {3, 0, 100, 100, 100, 0, 0, 0, 0}) == 0 && entries.empty());
  CHECK(run("ipu_stack_adjust_logits_f16", m, in, {0, 3, 100, 100, 100, 0, 0, 0, 0}) == 0 && entries.empty());
  // Every chunk of every group of rows has a workgroup, whatever the sequences' rows: a group
  // takes up to 8 fp16 rows of a sequence, each sequence a partial one more at most.
  for (uint32_t sequences : {1u, 3u, 64u, 1000u, 70000u})
    for (uint32_t rows : {1u, 5u, 700u, 4000u, 200000u, 1u << 28})
      for (uint32_t columns : {1u, 4096u, 4097u, 131072u, 1000001u}) {
        CHECK(run("ipu_stack_adjust_logits_f16", m, in, {sequences, rows, columns, columns, columns, 0, 0, 0, 0}) == 0);
        const uint64_t chunks = (columns + 4095) / 4096, fill = rows * chunks / 2048;
        const uint64_t group = rows <= sequences || fill < 1 ? 1 : fill > 8 ? 8 : fill;
        uint64_t next = 0;
        for (const Entry& e : entries) {
          CHECK(e.words[0] == next && e.grid.x == chunks && e.grid.y <= 65535 && e.block.x == 512);
          next += e.grid.y;
        }
        CHECK(next == std::min<uint64_t>(rows, group == 1 ? rows : rows / group + sequences));
      }
  // A tree's mask has whole words.
  std::vector<const void*> tree = {m, m, m, m, m, m + 2};
  CHECK(run("ipu_stack_attention_tree_pages_f16", m, tree, {2, 8, 4, 8, 2, 64, 512, 10, 16, 4, 1, 0}) == IPUS_ERROR_INVALID_ARGUMENT);
  tree[5] = m;
  CHECK(run("ipu_stack_attention_tree_pages_f16", m, tree, {2, 8, 4, 8, 2, 64, 512, 10, 16, 4, 1, 0}) == 0 && !entries.empty());
  return failures != 0;
}
"""


def test_grids(tmp_path):
    run_program(tmp_path, GRIDS)


def test_the_form_of_page_tables_keeps_every_page():
    """The definition that the device is held to: no page is lost, doubled or held twice."""
    rng = np.random.default_rng(3)
    free, rows = list(rng.permutation(40)), []
    for _ in range(200):
        count = int(rng.integers(0, 7))
        source = [int(x) for x in rng.integers(-1, max(1, len(rows)) + 1, count)]
        lengths = [int(x) for x in rng.integers(-3, 70, count)]
        before = sorted(free + sum(rows, []))
        free, rows, missing = fit_tables(free, rows, source, lengths, 4, 12)
        assert sorted(free + sum(rows, [])) == before and missing >= 0
        assert all(len(r) <= min(12, max(0, (x + 3) // 4)) for r, x in zip(rows, lengths))
        assert missing == 0 or not free
        state = table_state(free, rows, 40, 12, missing)
        assert state[0] == len(free) and len(state) == 2 + 40 + count * 13
