"""Lookups in a ragged batch and a paged cache (csrc/page_lookup.h), compiled for
the host: arrays of any content stay within their bounds."""
from __future__ import annotations

import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

SOURCE = r"""
#include <limits.h>
#include <stdio.h>
#include <vector>
#include "page_lookup.h"
using namespace ipus;
static int failures = 0;
#define CHECK(x) do { if (!(x)) { printf("line %d: %s\n", __LINE__, #x); ++failures; } } while (0)
int main() {
  // Exactly as large as the batch says: an access past an end is seen by the
  // address sanitizer that the test builds this with.
  const int kLow = INT_MIN, kHigh = INT_MAX;
  std::vector<int> table = {3, -1, 10, kLow, 0, 9, kHigh, 2};
  std::vector<int> offsets = {0, 5, 2}, lengths = {7, kHigh};
  PagedBatch b{table.data(), offsets.data(), lengths.data(), 2, 4, 10, 16, 4, 0, 0};
  CHECK(page_of(b, 0, 0) == 3 && page_of(b, 0, 15) == 3);
  CHECK(page_of(b, 0, 16) == -1);            // below 0
  CHECK(page_of(b, 0, 32) == -1);            // == pages
  CHECK(page_of(b, 0, 48) == -1);            // INT_MIN
  CHECK(page_of(b, 0, 64) == -1);            // past the table
  CHECK(page_of(b, 1, 0xffffffffu) == -1);
  CHECK(page_of(b, 1, 0) == 0 && page_of(b, 1, 31) == 9 && page_of(b, 1, 32) == -1 && page_of(b, 1, 63) == 2);
  b.shared_rows = 5;                          // through the first table below it
  CHECK(page_of(b, 1, 4) == 3 && page_of(b, 1, 5) == 0);
  b.pages = 0;
  CHECK(page_of(b, 0, 0) == -1);
  b.pages = 0xffffffffu;
  CHECK(page_of(b, 0, 16) == -1 && page_of(b, 1, 47) == kHigh);
  b.pages = 10;
  // Rows: offsets that decrease or pass the rows are cut off, keys end with the table.
  BatchSequence q = sequence_at(b, 0, 8);
  CHECK(q.first == 0 && q.rows == 5 && q.keys == 7 && q.length == 7 && q.end == 5);
  q = sequence_at(b, 0, 3);                   // fewer rows than the offsets say: the first three
  CHECK(q.first == 0 && q.rows == 3 && q.end == 5 && row_position(q.length, q.end, 2) == 4);
  q = sequence_at(b, 1, 8);
  CHECK(q.rows == 0 && q.first <= 8 && q.keys == 64);
  offsets = {kLow, kHigh, kHigh};
  b.row_offsets = offsets.data();
  q = sequence_at(b, 0, 8);
  CHECK(q.first == 0 && q.rows == 8);
  q = sequence_at(b, 1, 8);
  CHECK(q.first == 8 && q.rows == 0);
  lengths = {kLow, 0};
  CHECK(sequence_at(b, 0, 8).keys == 0 && sequence_at(b, 1, 8).keys == 0);
  // Positions: the last row at length - 1, none below 0 or past an int.
  CHECK(row_position(7, 5, 4) == 6 && row_position(7, 5, 0) == 2 && row_position(2, 5, 2) == -1);
  CHECK(row_position(2, 5, 3) == 0 && row_position(kLow, kHigh, 0) == -1 && row_position(kHigh, kLow, 9) == -1);
  BatchSequence keys{0, 1, 64, 100, 1};
  CHECK(readable_keys(keys, -1, true) == 0 && readable_keys(keys, 0, true) == 1);
  CHECK(readable_keys(keys, 63, true) == 64 && readable_keys(keys, kHigh, true) == 64);
  CHECK(readable_keys(keys, -1, false) == 64);
  printf("%d failures\n", failures);
  return failures != 0;
}
"""


def test_lookups_hold_for_any_content(tmp_path):
    compiler = shutil.which("g++") or shutil.which("c++")
    if compiler is None:
        pytest.skip("no host compiler")
    (tmp_path / "lookup.cpp").write_text(SOURCE)
    subprocess.run([compiler, "-std=c++20", "-g", "-fsanitize=address,undefined",
                    "-I", os.path.join(ROOT, "ipu-stack_amd", "csrc"),
                    "-o", str(tmp_path / "lookup"), str(tmp_path / "lookup.cpp")], check=True)
    done = subprocess.run([str(tmp_path / "lookup")], capture_output=True, text=True)
    assert done.returncode == 0, done.stdout + done.stderr
