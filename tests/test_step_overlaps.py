"""Which addresses of outputs and inputs the operators of a drafted step refuse, before any
device work (CPU)."""
from __future__ import annotations

from host_programs import run_program

START = r"""
#include "host_runtime.h"
static char memory[1 << 16] __attribute__((aligned(256)));
static const char* const m = memory;       // outputs
static const char* const n = memory + 32768;  // inputs apart from them
static ipus_context* ctx;
static int run(const char* symbol, const void* out, std::vector<const void*> in, std::vector<uint32_t> s) {
  entries.clear();
  return ipus_launch(ctx, symbol, (void*)out, in.data(), (int)in.size(), s.data(), (int)s.size());
}
int main() {
  CHECK(ipus_context_create(0, &ctx) == 0);
"""
END = r"""
  return failures != 0;
}
"""

EMPTY = START + r"""
  // Slot maps of 3 sequences and 5 rows are 14 words: a mask of no words, a table of no columns.
  for (int at : {0, 4, 20, 52}) {
    CHECK(run("ipu_stack_slot_maps", m, {n, n, n, m + at}, {3, 5, 10, 16, 4, 0}) == 0 && entries.size() == 1);
    CHECK(run("ipu_stack_slot_maps", m, {n, n, m + at, n}, {3, 5, 10, 16, 0, 1}) == 0 && entries.size() == 1);
    CHECK(run("ipu_stack_slot_maps", m, {n, n, n, m + at}, {3, 5, 10, 16, 4, 1}) == IPUS_ERROR_INVALID_ARGUMENT);
    CHECK(run("ipu_stack_slot_maps", m, {n, n, m + at, n}, {3, 5, 10, 16, 1, 0}) == IPUS_ERROR_INVALID_ARGUMENT);
    // No sequences: no counts and no lengths either.
    CHECK(run("ipu_stack_slot_maps", m, {m + at % 44, m + at % 44, m + at % 44, n}, {0, 5, 10, 16, 4, 1}) == 0);
    // No rows: no mask.
    CHECK(run("ipu_stack_slot_maps", m, {n, n, n, m + at % 16}, {3, 0, 10, 16, 4, 1}) == 0);
  }
  // Page tables of no sequences: 2 + 27 words, no sources and no lengths.
  for (int at : {0, 4, 112})
    CHECK(run("ipu_stack_page_tables", m, {n, m + at, m + at}, {0, 2, 27, 16, 10}) == 0 && entries.size() == 1);
  CHECK(run("ipu_stack_page_tables", m, {n, m + 4, n}, {1, 2, 27, 16, 10}) == IPUS_ERROR_INVALID_ARGUMENT);
""" + END


def test_empty_inputs_lie_anywhere(tmp_path):
    """An input that a scalar of 0 leaves empty is not read: its pointer may be any, also one
    into the output."""
    run_program(tmp_path, EMPTY)
