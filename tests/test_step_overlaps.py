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


LOGITS = START + r"""
  // 6 rows of 100 columns, 3 sequences, one word of a tree's mask, 5 columns of history, 4 biases,
  // 4 words of allowed tokens; rows 104 apart.
  const std::vector<uint32_t> bytes = {0, 16, 24, 24, 60, 24, 36, 16, 32, 96};  // of the lists, in their order
  for (uint32_t element : {2u, 4u}) {
    const char* symbol = element == 2 ? "ipu_stack_adjust_logits_f16" : "ipu_stack_adjust_logits_f32";
    const uint32_t row = 104 * element, all = 5 * row + 100 * element;
    const char* x = m + 16384;
    auto call = [&](const char* out, const char* logits, uint32_t in_stride = 104, uint32_t out_stride = 104, uint32_t rows = 6) {
      std::vector<const void*> in(10, n);
      in[0] = logits;
      return run(symbol, out, in, {3, rows, 100, in_stride, out_stride, 1, 5, 4, 4});
    };
    CHECK(call(x, x) == 0 && entries.size() == 1);  // in place
    for (int sign : {1, -1}) {
      for (uint32_t shift : {element, 16u, 99 * element, row, row + 8, 2 * row, 5 * row, 5 * row + 99 * element})
        CHECK(call(x + sign * (int)shift, x) == IPUS_ERROR_INVALID_ARGUMENT && entries.empty());
      CHECK(call(x + sign * (int)(6 * row), x) == 0);
      CHECK(call(x + sign * (int)all, x) == 0);  // the last row's padding is not the input's
      CHECK(call(x + sign * (int)(100 * element), x) == IPUS_ERROR_INVALID_ARGUMENT);  // over the next row's beginning
      // Rows of the output between those of the input.
      CHECK(call(x + sign * (int)(100 * element), x, 200, 200) == 0 && entries.size() == 1);
      CHECK(call(x + sign * (int)(99 * element), x, 200, 200) == IPUS_ERROR_INVALID_ARGUMENT);
      CHECK(call(x + sign * (int)(101 * element), x, 200, 200) == IPUS_ERROR_INVALID_ARGUMENT);
      CHECK(call(x + sign * (int)(101 * element), x, 201, 201) == 0);
      CHECK(call(x + sign * (int)(4 * 200 + 100) * (int)element, x, 200, 200) == 0);
    }
    // Other strides: where no two rows meet.
    CHECK(call(x, x, 104, 100) == IPUS_ERROR_INVALID_ARGUMENT && call(x, x, 100, 104) == IPUS_ERROR_INVALID_ARGUMENT);
    CHECK(call(x + 100 * element, x, 700, 100) == 0 && call(x, x + 100 * element, 100, 700) == 0);
    CHECK(call(x + 101 * element, x, 700, 100) == IPUS_ERROR_INVALID_ARGUMENT);  // the last one
    CHECK(call(x, x + 101 * element, 100, 700) == IPUS_ERROR_INVALID_ARGUMENT);
    CHECK(call(x + 101 * element, x, 700, 100, 5) == 0);
    CHECK(call(x, x + 300 * element, 104, 250) == IPUS_ERROR_INVALID_ARGUMENT);
    // Each list: apart from the output, also between its rows, or refused.
    for (int list = 1; list < 10; ++list) {
      auto with = [&](const char* at, std::vector<uint32_t> s = {3, 6, 100, 104, 104, 1, 5, 4, 4}) {
        std::vector<const void*> in(10, n);
        in[0] = n + 8192;
        in[list] = at;
        return run(symbol, x, in, s);
      };
      const int size = (int)bytes[list];
      for (int at : {0, 4, (int)all / 2 / 4 * 4, (int)all - 4, 4 - size})
        CHECK(with(x + at) == IPUS_ERROR_INVALID_ARGUMENT && entries.empty());
      CHECK(with(x + all) == 0 && with(x - size) == 0 && entries.size() == 1);
      CHECK(with(x + 100 * element, {3, 6, 100, 104, 200, 1, 5, 4, 4}) == 0);
      CHECK(with(x + 200 * element - size, {3, 6, 100, 104, 200, 1, 5, 4, 4}) == 0);
      CHECK(with(x + 200 * element - size + 4, {3, 6, 100, 104, 200, 1, 5, 4, 4}) == IPUS_ERROR_INVALID_ARGUMENT);
      // A list that is not read lies anywhere.
      const bool always = list == 1 || list == 2 || list == 6;
      CHECK(with(x + 4, {3, 6, 100, 104, 104, 0, 0, 0, 0}) == (always ? IPUS_ERROR_INVALID_ARGUMENT : 0));
    }
  }
""" + END


def test_logits_apart_from_their_inputs(tmp_path):
    """A row of the output over another's input, or over a list that other workgroups still
    read, would be a race."""
    run_program(tmp_path, LOGITS)
