"""The rotary kernels' launches cover all rows and heads within the limits of a grid, for any
sizes (CPU: over a runtime that logs its launches)."""
from __future__ import annotations

from host_programs import run_program

SOURCE = r"""
#include "host_runtime.h"
static char memory[4096] __attribute__((aligned(256)));
static ipus_context* ctx;
static void check(int status, uint32_t rows, uint32_t heads) {
  CHECK(status == 0);
  if (rows == 0 || heads == 0) {
    CHECK(entries.empty());
    return;
  }
  uint64_t next = 0;
  for (const Entry& e : entries) {
    const uint32_t first = e.words[0], per_block = e.words[1], head_block = e.words[2], lanes = e.words[3];
    CHECK(e.block.x == 256 && e.block.y == 1 && e.block.z == 1 && e.grid.z == 1);
    CHECK((uint64_t)e.grid.x * e.block.x < 1ull << 32 && e.grid.y <= 65535 && e.shared <= 16384);
    CHECK(first == next && per_block >= 1 && per_block <= 32 && lanes >= 1 && lanes <= 64 && (lanes & (lanes - 1)) == 0);
    next += (uint64_t)e.grid.x * per_block;
    CHECK((uint64_t)e.grid.y * head_block >= heads && (uint64_t)(e.grid.y - 1) * head_block < heads);
    if (failures) return;
  }
  CHECK(next >= rows && next - rows < 32);
}
int main() {
  CHECK(ipus_context_create(0, &ctx) == 0);
  first_words = 4;
  const void* in[] = {memory, memory, memory, memory, memory, memory};
  const uint32_t all_rows[] = {0, 1, 3, 64, 1000, 1023, 1024, 1025, 4095, 4096, 32767, 32768, 100003, (1u << 23) - 1,
                               1u << 23, (1u << 23) + 1, (1u << 28) + 5, 0x7ffffffe, 0x7fffffff};
  const uint32_t all_heads[] = {1, 2, 5, 16, 17, 40, 64, 255, 300, 1025, 32767, 65536, 70001, 16777215, 0x7fffffff};
  for (uint32_t width : {1u, 2u, 24u, 64u, 65u, 128u, 1000u, 2048u})
    for (uint32_t rotary : {0u, width / 4 * 2, width / 2 * 2})
      for (uint32_t rows : all_rows)
        for (uint32_t heads : all_heads) {
          const uint64_t row = (uint64_t)heads * width;
          if (row <= 0xffffffffu || rows <= 1) {
            const uint32_t s[] = {rows, heads, width, rotary, 0, (uint32_t)row, width, (uint32_t)row, width, 0};
            entries.clear();
            check(ipus_launch(ctx, width % 3 ? "ipu_stack_rotary_f16" : "ipu_stack_rotary_f32", memory + 1024, in, 3, s, 10), rows, heads);
            const uint32_t n[] = {rows, heads / 3, heads - heads / 3, width, rotary, 1, (uint32_t)row, (uint32_t)row, 0, 0};
            entries.clear();
            check(ipus_launch(ctx, width % 3 ? "ipu_stack_norm_rotary_f32" : "ipu_stack_norm_rotary_f16", memory + 1024, in, 5, n, 10), rows, heads);
          }
          if (heads > 32767) continue;
          const uint32_t a[] = {7, rows, heads, width, (uint32_t)row, (uint32_t)row, rotary, 0, 0, 10, 16, 4};
          entries.clear();
          check(ipus_launch(ctx, "ipu_stack_append_pages_f16", memory + 1024, in, 6, a, 12), rows, 2 * heads);
          if (failures) return printf("%u rows, %u heads, %u of %u columns\n", rows, heads, rotary, width), 1;
        }
  return failures != 0;
}
"""


def test_rotary_grids(tmp_path):
    run_program(tmp_path, SOURCE)
