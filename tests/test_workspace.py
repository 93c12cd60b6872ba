"""A context's workspace where device memory is short (CPU: over a runtime whose
allocations fail past a size)."""
from __future__ import annotations

from host_programs import run_program

SOURCE = r"""
#include "host_runtime.h"
static char memory[1 << 16];
struct Launch {
  const void* kernel;
  uint32_t groups;
  bool operator==(const Launch&) const = default;
};
static std::vector<Launch> launches(ipus_context* ctx) {
  entries.clear();
  const uint32_t product[] = {1, 8, 1024, 4096, 0, 0, 0, 0};
  const uint32_t decode[] = {4, 1, 2048, 64, 64, 0, 0, 0};
  const uint32_t pages[] = {1, 70, 70, 4, 1, 64, 256, 300, 16, 260, 1, 0};
  const void* in[] = {memory, memory, memory, memory, memory};
  CHECK(ipus_launch(ctx, "ipu_stack_gemm_f16", memory, in, 2, product, 8) == 0);
  CHECK(ipus_launch(ctx, "ipu_stack_flash_attention_online_f16", memory, in, 3, decode, 8) == 0);
  CHECK(ipus_launch(ctx, "ipu_stack_attention_pages_f16", memory, in, 5, pages, 12) == 0);
  std::vector<Launch> all;
  for (const Entry& e : entries) all.push_back({e.kernel, e.grid.x * e.grid.y * e.grid.z});
  return all;
}
int main() {
  std::vector<Launch> split, unsplit;
  struct { size_t room, taken; } cases[] = {{~0ull, 96u << 20}, {96u << 20, 32u << 20}, {33u << 20, 32u << 20}, {32u << 20, 0}};
  for (auto& c : cases) {
    largest_allocation = c.room;
    allocations.clear();
    ipus_context* ctx;
    CHECK(ipus_context_create(0, &ctx) == 0);
    const size_t counters = 16384 * 4;
    if (c.taken)
      CHECK(allocations.size() == 1 && allocations[0] == c.taken + counters);
    else
      CHECK(allocations.empty());
    const std::vector<Launch> got = launches(ctx);
    if (c.room == ~0ull) split = got;
    if (c.taken) {
      CHECK(got == split && got.size() == 4);  // the paged attention's blocks and their join
    } else {
      CHECK(got.size() == 3 && got[0] != split[0] && got[1] != split[1]);
    }
    CHECK(ipus_context_destroy(ctx) == 0);
  }
  printf("%d failures\n", failures);
  return failures != 0;
}
"""


def test_the_workspace_is_smaller_where_memory_is_short(tmp_path):
    run_program(tmp_path, SOURCE)
