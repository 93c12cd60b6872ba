"""Norm with rotation where one of the two groups has no heads: its weight pointer
is passed on to no kernel (CPU: over a runtime that logs its launches)."""
from __future__ import annotations

import pytest

from host_programs import run_program

SOURCE = r"""
#include "host_runtime.h"
#include "kernels.h"
using namespace ipus;
static char memory[4096] __attribute__((aligned(256)));
int main() {
  ipus_context* ctx;
  CHECK(ipus_context_create(0, &ctx) == 0);
  first_bytes = sizeof(RotaryArgs);
  char* const weight = memory + 1024;
  char* const placeholder = (char*)3;  // not null, of no alignment, no memory
  const bool f32 = FLOATS;
  auto launch = [&](uint32_t query, uint32_t key, void* wq, void* wk) {
    entries.clear();
    const void* in[] = {memory, wq, wk, memory, memory};
    const uint32_t s[] = {4, query, key, 64, 64, 0, 192, 192, 0x358637bd, 0};
    return ipus_launch(ctx, f32 ? "ipu_stack_norm_rotary_f32" : "ipu_stack_norm_rotary_f16", memory + 2048, in, 5, s, 10);
  };
  auto weights_are = [&](size_t i, const void* wq, const void* wk) {
    const RotaryArgs* a = (const RotaryArgs*)entries.at(i).first.data();
    CHECK(a->query_weight == wq && a->key_weight == wk);
  };
  CHECK(launch(2, 1, weight, weight + 512) == 0 && entries.size() == 1);
  weights_are(0, weight, weight + 512);
  const void* const kernel = entries[0].kernel;
  CHECK(launch(3, 0, weight, placeholder) == 0 && entries.size() == 1 && entries[0].kernel == kernel);
  weights_are(0, weight, weight);
  CHECK(launch(0, 3, placeholder, weight) == 0 && entries.size() == 1 && entries[0].kernel == kernel);
  weights_are(0, weight, weight);
  CHECK(launch(0, 0, placeholder, placeholder) == 0 && entries.empty());
  CHECK(launch(3, 0, weight, nullptr) == IPUS_ERROR_INVALID_ARGUMENT);
  CHECK(launch(3, 0, weight + 1, weight) == IPUS_ERROR_INVALID_ARGUMENT);
  printf("%d failures\n", failures);
  return failures != 0;
}
"""


@pytest.mark.parametrize("floats", ["false", "true"])
def test_the_weight_of_no_heads_is_not_read(tmp_path, floats):
    run_program(tmp_path, SOURCE.replace("FLOATS", floats))
