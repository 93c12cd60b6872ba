"""The launches of one call stand together on a context's stream, whatever other
threads enqueue (CPU: the library's host side over a runtime that logs its launches)."""
from __future__ import annotations

from host_programs import run_program

SOURCE = r"""
#include "host_runtime.h"
static char memory[1 << 16];
static ipus_context* ctx;

// Attention of 70 rows on one key head against a table of 4,160 keys: split blocks and
// their join; and of 300 single rows behind 1,000 shared keys: those, then the decode.
static int split_keys() {
  const uint32_t s[] = {1, 70, 70, 4, 1, 64, 256, 300, 16, 260, 1, 0};
  const void* in[] = {memory, memory, memory, memory, memory};
  return ipus_launch(ctx, "ipu_stack_attention_pages_f16", memory, in, 5, s, 12);
}
static int shared_keys() {
  const uint32_t s[] = {300, 300, 1, 16, 4, 64, 1024, 600, 16, 64, 1, 0, 1000};
  const void* in[] = {memory, memory, memory, memory, memory};
  return ipus_launch(ctx, "ipu_stack_attention_shared_pages_f16", memory, in, 5, s, 13);
}
static int product() {  // splits its sum in the same workspace
  const uint32_t s[] = {1, 8, 1024, 4096, 0, 0, 0, 0};
  const void* in[] = {memory, memory};
  return ipus_launch(ctx, "ipu_stack_gemm_f16", memory, in, 2, s, 8);
}
static int split_product() {  // partial products in the library's own array, then their sum
  return ipus_gemm_f16_split_noalloc(ctx, memory, memory, memory, 1, 8, 512, 4096, 0, 0, 0, 0, 4, 0);
}
static ipus_session* two_products() {
  ipus_graph* g;
  ipus_value x, w, y, out;
  const uint32_t dx[] = {8, 512}, dw[] = {512, 512};
  ipus_graph_create(&g);
  ipus_graph_host_input(g, "x", dx, 2, &x);
  ipus_graph_parameter(g, "w", dw, 2, &w);
  ipus_graph_gemm(g, x, w, 0, 0, &y);
  ipus_graph_gemm(g, y, w, 0, 0, &out);
  ipus_graph_set_outputs(g, &out, 1);
  ipus_package_config config = {};
  config.compute_precision = IPUS_PRECISION_F32;
  ipus_package* p;
  ipus_session* s;
  CHECK(ipus_build_package(g, &config, &p) == 0 && ipus_session_create(ctx, p, &s) == 0);
  return s;
}

template <typename A, typename B>
static void together(A a, B b, std::thread::id* ia, std::thread::id* ib) {
  entries.clear();
  std::atomic<int> ready{0};
  auto both = [&](auto f) {
    ++ready;
    while (ready < 2) {}
    f();
  };
  std::thread ta([&] { both(a); }), tb([&] { both(b); });
  *ia = ta.get_id();
  *ib = tb.get_id();
  ta.join();
  tb.join();
}
// Entries of `by` come in whole runs of `each`.
static void stands_together(std::thread::id by, size_t each) {
  size_t run = 0, all = 0;
  for (const Entry& e : entries) {
    if (e.by == by) {
      ++run;
      ++all;
    } else {
      CHECK(run % each == 0);
      run = 0;
    }
  }
  CHECK(run % each == 0 && all > 0);
}

// Sessions captured, run and closed by one thread; another's entries stand outside of captures.
static void captures(int n) {
  for (int i = 0; i < n; ++i) {
    ipus_session* t = two_products();
    CHECK(ipus_session_capture(t) == 0 && ipus_session_capture(t) == 0);
    CHECK(ipus_session_run(t) == 0 && ipus_session_destroy(t) == 0);
  }
}
static void stands_outside(std::thread::id capturing, int n) {
  bool recording = false;
  int begun = 0, replayed = 0, beside = 0;
  for (const Entry& e : entries) {
    if (e.what == "begin") recording = true, ++begun;
    if (e.what == "end") recording = false;
    if (e.what == "replay") ++replayed;
    if (e.by != capturing) ++beside;
    CHECK(!recording || e.by == capturing);
  }
  CHECK(begun == n && replayed == n && beside > 0);
}

int main() {
  CHECK(ipus_context_create(0, &ctx) == 0);
  entries.clear();
  CHECK(split_keys() == 0 && entries.size() == 2);
  entries.clear();
  CHECK(shared_keys() == 0 && entries.size() == 2);
  entries.clear();
  CHECK(product() == 0 && entries.size() == 1);
  entries.clear();
  CHECK(split_product() == 0 && entries.size() == 2);
  pause_us = 300;
  auto loop = [](auto f, int n) { return [=] { for (int i = 0; i < n; ++i) CHECK(f() == 0); }; };
  std::thread::id a, b;
  together(loop(split_keys, 30), loop(product, 60), &a, &b);
  stands_together(a, 2);
  together(loop(shared_keys, 30), loop(product, 60), &a, &b);
  stands_together(a, 2);
  together(loop(split_keys, 30), loop(shared_keys, 30), &a, &b);
  stands_together(a, 2);
  stands_together(b, 2);
  together(loop(split_product, 30), loop(split_product, 30), &a, &b);
  stands_together(a, 2);
  stands_together(b, 2);
  // A session's run, its replays and its capture.
  ipus_session* s = two_products();
  auto run = [=] { return ipus_session_run(s); };
  together(loop(split_keys, 30), loop(run, 30), &a, &b);
  stands_together(a, 2);
  stands_together(b, 2);
  together(loop(split_keys, 20), [] { captures(10); }, &a, &b);
  stands_together(a, 2);
  stands_outside(b, 10);
  together(loop(split_product, 20), [] { captures(10); }, &a, &b);
  stands_outside(b, 10);
  // Copies, fills, waits and events beside captures.
  ipus_event* event;
  CHECK(ipus_event_create(ctx, &event) == 0);
  static char host[64];
  auto others = [=] {
    const int done[] = {ipus_buffer_upload(ctx, memory, host, 64), ipus_buffer_download(ctx, host, memory, 64),
                        ipus_buffer_copy(ctx, memory, memory + 64, 64), ipus_buffer_memset(ctx, memory, 0, 64),
                        ipus_stream_sync(ctx), ipus_event_record(ctx, event)};
    for (int e : done) if (e) return e;
    return 0;
  };
  together(loop(others, 15), [] { captures(10); }, &a, &b);
  stands_outside(b, 10);
  printf("%d failures\n", failures);
  return failures != 0;
}
"""


def test_launches_of_a_call_stand_together(tmp_path):
    run_program(tmp_path, SOURCE)
