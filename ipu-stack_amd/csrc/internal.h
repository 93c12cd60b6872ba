// Internal host-side declarations shared by the libipus translation units.
#pragma once

#include <hip/hip_runtime.h>

#include <cstddef>
#include <cstdint>

#include "../../include/ipus.h"

#include <atomic>
#include <mutex>
#include <shared_mutex>
#include <unordered_map>

struct ipus_context {
  int device = 0;
  hipStream_t stream = nullptr;
  // Buffers allocated through this context and not yet freed (pointer ->
  // bytes); ipus_context_destroy releases whatever is left.
  std::mutex live_mutex;
  std::unordered_map<void*, size_t> live;
  // Failure injection (ipus_context_inject_launch_failure): after
  // inject_after more launches, the next one returns inject_status.
  uint32_t inject_after = 0;
  int inject_status = 0;
  // Workspace of the kernels that split a reduction over workgroups
  // (context_workspace): allocated with the context, not counted among the
  // buffers above.
  void* workspace = nullptr;
  size_t workspace_bytes = 0;
  uint32_t* workspace_counters = nullptr;
  // Held while a call enqueues its launches on the stream: by ipus_launch (some
  // operators are two launches with parts in the workspace between them), by
  // ipus_gemm_f16_split_noalloc, by a session's replay, and over the whole of ipus_session_capture, whose steps come
  // through ipus_launch again.
  std::recursive_mutex enqueue_mutex;
  // Held by ipus_session_capture, shared by copies, fills, events and waits: on a stream
  // that is being captured those would be recorded, or end the capture.
  std::shared_mutex capture_mutex;
  // ipus_session_capture is recording this context's stream into a graph
  // that will only be launched on it.
  std::atomic<bool> capturing_session{false};
};

namespace ipus {

struct Workspace;
// The context's workspace, for the launches of one call on its stream.  Launches
// there run one after the other, and enqueue_mutex, which the caller holds, keeps
// other threads' launches from coming between those of one call: so all can share it.
// Empty where the allocation failed, and while a caller records the stream
// into a graph of its own (which it may launch on other streams, several at
// once): the unsplit kernels run then.  paged: all of it, for the paged attention.
Workspace context_workspace(const ipus_context* ctx, bool paged = false);
// The context's stream is being recorded into a graph (or cannot tell).
bool stream_recorded(const ipus_context* ctx);

// Records a formatted message as the thread's last error and returns `code`.
int fail(int code, const char* fmt, ...) __attribute__((format(printf, 2, 3)));
int hip_fail(hipError_t e, const char* what);
// Makes the context's device current for the calling thread.
int use_device(const ipus_context* ctx);
// Turns a launcher status into a recorded error for `symbol`.
int check_launch(int status, const char* symbol);

int run_flat_add(ipus_context* c, void* o, const void* const* i, const uint32_t* s, int precision);
int run_broadcast_add(ipus_context* c, void* o, const void* const* i, const uint32_t* s,
                      int precision);

}  // namespace ipus
