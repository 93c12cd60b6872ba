// A HIP runtime without a device, linked ahead of the real one into programs that test
// libipus.so's host side: memory is the host's, and a launch is an entry of a log.
#pragma once

#include <hip/hip_runtime_api.h>
#include <stdio.h>
#include <stdlib.h>
#include <string.h>

#include <atomic>
#include <chrono>
#include <mutex>
#include <string>
#include <thread>
#include <vector>

#include "ipus.h"
#include "ipus_graph.h"

struct Entry {
  std::string what;     // "launch", "replay", "begin", "end", "copy", "fill", "wait", "event"
  std::thread::id by;
  dim3 grid;
  const void* kernel;
  std::vector<char> first;  // bytes of a kernel's first argument
  dim3 block;
  size_t shared;
  std::vector<uint32_t> words;  // its arguments behind the first, of 32 bits each
};
inline std::mutex log_mutex;
inline std::vector<Entry> entries;
inline int pause_us = 0;                 // how long an entry takes
inline size_t first_bytes = 0;           // of each launch's first argument, to be logged
inline size_t first_words = 0;           // how many arguments of 32 bits behind it
inline size_t largest_allocation = ~0ull;
inline std::vector<size_t> allocations;  // that succeeded
inline std::atomic<bool> stream_captured{false};
inline int failures = 0;
#define CHECK(x) do { if (!(x)) { printf("line %d: %s\n", __LINE__, #x); ++failures; } } while (0)

inline void record(Entry e, const void* first = nullptr) {
  e.by = std::this_thread::get_id();
  if (first && first_bytes) e.first.assign((const char*)first, (const char*)first + first_bytes);
  {
    std::lock_guard<std::mutex> lock(log_mutex);
    entries.push_back(std::move(e));
  }
  if (pause_us) std::this_thread::sleep_for(std::chrono::microseconds(pause_us));
}

inline void record(const char* what) { record(Entry{what}); }

struct Configuration {
  dim3 grid, block;
  size_t shared;
  hipStream_t stream;
};
inline thread_local Configuration pushed;

extern "C" {
hipError_t __hipPushCallConfiguration(dim3 grid, dim3 block, size_t shared, hipStream_t stream) {
  pushed = {grid, block, shared, stream};
  return hipSuccess;
}
hipError_t __hipPopCallConfiguration(dim3* grid, dim3* block, size_t* shared, hipStream_t* stream) {
  *grid = pushed.grid;
  *block = pushed.block;
  *shared = pushed.shared;
  *stream = pushed.stream;
  return hipSuccess;
}
void** __hipRegisterFatBinary(const void*) {
  static void* handle;
  return &handle;
}
void __hipRegisterFunction(void**, const void*, char*, const char*, unsigned, void*, void*, dim3*, dim3*, int*) {}
void __hipRegisterVar(void**, void*, char*, char*, int, size_t, int, int) {}
void __hipUnregisterFatBinary(void**) {}
hipError_t hipLaunchKernel(const void* kernel, dim3 grid, dim3 block, void** args, size_t shared, hipStream_t) {
  Entry e{"launch", {}, grid, kernel, {}, block, shared, {}};
  for (size_t i = 0; i < first_words; ++i) e.words.push_back(*(const uint32_t*)args[1 + i]);
  record(std::move(e), args ? args[0] : nullptr);
  return hipSuccess;
}
hipError_t hipGetDeviceCount(int* n) { return *n = 1, hipSuccess; }
hipError_t hipSetDevice(int) { return hipSuccess; }
hipError_t hipGetLastError() { return hipSuccess; }
const char* hipGetErrorString(hipError_t) { return ""; }
hipError_t hipGetSymbolAddress(void** p, const void*) { return *p = malloc(64), hipSuccess; }
hipError_t hipMalloc(void** p, size_t bytes) {
  if (bytes > largest_allocation) return hipErrorOutOfMemory;
  allocations.push_back(bytes);
  return *p = aligned_alloc(256, (bytes + 255) / 256 * 256), *p ? hipSuccess : hipErrorOutOfMemory;
}
hipError_t hipFree(void* p) { return free(p), hipSuccess; }
hipError_t hipMemcpyAsync(void* to, const void* from, size_t n, hipMemcpyKind, hipStream_t) {
  record("copy");
  return memcpy(to, from, n), hipSuccess;
}
hipError_t hipMemsetAsync(void* p, int v, size_t n, hipStream_t) {
  record("fill");
  return memset(p, v, n), hipSuccess;
}
hipError_t hipStreamCreateWithFlags(hipStream_t* s, unsigned) { return *s = (hipStream_t)malloc(1), hipSuccess; }
hipError_t hipStreamDestroy(hipStream_t s) { return free(s), hipSuccess; }
hipError_t hipStreamSynchronize(hipStream_t) { return record("wait"), hipSuccess; }
hipError_t hipEventCreate(hipEvent_t* e) { return *e = (hipEvent_t)malloc(1), hipSuccess; }
hipError_t hipEventDestroy(hipEvent_t e) { return free(e), hipSuccess; }
hipError_t hipEventRecord(hipEvent_t, hipStream_t) { return record("event"), hipSuccess; }
hipError_t hipStreamIsCapturing(hipStream_t, hipStreamCaptureStatus* s) {
  return *s = stream_captured ? hipStreamCaptureStatusActive : hipStreamCaptureStatusNone, hipSuccess;
}
hipError_t hipStreamBeginCapture(hipStream_t, hipStreamCaptureMode) {
  stream_captured = true;
  return record("begin"), hipSuccess;
}
hipError_t hipStreamEndCapture(hipStream_t, hipGraph_t* g) {
  stream_captured = false;
  return record("end"), *g = (hipGraph_t)malloc(1), hipSuccess;
}
hipError_t hipGraphInstantiate(hipGraphExec_t* x, hipGraph_t, hipGraphNode_t*, char*, size_t) {
  return *x = (hipGraphExec_t)malloc(1), hipSuccess;
}
hipError_t hipGraphLaunch(hipGraphExec_t, hipStream_t) { return record("replay"), hipSuccess; }
hipError_t hipGraphDestroy(hipGraph_t g) { return free(g), hipSuccess; }
hipError_t hipGraphExecDestroy(hipGraphExec_t x) { return free(x), hipSuccess; }
}
