// Penalties for repeated tokens, biases and masks on the logits of a step's rows:
//   x' = x / r (x > 0) or x r (else) of a token that stands in the sequence's history or
//        the row's path, then x' - (f g + p [g > 0]) with g its uses behind the prompt,
//   then x' + its bias, and -inf for a token that the row's mask does not allow.
// The path of a row is the rows of its sequence that its mask names, or those up to itself.
// Bound by HBM: the logits once in, once out.
#include "../../include/ipus.h"
#include "kernels.h"
#include "pages.h"
#include "wave_scan.h"

namespace ipus {
namespace {

inline int hip_status(hipError_t e) { return e == hipSuccess ? 0 : IPUS_ERROR_HIP_BASE - (int)e; }

// A workgroup takes a chunk of a row's tokens: how often each stands where is counted
// in LDS (integers: any order gives the same), then the chunk's logits pass through once.
constexpr uint32_t kLogitThreads = 256, kChunk = 4096;
constexpr uint32_t kInPrompt = 1u << 31;  // beside the uses behind the prompt
template <typename T>
__global__ __launch_bounds__(kLogitThreads) void adjust_logits_kernel(LogitArgs a, uint32_t first_row) {
  constexpr uint32_t kPer = 16 / sizeof(T);
  typedef T Pack __attribute__((ext_vector_type(kPer)));
  typedef Pack Loose __attribute__((aligned(sizeof(T))));  // rows of any alignment
  __shared__ uint32_t uses[kChunk];
  __shared__ uint32_t bias_entry[kChunk];  // 1 + the last entry of the token, 0: none
  const uint32_t row = first_row + blockIdx.y, chunk0 = blockIdx.x * kChunk, tid = threadIdx.x;
  PagedBatch b{};
  b.row_offsets = a.row_offsets;
  b.sequences = a.sequences;
  const uint32_t s = uniform(find_sequence(b, row));
  if (s >= a.sequences) return;
  const int64_t first = a.row_offsets[s], end = a.row_offsets[s + 1];
  if ((int64_t)row < first) return;
  const uint32_t tokens = a.columns - chunk0 < kChunk ? a.columns - chunk0 : kChunk;

  for (uint32_t i = tid; i < kChunk; i += kLogitThreads) uses[i] = bias_entry[i] = 0;
  __syncthreads();
  auto use = [&](int token, uint32_t prompt) __attribute__((always_inline)) {
    const uint32_t at = (uint32_t)token - chunk0;
    if (token >= 0 && at < tokens) prompt ? atomicOr(uses + at, kInPrompt) : atomicAdd(uses + at, 1u);
  };
  if (a.history_columns > 0) {
    const int given = a.history_counts[2 * (uint64_t)s], all = a.history_counts[2 * (uint64_t)s + 1];
    const uint32_t total = all <= 0 ? 0 : (uint32_t)all < a.history_columns ? (uint32_t)all : a.history_columns;
    const uint32_t prompt = given <= 0 ? 0 : (uint32_t)given < total ? (uint32_t)given : total;
    const int* history = a.history + (uint64_t)s * a.history_columns;
    for (uint32_t i = tid; i < total; i += kLogitThreads) use(history[i], i < prompt);
  }
  {
    const uint32_t* mask = a.mask + (uint64_t)row * a.mask_words;
    const uint64_t count = a.mask_words ? (uint64_t)(end - first) : (uint64_t)(row - first) + 1;
    const uint64_t reach = a.mask_words ? 32ull * a.mask_words : count;
    for (uint64_t j = tid; j < (count < reach ? count : reach); j += kLogitThreads) {
      const int64_t from = first + (int64_t)j;
      if (from < 0 || from >= (int64_t)a.rows) continue;
      if (a.mask_words == 0 || (mask[j / 32] >> j % 32 & 1)) use(a.tokens[from], 0);
    }
  }
  const int* entries = a.biases;
  if (a.bias_entries > 0) {
    auto within = [&](int x) { return x <= 0 ? 0u : (uint32_t)x < a.bias_entries ? (uint32_t)x : a.bias_entries; };
    const uint32_t begin = within(a.bias_offsets[s]), last = within(a.bias_offsets[s + 1]);
    entries += 2 * (uint64_t)begin;
    for (uint32_t i = tid; begin + i < last; i += kLogitThreads) {
      const int token = entries[2 * (uint64_t)i];
      const uint32_t at = (uint32_t)token - chunk0;
      if (token >= 0 && at < tokens) atomicMax(bias_entry + at, i + 1);
    }
  }
  __syncthreads();

  const float repetition = a.penalties[3 * (uint64_t)s], frequency = a.penalties[3 * (uint64_t)s + 1];
  const float presence = a.penalties[3 * (uint64_t)s + 2];
  const T* from = (const T*)a.logits + (uint64_t)row * a.input_row_stride + chunk0;
  T* to = (T*)a.out + (uint64_t)row * a.output_row_stride + chunk0;
  const uint32_t* allowed = a.allowed + (uint64_t)row * a.allowed_words + chunk0 / 32;
  auto adjust = [&](uint32_t at, float x, uint32_t bits) __attribute__((always_inline)) {
    const uint32_t u = uses[at], e = bias_entry[at];
    if (u != 0) {
      const uint32_t made = u & ~kInPrompt;
      x = x > 0.0f ? x / repetition : x * repetition;
      if (made > 0) x -= fmaf(frequency, (float)made, presence);
    }
    if (e != 0) x += __int_as_float(entries[2 * (uint64_t)(e - 1) + 1]);
    return bits & 1 ? x : -INFINITY;
  };
  for (uint32_t at = tid * kPer; at < tokens; at += kLogitThreads * kPer) {
    const uint32_t bits = a.allowed_words ? allowed[at / 32] >> at % 32 : ~0u;
    if (tokens - at >= kPer) {
      Pack x = *(const Loose*)(from + at);
#pragma unroll
      for (uint32_t k = 0; k < kPer; ++k) x[k] = (T)adjust(at + k, (float)x[k], bits >> k);
      *(Loose*)(to + at) = x;
    } else {
      for (uint32_t k = 0; at + k < tokens; ++k) to[at + k] = (T)adjust(at + k, (float)from[at + k], bits >> k);
    }
  }
}

template <typename T>
int launch_as(hipStream_t stream, const LogitArgs& a) {
  constexpr uint32_t kMostRows = 65535;  // the grid's second dimension
  for (uint64_t done = 0; done < a.rows; done += kMostRows) {
    const uint32_t rows = a.rows - done < kMostRows ? (uint32_t)(a.rows - done) : kMostRows;
    hipLaunchKernelGGL(adjust_logits_kernel<T>, dim3((uint32_t)(((uint64_t)a.columns + kChunk - 1) / kChunk), rows),
                       dim3(kLogitThreads), 0, stream, a, (uint32_t)done);
    if (int e = hip_status(hipGetLastError())) return e;
  }
  return 0;
}

}  // namespace

int launch_adjust_logits(hipStream_t stream, const LogitArgs& a) {
  if (a.rows == 0 || a.sequences == 0) return 0;
  const uintptr_t words = (uintptr_t)a.row_offsets | (uintptr_t)a.tokens | (uintptr_t)a.mask | (uintptr_t)a.history |
                          (uintptr_t)a.history_counts | (uintptr_t)a.penalties | (uintptr_t)a.bias_offsets |
                          (uintptr_t)a.biases | (uintptr_t)a.allowed;
  if (words % 4 != 0 || ((uintptr_t)a.out | (uintptr_t)a.logits) % (a.f32 ? 4 : 2) != 0)
    return IPUS_ERROR_INVALID_ARGUMENT;
  // In place only where every element is read and written by the same thread.
  if (a.out == a.logits && a.input_row_stride != a.output_row_stride) return IPUS_ERROR_INVALID_ARGUMENT;
  return a.f32 ? launch_as<float>(stream, a) : launch_as<half_t>(stream, a);
}

}  // namespace ipus
