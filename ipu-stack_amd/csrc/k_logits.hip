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

// A workgroup takes a chunk of the tokens, and a few rows one after the other.  How often each
// token of the chunk stands in the history is counted in LDS, once for the rows of a sequence
// (integers: any order gives the same); each row's path is added to that and taken off again.
// The next row's logits, mask words and path are on their way while this one's are adjusted.
constexpr uint32_t kLogitThreads = 256, kLogitWaves = kLogitThreads / kWave, kChunk = 4096, kMostGroup = 16;
// A token's word: its uses behind the prompt, whether it stands in the prompt, and whether it
// has a bias.
constexpr uint32_t kInPrompt = 1u << 31, kBiased = 1u << 30, kUses = kBiased - 1;
template <typename T>
__global__ __launch_bounds__(kLogitThreads) void adjust_logits_kernel(LogitArgs a, uint32_t first_row, uint32_t group) {
  constexpr uint32_t kPer = 16 / sizeof(T), kPacks = kChunk / (kLogitThreads * kPer);
  typedef T Pack __attribute__((ext_vector_type(kPer)));
  typedef Pack Loose __attribute__((aligned(sizeof(T))));  // rows of any alignment
  __shared__ __attribute__((aligned(16))) uint32_t words[kChunk];
  __shared__ uint32_t bias_entry[kChunk];  // 1 + the last entry of the token, 0: none
  __shared__ uint32_t row_sequence[kMostGroup];
  const uint32_t row0 = first_row + blockIdx.y * group, chunk0 = blockIdx.x * kChunk;
  const uint32_t tid = threadIdx.x, wave = tid / kWave;
  const uint32_t rows = a.rows - row0 < group ? a.rows - row0 : group;
  const uint32_t tokens = a.columns - chunk0 < kChunk ? a.columns - chunk0 : kChunk;
  PagedBatch b{};
  b.row_offsets = a.row_offsets;
  b.sequences = a.sequences;
  for (uint32_t r = wave; r < rows; r += kLogitWaves) {
    const uint32_t s = find_sequence(b, row0 + r);
    if (tid % kWave == 0)
      row_sequence[r] = s < a.sequences && (int64_t)a.row_offsets[s] <= (int64_t)(row0 + r) ? s : a.sequences;
  }
  // Pack i of a thread: tokens from 16 bytes of it on; the mask's bits of these.
  auto place = [&](uint32_t i) __attribute__((always_inline)) { return (i * kLogitThreads + tid) * kPer; };
  Pack next[kPacks];
  uint32_t next_bits[kPacks];
  auto load = [&](uint32_t row) __attribute__((always_inline)) {
    const T* from = (const T*)a.logits + (uint64_t)row * a.input_row_stride + chunk0;
    const uint32_t* allowed = a.allowed + (uint64_t)row * a.allowed_words + chunk0 / 32;
#pragma unroll
    for (uint32_t i = 0; i < kPacks; ++i) {
      const uint32_t at = place(i);
      next_bits[i] = ~0u;
      if (at < tokens && a.allowed_words) next_bits[i] = allowed[at / 32];
      if (at + kPer <= tokens) {
        next[i] = __builtin_nontemporal_load((const Loose*)(from + at));
      } else {
#pragma unroll
        for (uint32_t k = 0; k < kPer; ++k)
          if (at + k < tokens) next[i][k] = from[at + k];
      }
    }
  };
  load(row0);
  __syncthreads();

  uint32_t held = a.sequences;  // the sequence whose history the words hold
  const int* entries = a.biases;
  float repetition = 1.0f, inverse = 1.0f, frequency = 0.0f, presence = 0.0f;
  bool penal = false;
  int64_t first = 0, end = 0;
  int token = -1;                 // of the sequence's row `tid`
  uint32_t mine = 0, before = 0;  // this thread's part of the path: in this row, in the one before
  auto inside = [&](int t) __attribute__((always_inline)) { return t >= 0 && (uint32_t)t - chunk0 < tokens; };
  auto path_at = [&](uint32_t row, uint64_t j) __attribute__((always_inline)) {
    if (a.mask_words == 0) return (int64_t)j <= (int64_t)row - first;
    return j / 32 < a.mask_words && (a.mask[(uint64_t)row * a.mask_words + j / 32] >> j % 32 & 1) != 0;
  };
  auto token_at = [&](uint64_t j) __attribute__((always_inline)) {
    const int64_t from = first + (int64_t)j;
    return from < end && from >= 0 && from < (int64_t)a.rows ? a.tokens[from] : -1;
  };
  for (uint32_t r = 0; r < rows; ++r) {
    const uint32_t row = row0 + r, s = uniform(row_sequence[r]);
    Pack x[kPacks];
    uint32_t bits[kPacks];
#pragma unroll
    for (uint32_t i = 0; i < kPacks; ++i) {
      x[i] = next[i];
      bits[i] = next_bits[i];
    }
    if (r + 1 < rows) load(row + 1);
    if (s >= a.sequences) continue;
    if (s != held) {
      held = s;
      before = 0;
      first = a.row_offsets[s];
      end = a.row_offsets[s + 1];
      repetition = a.penalties[3 * (uint64_t)s];
      frequency = a.penalties[3 * (uint64_t)s + 1];
      presence = a.penalties[3 * (uint64_t)s + 2];
      inverse = 1.0f / repetition;
      penal = !(repetition == 1.0f && frequency == 0.0f && presence == 0.0f);
      if (r > 0) __syncthreads();  // the row before has read its words
      for (uint32_t i = tid; i < kChunk / 4; i += kLogitThreads)
        *reinterpret_cast<u32x4*>(words + 4 * i) = u32x4{0, 0, 0, 0};
      if (a.bias_entries > 0)
        for (uint32_t i = tid; i < kChunk; i += kLogitThreads) bias_entry[i] = 0;
      token = token_at(tid);
      __syncthreads();
      if (penal && a.history_columns > 0) {
        const int given = a.history_counts[2 * (uint64_t)s], all = a.history_counts[2 * (uint64_t)s + 1];
        const uint32_t total = all <= 0 ? 0 : (uint32_t)all < a.history_columns ? (uint32_t)all : a.history_columns;
        const uint32_t prompt = given <= 0 ? 0 : (uint32_t)given < total ? (uint32_t)given : total;
        const int* history = a.history + (uint64_t)s * a.history_columns;
        auto use = [&](int t, bool in_prompt) __attribute__((always_inline)) {
          if (inside(t)) in_prompt ? atomicOr(words + (t - chunk0), kInPrompt) : atomicAdd(words + (t - chunk0), 1u);
        };
        typedef int Four __attribute__((ext_vector_type(4)));
        typedef Four LooseFour __attribute__((aligned(4)));
        for (uint32_t i = 4 * tid; i < total; i += 4 * kLogitThreads) {
          if (total - i >= 4) {
            const Four t = *(const LooseFour*)(history + i);
#pragma unroll
            for (uint32_t k = 0; k < 4; ++k) use(t[k], i + k < prompt);
          } else {
            for (uint32_t k = 0; i + k < total; ++k) use(history[i + k], i + k < prompt);
          }
        }
      }
      if (a.bias_entries > 0) {
        auto within = [&](int t) { return t <= 0 ? 0u : (uint32_t)t < a.bias_entries ? (uint32_t)t : a.bias_entries; };
        const uint32_t begin = within(a.bias_offsets[s]), last = within(a.bias_offsets[s + 1]);
        entries = a.biases + 2 * (uint64_t)begin;
        for (uint32_t i = tid; begin + i < last; i += kLogitThreads) {
          const int t = entries[2 * (uint64_t)i];
          if (inside(t)) {
            atomicMax(bias_entry + (t - chunk0), i + 1);
            atomicOr(words + (t - chunk0), kBiased);
          }
        }
      }
    } else {
      __syncthreads();  // the row before has read its words
    }
    if (penal) {
      // This row's path on, the last one's off.
      mine = path_at(row, tid) && inside(token);
      if (mine != before) mine ? atomicAdd(words + (token - chunk0), 1u) : atomicSub(words + (token - chunk0), 1u);
      before = mine;
      for (uint64_t j = tid + kLogitThreads; (int64_t)j < end - first; j += kLogitThreads) {  // long paths
        const bool now = path_at(row, j), was = r > 0 && row_sequence[r - 1] == s && path_at(row - 1, j);
        if (now == was) continue;
        const int t = token_at(j);
        if (inside(t)) now ? atomicAdd(words + (t - chunk0), 1u) : atomicSub(words + (t - chunk0), 1u);
      }
    }
    __syncthreads();

    auto adjust = [&](float y, uint32_t word, uint32_t at) __attribute__((always_inline)) {
      const uint32_t uses = word & kUses;
      if (word & ~kBiased) {
        // y / repetition, rounded once: the quotient by the inverse, and what it leaves.
        const float quotient = y * inverse, left = fmaf(-quotient, repetition, y), better = fmaf(left, inverse, quotient);
        const float less = fabsf(better) < INFINITY ? better : y / repetition;
        y = y > 0.0f ? less : y * repetition;
        if (uses > 0) y -= fmaf(frequency, (float)uses, presence);
      }
      if (word & kBiased) y += __int_as_float(entries[2 * (uint64_t)(bias_entry[at] - 1) + 1]);
      return y;
    };
    T* to = (T*)a.out + (uint64_t)row * a.output_row_stride + chunk0;
#pragma unroll
    for (uint32_t i = 0; i < kPacks; ++i) {
      const uint32_t at = place(i);
      if (at >= tokens) continue;
      uint32_t word[kPer], any = 0;
#pragma unroll
      for (uint32_t k = 0; k < kPer; k += 4) {
        const u32x4 w = *reinterpret_cast<const u32x4*>(words + at + k);
#pragma unroll
        for (uint32_t e = 0; e < 4; ++e) {
          word[k + e] = w[e];
          any |= w[e];
        }
      }
      if (any) {
#pragma unroll
        for (uint32_t k = 0; k < kPer; ++k)
          if (word[k]) x[i][k] = (T)adjust((float)x[i][k], word[k], at + k);
      }
      const uint32_t allowed = bits[i] >> at % 32;
#pragma unroll
      for (uint32_t k = 0; k < kPer; ++k) x[i][k] = allowed >> k & 1 ? x[i][k] : (T)-INFINITY;
      if (at + kPer <= tokens) {
        __builtin_nontemporal_store(x[i], (Loose*)(to + at));
      } else {
#pragma unroll
        for (uint32_t k = 0; k < kPer; ++k)
          if (at + k < tokens) to[at + k] = x[i][k];
      }
    }
  }
}

// Rows of a workgroup: as many as leave two rounds of the workgroups that the chip holds (five
// per CU, by LDS); rows of one sequence then count its history once.
template <typename T>
int launch_as(hipStream_t stream, const LogitArgs& a) {
  constexpr uint64_t kWant = 2 * 5 * 256, kMostGroups = 65535;  // the grid's second dimension
  const uint64_t chunks = ((uint64_t)a.columns + kChunk - 1) / kChunk;
  uint64_t group = a.rows * chunks / kWant;
  group = group < 1 ? 1 : group > kMostGroup ? kMostGroup : group;
  for (uint64_t done = 0; done < a.rows; done += kMostGroups * group) {
    const uint64_t groups = (a.rows - done + group - 1) / group;
    hipLaunchKernelGGL(adjust_logits_kernel<T>, dim3((uint32_t)chunks, (uint32_t)(groups < kMostGroups ? groups : kMostGroups)),
                       dim3(kLogitThreads), 0, stream, a, (uint32_t)done, (uint32_t)group);
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
