// Penalties for repeated tokens, biases and masks on the logits of a step's rows:
//   x' = x / r (x > 0) or x r (else) of a token that stands in the sequence's history or
//        the row's path, then x' - (f g + p [g > 0]) with g its uses behind the prompt,
//   then x' + its bias, and -inf for a token that the row's mask does not allow.
// The path of a row is the rows of its sequence that its mask names, or those up to itself.
// Bound by HBM: the logits once in, once out.
#include "attention_pages.h"

namespace ipus {
namespace {

// A workgroup takes a chunk of the tokens and up to `group` rows of a sequence, one after the
// other.  How often each token of the chunk stands in the history is counted in LDS, once for
// these rows (integers: any order gives the same); each row's path is added to that and taken
// off again.  The next row's logits and mask words are on their way while this one's are
// adjusted.
constexpr uint32_t kLogitThreads = 512, kChunk = 4096;
// A token's word: its uses behind the prompt, whether it stands in the prompt, and whether it
// has a bias.
constexpr uint32_t kInPrompt = 1u << 31, kBiased = 1u << 30, kUses = kBiased - 1;
// Rows [first, first + rows) of sequence s, offsets outside the rows cut off.
struct LogitRows {
  uint32_t first, rows;
};
__device__ __forceinline__ LogitRows logit_rows(const LogitArgs& a, uint32_t s) {
  const int64_t from = a.row_offsets[s], to = a.row_offsets[s + 1], most = a.rows;
  const int64_t first = from < 0 ? 0 : from > most ? most : from, last = to > most ? most : to;
  return {(uint32_t)first, last > first ? (uint32_t)(last - first) : 0};
}
template <typename T>
__global__ __launch_bounds__(kLogitThreads, 8) void adjust_logits_kernel(LogitArgs a, uint32_t first_unit, uint32_t group) {
  constexpr uint32_t kPer = 16 / sizeof(T), kPacks = kChunk / (kLogitThreads * kPer);
  typedef T Pack __attribute__((ext_vector_type(kPer)));
  typedef Pack Loose __attribute__((aligned(sizeof(T))));  // rows of any alignment
  typedef int Four __attribute__((ext_vector_type(4)));
  typedef Four LooseFour __attribute__((aligned(4)));
  __shared__ __attribute__((aligned(16))) uint32_t words[kChunk];
  // A biased token's 1 + last entry, then that entry's value.
  __shared__ __attribute__((aligned(16))) uint32_t bias[kChunk];
  const uint32_t chunk0 = blockIdx.x * kChunk, tid = threadIdx.x;
  const uint32_t tokens = a.columns - chunk0 < kChunk ? a.columns - chunk0 : kChunk;

  // ---- the sequence and its rows ----
  PagedBatch b{};
  b.sequences = a.sequences;
  auto units = [&](uint32_t s) __attribute__((always_inline)) { return (uint64_t)((logit_rows(a, s).rows + group - 1) / group); };
  const UnitLine line = count_units(b, units);
  const uint32_t unit = first_unit + blockIdx.y;
  if (unit >= line.total) return;
  const UnitPlace found = find_unit(b, line, unit, units);
  const uint32_t s = uniform(found.sequence);
  if (s >= a.sequences) return;
  const LogitRows all = logit_rows(a, s);
  const uint32_t row0 = all.first + (unit - (uint32_t)found.first) * group, left = all.first + all.rows - row0;
  const uint32_t rows = left < group ? left : group;

  // Pack i of a thread: the tokens from place(i) on.
  auto place = [&](uint32_t i) __attribute__((always_inline)) { return (i * kLogitThreads + tid) * kPer; };
  Pack next[kPacks];
  uint32_t next_bits[kPacks], next_path = 0;
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
    if (tid < all.rows && tid / 32 < a.mask_words) next_path = a.mask[(uint64_t)row * a.mask_words + tid / 32];
  };
  load(row0);
  const float repetition = a.penalties[3 * (uint64_t)s], frequency = a.penalties[3 * (uint64_t)s + 1];
  const float presence = a.penalties[3 * (uint64_t)s + 2], inverse = 1.0f / repetition;
  const bool penal = !(repetition == 1.0f && frequency == 0.0f && presence == 0.0f);
  auto inside = [&](int t) __attribute__((always_inline)) { return t >= 0 && (uint32_t)t - chunk0 < tokens; };
  const int token = tid < all.rows ? a.tokens[all.first + tid] : -1;  // of the sequence's row `tid`
  uint32_t begin = 0, end = 0;                                       // biases
  if (a.bias_entries > 0) {
    auto within = [&](int t) { return t <= 0 ? 0u : (uint32_t)t < a.bias_entries ? (uint32_t)t : a.bias_entries; };
    begin = within(a.bias_offsets[s]);
    end = within(a.bias_offsets[s + 1]);
  }

  // ---- the history's tokens, and the biases' ----
  for (uint32_t i = tid; i < kChunk / 4; i += kLogitThreads) {
    *reinterpret_cast<u32x4*>(words + 4 * i) = u32x4{0, 0, 0, 0};
    if (begin < end) *reinterpret_cast<u32x4*>(bias + 4 * i) = u32x4{0, 0, 0, 0};
  }
  __syncthreads();
  if (penal && a.history_columns > 0) {
    const int given = a.history_counts[2 * (uint64_t)s], known = a.history_counts[2 * (uint64_t)s + 1];
    const uint32_t total = known <= 0 ? 0 : (uint32_t)known < a.history_columns ? (uint32_t)known : a.history_columns;
    const uint32_t prompt = given <= 0 ? 0 : (uint32_t)given < total ? (uint32_t)given : total;
    const int* history = a.history + (uint64_t)s * a.history_columns;
    auto use = [&](int t, bool in_prompt) __attribute__((always_inline)) {
      if (inside(t)) in_prompt ? atomicOr(words + (t - chunk0), kInPrompt) : atomicAdd(words + (t - chunk0), 1u);
    };
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
  // A token's last entry is found by its number, then its value put in its place: 32 entries
  // of a thread at a time, from the end of the list, so that later ones are there already.
  for (uint32_t upto = end; upto > begin;) {
    constexpr uint32_t kAtOnce = 32 * kLogitThreads;
    const uint32_t from = upto - begin > kAtOnce ? upto - kAtOnce : begin;
    uint32_t lasts = 0;
    auto over = [&](auto f) __attribute__((always_inline)) {
      for (uint32_t k = 0; k < 32 && from + k * kLogitThreads + tid < upto; ++k) {
        const int t = a.biases[2 * (uint64_t)(from + k * kLogitThreads + tid)];
        if (inside(t)) f(k, (uint32_t)t - chunk0);
      }
    };
    over([&](uint32_t k, uint32_t at) __attribute__((always_inline)) {
      if (!(words[at] & kBiased)) {
        lasts |= 1u << k;
        atomicMax(bias + at, 1 + k * kLogitThreads + tid);
      }
    });
    __syncthreads();
    over([&](uint32_t k, uint32_t at) __attribute__((always_inline)) {
      if (bias[at] != 1 + k * kLogitThreads + tid) lasts &= ~(1u << k);
    });
    __syncthreads();
    over([&](uint32_t k, uint32_t at) __attribute__((always_inline)) {
      if (lasts >> k & 1) {
        bias[at] = (uint32_t)a.biases[2 * (uint64_t)(from + k * kLogitThreads + tid) + 1];
        atomicOr(words + at, kBiased);
      }
    });
    upto = from;
    if (upto > begin) __syncthreads();
  }

  uint32_t before = 0;  // whether this thread's token stood in the path of the row before
  for (uint32_t r = 0; r < rows; ++r) {
    const uint32_t row = row0 + r, path = next_path;
    Pack x[kPacks];
    uint32_t bits[kPacks];
#pragma unroll
    for (uint32_t i = 0; i < kPacks; ++i) {
      x[i] = next[i];
      bits[i] = next_bits[i];
    }
    if (r + 1 < rows) load(row + 1);
    if (penal) {
      if (r > 0) __syncthreads();  // the row before has read its words
      // This row's path on, the last one's off.
      const uint32_t index = row - all.first;
      const uint32_t mine = inside(token) && (a.mask_words ? path >> tid % 32 & 1 : tid <= index);
      if (mine != before) mine ? atomicAdd(words + (token - chunk0), 1u) : atomicSub(words + (token - chunk0), 1u);
      before = mine;
      for (uint32_t j = tid + kLogitThreads; j < all.rows; j += kLogitThreads) {  // long paths
        auto stands = [&](uint32_t i) __attribute__((always_inline)) {
          if (a.mask_words == 0) return j <= i;
          return j / 32 < a.mask_words && (a.mask[(uint64_t)(all.first + i) * a.mask_words + j / 32] >> j % 32 & 1) != 0;
        };
        const bool now = stands(index), was = r > 0 && stands(index - 1);
        if (now == was) continue;
        const int t = a.tokens[all.first + j];
        if (inside(t)) now ? atomicAdd(words + (t - chunk0), 1u) : atomicSub(words + (t - chunk0), 1u);
      }
    }
    if (penal || r == 0) __syncthreads();

    auto adjust = [&](float y, uint32_t word, uint32_t at) __attribute__((always_inline)) {
      const uint32_t uses = word & kUses;
      if (word & ~kBiased) {
        // y / repetition, rounded once: the quotient by the inverse, and what it leaves.
        const float quotient = y * inverse, rest = fmaf(-quotient, repetition, y), better = fmaf(rest, inverse, quotient);
        const float less = fabsf(better) < INFINITY ? better : y / repetition;
        y = y > 0.0f ? less : y * repetition;
        if (uses > 0) y -= fmaf(frequency, (float)uses, presence);
      }
      if (word & kBiased) y += __uint_as_float(bias[at]);
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

// Rows of a workgroup: all of a sequence's, as far as that leaves two rounds of the workgroups
// that the chip holds (four per CU).
template <typename T>
int launch_as(hipStream_t stream, const LogitArgs& a) {
  constexpr uint64_t kWant = 2 * 4 * 256, kMostUnits = 65535;  // the grid's second dimension
  const uint64_t chunks = ((uint64_t)a.columns + kChunk - 1) / kChunk;
  uint64_t group = a.rows * chunks / kWant;
  group = group < 1 ? 1 : group > 64 ? 64 : group;
  if (a.sequences * chunks >= kWant) group = 64;
  // At most a partial group more for each sequence.
  uint64_t units = a.rows / group + a.sequences;
  if (units > a.rows) units = a.rows;
  for (uint64_t done = 0; done < units; done += kMostUnits) {
    hipLaunchKernelGGL(adjust_logits_kernel<T>, dim3((uint32_t)chunks, (uint32_t)(units - done < kMostUnits ? units - done : kMostUnits)),
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
