// Penalties for repeated tokens, biases and masks on the logits of a step's rows:
//   x' = x / r (x > 0) or x r (else) of a token that stands in the sequence's history or
//        the row's path, then x' - (f g + p [g > 0]) with g its uses behind the prompt,
//   then x' + its bias, and -inf for a token that the row's mask does not allow.
// The path of a row is the rows of its sequence that its mask names, or those up to itself.
// Bound by HBM, the logits once in, once out, where there are rows enough: 64 trees of 8 to 16 rows
// x 131072 fp32 behind 8192 tokens with 300 biases and masks 143 us, 5.8 TB/s, fp16 80 us, 5.1;
// by latency where there are few (64 single rows x 50001 fp16 6.9 us, 13 MB).
#include "attention_pages.h"

namespace ipus {
namespace {

// Two kernels: for single rows of many sequences (a token each), where the launch and the loads
// that wait for each other count, and for several rows of a sequence.
//
// Both: a workgroup takes a chunk of the tokens.  How often each of them stands in the history
// is counted in LDS (integers: any order gives the same).
constexpr uint32_t kLogitThreads = 512, kChunk = 4096;
// A token's word: its uses behind the prompt, and whether it stands in the prompt, has a bias,
// or stands in some row's path.
constexpr uint32_t kInPrompt = 1u << 31, kBiased = 1u << 30, kInPath = 1u << 29, kUses = kInPath - 1;

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
struct LogitPacks {
  static constexpr uint32_t kPer = 16 / sizeof(T), kPacks = kChunk / (kLogitThreads * kPer);
  typedef T Pack __attribute__((ext_vector_type(kPer)));
  typedef Pack Loose __attribute__((aligned(sizeof(T))));  // rows of any alignment
  static __device__ __forceinline__ uint32_t place(uint32_t i) { return (i * kLogitThreads + threadIdx.x) * kPer; }
  // This thread's packs of a row's chunk, and the words of the row's mask that hold their bits.
  Pack x[kPacks];
  uint32_t bits[kPacks];
  __device__ __forceinline__ void load(const LogitArgs& a, uint32_t row, uint32_t chunk0, uint32_t tokens) {
    const T* from = (const T*)a.logits + (uint64_t)row * a.input_row_stride + chunk0;
    const uint32_t* allowed = a.allowed + (uint64_t)row * a.allowed_words + chunk0 / 32;
#pragma unroll
    for (uint32_t i = 0; i < kPacks; ++i) {
      const uint32_t at = place(i);
      bits[i] = ~0u;
      if (at < tokens && a.allowed_words) bits[i] = allowed[at / 32];
      if (at + kPer <= tokens) {
        x[i] = __builtin_nontemporal_load((const Loose*)(from + at));
      } else {
#pragma unroll
        for (uint32_t k = 0; k < kPer; ++k)
          if (at + k < tokens) x[i][k] = from[at + k];
      }
    }
  }
  __device__ __forceinline__ void store(const LogitArgs& a, uint32_t row, uint32_t chunk0, uint32_t tokens) {
    T* to = (T*)a.out + (uint64_t)row * a.output_row_stride + chunk0;
#pragma unroll
    for (uint32_t i = 0; i < kPacks; ++i) {
      const uint32_t at = place(i), allowed = bits[i] >> at % 32;
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
};
struct Penalties {
  float repetition, frequency, presence;
  __device__ __forceinline__ bool any() const { return !(repetition == 1.0f && frequency == 0.0f && presence == 0.0f); }
  __device__ __forceinline__ float operator()(float y, uint32_t word) const {
    if (word & (kInPrompt | kUses)) {
      y = y > 0.0f ? y / repetition : y * repetition;
      if (word & kUses) y -= fmaf(frequency, (float)(word & kUses), presence);
    }
    return y;
  }
};
__device__ __forceinline__ Penalties penalties_of(const LogitArgs& a, uint32_t s) {
  const float* p = a.penalties + 3 * (uint64_t)s;
  return {p[0], p[1], p[2]};
}
// Entries [begin, end) of the biases are sequence s's.
struct BiasRange {
  uint32_t begin, end;
};
__device__ __forceinline__ BiasRange biases_of(const LogitArgs& a, uint32_t s) {
  if (a.bias_entries == 0) return {0, 0};
  auto within = [&](int t) { return t <= 0 ? 0u : (uint32_t)t < a.bias_entries ? (uint32_t)t : a.bias_entries; };
  return {within(a.bias_offsets[s]), within(a.bias_offsets[s + 1])};
}
// Marks the history of sequence s in a chunk's words.
__device__ __forceinline__ void mark_history(const LogitArgs& a, uint32_t s, uint32_t* words, uint32_t chunk0, uint32_t tokens) {
  typedef int Four __attribute__((ext_vector_type(4)));
  typedef Four LooseFour __attribute__((aligned(4)));
  if (a.history_columns == 0) return;
  const int* history = a.history + (uint64_t)s * a.history_columns;
  auto fetch = [&](uint32_t i) __attribute__((always_inline)) {
    Four t = {-1, -1, -1, -1};
    if (i + 4 <= a.history_columns)
      t = *(const LooseFour*)(history + i);
    else
      for (uint32_t k = 0; i + k < a.history_columns; ++k) t[k] = history[i + k];
    return t;
  };
  // The first tokens are asked for beside the counts that say how many of them there are (256 rows
  // x 32000 behind 4000 tokens 17.4 us, after them 18.0).
  Four t = fetch(4 * threadIdx.x);
  const int given = a.history_counts[2 * (uint64_t)s], known = a.history_counts[2 * (uint64_t)s + 1];
  const uint32_t total = known <= 0 ? 0 : (uint32_t)known < a.history_columns ? (uint32_t)known : a.history_columns;
  const uint32_t prompt = given <= 0 ? 0 : (uint32_t)given < total ? (uint32_t)given : total;
  for (uint32_t i = 4 * threadIdx.x; i < total;) {
#pragma unroll
    for (uint32_t k = 0; k < 4; ++k)
      if (i + k < total && t[k] >= 0 && (uint32_t)t[k] - chunk0 < tokens) {
        uint32_t* const word = words + ((uint32_t)t[k] - chunk0);
        i + k < prompt ? atomicOr(word, kInPrompt) : atomicAdd(word, 1u);
      }
    i += 4 * kLogitThreads;
    if (i < total) t = fetch(i);
  }
}

// A row's logits are on their way while its history is counted, and adjusted in registers.
// They are asked for behind what the counting waits for: loads arrive in order.
template <typename T>
__global__ __launch_bounds__(kLogitThreads, 8) void adjust_row_kernel(LogitArgs a, uint32_t first_row) {
  using P = LogitPacks<T>;
  __shared__ __attribute__((aligned(16))) uint32_t words[kChunk];
  __shared__ __attribute__((aligned(16))) uint32_t entry[kChunk];  // a biased token's 1 + last entry
  const uint32_t chunk0 = blockIdx.x * kChunk, row = first_row + blockIdx.y, tid = threadIdx.x;
  const uint32_t tokens = a.columns - chunk0 < kChunk ? a.columns - chunk0 : kChunk;
  P p;
  PagedBatch b{};
  b.row_offsets = a.row_offsets;
  b.sequences = a.sequences;
  const uint32_t s = uniform(find_sequence(b, row));
  if (s >= a.sequences) return;
  const LogitRows all = logit_rows(a, s);
  if (row < all.first) return;
  const Penalties penalties = penalties_of(a, s);
  const BiasRange biases = biases_of(a, s);
  p.load(a, row, chunk0, tokens);
  for (uint32_t i = tid; i < kChunk / 4; i += kLogitThreads) {
    *reinterpret_cast<u32x4*>(words + 4 * i) = u32x4{0, 0, 0, 0};
    if (biases.begin < biases.end) *reinterpret_cast<u32x4*>(entry + 4 * i) = u32x4{0, 0, 0, 0};
  }
  __syncthreads();
  auto inside = [&](int t) __attribute__((always_inline)) { return t >= 0 && (uint32_t)t - chunk0 < tokens; };
  if (penalties.any()) {
    mark_history(a, s, words, chunk0, tokens);
    for (uint32_t j = tid; j < all.rows; j += kLogitThreads) {
      const bool stands = a.mask_words == 0 ? j <= row - all.first
                                            : j / 32 < a.mask_words && (a.mask[(uint64_t)row * a.mask_words + j / 32] >> j % 32 & 1);
      const int t = stands ? a.tokens[all.first + j] : -1;
      if (inside(t)) atomicAdd(words + ((uint32_t)t - chunk0), 1u);
    }
  }
  for (uint32_t i = biases.begin + tid; i < biases.end; i += kLogitThreads) {
    const int t = a.biases[2 * (uint64_t)i];
    if (inside(t)) {
      atomicOr(words + ((uint32_t)t - chunk0), kBiased);
      atomicMax(entry + ((uint32_t)t - chunk0), 1 + i);
    }
  }
  __syncthreads();
#pragma unroll
  for (uint32_t i = 0; i < P::kPacks; ++i) {
    const uint32_t at = P::place(i);
    uint32_t word[P::kPer], any = 0;
#pragma unroll
    for (uint32_t k = 0; k < P::kPer; k += 4) {
      const u32x4 w = *reinterpret_cast<const u32x4*>(words + at + k);
#pragma unroll
      for (uint32_t e = 0; e < 4; ++e) {
        word[k + e] = w[e];
        any |= w[e];
      }
    }
    if (any == 0) continue;
#pragma unroll
    for (uint32_t k = 0; k < P::kPer; ++k)
      if (word[k] != 0) {
        float y = penalties((float)p.x[i][k], word[k]);
        if (word[k] & kBiased) y += __int_as_float(a.biases[2 * (uint64_t)(entry[at + k] - 1) + 1]);
        p.x[i][k] = (T)y;
      }
  }
  p.store(a, row, chunk0, tokens);
}

// A workgroup takes up to `group` rows of a sequence, one after the other, and counts the history
// once for them; the few tokens that anything changes are listed.  A row's logits pass from registers through LDS back to registers, where
// between two barriers the listed ones are adjusted, a thread each: a test of every token in
// its registers costs more, since most waves hold a listed one.  The next row's logits and mask
// words are on their way meanwhile.
template <typename T>
__global__ __launch_bounds__(kLogitThreads, 8) void adjust_rows_kernel(LogitArgs a, uint32_t first_unit, uint32_t group) {
  using P = LogitPacks<T>;
  constexpr uint32_t kSlots = kChunk / kLogitThreads;  // of the list, per thread
  __shared__ __attribute__((aligned(16))) uint32_t words[kChunk];
  // A row's logits; before the first row a biased token's 1 + last entry.
  __shared__ __attribute__((aligned(16))) uint32_t stage[kChunk];
  __shared__ __attribute__((aligned(16))) uint16_t list[kChunk];  // before it is written, the waves' counts of it
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
  const uint32_t ahead = (unit - (uint32_t)found.first) * group;
  if (ahead >= all.rows) return;  // offsets that change meanwhile
  const uint32_t row0 = all.first + ahead, left = all.rows - ahead, rows = left < group ? left : group;

  P next;
  uint32_t next_path = 0;
  auto load = [&](uint32_t row) __attribute__((always_inline)) {
    next.load(a, row, chunk0, tokens);
    if (tid < all.rows && tid / 32 < a.mask_words) next_path = a.mask[(uint64_t)row * a.mask_words + tid / 32];
  };
  load(row0);
  const Penalties penalties = penalties_of(a, s);
  const BiasRange biases = biases_of(a, s);
  const uint32_t begin = biases.begin, end = biases.end;
  const bool penal = penalties.any();
  auto inside = [&](int t) __attribute__((always_inline)) { return t >= 0 && (uint32_t)t - chunk0 < tokens; };
  const int token = tid < all.rows ? a.tokens[all.first + tid] : -1;  // of the sequence's row `tid`

  // ---- the tokens of the history, the paths and the biases ----
  for (uint32_t i = tid; i < kChunk / 4; i += kLogitThreads) {
    *reinterpret_cast<u32x4*>(words + 4 * i) = u32x4{0, 0, 0, 0};
    if (begin < end) *reinterpret_cast<u32x4*>(stage + 4 * i) = u32x4{0, 0, 0, 0};
  }
  __syncthreads();
  if (penal) {
    mark_history(a, s, words, chunk0, tokens);
    if (inside(token)) atomicOr(words + (token - chunk0), kInPath);
    for (uint32_t j = tid + kLogitThreads; j < all.rows; j += kLogitThreads) {
      const int t = a.tokens[all.first + j];
      if (inside(t)) atomicOr(words + (t - chunk0), kInPath);
    }
  }
  for (uint32_t i = begin + tid; i < end; i += kLogitThreads) {
    const int t = a.biases[2 * (uint64_t)i];
    if (inside(t)) {
      atomicOr(words + (t - chunk0), kBiased);
      atomicMax(stage + (t - chunk0), 1 + i);
    }
  }
  __syncthreads();
  // The list.
  uint32_t count = 0;
  {
    uint32_t mine = 0;
    u32x4 w[kSlots / 4];
#pragma unroll
    for (uint32_t q = 0; q < kSlots / 4; ++q) {
      w[q] = *reinterpret_cast<const u32x4*>(words + 4 * (q * kLogitThreads + tid));
#pragma unroll
      for (uint32_t k = 0; k < 4; ++k) mine += w[q][k] != 0;
    }
    const uint32_t upto = scan(mine), wave = tid / kWave;
    uint32_t* const counts = reinterpret_cast<uint32_t*>(list);
    if (tid % kWave == kWave - 1) counts[wave] = upto;
    __syncthreads();
    uint32_t at = upto - mine;
#pragma unroll
    for (uint32_t v = 0; v < kLogitThreads / kWave; ++v) {
      if (v == wave) at += count;
      count += counts[v];
    }
    count = uniform(count);
    __syncthreads();
#pragma unroll
    for (uint32_t q = 0; q < kSlots / 4; ++q)
#pragma unroll
      for (uint32_t k = 0; k < 4; ++k)
        if (w[q][k] != 0) list[at++] = (uint16_t)(4 * (q * kLogitThreads + tid) + k);
  }
  if (count > 0) __syncthreads();
  float value[kSlots];  // biases of this thread's listed tokens
#pragma unroll
  for (uint32_t u = 0; u < kSlots; ++u) {
    value[u] = 0.0f;
    const uint32_t e = u * kLogitThreads + tid;
    if (begin < end && e < count && (words[list[e]] & kBiased))
      value[u] = __int_as_float(a.biases[2 * (uint64_t)(stage[list[e]] - 1) + 1]);
  }
  if (begin < end && count > 0) __syncthreads();

  T* const logits = reinterpret_cast<T*>(stage);
  uint32_t before = 0;  // whether this thread's token stood in the path of the row before
  for (uint32_t r = 0; r < rows; ++r) {
    const uint32_t row = row0 + r, path = next_path;
    P p = next;
    if (r + 1 < rows) load(row + 1);
    if (count > 0) {
#pragma unroll
      for (uint32_t i = 0; i < P::kPacks; ++i) *reinterpret_cast<typename P::Pack*>(logits + P::place(i)) = p.x[i];
      if (penal) {
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
      __syncthreads();
#pragma unroll
      for (uint32_t u = 0; u < kSlots; ++u) {
        if (u * kLogitThreads >= count) break;
        const uint32_t e = u * kLogitThreads + tid;
        if (e >= count) break;
        const uint32_t at = list[e], word = words[at];
        float y = penalties((float)logits[at], word);
        if (word & kBiased) y += value[u];
        logits[at] = (T)y;
      }
      __syncthreads();
#pragma unroll
      for (uint32_t i = 0; i < P::kPacks; ++i) p.x[i] = *reinterpret_cast<const typename P::Pack*>(logits + P::place(i));
    }
    p.store(a, row, chunk0, tokens);
  }
}

// Several rows per workgroup where sequences have them and there are enough for two rounds of the
// workgroups that the chip holds (four per CU), but not so many that the last round is long (us,
// 64 trees of 8 to 16 rows x 131072: fp32 3 / 4 / 6 / 8 rows 145 / 146 / 151 / 155, fp16 8 / 12 / 16
// rows 81 / 83 / 83).
template <typename T>
int launch_as(hipStream_t stream, const LogitArgs& a) {
  constexpr uint64_t kWant = 2 * 4 * 256, kMostUnits = 65535;  // the grid's second dimension
  constexpr uint64_t kMostGroup = sizeof(T) == 4 ? 4 : 8;
  const uint64_t chunks = ((uint64_t)a.columns + kChunk - 1) / kChunk;
  uint64_t group = a.rows * chunks / kWant;
  group = group < 1 || a.rows <= a.sequences ? 1 : group > kMostGroup ? kMostGroup : group;
  // At most a partial group more for each sequence.
  uint64_t units = group == 1 ? a.rows : a.rows / group + a.sequences;
  if (units > a.rows) units = a.rows;
  for (uint64_t done = 0; done < units; done += kMostUnits) {
    const dim3 grid((uint32_t)chunks, (uint32_t)(units - done < kMostUnits ? units - done : kMostUnits));
    if (group == 1)
      hipLaunchKernelGGL(adjust_row_kernel<T>, grid, dim3(kLogitThreads), 0, stream, a, (uint32_t)done);
    else
      hipLaunchKernelGGL(adjust_rows_kernel<T>, grid, dim3(kLogitThreads), 0, stream, a, (uint32_t)done, (uint32_t)group);
    if (int e = hip_status(hipGetLastError())) return e;
  }
  return 0;
}

// Rows of `bytes` each, `stride` apart (at least their bytes).
struct RowSpan {
  uint64_t at, stride, rows, bytes;
  uint64_t end() const { return at + (rows - 1) * stride + bytes; }
  // Whether one of them shares memory with `count` bytes from `from` on.
  bool meets(uint64_t from, uint64_t count) const {
    if (count == 0 || from + count <= at || from >= end()) return false;
    uint64_t row = (from + count - 1 - at) / stride;  // the last that begins before their end
    if (row >= rows) row = rows - 1;
    return at + row * stride + bytes > from;
  }
  bool meets(const RowSpan& other) const {
    if (other.end() <= at || other.at >= end()) return false;
    // With one stride a pair's distance goes by its rows' difference alone: pairs with the first or the
    // last row are all that there are.
    const uint64_t step = stride == other.stride && other.rows > 1 ? other.rows - 1 : 1;
    for (uint64_t r = 0; r < other.rows; r += step)
      if (meets(other.at + r * other.stride, other.bytes)) return true;
    return false;
  }
};
// Whether the output shares memory with an input other than row by row, in place: workgroups
// read the lists, and rows ahead of the one that they write, while others write.  Where the tokens'
// list begins at the logits' own address, all are taken for placeholders, of a launch that is
// only looked at.
bool races(const LogitArgs& a) {
  if ((const void*)a.tokens == a.logits) return a.out == a.logits && a.input_row_stride != a.output_row_stride;
  const uint64_t element = a.f32 ? 4 : 2, sequences = a.sequences, rows = a.rows;
  const RowSpan out{(uintptr_t)a.out, a.output_row_stride * element, rows, a.columns * element};
  const RowSpan in{(uintptr_t)a.logits, a.input_row_stride * element, rows, a.columns * element};
  if (!(out.at == in.at && out.stride == in.stride) && out.meets(in)) return true;
  auto over = [&](const void* list, uint64_t bytes) { return out.meets((uintptr_t)list, bytes); };
  return over(a.row_offsets, 4 * (sequences + 1)) || over(a.tokens, 4 * rows) || over(a.penalties, 12 * sequences) ||
         over(a.mask, 4 * rows * a.mask_words) || over(a.history, 4 * sequences * a.history_columns) ||
         (a.history_columns && over(a.history_counts, 8 * sequences)) ||
         (a.bias_entries && over(a.bias_offsets, 4 * (sequences + 1))) || over(a.biases, 8ull * a.bias_entries) ||
         over(a.allowed, 4 * rows * a.allowed_words);
}

}  // namespace

int launch_adjust_logits(hipStream_t stream, const LogitArgs& a) {
  if (a.rows == 0 || a.sequences == 0) return 0;
  const uintptr_t words = (uintptr_t)a.row_offsets | (uintptr_t)a.tokens | (uintptr_t)a.mask | (uintptr_t)a.history |
                          (uintptr_t)a.history_counts | (uintptr_t)a.penalties | (uintptr_t)a.bias_offsets |
                          (uintptr_t)a.biases | (uintptr_t)a.allowed;
  if (words % 4 != 0 || ((uintptr_t)a.out | (uintptr_t)a.logits) % (a.f32 ? 4 : 2) != 0)
    return IPUS_ERROR_INVALID_ARGUMENT;
  // In place every element is read and written by the same thread.
  if (races(a)) return IPUS_ERROR_INVALID_ARGUMENT;
  return a.f32 ? launch_as<float>(stream, a) : launch_as<half_t>(stream, a);
}

}  // namespace ipus
