// What a decoder's step keeps in order around its paged cache (pages.h): the page tables
// as requests begin, grow, shrink and end; the step's row offsets, positions and cache
// slots; and the cache's rows of drafted tokens that were accepted, side by side again.
#include "../../include/ipus.h"
#include "kernels.h"
#include "pages.h"
#include "wave_scan.h"

namespace ipus {
namespace {

// Whether `bytes` from a on share memory with `others` from b on: none of an empty list,
// whose address may be any.
inline bool overlaps(const void* a, uint64_t bytes, const void* b, uint64_t others) {
  if (bytes == 0 || others == 0) return false;
  return (uintptr_t)a < (uintptr_t)b ? (uintptr_t)b - (uintptr_t)a < bytes : (uintptr_t)a - (uintptr_t)b < others;
}
inline int hip_status(hipError_t e) { return e == hipSuccess ? 0 : IPUS_ERROR_HIP_BASE - (int)e; }

// Sum over the threads up to this one of a workgroup of Waves waves, and of all; `waves`:
// LDS.  Called by all threads, again only after a barrier.
template <uint32_t Waves, typename T>
__device__ __forceinline__ T scan_threads(T x, T* waves, T* all) {
  const uint32_t lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  T upto = scan(x);
  if (lane == kWave - 1) waves[wave] = upto;
  __syncthreads();
  T sum = 0;
#pragma unroll
  for (uint32_t w = 0; w < Waves; ++w) {
    if (w == wave) upto += sum;
    sum += waves[w];
  }
  *all = sum;
  return upto;
}

// ---------------------------------------------------------------------------
// Page tables
// ---------------------------------------------------------------------------
// The state is int32 [free][missing][free pages: pages][held: sequences][table: sequences x
// columns].  Every workgroup works the whole step out for itself - who goes on with which row,
// what each gives back and takes, as running sums in LDS - and writes its share of the new
// state: one launch without a word between workgroups.  Entry i of the list of free pages is
// the previous list's, behind it the pages given back in the order of the previous rows;
// pages are taken from its end.
// Bound by the launch and the loads that wait for each other: 64 sequences x 256 pages 3.6 us on
// the GPU; of 512 sequences the sums alone 4.3 us (2 columns, 2000 pages), 5.7 with a word of the
// state for every thread (256 columns, 80,000 pages), 7.5 with seven (2048 columns, 624,000 pages,
// 7.7 MB): all workgroups are on the chip at once, and a thread's words behind its first take turns,
// an entry's with a division and two loads that wait for each other (its source, then the page).
// Entries and free pages are below 2^31 each (checked with the scalars), and a grid has at most
// 2^18 threads: their numbers fit 32 bits.
// The words that decide are loaded first, together, and so is what each thread will most
// likely write; all else is LDS.
constexpr uint32_t kTableThreads = 512, kTableWaves = kTableThreads / kWave;
__global__ __launch_bounds__(kTableThreads) void page_tables_kernel(PageTableArgs a) {
  extern __shared__ uint32_t lds[];
  uint32_t* const need = lds;                           // [sequences] pages
  uint32_t* const wanted = need + a.sequences;          // first the sources; then pages to take, of those up to and with
  uint32_t* const owner = wanted + a.sequences;         // [previous] the sequence that goes on with the row
  uint32_t* const back = owner + a.previous_sequences;  // first those held; then given back, of the rows up to and with
  __shared__ uint32_t waves[kTableWaves];
  const uint32_t tid = threadIdx.x;
  const int* const spare = a.previous + 2;
  const int* const held = spare + a.pages;
  const int* const old = held + a.previous_sequences;
  auto within = [](int x, uint32_t most) __attribute__((always_inline)) {
    return x <= 0 ? 0u : (uint32_t)x < most ? (uint32_t)x : most;
  };
  const uint32_t entries = a.sequences * a.columns, stride = gridDim.x * kTableThreads;
  const uint32_t i0 = blockIdx.x * kTableThreads + tid;  // this thread's first entry and free page

  const uint32_t free = within(a.previous[0], a.pages);
  const int early_spare = i0 < a.pages ? spare[i0] : -1;
  for (uint32_t p = tid; p < a.previous_sequences; p += kTableThreads) {
    owner[p] = a.sequences;
    back[p] = within(held[p], a.columns);
  }
  for (uint32_t s = tid; s < a.sequences; s += kTableThreads) {
    const int length = a.lengths[s];
    const uint32_t pages = length <= 0 ? 0 : (((uint32_t)length - 1) >> a.page_shift) + 1;
    need[s] = pages < a.columns ? pages : a.columns;
    wanted[s] = (uint32_t)a.source[s];
  }
  __syncthreads();
  int early_page = -1;
  if (i0 < entries) {
    const uint32_t s = i0 / a.columns, from = wanted[s];
    if (from < a.previous_sequences) early_page = old[(uint64_t)from * a.columns + (i0 - s * a.columns)];
  }
  for (uint32_t s = tid; s < a.sequences; s += kTableThreads) {
    const uint32_t from = wanted[s];
    if (from < a.previous_sequences) atomicMin(owner + from, s);
  }
  __syncthreads();
  uint32_t given = 0, taken = 0;  // in all
  for (uint32_t s1 = 0; s1 < a.sequences; s1 += kTableThreads) {
    const uint32_t s = s1 + tid;
    uint32_t x = 0, all;
    if (s < a.sequences) {
      const uint32_t from = wanted[s], base = from < a.previous_sequences && owner[from] == s ? back[from] : 0;
      x = need[s] > base ? need[s] - base : 0;
    }
    const uint32_t upto = taken + scan_threads<kTableWaves>(x, waves, &all);
    if (s < a.sequences) wanted[s] = upto;
    taken += all;
    __syncthreads();
  }
  for (uint32_t p0 = 0; p0 < a.previous_sequences; p0 += kTableThreads) {
    const uint32_t p = p0 + tid;
    uint32_t x = 0, all;
    if (p < a.previous_sequences) {
      const uint32_t h = back[p], o = owner[p], stay = o < a.sequences ? need[o] : 0;
      x = h > stay ? h - stay : 0;
    }
    const uint32_t upto = given + scan_threads<kTableWaves>(x, waves, &all);
    if (p < a.previous_sequences) back[p] = upto;
    given += all;
    __syncthreads();
  }
  const uint32_t total = free + given;
  const uint32_t left = total > taken ? total - taken : 0;

  auto listed_page = [&](uint32_t i) __attribute__((always_inline)) {  // i < total
    if (i < free) return spare[i];
    i -= free;
    uint32_t low = 0, count = a.previous_sequences;  // the first row with back > i
    while (count > 0) {
      const uint32_t half = count / 2;
      const bool before = back[low + half] <= i;
      low = before ? low + half + 1 : low;
      count = before ? count - half - 1 : half;
    }
    const uint32_t first = low > 0 ? back[low - 1] : 0;
    const uint32_t column = within(held[low], a.columns) - (back[low] - first) + (i - first);
    return old[(uint64_t)low * a.columns + column];
  };
  int* const out_spare = a.out + 2;
  int* const out_held = out_spare + a.pages;
  int* const out_table = out_held + a.sequences;
  for (uint32_t i = i0; i < a.pages; i += stride) {
    int page = -1;
    if (i < left) page = i == i0 && i < free ? early_spare : listed_page(i);
    out_spare[i] = page;
  }
  for (uint32_t i = i0; i < entries; i += stride) {
    const uint32_t s = i / a.columns, c = i - s * a.columns;
    const uint32_t before = s > 0 ? wanted[s - 1] : 0, kept = need[s] - (wanted[s] - before);
    int page = -1;
    if (c < kept) {
      page = i == i0 ? early_page : old[(uint64_t)(uint32_t)a.source[s] * a.columns + c];
    } else if (c < need[s]) {
      const uint32_t turn = before + (c - kept);
      if (turn < total) page = listed_page(total - 1 - turn);
    }
    out_table[i] = page;
  }
  if (blockIdx.x > 0) return;
  for (uint32_t s = tid; s < a.sequences; s += kTableThreads) {
    const uint32_t before = s > 0 ? wanted[s - 1] : 0, want = wanted[s] - before;
    const uint32_t got = total <= before ? 0 : total - before < want ? total - before : want;
    out_held[s] = (int)(need[s] - want + got);
  }
  if (tid == 0) {
    a.out[0] = (int)(left < a.pages ? left : a.pages);
    a.out[1] = (int)(taken > total ? taken - total : 0);
  }
}

// ---------------------------------------------------------------------------
// Slot maps
// ---------------------------------------------------------------------------
// A thread per row; every workgroup adds the counts up for itself, a thread per sequence at
// a time, and looks its rows up among the sums.  The first one writes the offsets too.  Bound
// by latency (count, sum, length, table entry): 64 rows 2.7 us on the GPU, 1000 trees of 64 rows 4.6.
constexpr uint32_t kSlotThreads = 512, kSlotWaves = kSlotThreads / kWave;
__global__ __launch_bounds__(kSlotThreads) void slot_maps_kernel(SlotMapArgs a, uint32_t first_block) {
  __shared__ uint32_t ends[kSlotThreads];  // of the sequences' rows, within a.rows
  __shared__ uint64_t waves[kSlotWaves];
  const uint32_t tid = threadIdx.x, block = first_block + blockIdx.x;
  const uint64_t row = (uint64_t)block * kSlotThreads + tid, last = (uint64_t)block * kSlotThreads + kSlotThreads - 1;
  uint32_t sequence = a.batch.sequences, first = 0, count = 0;
  uint64_t before = 0;
  for (uint32_t s0 = 0; s0 < a.batch.sequences; s0 += kSlotThreads) {
    const uint32_t s = s0 + tid;
    const int n = s < a.batch.sequences ? a.counts[s] : 0;
    uint64_t all;
    const uint64_t upto = before + scan_threads<kSlotWaves>((uint64_t)(n > 0 ? n : 0), waves, &all);
    const uint32_t end = upto < a.rows ? (uint32_t)upto : a.rows;
    ends[tid] = end;
    if (block == 0 && s < a.batch.sequences) a.out[1 + (uint64_t)s] = (int)end;
    __syncthreads();
    const uint32_t begin = before < a.rows ? (uint32_t)before : a.rows;
    if (row >= begin && row < ends[kSlotThreads - 1]) {
      uint32_t low = 0, span = kSlotThreads;  // the first that ends past the row
      while (span > 0) {
        const uint32_t half = span / 2;
        const bool past = ends[low + half] <= row;
        low = past ? low + half + 1 : low;
        span = past ? span - half - 1 : half;
      }
      sequence = s0 + low;
      first = low > 0 ? ends[low - 1] : begin;
      count = ends[low] - first;
    }
    before += all;
    if (block > 0 && before > last) break;
    __syncthreads();
  }
  if (block == 0 && tid == 0) a.out[0] = 0;
  if (row >= a.rows) return;
  int position = 0, slot = -1;
  if (sequence < a.batch.sequences) {
    const int64_t base = (int64_t)a.batch.lengths[sequence] - count;
    const uint32_t i = (uint32_t)row - first;
    const int64_t place = base + i;
    int64_t p = place;
    if (a.mask_words > 0) {
      const uint32_t* mask = a.mask + row * a.mask_words;
      uint32_t others = 0;
      for (uint32_t w = 0; w < a.mask_words && w * 32 < count; ++w) {
        uint32_t x = mask[w];
        if (count - w * 32 < 32) x &= (1u << (count - w * 32)) - 1;
        if (i / 32 == w) x &= ~(1u << i % 32);
        others += (uint32_t)__popc(x);
      }
      p = base + others;
    }
    position = p < 0 ? -1 : p > 0x7fffffff ? 0x7fffffff : (int)p;
    const int page = place < 0 || place > 0x7fffffff ? -1 : page_of(a.batch, sequence, (uint32_t)place);
    if (page >= 0) slot = (int)((uint64_t)page * a.batch.page_rows + ((uint32_t)place & (a.batch.page_rows - 1)));
  }
  int* const positions = a.out + 1 + (uint64_t)a.batch.sequences;
  positions[row] = position;
  positions[(uint64_t)a.rows + row] = slot;
}

// ---------------------------------------------------------------------------
// Accepted drafts
// ---------------------------------------------------------------------------
// Row path[i] of a sequence's new rows moves to row i, in the caches of all layers.  The path
// increases, so that a row is read before, or by the same entry as, it is written when entries
// go in order: a thread takes the same columns of all of them, in groups whose loads are in
// flight together.  Bound by HBM behind three loads that wait for each other (path, page, row):
// 64 sequences x up to 12 rows x 16 layers x 8 heads x 128, 52 MB, 11.3 us (4.6 TB/s; 12.4 on another
// card; sixteen rows in flight 11.2, but 7.0 against 6.3 for paths of up to 4 in 32 layers).
constexpr uint32_t kKeepThreads = 256, kKeepEntries = 64, kKeepAtOnce = 8;
template <int V>
__global__ __launch_bounds__(kKeepThreads) void keep_pages_kernel(KeepArgs a, uint32_t first_sequence) {
  typedef half_t Pack __attribute__((ext_vector_type(V)));
  __shared__ uint64_t from[kKeepEntries], to[kKeepEntries];  // elements of a layer's cache
  __shared__ uint32_t usable;
  const uint32_t s = first_sequence + blockIdx.x, tid = threadIdx.x, layer = blockIdx.z;
  const BatchSequence q = sequence_at(a.batch, s, a.rows);
  const int64_t begin = a.batch.row_offsets[s], rows = (int64_t)a.batch.row_offsets[s + 1] - begin;
  const int64_t base = (int64_t)q.length - rows;
  const int counted = a.path_counts[s];
  const uint32_t entries = counted <= 0 ? 0 : (uint32_t)counted < a.path_columns ? (uint32_t)counted : a.path_columns;
  const int* const path = a.path + (uint64_t)s * a.path_columns;
  const uint32_t unit = blockIdx.y * kKeepThreads + tid, chunks = a.width / V;
  const uint32_t units = 2 * a.key_heads * chunks, head = unit / chunks;
  half_t* const mine = (half_t*)a.caches + (uint64_t)layer * a.batch.pages * a.batch.page_elements +
                       (uint64_t)head * a.batch.page_rows * a.width + (unit - head * chunks) * V;
  for (uint32_t i0 = 0; i0 < entries; i0 += kKeepEntries) {
    // Entries up to the first that is not past the one before, or not a row.
    if (tid < kKeepEntries) {
      const uint32_t i = i0 + tid;
      const int row = i < entries ? path[i] : -1, previous = i > 0 && i < entries ? path[i - 1] : -1;
      const uint64_t bad = __ballot(!(row > previous && row < rows && begin + row >= 0 && begin + row < (int64_t)a.rows));
      if (tid == 0) usable = bad ? (uint32_t)__builtin_ctzll(bad) : kKeepEntries;
      auto element = [&](int64_t position) __attribute__((always_inline)) {
        if (position < 0 || position >= (int64_t)q.keys) return ~0ull;
        const int page = page_of(a.batch, s, (uint32_t)position);
        return page < 0 ? ~0ull
                        : (uint64_t)page * a.batch.page_elements + (uint64_t)((uint32_t)position & (a.batch.page_rows - 1)) * a.width;
      };
      from[tid] = row == (int)i ? ~0ull : element(base + row);
      to[tid] = element(base + i);
    }
    __syncthreads();
    const uint32_t count = usable;
    if (unit < units) {
      for (uint32_t e = 0; e < count; e += kKeepAtOnce) {
        Pack x[kKeepAtOnce];
#pragma unroll
        for (uint32_t k = 0; k < kKeepAtOnce; ++k)
          if (e + k < count && from[e + k] != ~0ull && to[e + k] != ~0ull) x[k] = *(const Pack*)(mine + from[e + k]);
#pragma unroll
        for (uint32_t k = 0; k < kKeepAtOnce; ++k)
          if (e + k < count && from[e + k] != ~0ull && to[e + k] != ~0ull) *(Pack*)(mine + to[e + k]) = x[k];
      }
    }
    if (count < kKeepEntries) break;
    __syncthreads();
  }
}

}  // namespace

int launch_page_tables(hipStream_t stream, const PageTableArgs& a) {
  if (((uintptr_t)a.out | (uintptr_t)a.previous | (uintptr_t)a.source | (uintptr_t)a.lengths) % 4 != 0)
    return IPUS_ERROR_INVALID_ARGUMENT;
  // The inputs are read while the new state is written.
  const uint64_t rows = 1 + (uint64_t)a.columns, bytes = 4 * (2 + a.pages + a.sequences * rows);
  if (overlaps(a.out, bytes, a.previous, 4 * (2 + a.pages + a.previous_sequences * rows)) ||
      overlaps(a.out, bytes, a.source, 4ull * a.sequences) || overlaps(a.out, bytes, a.lengths, 4ull * a.sequences))
    return IPUS_ERROR_INVALID_ARGUMENT;
  // A word per thread, up to two workgroups per CU, whose own sums then take longer than the
  // words of another (us, a word per thread / four: 64 sequences x 256 pages 4.2 / 5.0; 2000 x 500
  // pages 12.0 of 512 workgroups, 12.2 of 1024, 14.5 of 256).
  constexpr uint64_t kEach = kTableThreads, kMostGroups = 512;
  uint64_t groups = (a.pages + a.sequences * rows + kEach - 1) / kEach;
  groups = groups < 1 ? 1 : groups > kMostGroups ? kMostGroups : groups;
  const uint32_t lds = 8 * (a.sequences + a.previous_sequences);
  hipLaunchKernelGGL(page_tables_kernel, dim3((uint32_t)groups), dim3(kTableThreads), lds, stream, a);
  return hip_status(hipGetLastError());
}

int launch_slot_maps(hipStream_t stream, const SlotMapArgs& a) {
  if ((batch_addresses(a.batch) | (uintptr_t)a.counts | (uintptr_t)a.mask | (uintptr_t)a.out) % 4 != 0)
    return IPUS_ERROR_INVALID_ARGUMENT;
  const uint64_t sequences = a.batch.sequences, bytes = 4 * (sequences + 1 + 2ull * a.rows);
  if (overlaps(a.out, bytes, a.counts, 4 * sequences) || overlaps(a.out, bytes, a.batch.lengths, 4 * sequences) ||
      overlaps(a.out, bytes, a.batch.table, 4 * sequences * a.batch.table_columns) ||
      overlaps(a.out, bytes, a.mask, 4ull * a.rows * a.mask_words))
    return IPUS_ERROR_INVALID_ARGUMENT;
  constexpr uint64_t kMostBlocks = 1u << 22;  // a grid dimension holds less than 2^32 threads
  const uint64_t blocks = a.rows == 0 ? 1 : ((uint64_t)a.rows + kSlotThreads - 1) / kSlotThreads;
  for (uint64_t done = 0; done < blocks; done += kMostBlocks) {
    const uint32_t some = blocks - done < kMostBlocks ? (uint32_t)(blocks - done) : (uint32_t)kMostBlocks;
    hipLaunchKernelGGL(slot_maps_kernel, dim3(some), dim3(kSlotThreads), 0, stream, a, (uint32_t)done);
    if (int e = hip_status(hipGetLastError())) return e;
  }
  return 0;
}

namespace {
template <int V>
int launch_keep_as(hipStream_t stream, const KeepArgs& a) {
  const uint64_t across = (2ull * a.key_heads * (a.width / V) + kKeepThreads - 1) / kKeepThreads;
  if (across > 65535 || a.layers > 65535) return IPUS_ERROR_UNAVAILABLE;  // the grid's other dimensions
  constexpr uint32_t kMostSequences = 1u << 23;
  for (uint64_t done = 0; done < a.batch.sequences; done += kMostSequences) {
    const uint64_t left = a.batch.sequences - done;
    hipLaunchKernelGGL(keep_pages_kernel<V>, dim3((uint32_t)(left < kMostSequences ? left : kMostSequences), (uint32_t)across, a.layers),
                       dim3(kKeepThreads), 0, stream, a, (uint32_t)done);
    if (int e = hip_status(hipGetLastError())) return e;
  }
  return 0;
}
}  // namespace

int launch_keep_pages(hipStream_t stream, const KeepArgs& a) {
  if (a.batch.sequences == 0 || a.layers == 0 || a.path_columns == 0 || a.rows == 0) return 0;
  if ((uintptr_t)a.caches % 2 != 0 || (batch_addresses(a.batch) | (uintptr_t)a.path | (uintptr_t)a.path_counts) % 4 != 0)
    return IPUS_ERROR_INVALID_ARGUMENT;
  const uintptr_t at = (uintptr_t)a.caches;
  if (a.width % 8 == 0 && at % 16 == 0) return launch_keep_as<8>(stream, a);
  if (a.width % 4 == 0 && at % 8 == 0) return launch_keep_as<4>(stream, a);
  if (a.width % 2 == 0 && at % 4 == 0) return launch_keep_as<2>(stream, a);
  return launch_keep_as<1>(stream, a);
}

}  // namespace ipus
