// The paged cache and the ragged batch that the append and attention kernels
// share, and the lookups in them.
//
// Cache: fp16 [pages][2][key heads][page_rows][width], keys before values.  Row p
// of sequence s lies in page table[s][p / page_rows] at row p % page_rows.
// Batch: rows row_offsets[s] .. row_offsets[s + 1] - 1 belong to sequence s, the
// last of them at position lengths[s] - 1; rows past row_offsets[sequences] to none.
//
// The arrays are device memory that the host never reads, so the lookups hold
// for any content: a row outside every sequence, a position outside the table and a
// page outside the cache have no place.
#pragma once

#include "device_common.h"
#include "kernels.h"

namespace ipus {

inline uintptr_t batch_addresses(const PagedBatch& b) {
  return (uintptr_t)b.table | (uintptr_t)b.row_offsets | (uintptr_t)b.lengths;
}

// Page of position `position` of a sequence, -1 if it has none.
__device__ __forceinline__ int64_t page_of(const PagedBatch& b, uint32_t sequence, uint32_t position) {
  const uint32_t column = position >> b.page_shift;
  if (column >= b.table_columns) return -1;
  const uint32_t from = position < b.shared_rows ? 0 : sequence;
  const uint32_t page = (uint32_t)b.table[(uint64_t)from * b.table_columns + column];
  return page < b.pages ? (int64_t)page : -1;
}

// Sequence of row t: the number of sequences that end at or before it (sequences
// if it lies behind the last).  A wave's 64 lanes probe 64 ends at a time.
__device__ __forceinline__ uint32_t find_sequence(const PagedBatch& b, uint32_t t) {
  const uint32_t lane = threadIdx.x % kWave;
  uint32_t low = 0, left = b.sequences;
  while (left > (uint32_t)kWave) {
    const uint32_t step = (left + kWave - 1) / kWave;
    const uint32_t probe = (lane + 1) * step - 1;
    const bool ended = probe < left && (int64_t)b.row_offsets[low + probe + 1] <= (int64_t)t;
    const uint32_t past = (uint32_t)__popcll(__ballot(ended)) * step;
    low += past;
    left = left - past < step ? left - past : step;
  }
  const bool ended = lane < left && (int64_t)b.row_offsets[low + lane + 1] <= (int64_t)t;
  return low + (uint32_t)__popcll(__ballot(ended));
}

struct RowPlace {
  uint32_t sequence;
  int position;  // < 0: none
};
// Sequence and position of row t; called by a whole wave.
__device__ __forceinline__ RowPlace find_row(const PagedBatch& b, uint32_t t) {
  RowPlace p{find_sequence(b, t), -1};
  if (p.sequence >= b.sequences) return p;
  const int64_t start = b.row_offsets[p.sequence], end = b.row_offsets[p.sequence + 1];
  const int64_t position = (int64_t)b.lengths[p.sequence] - (end - (int64_t)t);
  if ((int64_t)t >= start && position >= 0 && position <= 0x7fffffff) p.position = (int)position;
  return p;
}

}  // namespace ipus
