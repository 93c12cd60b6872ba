// Wave-wide lookups in a ragged batch (page_lookup.h), shared by the append and
// attention kernels.
#pragma once

#include "device_common.h"
#include "kernels.h"

namespace ipus {

inline uintptr_t batch_addresses(const PagedBatch& b) {
  return (uintptr_t)b.table | (uintptr_t)b.row_offsets | (uintptr_t)b.lengths;
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
  uint32_t sequence;  // sequences: the row belongs to none
  int position;       // -1: none
};
// Sequence and position of row t; called by a whole wave.
__device__ __forceinline__ RowPlace find_row(const PagedBatch& b, uint32_t t) {
  RowPlace p{find_sequence(b, t), -1};
  if (p.sequence >= b.sequences) return p;
  if ((int64_t)t < (int64_t)b.row_offsets[p.sequence])
    p.sequence = b.sequences;
  else
    p.position = row_position(b.lengths[p.sequence], b.row_offsets[p.sequence + 1], t);
  return p;
}

}  // namespace ipus
