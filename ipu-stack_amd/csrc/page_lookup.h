// The ragged batch and the paged cache as the kernels see them: the arrays are
// device memory that the host never reads, so every lookup holds for any content.
// A row outside every sequence, a position outside the table and a page outside
// the cache have no place.  Also compiled for the host, by the tests.
#pragma once

#include <stdint.h>

#include "layout_maps.h"

namespace ipus {

// A ragged batch over a paged cache.
//
// Cache: fp16 [pages][2][key heads][page_rows][width], keys before values.  Row p
// of sequence s lies in page table[s][p / page_rows] at row p % page_rows.
// Batch: rows row_offsets[s] .. row_offsets[s + 1] - 1 belong to sequence s, the
// last of them at position lengths[s] - 1; rows past row_offsets[sequences] to none.
struct PagedBatch {
  const int* table;        // [sequences][table_columns]
  const int* row_offsets;  // [sequences + 1]
  const int* lengths;      // [sequences]
  uint32_t sequences, table_columns, pages, page_rows, page_shift;
  uint32_t shared_rows = 0;  // positions that every sequence reads through the first one's table
  uint64_t page_elements;    // 2 x key heads x page_rows x width
};

// Page of position `position` of a sequence, -1 if it has none.
IPUS_HD int page_of(const PagedBatch& b, uint32_t sequence, uint32_t position) {
  const uint32_t column = position >> b.page_shift;
  if (column >= b.table_columns) return -1;
  const uint32_t from = position < b.shared_rows ? 0 : sequence;
  const uint32_t page = (uint32_t)b.table[(uint64_t)from * b.table_columns + column];
  return page < b.pages && page <= 0x7fffffffu ? (int)page : -1;
}

// Rows and keys of a sequence: rows first .. first + rows - 1 of the batch's
// row_count (offsets outside it are cut off), keys [0, keys) that its table reaches,
// and its length and the end of its rows as given.
struct BatchSequence {
  uint32_t first, rows, keys;
  int length, end;
};
IPUS_HD BatchSequence sequence_at(const PagedBatch& b, uint32_t s, uint32_t row_count) {
  const int64_t from = b.row_offsets[s], to = b.row_offsets[s + 1];
  BatchSequence q;
  const int64_t first = from < 0 ? 0 : from > (int64_t)row_count ? (int64_t)row_count : from;
  const int64_t last = to > (int64_t)row_count ? (int64_t)row_count : to;
  q.first = (uint32_t)first;
  q.rows = last > first ? (uint32_t)(last - first) : 0;
  q.length = b.lengths[s];
  q.end = (int)to;
  const uint64_t reach = (uint64_t)b.table_columns * b.page_rows;
  q.keys = q.length <= 0 ? 0 : (uint64_t)q.length < reach ? (uint32_t)q.length : (uint32_t)reach;
  return q;
}

// Position of row t of a sequence whose rows end at `end`: its length less the
// rows from t on; -1 where that is negative.
IPUS_HD int row_position(int length, int end, uint32_t t) {
  const int64_t p = (int64_t)length - ((int64_t)end - (int64_t)t);
  return p >= 0 && p <= 0x7fffffff ? (int)p : -1;
}

// Keys that a row at `position` may read of a sequence: [0, count).
IPUS_HD uint32_t readable_keys(const BatchSequence& q, int position, bool causal) {
  if (!causal) return q.keys;
  const uint32_t upto = (uint32_t)(position + 1);  // -1: none
  return upto < q.keys ? upto : q.keys;
}

}  // namespace ipus
