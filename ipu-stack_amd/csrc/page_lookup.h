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

// A tree of drafted tokens: the sequence's rows, and which of them each reads.  A row's
// mask says so by bit j for the j-th of them, whose key stands at position base + j;
// the keys before `base` are every row's.
struct TreeRows {
  int64_t base;   // of the first row, negative where the sequence has more rows than keys
  uint32_t bits;  // of a mask that are read: one per row, as far as the mask reaches
};
IPUS_HD TreeRows tree_rows(const PagedBatch& b, uint32_t s, uint32_t row_count, uint32_t mask_words) {
  const int64_t from = b.row_offsets[s], to = b.row_offsets[s + 1];
  const int64_t rows = to > from ? to - from : 0;
  const uint64_t most = rows < (int64_t)row_count ? (uint64_t)rows : row_count, reach = 32ull * mask_words;
  return {(int64_t)b.lengths[s] - rows, (uint32_t)(most < reach ? most : reach)};
}
// Which of the 64 keys from position `key` on a row with this mask reads: bit i for key + i.
IPUS_HD uint64_t tree_window(const uint32_t* mask, const TreeRows& t, uint32_t key) {
  const int64_t first = (int64_t)key - t.base;  // bit of the mask, negative before the rows
  if (first >= (int64_t)t.bits) return 0;
  if (first <= -64) return ~0ull;
  const uint32_t at = first > 0 ? (uint32_t)first : 0, word = at / 32, shift = at % 32;
  uint64_t x = 0;
  if (t.bits > at) {
    const uint32_t last = (t.bits - 1) / 32;
    x = mask[word];
    if (word < last) x |= (uint64_t)mask[word + 1] << 32;
    x >>= shift;
    if (shift > 0 && word + 1 < last) x |= (uint64_t)mask[word + 2] << (64 - shift);
    const uint32_t left = t.bits - at;
    if (left < 64) x &= (1ull << left) - 1;
  }
  return first >= 0 ? x : x << -first | ((1ull << -first) - 1);
}

}  // namespace ipus
