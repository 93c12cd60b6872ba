// Attention over a paged cache (pages.h) for many query rows per key head: chunks of
// prompts, and the rows of a whole batch over the keys that it shares.  Bound by the
// matrix pipes and the softmax beside them.
//
// A sequence's rows times the query heads of one key head are packed into blocks of
// 64 QT queries; a workgroup of 4 waves takes one block of one key head, a wave 16 QT
// queries of it.  The key loop is the one of k_attention.hip: blocks of 64 keys (32 at 256
// columns) by LDS DMA into two stages, S^T = K Q^T of block j and O^T += V^T P^T of
// block j - 1 as one MFMA cluster, the softmax of block j behind it, a reference point
// that moves only when a block's probabilities pass 2^8 against it.  Keys and values lie
// in pages: a lane holds the page of one of the block's rows, loaded two blocks
// ahead, and every DMA takes its row's page from the lane that has it.  Probabilities are
// rounded to one fp16 value (2^-11) for the second product, and row sums taken in fp32 of what
// it sees: a second value for what the first loses would be a half more MFMAs where those bound
// (4 x 2048 rows against 8192 keys 1304 us against 955, 5 x 796 rows 39.9 against 31.6; trees, which
// wait for HBM too, 8 to 25% more: 16 of 64 rows against 8192 keys 229 us against 186, 64 of 8 to 16
// against 256 to 4096 121 against 106, 7 of 50 to 99 against up to 3001 (16 heads of 72 columns) 27.3
// against 23.1).  Against float64 trees' results are off by 2.6e-4 to 2.9e-4 of their size so (root
// mean square), where their own rounding to fp16 alone makes 2.1e-4.
//
// A workgroup finds its block by a scan over the sequences; workgroups of one XCD
// take a contiguous range of blocks, the query blocks of one (sequence, key head)
// together, the longest first, so that its keys and values stay in that XCD's L2.
// Where the blocks are too few for the chip, each one's keys are split over several
// workgroups, whose parts a second launch joins: the parts are 128 rows each, and joined
// in the same launch they would go past the XCD's L2 (about 2 us per MB) to one workgroup
// per block (333 rows x 16 heads x 72 columns against 2800 keys, 16 MB of parts: 62 us
// for blocks and join, 28 in two launches).
//
// Measured, causal, 64-row pages (TFLOP/s of the products that the mask leaves): 32 query heads
// on 8 x 128: 4 x 2048 rows against 8192 keys 945 to 960 us, 1000 to 1020; a prompt of 16384
// 1030, of 4096 880, of 512 18.7 us; 64 columns 830, 96 910, 256 580 (one tile of queries
// per wave: four accumulators of 256 columns do not fit beside two).
#include "attention_pages.h"

namespace ipus {
namespace {

constexpr float kSumLimit = 256.0f;  // as in k_attention.hip
// A reference point is a score's product with scale_log2, rounded; the probabilities are
// taken from the products unrounded, by one FMA.  From this point on (log2 units) the rounding
// alone could make the largest of them overflow or vanish: there they are taken from
// rounded products, block by block.
constexpr float kFarPoint = 1 << 24;

typedef _Float16 half2_t __attribute__((ext_vector_type(2)));

// Split keys: unnormalised rows [rows * query_heads][parts][width] fp32, their
// (reference point, sum) pairs, and how many parts a row has (unless all have `parts`).
struct SplitKeys {
  float* rows;
  float* sums;
  uint32_t* counts;
  uint32_t parts;  // at most; 1: not split
};
constexpr uint32_t kMaxSplits = 16;
// Key blocks from which they are split, and of a part at least.  The parts' rows and the
// second launch cost what 8 to 16 key blocks take (128 columns, 32 query heads, us split /
// whole: 512 rows against 1024 keys 37.2 / 28.9, against 2048 40.4 / 49.1, 128 against 4096
// 36.9 / 88.8; 256 columns, 16 heads: 512 against 512 (16 blocks) 26.8 / 22.2, against 1024
// 31.3 / 36.6).  Where the table cannot hold so many keys there is no second launch either
// (512 rows against 512 keys 18.7, with both 28.8).
constexpr uint32_t kLeastSplit = 17, kLeastPart = 4;

template <int D, int QT>
struct Block {
  static constexpr uint32_t kKeys = D > 128 ? 32 : 64;
  static constexpr uint32_t kQueriesPerWave = 16 * QT, kQueries = kWaves * kQueriesPerWave;
  static constexpr uint32_t kRowBytes = D * 2, kTile = kKeys * kRowBytes;
  static constexpr uint32_t kDma = kTile / 16 / kThreads;     // DMA instructions per thread and tile
  static constexpr uint32_t kDmaRows = kThreads / (D / 8);    // rows per DMA instruction
};

// K tile rows, as value_swizzle: read with ds_read_b128, 16 rows of one chunk.
template <int D>
__device__ __forceinline__ uint32_t key_swizzle(uint32_t row) {
  return D >= 128 ? (row & 15u) : (row & 7u);
}

// Query blocks of all key heads of a sequence; none if it has so few queries that
// the other kernel takes it.
template <uint32_t Queries>
__device__ __forceinline__ uint64_t blocks_of(const BatchSequence& q, uint32_t group, uint32_t key_heads, uint32_t few) {
  const uint32_t queries = q.rows * group;  // launch_attention_pages
  return queries <= few ? 0 : (uint64_t)((queries + Queries - 1) / Queries) * key_heads;
}

// A tree's rows all read their sequence's keys, and a batch's sequences may be of very different
// lengths: the key blocks of a part at most, by all of them, so that the work is even.  Costs
// in key blocks: of as many parts as the chip holds workgroups, the longest; of twice as many,
// which follow one another, an even share and the longest; the join, where there are parts.
// Parts of fewer than kTreePart cost more than they save.  us, 32 query heads on 8 x 128, so /
// by the rule of the other rows: 64 trees of 8 to 16 rows against 256 to 4096 keys 101 / 118, 40
// of 12 to 24 against up to 3000 (96 columns) 47 / 77, 16 of 64 against 8192 186 / 198; where
// no part is of use the join's launch is lost, 20 of 64 against 2000 77 / 74.
constexpr uint32_t kJoinBlocks = 8, kTreePart = 12, kPlannedSequences = 256;
struct TreeWork {
  uint32_t blocks, key_blocks;  // query blocks of all key heads of a sequence, key blocks of each
  __device__ __forceinline__ uint32_t parts(uint32_t each) const {
    return key_blocks < kLeastSplit || each >= key_blocks ? 1 : (key_blocks + each - 1) / each;
  }
};
// held: of the first 64 sequences, one per lane.
template <typename F>
__device__ __forceinline__ uint32_t tree_part(const PagedBatch& b, uint32_t most_parts, const TreeWork& held, F work) {
  const uint32_t lane = threadIdx.x % kWave;
  uint64_t steps = (uint64_t)held.blocks * held.key_blocks, total = held.blocks;
  uint32_t longest = held.blocks > 0 ? held.key_blocks : 0;
  for (uint32_t s = kWave + lane; s < b.sequences; s += kWave) {
    const TreeWork w = work(s);
    steps += (uint64_t)w.blocks * w.key_blocks;
    total += w.blocks;
    if (w.blocks > 0 && w.key_blocks > longest) longest = w.key_blocks;
  }
  longest = largest(longest);
  total = from_lane(scan(total), kWave - 1);
  if (most_parts <= 1 || longest < kLeastSplit || total > 2 * kFullChip || b.sequences > kPlannedSequences) return longest;
  const uint32_t share = (uint32_t)((from_lane(scan(steps), kWave - 1) + kFullChip - 1) / kFullChip);
  uint32_t least = (longest + most_parts - 1) / most_parts;
  if (least < kTreePart) least = kTreePart;
  auto smallest = [&](uint32_t room) __attribute__((always_inline)) {  // of which there are at most `room`
    uint32_t low = least, high = longest;
    while (low < high) {
      const uint32_t each = (low + high) / 2;
      uint32_t items = held.blocks * held.parts(each);
      for (uint32_t s = kWave + lane; s < b.sequences; s += kWave) {
        const TreeWork w = work(s);
        items += w.blocks * w.parts(each);
      }
      if ((uint32_t)__builtin_amdgcn_readlane(scan(items), kWave - 1) <= room)
        high = each;
      else
        low = each + 1;
    }
    return low;
  };
  uint32_t best = longest, cost = total <= kFullChip ? longest : share + longest;
  if (total <= kFullChip) {
    const uint32_t each = smallest(kFullChip);
    if (each + kJoinBlocks < cost) {
      best = each;
      cost = each + kJoinBlocks;
    }
  }
  if (share + least + kJoinBlocks >= cost) return best;
  const uint32_t each = smallest(2 * kFullChip);
  return share + each + kJoinBlocks < cost ? each : best;
}

// Shared: the rows of the whole batch over the keys below shared_rows, as parts for
// another launch.  Tree: the masks of a sequence's rows, looked up for the key blocks that hold
// their keys.
template <int D, int DC, int QT, bool Shared, bool Tree>
__global__ __launch_bounds__(kThreads, 2) void attention_blocks_kernel(PagedAttentionArgs a, float scale_log2,
                                                                       uint32_t few, SplitKeys split) {
  using F = Block<D, QT>;
  constexpr uint32_t kKeys = F::kKeys, kTile = F::kTile, kRowBytes = F::kRowBytes;
  constexpr uint32_t kQPW = F::kQueriesPerWave, kQueries = F::kQueries;
  constexpr uint32_t kKT = kKeys / 16, kHalves = kKeys / 32, kKS = DC / 32, kDT = DC / 16;
  constexpr uint32_t kScoreGroups = kKT * kKS, kOutGroups = kHalves * kDT;
  constexpr uint32_t kPairs = kScoreGroups > kOutGroups ? kScoreGroups : kOutGroups;
  __shared__ __attribute__((aligned(1024))) uint8_t lds_k0[kTile];
  __shared__ __attribute__((aligned(1024))) uint8_t lds_v0[kTile];
  __shared__ __attribute__((aligned(1024))) uint8_t lds_k1[kTile];
  __shared__ __attribute__((aligned(1024))) uint8_t lds_v1[kTile];
  __shared__ uint32_t wave_word[kWaves];

  const uint32_t lane = threadIdx.x % kWave, r16 = lane % 16, g4 = lane / 16;
  const uint32_t wave = uniform(threadIdx.x / kWave);
  const uint32_t group = a.query_heads / a.key_heads;
  const PagedBatch& b = a.batch;

  // ---- this workgroup's block: sequence s, key head, queries from query0 on ----
  uint32_t s = 0, key_head;
  uint32_t query0;
  BatchSequence q{0, a.rows, 0, 0, 0};  // Shared: all rows
  uint32_t queries;                   // of the sequence
  uint64_t block;                     // in the line of all blocks
  uint32_t part, splits = split.parts;
  if constexpr (Tree) {
    auto work = [&](uint32_t x) __attribute__((always_inline)) {
      const BatchSequence w = sequence_at(b, x, a.rows);
      return TreeWork{(uint32_t)blocks_of<kQueries>(w, group, a.key_heads, few), (w.keys + kKeys - 1) / kKeys};
    };
    const TreeWork held = lane < b.sequences ? work(lane) : TreeWork{0, 0};
    const uint32_t each = tree_part(b, split.parts, held, work);
    auto items_in = [&](uint32_t x) __attribute__((always_inline)) {
      const TreeWork w = work(x);
      return (uint64_t)w.blocks * w.parts(each);
    };
    UnitLine line{scan((uint64_t)held.blocks * held.parts(each)), 0};
    line.total = from_lane(line.upto, kWave - 1);
    if (b.sequences > (uint32_t)kWave) line = count_units(b, items_in);
    // An XCD's range of the line: what reads the same keys stands together.
    const uint64_t per_xcd = (line.total + 7) / 8, local = blockIdx.x / 8, item = blockIdx.x % 8 * per_xcd + local;
    if (local >= per_xcd || item >= line.total || item >= gridDim.x) return;
    const UnitPlace place = find_unit(b, line, item, items_in);
    s = place.sequence;
    q = uniform(sequence_at(b, s, a.rows));
    queries = q.rows * group;
    const uint32_t per_head = (queries + kQueries - 1) / kQueries, within = (uint32_t)(item - place.first);
    splits = work(s).parts(each);
    const uint32_t keys_of = within / per_head;  // of one key head and part
    key_head = keys_of / splits;
    part = keys_of - key_head * splits;
    query0 = (within - keys_of * per_head) * kQueries;
  } else {
    auto blocks_in = [&](uint32_t x) __attribute__((always_inline)) {
      return blocks_of<kQueries>(sequence_at(b, x, a.rows), group, a.key_heads, few);
    };
    UnitLine line{0, blocks_of<kQueries>(q, group, a.key_heads, 0)};
    if (!Shared) line = count_units(b, blocks_in);
    const uint64_t total = line.total;
    if (total == 0) return;
    // Parts of the keys where the blocks are fewer than half of the workgroups that
    // the chip holds at once.
    if (!Shared) {
      const uint32_t want = total < kFullChip / 2 ? kFullChip / (uint32_t)total : 1;
      splits = want < split.parts ? want : split.parts;
    }
    // An XCD's range of the line, all blocks' first parts first: of blocks with fewer keys
    // the other parts have nothing to do, and workgroups at a fixed distance meet on the same
    // CUs (64 blocks of 8 possible parts, one in use: 41.5 us, so 29).
    const uint64_t items = total * splits, per_xcd = (items + 7) / 8;
    uint64_t local = blockIdx.x / 8;
    if (!Shared && splits > 1) {
      const uint32_t across = (uint32_t)quotient(per_xcd + splits - 1, splits);
      const uint32_t turn = (uint32_t)local / across;
      local = turn < splits ? (uint64_t)((uint32_t)local - turn * across) * splits + turn : per_xcd;
    }
    const uint64_t item = blockIdx.x % 8 * per_xcd + local;
    block = quotient(item, splits);
    part = (uint32_t)(item - block * splits);
    // Offsets that decrease can make more blocks than the host expects (and has memory
    // for the parts of); what lies past the grid is not computed.
    if (local >= per_xcd || item >= items || item >= gridDim.x) return;
    uint64_t within = block;
    if (!Shared) {
      const UnitPlace place = find_unit(b, line, block, blocks_in);
      s = place.sequence;
      within -= place.first;
      q = uniform(sequence_at(b, s, a.rows));
    }
    queries = q.rows * group;
    const uint32_t per_head = (queries + kQueries - 1) / kQueries;
    key_head = (uint32_t)within / per_head;
    query0 = (per_head - 1 - (uint32_t)within % per_head) * kQueries;  // the longest first
  }

  // ---- the wave's queries ----
  // Fragment (qt, ks) holds columns 32 ks + 8 (l / 16) .. + 7 of query 16 qt + l % 16;
  // queries past the last repeat it, with no key to read.
  half8_t qf[QT][kKS];
  uint32_t limit[QT];         // keys that this lane's query may read
  uint32_t least = 0xffffffffu;
  const uint32_t wave0 = query0 + wave * kQPW;
#pragma unroll
  for (uint32_t qt = 0; qt < QT; ++qt) {
    uint32_t m = wave0 + 16 * qt + r16;
    const bool real = m < queries;
    m = real ? m : queries - 1;
    const uint32_t row = q.first + m / group, head = m % group;
    const half_t* from = (const half_t*)a.query + (uint64_t)row * a.query_row_stride +
                         (uint64_t)(key_head * group + head) * a.width;
    BatchSequence mine = q;
    bool inside = real;
    if (Shared) {
      // The row's sequence: the number that end at or before it.
      uint32_t low = 0, left = b.sequences;
      while (left > 0) {
        const uint32_t half = left / 2;
        const bool past = (int64_t)b.row_offsets[low + half + 1] <= (int64_t)row;
        low = past ? low + half + 1 : low;
        left = past ? left - half - 1 : half;
      }
      inside = real && low < b.sequences;
      mine = inside ? sequence_at(b, low, a.rows) : BatchSequence{};
      inside = inside && row >= mine.first && row - mine.first < mine.rows;
      mine.keys = mine.keys < b.shared_rows ? mine.keys : b.shared_rows;
    }
    const int position = row_position(mine.length, mine.end, row);
    limit[qt] = inside ? readable_keys(mine, position, a.causal) : 0;
    if (inside && limit[qt] < least) least = limit[qt];  // what the others compute is not used
#pragma unroll
    for (uint32_t ks = 0; ks < kKS; ++ks) {
      const uint32_t d0 = ks * 32 + g4 * 8;
      qf[qt][ks] = __builtin_bit_cast(half8_t, d0 < a.width ? load16(from + d0) : u32x4{0, 0, 0, 0});
    }
  }
  for (uint32_t o = 32; o > 0; o >>= 1) {
    const uint32_t x = __shfl_xor(least, o, kWave);
    least = x < least ? x : least;
  }
  const TreeRows tree = Tree ? tree_rows(b, s, a.rows, a.mask_words) : TreeRows{0, 0};
  if (Tree) least = tree.base <= 0 ? 0 : tree.base < (int64_t)q.keys ? (uint32_t)tree.base : q.keys;
  least = uniform(least);  // every query of the wave reads the keys below it
  if (lane == 0) wave_word[wave] = least;
  __syncthreads();
  uint32_t block_least = wave_word[0];  // every query of the workgroup
#pragma unroll
  for (uint32_t w = 1; w < kWaves; ++w) block_least = wave_word[w] < block_least ? wave_word[w] : block_least;
  block_least = uniform(block_least);

  // Keys of the block: those of its last query (Shared: all of the shared ones; the host
  // has checked that the table reaches them).
  uint32_t key_end;
  if (Shared) {
    const uint64_t reach = (uint64_t)b.table_columns * b.page_rows;
    key_end = b.shared_rows < reach ? b.shared_rows : (uint32_t)reach;
  } else {
    const uint32_t last = query0 + kQueries < queries ? query0 + kQueries - 1 : queries - 1;
    const uint32_t row = q.first + last / group;
    key_end = readable_keys(q, row_position(q.length, q.end, row), a.causal);
  }
  // This part's: every part has a block of keys, but for the first of none at all.
  const uint32_t all_blocks = (key_end + kKeys - 1) / kKeys;
  uint32_t per_part = (all_blocks + splits - 1) / splits;
  if (!Shared && !Tree && splits > 1 && per_part < kLeastPart) per_part = kLeastPart;
  if (!Shared && !Tree && all_blocks < kLeastSplit) per_part = all_blocks;
  if (per_part == 0) per_part = 1;
  uint32_t parts = (all_blocks + per_part - 1) / per_part;
  if (parts == 0) parts = 1;
  if (part >= parts) return;
  const uint32_t block0 = part * per_part;
  const uint32_t nblocks = all_blocks - block0 < per_part ? all_blocks - block0 : per_part;

  float4_t o[kDT][QT];
  float m_run[QT], l_run[QT];  // reference points (log2 units), this lane's share of the row sums
  float near[QT];              // -m_run, or infinity, with which no block is accepted
  half8_t pp[kHalves][QT];     // fp16 probabilities of the last softmax
#pragma unroll
  for (uint32_t qt = 0; qt < QT; ++qt) {
    m_run[qt] = -INFINITY;
    l_run[qt] = 0.0f;
    near[qt] = INFINITY;
#pragma unroll
    for (uint32_t dt = 0; dt < kDT; ++dt) o[dt][qt] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (uint32_t kk = 0; kk < kHalves; ++kk)
#pragma unroll
      for (int e = 0; e < 8; ++e) pp[kk][qt][e] = (half_t)0.0f;
  }

  // ---- loads ----
  const uint64_t head_bytes = (uint64_t)b.page_rows * a.width * 2;
  const uint64_t cache = (uint64_t)a.cache + key_head * head_bytes, value_bytes = a.key_heads * head_bytes;
  const uint32_t page_bytes = (uint32_t)(b.page_elements * 2);  // launch_attention_pages
  const uint32_t row_mask = b.page_rows - 1, row_bytes = a.width * 2;
  const uint64_t zeros = (uint64_t)kZeros;
  const uint64_t table = (uint64_t)(b.table + (uint64_t)s * b.table_columns);
  const uint64_t first_table = (uint64_t)b.table;
  const uint32_t last_key = block0 * kKeys + nblocks * kKeys < key_end ? block0 * kKeys + nblocks * kKeys : key_end;
  const uint32_t lane_last = lane < kKeys ? last_key : 0;
  // Table entry of this lane's row of key block j (of all), and its page, -1 for none.
  auto entry = [&](uint32_t j) __attribute__((always_inline)) {
    const uint32_t key = j * kKeys + lane;
    const uint64_t at = (key < b.shared_rows ? first_table : table) + (uint64_t)(key >> b.page_shift) * 4;
    return *(const GLOBAL_AS int*)pick(key < lane_last, at, zeros);
  };
  auto page_at = [&](uint32_t j, int e) __attribute__((always_inline)) {
    const bool has = (j * kKeys + lane < lane_last) & ((uint32_t)e < b.pages);
    return has ? e : -1;
  };
  // Addresses of the rows that this thread's DMA instructions fetch, 0: none.
  auto bases = [&](uint32_t j, int page, uint64_t (&base)[F::kDma]) __attribute__((always_inline)) {
#pragma unroll
    for (uint32_t i = 0; i < F::kDma; ++i) {
      const uint32_t row = i * F::kDmaRows + threadIdx.x / (D / 8);
      const int p = __shfl(page, row, kWave);
      const uint64_t at = cache + (uint64_t)(uint32_t)p * page_bytes + ((j * kKeys + row) & row_mask) * row_bytes;
      base[i] = pick(p >= 0, at, 0);
    }
  };
  const uint32_t dma_row = threadIdx.x / (D / 8), dma_chunk = threadIdx.x % (D / 8);
  // Columns of the chunks that the swizzles place at this thread's slots.  A step of
  // kDmaRows rows leaves the value swizzle alone, and the key swizzle but at 256 columns,
  // where the odd instructions' rows are 8 further on.
  const uint32_t k_column = (dma_chunk ^ key_swizzle<D>(dma_row)) * 8;
  const uint32_t k_column_odd = F::kDmaRows % 16 == 0 ? k_column : (dma_chunk ^ key_swizzle<D>(dma_row + F::kDmaRows)) * 8;
  const uint32_t v_column = (dma_chunk ^ value_swizzle<D>(dma_row)) * 8;
  auto dma = [&](uint32_t i, uint64_t base, uint64_t offset, uint32_t column, uint8_t* to) __attribute__((always_inline)) {
    dma16(pick((base != 0) & (column < a.width), base + offset + column * 2, zeros), to + (i * kThreads + wave * kWave) * 16);
  };

  const uint32_t kbase = r16 * kRowBytes + ((g4 ^ key_swizzle<D>(r16)) << 4);
  uint32_t vbase;
  {
    const uint32_t row = 4 * g4 + r16 / 4, c1 = (r16 % 4) / 2;
    vbase = row * kRowBytes + ((c1 ^ value_swizzle<D>(row)) << 4) + 8 * (r16 % 2);
  }
  auto kfrag = [&](const uint8_t* lk, uint32_t kt, uint32_t ks) __attribute__((always_inline)) {
    return __builtin_bit_cast(half8_t, *reinterpret_cast<const u32x4*>(lk + (kbase ^ (ks << 6)) + 16 * kt * kRowBytes));
  };
  auto vfrag = [&](const uint8_t* lv, uint32_t dt, uint32_t kk) __attribute__((always_inline)) {
    const uint8_t* p = lv + (vbase ^ (dt << 5)) + 32 * kk * kRowBytes;
    const short4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LDS_AS short4_t*)p);
    const short4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LDS_AS short4_t*)(p + 16 * kRowBytes));
    return __builtin_bit_cast(half8_t, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
  };

  uint64_t k_rows[F::kDma], v_rows[F::kDma];  // of key block j + 1 and j in step j
  // Scores of block j and the output of block j - 1, with the DMA of the next keys
  // and this block's values spread over them.
  auto cluster = [&](float4_t (&sc)[kKT][QT], const uint8_t* lk, const uint8_t* lv, uint8_t* nk, uint8_t* nv)
      __attribute__((always_inline)) {
#pragma unroll
    for (uint32_t kt = 0; kt < kKT; ++kt)
#pragma unroll
      for (uint32_t qt = 0; qt < QT; ++qt) sc[kt][qt] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
    constexpr uint32_t kAhead = QT == 2 && kKS == 3 ? 1 : 2;  // fragments ahead, as in k_attention.hip
    half8_t kf[kAhead], vf[kAhead];
#pragma unroll
    for (uint32_t p = 0; p < kAhead; ++p) {
      if (p < kScoreGroups) kf[p] = kfrag(lk, p % kKT, p / kKT);
      if (p < kOutGroups) vf[p] = vfrag(lv, p % kDT, p / kDT);
    }
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (uint32_t p = 0; p < kPairs; ++p) {
      const uint32_t ks = p / kKT, kt = p % kKT, kk = p / kDT, dt = p % kDT;
#pragma unroll
      for (uint32_t qt = 0; qt < QT; ++qt) {
        if (p < kScoreGroups)
          sc[kt][qt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[p % kAhead], qf[qt][ks], sc[kt][qt], 0, 0, 0);
        if (p < kOutGroups)
          o[dt][qt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf[p % kAhead], pp[kk][qt], o[dt][qt], 0, 0, 0);
      }
      if (p + kAhead < kScoreGroups) kf[p % kAhead] = kfrag(lk, (p + kAhead) % kKT, (p + kAhead) / kKT);
      if (p + kAhead < kOutGroups) vf[p % kAhead] = vfrag(lv, (p + kAhead) % kDT, (p + kAhead) / kDT);
      constexpr uint32_t kDmaPer = (2 * F::kDma + kPairs - 1) / kPairs;
#pragma unroll
      for (uint32_t u = 0; u < kDmaPer; ++u) {
        const uint32_t i = p * kDmaPer + u;
        if (i < F::kDma)
          dma(i, k_rows[i], 0, i % 2 ? k_column_odd : k_column, nk);
        else if (i < 2 * F::kDma)
          dma(i - F::kDma, v_rows[i - F::kDma], value_bytes, v_column, nv);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    __builtin_amdgcn_s_setprio(0);
  };
  // Of the 64 keys from key0 on, those that the mask of query 16 qt + l % 16 names.
  auto seen = [&](uint32_t qt, uint32_t key0) __attribute__((always_inline)) {
    uint32_t m = threadIdx.x % 16;
    asm volatile("" : "+v"(m));  // nothing of this is kept in registers
    m += wave0 + 16 * qt;
    m = m < queries ? m : queries - 1;
    return tree_window(a.tree_mask + (uint64_t)(q.first + m / group) * a.mask_words, tree, key0);
  };
  // Softmax of block j (of all), whose rows with a page are `valid`; result in pp.
  auto softmax = [&](float4_t (&sc)[kKT][QT], uint32_t j, uint64_t valid) __attribute__((always_inline)) {
    constexpr uint64_t kAll = ~0ull >> (64 - kKeys);
    const uint32_t key0 = j * kKeys;
    if (valid != kAll || key0 + kKeys > least) {
      // sc[kt][qt][e]: key 16 kt + 4 (l / 16) + e of query 16 qt + l % 16.
      const uint64_t here = valid >> (4 * g4);
#pragma unroll
      for (uint32_t qt = 0; qt < QT; ++qt) {
        const uint64_t mine = Tree ? here & seen(qt, key0) >> (4 * g4) : here;
        const uint32_t left = limit[qt] > key0 + 4 * g4 ? limit[qt] - (key0 + 4 * g4) : 0;
#pragma unroll
        for (uint32_t kt = 0; kt < kKT; ++kt)
#pragma unroll
          for (uint32_t e = 0; e < 4; ++e) {
            const uint32_t x = 16 * kt + e;
            const bool keep = (x < left) & (int)(mine >> x & 1);
            sc[kt][qt][e] = keep ? sc[kt][qt][e] : -INFINITY;
          }
      }
    }
    // Probabilities against the reference points, and this lane's share of their sums, of
    // scores or (Products) their products.
    auto exps = [&]<bool Products>(const float* neg_m, half8_t (&pf)[kHalves][QT], float* sum) __attribute__((always_inline)) {
#pragma unroll
      for (uint32_t qt = 0; qt < QT; ++qt) {
        sum[qt] = 0.0f;
#pragma unroll
        for (uint32_t kk = 0; kk < kHalves; ++kk) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float x = sc[2 * kk + e / 4][qt][e % 4];
            pf[kk][qt][e] = (half_t)__builtin_amdgcn_exp2f(Products ? x + neg_m[qt] : fmaf(x, scale_log2, neg_m[qt]));
          }
#pragma unroll
          for (int e = 0; e < 8; e += 2)
            sum[qt] = __builtin_amdgcn_fdot2(half2_t{pf[kk][qt][e], pf[kk][qt][e + 1]}, half2_t{1, 1}, sum[qt], false);
        }
      }
    };
    half8_t pf[kHalves][QT];
    float sum[QT], neg_m[QT];
    exps.template operator()<false>(near, pf, sum);
    bool over = false;
#pragma unroll
    for (uint32_t qt = 0; qt < QT; ++qt) over = over || !(sum[qt] <= kSumLimit);
    if (__any(over)) {
#pragma unroll
      for (uint32_t qt = 0; qt < QT; ++qt) {
        float top = -INFINITY;
#pragma unroll
        for (uint32_t kt = 0; kt < kKT; ++kt) {
#pragma clang fp contract(off)  // rounded, not one FMA with what follows
          sc[kt][qt] *= scale_log2;
#pragma unroll
          for (int e = 0; e < 4; ++e) top = fmaxf(top, sc[kt][qt][e]);
        }
        top = max_of_query(top);
        const float m_new = fmaxf(m_run[qt], top);
        const float m_use = m_new == -INFINITY ? 0.0f : m_new;  // no NaN from (-inf) - (-inf)
        const float alpha = __builtin_amdgcn_exp2f(m_run[qt] - m_use);
        m_run[qt] = m_new;
        near[qt] = fabsf(m_new) < kFarPoint ? -m_new : INFINITY;
        neg_m[qt] = -m_use;
        l_run[qt] *= alpha;
#pragma unroll
        for (uint32_t dt = 0; dt < kDT; ++dt) o[dt][qt] *= alpha;
      }
      exps.template operator()<true>(neg_m, pf, sum);
    }
#pragma unroll
    for (uint32_t qt = 0; qt < QT; ++qt) l_run[qt] += sum[qt];
#pragma unroll
    for (uint32_t kk = 0; kk < kHalves; ++kk)
#pragma unroll
      for (uint32_t qt = 0; qt < QT; ++qt) pp[kk][qt] = pf[kk][qt];
  };

  // Before the output products of block j with the values in lv: those that are not finite, where
  // some query of the workgroup may not read all of its keys.  A wave looks through a quarter.
  auto look_through = [&](uint32_t j, uint8_t* lv) __attribute__((always_inline)) {
    const uint32_t upto = j * kKeys + kKeys < key_end ? j * kKeys + kKeys : key_end;
    if (upto <= block_least) return;
    const bool mine = has_non_finite<kTile / kWaves>(lv + wave * (kTile / kWaves));
    if (lane == 0) wave_word[wave] = mine;
    __syncthreads();
    if (wave_word[0] | wave_word[1] | wave_word[2] | wave_word[3]) {
      auto weight = [&](uint32_t kk, uint32_t qt, uint32_t e) __attribute__((always_inline)) { return (float)pp[kk][qt][e]; };
      auto chunk = [&](uint32_t row, uint32_t column) __attribute__((always_inline)) {
        return row * kRowBytes + (((column / 8) ^ value_swizzle<D>(row)) << 4) + column % 8 * 2;
      };
      if constexpr (Tree) {
        uint64_t bits[QT];
#pragma unroll
        for (uint32_t qt = 0; qt < QT; ++qt) bits[qt] = seen(qt, j * kKeys);
        add_non_finite<kHalves, kDT, QT>(o, weight, lv, chunk, limit, j * kKeys,
                                         [&](uint32_t qt, uint32_t row) __attribute__((always_inline)) { return bits[qt] >> row & 1; });
      } else {
        add_non_finite<kHalves, kDT, QT>(o, weight, lv, chunk, limit, j * kKeys);
      }
      __syncthreads();
      clear_non_finite<kTile>(lv, threadIdx.x, kThreads);
      __syncthreads();
    }
  };

  // Block j of this part lives in stage j % 2.  Step j: every wave's DMA of K(j) and
  // V(j - 1) has landed, and every wave is done with K(j - 1) and V(j - 2), whose
  // stages this step's DMA overwrites.  Past the last block there is no page, and
  // the DMA fetches zeros.
  int page = page_at(block0, entry(block0)), e = entry(block0 + 1);
  uint64_t valid = __ballot(page >= 0);
  bases(block0, page, k_rows);
  auto step = [&](const uint8_t* lk, uint8_t* lv, uint8_t* nk, uint8_t* nv, uint32_t j)
      __attribute__((always_inline)) {
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    if (j > block0) look_through(j - 1, lv);
    page = page_at(j + 1, e);
    e = entry(j + 2);
    const uint64_t now = valid;
    valid = __ballot(page >= 0);
#pragma unroll
    for (uint32_t i = 0; i < F::kDma; ++i) v_rows[i] = k_rows[i];
    bases(j + 1, page, k_rows);
    float4_t sc[kKT][QT];
    cluster(sc, lk, lv, nk, nv);
    softmax(sc, j, now);
  };
  auto output = [&](const uint8_t* lv) __attribute__((always_inline)) {
#pragma unroll
    for (uint32_t kk = 0; kk < kHalves; ++kk)
#pragma unroll
      for (uint32_t dt = 0; dt < kDT; ++dt) {
        const half8_t v = vfrag(lv, dt, kk);
#pragma unroll
        for (uint32_t qt = 0; qt < QT; ++qt)
          o[dt][qt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, pp[kk][qt], o[dt][qt], 0, 0, 0);
      }
  };
  if (nblocks > 0) {
#pragma unroll
    for (uint32_t i = 0; i < F::kDma; ++i) dma(i, k_rows[i], 0, i % 2 ? k_column_odd : k_column, lds_k0);
    // The first step's output products meet zero probabilities with V stage 1, which
    // may hold anything: zeroed.
#pragma unroll
    for (uint32_t i = 0; i < kTile / 16 / kThreads; ++i)
      *reinterpret_cast<u32x4*>(lds_v1 + (i * kThreads + threadIdx.x) * 16) = u32x4{0, 0, 0, 0};
    uint32_t j = 0;
    for (; j + 1 < nblocks; j += 2) {
      step(lds_k0, lds_v1, lds_k1, lds_v0, block0 + j);
      step(lds_k1, lds_v0, lds_k0, lds_v1, block0 + j + 1);
    }
    if (j < nblocks) step(lds_k0, lds_v1, lds_k1, lds_v0, block0 + j);
    asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
    uint8_t* last = (nblocks - 1) % 2 == 0 ? lds_v0 : lds_v1;
    look_through(block0 + nblocks - 1, last);
    output(last);
  }

  // ---- results: o[dt][qt][e] = O^T[16 dt + 4 (l / 16) + e][query], unnormalised ----
  auto output_row = [&](uint32_t m) __attribute__((always_inline)) {
    const uint32_t row = m / group;
    return (uint64_t)(q.first + row) * a.query_heads + key_head * group + (m - row * group);
  };
  if (!Shared && parts == 1) {
    if (split.parts > 1 && g4 == 0) {
#pragma unroll
      for (uint32_t qt = 0; qt < QT; ++qt)
        if (wave0 + 16 * qt + r16 < queries) split.counts[output_row(wave0 + 16 * qt + r16)] = 1;
    }
#pragma unroll
    for (uint32_t qt = 0; qt < QT; ++qt) {
      const float l = sum_of_query(l_run[qt]);
      const float inverse = l == 0.0f ? 0.0f : 1.0f / l;
      const uint32_t m = wave0 + 16 * qt + r16;
      if (m < queries) {
        half_t* to = (half_t*)a.out + output_row(m) * a.width;
#pragma unroll
        for (uint32_t dt = 0; dt < kDT; ++dt) {
          const uint32_t d = dt * 16 + 4 * g4;
          if (d >= a.width) continue;  // padding (a multiple of 8)
          half4_t h;
#pragma unroll
          for (int x = 0; x < 4; ++x) h[x] = (half_t)(o[dt][qt][x] * inverse);
          *reinterpret_cast<half4_t*>(to + d) = h;
        }
      }
    }
    return;
  }
#pragma unroll
  for (uint32_t qt = 0; qt < QT; ++qt) {
    const float l = sum_of_query(l_run[qt]);
    const uint32_t m = wave0 + 16 * qt + r16;
    if (m < queries) {
      const uint64_t row = output_row(m), at = row * split.parts + part;
      if (g4 == 0) {
        split.sums[at * 2] = m_run[qt];
        split.sums[at * 2 + 1] = l;
        if (!Shared && part == 0) split.counts[row] = parts;
      }
#pragma unroll
      for (uint32_t dt = 0; dt < kDT; ++dt) {
        const uint32_t d = dt * 16 + 4 * g4;
        if (d < a.width) *reinterpret_cast<float4_t*>(split.rows + at * a.width + d) = o[dt][qt];
      }
    }
  }
}

// Joins the parts of the split blocks: a wave per row and query head.
__global__ __launch_bounds__(kThreads) void join_parts_kernel(PagedAttentionArgs a, uint32_t few, SplitKeys split) {
  const uint32_t row = blockIdx.x, lane = threadIdx.x % kWave;
  const uint32_t head = blockIdx.y * kWaves + threadIdx.x / kWave;
  if (head >= a.query_heads) return;
  const uint64_t at = (uint64_t)row * a.query_heads + head;
  const uint32_t written = split.counts[at];
  // Rows of no split block: what stands there is not theirs.
  const uint32_t s = find_sequence(a.batch, row);
  if (s >= a.batch.sequences) return;
  const BatchSequence q = sequence_at(a.batch, s, a.rows);
  const uint32_t parts = uniform(written);
  if (parts < 2 || parts > split.parts) return;  // 1: its block has written the output
  // Lane z holds part z's weight, exp2(m - max m) / sum.
  const float* pair = split.sums + (at * split.parts + (lane < parts ? lane : 0)) * 2;
  const float m0 = pair[0], l0 = pair[1];
  const float* rows = split.rows + at * split.parts * a.width;
  const uint32_t c = lane * 4 < a.width ? lane * 4 : 0;
  constexpr uint32_t kAtOnce = 8;  // loads in flight (past the last part: the last one again, not added)
  float4_t y[kAtOnce];
  auto load = [&](uint32_t z0) __attribute__((always_inline)) {
#pragma unroll
    for (uint32_t z = 0; z < kAtOnce; ++z)
      y[z] = *reinterpret_cast<const float4_t*>(rows + (uint64_t)(z0 + z < parts ? z0 + z : parts - 1) * a.width + c);
  };
  load(0);
  if (row < q.first || q.rows * (a.query_heads / a.key_heads) <= few) return;
  const float m = lane < parts ? m0 : -INFINITY;
  float top = m;
  for (uint32_t o = 8; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, kWave));
  top = __shfl(top, 0, kWave);  // of the first 16 lanes
  const float f = __builtin_amdgcn_exp2f(m - (top == -INFINITY ? 0.0f : top));
  const float sum = wave_sum(lane < parts ? f * l0 : 0.0f);
  const float weight = sum == 0.0f ? 0.0f : f / sum;
  float4_t x = {0.0f, 0.0f, 0.0f, 0.0f};
  for (uint32_t z0 = 0;;) {
#pragma unroll
    for (uint32_t z = 0; z < kAtOnce; ++z) {
      const float w = __shfl(weight, z0 + z, kWave);
      if (z0 + z < parts) x += y[z] * w;
    }
    z0 += kAtOnce;
    if (z0 >= parts) break;
    load(z0);
  }
  if (lane * 4 < a.width) {
    half4_t h;
#pragma unroll
    for (int e = 0; e < 4; ++e) h[e] = (half_t)x[e];
    *reinterpret_cast<half4_t*>((half_t*)a.out + at * a.width + lane * 4) = h;
  }
}
static_assert(kMaxSplits == 16, "join_parts_kernel folds the parts over 16 lanes");

template <int D, int DC, int QT, bool Shared, bool Tree>
int launch_as(hipStream_t stream, const PagedAttentionArgs& a, float scale_log2, uint32_t few, const SplitKeys& given) {
  const uint64_t queries = (uint64_t)a.rows * (a.query_heads / a.key_heads);
  constexpr uint64_t kQueries = Block<D, QT>::kQueries;
  // Blocks: at most a partial one more for each sequence of more than `few` queries.
  uint64_t blocks = (queries + kQueries - 1) / kQueries;
  if (!Shared) {
    const uint64_t sequences = queries / ((uint64_t)few + 1);
    blocks += a.batch.sequences < sequences ? a.batch.sequences : sequences;
  }
  blocks *= a.key_heads;
  SplitKeys split = given;
  // Parts where the blocks may leave half of the chip's workgroups idle and the table
  // holds keys enough; how many, the kernel decides by the blocks that there are.
  const uint64_t reach = (uint64_t)a.batch.table_columns * a.batch.page_rows;
  // Known exactly where every sequence has max_rows.
  uint64_t least = 0;
  if (few == 0 && (uint64_t)a.batch.sequences * a.max_rows == a.rows)
    least = ((uint64_t)a.max_rows * (a.query_heads / a.key_heads) + kQueries - 1) / kQueries * a.batch.sequences * a.key_heads;
  const uint64_t room = Tree ? 2 * kFullChip + 1 : kFullChip / 2;  // tree_part
  const bool may_split = least < room && !(Tree && a.batch.sequences > kPlannedSequences) &&
                         reach > (uint64_t)(kLeastSplit - 1) * Block<D, QT>::kKeys;
  const uint64_t most = Tree ? 4 * kFullChip : kFullChip;
  if (!Shared && a.workspace.data && blocks < most && may_split) {
    const uint64_t rows = (uint64_t)a.rows * a.query_heads;
    uint64_t parts = a.workspace.bytes / sizeof(float) / rows;  // floats per row, then parts
    parts = parts > 0 ? (parts - 1) / (a.width + 2) : 0;
    if (parts > kMaxSplits) parts = kMaxSplits;
    if (parts > 1) {
      split.parts = (uint32_t)parts;
      split.rows = (float*)a.workspace.data;
      split.sums = split.rows + rows * parts * a.width;
      split.counts = (uint32_t*)(split.sums + rows * parts * 2);
    }
  }
  // Split blocks make at most kFullChip workgroups, in ranges of whole blocks' parts (Shared: the
  // given parts of each).
  // Tree: whole blocks, or parts of which there are at most twice kFullChip.
  uint64_t grid = Shared ? blocks * split.parts : split.parts > 1 ? kFullChip + 8 * kMaxSplits : blocks;
  if (Tree) grid = split.parts > 1 && blocks < 2 * kFullChip ? 2 * kFullChip : blocks;
  grid = (grid + 7) / 8 * 8;
  if (grid > 0xffffffull) return IPUS_ERROR_UNAVAILABLE;  // a grid dimension holds less than 2^32 threads
  hipLaunchKernelGGL((attention_blocks_kernel<D, DC, QT, Shared, Tree>), dim3((uint32_t)grid), dim3(kThreads), 0, stream, a,
                     scale_log2, few, split);
  if (int e = hip_status(hipGetLastError())) return e;
  if (Shared || split.parts <= 1) return 0;
  // So few blocks hold fewer than 2^20 rows.
  hipLaunchKernelGGL(join_parts_kernel, dim3(a.rows, (a.query_heads + kWaves - 1) / kWaves), dim3(kThreads), 0, stream, a,
                     few, split);
  return hip_status(hipGetLastError());
}
template <bool Shared, bool Tree>
int launch(hipStream_t stream, const PagedAttentionArgs& a, float scale_log2, uint32_t few, const SplitKeys& split) {
  if (a.width > 192) return launch_as<256, 256, 1, Shared, Tree>(stream, a, scale_log2, few, split);
  if (a.width > 128) return launch_as<256, 192, 1, Shared, Tree>(stream, a, scale_log2, few, split);
  if (a.width > 96) return launch_as<128, 128, 2, Shared, Tree>(stream, a, scale_log2, few, split);
  if (a.width > 64) return launch_as<128, 96, 2, Shared, Tree>(stream, a, scale_log2, few, split);
  if (a.width > 32) return launch_as<64, 64, 2, Shared, Tree>(stream, a, scale_log2, few, split);
  return launch_as<64, 32, 2, Shared, Tree>(stream, a, scale_log2, few, split);
}

}  // namespace

int launch_attention_blocks(hipStream_t stream, const PagedAttentionArgs& a, float scale_log2, uint32_t few) {
  const SplitKeys whole{nullptr, nullptr, nullptr, 1};
  return a.tree_mask ? launch<false, true>(stream, a, scale_log2, few, whole)
                     : launch<false, false>(stream, a, scale_log2, few, whole);
}
int launch_shared_parts(hipStream_t stream, const PagedAttentionArgs& a, float scale_log2, const SharedParts& parts) {
  return launch<true, false>(stream, a, scale_log2, 0, SplitKeys{parts.rows, parts.sums, nullptr, parts.parts});
}
uint32_t shared_part_count(const PagedAttentionArgs& a, uint32_t most) {
  const uint32_t block_queries = a.width > 128 ? 64 : 128, block_keys = a.width > 128 ? 32 : 64;
  const uint64_t queries = (uint64_t)a.rows * (a.query_heads / a.key_heads);
  const uint64_t blocks = (queries + block_queries - 1) / block_queries * a.key_heads;
  const uint64_t reach = (uint64_t)a.batch.table_columns * a.batch.page_rows;
  const uint32_t keys = a.batch.shared_rows < reach ? a.batch.shared_rows : (uint32_t)reach;
  const uint32_t key_blocks = (keys + block_keys - 1) / block_keys;
  uint64_t parts = (kFullChip + blocks - 1) / blocks;
  if (parts > most) parts = most;
  if (parts > key_blocks) parts = key_blocks;
  if (parts == 0) return 0;
  const uint32_t per_part = (key_blocks + (uint32_t)parts - 1) / (uint32_t)parts;
  return (key_blocks + per_part - 1) / per_part;  // every part has a block of keys
}

}  // namespace ipus
