// Attention of a ragged batch over a paged cache (pages.h) on gfx950:
//   out = softmax(scale q K^T [+ causal mask]) V
// for every row of every sequence, query head h reading key head
// h / (query_heads / key_heads).  Row i of the n rows of sequence s stands at
// position lengths[s] - n + i; it reads the keys below lengths[s], when causal
// those up to its own position, of a tree all before the sequence's rows and those of
// the rows that its mask names.  Keys without a page carry no weight, and a row
// whose weights are all zero (no key, or only scores of -inf) gives zeros.
#include "attention_pages.h"

#include <type_traits>

namespace ipus {
namespace {

// Any width up to 1024, any alignment: a workgroup per row and query head, its waves eight
// keys each at a time, whose loads wait for memory together, joined in LDS (4 sequences x
// 16 heads x 1000 keys of 65 columns 69 us, of 2000 of 500 columns 434; one key after the
// other by one wave 859 and 8,530).
constexpr uint32_t kGeneralWidth = 1024, kGeneralPerLane = kGeneralWidth / kWave, kGeneralKeys = 8;
template <bool Tree>
__global__ __launch_bounds__(kThreads) void attention_pages_general_kernel(PagedAttentionArgs a, uint32_t first_row,
                                                                           float scale_log2) {
  __shared__ float wave_rows[kWaves][kGeneralWidth], wave_sums[kWaves][2];
  const uint32_t row = first_row + blockIdx.x, head = blockIdx.y;
  const uint32_t lane = threadIdx.x % kWave, wave = uniform(threadIdx.x / kWave);
  const RowPlace place = find_row(a.batch, row);
  if (place.sequence >= a.batch.sequences) return;
  const uint32_t s = uniform(place.sequence);
  const uint32_t count = uniform(readable_keys(sequence_at(a.batch, s, a.rows), place.position, a.causal));
  const half_t* from = (const half_t*)a.query + (uint64_t)row * a.query_row_stride + (uint64_t)head * a.width;
  const uint32_t key_head = head / (a.query_heads / a.key_heads);
  const uint64_t head_elements = (uint64_t)a.batch.page_rows * a.width;
  TreeRows tree = Tree ? tree_rows(a.batch, s, a.rows, a.mask_words) : TreeRows{0, 0};
  if (Tree) asm volatile("" : "+v"(tree.base), "+v"(tree.bits));  // not in scalar registers
  float q[kGeneralPerLane], acc[kGeneralPerLane];
#pragma unroll
  for (uint32_t i = 0; i < kGeneralPerLane; ++i) {
    const uint32_t d = lane + kWave * i;
    q[i] = d < a.width ? (float)from[d] : 0.0f;
    acc[i] = 0.0f;
  }
  float m = -INFINITY, l = 0.0f;
  for (uint32_t j0 = wave * kGeneralKeys; j0 < count; j0 += kWaves * kGeneralKeys) {
    // Keys without a page: the query is loaded in their place, and not used.
    const half_t *key[kGeneralKeys], *value[kGeneralKeys];
    bool has[kGeneralKeys];
    float dot[kGeneralKeys];
    int mine = lane < kGeneralKeys && j0 + lane < count ? page_of(a.batch, s, j0 + lane) : -1;
    if (Tree && (int64_t)j0 + kGeneralKeys > tree.base)
      mine = tree_window(a.tree_mask + (uint64_t)row * a.mask_words, tree, j0) >> lane & 1 ? mine : -1;
#pragma unroll
    for (uint32_t u = 0; u < kGeneralKeys; ++u) {
      const int page = __builtin_amdgcn_readlane(mine, u);
      const half_t* at = (const half_t*)a.cache + (uint64_t)(uint32_t)page * a.batch.page_elements +
                         key_head * head_elements + (uint64_t)((j0 + u) & (a.batch.page_rows - 1)) * a.width;
      has[u] = page >= 0;
      key[u] = has[u] ? at : from;
      value[u] = has[u] ? at + a.key_heads * head_elements : from;
      dot[u] = 0.0f;
    }
#pragma unroll
    for (uint32_t i = 0; i < kGeneralPerLane; ++i) {
      const uint32_t d = lane + kWave * i;
      if (kWave * i >= a.width) break;
      half_t x[kGeneralKeys];
#pragma unroll
      for (uint32_t u = 0; u < kGeneralKeys; ++u) x[u] = key[u][d < a.width ? d : 0];
#pragma unroll
      for (uint32_t u = 0; u < kGeneralKeys; ++u) dot[u] = d < a.width ? fmaf(q[i], (float)x[u], dot[u]) : dot[u];
    }
    float top = m;
#pragma unroll
    for (uint32_t u = 0; u < kGeneralKeys; ++u) {
      const float score = wave_sum(dot[u]) * scale_log2;
      dot[u] = has[u] ? score : -INFINITY;
      top = fmaxf(top, dot[u]);
    }
    const float use = top == -INFINITY ? 0.0f : top;  // no NaN from (-inf) - (-inf)
    const float alpha = exp2f(m - use);
    m = top;
    l *= alpha;
#pragma unroll
    for (uint32_t u = 0; u < kGeneralKeys; ++u) {
      dot[u] = exp2f(dot[u] - use);
      l += dot[u];
    }
#pragma unroll
    for (uint32_t i = 0; i < kGeneralPerLane; ++i) {
      const uint32_t d = lane + kWave * i;
      if (kWave * i >= a.width) break;
      half_t x[kGeneralKeys];
#pragma unroll
      for (uint32_t u = 0; u < kGeneralKeys; ++u) x[u] = value[u][d < a.width ? d : 0];
      acc[i] *= alpha;
#pragma unroll
      for (uint32_t u = 0; u < kGeneralKeys; ++u) acc[i] = has[u] ? fmaf(dot[u], (float)x[u], acc[i]) : acc[i];
    }
  }
#pragma unroll
  for (uint32_t i = 0; i < kGeneralPerLane; ++i) {
    const uint32_t d = lane + kWave * i;
    if (d < a.width) wave_rows[wave][d] = acc[i];
  }
  if (lane == 0) {
    wave_sums[wave][0] = m;
    wave_sums[wave][1] = l;
  }
  __syncthreads();
  float top = -INFINITY, sum = 0.0f, weight[kWaves];
#pragma unroll
  for (uint32_t w = 0; w < kWaves; ++w) top = fmaxf(top, wave_sums[w][0]);
  const float use = top == -INFINITY ? 0.0f : top;
#pragma unroll
  for (uint32_t w = 0; w < kWaves; ++w) {
    weight[w] = exp2f(wave_sums[w][0] - use);
    sum += weight[w] * wave_sums[w][1];
  }
  const float inverse = sum == 0.0f ? 0.0f : 1.0f / sum;
  half_t* out = (half_t*)a.out + ((uint64_t)row * a.query_heads + head) * a.width;
  for (uint32_t d = threadIdx.x; d < a.width; d += kThreads) {
    float x = 0.0f;
#pragma unroll
    for (uint32_t w = 0; w < kWaves; ++w) x += weight[w] * wave_rows[w][d];
    out[d] = (half_t)(x * inverse);
  }
}

// ---------------------------------------------------------------------------
// Few query rows per key head: the keys are read once, bound by HBM.
//
// A sequence's rows times the query heads of one key head are packed into tiles
// of 16 or 32 queries, so a key head's keys and values serve all of its query
// heads.  The work of the whole batch - every (sequence, query tile, key head)
// with its tiles of kKeys keys - is one line of units, cut into equal chunks, one
// per workgroup: sequences of any mix of lengths load the chip evenly.  A
// (sequence, query tile, key head) that lies in several chunks is merged by the
// last of their workgroups to finish, in the order of the keys.  Every workgroup finds
// its place by a scan over the sequences' lengths (two reads of a few words, in L2).
//
// Waves work alone: wave w takes the chunk's key tiles w, w + 4, ...  A tile's keys go
// to registers in the layout of the first MFMA operand, its values by LDS DMA into the
// wave's own stage (the transposing LDS read needs them there), the next tile's loads run
// under this one's arithmetic, and the page numbers of the one after under both.  At 8
// waves per CU 128 KiB are in flight, without a barrier until the waves' results are
// joined at the end of a segment.
//
// Measured (width 128, 32 query heads on 8): 64 sequences of 2048 to 32768 keys, 2.8 GB,
// 481 us, 5.9 TB/s of a copy's 6.3; 64 of 4000 181 us, 5.8; 256 of 300 67 us, 4.7; 64 of 300 20 us,
// where a segment's start (five loads that wait for each other, about 6 us) and end (2 us)
// are as long as its keys' loads.
//
// Scores are computed transposed, S^T = K Q^T, and the output as O^T += V^T P^T
// (v_mfma_f32_16x16x32_f16, fp32 accumulation), as in k_attention.hip.  The probabilities
// enter the second product as the sum of two fp16 values (22 bits): the matrix pipes have
// time for it here, and the result is off by little more than its own rounding.  With 32
// queries per tile, but for 128 columns, they are one fp16 value (2^-11), as in the kernel
// for many rows, and so are the sums' terms.

// Partial results of a launch: two slots per workgroup, each 16 * MT rows of D fp32
// and their (reference point, sum) pairs; without memory every segment is one
// workgroup's.
struct DecodeSplit {
  float* rows;
  float* sums;
  uint32_t* counters;  // by a segment's first part
};
constexpr uint32_t kMaxParts = 64;       // of one segment
constexpr uint32_t kMostGroups = 2048;   // workgroups of a launch at most
constexpr uint32_t kMostResident = 512;  // workgroups on the chip at most (Decode::kResident)

// How a launch's segments (a sequence's query tile and key head, with its key tiles) are
// dealt to the workgroups.  A segment's start and end cost about as much as four tiles per
// wave, joining parts of it as much again:
//  - none of more than 32 tiles (with shared keys' parts, which a wave alone joins slowly, 8;
//    past 128 columns never), and 600 times the longest in all: a wave takes a segment
//    alone, so that the starts of four run at once and nothing is joined (us, alone / by
//    a workgroup's waves together; 128 columns: 256 sequences x 8 heads x 300 keys
//    66.7 / 82.2, 128 x 8 x 616 63.4 / 65.3, 300 x 8 of 37 to 600 keys 72 / 123; 64
//    columns: 256 x 16 x 60 27 / 62, 40 x 16 x 200 (640 segments) 14.4 / 18.2; not 64 x 8 x 300
//    at 128 columns (512 segments) 23.3 / 20.5, where a wave's own latency counts; behind 2048
//    shared keys, 256 x 16 x 52 of 64 columns 54 / 93, 256 x 8 x 52 of 128 55 / 71, but 113 x 12 x
//    30 of 256 columns 151 / 92);
//  - no segment of more than 16 tiles: all whole;
//  - at least 40 tiles per resident workgroup (of trees 200): the tiles of all segments are one line, cut
//    into an equal chunk for each, wherever the cuts fall (128 segments of 125 tiles, 31 per
//    workgroup, 61.6 us so, in parts 54.6);
//  - in between: every segment in parts of its own, of at least 8 tiles, one per
//    workgroup (cut at any place, a workgroup would pay two segments' starts for a few tiles:
//    2 x 8 segments of 34 tiles 18.1 us, of 48 tiles, where the cuts coincide, 13.0), and
//    about one per CU (two make twice the parts to join: 8 segments of 500 tiles 24.5 us
//    against 21.6, 32 of 66 18.2 against 16.1).
// The line's units are tiles (part_tiles = 0) or parts of at most part_tiles tiles.
// Trees: hundreds of segments of very different lengths are whole, or in few parts, up to 200
// tiles per workgroup, which begins the next one as it ends (us, so / in equal chunks from 40 on,
// 8 key heads x 128: 128 trees against 125 to 2000 keys 95 / 125, 64 against 250 to 4000 84 / 91, 128
// against 250 to 4000 164 / 177; 64 against 500 to 8000 148 / 144, of equal lengths the same).  Single
// rows and causal ones keep the 40, and with it the order in which their parts are added.
constexpr uint32_t kAloneTiles = 32, kAloneShared = 8, kChunkTiles = 40, kTreeChunkTiles = 200;
struct Shares {
  uint32_t part_tiles;
  uint64_t chunk;  // units per workgroup, or per wave
  uint64_t parts;  // units of the line, or a bound on them
  bool alone;      // every wave has segments of its own
  __device__ __forceinline__ uint32_t units(uint32_t tiles) const {
    return part_tiles == 0 ? tiles : part_tiles >= tiles ? 1 : (tiles + part_tiles - 1) / part_tiles;
  }
  __device__ __forceinline__ uint64_t total(uint64_t tiles, uint64_t segments) const {
    return part_tiles == 0 ? tiles : parts;
  }
};
__device__ __forceinline__ Shares share_out(uint64_t tiles, uint64_t segments, uint32_t longest, uint32_t groups,
                                            uint32_t resident, bool may_split, uint32_t alone_tiles, uint32_t chunk_tiles) {
  constexpr uint32_t kAloneSegments = 600;
  constexpr uint32_t kWholeTiles = 16, kLeastTiles = 8, kCus = 256;
  if (longest <= alone_tiles && (uint64_t)longest * kAloneSegments <= tiles) {
    const uint32_t waves = groups * kWaves;
    return {0xffffffffu, quotient(segments + waves - 1, waves), segments, true};
  }
  if (!may_split || longest <= kWholeTiles)
    return {0xffffffffu, quotient(segments + groups - 1, groups), segments, false};
  if (resident > groups) resident = groups;
  const uint64_t each = quotient(tiles + resident - 1, resident);
  if (each < chunk_tiles) {
    uint32_t part = (uint32_t)((tiles + kCus - 1) / kCus);
    if (part < kLeastTiles) part = kLeastTiles;
    const uint32_t least = (longest + kMaxParts - 1) / kMaxParts;
    if (part < least) part = least;
    const uint64_t parts = quotient(tiles, part) + segments;  // at most
    if (parts <= groups) return {part, 1, parts, false};
  }
  const uint64_t least = (longest + kMaxParts - 2) / (kMaxParts - 1);
  return {0, each < least ? least : each, 0, false};
}

// D: the width rounded up to 32, 64, 96, 128, 192 or 256 columns, which are computed and
// are an LDS row.
template <int D, int MT>
struct Decode {
  static constexpr uint32_t kKeys = D > 64 ? 32 : 64;  // per tile
  static constexpr uint32_t kRowBytes = D * 2, kChunks = D / 8;
  static constexpr uint32_t kTileBytes = kKeys * kRowBytes;
  static constexpr uint32_t kKT = kKeys / 16, kKS = D / 32, kDT = D / 16, kHalves = kKeys / 32;
  static constexpr uint32_t kQueries = 16 * MT;
  static constexpr uint32_t kDma = kTileBytes / 1024;  // DMA instructions of a wave per tile
  // Workgroups per CU, by LDS (two stages of a tile per wave) and registers.  One keeps
  // nearly the bandwidth of two (64 sequences x 8 heads x 4096 keys x 128: 191 us against 185); three, where
  // they fit, lose some (96 columns: 167 against 139).
  static constexpr uint32_t kPerCu = D > 128 || (D == 128 && MT == 2) ? 1 : 2;
  // Probabilities as two fp16 values; with two tiles of queries as one, for the registers,
  // where a CU holds two workgroups: at 64 and 96 columns the second value spills, at 32 it
  // costs 6% (64 sequences x 3 rows x 24 heads on 4 x 3000 keys, 30.9 us against 29.2); at 128
  // nothing (16 x 3 x 64 on 8 x 8000 keys 107.3 against 106.4, 64 x 2000 101.5 against 101.3).
  static constexpr bool kTwoHalves = MT == 1 || kPerCu == 1;
  static constexpr uint32_t kResident = 256 * kPerCu;
};
// 16-byte chunk c of a tile's row r lies at chunk c ^ swizzle(r): the 4 rows x 32 bytes that
// 16 lanes of ds_read_b64_tr_b16 take then touch every bank once.  Rows of 64 and 192 bytes do
// without; those of 384 bytes meet in pairs.
template <int D>
__device__ __forceinline__ uint32_t tile_swizzle(uint32_t row) {
  return D == 64 || D == 128 || D == 256 ? value_swizzle<D>(row) : 0;
}

// Units of sequence q: query tiles x key heads, each of `tiles` key tiles (at
// least one, so that rows without keys are written).  A sequence of more than `few`
// queries is the other kernel's.
struct Units {
  uint64_t segments;
  uint32_t tiles;
};
template <uint32_t Keys, uint32_t Queries>
__device__ __forceinline__ Units units_of(const BatchSequence& q, uint32_t group, uint32_t key_heads, uint32_t first_key,
                                          uint32_t few) {
  Units u;
  const uint32_t queries = q.rows * group;  // launch_attention_pages
  u.segments = queries <= few ? (uint64_t)((queries + Queries - 1) / Queries) * key_heads : 0;
  const uint32_t keys = q.keys > first_key ? q.keys - first_key : 0;
  u.tiles = keys == 0 ? 1 : (uint32_t)(((uint64_t)keys + Keys - 1) / Keys);
  return u;
}

// Shared: the keys from first_key on, joined with the parts of those before it.  Tree: the
// masks of a sequence's rows, looked up for the tiles that hold their keys.
template <int D, int MT, bool Shared, bool Tree>
__global__ __launch_bounds__(kThreads, (Decode<D, MT>::kPerCu)) void attention_pages_decode_kernel(
    PagedAttentionArgs a, float scale_log2, uint32_t keys_from, uint32_t few, DecodeSplit split,
    SharedParts given) {
  const uint32_t first_key = Shared ? keys_from : 0;
  const SharedParts shared = Shared ? given : SharedParts{nullptr, nullptr, 0};
  using C = Decode<D, MT>;
  constexpr uint32_t kKeys = C::kKeys, kKT = C::kKT, kKS = C::kKS, kDT = C::kDT, kHalves = C::kHalves;
  constexpr uint32_t kQueries = C::kQueries, kTile = C::kTileBytes, kRowBytes = C::kRowBytes;
  // Two stages, distinct objects, so that the compiler sees that the DMA into
  // one never meets the reads of the other; a wave's tile at wave * kTile.
  __shared__ __attribute__((aligned(1024))) uint8_t stage0[kWaves * kTile];
  __shared__ __attribute__((aligned(1024))) uint8_t stage1[kWaves * kTile];
  __shared__ float wave_sums[kWaves][kQueries][2];
  // Weights of a query's parts and their sums: the waves' and the shared keys'.  Where a
  // segment of several workgroups is merged, its parts' and the shared keys', in the stages.
  constexpr uint32_t kShared = Shared ? kMaxSharedParts : 0;
  constexpr uint32_t kFewParts = kWaves + kShared, kManyParts = kMaxParts + kShared;
  __shared__ float few_weights[kQueries * kFewParts], few_sums[kQueries * kFewParts];
  static_assert(kQueries * kManyParts * 4 <= kWaves * kTile, "the weights of a merge fit a stage");
  __shared__ uint32_t arrived;

  const uint32_t lane = threadIdx.x % kWave, r16 = lane % 16, g4 = lane / 16;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const uint32_t group = a.query_heads / a.key_heads;
  const PagedBatch& b = a.batch;

  // ---- this workgroup's share of the batch ----
  auto units_at = [&](uint32_t s) __attribute__((always_inline)) {
    return units_of<kKeys, kQueries>(sequence_at(b, s, a.rows), group, a.key_heads, first_key, few);
  };
  const Units held = lane < b.sequences ? units_at(lane) : Units{0, 1};  // of the first 64 sequences
  uint64_t tiles = held.segments * held.tiles, segments = held.segments;
  uint32_t longest = held.segments > 0 ? held.tiles : 0;
  for (uint32_t s = kWave + lane; s < b.sequences; s += kWave) {
    const Units u = units_at(s);
    tiles += u.segments * u.tiles;
    segments += u.segments;
    if (u.segments > 0 && u.tiles > longest) longest = u.tiles;
  }
  tiles = from_lane(scan(tiles), kWave - 1);
  segments = from_lane(scan(segments), kWave - 1);
  longest = largest(longest);
  if (segments == 0) return;
  const Shares shares = share_out(tiles, segments, longest, gridDim.x, C::kResident, split.rows != nullptr,
                                  !Shared ? kAloneTiles : D <= 128 ? kAloneShared : 0,
                                  Tree ? kTreeChunkTiles : kChunkTiles);
  auto line_units = [&](const Units& u) __attribute__((always_inline)) { return u.segments * shares.units(u.tiles); };
  auto units_in = [&](uint32_t s) __attribute__((always_inline)) { return line_units(units_at(s)); };
  UnitLine line{scan(line_units(held)), 0};
  const bool alone = shares.alone;
  const uint64_t begin = (alone ? (uint64_t)blockIdx.x * kWaves + wave : blockIdx.x) * shares.chunk;
  if (begin >= shares.total(tiles, segments)) return;
  const UnitPlace place = find_unit(b, line, begin, units_in);
  uint32_t s = place.sequence;
  uint64_t sequence_begin = place.first;  // first unit of sequence s
  uint64_t end = begin + shares.chunk;

  // Per-lane offsets of the tile accesses.
  const uint64_t head_bytes = (uint64_t)b.page_rows * a.width * 2;
  const uint32_t row_mask = b.page_rows - 1;
  uint32_t vbase;
  {
    const uint32_t row = 4 * g4 + r16 / 4, c1 = (r16 % 4) / 2;
    vbase = row * kRowBytes + ((c1 ^ tile_swizzle<D>(row)) << 4) + 8 * (r16 % 2);
  }
  uint8_t* const my0 = stage0 + wave * kTile;
  uint8_t* const my1 = stage1 + wave * kTile;

  uint64_t unit = begin;
  while (unit < end) {
    if (s >= b.sequences) break;  // the line's end
    const BatchSequence q = uniform(sequence_at(b, s, a.rows));
    const Units u = units_of<kKeys, kQueries>(q, group, a.key_heads, first_key, few);
    const uint32_t per_segment = shares.units(u.tiles);
    const uint64_t units = u.segments * per_segment;
    if (unit >= sequence_begin + units) {  // also a sequence without rows
      sequence_begin += units;
      ++s;
      continue;
    }
    const uint64_t within = unit - sequence_begin;
    const uint64_t segment = quotient(within, per_segment);
    const uint32_t unit_first = (uint32_t)(within - segment * per_segment);
    const uint64_t segment_begin = unit - unit_first, segment_end = segment_begin + per_segment;
    const uint32_t query_tile = (uint32_t)segment / a.key_heads, key_head = (uint32_t)segment - query_tile * a.key_heads;
    const uint32_t query0 = query_tile * kQueries;  // of the sequence's rows x group
    // Its key tiles: those of one part, or (cut into chunks) up to the chunk's end.
    uint32_t tile_first = unit_first, tile_last;
    uint64_t stop;
    if (shares.part_tiles) {
      const uint32_t each = (u.tiles + per_segment - 1) / per_segment;  // every part has a tile
      stop = unit + 1;
      tile_first = unit_first * each;
      tile_last = u.tiles - tile_first < each ? u.tiles : tile_first + each;
    } else {
      stop = segment_end < end ? segment_end : end;
      tile_last = tile_first + (uint32_t)(stop - unit);
    }

    // The wave's queries: fragment (mt, ks) holds columns 32 ks + 8 (l / 16) .. + 7 of
    // query 16 mt + l % 16; padding queries repeat the last one, with no key allowed.
    const uint32_t queries = q.rows * group - query0;  // left, at least 1
    half8_t qf[MT][kKS];
    uint32_t limit[MT];  // keys that this lane's query may read
    // Its mask, where that is one word, asked for with the query (in the last tile, where it is
    // used, its load would be waited for: 4 trees of 8 rows against 1000 keys 13.3 us, so 13.9).
    constexpr bool kEarly = Tree && MT == 1;
    uint32_t early = 0;
#pragma unroll
    for (uint32_t mt = 0; mt < MT; ++mt) {
      uint32_t m = 16 * mt + r16;
      const bool real = m < queries;
      m = real ? m : queries - 1;
      const uint32_t row = q.first + (query0 + m) / group, head = (query0 + m) % group;
      const half_t* from = (const half_t*)a.query + (uint64_t)row * a.query_row_stride +
                           (uint64_t)(key_head * group + head) * a.width;
      const int position = row_position(q.length, q.end, row);
      limit[mt] = real ? readable_keys(q, position, a.causal) : 0;
      if (kEarly) early = a.tree_mask[(uint64_t)row * a.mask_words];
#pragma unroll
      for (uint32_t ks = 0; ks < kKS; ++ks) {
        const uint32_t d0 = ks * 32 + g4 * 8;
        qf[mt][ks] = __builtin_bit_cast(half8_t, d0 < a.width ? load16(from + d0) : u32x4{0, 0, 0, 0});
      }
    }
    // Every query of the tile reads the keys below `least`: causal rows stand in the order
    // of their positions.
    const TreeRows tree = Tree ? tree_rows(b, s, a.rows, a.mask_words) : TreeRows{0, 0};
    const uint32_t least = !Tree ? readable_keys(q, row_position(q.length, q.end, q.first + query0 / group), a.causal)
                           : tree.base <= 0 ? 0 : tree.base < (int64_t)q.keys ? (uint32_t)tree.base : q.keys;
    float4_t o[kDT][MT];
    float m_run[MT], l_run[MT];
#pragma unroll
    for (uint32_t mt = 0; mt < MT; ++mt) {
      m_run[mt] = -INFINITY;
      l_run[mt] = 0.0f;
#pragma unroll
      for (uint32_t dt = 0; dt < kDT; ++dt) o[dt][mt] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
    }

    const uint64_t cache = (uint64_t)a.cache + key_head * head_bytes, value_bytes = a.key_heads * head_bytes;
    const uint32_t page_bytes = (uint32_t)(b.page_elements * 2);  // launch_attention_pages
    const uint64_t zeros = (uint64_t)kZeros;
    // Keys of this part, from first_key on; lanes past a tile's rows have none.
    const uint32_t all_keys = q.keys > first_key ? q.keys - first_key : 0;
    const uint32_t part_keys = (uint64_t)tile_last * kKeys < all_keys ? tile_last * kKeys : all_keys;
    const uint32_t lane_keys = lane < kKeys ? part_keys : 0;
    // Table entry of this lane's row of tile t; page_at: its page, -1 for none.
    auto entry = [&](uint32_t t) __attribute__((always_inline)) {
      const uint32_t key = first_key + t * kKeys + lane;
      const uint64_t at = (uint64_t)(b.table + (uint64_t)(key < b.shared_rows ? 0 : s) * b.table_columns + (key >> b.page_shift));
      return *(const GLOBAL_AS int*)pick(t * kKeys + lane < lane_keys, at, zeros);
    };
    auto page_at = [&](uint32_t t, int e) __attribute__((always_inline)) {
      const bool has = (t * kKeys + lane < lane_keys) & ((uint32_t)e < b.pages);
      return has ? e : -1;
    };
    auto row_address = [&](uint32_t t, uint32_t row, int p) __attribute__((always_inline)) {
      const uint32_t key = first_key + t * kKeys + row;
      return cache + (uint64_t)(uint32_t)p * page_bytes + (key & row_mask) * (a.width * 2);
    };
    // Opaque, so that rows and chunks are not kept in registers between tiles.
    auto opaque = [](uint32_t x) __attribute__((always_inline)) {
      asm volatile("" : "+v"(x));
      return x;
    };
    // Tile t's keys into registers and its values into LDS; zeros for rows without a page.
    half8_t kf[kKT][kKS];
    auto fetch_keys = [&](uint32_t t, int page) __attribute__((always_inline)) {
      const uint32_t lane_v = opaque(lane);
#pragma unroll
      for (uint32_t kt = 0; kt < kKT; ++kt) {
        const uint32_t row = 16 * kt + lane_v % 16;
        const int p = __shfl(page, row, kWave);
        const uint64_t at = row_address(t, row, p);
#pragma unroll
        for (uint32_t ks = 0; ks < kKS; ++ks) {
          const uint32_t d0 = ks * 32 + (lane_v / 16) * 8;
          kf[kt][ks] = __builtin_bit_cast(half8_t, load16_at(pick((p >= 0) & (d0 < a.width), at + d0 * 2, zeros)));
        }
      }
      __builtin_amdgcn_sched_barrier(0);  // on the way before the arithmetic that follows
    };
    auto fetch_values = [&](uint32_t t, int page, uint8_t* lv) __attribute__((always_inline)) {
      const uint32_t lane_v = opaque(lane);
#pragma unroll
      for (uint32_t i = 0; i < C::kDma; ++i) {
        const uint32_t slot = i * kWave + lane_v, row = slot / C::kChunks;
        const uint32_t column = ((slot % C::kChunks) ^ tile_swizzle<D>(row)) * 8;
        const int p = __shfl(page, row, kWave);
        dma16(pick((p >= 0) & (column < a.width), row_address(t, row, p) + value_bytes + column * 2, zeros), lv + i * 1024);
      }
      __builtin_amdgcn_sched_barrier(0);
    };
    auto scores = [&](float4_t (&sc)[kKT][MT]) __attribute__((always_inline)) {
#pragma unroll
      for (uint32_t kt = 0; kt < kKT; ++kt)
#pragma unroll
        for (uint32_t mt = 0; mt < MT; ++mt) {
          sc[kt][mt] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
          for (uint32_t ks = 0; ks < kKS; ++ks)
            sc[kt][mt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[kt][ks], qf[mt][ks], sc[kt][mt], 0, 0, 0);
        }
      __builtin_amdgcn_sched_barrier(0);
    };
    // Softmax of tile t's scores, rows of `valid`, and the output with the values in lv.
    auto update = [&](uint32_t t, uint64_t valid, float4_t (&sc)[kKT][MT], uint8_t* lv) __attribute__((always_inline)) {
      const uint32_t key0 = first_key + t * kKeys;
      const uint32_t upto = (t + 1) * kKeys < all_keys ? key0 + kKeys : q.keys;
      half8_t high[kHalves][MT], low[kHalves][MT];
      // Of the tile's keys, those that the query's mask names.
      auto seen = [&](uint32_t mt) __attribute__((always_inline)) {
        if (kEarly && tree.bits <= 32) return tree_window(&early, tree, key0);
        uint32_t m = 16 * mt + opaque(lane) % 16;
        m = m < queries ? m : queries - 1;
        const uint32_t row = q.first + (query0 + m) / group;
        return tree_window(a.tree_mask + (uint64_t)row * a.mask_words, tree, key0);
      };
#pragma unroll
      for (uint32_t mt = 0; mt < MT; ++mt) {
        // sc[kt][mt][e]: key 16 kt + 4 (l / 16) + e of query 16 mt + l % 16.
        uint64_t here = valid;
        if (Tree && upto > least) here &= seen(mt);
        const uint64_t mine = here >> (4 * g4);
        const uint32_t left = limit[mt] > key0 + 4 * g4 ? limit[mt] - (key0 + 4 * g4) : 0;
        float top = -INFINITY;
#pragma unroll
        for (uint32_t kt = 0; kt < kKT; ++kt)
#pragma unroll
          for (uint32_t e = 0; e < 4; ++e) {
            const uint32_t x = 16 * kt + e;
            sc[kt][mt][e] = (mine >> x & 1) && x < left ? sc[kt][mt][e] * scale_log2 : -INFINITY;
            top = fmaxf(top, sc[kt][mt][e]);
          }
        top = max_of_query(top);
        const float m_new = fmaxf(m_run[mt], top);
        const float m_use = m_new == -INFINITY ? 0.0f : m_new;  // no NaN from (-inf) - (-inf)
        const float alpha = __builtin_amdgcn_exp2f(m_run[mt] - m_use);
        m_run[mt] = m_new;
        float sum = 0.0f;
#pragma unroll
        for (uint32_t kk = 0; kk < kHalves; ++kk)
#pragma unroll
          for (uint32_t e = 0; e < 8; ++e) {
            const float p = __builtin_amdgcn_exp2f(sc[2 * kk + e / 4][mt][e % 4] - m_use);
            high[kk][mt][e] = (half_t)p;
            // What the second product sees: equal values come out as they are.
            sum += C::kTwoHalves ? p : (float)high[kk][mt][e];
            low[kk][mt][e] = C::kTwoHalves ? (half_t)(p - (float)high[kk][mt][e]) : (half_t)0.0f;
          }
        l_run[mt] = l_run[mt] * alpha + sum;
#pragma unroll
        for (uint32_t dt = 0; dt < kDT; ++dt) o[dt][mt] *= alpha;
      }
      __builtin_amdgcn_sched_barrier(0);
      if (upto > least && has_non_finite<kTile>(lv)) {
        auto weight = [&](uint32_t kk, uint32_t mt, uint32_t e) __attribute__((always_inline)) {
          return (float)high[kk][mt][e] + (float)low[kk][mt][e];
        };
        auto chunk = [&](uint32_t row, uint32_t column) __attribute__((always_inline)) {
          return row * kRowBytes + (((column / 8) ^ tile_swizzle<D>(row)) << 4) + column % 8 * 2;
        };
        if constexpr (Tree) {
          std::conditional_t<kKeys == 64, uint64_t, uint32_t> bits[MT];
#pragma unroll
          for (uint32_t mt = 0; mt < MT; ++mt) bits[mt] = seen(mt);
          add_non_finite<kHalves, kDT, MT>(o, weight, lv, chunk, limit, key0,
                                           [&](uint32_t mt, uint32_t row) __attribute__((always_inline)) { return bits[mt] >> row & 1; });
        } else {
          add_non_finite<kHalves, kDT, MT>(o, weight, lv, chunk, limit, key0);
        }
        clear_non_finite<kTile>(lv, lane, kWave);
      }
      uint32_t vbase_v = vbase;
      asm volatile("" : "+v"(vbase_v));
#pragma unroll
      for (uint32_t kk = 0; kk < kHalves; ++kk)
#pragma unroll
        for (uint32_t dt = 0; dt < kDT; ++dt) {
          // The chunks of column tile dt: its number XORed in, or added where rows are not swizzled.
          constexpr bool kSwizzled = D == 64 || D == 128 || D == 256;
          const uint8_t* p = lv + (kSwizzled ? vbase_v ^ (dt << 5) : vbase_v + (dt << 5)) + 32 * kk * kRowBytes;
          const short4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LDS_AS short4_t*)p);
          const short4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LDS_AS short4_t*)(p + 16 * kRowBytes));
          const half8_t v = __builtin_bit_cast(half8_t, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
          for (uint32_t mt = 0; mt < MT; ++mt) {
            o[dt][mt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, high[kk][mt], o[dt][mt], 0, 0, 0);
            if constexpr (C::kTwoHalves)
              o[dt][mt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, low[kk][mt], o[dt][mt], 0, 0, 0);
          }
        }
    };
    // What this wave has asked for has arrived, and its reads of the other
    // stage are done.
    auto settle = [&]() __attribute__((always_inline)) {
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    };

    const uint32_t stride = alone ? 1 : kWaves;
    uint32_t t = tile_first + (alone ? 0 : wave);
    if (t < tile_last) {
      int page = page_at(t, entry(t));
      int e = entry(t + stride);
      uint64_t valid = __ballot(page >= 0);
      fetch_values(t, page, my0);
      fetch_keys(t, page);
      // One tile: the next one's values on their way, the scores, the next one's keys on
      // their way into the registers just read, the rest.
      auto step = [&](uint8_t* lv, uint8_t* next) __attribute__((always_inline)) {
        settle();
        page = page_at(t + stride, e);
        e = entry(t + 2 * stride);
        fetch_values(t + stride, page, next);
        float4_t sc[kKT][MT];
        scores(sc);
        fetch_keys(t + stride, page);
        update(t, valid, sc, lv);
        valid = __ballot(page >= 0);
        t += stride;
      };
      while (true) {
        step(my0, my1);
        if (t >= tile_last) break;
        step(my1, my0);
        if (t >= tile_last) break;
      }
    }
    settle();

    // ---- the waves' results joined ----
    // Lane numbers made opaque, so that nothing of this is computed before the key loop.
    const uint32_t tid = opaque(threadIdx.x), r16 = tid % 16, g4 = tid % kWave / 16;
    // (row, head) of query m, for the shared keys' parts and the output.
    auto output_row = [&](uint32_t m) __attribute__((always_inline)) {
      const uint32_t row = (query0 + m) / group;
      return (uint64_t)(q.first + row) * a.query_heads + key_head * group + (query0 + m - row * group);
    };
    if (alone) {  // nothing to join but the shared keys' parts
#pragma unroll
      for (uint32_t mt = 0; mt < MT; ++mt) {
        const uint32_t m = 16 * mt + r16;
        const uint64_t at = output_row(m < queries ? m : queries - 1);
        const float l = sum_of_query(l_run[mt]);
        float inverse = l == 0.0f ? 0.0f : 1.0f / l;
        if constexpr (Shared && D <= 128) {
          // A query's four lanes hold every fourth part's weight.
          constexpr uint32_t kHeld = kMaxSharedParts / 4, kAtOnce = MT == 1 ? 4 : 2;
          float w[kHeld], sums[kHeld], top = m_run[mt], sum = 0.0f;
#pragma unroll
          for (uint32_t j = 0; j < kHeld; ++j) {
            const uint32_t z = 4 * j + g4;
            const float* pair = shared.sums + (at * shared.parts + (z < shared.parts ? z : 0)) * 2;
            w[j] = pair[0];
            sums[j] = pair[1];
          }
#pragma unroll
          for (uint32_t j = 0; j < kHeld; ++j) {
            w[j] = 4 * j + g4 < shared.parts ? w[j] : -INFINITY;
            top = fmaxf(top, w[j]);
          }
          top = max_of_query(top);
          top = top == -INFINITY ? 0.0f : top;
#pragma unroll
          for (uint32_t j = 0; j < kHeld; ++j) {
            w[j] = __builtin_amdgcn_exp2f(w[j] - top);
            sum += 4 * j + g4 < shared.parts ? w[j] * sums[j] : 0.0f;
          }
          const float own = __builtin_amdgcn_exp2f(m_run[mt] - top);
          sum = sum_of_query(sum) + own * l;
          inverse = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
          for (uint32_t dt = 0; dt < kDT; ++dt) o[dt][mt] *= own;
          const float* from = shared.rows + at * shared.parts * a.width;
#pragma unroll
          for (uint32_t j = 0; j < kHeld; ++j)
#pragma unroll
            for (uint32_t z0 = 0; z0 < 4; z0 += kAtOnce) {  // parts, whose loads are in flight together
              if (4 * j + z0 >= shared.parts) break;
              float4_t y[kAtOnce][kDT];
#pragma unroll
              for (uint32_t k = 0; k < kAtOnce; ++k) {
                const uint32_t z = 4 * j + z0 + k < shared.parts ? 4 * j + z0 + k : shared.parts - 1;
#pragma unroll
                for (uint32_t dt = 0; dt < kDT; ++dt) {
                  const uint32_t d = 16 * dt + 4 * g4;
                  y[k][dt] = *reinterpret_cast<const float4_t*>(from + z * a.width + (d < a.width ? d : 0));
                }
              }
#pragma unroll
              for (uint32_t k = 0; k < kAtOnce; ++k) {
                const float weight = __shfl(w[j], 16 * (z0 + k) + r16, kWave);
                if (4 * j + z0 + k < shared.parts) {
#pragma unroll
                  for (uint32_t dt = 0; dt < kDT; ++dt) o[dt][mt] += y[k][dt] * weight;
                }
              }
            }
        }
#pragma unroll
        for (uint32_t dt = 0; dt < kDT; ++dt) {
          const uint32_t d = 16 * dt + 4 * g4;
          half4_t h;
#pragma unroll
          for (int e = 0; e < 4; ++e) h[e] = (half_t)(o[dt][mt][e] * inverse);
          if (m < queries && d < a.width) *reinterpret_cast<half4_t*>((half_t*)a.out + at * a.width + d) = h;
        }
      }
      unit = stop;
      continue;
    }
    // A wave's rows, fp32 [kQueries][D], fill its stage 0 and 1 (16 rows of each).
    static_assert(16 * D * 4 <= kTile, "a stage holds 16 rows");
#pragma unroll
    for (uint32_t mt = 0; mt < MT; ++mt) {
      const float l = sum_of_query(l_run[mt]);
      if (g4 == 0) {
        wave_sums[wave][16 * mt + r16][0] = m_run[mt];
        wave_sums[wave][16 * mt + r16][1] = l;
      }
      float* mine = reinterpret_cast<float*>(mt == 0 ? my0 : my1) + r16 * D;
#pragma unroll
      for (uint32_t dt = 0; dt < kDT; ++dt)
        *reinterpret_cast<float4_t*>(mine + ((dt * 4 + g4) ^ (r16 & 7)) * 4) = o[dt][mt];
    }
    const uint32_t real = queries < kQueries ? queries : kQueries;
    __syncthreads();
    const uint32_t quads = a.width / 4;
    auto wave_quad = [&](uint32_t w, uint32_t m, uint32_t c) __attribute__((always_inline)) {
      const float* from = reinterpret_cast<const float*>((m < 16 ? stage0 : stage1) + w * kTile) + (m % 16) * D;
      return *reinterpret_cast<const float4_t*>(from + (c ^ (m & 7)) * 4);
    };
    auto store = [&](uint32_t m, uint32_t c, float4_t x) __attribute__((always_inline)) {
      half4_t h;
#pragma unroll
      for (int e = 0; e < 4; ++e) h[e] = (half_t)x[e];
      *reinterpret_cast<half4_t*>((half_t*)a.out + output_row(m) * a.width + c * 4) = h;
    };
    // Weights of `parts` results and of the shared keys' parts of each query,
    // exp2(m - max m) / sum, of which `load` gives the (reference point, sum) pairs: a
    // thread loads a pair, a wave folds a query.
    auto weigh = [&](float* weights, float* sums, uint32_t most, uint32_t parts, auto load) __attribute__((always_inline)) {
      const uint32_t all = parts + shared.parts;
      for (uint32_t i = tid; i < real * all; i += kThreads) {
        const uint32_t m = i / all, z = i - m * all;
        const float* pair = shared.sums + (output_row(m) * shared.parts + (z - parts)) * 2;
        weights[m * most + z] = z < parts ? load(z, m, 0) : pair[0];
        sums[m * most + z] = z < parts ? load(z, m, 1) : pair[1];
      }
      __syncthreads();
      for (uint32_t m = wave; m < real; m += kWaves) {
        float* w = weights + m * most;
        float top = -INFINITY, sum = 0.0f;
        for (uint32_t z = lane; z < all; z += kWave) top = fmaxf(top, w[z]);
        for (uint32_t o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, kWave));
        top = top == -INFINITY ? 0.0f : top;
        for (uint32_t z = lane; z < all; z += kWave) sum += __builtin_amdgcn_exp2f(w[z] - top) * sums[m * most + z];
        sum = wave_sum(sum);
        const float inverse = sum == 0.0f ? 0.0f : 1.0f / sum;
        for (uint32_t z = lane; z < all; z += kWave) w[z] = __builtin_amdgcn_exp2f(w[z] - top) * inverse;
      }
      __syncthreads();
    };
    auto shared_quads = [&](const float* w, uint32_t m, uint32_t c, float4_t x) __attribute__((always_inline)) {
      const float* from = shared.rows + output_row(m) * shared.parts * a.width + c * 4;
      for (uint32_t z0 = 0; z0 < shared.parts; z0 += 8) {  // eight loads in flight
        float4_t y[8];
#pragma unroll
        for (uint32_t j = 0; j < 8; ++j) {
          const uint32_t z = z0 + j < shared.parts ? z0 + j : shared.parts - 1;
          y[j] = *reinterpret_cast<const float4_t*>(from + (uint64_t)z * a.width);
        }
#pragma unroll
        for (uint32_t j = 0; j < 8; ++j)
          if (z0 + j < shared.parts) x += y[j] * w[z0 + j];
      }
      return x;
    };

    if (tile_last - tile_first == u.tiles) {  // the whole segment
      weigh(few_weights, few_sums, kFewParts, kWaves, [&](uint32_t z, uint32_t m, uint32_t which) { return wave_sums[z][m][which]; });
      for (uint32_t i = tid; i < real * quads; i += kThreads) {
        const uint32_t m = i / quads, c = i % quads;
        float4_t x = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (uint32_t w = 0; w < kWaves; ++w) x += wave_quad(w, m, c) * few_weights[m * kFewParts + w];
        store(m, c, shared_quads(few_weights + m * kFewParts + kWaves, m, c, x));
      }
    } else {
      // This part's slot: by its unit; cut into chunks, 2 w of workgroup w for the segment
      // in which its chunk begins, 2 w + 1 for one that begins later in it.
      const bool chunks = shares.part_tiles == 0;
      const uint64_t first_part = chunks ? quotient(segment_begin, shares.chunk) : segment_begin;
      const uint64_t last_part = chunks ? quotient(segment_end - 1, shares.chunk) : segment_end - 1;
      const uint32_t parts = (uint32_t)(last_part - first_part) + 1;
      auto slot_of = [&](uint64_t w) { return chunks ? 2 * w + (segment_begin > w * shares.chunk ? 1 : 0) : w; };
      const uint64_t slot = slot_of(chunks ? blockIdx.x : unit);
      float* rows = split.rows + slot * kQueries * D;
      float* sums = split.sums + slot * kQueries * 2;
      for (uint32_t i = tid; i < real * quads; i += kThreads) {
        const uint32_t m = i / quads, c = i % quads;
        float top = -INFINITY;
#pragma unroll
        for (uint32_t w = 0; w < kWaves; ++w) top = fmaxf(top, wave_sums[w][m][0]);
        const float use = top == -INFINITY ? 0.0f : top;
        float4_t x = {0.0f, 0.0f, 0.0f, 0.0f};
        float l = 0.0f;
#pragma unroll
        for (uint32_t w = 0; w < kWaves; ++w) {
          const float f = __builtin_amdgcn_exp2f(wave_sums[w][m][0] - use);
          l += f * wave_sums[w][m][1];
          x += wave_quad(w, m, c) * f;
        }
        store_device4(rows + m * D + c * 4, x);
        if (c == 0) {
          store_device(sums + 2 * m, top);
          store_device(sums + 2 * m + 1, l);
        }
      }
      if (arrive(split.counters + first_part, parts, &arrived)) {
        float* weights = reinterpret_cast<float*>(stage0);
        weigh(weights, reinterpret_cast<float*>(stage1), kManyParts, parts, [&](uint32_t z, uint32_t m, uint32_t which) {
          return load_device(split.sums + (slot_of(first_part + z) * kQueries + m) * 2 + which);
        });
        for (uint32_t i = tid; i < real * quads; i += kThreads) {
          const uint32_t m = i / quads, c = i % quads;
          const float* w = weights + m * kManyParts;
          float4_t x = {0.0f, 0.0f, 0.0f, 0.0f};
          // Eight loads in flight (past the last part: the last one again, not added).
          for (uint32_t z0 = 0; z0 < parts; z0 += 8) {
            float4_t y[8];
#pragma unroll
            for (uint32_t j = 0; j < 8; ++j) {
              const uint32_t z = z0 + j < parts ? z0 + j : parts - 1;
              y[j] = load_device4(split.rows + (slot_of(first_part + z) * kQueries + m) * D + c * 4);
            }
#pragma unroll
            for (uint32_t j = 0; j < 8; ++j)
              if (z0 + j < parts) x += y[j] * w[z0 + j];
          }
          store(m, c, shared_quads(w + parts, m, c, x));
        }
      }
    }
    __syncthreads();  // the stages, sums and weights are free for the next segment
    unit = stop;
  }
}

int launch_general(hipStream_t stream, const PagedAttentionArgs& a, float scale_log2) {
  constexpr uint32_t kMostRows = 1u << 23;  // a grid dimension holds less than 2^32 threads
  for (uint64_t done = 0; done < a.rows; done += kMostRows) {
    const uint32_t rows = a.rows - done < kMostRows ? (uint32_t)(a.rows - done) : kMostRows;
    if (a.tree_mask)
      hipLaunchKernelGGL(attention_pages_general_kernel<true>, dim3(rows, a.query_heads), dim3(kThreads), 0, stream, a,
                         (uint32_t)done, scale_log2);
    else
      hipLaunchKernelGGL(attention_pages_general_kernel<false>, dim3(rows, a.query_heads), dim3(kThreads), 0, stream, a,
                         (uint32_t)done, scale_log2);
    if (int e = hip_status(hipGetLastError())) return e;
  }
  return 0;
}

// One launch over the sequences of at most `few` queries, keys from first_key on.
struct DecodeLaunch {
  uint32_t first_key;
  uint32_t few;
  SharedParts shared;
};
template <int D, int MT, bool Shared, bool Tree>
int launch_decode_as(hipStream_t stream, const PagedAttentionArgs& a, float scale_log2, const DecodeLaunch& l) {
  constexpr uint64_t kResident = Decode<D, MT>::kResident, kQueries = Decode<D, MT>::kQueries;
  constexpr uint64_t kSlotBytes = kQueries * (D + 2) * sizeof(float);
  // A workgroup per segment (at most a partial query tile more per sequence) and one more per
  // resident one, for segments in parts.
  const uint64_t queries = (uint64_t)a.rows * (a.query_heads / a.key_heads);
  const uint64_t sequences = a.batch.sequences < a.rows ? a.batch.sequences : a.rows;
  uint64_t groups = ((queries + kQueries - 1) / kQueries + sequences) * a.key_heads + kResident;
  if (groups > kMostGroups) groups = kMostGroups;
  DecodeSplit split{nullptr, nullptr, nullptr};
  if (a.workspace.data) {
    const uint64_t fit = a.workspace.bytes / (2 * kSlotBytes);
    const uint64_t most = fit < a.workspace.counter_count ? fit : a.workspace.counter_count;
    if (most >= kResident) {
      if (groups > most) groups = most;
      split.rows = (float*)a.workspace.data;
      split.sums = split.rows + 2 * groups * kQueries * D;
      split.counters = a.workspace.counters;
    }
  }
  hipLaunchKernelGGL((attention_pages_decode_kernel<D, MT, Shared, Tree>), dim3((uint32_t)groups), dim3(kThreads), 0, stream,
                     a, scale_log2, l.first_key, l.few, split, l.shared);
  return hip_status(hipGetLastError());
}
template <int D, bool Shared, bool Tree>
int launch_decode_queries(hipStream_t stream, const PagedAttentionArgs& a, float scale_log2, const DecodeLaunch& l) {
  // Two tiles of queries at 256 columns do not fit the registers.
  if constexpr (D <= 128)
    if ((uint64_t)a.max_rows * (a.query_heads / a.key_heads) > 16) return launch_decode_as<D, 2, Shared, Tree>(stream, a, scale_log2, l);
  return launch_decode_as<D, 1, Shared, Tree>(stream, a, scale_log2, l);
}
template <bool Shared, bool Tree>
int launch_decode_width(hipStream_t stream, const PagedAttentionArgs& a, float scale_log2, const DecodeLaunch& l) {
  if (a.width > 192) return launch_decode_queries<256, Shared, Tree>(stream, a, scale_log2, l);
  if (a.width > 128) return launch_decode_queries<192, Shared, Tree>(stream, a, scale_log2, l);
  if (a.width > 96) return launch_decode_queries<128, Shared, Tree>(stream, a, scale_log2, l);
  if (a.width > 64) return launch_decode_queries<96, Shared, Tree>(stream, a, scale_log2, l);
  if (a.width > 32) return launch_decode_queries<64, Shared, Tree>(stream, a, scale_log2, l);
  return launch_decode_queries<32, Shared, Tree>(stream, a, scale_log2, l);
}
int launch_decode(hipStream_t stream, const PagedAttentionArgs& a, float scale_log2, const DecodeLaunch& l) {
  if (a.tree_mask) return launch_decode_width<false, true>(stream, a, scale_log2, l);
  return l.shared.parts > 0 ? launch_decode_width<true, false>(stream, a, scale_log2, l)
                            : launch_decode_width<false, false>(stream, a, scale_log2, l);
}

// Queries of a key head (rows x query heads) up to which a sequence is the decode kernel's.
// Up to 16, one tile, it is ahead everywhere; of 17 to 32 it wins where there are few
// segments and loses a little where there are many (us, decode / blocks at 32 queries: 16
// sequences x 16 heads x 8000 keys x 128 190 / 220, x 64 118 / 150; 64 x 16 x 2000 x 128
// 228 / 205, 64 x 8 x 2000 x 64 58 / 64); at 48, three tiles or two that read the keys
// twice, it is behind (64 x 16 x 2000 x 128 372 / 206).
constexpr uint32_t kFewQueries = 32;
// Beside sequences of more the blocks' launch is there anyway: only sequences of one tile.
constexpr uint32_t kFewBeside = 16;
// Where the table holds few keys and there are few segments, the blocks take those too: one
// launch, and their time hardly counts (us, one launch / two; a prompt of 100 rows beside
// single ones, 128 columns, 32 query heads on 8: 17 sequences x 256 keys 12.9 / 23.8, x 1000
// 27.8 / 47.9, x 2000 32.1 / 48.2, 65 x 1000 54 / 71; not 17 x 4000 84 / 79, nor 257 x 128 (2056
// segments) 53 / 43; of 64 columns, 16 heads: 65 x 1000 60 / 66, 120 x 1000 (1920) 102 / 98).
// So it is with sequences of 17 to 32 queries alone (24 queries, one launch of blocks / decode:
// 64 x 8 segments x 128 keys x 128 13.2 / 30.9, x 500 27.7 / 44.4, x 1000 54 / 70, 16 x 8 x 2000
// 32 / 36), but not of up to 16 (64 x 16 x 200 x 64 21.8 / 16.0).
constexpr uint32_t kShortReach = 2560, kShortSegments = 1280;

// The shared keys in a launch of their own: their parts in the workspace's lower
// end, what is left to the launch that joins them.  That launch costs 8 us and more
// (it writes the parts), reading the keys once per sequence what the caches give, about
// 14 TB/s: worth it from some 160 MB saved.  Measured at width 128 with 64 keys of their own
// each (us, shared / read per sequence): 8 sequences x 4096 keys x 8 heads (117 MB) 21.7 / 22.2,
// 32 x 1024 x 16 (260 MB) 23.1 / 28.8, 8 x 4096 x 16 (235 MB) 25.6 / 50.4, 128 x 16384 x 8 (8.5 GB)
// 70.9 / 598; not 2 x 16384 x 8 (67 MB) 35.8 / 26.1, 128 x 256 x 8 (134 MB) 34.0 / 29.8.
constexpr uint64_t kSharedSaving = 160u << 20;
bool plan_shared(const PagedAttentionArgs& a, SharedParts* parts, Workspace* rest) {
  if (a.batch.shared_rows == 0 || a.batch.sequences < 2 || !a.workspace.data) return false;
  const uint64_t reach = (uint64_t)a.batch.table_columns * a.batch.page_rows;
  const uint64_t keys = a.batch.shared_rows < reach ? a.batch.shared_rows : reach;
  if ((a.batch.sequences - 1) * keys < kSharedSaving / ((uint64_t)a.key_heads * a.width * 4)) return false;
  const uint64_t row_floats = (uint64_t)a.rows * a.query_heads * (a.width + 2);
  // What stays for the keys behind the shared ones: two slots per resident workgroup.
  const uint64_t queries = (uint64_t)a.max_rows * (a.query_heads / a.key_heads) > 16 && a.width <= 128 ? 32 : 16;
  const uint64_t width = a.width > 128 ? 256 : a.width > 64 ? 128 : 64;  // at least the columns computed
  const uint64_t rest_bytes = 2 * kMostResident * queries * (width + 2) * sizeof(float);
  const uint64_t room = a.workspace.bytes > rest_bytes ? (a.workspace.bytes - rest_bytes) / sizeof(float) : 0;
  const uint64_t most = room / row_floats < kMaxSharedParts ? room / row_floats : kMaxSharedParts;
  parts->parts = most == 0 ? 0 : shared_part_count(a, (uint32_t)most);
  if (parts->parts == 0) return false;
  parts->rows = (float*)a.workspace.data;
  parts->sums = parts->rows + (uint64_t)a.rows * a.query_heads * parts->parts * a.width;
  const uint64_t used = (row_floats * parts->parts * sizeof(float) + 255) & ~255ull;
  *rest = a.workspace;
  rest->data = (uint8_t*)a.workspace.data + used;
  rest->bytes = a.workspace.bytes - used;
  return true;
}

}  // namespace

int launch_attention_pages(hipStream_t stream, const PagedAttentionArgs& a) {
  if (a.rows == 0 || a.batch.sequences == 0) return 0;
  if (((uintptr_t)a.query | (uintptr_t)a.cache | (uintptr_t)a.out) % 2 != 0 ||
      (batch_addresses(a.batch) | (uintptr_t)a.tree_mask) % 4 != 0)
    return IPUS_ERROR_INVALID_ARGUMENT;
  const float scale_log2 = a.scale * kLog2e;
  const bool vectors = a.width % 8 == 0 && a.query_row_stride % 8 == 0 &&
                       ((uintptr_t)a.query | (uintptr_t)a.cache) % 16 == 0 && (uintptr_t)a.out % 8 == 0;
  // A page's bytes fit 32 bits, for the tile loads' addresses, and the batch's queries.
  if (!vectors || a.width > 256 || a.batch.page_elements * 2 > 0xffffffffull ||
      (uint64_t)a.rows * (a.query_heads / a.key_heads) > 0x7fffffffull)
    return launch_general(stream, a, scale_log2);
  const uint64_t queries = (uint64_t)a.max_rows * (a.query_heads / a.key_heads);
  const DecodeLaunch unshared{0, ~0u, {nullptr, nullptr, 0}};
  const bool small = (uint64_t)a.batch.table_columns * a.batch.page_rows <= kShortReach &&
                     (uint64_t)a.batch.sequences * a.key_heads <= kShortSegments;
  if (queries <= (small && a.batch.shared_rows == 0 ? kFewBeside : kFewQueries)) {
    SharedParts parts;
    Workspace rest;
    if (plan_shared(a, &parts, &rest)) {
      if (int e = launch_shared_parts(stream, a, scale_log2, parts)) return e;
      PagedAttentionArgs behind = a;
      behind.workspace = rest;
      return launch_decode(stream, behind, scale_log2, {a.batch.shared_rows, ~0u, parts});
    }
    return launch_decode(stream, a, scale_log2, unshared);
  }
  // Sequences of many rows, and those of few beside them, of which there are none
  // where every sequence has max_rows.
  if (small || (uint64_t)a.batch.sequences * a.max_rows == a.rows)
    return launch_attention_blocks(stream, a, scale_log2, 0);
  if (int e = launch_attention_blocks(stream, a, scale_log2, kFewBeside)) return e;
  PagedAttentionArgs beside = a;
  beside.max_rows = 1;  // one tile of queries
  return launch_decode(stream, beside, scale_log2, {0, kFewBeside, {nullptr, nullptr, 0}});
}

}  // namespace ipus
