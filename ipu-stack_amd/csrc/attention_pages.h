// Device helpers of the paged attention kernels: loads that need no branch, LDS tiles,
// and the scan that finds a workgroup's place in a ragged batch.
#pragma once

#include "../../include/ipus.h"
#include "kernels.h"
#include "pages.h"
#include "wave_scan.h"

#define LDS_AS __attribute__((address_space(3)))
#define GLOBAL_AS __attribute__((address_space(1)))
typedef short short4_t __attribute__((vector_size(8)));

namespace ipus {

constexpr uint32_t kThreads = 256;
constexpr uint32_t kWaves = kThreads / kWave;

constexpr float kLog2e = 1.4426950408889634f;

inline int hip_status(hipError_t e) { return e == hipSuccess ? 0 : IPUS_ERROR_HIP_BASE - (int)e; }

// 16 bytes of zeros: what a lane loads for keys that are not to be read and for columns
// past the width, so that loads need no branch (with branches the compiler cannot count
// them and waits for all) and nothing that is not the sequence's meets a product.
alignas(16) __device__ const uint32_t kZeros[4] = {0, 0, 0, 0};

// LDS rows of D fp16, 16-byte chunk c of row r at chunk c ^ value_swizzle(r): both the DMA's
// 64 chunks and ds_read_b64_tr_b16's (4 rows x 32 bytes per 16 lanes) touch every bank once.
template <int D>
__device__ __forceinline__ uint32_t value_swizzle(uint32_t row) {
  return D >= 128 ? (row & 7u) << 1 : row & 7u;
}

// Loads from addresses as numbers, of global memory (without the address space they
// would be flat loads, which count as LDS accesses too).
__device__ __forceinline__ void dma16(uint64_t from, uint8_t* lds) {
  __builtin_amdgcn_global_load_lds((const GLOBAL_AS void*)from, (LDS_AS void*)lds, 16, 0, 0);
}
__device__ __forceinline__ u32x4 load16_at(uint64_t from) { return *(const GLOBAL_AS u32x4*)from; }
// at if use, else otherwise, selected without a branch.
__device__ __forceinline__ uint64_t pick(bool use, uint64_t at, uint64_t otherwise) {
  asm volatile("" : "+v"(at));
  return use ? at : otherwise;
}

__device__ __forceinline__ float max_of_query(float x) {  // the four lanes that hold one query
  x = fmaxf(x, __shfl_xor(x, 16, kWave));
  return fmaxf(x, __shfl_xor(x, 32, kWave));
}
__device__ __forceinline__ float sum_of_query(float x) {
  x += __shfl_xor(x, 16, kWave);
  return x + __shfl_xor(x, 32, kWave);
}

__device__ __forceinline__ BatchSequence uniform(BatchSequence q) {
  return {uniform(q.first), uniform(q.rows), uniform(q.keys), (int)uniform((uint32_t)q.length), (int)uniform((uint32_t)q.end)};
}

// Quotient of values that mostly fit 32 bits (a 64-bit division takes about 100
// instructions).
__device__ __forceinline__ uint64_t quotient(uint64_t x, uint64_t y) {
  return ((x | y) >> 32) == 0 ? (uint32_t)x / (uint32_t)y : x / y;
}

// The batch's work as one line of units, `units(sequence)` of them for each in turn:
// how many there are, and the sequence that holds unit `at` (with its first unit).
// Used by whole waves.  The lengths of up to 64 sequences are read once.
struct UnitLine {
  uint64_t upto, total;  // units up to and with this lane's sequence of the first 64; of all
};
template <typename F>
__device__ __forceinline__ UnitLine count_units(const PagedBatch& b, F units) {
  const uint32_t lane = threadIdx.x % kWave;
  UnitLine l;
  l.upto = scan(lane < b.sequences ? units(lane) : 0);
  l.total = from_lane(l.upto, kWave - 1);
  if (b.sequences > (uint32_t)kWave) {
    uint64_t more = 0;
    for (uint32_t s = kWave + lane; s < b.sequences; s += kWave) more += units(s);
    l.total += from_lane(scan(more), kWave - 1);
  }
  return l;
}
struct UnitPlace {
  uint32_t sequence;
  uint64_t first;
};
template <typename F>
__device__ __forceinline__ UnitPlace find_unit(const PagedBatch& b, const UnitLine& line, uint64_t at, F units) {
  const uint32_t lane = threadIdx.x % kWave;
  UnitPlace p{0, 0};
  uint64_t upto = line.upto;
  while (true) {
    const uint64_t all = from_lane(upto, kWave - 1);
    if (at < p.first + all) break;
    p.first += all;
    p.sequence += kWave;
    if (p.sequence >= b.sequences) break;  // not in the line
    upto = scan(p.sequence + lane < b.sequences ? units(p.sequence + lane) : 0);
  }
  const uint64_t past = __ballot(p.first + upto > at);
  const uint32_t holder = past ? (uint32_t)__builtin_ctzll(past) : 0;
  p.sequence += holder;
  if (holder > 0) p.first += from_lane(upto, holder - 1);
  return p;
}

// Non-finite values.  A key that a row may not read has probability 0 there, and 0 times a
// non-finite value would be NaN, so that one bad value would spoil the rows of a tile that
// stand before it.  Tiles with a key that some of a wave's queries may not read are
// therefore looked through; where one holds such a value, its products are added one by one to the
// rows that read it, and the value is cleared before the tile's MFMAs.
__device__ __forceinline__ uint32_t non_finite_halves(uint32_t x) {  // the top bit of each such half
  return ((x & 0x7c007c00u) + 0x04000400u) & 0x80008000u;            // an exponent of all ones carries
}
template <uint32_t Bytes>
__device__ __forceinline__ bool has_non_finite(const uint8_t* tile) {  // fp16, by one wave
  uint32_t found = 0;
#pragma unroll
  for (uint32_t i = 0; i < Bytes / (16 * kWave); ++i) {
    const u32x4 x = *reinterpret_cast<const u32x4*>(tile + (i * kWave + threadIdx.x % kWave) * 16);
#pragma unroll
    for (int w = 0; w < 4; ++w) found |= non_finite_halves(x[w]);
  }
  return __any(found != 0);
}
// Clears them, `threads` threads together, this one `thread`.
template <uint32_t Bytes>
__device__ __forceinline__ void clear_non_finite(uint8_t* tile, uint32_t thread, uint32_t threads) {
#pragma unroll 1
  for (uint32_t i = thread; i < Bytes / 16; i += threads) {
    u32x4 x = *reinterpret_cast<const u32x4*>(tile + i * 16);
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const uint32_t f = non_finite_halves(x[w]);
      x[w] &= ~((f >> 15) * 0xffffu);
    }
    *reinterpret_cast<u32x4*>(tile + i * 16) = x;
  }
}
// Adds the products of a tile's non-finite values, in the layout of the kernels' MFMAs: o[dt][qt][c]
// is column 16 dt + 4 (l / 16) + c of query 16 qt + l % 16, and p(kk, qt, e) the probability of
// key 32 kk + 4 (l / 16) + e % 4 + 16 (e / 4).  chunk(row, column): where 4 columns lie in the tile;
// this lane's query reads the keys below its limit that named(qt, row) names, by their row of the tile.
struct AllNamed {
  __device__ __forceinline__ bool operator()(uint32_t, uint32_t) const { return true; }
};
template <uint32_t Halves, uint32_t DT, uint32_t QT, typename P, typename Chunk, typename Named = AllNamed>
__device__ __forceinline__ void add_non_finite(float4_t (&o)[DT][QT], P p, const uint8_t* tile, Chunk chunk,
                                               const uint32_t (&limit)[QT], uint32_t key0, Named named = {}) {
#pragma unroll
  for (uint32_t kk = 0; kk < Halves; ++kk)
#pragma unroll
    for (uint32_t e = 0; e < 8; ++e)
#pragma unroll 1
      for (uint32_t g = 0; g < 4; ++g) {
        uint32_t lane = threadIdx.x % kWave;
        asm volatile("" : "+v"(lane));  // nothing of this is kept in registers
        const uint32_t r16 = lane % 16, g4 = lane / 16;
        const uint32_t row = 32 * kk + 4 * g + e % 4 + 16 * (e / 4);
        float w[QT];
#pragma unroll
        for (uint32_t qt = 0; qt < QT; ++qt) w[qt] = __shfl(p(kk, qt, e), 16 * g + r16, kWave);
#pragma unroll
        for (uint32_t dt = 0; dt < DT; ++dt) {
          __builtin_amdgcn_sched_barrier(0);
          const half4_t x = *reinterpret_cast<const half4_t*>(tile + chunk(row, 16 * dt + 4 * g4));
#pragma unroll
          for (uint32_t c = 0; c < 4; ++c) {
            const float v = (float)x[c];
            const bool bad = !(fabsf(v) <= 65504.0f);
#pragma unroll
            for (uint32_t qt = 0; qt < QT; ++qt) o[dt][qt][c] += bad && key0 + row < limit[qt] && named(qt, row) ? w[qt] * v : 0.0f;
          }
        }
      }
}

// Results over the shared keys, from a launch before the one that joins them: for
// every (row, query head) `parts` unnormalised rows and (reference point, sum) pairs.
struct SharedParts {
  float* rows;
  float* sums;
  uint32_t parts;
};
constexpr uint32_t kMaxSharedParts = 32;
constexpr uint32_t kFullChip = 512;  // workgroups that the chip holds at once, two per CU

// The kernels for many query rows per key head (k_attention_blocks.hip): sequences of more
// than `few` queries (rows x query heads of a key head); and the rows of the whole
// batch over the shared keys alone.  shared_part_count: into how many parts, at
// most `most`, those keys are split to fill the chip.
int launch_attention_blocks(hipStream_t stream, const PagedAttentionArgs& a, float scale_log2, uint32_t few);
int launch_shared_parts(hipStream_t stream, const PagedAttentionArgs& a, float scale_log2, const SharedParts& parts);
uint32_t shared_part_count(const PagedAttentionArgs& a, uint32_t most);

}  // namespace ipus
