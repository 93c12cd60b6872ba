// Wave-wide scalars, sums and maxima of 32 and 64 bits, by lane moves alone.
#pragma once

#include "device_common.h"

namespace ipus {

// Values that all lanes hold alike, into scalar registers.
__device__ __forceinline__ uint32_t uniform(uint32_t x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ uint64_t uniform(uint64_t x) {
  return uniform((uint32_t)x) | (uint64_t)uniform((uint32_t)(x >> 32)) << 32;
}
__device__ __forceinline__ uint64_t from_lane(uint64_t x, uint32_t lane) {  // lane: alike in all lanes
  return (uint32_t)__builtin_amdgcn_readlane((uint32_t)x, lane) |
         (uint64_t)(uint32_t)__builtin_amdgcn_readlane((uint32_t)(x >> 32), lane) << 32;
}
// x of the lane that the DPP control names, 0 where there is none.
template <int Control, int RowMask>
__device__ __forceinline__ uint32_t neighbour(uint32_t x) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, Control, RowMask, 0xf, false);
}
template <int Control, int RowMask>
__device__ __forceinline__ uint64_t neighbour(uint64_t x) {
  return neighbour<Control, RowMask>((uint32_t)x) | (uint64_t)neighbour<Control, RowMask>((uint32_t)(x >> 32)) << 32;
}
// Sum over the lanes up to this one, and the largest of all lanes: four steps inside rows
// of 16 lanes (row_shr), then the rows before (row_bcast:15 and :31).
template <typename T>
__device__ __forceinline__ T scan(T x) {
  x += neighbour<0x111, 0xf>(x);
  x += neighbour<0x112, 0xf>(x);
  x += neighbour<0x114, 0xf>(x);
  x += neighbour<0x118, 0xf>(x);
  x += neighbour<0x142, 0xa>(x);
  x += neighbour<0x143, 0xc>(x);
  return x;
}
template <int Control, int RowMask>
__device__ __forceinline__ uint32_t larger(uint32_t x) {
  const uint32_t y = neighbour<Control, RowMask>(x);
  return x > y ? x : y;
}
__device__ __forceinline__ uint32_t largest(uint32_t x) {
  x = larger<0x111, 0xf>(x);
  x = larger<0x112, 0xf>(x);
  x = larger<0x114, 0xf>(x);
  x = larger<0x118, 0xf>(x);
  x = larger<0x142, 0xa>(x);
  x = larger<0x143, 0xc>(x);
  return (uint32_t)__builtin_amdgcn_readlane(x, kWave - 1);
}

}  // namespace ipus
