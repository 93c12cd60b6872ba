// Rotary positions on gfx950: the rotation of query and key heads, the norm of
// those heads with the rotation in the same pass, and the append of keys (rotated
// on the way) and values to a paged cache.
//
// Pair i of a head at position p turns by the angle t = p f_i:
//   a' = m (a cos t - b sin t),  b' = m (b cos t + a sin t)
// with (a, b) = (x[i], x[i + r / 2]) in the half layout and (x[2 i], x[2 i + 1])
// in the interleaved one, r the rotated width, m a magnitude; elements from r on
// are copied.  The norm is y = x w / sqrt(mean(x^2) + epsilon) over the head.
//
// Bound by memory: every element is read once and written once, in 16-byte
// accesses where widths, strides and addresses allow.  An angle serves every head
// of its row, so a workgroup takes whole rows, computes their sines and cosines
// once (the angle in 64 bits: p f_i passes 2^20 rad in long contexts, where fp32
// holds 2^-4) into LDS, with the first elements' loads already under way.
//
// Measured against a copy's 6.3 TB/s: 16384 rows x 16 heads x 128 fp32 43.5 us (6.2 TB/s);
// 16384 rows x 40 heads x 128 fp16 with the norm 58.2 us (5.8: the sum over the head stands
// between its loads and stores); 32000 rows x 8 key heads x 128 into pages 37.8 us (5.3 of the rows
// in use: a row's keys and values go to 16 places).  A step of few rows takes 4.2 to 4.5 us,
// 2.8 to 3.7 of them on the GPU: a launch and four loads that wait for each other.
#include "../../include/ipus.h"
#include "kernels.h"
#include "pages.h"

#include <type_traits>

namespace ipus {
namespace {

constexpr uint32_t kThreads = 256;
constexpr uint32_t kMaxRows = 32;  // of a workgroup

inline int hip_status(hipError_t e) { return e == hipSuccess ? 0 : IPUS_ERROR_HIP_BASE - (int)e; }

template <typename T, int V>
struct alignas(V * sizeof(T)) Pack {
  T e[V];
};

// A chunk as one word, read and written once: non-temporal accesses (a copy of 268 MB:
// 6.3 TB/s with them, 5.0-5.8 without).
template <int Bytes> struct Word;
template <> struct Word<16> { typedef u32x4 type; };
template <> struct Word<8> { typedef u32x2 type; };
template <> struct Word<4> { typedef uint32_t type; };
template <> struct Word<2> { typedef uint16_t type; };
template <typename P>
__device__ __forceinline__ P load_once(const void* p) {
  typedef typename Word<sizeof(P)>::type W;
  return __builtin_bit_cast(P, __builtin_nontemporal_load(reinterpret_cast<const W*>(p)));
}
template <typename P>
__device__ __forceinline__ void store_once(void* p, const P& x) {
  typedef typename Word<sizeof(P)>::type W;
  __builtin_nontemporal_store(__builtin_bit_cast(W, x), reinterpret_cast<W*>(p));
}

// cos and sin of position x frequency.  The angle is reduced to a quarter turn
// in 64 bits: (position f / 2 pi) has 52 bits, of which a position below 2^31
// and f <= 1 leave 23 behind the point.  The reduced angle's series up to r^9
// and r^10 are within 2^-29 for |r| <= pi / 4.
__device__ __forceinline__ void cos_sin(int position, float frequency, float* c, float* s) {
  const double turns = (double)position * ((double)frequency * 0.15915494309189533577);
  const double part = turns - __builtin_rint(turns);  // exact, |part| <= 1/2
  const double quarter = __builtin_rint(4.0 * part);
  const float r = (float)((4.0 * part - quarter) * 1.57079632679489661923);
  const int k = (int)quarter;
  const float z = r * r;
  const float sr = fmaf(r * z, fmaf(z, fmaf(z, fmaf(z, 1.0f / 362880, -1.0f / 5040), 1.0f / 120), -1.0f / 6), r);
  const float cr = fmaf(z, fmaf(z, fmaf(z, fmaf(z, fmaf(z, -1.0f / 3628800, 1.0f / 40320), -1.0f / 720), 1.0f / 24), -0.5f), 1.0f);
  const float sk = k & 1 ? cr : sr, ck = k & 1 ? sr : cr;
  *s = k & 2 ? -sk : sk;
  *c = (k + 1) & 2 ? -ck : ck;
}

// A head is cut into units of two chunks of V elements each, half a part apart, so that
// neighbouring lanes access neighbouring chunks: first the units of the rotated part,
// whose chunks hold the two sides of V pairs (half) or V / 2 pairs each (interleaved;
// for V = 1 the two elements of a pair), then those of the copied part.  With an odd
// number of copied elements (V = 1) the last unit has no second chunk.
struct Unit {
  uint32_t a, b;  // first elements of the chunks
  bool turned, second;
};
template <int V, bool Interleaved>
__device__ __forceinline__ Unit unit_at(uint32_t u, uint32_t half, uint32_t width) {
  const uint32_t turned = half / V;
  Unit n;
  n.turned = u < turned;
  if (n.turned) {
    n.a = Interleaved && V == 1 ? 2 * u : u * V;
    n.b = Interleaved && V == 1 ? n.a + 1 : n.a + half;
  } else {
    n.a = 2 * half + (u - turned) * V;
    n.b = n.a + (width - 2 * half + 1) / 2;
  }
  n.second = V > 1 || n.b < width;
  return n;
}

// Turns the chunks of unit `index` by the cosines and sines of its row (results unrounded).
template <int V, bool Interleaved>
__device__ __forceinline__ void turn(float (&a)[V], float (&b)[V], uint32_t index, uint32_t half, const float* c,
                                     const float* s) {
  if constexpr (Interleaved && V > 1) {
    const uint32_t ia = index * V / 2, ib = ia + half / 2;
#pragma unroll
    for (int e = 0; e < V; e += 2) {
      const float xa = a[e], ya = a[e + 1], xb = b[e], yb = b[e + 1];
      a[e] = xa * c[ia + e / 2] - ya * s[ia + e / 2];
      a[e + 1] = ya * c[ia + e / 2] + xa * s[ia + e / 2];
      b[e] = xb * c[ib + e / 2] - yb * s[ib + e / 2];
      b[e + 1] = yb * c[ib + e / 2] + xb * s[ib + e / 2];
    }
  } else {
    const uint32_t i = index * V;
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const float x = a[e], y = b[e];
      a[e] = x * c[i + e] - y * s[i + e];
      b[e] = y * c[i + e] + x * s[i + e];
    }
  }
}

template <typename T, int V>
__device__ __forceinline__ void widen(const Pack<T, V>& p, float (&x)[V]) {
#pragma unroll
  for (int e = 0; e < V; ++e) x[e] = (float)p.e[e];
}
template <typename T, int V>
__device__ __forceinline__ Pack<T, V> narrow(const float (&x)[V]) {
  Pack<T, V> p;
#pragma unroll
  for (int e = 0; e < V; ++e) p.e[e] = (T)x[e];
  return p;
}

// Lane groups of `lanes` (a power of two, at most a wave) walk the heads of the
// workgroup's rows: (row, head) and the step to this group's next one.
struct Walk {
  uint32_t row, head, heads, step;
  __device__ __forceinline__ Walk(uint32_t slot, uint32_t heads_, uint32_t step_)
      : row(slot / heads_), head(slot % heads_), heads(heads_), step(step_) {}
  __device__ __forceinline__ void next() {
    head += step;
    while (head >= heads) {
      head -= heads;
      ++row;
    }
  }
};

// trig: cos of pair i of the workgroup's row r at [r * half + i], sin behind all
// of them.  Called by all threads.
template <typename Position>
__device__ __forceinline__ void fill_trig(float* trig, uint32_t rows, uint32_t half, float magnitude,
                                          const float* frequencies, Position position) {
  const uint32_t count = rows * half;
  for (uint32_t i = threadIdx.x; i < count; i += kThreads) {
    const uint32_t r = i / half;
    float c, s;
    cos_sin(position(r), frequencies[i - r * half], &c, &s);
    trig[i] = c * magnitude;
    trig[count + i] = s * magnitude;
  }
  __syncthreads();
}

// One workgroup: rows_per_block rows and heads_per_block heads of them.  A group
// of lanes takes a head, a lane one of its units (Loop: several, read twice by the norm).
template <typename T, int V, bool Interleaved, bool Norm, bool Loop>
__global__ __launch_bounds__(kThreads) void rotary_kernel(RotaryArgs a, uint32_t first_row,
                                                          uint32_t rows_per_block,
                                                          uint32_t heads_per_block, uint32_t lanes) {
  extern __shared__ float trig[];
  using P = Pack<T, V>;
  // The squares of fp32 elements and their sum pass fp32 from 2^64 / sqrt(width) on and
  // vanish below 2^-75: they and their sum are taken in 64 bits, and the elements brought
  // near 1 by a power of 2 before they meet its root.
  using Sum = std::conditional_t<std::is_same_v<T, float>, double, float>;
  struct Inverse {  // root x 2^shift
    float root;
    int shift;
  };
  const uint32_t half = a.rotary_width / 2;
  const uint32_t units = half / V + (a.width - a.rotary_width + 2 * V - 1) / (2 * V);
  const uint32_t row0 = first_row + blockIdx.x * rows_per_block, head0 = blockIdx.y * heads_per_block;
  const uint32_t rows = a.rows - row0 < rows_per_block ? a.rows - row0 : rows_per_block;
  const uint32_t heads = a.heads - head0 < heads_per_block ? a.heads - head0 : heads_per_block;
  const uint32_t lane = threadIdx.x & (lanes - 1);
  Walk at(threadIdx.x / lanes, heads, kThreads / lanes);
  const T* in = (const T*)a.input + (uint64_t)row0 * a.input_row_stride + (uint64_t)head0 * a.input_head_stride;
  T* out = (T*)a.out + (uint64_t)row0 * a.output_row_stride + (uint64_t)head0 * a.output_head_stride;
  const Unit own = unit_at<V, Interleaved>(lane, half, a.width);
  const bool on = lane < units;
  const float per_element = 1.0f / (float)a.width;
  P xa, xb, wq[2], wk[2];
  auto load = [&](const T* x, const Unit& u, P* pa, P* pb) __attribute__((always_inline)) {
    *pa = *reinterpret_cast<const P*>(x + u.a);
    if (u.second) *pb = *reinterpret_cast<const P*>(x + u.b);
  };
  auto stream = [&](const T* x, const Unit& u, P* pa, P* pb) __attribute__((always_inline)) {
    *pa = load_once<P>(x + u.a);
    if (u.second) *pb = load_once<P>(x + u.b);
  };
  if (!Loop && on) {
    if (at.row < rows)
      stream(in + (uint64_t)at.row * a.input_row_stride + (uint64_t)at.head * a.input_head_stride, own, &xa, &xb);
    if (Norm) {
      load((const T*)a.query_weight, own, &wq[0], &wq[1]);
      load((const T*)a.key_weight, own, &wk[0], &wk[1]);
    }
  }
  fill_trig(trig, rows, half, a.magnitude, a.frequencies, [&](uint32_t r) { return a.positions[row0 + r]; });
  const float* sines = trig + rows * half;

  // Squares of a unit's elements.
  auto squares = [&](const Unit& u, const P& pa, const P& pb) __attribute__((always_inline)) {
    Sum sum = 0;
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const Sum xa = (Sum)pa.e[e], xb = u.second ? (Sum)pb.e[e] : (Sum)0;
      sum = __builtin_elementwise_fma(xa, xa, sum);
      sum = __builtin_elementwise_fma(xb, xb, sum);
    }
    return sum;
  };
  auto finish = [&](const Unit& u, uint32_t index, const P& pa, const P& pb, const P& va, const P& vb,
                    Inverse inverse, T* y, uint32_t row) __attribute__((always_inline)) {
    float fa[V], fb[V] = {};
    widen(pa, fa);
    if (u.second) widen(pb, fb);
    if (Norm) {
#pragma unroll
      for (int e = 0; e < V; ++e) {
        if constexpr (std::is_same_v<Sum, double>) {
          fa[e] = __builtin_amdgcn_ldexpf(fa[e], inverse.shift);
          fb[e] = __builtin_amdgcn_ldexpf(fb[e], inverse.shift);
        }
        fa[e] = fa[e] * inverse.root * (float)va.e[e];
        if (u.second) fb[e] = fb[e] * inverse.root * (float)vb.e[e];
      }
    }
    if (u.turned) {
      turn<V, Interleaved>(fa, fb, index, half, trig + row * half, sines + row * half);
    }
    store_once(y + u.a, narrow<T, V>(fa));
    if (u.second) store_once(y + u.b, narrow<T, V>(fb));
  };
  auto norm = [&](Sum sum) __attribute__((always_inline)) {
    for (uint32_t o = lanes / 2; o > 0; o >>= 1) sum += __shfl_xor(sum, o, kWave);
    if constexpr (std::is_same_v<Sum, float>) {
      return Inverse{1.0f / sqrtf(sum / (float)a.width + a.epsilon), 0};
    } else {
      const double mean = fma(sum, (double)per_element, (double)a.epsilon);
      const int j = __builtin_amdgcn_frexp_exp(mean) >> 1;
      return Inverse{1.0f / sqrtf((float)__builtin_amdgcn_ldexp(mean, -2 * j)), -j};
    }
  };

  while (at.row < rows) {
    const uint32_t row = at.row, head = at.head;
    const T* x = in + (uint64_t)row * a.input_row_stride + (uint64_t)head * a.input_head_stride;
    T* y = out + (uint64_t)row * a.output_row_stride + (uint64_t)head * a.output_head_stride;
    const bool query = head0 + head < a.query_heads;
    at.next();
    if constexpr (Loop) {
      Inverse inverse{1.0f, 0};
      if (Norm) {
        Sum sum = 0;
        for (uint32_t i = lane; i < units; i += lanes) {
          const Unit u = unit_at<V, Interleaved>(i, half, a.width);
          load(x, u, &xa, &xb);
          sum += squares(u, xa, xb);
        }
        inverse = norm(sum);
      }
      const T* w = (const T*)(query ? a.query_weight : a.key_weight);
      for (uint32_t i = lane; i < units; i += lanes) {
        const Unit u = unit_at<V, Interleaved>(i, half, a.width);
        load(x, u, &xa, &xb);
        if (Norm) load(w, u, &wq[0], &wq[1]);
        finish(u, i, xa, xb, wq[0], wq[1], inverse, y, row);
      }
    } else {
      // The next head's elements, on the way while this one's are turned.
      P na, nb;
      if (on && at.row < rows)
        stream(in + (uint64_t)at.row * a.input_row_stride + (uint64_t)at.head * a.input_head_stride, own, &na, &nb);
      const Inverse inverse = Norm ? norm(on ? squares(own, xa, xb) : (Sum)0) : Inverse{1.0f, 0};
      if (on) finish(own, lane, xa, xb, query ? wq[0] : wk[0], query ? wq[1] : wk[1], inverse, y, row);
      xa = na;
      xb = nb;
    }
  }
}

// Keys and values of rows_per_block new rows into the cache, both as heads of
// one walk: heads [0, key_heads) are keys, turned, the rest values, copied.
template <int V, bool Interleaved, bool Loop>
__global__ __launch_bounds__(kThreads) void append_kernel(AppendArgs a, uint32_t first_row,
                                                          uint32_t rows_per_block,
                                                          uint32_t heads_per_block, uint32_t lanes) {
  extern __shared__ float trig[];
  __shared__ int64_t target[kMaxRows];  // element of the cache, < 0: none
  __shared__ int place[kMaxRows];
  using P = Pack<half_t, V>;
  const uint32_t half = a.rotary_width / 2;
  const uint32_t units = half / V + (a.width - a.rotary_width + 2 * V - 1) / (2 * V);
  const uint32_t row0 = first_row + blockIdx.x * rows_per_block, head0 = blockIdx.y * heads_per_block;
  const uint32_t rows = a.rows - row0 < rows_per_block ? a.rows - row0 : rows_per_block;
  const uint32_t heads = 2 * a.key_heads - head0 < heads_per_block ? 2 * a.key_heads - head0 : heads_per_block;
  const uint32_t lane = threadIdx.x & (lanes - 1);
  Walk at(threadIdx.x / lanes, heads, kThreads / lanes);
  const Unit own = unit_at<V, Interleaved>(lane, half, a.width);
  const bool on = lane < units;
  auto source = [&](uint32_t row, uint32_t head) __attribute__((always_inline)) {
    const uint64_t r = row0 + row;
    return head < a.key_heads ? (const half_t*)a.keys + r * a.key_row_stride + (uint64_t)head * a.width
                              : (const half_t*)a.values + r * a.value_row_stride +
                                    (uint64_t)(head - a.key_heads) * a.width;
  };
  auto load = [&](const half_t* x, const Unit& u, P* pa, P* pb) __attribute__((always_inline)) {
    *pa = load_once<P>(x + u.a);
    if (u.second) *pb = load_once<P>(x + u.b);
  };
  P xa, xb;
  if (!Loop && on && at.row < rows) load(source(at.row, head0 + at.head), own, &xa, &xb);
  // A wave finds each row's place.
  for (uint32_t r = threadIdx.x / kWave; r < rows; r += kThreads / kWave) {
    const RowPlace p = find_row(a.batch, row0 + r);
    const int page = p.position < 0 ? -1 : page_of(a.batch, p.sequence, (uint32_t)p.position);
    if (threadIdx.x % kWave == 0) {
      const uint64_t in_page = (uint32_t)p.position & (a.batch.page_rows - 1);
      target[r] = page < 0 ? -1 : (int64_t)((uint64_t)page * a.batch.page_elements + in_page * a.width);
      place[r] = p.position;
    }
  }
  __syncthreads();
  fill_trig(trig, rows, half, a.magnitude, a.frequencies, [&](uint32_t r) { return place[r]; });
  const float* sines = trig + rows * half;

  auto finish = [&](const Unit& u, uint32_t index, const P& pa, const P& pb, half_t* y, uint32_t row,
                    bool key) __attribute__((always_inline)) {
    if (u.turned && key) {
      float fa[V], fb[V];
      widen(pa, fa);
      widen(pb, fb);
      turn<V, Interleaved>(fa, fb, index, half, trig + row * half, sines + row * half);
      store_once(y + u.a, narrow<half_t, V>(fa));
      store_once(y + u.b, narrow<half_t, V>(fb));
    } else {
      store_once(y + u.a, pa);
      if (u.second) store_once(y + u.b, pb);
    }
  };
  while (at.row < rows) {
    const uint32_t row = at.row, head = head0 + at.head;
    at.next();
    const int64_t to = target[row];
    half_t* y = (half_t*)a.cache + to + (uint64_t)head * a.batch.page_rows * a.width;
    if constexpr (Loop) {
      if (to < 0) continue;
      const half_t* x = source(row, head);
      for (uint32_t i = lane; i < units; i += lanes) {
        const Unit u = unit_at<V, Interleaved>(i, half, a.width);
        load(x, u, &xa, &xb);
        finish(u, i, xa, xb, y, row, head < a.key_heads);
      }
    } else {
      P na, nb;
      if (on && at.row < rows) load(source(at.row, head0 + at.head), own, &na, &nb);
      if (on && to >= 0) finish(own, lane, xa, xb, y, row, head < a.key_heads);
      xa = na;
      xb = nb;
    }
  }
}

// Elements per access, of which 16 bytes are the most: chunks of the rotated
// pairs and of the copied elements must be whole, strides and addresses aligned.
inline uint32_t chunk_elements(uint32_t size, uint32_t width, uint32_t rotary_width, uint64_t strides,
                               uintptr_t addresses) {
  for (uint32_t v = 16 / size; v > 1; v /= 2)
    if ((rotary_width / 2) % v == 0 && (width - rotary_width) % (2 * v) == 0 && strides % v == 0 &&
        addresses % (v * size) == 0)
      return v;
  return 1;
}

// An append's rows at least: a wave finds a row's place (16 heads of 32000 rows, 32 groups:
// 4 rows 37.7 us, 2 rows 38.3, 8 rows 39.7).
constexpr uint32_t kAppendRows = kThreads / kWave;
struct Plan {
  uint32_t rows, heads, lanes, blocks_y, lds;
  bool loop;
};
// Whole rows per workgroup, the fewest (from `least` on) whose heads keep four fifths of
// its lane groups' turns busy, or as many as they can be: an angle is computed once per row
// and workgroup in any case, and small workgroups end together (16384 rows of 40 heads in 32
// groups: 2 rows 58.5 us, 1 row 65.0, 3 rows 62.9, 6 rows 73.1; of 16 heads in 16 groups,
// fp32: 1 row 43.2, 4 rows 46.6, 8 rows 50.7).  Not so many that they make fewer than 1024
// workgroups; where `least` does, one row and as many heads as it has groups for.
inline Plan plan_rows(uint32_t rows, uint32_t heads, uint32_t width, uint32_t rotary_width, uint32_t v,
                      uint32_t least) {
  const uint32_t half = rotary_width / 2;
  const uint32_t units = half / v + (width - rotary_width + 2 * v - 1) / (2 * v);
  Plan p;
  p.lanes = 1;
  while (p.lanes < units && p.lanes < (uint32_t)kWave) p.lanes *= 2;
  p.loop = units > p.lanes;
  const uint32_t slots = kThreads / p.lanes;
  uint32_t most = half > 0 && kMaxRows > 2048 / half ? 2048 / half : kMaxRows;  // 16 KiB of angles
  if (heads > 4 * slots) most = 1;
  if (rows / 1024 >= least && most > rows / 1024) most = rows / 1024;
  // Busy parts of rows x heads on turns of slots, compared crosswise.
  auto turns = [&](uint32_t r) { return (r * heads + slots - 1) / slots; };
  p.rows = least < most ? least : most;
  for (uint32_t r = p.rows; r <= most && heads <= 4 * slots; ++r) {
    if ((uint64_t)r * turns(p.rows) > (uint64_t)p.rows * turns(r)) p.rows = r;
    if (5ull * p.rows * heads >= 4ull * slots * turns(p.rows)) break;
  }
  if (p.rows < 1) p.rows = 1;
  p.heads = heads;
  if ((rows + p.rows - 1) / p.rows < 1024) {
    p.rows = 1;
    p.heads = heads < slots ? heads : slots;
  }
  p.blocks_y = (heads + p.heads - 1) / p.heads;
  if (p.blocks_y > 65535) {  // the grid's second dimension
    p.heads = heads;
    p.blocks_y = 1;
  }
  p.lds = p.rows * half * 2 * (uint32_t)sizeof(float);
  return p;
}

// Calls launch(first row, workgroups) until all rows are covered: a grid holds
// less than 2^24 workgroups of 256 threads.
template <typename F>
int over_rows(uint32_t rows, uint32_t rows_per_block, const F& launch) {
  constexpr uint32_t kMostBlocks = 1u << 23;
  const uint64_t blocks = ((uint64_t)rows + rows_per_block - 1) / rows_per_block;
  for (uint64_t done = 0; done < blocks; done += kMostBlocks) {
    launch((uint32_t)(done * rows_per_block), (uint32_t)(blocks - done < kMostBlocks ? blocks - done : kMostBlocks));
    if (int e = hip_status(hipGetLastError())) return e;
  }
  return 0;
}

template <typename T, int V, bool Interleaved, bool Norm>
int launch_rotary_as(hipStream_t stream, const RotaryArgs& a) {
  const Plan p = plan_rows(a.rows, a.heads, a.width, a.rotary_width, V, 1);
  return over_rows(a.rows, p.rows, [&](uint32_t first, uint32_t blocks) {
    const dim3 grid(blocks, p.blocks_y), block(kThreads);
    if (p.loop)
      hipLaunchKernelGGL((rotary_kernel<T, V, Interleaved, Norm, true>), grid, block, p.lds, stream, a, first, p.rows, p.heads, p.lanes);
    else
      hipLaunchKernelGGL((rotary_kernel<T, V, Interleaved, Norm, false>), grid, block, p.lds, stream, a, first, p.rows, p.heads, p.lanes);
  });
}
template <typename T, int V>
int launch_rotary_v(hipStream_t stream, const RotaryArgs& a) {
  const bool norm = a.query_weight != nullptr;
  if (a.interleaved) return norm ? launch_rotary_as<T, V, true, true>(stream, a) : launch_rotary_as<T, V, true, false>(stream, a);
  return norm ? launch_rotary_as<T, V, false, true>(stream, a) : launch_rotary_as<T, V, false, false>(stream, a);
}

template <int V, bool Interleaved>
int launch_append_as(hipStream_t stream, const AppendArgs& a) {
  const Plan p = plan_rows(a.rows, 2 * a.key_heads, a.width, a.rotary_width, V, kAppendRows);
  return over_rows(a.rows, p.rows, [&](uint32_t first, uint32_t blocks) {
    const dim3 grid(blocks, p.blocks_y), block(kThreads);
    if (p.loop)
      hipLaunchKernelGGL((append_kernel<V, Interleaved, true>), grid, block, p.lds, stream, a, first, p.rows, p.heads, p.lanes);
    else
      hipLaunchKernelGGL((append_kernel<V, Interleaved, false>), grid, block, p.lds, stream, a, first, p.rows, p.heads, p.lanes);
  });
}
template <int V>
int launch_append_v(hipStream_t stream, const AppendArgs& a) {
  return a.interleaved ? launch_append_as<V, true>(stream, a) : launch_append_as<V, false>(stream, a);
}

}  // namespace

int launch_rotary(hipStream_t stream, const RotaryArgs& a) {
  if (a.rows == 0 || a.heads == 0) return 0;
  const uint32_t size = a.f32 ? 4 : 2;
  const uintptr_t addresses = (uintptr_t)a.input | (uintptr_t)a.out | (uintptr_t)a.query_weight | (uintptr_t)a.key_weight;
  if (addresses % size != 0 || ((uintptr_t)a.positions | (uintptr_t)a.frequencies) % 4 != 0)
    return IPUS_ERROR_INVALID_ARGUMENT;
  // In place only where every element is read and written by the same lane.
  if (a.out == a.input &&
      (a.input_row_stride != a.output_row_stride || a.input_head_stride != a.output_head_stride))
    return IPUS_ERROR_INVALID_ARGUMENT;
  const uint64_t strides = (uint64_t)a.input_row_stride | a.output_row_stride | a.input_head_stride | a.output_head_stride;
  const uint32_t v = chunk_elements(size, a.width, a.rotary_width, strides, addresses);
  if (a.f32) {
    if (v == 4) return launch_rotary_v<float, 4>(stream, a);
    if (v == 2) return launch_rotary_v<float, 2>(stream, a);
    return launch_rotary_v<float, 1>(stream, a);
  }
  if (v == 8) return launch_rotary_v<half_t, 8>(stream, a);
  if (v == 4) return launch_rotary_v<half_t, 4>(stream, a);
  if (v == 2) return launch_rotary_v<half_t, 2>(stream, a);
  return launch_rotary_v<half_t, 1>(stream, a);
}

int launch_append_pages(hipStream_t stream, const AppendArgs& a) {
  if (a.rows == 0 || a.batch.sequences == 0) return 0;
  const uintptr_t addresses = (uintptr_t)a.keys | (uintptr_t)a.values | (uintptr_t)a.cache;
  if (addresses % 2 != 0 || (uintptr_t)a.frequencies % 4 != 0 || batch_addresses(a.batch) % 4 != 0)
    return IPUS_ERROR_INVALID_ARGUMENT;
  const uint64_t strides = (uint64_t)a.key_row_stride | a.value_row_stride | a.width;
  const uint32_t v = chunk_elements(2, a.width, a.rotary_width, strides, addresses);
  if (v == 8) return launch_append_v<8>(stream, a);
  if (v == 4) return launch_append_v<4>(stream, a);
  if (v == 2) return launch_append_v<2>(stream, a);
  return launch_append_v<1>(stream, a);
}

}  // namespace ipus
