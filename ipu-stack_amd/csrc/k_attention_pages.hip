// Attention of a ragged batch over a paged cache (pages.h) on gfx950:
//   out = softmax(scale q K^T [+ causal mask]) V
// for every row of every sequence, query head h reading key head
// h / (query_heads / key_heads).  Row i of the n rows of sequence s stands at
// position lengths[s] - n + i; it reads the keys below lengths[s], when causal
// those up to its own position.  Keys without a page carry no weight, and a row
// whose weights are all zero (no key, or only scores of -inf) gives zeros.
#include "../../include/ipus.h"
#include "kernels.h"
#include "pages.h"

namespace ipus {
namespace {

constexpr float kLog2e = 1.4426950408889634f;

inline int hip_status(hipError_t e) { return e == hipSuccess ? 0 : IPUS_ERROR_HIP_BASE - (int)e; }

// Keys that row t may read: [0, count) of a sequence.  sequence >= sequences:
// the row belongs to none.  Called by a whole wave.
struct RowKeys {
  uint32_t sequence, count;
};
__device__ __forceinline__ RowKeys row_keys(const PagedBatch& b, uint32_t t, bool causal) {
  RowKeys k{find_sequence(b, t), 0};
  if (k.sequence >= b.sequences) return k;
  const int64_t start = b.row_offsets[k.sequence], end = b.row_offsets[k.sequence + 1];
  if ((int64_t)t < start) {
    k.sequence = b.sequences;
    return k;
  }
  const int64_t length = b.lengths[k.sequence];
  const int64_t count = causal ? length - (end - (int64_t)t) + 1 : length;
  k.count = count > 0 ? (uint32_t)count : 0;
  return k;
}

// Any width up to 1024, any alignment: a wave per row and query head, one key
// after the other.
constexpr uint32_t kGeneralPerLane = 16;
__global__ __launch_bounds__(kWave) void attention_pages_general_kernel(PagedAttentionArgs a, uint32_t first_row,
                                                                        float scale_log2) {
  const uint32_t row = first_row + blockIdx.x, head = blockIdx.y, lane = threadIdx.x;
  const RowKeys k = row_keys(a.batch, row, a.causal);
  if (k.sequence >= a.batch.sequences) return;
  const half_t* q = (const half_t*)a.query + (uint64_t)row * a.query_row_stride + (uint64_t)head * a.width;
  const uint32_t key_head = head / (a.query_heads / a.key_heads);
  const uint64_t head_elements = (uint64_t)a.batch.page_rows * a.width;
  float acc[kGeneralPerLane];
#pragma unroll
  for (uint32_t i = 0; i < kGeneralPerLane; ++i) acc[i] = 0.0f;
  float m = -INFINITY, l = 0.0f;
  for (uint32_t j = 0; j < k.count; ++j) {
    if (j >> a.batch.page_shift >= a.batch.table_columns) break;
    const int64_t page = page_of(a.batch, k.sequence, j);
    if (page < 0) continue;
    const half_t* key = (const half_t*)a.cache + (uint64_t)page * a.batch.page_elements + key_head * head_elements +
                        (uint64_t)(j & (a.batch.page_rows - 1)) * a.width;
    const half_t* value = key + a.key_heads * head_elements;
    float dot = 0.0f;
    for (uint32_t d = lane; d < a.width; d += kWave) dot = fmaf((float)q[d], (float)key[d], dot);
    dot = wave_sum(dot) * scale_log2;
    const float m_new = fmaxf(m, dot);
    const float m_use = m_new == -INFINITY ? 0.0f : m_new;  // no NaN from (-inf) - (-inf)
    const float alpha = exp2f(m - m_use), p = exp2f(dot - m_use);
    l = l * alpha + p;
#pragma unroll
    for (uint32_t i = 0; i < kGeneralPerLane; ++i) {
      const uint32_t d = lane + kWave * i;
      if (d < a.width) acc[i] = acc[i] * alpha + p * (float)value[d];
    }
    m = m_new;
  }
  const float inverse = l == 0.0f ? 0.0f : 1.0f / l;
  half_t* out = (half_t*)a.out + ((uint64_t)row * a.query_heads + head) * a.width;
#pragma unroll
  for (uint32_t i = 0; i < kGeneralPerLane; ++i) {
    const uint32_t d = lane + kWave * i;
    if (d < a.width) out[d] = (half_t)(acc[i] * inverse);
  }
}

int launch_general(hipStream_t stream, const PagedAttentionArgs& a, float scale_log2) {
  constexpr uint32_t kMostRows = 1u << 24;  // a grid dimension holds less than 2^32 threads
  for (uint64_t done = 0; done < a.rows; done += kMostRows) {
    const uint32_t rows = a.rows - done < kMostRows ? (uint32_t)(a.rows - done) : kMostRows;
    hipLaunchKernelGGL(attention_pages_general_kernel, dim3(rows, a.query_heads), dim3(kWave), 0, stream, a,
                       (uint32_t)done, scale_log2);
    if (int e = hip_status(hipGetLastError())) return e;
  }
  return 0;
}

}  // namespace

int launch_attention_pages(hipStream_t stream, const PagedAttentionArgs& a) {
  if (a.rows == 0 || a.batch.sequences == 0) return 0;
  if (((uintptr_t)a.query | (uintptr_t)a.cache | (uintptr_t)a.out) % 2 != 0 || batch_addresses(a.batch) % 4 != 0)
    return IPUS_ERROR_INVALID_ARGUMENT;
  const float scale_log2 = a.scale * kLog2e;
  return launch_general(stream, a, scale_log2);
}

}  // namespace ipus
