// q8_params.h -- parameters of norms, their gradients, and rows as they lie in memory: what the kernels of norms share.
#pragma once
#include "q8_block.h"

namespace cswap {
namespace q8 {

struct Params {
  const void* p;  // NULL: none
  int dtype;
};

// eight parameters from `at` on, as fp32; `none` where there are no such parameters
__device__ inline void load_params(const Params& q, uint32_t at, int valid, float none, float v[8])
{
  if (!q.p) {
#pragma unroll
    for (int i = 0; i < kChunk; ++i) v[i] = none;
  } else if (q.dtype == CSWAP_DT_F32) {
    load_chunk<F32>(static_cast<const float*>(q.p) + at, valid, v);
  } else if (q.dtype == CSWAP_DT_BF16) {
    load_chunk<BF16>(static_cast<const uint16_t*>(q.p) + at, valid, v);
  } else {
    load_chunk<F16>(static_cast<const uint16_t*>(q.p) + at, valid, v);
  }
}

struct GradParams {
  void *dgamma, *dbeta;  // NULL: not wanted
  int dtype;
  __device__ inline void store(bool gamma, uint32_t at, float v) const
  {
    void* to = gamma ? dgamma : dbeta;
    if (!to) return;
    if (dtype == CSWAP_DT_F32) static_cast<float*>(to)[at] = v;
    else if (dtype == CSWAP_DT_BF16) static_cast<uint16_t*>(to)[at] = from_float<BF16>(v);
    else static_cast<uint16_t*>(to)[at] = from_float<F16>(v);
  }
};

__device__ inline int valid_at(uint32_t col, uint32_t cols)
{
  return col + kChunk <= cols ? kChunk : col < cols ? (int)(cols - col) : 0;
}

template <typename T> __device__ inline void widen(const u4_any raw[T::bytes / 2], float v[8])
{
#pragma unroll
  for (int e = 0; e < kChunk; ++e) {
    if constexpr (T::bytes == 4) v[e] = __uint_as_float(raw[e / 4][e % 4]);
    else v[e] = to_float<T>((typename T::value)(raw[0][e / 2] >> (16 * (e & 1))));
  }
}

// The gradients from `parts` shares part[share][0 = gamma, 1 = beta][cols], in a fixed order: 32 columns a workgroup of 32 * SEGS threads,
// SEGS lanes to a column.  `sum`: SEGS * 33 values of LDS.
template <int SEGS>
__device__ inline void sum_shares(const float* __restrict__ part, uint32_t parts, uint32_t cols, uint32_t group, const GradParams& grads, float* sum)
{
  const uint32_t lane = threadIdx.x & 31, seg = threadIdx.x >> 5, n = 2 * cols, i = group * 32 + lane;
  float v = 0.0f;
  if (i < n) {
#pragma unroll 8
    for (uint32_t p = seg; p < parts; p += SEGS) v += part[(size_t)p * n + i];
  }
  sum[seg * 33 + lane] = v;
  __syncthreads();
  if (seg == 0 && i < n) {
#pragma unroll
    for (int k = 1; k < SEGS; ++k) v += sum[k * 33 + lane];
    grads.store(i < cols, i < cols ? i : i - cols, v);
  }
}

template <typename Fn> static int with_type(int dtype, Fn&& fn)
{
  switch (dtype) {
    case CSWAP_DT_F32: return fn(F32());
    case CSWAP_DT_BF16: return fn(BF16());
    default: return fn(F16());
  }
}

}  // namespace q8
}  // namespace cswap
