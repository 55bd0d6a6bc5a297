// norm_kernels.hip -- layer norm for training: the forward pass leaves the 8-bit checkpoint of its input where that is wanted,
// the backward pass reads the checkpoint (or the input) and reduces the parameters' gradients in a fixed order.
//
//   forward   mu = mean(x), r = 1 / sqrt(mean((x - mu)^2) + eps), y = (x - mu) r g + b
//   backward  h = (x - mu) r, u = dy g, dx = r (u - mean(u) - h mean(u h)), dg = sum over rows of dy h, db = sum over rows of dy
//
// Memory bounds both.  A row lives in the registers of L lanes from its load to its store, so it is read once and the variance
// is taken around the mean (two passes over registers): no cancellation where |mu| >> 1/r.  All sums are fp32.
#include <hip/hip_runtime.h>
#include "../../include/cswap_hip.h"
#include "common.h"
#include "q8_block.h"

namespace cswap {
namespace q8 {

// Lanes that share a row and chunks of 8 values that each of them holds.  A workgroup has 256 threads, as many as one row needs
// where that is more.
template <int L, int NC> struct Form {
  static constexpr int lanes = L, chunks = NC;
  static constexpr int threads = L > 256 ? L : 256, rows = threads / L, waves = threads / 64;
};

// The sum over the L lanes of a row, in all of them, the same bits in each.  `red` (threads / 64 floats) only where a row has
// more lanes than a wavefront.
template <int L> __device__ inline float row_sum(float v, float* red)
{
  v += __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), 0xb1, 0xf, 0xf, true));   // lane ^ 1
  v += __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), 0x4e, 0xf, 0xf, true));   // lane ^ 2
  v += __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), 0x141, 0xf, 0xf, true));  // 7 - lane
  v += __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), 0x140, 0xf, 0xf, true));  // 15 - lane
  if (L >= 32) v += __shfl_xor(v, 16);
  if (L >= 64) v += __shfl_xor(v, 32);
  if (L > 64) {
    constexpr int W = L / 64;
    __syncthreads();  // red may still be read by the sum before
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.0f;
#pragma unroll
    for (int w = 0; w < W; ++w) v += red[w];
  }
  return v;
}

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

struct NormShape {
  uint32_t rows, cols, code_chunks;  // code_chunks: chunks of a checkpoint's row, padding included
  float inv_cols, eps;
};

__device__ inline int valid_at(uint32_t col, uint32_t cols)
{
  return col + kChunk <= cols ? kChunk : col < cols ? (int)(cols - col) : 0;
}

template <typename T, typename F, bool HOLD>
__global__ __launch_bounds__(F::threads) void norm_forward_kernel(const typename T::value* __restrict__ x, size_t x_stride,
                                                                  NormShape s, Params gamma, Params beta,
                                                                  typename T::value* __restrict__ y, size_t y_stride,
                                                                  float* __restrict__ mean, float* __restrict__ rstd,
                                                                  uint2* __restrict__ codes, uint8_t* __restrict__ scales)
{
  __shared__ float red[F::waves];
  const uint32_t lane = threadIdx.x % F::lanes;
  float g[F::chunks][8], b[F::chunks][8];
  int valid[F::chunks];
#pragma unroll
  for (int c = 0; c < F::chunks; ++c) {
    const uint32_t col = (lane + c * F::lanes) * kChunk;
    valid[c] = valid_at(col, s.cols);
    load_params(gamma, col, valid[c], 1.0f, g[c]);
    load_params(beta, col, valid[c], 0.0f, b[c]);
  }
  // the rows of a workgroup walk together: every lane runs every exchange and barrier
  for (uint32_t base = blockIdx.x * F::rows; base < s.rows; base += gridDim.x * F::rows) {
    const uint32_t row = base + threadIdx.x / F::lanes;
    const bool here = row < s.rows;
    float v[F::chunks][8], sum = 0.0f;
#pragma unroll
    for (int c = 0; c < F::chunks; ++c) {
      const uint32_t col = (lane + c * F::lanes) * kChunk;
      load_chunk<T>(x + (size_t)row * x_stride + col, here ? valid[c] : 0, v[c]);
#pragma unroll
      for (int i = 0; i < kChunk; ++i) sum += v[c][i];
    }
    if (HOLD) {
#pragma unroll
      for (int c = 0; c < F::chunks; ++c) {
        const uint32_t chunk = lane + c * F::lanes;
        uint32_t scale;
        const uint2 q = encode_chunk(v[c], quad_max_bits(v[c]), &scale);
        if (here && chunk < s.code_chunks) {
          const size_t at = (size_t)row * s.code_chunks + chunk;
          codes[at] = q;
          if ((chunk & (kChunksPerGroup - 1)) == 0) scales[at / kChunksPerGroup] = (uint8_t)scale;
        }
      }
    }
    const float mu = row_sum<F::lanes>(sum, red) * s.inv_cols;
    float squares = 0.0f;
#pragma unroll
    for (int c = 0; c < F::chunks; ++c)
#pragma unroll
      for (int i = 0; i < kChunk; ++i) {
        v[c][i] -= mu;
        if (i < valid[c]) squares = __builtin_fmaf(v[c][i], v[c][i], squares);
      }
    const float r = 1.0f / __builtin_sqrtf(row_sum<F::lanes>(squares, red) * s.inv_cols + s.eps);
#pragma unroll
    for (int c = 0; c < F::chunks; ++c) {
#pragma unroll
      for (int i = 0; i < kChunk; ++i) v[c][i] = __builtin_fmaf(v[c][i] * r, g[c][i], b[c][i]);
      if (here) store_chunk<T>(y + (size_t)row * y_stride + (lane + c * F::lanes) * kChunk, valid[c], v[c]);
    }
    if (here && lane == 0) mean[row] = mu, rstd[row] = r;
  }
}

// One workgroup's share of the parameters' gradients: part[workgroup][0 = gamma, 1 = beta][cols].
template <typename T, typename F, bool HELD>
__global__ __launch_bounds__(F::threads) void norm_backward_kernel(const typename T::value* __restrict__ dy, size_t dy_stride,
                                                                   const typename T::value* __restrict__ x, size_t x_stride,
                                                                   const uint2* __restrict__ codes,
                                                                   const uint8_t* __restrict__ scales, NormShape s,
                                                                   const float* __restrict__ mean, const float* __restrict__ rstd,
                                                                   Params gamma, typename T::value* __restrict__ dx,
                                                                   size_t dx_stride, float* __restrict__ part)
{
  __shared__ float red[F::waves];
  const uint32_t lane = threadIdx.x % F::lanes;
  float g[F::chunks][8], dg[F::chunks][8], db[F::chunks][8];
  int valid[F::chunks];
#pragma unroll
  for (int c = 0; c < F::chunks; ++c) {
    const uint32_t col = (lane + c * F::lanes) * kChunk;
    valid[c] = valid_at(col, s.cols);
    load_params(gamma, col, valid[c], 1.0f, g[c]);
#pragma unroll
    for (int i = 0; i < kChunk; ++i) dg[c][i] = db[c][i] = 0.0f;
  }
  for (uint32_t base = blockIdx.x * F::rows; base < s.rows; base += gridDim.x * F::rows) {
    const uint32_t row = base + threadIdx.x / F::lanes;
    const bool here = row < s.rows;
    const float mu = here ? mean[row] : 0.0f, r = here ? rstd[row] : 0.0f;
    float h[F::chunks][8], u[F::chunks][8], s1 = 0.0f, s2 = 0.0f;
#pragma unroll
    for (int c = 0; c < F::chunks; ++c) {
      const uint32_t chunk = lane + c * F::lanes, col = chunk * kChunk;
      const int n = here ? valid[c] : 0;
      load_chunk<T>(dy + (size_t)row * dy_stride + col, n, u[c]);
      if (HELD) {
        const size_t at = (size_t)row * s.code_chunks + chunk;
        uint2 q = {0u, 0u};
        uint32_t scale = 1;
        if (n) q = codes[at], scale = scales[at / kChunksPerGroup];
        decode_chunk(q, unit_of(scale), h[c]);
      } else {
        load_chunk<T>(x + (size_t)row * x_stride + col, n, h[c]);
      }
    }
#pragma unroll
    for (int c = 0; c < F::chunks; ++c) {
      const int n = here ? valid[c] : 0;
#pragma unroll
      for (int i = 0; i < kChunk; ++i) {
        h[c][i] = (h[c][i] - mu) * r;
        if (i >= n) h[c][i] = 0.0f;  // a group of NaN reaches behind the row's end
        dg[c][i] = __builtin_fmaf(u[c][i], h[c][i], dg[c][i]);
        db[c][i] += u[c][i];
        u[c][i] *= g[c][i];
        s1 += u[c][i];
        s2 = __builtin_fmaf(u[c][i], h[c][i], s2);
      }
    }
    s1 = row_sum<F::lanes>(s1, red) * s.inv_cols;
    s2 = row_sum<F::lanes>(s2, red) * s.inv_cols;
#pragma unroll
    for (int c = 0; c < F::chunks; ++c) {
#pragma unroll
      for (int i = 0; i < kChunk; ++i) u[c][i] = r * (u[c][i] - __builtin_fmaf(h[c][i], s2, s1));
      if (here) store_chunk<T>(dx + (size_t)row * dx_stride + (lane + c * F::lanes) * kChunk, valid[c], u[c]);
    }
  }
  if (!part) return;
  float* mine = part + (size_t)blockIdx.x * 2 * s.cols;
  // the rows of a workgroup one after the other, in a fixed order
  constexpr int kPass = F::rows > 1 ? F::lanes * F::chunks * kChunk : 1;
  __shared__ float sum[2][kPass];
  if (F::rows > 1) {
    for (int turn = 0; turn < F::rows; ++turn) {
      if ((int)(threadIdx.x / F::lanes) == turn) {
#pragma unroll
        for (int c = 0; c < F::chunks; ++c)
#pragma unroll
          for (int i = 0; i < kChunk; ++i) {
            const uint32_t at = ((lane + c * F::lanes) * kChunk + i) % kPass;
            if (turn) dg[c][i] += sum[0][at], db[c][i] += sum[1][at];
            sum[0][at] = dg[c][i], sum[1][at] = db[c][i];
          }
      }
      __syncthreads();
    }
    for (uint32_t i = threadIdx.x; i < s.cols; i += F::threads) mine[i] = sum[0][i % kPass], mine[s.cols + i] = sum[1][i % kPass];
  } else {
#pragma unroll
    for (int c = 0; c < F::chunks; ++c) {
      const uint32_t col = (lane + c * F::lanes) * kChunk;
      store_chunk<F32>(mine + col, valid[c], dg[c]);
      store_chunk<F32>(mine + s.cols + col, valid[c], db[c]);
    }
  }
}

// out[i] = sum over `parts` rows of part[.][i], n values a row; 32 columns a workgroup, eight lanes to a column
template <typename P>
__global__ __launch_bounds__(256) void norm_reduce_kernel(const float* __restrict__ part, uint32_t parts, uint32_t cols,
                                                          typename P::value* __restrict__ dgamma,
                                                          typename P::value* __restrict__ dbeta)
{
  __shared__ float sum[8][32];
  const uint32_t i = blockIdx.x * 32 + (threadIdx.x & 31), seg = threadIdx.x >> 5, n = 2 * cols;
  float v = 0.0f;
  if (i < n)
    for (uint32_t p = seg; p < parts; p += 8) v += part[(size_t)p * n + i];
  sum[seg][threadIdx.x & 31] = v;
  __syncthreads();
  if (seg == 0 && i < n) {
#pragma unroll
    for (int k = 1; k < 8; ++k) v += sum[k][threadIdx.x];
    typename P::value* out = i < cols ? dgamma : dbeta;
    if (out) out[i < cols ? i : i - cols] = from_float<P>(v);
  }
}

// ---------------------------------------------------------------- launches
// Rows up to 16384 values: 16 lanes hold 128 values of a row, 1024 lanes with two chunks each the longest.
constexpr size_t kMaxNormCols = 16384;
constexpr unsigned kMostForward = 2048, kMostBackward = 512;  // workgroups

template <typename F> static unsigned groups_for(size_t rows, unsigned most)
{
  const size_t want = (rows + F::rows - 1) / F::rows;
  return (unsigned)(want < most ? want : most);
}

template <typename Fn> static auto with_form(size_t cols, Fn&& fn)
{
  if (cols <= 128) return fn(Form<16, 1>());
  if (cols <= 256) return fn(Form<32, 1>());
  if (cols <= 512) return fn(Form<64, 1>());
  if (cols <= 1024) return fn(Form<64, 2>());
  if (cols <= 2048) return fn(Form<256, 1>());
  if (cols <= 4096) return fn(Form<256, 2>());
  if (cols <= 8192) return fn(Form<1024, 1>());
  return fn(Form<1024, 2>());
}

static unsigned backward_groups(size_t rows, size_t cols)
{
  return with_form(cols, [&](auto f) { return groups_for<decltype(f)>(rows, kMostBackward); });
}

template <typename Fn> static int with_type(int dtype, Fn&& fn)
{
  switch (dtype) {
    case CSWAP_DT_F32: return fn(F32());
    case CSWAP_DT_BF16: return fn(BF16());
    default: return fn(F16());
  }
}

static int norm_shape(size_t rows, size_t cols, float eps, NormShape* s)
{
  if (cols > kMaxNormCols || rows >= ((size_t)1 << 31)) return CSWAP_E_UNSUPPORTED;
  *s = {(uint32_t)rows, (uint32_t)cols, (uint32_t)(pitch_of(cols) / kChunk), (float)(1.0 / (double)cols), eps};
  return CSWAP_OK;
}

}  // namespace q8
}  // namespace cswap

using namespace cswap;
using namespace cswap::q8;

extern "C" size_t cswap_layer_norm_workspace_bytes(size_t rows, size_t cols)
{
  if (cols == 0 || cols > kMaxNormCols || rows == 0) return 0;
  return (size_t)backward_groups(rows, cols) * 2 * cols * sizeof(float);
}

extern "C" int cswap_layer_norm_forward(const void* d_x, int dtype, size_t rows, size_t cols, ptrdiff_t x_stride,
                                        const void* d_gamma, const void* d_beta, int param_dtype, float eps, void* d_y,
                                        ptrdiff_t y_stride, float* d_mean, float* d_rstd, int8_t* d_codes, uint8_t* d_scales,
                                        cswap_stream_t stream)
{
  NormShape s;
  if (int e = check_rows(rows, cols, &x_stride)) return e;
  if (int e = check_rows(rows, cols, &y_stride)) return e;
  if (!dtype_known(dtype) || !dtype_known(param_dtype) || !(eps >= 0.0f)) return CSWAP_E_ARG;
  if (int e = norm_shape(rows, cols, eps, &s)) return e;
  if (rows == 0) return CSWAP_OK;
  if (!value_ptr(d_x, dtype) || !value_ptr(d_y, dtype) || !value_ptr(d_mean, CSWAP_DT_F32) || !value_ptr(d_rstd, CSWAP_DT_F32))
    return CSWAP_E_ARG;
  if ((d_gamma && !value_ptr(d_gamma, param_dtype)) || (d_beta && !value_ptr(d_beta, param_dtype))) return CSWAP_E_ARG;
  if ((d_codes || d_scales) && !checkpoint_ptrs(d_codes, d_scales)) return CSWAP_E_ARG;
  const Params g = {d_gamma, param_dtype}, b = {d_beta, param_dtype};
  hipStream_t st = static_cast<hipStream_t>(stream);
  return with_type(dtype, [&](auto t) {
    typedef decltype(t) T;
    return with_form(cols, [&](auto f) {
      typedef decltype(f) F;
      auto k = d_codes ? norm_forward_kernel<T, F, true> : norm_forward_kernel<T, F, false>;
      hipLaunchKernelGGL(k, dim3(groups_for<F>(rows, kMostForward)), dim3(F::threads), 0, st,
                         static_cast<const typename T::value*>(d_x), (size_t)x_stride, s, g, b,
                         static_cast<typename T::value*>(d_y), (size_t)y_stride, d_mean, d_rstd,
                         reinterpret_cast<uint2*>(d_codes), d_scales);
      return check_launch();
    });
  });
}

extern "C" int cswap_layer_norm_backward(const void* d_dy, int dtype, size_t rows, size_t cols, ptrdiff_t dy_stride,
                                         const void* d_x, ptrdiff_t x_stride, const int8_t* d_codes, const uint8_t* d_scales,
                                         const float* d_mean, const float* d_rstd, const void* d_gamma, int param_dtype,
                                         void* d_dx, ptrdiff_t dx_stride, void* d_dgamma, void* d_dbeta, void* d_ws,
                                         size_t ws_bytes, cswap_stream_t stream)
{
  NormShape s;
  if (int e = check_rows(rows, cols, &dy_stride)) return e;
  if (int e = check_rows(rows, cols, &x_stride)) return e;
  if (int e = check_rows(rows, cols, &dx_stride)) return e;
  if (!dtype_known(dtype) || !dtype_known(param_dtype)) return CSWAP_E_ARG;
  if (int e = norm_shape(rows, cols, 0.0f, &s)) return e;
  if ((d_gamma && !value_ptr(d_gamma, param_dtype)) || (d_dgamma && !value_ptr(d_dgamma, param_dtype)) ||
      (d_dbeta && !value_ptr(d_dbeta, param_dtype)))
    return CSWAP_E_ARG;
  const bool reduce = d_dgamma || d_dbeta;
  if (rows) {
    const bool held = d_codes || d_scales;
    if (!value_ptr(d_dy, dtype) || !value_ptr(d_dx, dtype) || !value_ptr(d_mean, CSWAP_DT_F32) ||
        !value_ptr(d_rstd, CSWAP_DT_F32))
      return CSWAP_E_ARG;
    if (held ? (d_x || !checkpoint_ptrs(d_codes, d_scales)) : !value_ptr(d_x, dtype)) return CSWAP_E_ARG;
    if (reduce && !value_ptr(d_ws, CSWAP_DT_F32)) return CSWAP_E_ARG;
    if (reduce && ws_bytes < cswap_layer_norm_workspace_bytes(rows, cols)) return CSWAP_E_NOMEM;
  }
  hipStream_t st = static_cast<hipStream_t>(stream);
  const Params g = {d_gamma, param_dtype};
  const unsigned grid = rows ? backward_groups(rows, cols) : 0;
  if (rows) {
    const int e = with_type(dtype, [&](auto t) {
      typedef decltype(t) T;
      return with_form(cols, [&](auto f) {
        typedef decltype(f) F;
        auto k = d_codes ? norm_backward_kernel<T, F, true> : norm_backward_kernel<T, F, false>;
        hipLaunchKernelGGL(k, dim3(grid), dim3(F::threads), 0, st, static_cast<const typename T::value*>(d_dy), (size_t)dy_stride,
                           static_cast<const typename T::value*>(d_x), (size_t)x_stride, reinterpret_cast<const uint2*>(d_codes),
                           d_scales, s, d_mean, d_rstd, g, static_cast<typename T::value*>(d_dx), (size_t)dx_stride,
                           reduce ? static_cast<float*>(d_ws) : nullptr);
        return check_launch();
      });
    });
    if (e) return e;
  }
  if (!reduce) return CSWAP_OK;
  return with_type(param_dtype, [&](auto t) {
    typedef decltype(t) P;
    hipLaunchKernelGGL(norm_reduce_kernel<P>, dim3((unsigned)((2 * cols + 31) / 32)), dim3(256), 0, st,
                       static_cast<const float*>(d_ws), grid, (uint32_t)cols, static_cast<typename P::value*>(d_dgamma),
                       static_cast<typename P::value*>(d_dbeta));
    return check_launch();
  });
}
