// norm_kernels.hip -- layer norm for training: the forward pass leaves the 8-bit checkpoint of its input where that is wanted,
// the backward pass reads the checkpoint (or the input) and reduces the parameters' gradients in a fixed order.
//
//   forward   mu = mean(x), r = 1 / sqrt(mean((x - mu)^2) + eps), y = (x - mu) r g + b
//   backward  h = (x - mu) r, u = dy g, dx = r (u - mean(u) - h mean(u h)), dg = sum over rows of dy h, db = sum over rows of dy
//
// Memory bounds both.  A row lives in the registers of L lanes from its load to its store, so it is read once and the variance
// is taken around the mean (two passes over registers): no cancellation where |mu| >> 1/r.  All sums are fp32.  A row of up to
// 1024 values is one wavefront's or less, so nothing waits for a barrier; longer ones share a sum through LDS with one barrier
// each.  Either kernel asks for a workgroup's next row before it works on this one.
//
// Calls one behind the other, tensors in turn: 16384 x 768 bf16 forward 13.0 us (4.9 TB/s), backward with its sums 17.0 from the
// checkpoint and 18.0 from the input (3.7 and 4.2 TB/s; the backward 44 in the first form: a row at a time, 512 shares, 8 lanes to
// sum a column), fp32 19.1, 23.4 and 30.5; 2048 x 8192 fp32 28.5, 35.3 and 42.1; 4096 x 16384 bf16 64, 81 and 87.  Traced launch by
// launch 16384 x 768 bf16 takes 15.0-16.3, 15.0-16.0 and 3.0-4.0 for the sums, 2048 x 8192 fp32 30-31, 31-33 and 4.2-4.8.  Shares
// by wavefronts of 1024 threads in rows of 513 to 1024 values spill (16384 x 768 fp32 backward 38 : 24 us with 512 threads).
#include <hip/hip_runtime.h>
#include "../../include/cswap_hip.h"
#include "common.h"
#include "q8_block.h"

namespace cswap {
namespace q8 {

// L lanes share a row, each holds NC chunks of 8 values; a workgroup has NT threads.
template <int L, int NC, int NT> struct Form {
  static constexpr int lanes = L, chunks = NC, threads = NT, rows = NT / L, waves = NT / 64;
};

#define CSWAP_DPP(v, ctrl) __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), ctrl, 0xf, 0xf, true))

// The sums of two values over the L lanes of a row, in all of them, the same bits in each.  `red` (two buffers of `waves` pairs,
// taken in turn: a buffer is written again only behind the next sum's barrier) only where a row has more lanes than a wavefront.
template <int L, int WAVES> struct RowSum {
  float2 (*red)[WAVES];
  int turn = 0;
  __device__ inline float2 operator()(float x, float y)
  {
    x += CSWAP_DPP(x, 0xb1), y += CSWAP_DPP(y, 0xb1);    // lane ^ 1
    x += CSWAP_DPP(x, 0x4e), y += CSWAP_DPP(y, 0x4e);    // lane ^ 2
    x += CSWAP_DPP(x, 0x141), y += CSWAP_DPP(y, 0x141);  // 7 - lane
    x += CSWAP_DPP(x, 0x140), y += CSWAP_DPP(y, 0x140);  // 15 - lane
    if (L >= 32) x = join<16>(x), y = join<16>(y);
    if (L >= 64) x = join<32>(x), y = join<32>(y);
    if (L > 64) {
      constexpr int W = L / 64;
      const int wave = threadIdx.x >> 6;
      if ((threadIdx.x & 63) == 0) red[turn][wave] = make_float2(x, y);
      __syncthreads();
      x = y = 0.0f;
#pragma unroll
      for (int w = 0; w < W; ++w) {
        const float2 v = red[turn][wave / W * W + w];
        x += v.x, y += v.y;
      }
      turn ^= 1;
    }
    return make_float2(x, y);
  }
  // v + v of lane ^ N: the swap of halves gives either half to both
  template <int N> static __device__ inline float join(float v)
  {
    const unsigned u = __float_as_uint(v);
    const auto p = N == 16 ? __builtin_amdgcn_permlane16_swap(u, u, false, false) : __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return __uint_as_float(p[0]) + __uint_as_float(p[1]);
  }
};

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

struct NormShape {
  uint32_t rows, cols, code_chunks;  // code_chunks: chunks of a checkpoint's row, padding included
  float inv_cols, eps;
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

template <typename T, typename F, bool HOLD>
__global__ __launch_bounds__(F::threads) void norm_forward_kernel(const typename T::value* __restrict__ x, size_t x_stride,
                                                                  NormShape s, Params gamma, Params beta,
                                                                  typename T::value* __restrict__ y, size_t y_stride,
                                                                  float* __restrict__ mean, float* __restrict__ rstd,
                                                                  uint2* __restrict__ codes, uint8_t* __restrict__ scales)
{
  __shared__ float2 red[2][F::waves];
  RowSum<F::lanes, F::waves> row_sum = {red};
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
  u4_any next[F::chunks][T::bytes / 2];
  auto load = [&](uint32_t row) {
#pragma unroll
    for (int c = 0; c < F::chunks; ++c)
      load_raw<T>(x + (size_t)row * x_stride + (lane + c * F::lanes) * kChunk, row < s.rows ? valid[c] : 0, next[c]);
  };
  // the rows of a workgroup walk together: every lane runs every exchange and barrier
  const uint32_t mine = threadIdx.x / F::lanes;
  load(blockIdx.x * F::rows + mine);
  for (uint32_t base = blockIdx.x * F::rows; base < s.rows; base += gridDim.x * F::rows) {
    const uint32_t row = base + mine;
    const bool here = row < s.rows;
    float v[F::chunks][8], sum = 0.0f;
#pragma unroll
    for (int c = 0; c < F::chunks; ++c) {
      widen<T>(next[c], v[c]);
#pragma unroll
      for (int i = 0; i < kChunk; ++i) sum += v[c][i];
    }
    if (base + gridDim.x * F::rows < s.rows) load(row + gridDim.x * F::rows);
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
    const float mu = row_sum(sum, 0.0f).x * s.inv_cols;
    float squares = 0.0f;
#pragma unroll
    for (int c = 0; c < F::chunks; ++c)
#pragma unroll
      for (int i = 0; i < kChunk; ++i) {
        v[c][i] -= mu;
        const float d = i < valid[c] ? v[c][i] : 0.0f;
        squares = __builtin_fmaf(d, d, squares);
      }
    const float r = 1.0f / __builtin_sqrtf(row_sum(squares, 0.0f).x * s.inv_cols + s.eps);
#pragma unroll
    for (int c = 0; c < F::chunks; ++c) {
#pragma unroll
      for (int i = 0; i < kChunk; ++i) v[c][i] = __builtin_fmaf(v[c][i] * r, g[c][i], b[c][i]);
      if (here) store_chunk<T>(y + (size_t)row * y_stride + (lane + c * F::lanes) * kChunk, valid[c], v[c]);
    }
    if (here && lane == 0) mean[row] = mu, rstd[row] = r;
  }
}

// What a lane holds of the next row while it works on this one: values as they lie in memory.
template <typename T, bool HELD> struct RowChunk {
  u4_any dy[T::bytes / 2], x[HELD ? 1 : T::bytes / 2];
  uint2 q;
  uint32_t scale;
};

// Either the workgroup's share of the parameters' gradients, part[workgroup][0 = gamma, 1 = beta][cols], or, of a single
// workgroup (part NULL), the gradients.
template <typename T, typename F, bool HELD>
__global__ __launch_bounds__(F::threads) void norm_backward_kernel(const typename T::value* __restrict__ dy, size_t dy_stride,
                                                                   const typename T::value* __restrict__ x, size_t x_stride,
                                                                   const uint2* __restrict__ codes,
                                                                   const uint8_t* __restrict__ scales, NormShape s,
                                                                   const float* __restrict__ mean, const float* __restrict__ rstd,
                                                                   Params gamma, typename T::value* __restrict__ dx,
                                                                   size_t dx_stride, float* __restrict__ part, GradParams grads)
{
  __shared__ float2 red[2][F::waves];
  RowSum<F::lanes, F::waves> row_sum = {red};
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
  constexpr bool kAhead = F::chunks == 1 || F::lanes <= 64;  // registers for two rows
  RowChunk<T, HELD> next[F::chunks];
  float next_mu, next_r;
  auto load = [&](uint32_t row) {
    const bool here = row < s.rows;
    next_mu = here ? mean[row] : 0.0f, next_r = here ? rstd[row] : 0.0f;
#pragma unroll
    for (int c = 0; c < F::chunks; ++c) {
      const uint32_t chunk = lane + c * F::lanes, col = chunk * kChunk;
      const int n = here ? valid[c] : 0;
      load_raw<T>(dy + (size_t)row * dy_stride + col, n, next[c].dy);
      if (HELD) {
        const size_t at = (size_t)row * s.code_chunks + chunk;
        next[c].q = {0u, 0u}, next[c].scale = 1;
        if (n) next[c].q = codes[at], next[c].scale = scales[at / kChunksPerGroup];
      } else {
        load_raw<T>(x + (size_t)row * x_stride + col, n, next[c].x);
      }
    }
  };
  // the rows of a workgroup walk together: every lane runs every exchange and barrier
  const uint32_t mine = threadIdx.x / F::lanes;
  if (kAhead && blockIdx.x * F::rows < s.rows) load(blockIdx.x * F::rows + mine);
  for (uint32_t base = blockIdx.x * F::rows; base < s.rows; base += gridDim.x * F::rows) {
    const uint32_t row = base + mine;
    if (!kAhead) load(row);
    const float mu = next_mu, r = next_r;
    float h[F::chunks][8], u[F::chunks][8], s1 = 0.0f, s2 = 0.0f;
#pragma unroll
    for (int c = 0; c < F::chunks; ++c) {
      widen<T>(next[c].dy, u[c]);
      if constexpr (HELD) decode_chunk(next[c].q, unit_of(next[c].scale), h[c]);
      else widen<T>(next[c].x, h[c]);
    }
    if (kAhead && base + gridDim.x * F::rows < s.rows) load(row + gridDim.x * F::rows);
#pragma unroll
    for (int c = 0; c < F::chunks; ++c) {
#pragma unroll
      for (int i = 0; i < kChunk; ++i) h[c][i] = (h[c][i] - mu) * r;
      if (HELD && valid[c] < kChunk) {  // a group of NaN reaches behind the row's end
#pragma unroll
        for (int i = 0; i < kChunk; ++i) h[c][i] = i < valid[c] ? h[c][i] : 0.0f;
      }
#pragma unroll
      for (int i = 0; i < kChunk; ++i) {
        dg[c][i] = __builtin_fmaf(u[c][i], h[c][i], dg[c][i]);
        db[c][i] += u[c][i];
        u[c][i] *= g[c][i];
        s1 += u[c][i];
        s2 = __builtin_fmaf(u[c][i], h[c][i], s2);
      }
    }
    const float2 sums = row_sum(s1, s2);
    s1 = sums.x * s.inv_cols, s2 = sums.y * s.inv_cols;
#pragma unroll
    for (int c = 0; c < F::chunks; ++c) {
#pragma unroll
      for (int i = 0; i < kChunk; ++i) u[c][i] = r * (u[c][i] - __builtin_fmaf(h[c][i], s2, s1));
      if (row < s.rows) store_chunk<T>(dx + (size_t)row * dx_stride + (lane + c * F::lanes) * kChunk, valid[c], u[c]);
    }
  }
  if (!part && !grads.dgamma && !grads.dbeta) return;
  float* const share = part ? part + (size_t)blockIdx.x * 2 * s.cols : nullptr;
  if constexpr (F::rows > 1) {
    // the lanes that have the same columns, in a fixed order: those of a wavefront by exchanges, then the sets through LDS
    constexpr int kCols = F::lanes * F::chunks * kChunk, kWide = F::lanes < 64 ? 64 : F::lanes, kSets = F::threads / kWide;
    __shared__ __attribute__((aligned(16))) float sum[kSets * 2 * kCols];
#pragma unroll
    for (int c = 0; c < F::chunks; ++c)
#pragma unroll
      for (int i = 0; i < kChunk; ++i) {
        if (F::lanes <= 16) dg[c][i] = row_sum.template join<16>(dg[c][i]), db[c][i] = row_sum.template join<16>(db[c][i]);
        if (F::lanes <= 32) dg[c][i] = row_sum.template join<32>(dg[c][i]), db[c][i] = row_sum.template join<32>(db[c][i]);
      }
    if (threadIdx.x % kWide < F::lanes) {
      float* to = sum + (size_t)(threadIdx.x / kWide) * 2 * kCols;
#pragma unroll
      for (int c = 0; c < F::chunks; ++c)
#pragma unroll
        for (int i = 0; i < kChunk; i += 4) {
          const int at = (lane + c * F::lanes) * kChunk + i;
          *reinterpret_cast<float4*>(to + at) = make_float4(dg[c][i], dg[c][i + 1], dg[c][i + 2], dg[c][i + 3]);
          *reinterpret_cast<float4*>(to + kCols + at) = make_float4(db[c][i], db[c][i + 1], db[c][i + 2], db[c][i + 3]);
        }
    }
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < 2 * s.cols; i += F::threads) {
      const uint32_t col = i < s.cols ? i : i - s.cols;
      const float* from = sum + (i < s.cols ? 0 : kCols) + col;
      float v = 0.0f;
#pragma unroll
      for (int k = 0; k < kSets; ++k) v += from[k * 2 * kCols];
      if (share) share[i] = v;
      else grads.store(i < s.cols, col, v);
    }
  } else {
#pragma unroll
    for (int c = 0; c < F::chunks; ++c) {
      const uint32_t col = (lane + c * F::lanes) * kChunk;
      if (share) {
        store_chunk<F32>(share + col, valid[c], dg[c]);
        store_chunk<F32>(share + s.cols + col, valid[c], db[c]);
      } else {
#pragma unroll
        for (int i = 0; i < kChunk; ++i)
          if (i < valid[c]) grads.store(true, col + i, dg[c][i]), grads.store(false, col + i, db[c][i]);
      }
    }
  }
}

// The gradients from `parts` shares: 32 columns a workgroup, 32 lanes to a column
__global__ __launch_bounds__(1024) void norm_reduce_kernel(const float* __restrict__ part, uint32_t parts, uint32_t cols,
                                                           GradParams grads)
{
  __shared__ float sum[32][33];
  const uint32_t lane = threadIdx.x & 31, seg = threadIdx.x >> 5, n = 2 * cols, i = blockIdx.x * 32 + lane;
  float v = 0.0f;
  if (i < n) {
#pragma unroll 8
    for (uint32_t p = seg; p < parts; p += 32) v += part[(size_t)p * n + i];
  }
  sum[seg][lane] = v;
  __syncthreads();
  if (seg == 0 && i < n) {
#pragma unroll
    for (int k = 1; k < 32; ++k) v += sum[k][lane];
    grads.store(i < cols, i < cols ? i : i - cols, v);
  }
}

// ---------------------------------------------------------------- launches
// Rows up to 16384 values: 16 lanes hold 128 values of a row, 1024 lanes with two chunks each the longest.
constexpr size_t kMaxNormCols = 16384;
constexpr unsigned kForwardThreads = 256 * 1024;  // of all workgroups
constexpr unsigned kMostBackward = 256;            // workgroups

template <typename F> static unsigned groups_for(size_t rows, unsigned most)
{
  const size_t want = (rows + F::rows - 1) / F::rows;
  return (unsigned)(want < most ? want : most);
}

// Many rows of 513 to 768 values in a 16-bit type: half a wavefront with three chunks a lane, none idle at 768 and fewer
// everywhere.  This form : a wavefront with two chunks, us forward and backward, bf16: 16384 rows of 768 13.0 : 14.0 and 16.8 :
// 18.5, of 640 13.0 : 13.7 and 16.6 : 18.3, of 520 12.6 : 13.4 and 16.2 : 18.2; 8192 rows of 768 9.1 : 9.5 and 12.7 : 12.9, of 520
// 8.7 : 9.1 and 12.2 : 12.6; 4096 rows of 768 6.1 : 6.3 and 9.9 : 9.6.  In fp32 16384 rows of 768 28.5 : 26.5 and 29.6 : 29.3.
template <typename T> static bool half_wave(size_t rows, size_t cols)
{
  return T::bytes == 2 && cols > 512 && cols <= 768 && rows >= 8192;
}

template <typename T, typename Fn> static auto with_forward_form(size_t rows, size_t cols, Fn&& fn)
{
  if constexpr (T::bytes == 2)
    if (half_wave<T>(rows, cols)) return fn(Form<32, 3, 256>());
  if (cols <= 128) return fn(Form<16, 1, 256>());
  if (cols <= 256) return fn(Form<32, 1, 256>());
  if (cols <= 512) return fn(Form<64, 1, 256>());
  if (cols <= 1024) return fn(Form<64, 2, 256>());
  if (cols <= 2048) return fn(Form<128, 2, 256>());  // 8192 x 1536 bf16 14.7 us, with 256 lanes 17.7; fp32 25.3 and 24.7
  if (cols <= 4096) return fn(Form<256, 2, 256>());
  if (cols <= 8192) return fn(Form<512, 2, 512>());
  return fn(Form<1024, 2, 1024>());
}

// Large workgroups: as few shares of the parameters' gradients as there are compute units.
template <typename T, typename Fn> static auto with_backward_form(size_t rows, size_t cols, Fn&& fn)
{
  if constexpr (T::bytes == 2)
    if (half_wave<T>(rows, cols)) return fn(Form<32, 3, 512>());
  if (cols <= 128) return fn(Form<16, 1, 1024>());
  if (cols <= 256) return fn(Form<32, 1, 1024>());
  if (cols <= 512) return fn(Form<64, 1, 1024>());
  if (cols <= 1024) return fn(Form<64, 2, 512>());
  if (cols <= 2048) return fn(Form<256, 1, 1024>());
  if (cols <= 4096) return fn(Form<512, 1, 1024>());
  if (cols <= 8192) return fn(Form<1024, 1, 1024>());
  return fn(Form<1024, 2, 1024>());
}

// One workgroup for as many rows as it takes in four turns: it needs no second kernel for the parameters' gradients.
static unsigned backward_groups(size_t rows, size_t cols)
{
  return with_backward_form<F32>(rows, cols, [&](auto f) {  // of any type: there are kMostBackward where forms differ
    typedef decltype(f) F;
    return rows <= 4 * F::rows ? 1u : groups_for<F>(rows, kMostBackward);
  });
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
  const size_t groups = backward_groups(rows, cols);
  return groups > 1 ? groups * 2 * cols * sizeof(float) : 0;
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
    return with_forward_form<T>(rows, cols, [&](auto f) {
      typedef decltype(f) F;
      auto k = d_codes ? norm_forward_kernel<T, F, true> : norm_forward_kernel<T, F, false>;
      hipLaunchKernelGGL(k, dim3(groups_for<F>(rows, kForwardThreads / F::threads)), dim3(F::threads), 0, st,
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
    const size_t room = reduce ? cswap_layer_norm_workspace_bytes(rows, cols) : 0;
    if (room && !value_ptr(d_ws, CSWAP_DT_F32)) return CSWAP_E_ARG;
    if (ws_bytes < room) return CSWAP_E_NOMEM;
  }
  hipStream_t st = static_cast<hipStream_t>(stream);
  const Params g = {d_gamma, param_dtype};
  const unsigned grid = rows ? backward_groups(rows, cols) : 0;
  const GradParams grads = {d_dgamma, d_dbeta, param_dtype};
  if (rows) {
    const int e = with_type(dtype, [&](auto t) {
      typedef decltype(t) T;
      return with_backward_form<T>(rows, cols, [&](auto f) {
        typedef decltype(f) F;
        auto k = d_codes ? norm_backward_kernel<T, F, true> : norm_backward_kernel<T, F, false>;
        hipLaunchKernelGGL(k, dim3(grid), dim3(F::threads), 0, st, static_cast<const typename T::value*>(d_dy),
                           (size_t)dy_stride, static_cast<const typename T::value*>(d_x), (size_t)x_stride,
                           reinterpret_cast<const uint2*>(d_codes), d_scales, s, d_mean, d_rstd, g,
                           static_cast<typename T::value*>(d_dx), (size_t)dx_stride,
                           reduce && grid > 1 ? static_cast<float*>(d_ws) : nullptr,
                           grid > 1 ? GradParams{nullptr, nullptr, 0} : grads);
        return check_launch();
      });
    });
    if (e) return e;
  }
  if (!reduce || grid == 1) return CSWAP_OK;
  hipLaunchKernelGGL(norm_reduce_kernel, dim3((unsigned)((2 * cols + 31) / 32)), dim3(1024), 0, st, static_cast<const float*>(d_ws),
                     grid, (uint32_t)cols, grads);
  return check_launch();
}
