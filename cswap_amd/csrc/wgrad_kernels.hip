// wgrad_kernels.hip -- the gradients of a linear layer's weight and bias from the 8-bit checkpoint of its input:
//
//   dW[n][k] = sum over m of dY[m][n] x^[m][k],   db[n] = sum over m of dY[m][n],   x^ = code * 2^e
//
// x^ is one bf16 exactly (seven bits and a power of two), so a bf16 dY takes one matrix instruction per product and nothing is
// rounded before the fp32 sums.  An fp32 dY is cut into three bf16 of eight bits each, exactly: three matrix instructions of the
// 16-bit rate instead of one of the fp32 rate, which is a sixteenth of it.  An fp16 dY meets x^ as fp16, which is exact where
// the checkpoint was made from fp16.
//
// Both operands run along m in memory's slow direction, and a matrix instruction wants eight consecutive m of one row or
// column in a lane: they are turned round on their way into LDS.
#include <hip/hip_runtime.h>
#include "../../include/cswap_hip.h"
#include "common.h"
#include "q8_block.h"

namespace cswap {
namespace q8 {

typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef float f16v __attribute__((ext_vector_type(16)));

constexpr int kTile = 128, kStep = 32;   // tile of dW, rows of dY and x^ at a time
constexpr int kPitch = kStep + 8;        // of a tile's row in LDS, in 16-bit values: 16-byte pieces that spread over the banks

__device__ inline f16v mma(BF16, uint4 a, uint4 b, f16v c)
{
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf8, a), __builtin_bit_cast(bf8, b), c, 0, 0, 0);
}
__device__ inline f16v mma(F32, uint4 a, uint4 b, f16v c) { return mma(BF16(), a, b, c); }
__device__ inline f16v mma(F16, uint4 a, uint4 b, f16v c)
{
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
}

template <typename T> struct Feed {  // the type that the matrix instructions see, and how many of it make one dY
  typedef T type;
  static constexpr int parts = 1;
  static constexpr uint32_t one = 0x3f803f80u;
};
template <> struct Feed<F32> {
  typedef BF16 type;
  static constexpr int parts = 3;
  static constexpr uint32_t one = 0x3f803f80u;
};
template <> struct Feed<F16> {
  typedef F16 type;
  static constexpr int parts = 1;
  static constexpr uint32_t one = 0x3c003c00u;
};

struct GradShape {
  uint32_t rows, n, k, scale_pitch, step_rows;  // step_rows: rows of a split, a multiple of kStep
  size_t dy_stride, code_pitch;
};

// eight values of one column, m ascending, as three planes of bf16: the leading eight bits, the next, the last (cut, not rounded:
// the three add up to the value)
__device__ inline void split3(const float v[8], uint4 out[3])
{
  uint32_t a[3][8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    a[0][i] = __float_as_uint(v[i]) & 0xffff0000u;
    const float r = v[i] - __uint_as_float(a[0][i]);
    a[1][i] = __float_as_uint(r) & 0xffff0000u;
    a[2][i] = __float_as_uint(r - __uint_as_float(a[1][i]));
  }
#pragma unroll
  for (int p = 0; p < 3; ++p) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = __builtin_amdgcn_perm(a[p][2 * i + 1], a[p][2 * i], 0x07060302);
    out[p] = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

template <typename T> __global__ __launch_bounds__(256) void weight_grad_kernel(const typename T::value* __restrict__ dy,
                                                                                const int8_t* __restrict__ codes,
                                                                                const uint8_t* __restrict__ scales, GradShape s,
                                                                                float* __restrict__ dw, float* __restrict__ db)
{
  constexpr int P = Feed<T>::parts;
  typedef typename Feed<T>::type M;
  __shared__ uint16_t a_tile[P][kTile * kPitch], b_tile[kTile * kPitch];
  const uint32_t n0 = blockIdx.y * kTile, k0 = blockIdx.x * kTile;
  const uint32_t from = blockIdx.z * s.step_rows, to = min(s.rows, from + s.step_rows);
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int wn = (wave >> 1) * 64, wk = (wave & 1) * 64;
  const bool bias = db && blockIdx.x == 0 && (wave & 1) == 0;
  f16v acc[2][2] = {}, acc_b[2] = {};
  const int oct = threadIdx.x & 3, pair = threadIdx.x >> 2;  // this thread's eight m and two columns of both tiles
  for (uint32_t m0 = from; m0 < to; m0 += kStep) {
    __syncthreads();
    {
      float v[2][8];
      const uint32_t n = n0 + 2 * pair;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t m = m0 + oct * 8 + j;
#pragma unroll
        for (int e = 0; e < 2; ++e) v[e][j] = m < to && n + e < s.n ? to_float<T>(dy[(size_t)m * s.dy_stride + n + e]) : 0.0f;
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        uint4 w[P];
        if constexpr (P == 3) {
          split3(v[e], w);
        } else {
          w[0] = make_uint4(to_pair<M>(v[e][0], v[e][1]), to_pair<M>(v[e][2], v[e][3]), to_pair<M>(v[e][4], v[e][5]),
                            to_pair<M>(v[e][6], v[e][7]));
        }
#pragma unroll
        for (int p = 0; p < P; ++p) *reinterpret_cast<uint4*>(&a_tile[p][(2 * pair + e) * kPitch + oct * 8]) = w[p];
      }
    }
    {
      float v[2][8];
      const uint32_t k = k0 + 2 * pair;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t m = m0 + oct * 8 + j;
        const bool here = m < to && k < s.k;  // behind the last column codes are padding: k + 1 is there where k is
        const uint32_t q = here ? *reinterpret_cast<const uint16_t*>(codes + (size_t)m * s.code_pitch + k) : 0u;
        const float unit = here ? unit_of(scales[(size_t)m * s.scale_pitch + k / kGroup]) : 0.0f;
#pragma unroll
        for (int e = 0; e < 2; ++e) v[e][j] = code_value(q, e) * unit;
      }
#pragma unroll
      for (int e = 0; e < 2; ++e)
        *reinterpret_cast<uint4*>(&b_tile[(2 * pair + e) * kPitch + oct * 8]) =
            make_uint4(to_pair<M>(v[e][0], v[e][1]), to_pair<M>(v[e][2], v[e][3]), to_pair<M>(v[e][4], v[e][5]),
                       to_pair<M>(v[e][6], v[e][7]));
    }
    __syncthreads();
#pragma unroll
    for (int c = 0; c < kStep; c += 16) {
      uint4 b[2];
#pragma unroll
      for (int j = 0; j < 2; ++j)
        b[j] = *reinterpret_cast<const uint4*>(&b_tile[(wk + 32 * j + (lane & 31)) * kPitch + c + 8 * (lane >> 5)]);
#pragma unroll
      for (int p = P - 1; p >= 0; --p)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint4 a = *reinterpret_cast<const uint4*>(&a_tile[p][(wn + 32 * i + (lane & 31)) * kPitch + c + 8 * (lane >> 5)]);
#pragma unroll
          for (int j = 0; j < 2; ++j) acc[i][j] = mma(M(), a, b[j], acc[i][j]);
          if (bias) {
            const uint32_t o = Feed<T>::one;
            acc_b[i] = mma(M(), a, make_uint4(o, o, o, o), acc_b[i]);
          }
        }
    }
  }
  float* out = dw + (size_t)blockIdx.z * s.n * s.k;
  const uint32_t col = k0 + wk + (lane & 31);
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const uint32_t n = n0 + wn + 32 * i + 8 * (r / 4) + 4 * (lane >> 5) + r % 4;
      if (n >= s.n) continue;
#pragma unroll
      for (int j = 0; j < 2; ++j)
        if (col + 32 * j < s.k) out[(size_t)n * s.k + col + 32 * j] = acc[i][j][r];
      if (bias && (lane & 31) == 0) db[(size_t)blockIdx.z * s.n + n] = acc_b[i][r];
    }
}

// out[i] = sum over `parts` of part[.][i], rounded once
template <typename O> __global__ __launch_bounds__(256) void weight_grad_reduce_kernel(const float* __restrict__ part,
                                                                                       uint32_t parts, size_t count,
                                                                                       typename O::value* __restrict__ out)
{
  for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < count; i += (size_t)gridDim.x * 256) {
    float v = 0.0f;
    for (uint32_t p = 0; p < parts; ++p) v += part[(size_t)p * count + i];
    out[i] = from_float<O>(v);
  }
}

// ---------------------------------------------------------------- launches
constexpr size_t kMaxGradSide = (size_t)1 << 20;  // features on either side

struct GradPlan {
  unsigned tiles_n, tiles_k, splits;
  uint32_t step_rows;
};

static GradPlan grad_plan(size_t rows, size_t n, size_t k)
{
  GradPlan p;
  p.tiles_n = (unsigned)((n + kTile - 1) / kTile), p.tiles_k = (unsigned)((k + kTile - 1) / kTile);
  const size_t tiles = (size_t)p.tiles_n * p.tiles_k;
  size_t splits = tiles >= 512 ? 1 : (512 + tiles - 1) / tiles;
  const size_t most = (rows + 255) / 256;  // at least 256 rows to a split
  if (splits > most) splits = most < 1 ? 1 : most;
  size_t step = (rows + splits - 1) / splits;
  step = (step + kStep - 1) / kStep * kStep;
  if (step == 0) step = kStep;
  p.step_rows = (uint32_t)step;
  p.splits = (unsigned)(rows ? (rows + step - 1) / step : 1);
  return p;
}

}  // namespace q8
}  // namespace cswap

using namespace cswap;
using namespace cswap::q8;

static bool grad_sizes(size_t rows, size_t n, size_t k) { return n && k && n <= kMaxGradSide && k <= kMaxGradSide && rows < ((size_t)1 << 31); }

extern "C" size_t cswap_q8_weight_grad_workspace_bytes(size_t rows, size_t n, size_t k)
{
  if (!grad_sizes(rows, n, k)) return 0;
  return grad_plan(rows, n, k).splits * (n * k + n) * sizeof(float);
}

extern "C" int cswap_q8_weight_grad(const void* d_dy, int dtype, size_t rows, size_t n, ptrdiff_t dy_stride, const int8_t* d_codes,
                                    const uint8_t* d_scales, size_t k, void* d_dw, void* d_db, int out_dtype, void* d_ws,
                                    size_t ws_bytes, cswap_stream_t stream)
{
  ptrdiff_t unused = 0;
  if (int e = check_rows(rows, n, &dy_stride)) return e;
  if (int e = check_rows(rows, k, &unused)) return e;
  if (!dtype_known(dtype) || !dtype_known(out_dtype)) return CSWAP_E_ARG;
  if (!grad_sizes(rows, n, k)) return CSWAP_E_UNSUPPORTED;
  if (!value_ptr(d_dw, out_dtype) || (d_db && !value_ptr(d_db, out_dtype))) return CSWAP_E_ARG;
  if (rows && (!value_ptr(d_dy, dtype) || !checkpoint_ptrs(d_codes, d_scales))) return CSWAP_E_ARG;
  if (!value_ptr(d_ws, CSWAP_DT_F32)) return CSWAP_E_ARG;
  if (ws_bytes < cswap_q8_weight_grad_workspace_bytes(rows, n, k)) return CSWAP_E_NOMEM;
  const GradPlan p = grad_plan(rows, n, k);
  const GradShape s = {(uint32_t)rows, (uint32_t)n, (uint32_t)k, (uint32_t)groups_of(k), p.step_rows, (size_t)dy_stride, pitch_of(k)};
  float* part = static_cast<float*>(d_ws);
  float* part_b = part + (size_t)p.splits * n * k;
  hipStream_t st = static_cast<hipStream_t>(stream);
  const dim3 grid(p.tiles_k, p.tiles_n, p.splits);
  const auto launch = [&](auto t) {
    typedef decltype(t) T;
    hipLaunchKernelGGL(weight_grad_kernel<T>, grid, dim3(256), 0, st, static_cast<const typename T::value*>(d_dy), d_codes,
                       d_scales, s, part, d_db ? part_b : nullptr);
    return check_launch();
  };
  if (int e = dtype == CSWAP_DT_F32 ? launch(F32()) : dtype == CSWAP_DT_BF16 ? launch(BF16()) : launch(F16())) return e;
  const auto reduce = [&](auto t, const float* from, size_t count, void* out) {
    typedef decltype(t) O;
    const size_t want = (count + 255) / 256;
    hipLaunchKernelGGL(weight_grad_reduce_kernel<O>, dim3((unsigned)(want < 8192 ? want : 8192)), dim3(256), 0, st, from,
                       p.splits, count, static_cast<typename O::value*>(out));
    return check_launch();
  };
  const auto reduce_to = [&](const float* from, size_t count, void* out) {
    return out_dtype == CSWAP_DT_F32 ? reduce(F32(), from, count, out)
                                     : out_dtype == CSWAP_DT_BF16 ? reduce(BF16(), from, count, out) : reduce(F16(), from, count, out);
  };
  if (int e = reduce_to(part, n * k, d_dw)) return e;
  return d_db ? reduce_to(part_b, n, d_db) : CSWAP_OK;
}
