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
  uint32_t rows, n, k, scale_pitch, step_rows;  // step_rows: rows of a split, a multiple of 64
  uint32_t tiles_n, tiles_k;
  size_t dy_stride, code_pitch;
};

// eight values as three planes of bf16: the leading eight bits, the next, the last (cut, not rounded: the three add up to the
// value)
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

typedef short s4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s4* lds_s4;

// eight m of one column for each lane, from two transposing reads of four; `at` as `Reader` has it
__device__ inline uint4 read_turned(const uint16_t* at, int four_rows)
{
  const s4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)(at));
  const s4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)(at + four_rows));
  const uint2 x = __builtin_bit_cast(uint2, lo), y = __builtin_bit_cast(uint2, hi);
  return make_uint4(x.x, x.y, y.x, y.y);
}

// A workgroup of four wavefronts makes a TN x TK tile of dW from one split of the rows, BK rows at a time.
template <typename T, int TN, int TK, int BK>
__global__ __launch_bounds__(256, 1) void weight_grad_kernel(const typename T::value* __restrict__ dy,
                                                             const int8_t* __restrict__ codes,
                                                             const uint8_t* __restrict__ scales, GradShape s,
                                                             float* __restrict__ dw, float* __restrict__ db)
{
  constexpr int P = Feed<T>::parts;
  typedef typename Feed<T>::type M;
  constexpr int FN = TN / 64, FK = TK / 64;                       // 32 x 32 pieces of a wavefront's quarter
  constexpr int kAChunks = TN / 8, kARows = 256 / kAChunks, kALoads = BK / kARows;
  constexpr int kBPieces = TK / 16, kBRows = 256 / kBPieces, kBLoads = BK / kBRows;
  constexpr int kAPlane = BK * TN, kStage = P * kAPlane + BK * TK;  // 16-bit values
  __shared__ __attribute__((aligned(16))) uint16_t lds[2][kStage];

  const uint32_t tile = blockIdx.x;
  const uint32_t tk = tile % s.tiles_k, rest = tile / s.tiles_k, tn = rest % s.tiles_n, split = rest / s.tiles_n;
  const uint32_t n0 = tn * TN, k0 = tk * TK;
  const uint32_t from = split * s.step_rows, to = min(s.rows, from + s.step_rows);
  const uint32_t stages = (to - from + BK - 1) / BK;
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;

  // staging: this thread's column chunk and first row of either operand
  const int a_chunk = tid % kAChunks, a_row = tid / kAChunks, b_piece = tid % kBPieces, b_row = tid / kBPieces;
  const uint32_t a_col = n0 + 8 * a_chunk, b_col = k0 + 16 * b_piece;
  const int a_valid = a_col + 8 <= s.n ? 8 : a_col < s.n ? (int)(s.n - a_col) : 0;
  const bool b_here = b_col < s.code_pitch;
  const bool a_edge = n0 + TN > s.n, b_edge = k0 + TK > s.code_pitch;
  u4_any a_raw[kALoads][T::bytes / 2], b_raw[kBLoads];
  uint32_t b_scale[kBLoads];

  auto load = [&](uint32_t m0) {
    const bool whole = m0 + BK <= to;
#pragma unroll
    for (int i = 0; i < kALoads; ++i) {
      const uint32_t m = m0 + a_row + i * kARows;
      const typename T::value* p = dy + (size_t)m * s.dy_stride + a_col;
      if (whole && !a_edge) {
#pragma unroll
        for (int h = 0; h < T::bytes / 2; ++h) a_raw[i][h] = reinterpret_cast<const u4_any*>(p)[h];
      } else {
#pragma unroll
        for (int h = 0; h < T::bytes / 2; ++h) a_raw[i][h] = (u4_any){0, 0, 0, 0};
        if (m < to) {
          if (a_valid == 8) {
#pragma unroll
            for (int h = 0; h < T::bytes / 2; ++h) a_raw[i][h] = reinterpret_cast<const u4_any*>(p)[h];
          } else {
#pragma unroll
            for (int e = 0; e < 7; ++e)
              if (e < a_valid) {
                if (T::bytes == 4) a_raw[i][(e / 4) % (T::bytes / 2)][e % 4] = reinterpret_cast<const uint32_t*>(p)[e];
                else a_raw[i][0][e / 2] |= (uint32_t)reinterpret_cast<const uint16_t*>(p)[e] << (16 * (e & 1));
              }
          }
        }
      }
    }
#pragma unroll
    for (int i = 0; i < kBLoads; ++i) {
      const uint32_t m = m0 + b_row + i * kBRows;
      b_raw[i] = (u4_any){0, 0, 0, 0}, b_scale[i] = 1;
      if ((whole && !b_edge) || (b_here && m < to)) {
        b_raw[i] = *reinterpret_cast<const u4_any*>(codes + (size_t)m * s.code_pitch + b_col);
        b_scale[i] = scales[(size_t)m * s.scale_pitch + b_col / kGroup];
      }
    }
  };

  // The tile of a stage lies in LDS as it does in memory, m by m, in chunks of 16 bytes whose order within a row depends on m:
  // the transposing reads take four rows at once, which have to lie in different banks.
  auto store = [&](uint16_t* buf) {
#pragma unroll
    for (int i = 0; i < kALoads; ++i) {
      const int m = a_row + i * kARows;
      uint16_t* at = buf + m * TN + 8 * (a_chunk ^ ((m & 3) << 2));
      if constexpr (P == 3) {
        float v[8];
        uint4 w[3];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = __uint_as_float(a_raw[i][0][e]), v[4 + e] = __uint_as_float(a_raw[i][1][e]);
        split3(v, w);
#pragma unroll
        for (int p = 0; p < 3; ++p) *reinterpret_cast<uint4*>(at + p * kAPlane) = w[p];
      } else {
        *reinterpret_cast<uint4*>(at) = make_uint4(a_raw[i][0][0], a_raw[i][0][1], a_raw[i][0][2], a_raw[i][0][3]);
      }
    }
#pragma unroll
    for (int i = 0; i < kBLoads; ++i) {
      const int m = b_row + i * kBRows;
      const float unit = unit_of(b_scale[i]);
      uint16_t* row = buf + P * kAPlane + m * TK;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float v[8];
        decode_chunk(make_uint2(b_raw[i][2 * h], b_raw[i][2 * h + 1]), unit, v);
        *reinterpret_cast<uint4*>(row + 8 * (h * kBPieces + (b_piece ^ (2 * (m & 3)) ^ (TK == 256 ? 8 * h : 0)))) =
            make_uint4(to_pair<M>(v[0], v[1]), to_pair<M>(v[2], v[3]), to_pair<M>(v[4], v[5]), to_pair<M>(v[6], v[7]));
      }
    }
  };

  // reading: a lane supplies the address of four values of row 8 (lane / 32) + (lane % 16) / 4 and gets column lane % 32
  const int quad_row = (lane & 15) >> 2, m_lane = 8 * (lane >> 5) + quad_row;
  int a_at[FN], b_at[FK];
#pragma unroll
  for (int i = 0; i < FN; ++i) {
    const int col = ((wave >> 1) * FN + i) * 32 + 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
    a_at[i] = m_lane * TN + 8 * ((col >> 3) ^ (quad_row << 2)) + (col & 7);
  }
#pragma unroll
  for (int j = 0; j < FK; ++j) {
    const int col = ((wave & 1) * FK + j) * 32 + 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
    const int piece = col >> 4, h = (col >> 3) & 1;
    b_at[j] = P * kAPlane + m_lane * TK + 8 * (h * kBPieces + (piece ^ (2 * quad_row) ^ (TK == 256 ? 8 * h : 0))) + (col & 7);
  }

  f16v acc[FN][FK] = {}, acc_b[FN] = {};
  if (stages) {
    load(from);
    store(lds[0]);
    if (stages > 1) load(from + BK);
  }
  for (uint32_t st = 0; st < stages; ++st) {
    __syncthreads();
    const uint16_t* buf = lds[st & 1];
    // the sum of dY's columns: a product with ones, each stage by one of the wavefronts that have its columns
    const bool bias = db && st % (2 * s.tiles_k) == 2 * tk + (wave & 1);
#pragma unroll
    for (int c = 0; c < BK / 16; ++c) {
      uint4 b[FK];
#pragma unroll
      for (int j = 0; j < FK; ++j) b[j] = read_turned(buf + b_at[j] + c * 16 * TK, 4 * TK);
#pragma unroll
      for (int p = P - 1; p >= 0; --p) {
        uint4 a[FN];
#pragma unroll
        for (int i = 0; i < FN; ++i) a[i] = read_turned(buf + p * kAPlane + a_at[i] + c * 16 * TN, 4 * TN);
#pragma unroll
        for (int i = 0; i < FN; ++i)
#pragma unroll
          for (int j = 0; j < FK; ++j) acc[i][j] = mma(M(), a[i], b[j], acc[i][j]);
        if (bias) {
          const uint32_t o = Feed<T>::one;
#pragma unroll
          for (int i = 0; i < FN; ++i) acc_b[i] = mma(M(), a[i], make_uint4(o, o, o, o), acc_b[i]);
        }
      }
    }
    if (st + 1 < stages) {
      store(lds[(st + 1) & 1]);
      if (st + 2 < stages) load(from + (st + 2) * BK);
    }
  }

  float* out = dw + (size_t)split * s.n * s.k;
  float* out_b = db + (size_t)((split * s.tiles_k + tk) * 2 + (wave & 1)) * s.n;
#pragma unroll
  for (int i = 0; i < FN; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const uint32_t n = n0 + ((wave >> 1) * FN + i) * 32 + 8 * (r / 4) + 4 * (lane >> 5) + r % 4;
      if (n >= s.n) continue;
#pragma unroll
      for (int j = 0; j < FK; ++j) {
        const uint32_t k = k0 + ((wave & 1) * FK + j) * 32 + (lane & 31);
        if (k < s.k) out[(size_t)n * s.k + k] = acc[i][j][r];
      }
      if (db && (lane & 31) == 0) out_b[n] = acc_b[i][r];
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
  bool large;  // 256 x 256 tiles, else 128 x 128
  unsigned tiles_n, tiles_k, splits;
  uint32_t step_rows;
};

static GradPlan grad_plan(size_t rows, size_t n, size_t k)
{
  GradPlan p;
  p.large = (rows + 2047) / 2048 * ((n + 255) / 256) * ((k + 255) / 256) >= 256;
  const size_t side = p.large ? 256 : 128, resident = p.large ? 256 : 512;
  p.tiles_n = (unsigned)((n + side - 1) / side), p.tiles_k = (unsigned)((k + side - 1) / side);
  const size_t tiles = (size_t)p.tiles_n * p.tiles_k;
  size_t splits = tiles >= resident ? 1 : resident / tiles;
  const size_t most = (rows + 255) / 256;  // at least 256 rows to a split
  if (splits > most) splits = most < 1 ? 1 : most;
  size_t step = (rows + splits - 1) / splits;
  step = (step + 63) / 64 * 64;
  if (step == 0) step = 64;
  p.step_rows = (uint32_t)step;
  p.splits = (unsigned)(rows ? (rows + step - 1) / step : 1);
  return p;
}

static size_t bias_parts(const GradPlan& p) { return (size_t)p.splits * p.tiles_k * 2; }

}  // namespace q8
}  // namespace cswap

using namespace cswap;
using namespace cswap::q8;

static bool grad_sizes(size_t rows, size_t n, size_t k) { return n && k && n <= kMaxGradSide && k <= kMaxGradSide && rows < ((size_t)1 << 31); }

extern "C" size_t cswap_q8_weight_grad_workspace_bytes(size_t rows, size_t n, size_t k)
{
  if (!grad_sizes(rows, n, k)) return 0;
  const GradPlan p = grad_plan(rows, n, k);
  return ((size_t)p.splits * n * k + bias_parts(p) * n) * sizeof(float);
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
  const GradShape s = {(uint32_t)rows, (uint32_t)n, (uint32_t)k, (uint32_t)groups_of(k), p.step_rows, p.tiles_n, p.tiles_k,
                       (size_t)dy_stride, pitch_of(k)};
  float* part = static_cast<float*>(d_ws);
  float* part_b = part + (size_t)p.splits * n * k;
  hipStream_t st = static_cast<hipStream_t>(stream);
  const auto launch = [&](auto t) {
    typedef decltype(t) T;
    constexpr int BK = T::bytes == 4 ? 32 : 64;
    auto kernel = p.large ? weight_grad_kernel<T, 256, 256, BK> : weight_grad_kernel<T, 128, 128, BK>;
    hipLaunchKernelGGL(kernel, dim3(p.tiles_n * p.tiles_k * p.splits), dim3(256), 0, st,
                       static_cast<const typename T::value*>(d_dy), d_codes, d_scales, s, part, d_db ? part_b : nullptr);
    return check_launch();
  };
  if (int e = dtype == CSWAP_DT_F32 ? launch(F32()) : dtype == CSWAP_DT_BF16 ? launch(BF16()) : launch(F16())) return e;
  const auto reduce = [&](auto t, const float* from, size_t parts, size_t count, void* out) {
    typedef decltype(t) O;
    const size_t want = (count + 255) / 256;
    hipLaunchKernelGGL(weight_grad_reduce_kernel<O>, dim3((unsigned)(want < 8192 ? want : 8192)), dim3(256), 0, st, from,
                       (uint32_t)parts, count, static_cast<typename O::value*>(out));
    return check_launch();
  };
  const auto reduce_to = [&](const float* from, size_t parts, size_t count, void* out) {
    return out_dtype == CSWAP_DT_F32    ? reduce(F32(), from, parts, count, out)
           : out_dtype == CSWAP_DT_BF16 ? reduce(BF16(), from, parts, count, out)
                                        : reduce(F16(), from, parts, count, out);
  };
  if (int e = reduce_to(part, p.splits, n * k, d_dw)) return e;
  return d_db ? reduce_to(part_b, bias_parts(p), n, d_db) : CSWAP_OK;
}
