// q8_kernels.hip -- 8-bit activation checkpoints: codec, and activation functions whose forward pass leaves the checkpoint
// of its input and whose backward pass reads it.  The format is in q8_block.h.
//
// Memory bounds them all; a lane has 8 values, which is one or two 16-byte accesses and 8 bytes of codes, and a workgroup's are one
// run.  402 MB of fp32, tensors in turn, each kernel traced: to codes 103-111 us, back 79-91 (4.6-4.9 and 5.6-6.4 TB/s, read and
// written; a copy of 1 GB reaches 5.2).  GELU of 16384 x 768 fp32 so: forward 21.4-22.2, backward 21.5-22.4 us (5.1-5.3 TB/s); its
// tanh form of 16384 x 4096 bf16: 50-52 and 63-66 us (6.4-6.8 and 5.1-5.3 TB/s).  One tensor again and again, the form of the codec
// that hooks use : the plain one, us to codes and back: 402 MB of fp32 86 : 87 and 87 : 86, 134 MB of bf16 34.0 : 30.0 and 30.2 :
// 30.1, 201 MB of bf16 59 : 51.5 and 56 : 52.5, of fp16 57 : 50 and 54.5 : 52.  Two chunks a lane changed nothing (+-3 %).
// Nontemporal hints: loads cost where a tensor is still in the memory-side cache (50 MB fp32 GELU 18.3 -> 22), stores save 20 % of
// a bf16 tensor's decoding and cost 17-47 % of an fp32 one's; none is used.
#include <hip/hip_runtime.h>
#include "../../include/cswap_hip.h"
#include "common.h"
#include "q8_block.h"

namespace cswap {
namespace q8 {

constexpr int kThreads = 256;

// rows x cols values, a lane per chunk.  cpr: chunks of a row, its group padding included, so four neighbouring lanes are a
// group and no quad crosses a row.
// Columns are counted in chunks: a row may have more than 2^32 values, but fewer than 2^31 chunks.
struct Shape {
  uint32_t chunks, full;  // of the call; of a row those whose 8 values are all there
  int tail;               // values of the chunk behind these
  RowDivisor cpr;
};

struct Place {
  uint32_t row, at;  // the row, and the chunk in it
  int valid;         // values of the chunk that are there: 8, fewer at a row's end, 0 behind it
};

// FLAT: one row (a tensor whose rows are whole groups without gaps is one), chunk numbers are positions.
template <bool FLAT> __device__ inline Place place_of(uint32_t chunk, const Shape& s, size_t flat_cols)
{
  Place p;
  if (FLAT) {
    const size_t at = (size_t)chunk * kChunk;
    p.row = 0, p.at = 0;
    p.valid = at + kChunk <= flat_cols ? kChunk : at < flat_cols ? (int)(flat_cols - at) : 0;
  } else {
    p.row = divide(chunk, s.cpr);
    p.at = chunk - p.row * s.cpr.d;
    p.valid = p.at < s.full ? kChunk : p.at == s.full ? s.tail : 0;
  }
  return p;
}

template <bool FLAT> __device__ inline size_t offset_of(uint32_t chunk, const Place& p, size_t stride)
{
  return FLAT ? (size_t)chunk * kChunk : (size_t)p.row * stride + (size_t)p.at * kChunk;
}

__device__ inline void store_codes(uint32_t chunk, uint2 q, uint32_t scale, uint2* codes, uint8_t* scales)
{
  codes[chunk] = q;
  if ((chunk & (kChunksPerGroup - 1)) == 0) scales[chunk / kChunksPerGroup] = (uint8_t)scale;
}

template <typename T, bool FLAT, int SIGNS>
__global__ __launch_bounds__(kThreads) void q8_pack_kernel(const typename T::value* __restrict__ in, size_t stride, Shape s,
                                                           size_t flat_cols, uint2* __restrict__ codes,
                                                           uint8_t* __restrict__ scales)
{
  const uint32_t chunk = blockIdx.x * kThreads + threadIdx.x;
  if (chunk >= s.chunks) return;  // s.chunks is a multiple of 4: a quad leaves as a whole
  const Place p = place_of<FLAT>(chunk, s, flat_cols);
  float v[kChunk];
  load_chunk<T>(in + offset_of<FLAT>(chunk, p, stride), p.valid, v);
  uint32_t scale, max_bits = quad_max_bits(v), masked = 0;
  if (SIGNS == kHold && max_bits == 0x7f800000u) {  // a quad has one maximum: it goes this way as a whole
#pragma unroll
    for (int i = 0; i < kChunk; ++i)
      if (v[i] == -__builtin_inff()) masked |= 1u << i, v[i] = 0.0f;
    max_bits = quad_max_bits(v);
  }
  const uint2 q = encode_chunk<SIGNS>(v, max_bits, &scale, masked);
  store_codes(chunk, q, scale, codes, scales);
}

// MASKED: codes of -128 are minus infinity.  A form of its own, since the question costs up to 6 % (196608 x 512 bf16 52.5 : 56 us).
template <typename T, bool FLAT, bool MASKED>
__global__ __launch_bounds__(kThreads) void q8_unpack_kernel(const uint2* __restrict__ codes, const uint8_t* __restrict__ scales,
                                                             Shape s, size_t flat_cols, typename T::value* __restrict__ out,
                                                             size_t stride)
{
  const uint32_t chunk = blockIdx.x * kThreads + threadIdx.x;
  if (chunk >= s.chunks) return;
  const Place p = place_of<FLAT>(chunk, s, flat_cols);
  const float unit = unit_of(scales[chunk / kChunksPerGroup]);
  float v[kChunk];
  decode_chunk(codes[chunk], unit, v);
  if (MASKED) decode_masked(unit, v);
  store_chunk<T>(out + offset_of<FLAT>(chunk, p, stride), p.valid, v);
}

// ---------------------------------------------------------------- activation functions
// Each gives y(x) and its slope in fp32.  v_exp_f32 and v_rcp_f32 are off by one unit in the last place and take four turns of
// the vector unit each, of 18 to 30 in all for a value with its conversions: at 6 TB/s of 16-bit values these count.
constexpr float kLog2e = 1.4426950408889634f;

// s = 1 / (1 + e) and 1 - s = e s, the second without the cancellation, from e = 2^a, a = -z log2 e.  The callers hold a below 126,
// so that e and e s are finite.
struct Sigmoid {
  float s, one_minus;
};
__device__ inline Sigmoid sigmoid(float a)
{
  const float e = __builtin_amdgcn_exp2f(a);
  const float s = __builtin_amdgcn_rcpf(1.0f + e);
  return {s, e * s};
}

// x s(x).  Below -87 the function is less than 2e-36 off 0, and s must not meet a large x.
struct Silu {
  template <typename T> static __device__ inline float value(float x)
  {
    x = larger(x, -87.0f);
    return x * sigmoid(x * -kLog2e).s;
  }
  template <typename T> static __device__ inline float slope(float x)
  {
    x = larger(x, -87.0f);
    const Sigmoid g = sigmoid(x * -kLog2e);
    return g.s * __builtin_fmaf(x, g.one_minus, 1.0f);
  }
};

// x s(2 u), u = sqrt(2/pi) (x + 0.044715 x^3); below -10 the same.  Beyond 10 the sigmoid is 1, and the cubic's slope must not
// overflow.
struct GeluTanh {
  static constexpr float kC2 = 1.5957691216057308f, kC2A = kC2 * 0.044715f;  // 2 sqrt(2/pi) and that times a
  static __device__ inline Sigmoid parts(float x, float xx)
  {
    return sigmoid(x * __builtin_fmaf(-kLog2e * kC2A, xx, -kLog2e * kC2));
  }
  template <typename T> static __device__ inline float value(float x)
  {
    x = larger(x, -10.0f);
    return x * parts(x, x * x).s;
  }
  template <typename T> static __device__ inline float slope(float x)
  {
    x = smaller(larger(x, -10.0f), 10.0f);
    const float xx = x * x;
    const Sigmoid g = parts(x, xx);
    return g.s * __builtin_fmaf(x * g.one_minus, __builtin_fmaf(3.0f * kC2A, xx, kC2), 1.0f);
  }
};

// x Phi(x).  With z = |x| the tail Phi(-z) = exp(-z^2 / 2) R(z), R(z) = erfcx(z / sqrt 2) / 2: smooth, so a polynomial in
// t = 1 / (1 + p z) without a constant term holds it to a relative error, in the far tail too.  Coefficients: least squares
// weighted towards the smallest largest relative error over z from 0 to 40, 1.0e-7 for nine of them (fp32) and 1.1e-5 for six
// (16-bit types, whose half step is 4.9e-4 and more).  The library's erff costs some 40 instructions, this 22 and 18.
struct Gelu {
  struct Parts {
    float tail, e;  // Phi(-|x|), exp(-x^2 / 2)
  };
  template <typename T> static __device__ inline Parts parts(float x)
  {
    const float z = __builtin_fabsf(x);
    const float e = __builtin_amdgcn_exp2f(x * x * (-0.5f * kLog2e));
    float r;
    if (T::bytes == 4) {
      const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.28f, z, 1.0f));
      r = 0.025858310982584953f;
      r = __builtin_fmaf(r, t, -0.09804349392652512f);
      r = __builtin_fmaf(r, t, 0.09953393042087555f);
      r = __builtin_fmaf(r, t, -0.01241198368370533f);
      r = __builtin_fmaf(r, t, 0.07559163123369217f);
      r = __builtin_fmaf(r, t, 0.08288782089948654f);
      r = __builtin_fmaf(r, t, 0.10318589955568314f);
      r = __builtin_fmaf(r, t, 0.11169400811195374f);
      r = __builtin_fmaf(r, t, 0.11170392483472824f) * t;
    } else {
      const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.32f, z, 1.0f));
      r = -0.06677431613206863f;
      r = __builtin_fmaf(r, t, 0.13958518207073212f);
      r = __builtin_fmaf(r, t, 0.04961468279361725f);
      r = __builtin_fmaf(r, t, 0.12305107712745667f);
      r = __builtin_fmaf(r, t, 0.1268281787633896f);
      r = __builtin_fmaf(r, t, 0.12768970429897308f) * t;
    }
    return {r * e, e};
  }
  template <typename T> static __device__ inline float value(float x)
  {
    // x >= 0: x - x tail, else x tail; the product with the tail is 0 at infinity, not NaN (a NaN comes with the tail)
    const float z = __builtin_amdgcn_fmed3f(__builtin_fabsf(x), 0.0f, 1e30f);
    return __builtin_fmaf(-z, parts<T>(x).tail, __builtin_amdgcn_fmed3f(x, 0.0f, __builtin_inff()));
  }
  template <typename T> static __device__ inline float slope(float x)
  {
    const Parts p = parts<T>(x);
    return __builtin_fmaf(x * 0.3989422804014327f, p.e, x > 0.0f ? 1.0f - p.tail : p.tail);
  }
};

template <typename T, typename A, bool FLAT>
__global__ __launch_bounds__(kThreads) void q8_act_forward_kernel(const typename T::value* __restrict__ x, size_t x_stride,
                                                                  Shape s, size_t flat_cols, typename T::value* __restrict__ y,
                                                                  size_t y_stride, uint2* __restrict__ codes,
                                                                  uint8_t* __restrict__ scales)
{
  const uint32_t chunk = blockIdx.x * kThreads + threadIdx.x;
  if (chunk >= s.chunks) return;
  const Place p = place_of<FLAT>(chunk, s, flat_cols);
  float v[kChunk];
  load_chunk<T>(x + offset_of<FLAT>(chunk, p, x_stride), p.valid, v);
  if (codes) {
    uint32_t scale;
    const uint2 q = encode_chunk(v, quad_max_bits(v), &scale);
    store_codes(chunk, q, scale, codes, scales);
  }
#pragma unroll
  for (int i = 0; i < kChunk; ++i) v[i] = A::template value<T>(v[i]);
  store_chunk<T>(y + offset_of<FLAT>(chunk, p, y_stride), p.valid, v);
}

template <typename T, typename A, bool FLAT>
__global__ __launch_bounds__(kThreads) void q8_act_backward_kernel(const typename T::value* __restrict__ dy, size_t dy_stride,
                                                                   const uint2* __restrict__ codes,
                                                                   const uint8_t* __restrict__ scales, Shape s, size_t flat_cols,
                                                                   typename T::value* __restrict__ dx, size_t dx_stride)
{
  const uint32_t chunk = blockIdx.x * kThreads + threadIdx.x;
  if (chunk >= s.chunks) return;
  const Place p = place_of<FLAT>(chunk, s, flat_cols);
  float v[kChunk], g[kChunk];
  load_chunk<T>(dy + offset_of<FLAT>(chunk, p, dy_stride), p.valid, g);
  decode_chunk(codes[chunk], unit_of(scales[chunk / kChunksPerGroup]), v);
#pragma unroll
  for (int i = 0; i < kChunk; ++i) g[i] *= A::template slope<T>(v[i]);
  store_chunk<T>(dx + offset_of<FLAT>(chunk, p, dx_stride), p.valid, g);
}

// ---------------------------------------------------------------- launches
// What a call works on, after its checks.
struct Call {
  Shape s;
  size_t flat_cols;
  bool flat;
  unsigned grid;
};

// CSWAP_OK and *c, or an error.  Strides: 0 is `cols`; the call is flat where no operand has a gap between its rows.
static int plan(size_t rows, size_t cols, ptrdiff_t* stride_a, ptrdiff_t* stride_b, Call* c)
{
  if (int e = check_rows(rows, cols, stride_a)) return e;
  if (stride_b)
    if (int e = check_rows(rows, cols, stride_b)) return e;
  c->flat = rows <= 1 || (cols % kGroup == 0 && *stride_a == (ptrdiff_t)cols && (!stride_b || *stride_b == (ptrdiff_t)cols));
  const size_t cpr = pitch_of(cols) / kChunk, chunks = rows * cpr;
  c->flat_cols = rows * cols;
  c->s = {(uint32_t)chunks, (uint32_t)(cols / kChunk), (int)(cols % kChunk), c->flat ? RowDivisor{1, 0, 0} : row_divisor((uint32_t)cpr)};
  c->grid = (unsigned)((chunks + kThreads - 1) / kThreads);
  return CSWAP_OK;
}

template <typename T>
static int pack(const void* in, size_t stride, int keep_sign, const Call& c, int8_t* codes, uint8_t* scales, hipStream_t st)
{
  auto k = keep_sign == CSWAP_Q8_HOLD ? (c.flat ? q8_pack_kernel<T, true, kHold> : q8_pack_kernel<T, false, kHold>)
           : keep_sign                ? (c.flat ? q8_pack_kernel<T, true, kAllSigns> : q8_pack_kernel<T, false, kAllSigns>)
                                      : (c.flat ? q8_pack_kernel<T, true, kRounded> : q8_pack_kernel<T, false, kRounded>);
  hipLaunchKernelGGL(k, dim3(c.grid), dim3(kThreads), 0, st, static_cast<const typename T::value*>(in), stride, c.s, c.flat_cols,
                     reinterpret_cast<uint2*>(codes), scales);
  return check_launch();
}

template <typename T>
static int unpack(const int8_t* codes, const uint8_t* scales, const Call& c, void* out, size_t stride, bool masked, hipStream_t st)
{
  auto k = masked ? (c.flat ? q8_unpack_kernel<T, true, true> : q8_unpack_kernel<T, false, true>)
                  : (c.flat ? q8_unpack_kernel<T, true, false> : q8_unpack_kernel<T, false, false>);
  hipLaunchKernelGGL(k, dim3(c.grid), dim3(kThreads), 0, st, reinterpret_cast<const uint2*>(codes), scales, c.s, c.flat_cols,
                     static_cast<typename T::value*>(out), stride);
  return check_launch();
}

template <typename T, typename A>
static int forward(const void* x, size_t xs, const Call& c, void* y, size_t ys, int8_t* codes, uint8_t* scales, hipStream_t st)
{
  auto k = c.flat ? q8_act_forward_kernel<T, A, true> : q8_act_forward_kernel<T, A, false>;
  hipLaunchKernelGGL(k, dim3(c.grid), dim3(kThreads), 0, st, static_cast<const typename T::value*>(x), xs, c.s, c.flat_cols,
                     static_cast<typename T::value*>(y), ys, reinterpret_cast<uint2*>(codes), scales);
  return check_launch();
}

template <typename T, typename A>
static int backward(const void* dy, size_t dys, const int8_t* codes, const uint8_t* scales, const Call& c, void* dx, size_t dxs,
                    hipStream_t st)
{
  auto k = c.flat ? q8_act_backward_kernel<T, A, true> : q8_act_backward_kernel<T, A, false>;
  hipLaunchKernelGGL(k, dim3(c.grid), dim3(kThreads), 0, st, static_cast<const typename T::value*>(dy), dys,
                     reinterpret_cast<const uint2*>(codes), scales, c.s, c.flat_cols, static_cast<typename T::value*>(dx), dxs);
  return check_launch();
}

template <typename T>
static int forward_of(int kind, const void* x, size_t xs, const Call& c, void* y, size_t ys, int8_t* codes, uint8_t* scales,
                      hipStream_t st)
{
  switch (kind) {
    case CSWAP_ACT_GELU: return forward<T, Gelu>(x, xs, c, y, ys, codes, scales, st);
    case CSWAP_ACT_GELU_TANH: return forward<T, GeluTanh>(x, xs, c, y, ys, codes, scales, st);
    default: return forward<T, Silu>(x, xs, c, y, ys, codes, scales, st);
  }
}

template <typename T>
static int backward_of(int kind, const void* dy, size_t dys, const int8_t* codes, const uint8_t* scales, const Call& c, void* dx,
                       size_t dxs, hipStream_t st)
{
  switch (kind) {
    case CSWAP_ACT_GELU: return backward<T, Gelu>(dy, dys, codes, scales, c, dx, dxs, st);
    case CSWAP_ACT_GELU_TANH: return backward<T, GeluTanh>(dy, dys, codes, scales, c, dx, dxs, st);
    default: return backward<T, Silu>(dy, dys, codes, scales, c, dx, dxs, st);
  }
}

static bool act_known(int kind) { return kind >= CSWAP_ACT_GELU && kind <= CSWAP_ACT_SILU; }

}  // namespace q8
}  // namespace cswap

using namespace cswap;
using namespace cswap::q8;

extern "C" size_t cswap_q8_code_pitch(size_t cols) { return pitch_of(cols); }
extern "C" size_t cswap_q8_scale_pitch(size_t cols) { return groups_of(cols); }

extern "C" int cswap_q8_pack(const void* d_in, int dtype, size_t rows, size_t cols, ptrdiff_t stride, int keep_sign,
                             int8_t* d_codes, uint8_t* d_scales, cswap_stream_t stream)
{
  Call c;
  if (int e = plan(rows, cols, &stride, nullptr, &c)) return e;
  if (!dtype_known(dtype)) return CSWAP_E_ARG;
  if (rows == 0) return CSWAP_OK;
  if (!value_ptr(d_in, dtype) || !checkpoint_ptrs(d_codes, d_scales)) return CSWAP_E_ARG;
  hipStream_t st = static_cast<hipStream_t>(stream);
  switch (dtype) {
    case CSWAP_DT_F32: return pack<F32>(d_in, (size_t)stride, keep_sign, c, d_codes, d_scales, st);
    case CSWAP_DT_BF16: return pack<BF16>(d_in, (size_t)stride, keep_sign, c, d_codes, d_scales, st);
    default: return pack<F16>(d_in, (size_t)stride, keep_sign, c, d_codes, d_scales, st);
  }
}

static int unpack_any(const int8_t* d_codes, const uint8_t* d_scales, size_t rows, size_t cols, void* d_out, int dtype,
                      ptrdiff_t stride, bool masked, hipStream_t st)
{
  Call c;
  if (int e = plan(rows, cols, &stride, nullptr, &c)) return e;
  if (!dtype_known(dtype)) return CSWAP_E_ARG;
  if (rows == 0) return CSWAP_OK;
  if (!value_ptr(d_out, dtype) || !checkpoint_ptrs(d_codes, d_scales)) return CSWAP_E_ARG;
  switch (dtype) {
    case CSWAP_DT_F32: return unpack<F32>(d_codes, d_scales, c, d_out, (size_t)stride, masked, st);
    case CSWAP_DT_BF16: return unpack<BF16>(d_codes, d_scales, c, d_out, (size_t)stride, masked, st);
    default: return unpack<F16>(d_codes, d_scales, c, d_out, (size_t)stride, masked, st);
  }
}

extern "C" int cswap_q8_unpack(const int8_t* d_codes, const uint8_t* d_scales, size_t rows, size_t cols, void* d_out, int dtype,
                               ptrdiff_t stride, cswap_stream_t stream)
{
  return unpack_any(d_codes, d_scales, rows, cols, d_out, dtype, stride, false, static_cast<hipStream_t>(stream));
}

extern "C" int cswap_q8_unpack_held(const int8_t* d_codes, const uint8_t* d_scales, size_t rows, size_t cols, void* d_out, int dtype,
                                    ptrdiff_t stride, cswap_stream_t stream)
{
  return unpack_any(d_codes, d_scales, rows, cols, d_out, dtype, stride, true, static_cast<hipStream_t>(stream));
}

extern "C" int cswap_q8_act_forward(int kind, const void* d_x, int dtype, size_t rows, size_t cols, ptrdiff_t x_stride, void* d_y,
                                    ptrdiff_t y_stride, int8_t* d_codes, uint8_t* d_scales, cswap_stream_t stream)
{
  Call c;
  if (int e = plan(rows, cols, &x_stride, &y_stride, &c)) return e;
  if (!dtype_known(dtype) || !act_known(kind)) return CSWAP_E_ARG;
  if (rows == 0) return CSWAP_OK;
  if (!value_ptr(d_x, dtype) || !value_ptr(d_y, dtype)) return CSWAP_E_ARG;
  if ((d_codes || d_scales) && !checkpoint_ptrs(d_codes, d_scales)) return CSWAP_E_ARG;
  hipStream_t st = static_cast<hipStream_t>(stream);
  const size_t xs = (size_t)x_stride, ys = (size_t)y_stride;
  switch (dtype) {
    case CSWAP_DT_F32: return forward_of<F32>(kind, d_x, xs, c, d_y, ys, d_codes, d_scales, st);
    case CSWAP_DT_BF16: return forward_of<BF16>(kind, d_x, xs, c, d_y, ys, d_codes, d_scales, st);
    default: return forward_of<F16>(kind, d_x, xs, c, d_y, ys, d_codes, d_scales, st);
  }
}

extern "C" int cswap_q8_act_backward(int kind, const void* d_dy, int dtype, size_t rows, size_t cols, ptrdiff_t dy_stride,
                                     const int8_t* d_codes, const uint8_t* d_scales, void* d_dx, ptrdiff_t dx_stride,
                                     cswap_stream_t stream)
{
  Call c;
  if (int e = plan(rows, cols, &dy_stride, &dx_stride, &c)) return e;
  if (!dtype_known(dtype) || !act_known(kind)) return CSWAP_E_ARG;
  if (rows == 0) return CSWAP_OK;
  if (!value_ptr(d_dy, dtype) || !value_ptr(d_dx, dtype) || !checkpoint_ptrs(d_codes, d_scales)) return CSWAP_E_ARG;
  hipStream_t st = static_cast<hipStream_t>(stream);
  const size_t ds = (size_t)dy_stride, xs = (size_t)dx_stride;
  switch (dtype) {
    case CSWAP_DT_F32: return backward_of<F32>(kind, d_dy, ds, d_codes, d_scales, c, d_dx, xs, st);
    case CSWAP_DT_BF16: return backward_of<BF16>(kind, d_dy, ds, d_codes, d_scales, c, d_dx, xs, st);
    default: return backward_of<F16>(kind, d_dy, ds, d_codes, d_scales, c, d_dx, xs, st);
  }
}
