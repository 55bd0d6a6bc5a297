// q8_act.h -- activation functions and their slopes in fp32, for the kernels that apply them to values that are there anyway.
#pragma once
#include "q8_block.h"

namespace cswap {
namespace q8 {

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

struct Identity {
  template <typename T> static __device__ inline float value(float x) { return x; }
  template <typename T> static __device__ inline float slope(float) { return 1.0f; }
};

}  // namespace q8
}  // namespace cswap
