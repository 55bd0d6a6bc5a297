// q8_block.h -- 8-bit activation checkpoints: the format's arithmetic and the loads and stores that its kernels share.
//
// 32 consecutive values of a row share a power of two 2^e, e = clamp(floor(log2 max|x|) - 6, -126, 121), held as the byte
// e + 127; a value is the signed byte clamp(rint(x / 2^e), -127, 127).  A group that holds a NaN or an infinity has the byte
// 255 and codes of 0: 0 * 2^128 is NaN in fp32, so it decodes to 32 NaN without a comparison.
//
// Why a power of two: x / 2^e and q * 2^e are exact, so codes do not depend on who computes them, and q * 2^e, seven bits and
// a sign, is exactly one bf16, which is what feeds the matrix instructions of the weight gradient.  It costs up to one bit
// against a scale of max|x| / 127; a byte instead of 4 pays for groups of 32 where those have 128.
//
// A lane holds a chunk of 8 consecutive values (16 bytes of a 16-bit type, one code word pair), so a group is four neighbouring
// lanes and its maximum two DPP steps.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>
#include "../../include/cswap_hip.h"

namespace cswap {
namespace q8 {

constexpr int kGroup = 32, kChunk = 8, kChunksPerGroup = kGroup / kChunk;
constexpr size_t kMaxChunks = (size_t)1 << 31;  // of one call: chunk numbers are 32 bits (17 G values)

typedef uint32_t u4_any __attribute__((ext_vector_type(4), aligned(2)));  // 16 bytes at any address of a 16-bit value
typedef uint32_t u2_any __attribute__((ext_vector_type(2), aligned(2)));
typedef __bf16 bf2 __attribute__((ext_vector_type(2)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef float f2 __attribute__((ext_vector_type(2)));

struct F32 { typedef float value; static constexpr int bytes = 4; };
struct BF16 { typedef uint16_t value; static constexpr int bytes = 2; };
struct F16 { typedef uint16_t value; static constexpr int bytes = 2; };

inline size_t groups_of(size_t cols) { return (cols + kGroup - 1) / kGroup; }
inline size_t pitch_of(size_t cols) { return groups_of(cols) * kGroup; }

// ---------------------------------------------------------------- checks that the entry points share
inline bool dtype_known(int dtype) { return dtype == CSWAP_DT_F32 || dtype == CSWAP_DT_BF16 || dtype == CSWAP_DT_F16; }

inline bool value_ptr(const void* p, int dtype)
{
  return p && reinterpret_cast<uintptr_t>(p) % (dtype == CSWAP_DT_F32 ? 4 : 2) == 0;
}

inline bool checkpoint_ptrs(const int8_t* codes, const uint8_t* scales)
{
  return codes && scales && reinterpret_cast<uintptr_t>(codes) % 8 == 0;
}

// Extents of rows x cols values; a stride of 0 becomes cols.
inline int check_rows(size_t rows, size_t cols, ptrdiff_t* stride)
{
  if (cols == 0) return CSWAP_E_ARG;
  if (cols > kMaxChunks * kChunk || (rows && pitch_of(cols) / kChunk > (kMaxChunks - 1) / rows)) return CSWAP_E_UNSUPPORTED;
  if (*stride == 0) *stride = (ptrdiff_t)cols;
  if (*stride < (ptrdiff_t)cols && rows > 1) return CSWAP_E_ARG;
  if (*stride < 0 || (rows > 1 && (size_t)*stride > ((size_t)1 << 60) / rows)) return CSWAP_E_ARG;
  return CSWAP_OK;
}

// ---------------------------------------------------------------- values of a type
template <typename T> __device__ inline float to_float(typename T::value v);
template <> __device__ inline float to_float<F32>(float v) { return v; }
template <> __device__ inline float to_float<BF16>(uint16_t v) { return __uint_as_float((uint32_t)v << 16); }
template <> __device__ inline float to_float<F16>(uint16_t v) { return (float)__builtin_bit_cast(_Float16, v); }

// two values, rounded once to nearest even
template <typename T> __device__ inline uint32_t to_pair(float a, float b);
template <> __device__ inline uint32_t to_pair<BF16>(float a, float b)
{
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f2){a, b}, bf2));
}
template <> __device__ inline uint32_t to_pair<F16>(float a, float b)
{
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f2){a, b}, h2));
}

template <typename T> __device__ inline typename T::value from_float(float v);
template <> __device__ inline float from_float<F32>(float v) { return v; }
template <> __device__ inline uint16_t from_float<BF16>(float v) { return (uint16_t)to_pair<BF16>(v, 0.0f); }
template <> __device__ inline uint16_t from_float<F16>(float v) { return (uint16_t)to_pair<F16>(v, 0.0f); }

// ---------------------------------------------------------------- a chunk in memory
// `valid` of its 8 values are there (0 to 8); the others read as 0 and are not written.  Rows may start at any element: the
// 16-byte accesses need no alignment beyond the type's.
template <typename T> __device__ inline void load_chunk(const typename T::value* p, int valid, float v[8])
{
  if (valid >= kChunk) {
    if (T::bytes == 4) {
      const u4_any a = reinterpret_cast<const u4_any*>(p)[0], b = reinterpret_cast<const u4_any*>(p)[1];
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(a[i]), v[4 + i] = __uint_as_float(b[i]);
    } else {
      const u4_any a = *reinterpret_cast<const u4_any*>(p);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[2 * i] = to_float<T>((typename T::value)(a[i] & 0xffffu));
        v[2 * i + 1] = to_float<T>((typename T::value)(a[i] >> 16));
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < kChunk; ++i) v[i] = i < valid ? to_float<T>(p[i]) : 0.0f;
  }
}

// The same as it lies in memory.
template <typename T> __device__ inline void load_raw(const typename T::value* p, int valid, u4_any raw[T::bytes / 2])
{
  constexpr int W = T::bytes / 2;
  if (valid >= kChunk) {
#pragma unroll
    for (int h = 0; h < W; ++h) raw[h] = reinterpret_cast<const u4_any*>(p)[h];
  } else {
#pragma unroll
    for (int h = 0; h < W; ++h) raw[h] = (u4_any){0, 0, 0, 0};
#pragma unroll
    for (int e = 0; e < kChunk - 1; ++e)
      if (e < valid) {
        if constexpr (T::bytes == 4) raw[e / 4][e % 4] = __float_as_uint(p[e]);
        else raw[0][e / 2] |= (uint32_t)p[e] << (16 * (e & 1));
      }
  }
}

template <typename T> __device__ inline void store_chunk(typename T::value* p, int valid, const float v[8])
{
  if (valid >= kChunk) {
    if constexpr (T::bytes == 4) {
      u4_any a, b;
#pragma unroll
      for (int i = 0; i < 4; ++i) a[i] = __float_as_uint(v[i]), b[i] = __float_as_uint(v[4 + i]);
      reinterpret_cast<u4_any*>(p)[0] = a, reinterpret_cast<u4_any*>(p)[1] = b;
    } else {
      u4_any a;
#pragma unroll
      for (int i = 0; i < 4; ++i) a[i] = to_pair<T>(v[2 * i], v[2 * i + 1]);
      *reinterpret_cast<u4_any*>(p) = a;
    }
  } else {
#pragma unroll
    for (int i = 0; i < kChunk; ++i)
      if (i < valid) p[i] = from_float<T>(v[i]);
  }
}

// ---------------------------------------------------------------- the format
// The unit that a scale byte stands for; 255 gives infinity.
__device__ inline float unit_of(uint32_t scale) { return __uint_as_float(scale << 23); }

// The larger, the smaller of two values; NaN where either is.
__device__ inline float larger(float a, float b) { return __builtin_elementwise_maximum(a, b); }
__device__ inline float smaller(float a, float b) { return __builtin_elementwise_minimum(a, b); }

// The largest magnitude of the group that this lane's quad holds, as its bits: NaN compares largest, then infinity.  All four
// lanes of the quad have to run this.
__device__ inline uint32_t quad_max_bits(const float v[8])
{
  // v_maximum3_f32 takes magnitudes and passes NaN on
  float m = larger(__builtin_fabsf(v[0]), __builtin_fabsf(v[1]));
#pragma unroll
  for (int i = 2; i < kChunk; i += 2) m = larger(larger(m, __builtin_fabsf(v[i])), __builtin_fabsf(v[i + 1]));
  m = larger(m, __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, m), 0xb1, 0xf, 0xf, true)));  // lane ^ 1
  m = larger(m, __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, m), 0x4e, 0xf, 0xf, true)));  // lane ^ 2
  return __float_as_uint(m) & 0x7fffffffu;
}

// What becomes of a value that is not 0 but rounds to 0: the code 0, or 1 or -1, the nearest that has its sign, in every group or
// (kHold) in those that have no more than kMostLost of them.  Of one sign, as probabilities are, such codes add up to a bias: rows of a
// softmax over 512 logits N(0, 9) sum to 1.20 with all signs kept and to 0.991 with few or none (0.998 to 1.0002 for N(0, 1) to N(0, 2.25)
// with few).  kHold has minus infinity, which masks leave, as a value of its own, too: the code -128.
enum Signs { kRounded = 0, kAllSigns = 1, kHold = 2 };
constexpr int kMostLost = 2;
constexpr uint32_t kMaskCode = 0x80;

// Eight codes (byte i of the pair is value i) and the group's scale byte.  With kHold all four lanes of the quad have to run this, and v has 0
// in the places of `masked` (bit i: value i).
template <int SIGNS = kRounded>
__device__ inline uint2 encode_chunk(const float v[8], uint32_t max_bits, uint32_t* scale, uint32_t masked = 0)
{
  const int exponent = (int)(max_bits >> 23);
  const int b = max(exponent - 6, 1);
  const bool finite = exponent != 255;
  *scale = finite ? (uint32_t)b : 255u;
  const float inverse = __uint_as_float((uint32_t)(254 - b) << 23);
  // x * 2^-e + 1.5 * 2^23 is rint(x / 2^e) in the low byte: the product is exact, the sum rounds it to an integer
  constexpr float kMagic = 12582912.0f;
  uint32_t t[8];
#pragma unroll
  for (int i = 0; i < kChunk; ++i)
    t[i] = __float_as_uint(__builtin_amdgcn_fmed3f(__builtin_fmaf(v[i], inverse, kMagic), kMagic - 127.0f, kMagic + 127.0f));
  if (SIGNS != kRounded) {
    bool keep = true;
    if (SIGNS == kHold) {
      int lost = 0;
#pragma unroll
      for (int i = 0; i < kChunk; ++i) lost += t[i] == __float_as_uint(kMagic) && v[i] != 0.0f;
      lost += __builtin_amdgcn_mov_dpp(lost, 0xb1, 0xf, 0xf, true);  // lane ^ 1
      lost += __builtin_amdgcn_mov_dpp(lost, 0x4e, 0xf, 0xf, true);  // lane ^ 2
      keep = lost <= kMostLost;
    }
#pragma unroll
    for (int i = 0; i < kChunk; ++i)
      if (keep && t[i] == __float_as_uint(kMagic)) t[i] = v[i] > 0.0f ? 1u : v[i] < 0.0f ? 0xffu : 0u;
  }
  if (SIGNS == kHold) {
#pragma unroll
    for (int i = 0; i < kChunk; ++i)
      if (masked >> i & 1) t[i] = kMaskCode;
  }
  uint2 q;
  // v_perm_b32 numbers the bytes of its second operand 0 to 3 and those of its first 4 to 7
  q.x = __builtin_amdgcn_perm(__builtin_amdgcn_perm(t[3], t[2], 0x0c0c0400), __builtin_amdgcn_perm(t[1], t[0], 0x0c0c0400), 0x05040100);
  q.y = __builtin_amdgcn_perm(__builtin_amdgcn_perm(t[7], t[6], 0x0c0c0400), __builtin_amdgcn_perm(t[5], t[4], 0x0c0c0400), 0x05040100);
  if (!finite) q.x = q.y = 0u;
  return q;
}

__device__ inline float code_value(uint32_t word, int byte) { return (float)(int)(int8_t)(word >> (8 * byte)); }

__device__ inline void decode_chunk(uint2 q, float unit, float v[8])
{
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = code_value(q.x, i) * unit, v[4 + i] = code_value(q.y, i) * unit;
}

// Minus infinity where the code is -128, which no other value has.
__device__ inline void decode_masked(float unit, float v[8])
{
  const float code = -128.0f * unit;
  float least = smaller(v[0], v[1]);
#pragma unroll
  for (int i = 2; i < kChunk; i += 2) least = smaller(smaller(least, v[i]), v[i + 1]);
  if (least <= code) {
#pragma unroll
    for (int i = 0; i < kChunk; ++i)
      if (v[i] <= code) v[i] = -__builtin_inff();
  }
}

// ---------------------------------------------------------------- rows of chunks
// Division of a chunk number below 2^31 by the chunks of a row: n / d = (n * m) >> s with m = ceil(2^s / d), s = 31 + ceil(log2 d)
// (m < 2^32; the error n * (m d - 2^s) / (2^s d) stays below 1/d).
struct RowDivisor {
  uint32_t d, m, s;
};

inline RowDivisor row_divisor(uint32_t d)
{
  uint32_t l = 0;
  while (((uint64_t)1 << l) < d) ++l;
  const uint32_t s = 31 + l;
  return {d, (uint32_t)((((uint64_t)1 << s) + d - 1) / d), s};
}

__device__ inline uint32_t divide(uint32_t n, const RowDivisor& r) { return (uint32_t)(((uint64_t)n * r.m) >> r.s); }

}  // namespace q8
}  // namespace cswap
