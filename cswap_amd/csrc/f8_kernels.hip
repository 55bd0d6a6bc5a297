// f8_kernels.hip -- products of linear layers in 8-bit floating point (e4m3: sign, four bits of exponent, three of mantissa) with a power of two
// for each 128 values of a row of activations and for each 128 x 128 weights:
//
//   y[m][n] = sum over blocks c of 128 of  2^(sx[m][c] + sw[n / 128][c])  sum over k in c of x8[m][k] w8[n][k]  + bias[n]
//
// and the gradient of the input, dx = dy W, which is the same product with the codes of W turned round.  The scaled matrix instructions of
// this chip take a power of two for each lane's 32 values along k, so a block's two scales go into the instruction and nothing is
// multiplied behind it: that is why the scales are powers of two (it costs up to one bit of range against max / 448, none of precision).
//
// Traced: 16384 x 1024 x 4096 57 us (2.41 PFLOP/s; torch's fp8 product with one scale for all 61), 16384 x 4096 x 1024 70 (1.96; torch 70), 8192^3
// 387 at the clock of a first run (2.84), 480 at that of many; fp32 results 16384 x 768 x 768 28 (torch's bf16 product 26), 4096^3 119; a token through 4096 x 1024
// 4.1, through 8192 x 8192 19.5 (3.4 TB/s); 32 tokens 4.2 and 25.6 besides 2.6 and 4.0 to turn them into codes.
//
// Scale of a block: the least 2^s, s >= -126, with max|x| <= 448 * 2^s, held as the byte s + 127.  A block that holds a NaN or an infinity has
// codes of NaN (0x7f): every result that it goes into is NaN.
#include <hip/hip_runtime.h>
#include "../../include/cswap_hip.h"
#include "../../include/cswap_test_hooks.h"
#include "common.h"
#include "q8_block.h"
#include "q8_params.h"

namespace cswap {
namespace q8 {

constexpr int kBlock = 128;
constexpr size_t kMaxFeatures = (size_t)1 << 20;

typedef int i8v __attribute__((ext_vector_type(8)));
typedef uint32_t u4v __attribute__((ext_vector_type(4)));
typedef uint32_t u2v __attribute__((ext_vector_type(2)));
typedef float f16v __attribute__((ext_vector_type(16)));
typedef float f4v __attribute__((ext_vector_type(4)));

inline size_t blocks_of(size_t n) { return (n + kBlock - 1) / kBlock; }
constexpr size_t kRowPad = 256;  // activations' codes have room for whole tiles, so that products need not ask which rows are there
inline size_t padded(size_t rows) { return (rows + kRowPad - 1) / kRowPad * kRowPad; }

// The scale byte of a block whose largest magnitude has these bits; 0 where it is not finite.
__device__ inline uint32_t f8_scale(uint32_t max_bits)
{
  const int s = (int)(max_bits >> 23) - 8 + ((max_bits & 0x7fffffu) > 0x600000u);
  return max_bits >= 0x7f800000u ? 0u : (uint32_t)max(s, 1);
}

// Eight codes; a scale of 0: NaN.  The products are exact and at most 448.
__device__ inline uint2 f8_codes(const float v[8], uint32_t scale)
{
  const float inverse = __uint_as_float((254u - scale) << 23);
  int lo = 0, hi = 0;
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[0] * inverse, v[1] * inverse, lo, false);
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[2] * inverse, v[3] * inverse, lo, true);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(v[4] * inverse, v[5] * inverse, hi, false);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(v[6] * inverse, v[7] * inverse, hi, true);
  return scale ? make_uint2((uint32_t)lo, (uint32_t)hi) : make_uint2(0x7f7f7f7fu, 0x7f7f7f7fu);
}
__device__ inline uint8_t stored_scale(uint32_t scale) { return (uint8_t)(scale ? scale : 127u); }

// The largest magnitude of eight values, NaN if one is; then of the lanes of a row of 16.
__device__ inline float largest(const float v[8])
{
  float m = larger(__builtin_fabsf(v[0]), __builtin_fabsf(v[1]));
#pragma unroll
  for (int i = 2; i < 8; i += 2) m = larger(larger(m, __builtin_fabsf(v[i])), __builtin_fabsf(v[i + 1]));
  return m;
}
template <int CTRL> __device__ inline float larger_dpp(float m)
{
  return larger(m, __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, m), CTRL, 0xf, 0xf, true)));
}
__device__ inline float largest_of_16(float m)
{
  m = larger_dpp<0xb1>(m);          // lane ^ 1
  m = larger_dpp<0x4e>(m);          // lane ^ 2
  m = larger_dpp<0x141>(m);         // 7 - lane
  return larger_dpp<0x140>(m);      // 15 - lane
}

// ---------------------------------------------------------------- activations to codes
// 16 lanes to a block of 128 values of a row, 16 rows a workgroup: their scales, of one block, are neighbours in scales[block][row].
// Memory bounds it.
template <typename T>
__global__ __launch_bounds__(256) void f8_rows_kernel(const typename T::value* __restrict__ x, size_t stride, uint32_t rows, uint32_t cols, uint32_t blocks,
                                                      uint2* __restrict__ codes, uint8_t* __restrict__ scales, uint32_t scale_pitch)
{
  const uint32_t block = blockIdx.x % blocks, row = blockIdx.x / blocks * 16 + (threadIdx.x >> 4), lane = threadIdx.x & 15;
  const uint32_t at = min(row, rows - 1), col = block * kBlock + lane * kChunk;
  float v[8];
  load_chunk<T>(x + (size_t)at * stride + col, valid_at(col, cols), v);
  const uint32_t scale = f8_scale(__float_as_uint(largest_of_16(largest(v))) & 0x7fffffffu);
  const uint2 q = f8_codes(v, scale);
  if (row < rows) {
    codes[((size_t)row * blocks + block) * (kBlock / kChunk) + lane] = q;
    if (lane == 0) scales[(size_t)block * scale_pitch + row] = stored_scale(scale);
  }
}

// ---------------------------------------------------------------- weights to codes
// A workgroup has 128 x 128 weights in registers from load to store; the codes turned round go through LDS.
constexpr int kWeightThreads = 1024;
template <typename T>
__global__ __launch_bounds__(kWeightThreads) void f8_weight_kernel(const typename T::value* __restrict__ w, size_t stride, uint32_t n, uint32_t k, uint2* __restrict__ codes,
                                                        uint4* __restrict__ turned, uint8_t* __restrict__ scales)
{
  __shared__ uint32_t tile[kBlock][kBlock / 4 + 1];
  constexpr int kTurns = kBlock * 16 / kWeightThreads, kRows = kBlock / kTurns;  // of 16 lanes a row
  __shared__ float most[kWeightThreads / 64];
  const uint32_t kb = (k + kBlock - 1) / kBlock, nb = (n + kBlock - 1) / kBlock;
  const uint32_t bn = blockIdx.x / kb, bk = blockIdx.x % kb, lane = threadIdx.x & 15, first = threadIdx.x >> 4;
  const uint32_t col = bk * kBlock + lane * kChunk;
  const int valid = valid_at(col, k);
  u4_any raw[kTurns][T::bytes / 2];
#pragma unroll
  for (int i = 0; i < kTurns; ++i) {
    const uint32_t row = bn * kBlock + first + kRows * i;
    load_raw<T>(w + (size_t)min(row, n - 1) * stride + col, row < n ? valid : 0, raw[i]);
  }
  float m = 0.0f;
#pragma unroll
  for (int i = 0; i < kTurns; ++i) {
    float v[8];
    widen<T>(raw[i], v);
    m = larger(m, largest(v));
  }
  m = largest_of_16(m);
  m = larger(m, __shfl_xor(m, 16));
  m = larger(m, __shfl_xor(m, 32));
  if ((threadIdx.x & 63) == 0) most[threadIdx.x >> 6] = m;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kWeightThreads / 64; ++i) m = larger(m, most[i]);
  const uint32_t scale = f8_scale(__float_as_uint(m) & 0x7fffffffu);
  if (threadIdx.x == 0) scales[(size_t)bn * kb + bk] = stored_scale(scale);
#pragma unroll
  for (int i = 0; i < kTurns; ++i) {
    float v[8];
    widen<T>(raw[i], v);
    const uint2 q = f8_codes(v, scale);
    const uint32_t r = first + kRows * i;
    codes[((size_t)(bn * kBlock + r) * kb + bk) * (kBlock / kChunk) + lane] = q;
    if (turned) tile[r][2 * lane] = q.x, tile[r][2 * lane + 1] = q.y;
  }
  if (!turned) return;
  __syncthreads();
  // 16 codes of a column, from 16 rows
  for (uint32_t j = threadIdx.x; j < kBlock * (kBlock / 16); j += kWeightThreads) {
    const uint32_t c = j % kBlock, r = j / kBlock * 16;
    uint32_t out[4];
#pragma unroll
    for (int o = 0; o < 4; ++o) {
      uint32_t word = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) word |= ((tile[r + 4 * o + i][c >> 2] >> (8 * (c & 3))) & 0xffu) << (8 * i);
      out[o] = word;
    }
    turned[((size_t)(bk * kBlock + c) * nb + bn) * (kBlock / 16) + r / 16] = make_uint4(out[0], out[1], out[2], out[3]);
  }
}

// ---------------------------------------------------------------- products
struct F8Shape {
  uint32_t rows, n, blocks;        // of the result; blocks of 128 of what is summed over
  uint32_t scale_pitch;            // of the activations' scales[block][row]
  uint32_t step_n, step_k;         // of the weights' scales: from a block of the result's columns, of what is summed over, to the next
  uint32_t tiles_m, tiles_n;
  size_t y_stride;
};

// Memory from an address on that is the same in all lanes: loads take it from scalar registers, with a lane's offset and one that the lanes share,
// both 32 bits.  What is asked for behind its `bytes` reads as 0.
struct Window {
  __amdgpu_buffer_rsrc_t rsrc;
  __device__ inline Window(const uint8_t* p, uint32_t bytes) : rsrc(__builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(p), 0, (int)bytes, 0x00020000)) {}
  __device__ inline u4v load16(uint32_t lane, uint32_t all) const { return __builtin_amdgcn_raw_buffer_load_b128(rsrc, (int)lane, (int)all, 0); }
  __device__ inline u2v load8(uint32_t lane, uint32_t all) const { return __builtin_amdgcn_raw_buffer_load_b64(rsrc, (int)lane, (int)all, 0); }
  __device__ inline uint32_t load1(uint32_t lane, uint32_t all) const { return __builtin_amdgcn_raw_buffer_load_b8(rsrc, (int)lane, (int)all, 0); }
};
__device__ inline uint32_t scalar(uint32_t v) { return __builtin_amdgcn_readfirstlane(v); }

// Four neighbouring results of a row with their bias.
struct F8Out {
  void* y;
  const void* bias;  // NULL: none
  int dtype, bias_dtype;
};
// As it lies in memory, and its value: between the two a load is under way.
__device__ inline uint32_t bias_bits(const F8Out& o, uint32_t col)
{
  if (!o.bias) return 0;
  return o.bias_dtype == CSWAP_DT_F32 ? static_cast<const uint32_t*>(o.bias)[col] : static_cast<const uint16_t*>(o.bias)[col];
}
__device__ inline float bias_value(const F8Out& o, uint32_t bits)
{
  if (o.bias_dtype == CSWAP_DT_F32) return __uint_as_float(bits);
  return o.bias_dtype == CSWAP_DT_BF16 ? to_float<BF16>((uint16_t)bits) : to_float<F16>((uint16_t)bits);
}
__device__ inline float bias_at(const F8Out& o, uint32_t col) { return bias_value(o, bias_bits(o, col)); }
__device__ inline void store_one(const F8Out& o, size_t at, float v)
{
  if (o.dtype == CSWAP_DT_F32) static_cast<float*>(o.y)[at] = v;
  else static_cast<uint16_t*>(o.y)[at] = o.dtype == CSWAP_DT_BF16 ? from_float<BF16>(v) : from_float<F16>(v);
}

// Results in 16 bits come from the 8-bit matrix instructions.  These line up each eight neighbouring products before they add them, and cut each of them
// to a multiple of 2^-13 of the power of two in the largest (measured; the sums of eights are added in fp32): at most 7 * 2^-13 of the largest of
// eight, as a rule 3e-5 of the products' norm, a tenth of what rounding to fp16 costs and a fiftieth of bf16's, where values themselves are held to 2^-4.
// That is why it is taken: exact products are at half the rate.  Results in fp32 (EXACT) have them: they come from the codes as bf16, which hold them
// and their scales exactly, products are exact and sums fp32.
typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf2v __attribute__((ext_vector_type(2)));

// Eight codes as bf16.
__device__ inline uint4 f8_as_bf16(uint2 q, float unit)
{
  uint4 w;
  w.x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(q.x, unit, false));
  w.y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(q.x, unit, true));
  w.z = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(q.y, unit, false));
  w.w = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(q.y, unit, true));
  return w;
}

// Few rows: bound by the weights' bytes, which every workgroup reads once and no other reads.  A workgroup makes 16 columns; its eight wavefronts take
// blocks of k in turn, two of them under way, and add up through LDS.  A lane has 32 codes of one of 16 rows: that is one 16 x 16 x 128 matrix
// instruction a block, or four of 16 x 16 x 32 in bf16 (which of a lane's codes meet in which does not matter as long as both operands have
// them alike).  Up to 16 rows are turned into codes in registers, by every workgroup for itself: four lanes have a row's block.  More rows (PACKED,
// MF times 16) are codes already.
constexpr int kFewWaves = 8;
template <typename T, int MF, bool EXACT, bool PACKED>
__global__ __launch_bounds__(64 * kFewWaves) void f8_few_rows_kernel(const typename T::value* __restrict__ x, size_t x_stride, uint32_t k,
                                                                     const uint8_t* __restrict__ x_codes, const uint8_t* __restrict__ x_scales, F8Shape s,
                                                                     const uint8_t* __restrict__ w, const uint8_t* __restrict__ w_scales, F8Out out)
{
  __shared__ __attribute__((aligned(16))) float part[kFewWaves][MF * 256];
  const uint32_t wave = threadIdx.x >> 6, lane = threadIdx.x & 63, r = lane & 15, quarter = lane >> 4;
  const uint32_t col0 = blockIdx.x * 16, pitch = s.blocks * kBlock;
  f4v acc[MF];
#pragma unroll
  for (int f = 0; f < MF; ++f) acc[f] = (f4v){0, 0, 0, 0};
  const uint8_t* from = w + (size_t)(col0 + r) * pitch + quarter * 32;  // weights are filled up to whole blocks: the row is there
  struct Block {
    u4v w[2], x[PACKED ? MF : 1][2];
    u4_any raw[PACKED ? 1 : 4][T::bytes / 2];
    int w_scale, x_scale[MF];
  };
  auto load = [&](uint32_t b, Block& to) __attribute__((always_inline)) {
    const u4v* at = reinterpret_cast<const u4v*>(from + (size_t)b * kBlock);
    to.w[0] = at[0], to.w[1] = at[1];
    to.w_scale = w_scales[(size_t)(col0 / kBlock) * s.step_n + (size_t)b * s.step_k];
    if constexpr (PACKED) {
#pragma unroll
      for (int f = 0; f < MF; ++f) {  // there is room for whole tiles of rows
        const u4v* row = reinterpret_cast<const u4v*>(x_codes + (size_t)(16 * f + r) * pitch + b * kBlock + quarter * 32);
        to.x[f][0] = row[0], to.x[f][1] = row[1];
        to.x_scale[f] = x_scales[(size_t)b * s.scale_pitch + 16 * f + r];
      }
    } else {
      const uint32_t col = b * kBlock + quarter * 32;
#pragma unroll
      for (int c = 0; c < 4; ++c)
        load_raw<T>(x + (size_t)min(r, s.rows - 1) * x_stride + col + 8 * c, r < s.rows ? valid_at(col + 8 * c, k) : 0, to.raw[c]);
    }
  };
  auto multiply = [&](Block& of) __attribute__((always_inline)) {
    if constexpr (!PACKED) {
      float v[4][8];
#pragma unroll
      for (int c = 0; c < 4; ++c) widen<T>(of.raw[c], v[c]);
      float m = larger(larger(largest(v[0]), largest(v[1])), larger(largest(v[2]), largest(v[3])));
      m = larger(m, __shfl_xor(m, 16));
      m = larger(m, __shfl_xor(m, 32));
      const uint32_t scale = f8_scale(__float_as_uint(m) & 0x7fffffffu);
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const uint2 q = f8_codes(v[c], scale);
        of.x[0][c / 2][2 * (c & 1)] = q.x, of.x[0][c / 2][2 * (c & 1) + 1] = q.y;
      }
      of.x_scale[0] = stored_scale(scale);
    }
#pragma unroll
    for (int f = 0; f < MF; ++f) {
      if constexpr (EXACT) {
        const float unit = unit_of(of.x_scale[f]), w_unit = unit_of(of.w_scale);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const u4v a = of.w[c / 2], b = of.x[f][c / 2];
          const uint2 p = c & 1 ? make_uint2(a.z, a.w) : make_uint2(a.x, a.y), q = c & 1 ? make_uint2(b.z, b.w) : make_uint2(b.x, b.y);
          acc[f] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf8, f8_as_bf16(p, w_unit)), __builtin_bit_cast(bf8, f8_as_bf16(q, unit)), acc[f], 0, 0, 0);
        }
      } else {
        const i8v wf = __builtin_bit_cast(i8v, __builtin_shufflevector(of.w[0], of.w[1], 0, 1, 2, 3, 4, 5, 6, 7));
        const i8v xf = __builtin_bit_cast(i8v, __builtin_shufflevector(of.x[f][0], of.x[f][1], 0, 1, 2, 3, 4, 5, 6, 7));
        acc[f] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wf, xf, acc[f], 0, 0, 0, of.w_scale, 0, of.x_scale[f]);
      }
    }
  };
  for (uint32_t b = wave; b < s.blocks; b += 2 * kFewWaves) {
    Block one, two;
    load(b, one);
    const bool more = b + kFewWaves < s.blocks;
    if (more) load(b + kFewWaves, two);
    multiply(one);
    if (more) multiply(two);
  }
  // a lane has columns 4 * quarter and on of row r
#pragma unroll
  for (int f = 0; f < MF; ++f) *reinterpret_cast<float4*>(&part[wave][(f * 16 + r) * 16 + 4 * quarter]) = make_float4(acc[f][0], acc[f][1], acc[f][2], acc[f][3]);
  __syncthreads();
  for (uint32_t i = threadIdx.x; i < MF * 256; i += 64 * kFewWaves) {
    const uint32_t row = i / 16, col = col0 + i % 16;
    float sum = 0.0f;
#pragma unroll
    for (int p = 0; p < kFewWaves; ++p) sum += part[p][i];
    if (row < s.rows && col < s.n) store_one(out, (size_t)row * s.y_stride + col, sum + bias_at(out, col));
  }
}

// 16 bytes of results from place `at` on, of which `left` are wanted.
template <bool EXACT> __device__ inline void store_results(const F8Out& out, size_t at, uint32_t left, uint4 v)
{
  constexpr int kOut = EXACT ? 4 : 2, kEach = 16 / kOut;
  uint8_t* to = static_cast<uint8_t*>(out.y) + at * kOut;
  if (left >= kEach) {
    *reinterpret_cast<u4_any*>(to) = (u4_any){v.x, v.y, v.z, v.w};
  } else {
#pragma unroll 1
    for (uint32_t e = 0; e < left; ++e) {  // the first of them, then the others one place nearer
      if constexpr (EXACT) {
        reinterpret_cast<uint32_t*>(to)[e] = v.x;
        v = make_uint4(v.y, v.z, v.w, 0);
      } else {
        reinterpret_cast<uint16_t*>(to)[e] = (uint16_t)v.x;
        v = make_uint4(v.x >> 16 | v.y << 16, v.y >> 16 | v.z << 16, v.z >> 16 | v.w << 16, v.w >> 16);
      }
    }
  }
}

typedef int i4v __attribute__((ext_vector_type(4)));
template <bool EXACT> struct FragOf {
  typedef i8v type;
};
template <> struct FragOf<true> {
  typedef bf8 type;
};

// Many rows.  Four wavefronts, WM x WN of them, make a tile of TM rows x TN columns, a stage of 128 along k (EXACT: 64) at a time.  Stages lie in
// LDS row by row, 128 bytes each, as chunks of 16 whose order within a row depends on it, so that eight lanes that read eight rows meet in
// no bank; two stages, the next one on its way through registers while this one multiplies.  The results go out through LDS, too, in whole rows.
// Tiles of 256 x 256 and 256 x 192 leave a compute unit no room for a second workgroup that would multiply while this one begins or stores.  Their workgroups go on
// to further tiles instead, whose first two stages are on their way before the results go out (16384 x 4096 x 1024 71 us; 93 with a workgroup to a tile).  What that
// leaves is memory's: without storing results 59 to 65.
template <int TM, int TN, int WM, int WN, bool EXACT>
__global__ __launch_bounds__(64 * WM * WN, TM + TN > 256 ? WM * WN / 4 : 2) void f8_product_kernel(const uint8_t* __restrict__ x, const uint8_t* __restrict__ x_scales,
                                                                                       const uint8_t* __restrict__ w, const uint8_t* __restrict__ w_scales,
                                                                                       F8Shape s, F8Out out)
{
  constexpr int NT = 64 * WM * WN, FM = TM / WM / 32, FN = TN / WN / 32, kRows = TM + TN, kEach32 = NT / 8, kLoads = kRows / kEach32, kStage = kRows * kBlock;
  constexpr int kDeep = EXACT ? 64 : 128, kSteps = EXACT ? 4 : 2, kOut = EXACT ? 4 : 2;  // k of a stage, matrix instructions along it; bytes of a result
  static_assert(TM % kEach32 == 0 && TN % kEach32 == 0 && TN / WN <= kBlock, "loads within one operand, a wavefront's biases have room");
  constexpr bool kOn = TM + TN > 256;  // workgroups go on to further tiles
  static_assert(kOn || (TM * TN * kOut <= 2 * kStage && NT % (TN * kOut / 16) == 0), "a tile's results fit the stages, a pass is whole rows");
  constexpr bool kOneBlock = kBlock % (TN / WN) == 0;  // a wavefront's columns are of one block; else each 32 of them are
  // both stages of activations, then both of weights: a read's place in them is an instruction's 16-bit offset
  __shared__ __attribute__((aligned(16))) uint8_t lds[2 * kStage];
  __shared__ __attribute__((aligned(16))) uint8_t parts[kOn ? WM * WN * 4096 : 16];
  __shared__ __attribute__((aligned(16))) float bias[kOn ? WM * WN * 128 : TN];  // (a wavefront's columns for each)
  // XCDs take workgroups in turn; each gets neighbouring tiles, up to 16 along n before the next rows
  const uint32_t count = s.tiles_m * s.tiles_n, xcd = blockIdx.x % 8, each = count / 8, more = count % 8;
  struct Place {
    uint32_t m0, n0, stage;
  };
  auto begin_of = [&](uint32_t tile) __attribute__((always_inline)) {
    uint32_t at = xcd * each + min(xcd, more) + tile / 8;
    const uint32_t column = at / (16 * s.tiles_m), width = min(16u, s.tiles_n - 16 * column);
    at -= column * 16 * s.tiles_m;
    return Place{scalar(at / width * TM), scalar((16 * column + at % width) * TN), 0};
  };
  const int tid = threadIdx.x, wave = (int)scalar(tid >> 6), lane = tid & 63;
  Place now = begin_of(blockIdx.x);
  if constexpr (!kOn)
    for (int i = tid; i < TN; i += NT) bias[i] = bias_at(out, min(now.n0 + i, s.n - 1));
  const uint32_t pitch = s.blocks * kBlock;  // up to 2^20
  const uint32_t n_rows = (s.n + kBlock - 1) / kBlock * kBlock;

  // Staging: chunk tid % 8 of rows tid / 8 + 32 i.  Behind the last row of activations there is room, behind the last block of weights 0; either
  // goes into results that nobody stores.
  const int chunk = tid & 7, row = tid >> 3;
  constexpr int kCodes = kDeep / 8;  // codes of a chunk
  const uint32_t stages = s.blocks * (kBlock / kDeep), last = stages - 1, off = row * pitch + kCodes * chunk;
  u4v raw[EXACT ? 1 : kLoads];
  u2v raw8[EXACT ? kLoads : 1];
  uint32_t unit8[EXACT ? kLoads : 1];
  struct From {
    Window x, w;
  };
  auto from_of = [&](const Place& p) __attribute__((always_inline)) {
    return From{Window(x + (size_t)p.m0 * pitch, TM * pitch), Window(w + (size_t)p.n0 * pitch, min((uint32_t)TN, n_rows - p.n0) * pitch)};
  };
  auto load = [&](const Place& p, const From& window, int i) __attribute__((always_inline)) {
    const bool of_x = kEach32 * i < TM;
    const uint32_t from = (of_x ? kEach32 * i : kEach32 * i - TM) * pitch + p.stage * kDeep;
    if constexpr (EXACT) {
      raw8[i] = of_x ? window.x.load8(off, from) : window.w.load8(off, from);
      const uint32_t b = p.stage / 2;
      if (of_x) unit8[i] = x_scales[(size_t)b * s.scale_pitch + p.m0 + kEach32 * i + row];
      else unit8[i] = w_scales[(size_t)(min(p.n0 + kEach32 * i - TM, s.n - 1) / kBlock) * s.step_n + (size_t)b * s.step_k];
    } else {
      raw[i] = of_x ? window.x.load16(off, from) : window.w.load16(off, from);
    }
  };
  // addresses in LDS: a lane's, which the compiler takes as they are, and what an instruction adds to them
  typedef __attribute__((address_space(3))) uint8_t* Local;
  Local const stages_at = (Local)lds;
  auto as_it_is = [](Local p) __attribute__((always_inline)) {
    asm("" : "+v"(p));
    return p;
  };
  Local to_x = as_it_is(stages_at + row * kBlock + 16 * (chunk ^ ((row >> 1) & 7))), to_w = as_it_is(to_x + 2 * TM * kBlock);
  auto store = [&](int which, int i) __attribute__((always_inline)) {
    Local const to = kEach32 * i < TM ? to_x + (which * TM + kEach32 * i) * kBlock : to_w + (which * TN + kEach32 * i - TM) * kBlock;
    if constexpr (EXACT) {
      const uint4 v = f8_as_bf16(make_uint2(raw8[i].x, raw8[i].y), unit_of(unit8[i]));
      *(__attribute__((address_space(3))) u4v*)to = (u4v){v.x, v.y, v.z, v.w};
    } else {
      *(__attribute__((address_space(3))) u4v*)to = raw[i];
    }
  };

  // reading: lane l has 32 codes, or eight bf16, of row l % 32 from that many times l / 32 on
  const int wm = wave / WN, wn = wave % WN, r = lane & 31, half = lane >> 5;
  constexpr int kScales = kOneBlock ? 1 : FN;
  int xs[2][FM], ws[2][kScales];
  auto load_scales = [&](const Place& p, int which) __attribute__((always_inline)) {
    if constexpr (!EXACT) {
      const Window of_x(x_scales + (size_t)p.stage * s.scale_pitch + p.m0, TM);
#pragma unroll
      for (int i = 0; i < FM; ++i) xs[which][i] = (int)of_x.load1(wm * (TM / WM) + 32 * i + r, 0);
#pragma unroll
      for (int i = 0; i < kScales; ++i)
        ws[which][i] = w_scales[(size_t)(min(p.n0 + wn * (TN / WN) + 32 * i, s.n - 1) / kBlock) * s.step_n + (size_t)p.stage * s.step_k];
    }
  };
  constexpr int kWords = EXACT ? 1 : 2;  // of 16 bytes
  typedef typename FragOf<EXACT>::type Frag;
  Local x_at[kSteps * kWords], w_at[kSteps * kWords];
#pragma unroll
  for (int k = 0; k < kSteps * kWords; ++k) {
    const int c = 2 * kWords * (k / kWords) + kWords * half + k % kWords;
    x_at[k] = as_it_is(stages_at + (wm * (TM / WM) + r) * kBlock + 16 * (c ^ ((r >> 1) & 7)));
    w_at[k] = as_it_is(stages_at + (2 * TM + wn * (TN / WN) + r) * kBlock + 16 * (c ^ ((r >> 1) & 7)));
  }
  auto frag = [&](const Local* at, int first_row, int step) __attribute__((always_inline)) {
    if constexpr (EXACT) {
      return *(__attribute__((address_space(3))) Frag*)(at[step] + first_row * kBlock);
    } else {
      typedef __attribute__((address_space(3))) i4v* Half;
      return __builtin_shufflevector(*(Half)(at[2 * step] + first_row * kBlock), *(Half)(at[2 * step + 1] + first_row * kBlock), 0, 1, 2, 3, 4, 5, 6, 7);
    }
  };
  f16v acc[FN][FM] = {};
  Frag xf[FM], wf[2][FN];
  auto read_x = [&](int which, int step, int j) __attribute__((always_inline)) { xf[j] = frag(x_at, which * TM + 32 * j, step); };
  auto read_w = [&](int which, int step, int i) __attribute__((always_inline)) {
    wf[step & 1][i] = frag(w_at, which * TN + 32 * i, step);
  };
  auto multiply = [&](int step, int which, int i, int j) __attribute__((always_inline)) {
    if constexpr (EXACT) {
      acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(wf[step & 1][i], xf[j], acc[i][j], 0, 0, 0);
    } else {
      acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wf[step & 1][i], xf[j], acc[i][j], 0, 0, 0, ws[which][kOneBlock ? 0 : i], 0, xs[which][j]);
    }
  };
  {
    const From window = from_of(now);
#pragma unroll
    for (int i = 0; i < kLoads; ++i) load(now, window, i);
  }
  load_scales(now, 0);
#pragma unroll
  for (int i = 0; i < kLoads; ++i) store(0, i);
  {
    const Place second = {now.m0, now.n0, min(1u, last)};
    const From window = from_of(second);
#pragma unroll
    for (int i = 0; i < kLoads; ++i) load(second, window, i);
  }
  __syncthreads();
  auto read_first = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < FN; ++i) read_w(0, 0, i);
#pragma unroll
    for (int j = 0; j < FM; ++j) read_x(0, 0, j);
  };
  read_first();
  // A stage is kSteps times FM x FN products.  Beside a step's go the next step's fragments, those of the activations each into the registers of
  // the one that has just been multiplied for the last time; the last step's are the next stage's, behind a barrier before it.  Beside the
  // other steps the next stage goes from registers to LDS and the one after it is asked for.  The order is given, or the compiler
  // brings loads forward until registers run out.
  constexpr int kSlots = FM * FN, kMoveSlots = (kSteps - 1) * kSlots;
  auto one_stage = [&](int which, const Place& next, const Place& ahead) __attribute__((always_inline)) {
    load_scales(next, which ^ 1);
    const From window = from_of(ahead);
#pragma unroll
    for (int step = 0; step < kSteps; ++step) {
      const bool done = step + 1 == kSteps;
      const int from = done ? which ^ 1 : which, then = done ? 0 : step + 1;
      if (done) __syncthreads();
#pragma unroll
      for (int t = 0; t < kSlots; ++t) {
        const int j = t / FN, i = t % FN;
        multiply(step, which, i, j);
#pragma unroll
        for (int f = 0; f < FN; ++f)
          if (f * kSlots / FN == t) read_w(from, then, f);
        if (i == FN - 1) read_x(from, then, j);
        if (!done) {
#pragma unroll
          for (int l = 0; l < kLoads; ++l)
            if (l * kMoveSlots / kLoads == step * kSlots + t) {
              store(which ^ 1, l);
              load(ahead, window, l);
            }
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  };
  // A tile's stages, and the first two of the one that comes then.
  auto one_tile = [&](const Place& then) __attribute__((always_inline)) {
    for (uint32_t st = 0; st + 2 <= stages; st += 2) {
      const bool end = st + 2 >= stages;
      const Place second = {now.m0, now.n0, st + 1}, ahead = {end ? then.m0 : now.m0, end ? then.n0 : now.n0, end ? 0 : st + 2};
      one_stage(0, second, ahead);
      one_stage(1, ahead, Place{ahead.m0, ahead.n0, (uint32_t)min(ahead.stage + 1, last)});
    }
    if (stages & 1) {
      const Place again = {now.m0, now.n0, last};
      one_stage(0, again, again);
    }
  };
  if constexpr (kOn) {
    uint32_t mine[2];
    auto load_bias = [&]() __attribute__((always_inline)) {
#pragma unroll
      for (int e = 0; e < 2; ++e) mine[e] = bias_bits(out, min(now.n0 + wn * (TN / WN) + 64 * e + lane, s.n - 1));
    };
    load_bias();
    for (uint32_t tile = blockIdx.x;;) {
      const uint32_t then = tile + gridDim.x;
      const Place at = now, follows = then < count ? begin_of(then) : now;
      one_tile(follows);
      // Results while the next tile's first stages are in LDS and on their way: each wavefront turns 32 rows at a time, kWide of its fragments wide, in LDS of
      // its own, whose accesses it makes in order.
      constexpr int kWide = !EXACT && FN % 2 == 0 ? 2 : 1, kChunks = kWide * 2 * kOut, kEach = 16 / kOut, kAtOnce = 64 / kChunks;  // of 16 bytes in a row; results of one; rows
      float* const of_wave = bias + wave * 128;
      of_wave[lane] = bias_value(out, mine[0]), of_wave[64 + lane] = bias_value(out, mine[1]);
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
      auto results = [&](auto type) __attribute__((always_inline)) {
        typedef decltype(type) O;
        int l = lane;
        asm volatile("" : "+v"(l));  // places are made here, not kept in registers through the stages
        const int r = l & 31, half = l >> 5, below = l / kChunks, c = l % kChunks;
        uint8_t* const part = parts + wave * 4096;
        const uint32_t my_m = at.m0 + wm * (TM / WM), my_n = at.n0 + wn * (TN / WN);
        const bool whole = my_m + TM / WM <= s.rows && my_n + TN / WN <= s.n;
        uint8_t* const first = static_cast<uint8_t*>(out.y) + ((size_t)(my_m + below) * s.y_stride + my_n + kEach * c) * kOut;
#pragma unroll
        for (int h = 0; h < FN / kWide; ++h) {
          float4 b[kWide][4];
#pragma unroll
          for (int i = 0; i < kWide; ++i)
#pragma unroll
            for (int q = 0; q < 4; ++q) b[i][q] = *reinterpret_cast<const float4*>(&of_wave[32 * (kWide * h + i) + 8 * q + 4 * half]);
#pragma unroll
          for (int j = 0; j < FM; ++j) {
#pragma unroll
            for (int i = 0; i < kWide; ++i)
#pragma unroll
              for (int q = 0; q < 4; ++q) {
                const f16v& of = acc[kWide * h + i][j];
                const float v[4] = {of[4 * q] + b[i][q].x, of[4 * q + 1] + b[i][q].y, of[4 * q + 2] + b[i][q].z, of[4 * q + 3] + b[i][q].w};
                const int byte = (32 * i + 8 * q + 4 * half) * kOut;
                uint8_t* to = part + (r * kChunks + ((byte / 16) ^ (r & (kChunks - 1)))) * 16 + byte % 16;
                if constexpr (EXACT) *reinterpret_cast<float4*>(to) = make_float4(v[0], v[1], v[2], v[3]);
                else *reinterpret_cast<uint2*>(to) = make_uint2(to_pair<O>(v[0], v[1]), to_pair<O>(v[2], v[3]));
              }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
            __builtin_amdgcn_sched_barrier(0);
            uint4 v[32 / kAtOnce];
#pragma unroll
            for (int p = 0; p < 32 / kAtOnce; ++p) {
              const int row = kAtOnce * p + below;
              v[p] = *reinterpret_cast<const uint4*>(part + (row * kChunks + (c ^ (row & (kChunks - 1)))) * 16);
            }
            if (whole) {
#pragma unroll
              for (int p = 0; p < 32 / kAtOnce; ++p)
                *reinterpret_cast<u4_any*>(first + ((size_t)(32 * j + kAtOnce * p) * s.y_stride + 32 * kWide * h) * kOut) = (u4_any){v[p].x, v[p].y, v[p].z, v[p].w};
            } else {
#pragma unroll
              for (int p = 0; p < 32 / kAtOnce; ++p) {
                const uint32_t m = my_m + 32 * j + kAtOnce * p + below, n = my_n + 32 * kWide * h + kEach * c;
                if (m < s.rows && n < s.n) store_results<EXACT>(out, (size_t)m * s.y_stride + n, s.n - n, v[p]);
              }
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
          }
        }
      };
      if (EXACT || out.dtype == CSWAP_DT_BF16) results(BF16());
      else results(F16());
      if (then >= count) return;
      tile = then, now = follows;
#pragma unroll
      for (int i = 0; i < FN; ++i)
#pragma unroll
        for (int j = 0; j < FM; ++j) acc[i][j] = (f16v){};
      load_bias();
      read_first();  // again: there is no room for them beside the results
    }
  }
  if constexpr (!kOn) {
    const uint32_t m0 = now.m0, n0 = now.n0;
    one_tile(now);  // what it asks for of a next one goes nowhere
    // Results: lane l has row l % 32, columns 8 q + 4 (l / 32) + 0 to 3 for q = 0 to 3.  To LDS as rows of chunks of 16 bytes, in another order in
    // each row, and from there to memory.
    __syncthreads();  // the last stage asked for fragments of a stage that is not there
    constexpr int kChunks = TN * kOut / 16, kEach = 16 / kOut;  // chunks of a row, results of a chunk
    uint8_t* const tile = lds;
#pragma unroll
    for (int i = 0; i < FN; ++i)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int c = wn * (TN / WN) + 32 * i + 8 * q + 4 * half;
        const float4 b = *reinterpret_cast<const float4*>(bias + c);
#pragma unroll
        for (int j = 0; j < FM; ++j) {
          const int m = wm * (TM / WM) + 32 * j + r;
          uint8_t* to = tile + m * (TN * kOut) + 16 * ((c / kEach) ^ (m & (kChunks - 1))) + (c % kEach) * kOut;
          const float v[4] = {acc[i][j][4 * q] + b.x, acc[i][j][4 * q + 1] + b.y, acc[i][j][4 * q + 2] + b.z, acc[i][j][4 * q + 3] + b.w};
          if constexpr (EXACT) *reinterpret_cast<float4*>(to) = make_float4(v[0], v[1], v[2], v[3]);
          else if (out.dtype == CSWAP_DT_BF16) *reinterpret_cast<uint2*>(to) = make_uint2(to_pair<BF16>(v[0], v[1]), to_pair<BF16>(v[2], v[3]));
          else *reinterpret_cast<uint2*>(to) = make_uint2(to_pair<F16>(v[0], v[1]), to_pair<F16>(v[2], v[3]));
        }
      }
    __syncthreads();
    const uint32_t rows_here = min((uint32_t)TM, s.rows - m0);
#pragma unroll 8
    for (int pass = 0; pass < TM * kChunks / NT; ++pass) {
      const uint32_t m = (pass * NT + tid) / kChunks, c = tid % kChunks, n = n0 + c * kEach;
      if (m >= rows_here || n >= s.n) continue;
      const uint4 v = *reinterpret_cast<const uint4*>(tile + m * (TN * kOut) + 16 * (c ^ (m & (kChunks - 1))));
      store_results<EXACT>(out, (size_t)(m0 + m) * s.y_stride + n, s.n - n, v);
    }
  }
}

// ---------------------------------------------------------------- launches
constexpr size_t kFewRows = 16;  // up to which the product's kernel turns activations into codes itself
constexpr size_t kFewPacked = 32, kFewPackedSmall = 64, kSmallWeights = (size_t)1 << 24;

// Tiles of 256 rows are made by as many workgroups as there are compute units, each of which goes on to its next tile.  Stages lie in LDS in pairs,
// so that an odd number of them leaves the next tile's first one where a second would be: then a workgroup makes one tile (16384 x 4096 by 1024, 1152 and
// 1280 along k, 8, 9 and 10 blocks: 71, 85 and 83 us).
constexpr uint32_t kOnWorkgroups = 256;
static bool goes_on(size_t kb, bool exact) { return exact || kb % 2 == 0; }

// Few rows read the weights once, a workgroup to 16 columns; tiles of 128 x 128 have fewer workgroups but each value of the activations once for 128
// columns.  us with codes ready, the former : the latter, 32 rows through 4096 x 1024 4.2 : 7.6, 1024 x 4096 8.3 : 16.8, 8192 x 8192 25.6 :
// 30.0; 64 rows 6.0 : 7.8, 12.8 : 17.0, 42 : 31.
static bool few_rows(size_t rows, size_t weights) { return rows <= kFewPacked || (rows <= kFewPackedSmall && weights <= kSmallWeights); }

// Which kernel makes a product: 0 the one that turns few rows into codes itself, 32 and 64 the one for so many rows of codes, 128, 192 and 256 the one with tiles
// of so many columns.
static int product_form(size_t rows, size_t n, size_t k, bool exact)
{
  if (rows <= kFewRows) return 0;
  if (few_rows(rows, n * k)) return rows <= kFewPacked ? 32 : 64;
  const size_t kb = blocks_of(k);
  // By what rounds of tiles on all compute units take, us, in blocks along k: of 256 x 256 and 256 x 192, one to a compute unit (further rounds begin sooner
  // where workgroups go on), and of 128 x 128, two to one, of which one alone takes 0.62 of the time.  Measured, large : middle : small, bf16 16384 x 1024 x 4096
  // 57 : 80 : 70, 16384 x 4096 x 1024 70 : 87 : 82, 16384 x 768 x 2304 33 : 31 : 33, 16384 x 768 x 768 18 : 17 : 18, 8192 x 1152 x 1152 22 : 19 : 20, 2048^3 25 : - : 15;
  // fp32 4096^3 119 : 171 : 142, 16384 x 4096 x 1024 156 : 163 : 167, 25216 x 384 x 1536 51 : 41 : 44, 16384 x 768 x 768 34 : 28 : 29, 2048^3 53 : 45 : 26.
  const bool on = goes_on(kb, exact);
  auto tiles = [&](size_t tm, size_t tn) { return ((rows + tm - 1) / tm) * ((n + tn - 1) / tn); };
  auto one_each = [&](size_t count, double first, double further, double block) {
    const size_t rounds = (count + 255) / 256;
    return first + (rounds - 1) * (on ? further : first) + rounds * kb * block;
  };
  const size_t count = tiles(128, 128), rest = count % 512;
  const double small = 4.0 + (count / 512 + (rest == 0 ? 0.0 : rest <= 256 ? 0.62 : 1.0)) * (2.3 + (exact ? 2.25 : 1.02) * kb);
  const double middle = exact ? one_each(tiles(256, 192), 15.0, 9.0, 2.15) : one_each(tiles(256, 192), 10.5, 5.5, 1.12);
  const double large = exact ? one_each(tiles(256, 256), 13.0, 10.0, 3.34) : one_each(tiles(256, 256), 10.0, 4.3, 1.43);
  return large < small && large <= middle ? 256 : middle < small ? 192 : 128;
}

// Launches have fewer than 2^32 threads: 256 to 16 rows of a block, or to a tile of 128 x 128, 1024 to a block of weights.
static bool f8_shape(size_t rows, size_t n, size_t k)
{
  if (n > kMaxFeatures || k > kMaxFeatures || rows >= ((size_t)1 << 31)) return false;
  const size_t kb = blocks_of(k), nb = blocks_of(n), launch = (size_t)1 << 24;
  return (rows + 15) / 16 * kb < launch && blocks_of(rows) * nb < launch && nb * kb < launch / 4;
}

}  // namespace q8
}  // namespace cswap

using namespace cswap;
using namespace cswap::q8;

extern "C" int cswap_test_f8_linear_form(size_t rows, size_t n, size_t k, int out_dtype)
{
  return n == 0 || k == 0 || !f8_shape(rows, n, k) ? -1 : product_form(rows, n, k, out_dtype == CSWAP_DT_F32);
}

extern "C" size_t cswap_f8_linear_workspace_bytes(size_t rows, size_t k)
{
  if (rows <= kFewRows || k == 0 || !f8_shape(rows, 1, k)) return 0;
  return blocks_of(k) * padded(rows) * (kBlock + 1);
}

extern "C" int cswap_f8_pack_weight(const void* d_w, int dtype, size_t n, size_t k, ptrdiff_t stride, uint8_t* d_codes, uint8_t* d_turned,
                                    uint8_t* d_scales, cswap_stream_t stream)
{
  if (n == 0 || k == 0) return CSWAP_E_ARG;
  if (!f8_shape(1, n, k)) return CSWAP_E_UNSUPPORTED;
  if (int e = check_rows(n, k, &stride)) return e;
  if (!dtype_known(dtype) || !value_ptr(d_w, dtype) || !d_codes || !d_scales || reinterpret_cast<uintptr_t>(d_codes) % 16 ||
      reinterpret_cast<uintptr_t>(d_turned) % 16)
    return CSWAP_E_ARG;
  return with_type(dtype, [&](auto t) {
    typedef decltype(t) T;
    hipLaunchKernelGGL(f8_weight_kernel<T>, dim3((unsigned)(blocks_of(n) * blocks_of(k))), dim3(kWeightThreads), 0, static_cast<hipStream_t>(stream),
                       static_cast<const typename T::value*>(d_w), (size_t)stride, (uint32_t)n, (uint32_t)k, reinterpret_cast<uint2*>(d_codes),
                       reinterpret_cast<uint4*>(d_turned), d_scales);
    return check_launch();
  });
}

extern "C" int cswap_f8_linear(const void* d_x, int dtype, size_t rows, size_t k, ptrdiff_t x_stride, const uint8_t* d_codes, const uint8_t* d_scales,
                               size_t n, int turned, const void* d_bias, int bias_dtype, void* d_y, int out_dtype, ptrdiff_t y_stride, void* d_ws,
                               size_t ws_bytes, cswap_stream_t stream)
{
  if (n == 0 || k == 0) return CSWAP_E_ARG;
  if (!f8_shape(rows, n, k)) return CSWAP_E_UNSUPPORTED;
  if (int e = check_rows(rows, k, &x_stride)) return e;
  if (int e = check_rows(rows, n, &y_stride)) return e;
  if (!dtype_known(dtype) || !dtype_known(out_dtype) || !dtype_known(bias_dtype) || (turned != 0 && turned != 1)) return CSWAP_E_ARG;
  if (rows == 0) return CSWAP_OK;
  if (!value_ptr(d_x, dtype) || !value_ptr(d_y, out_dtype) || (d_bias && !value_ptr(d_bias, bias_dtype)) || !d_codes || !d_scales ||
      reinterpret_cast<uintptr_t>(d_codes) % 16)
    return CSWAP_E_ARG;
  const size_t need = cswap_f8_linear_workspace_bytes(rows, k);
  if (need && (!d_ws || reinterpret_cast<uintptr_t>(d_ws) % 16)) return CSWAP_E_ARG;
  if (ws_bytes < need) return CSWAP_E_NOMEM;
  hipStream_t st = static_cast<hipStream_t>(stream);
  const uint32_t kb = (uint32_t)blocks_of(k), nb = (uint32_t)blocks_of(n);
  F8Shape s = {(uint32_t)rows, (uint32_t)n, kb, (uint32_t)padded(rows), turned ? 1u : kb, turned ? nb : 1u, 0, 0, (size_t)y_stride};
  const F8Out out = {d_y, d_bias, out_dtype, bias_dtype};
  const bool exact = out_dtype == CSWAP_DT_F32;
  const int form = product_form(rows, n, k, exact);
  return with_type(dtype, [&](auto t) {
    typedef decltype(t) T;
    const typename T::value* x = static_cast<const typename T::value*>(d_x);
    const dim3 columns((unsigned)((n + 15) / 16)), threads(64 * kFewWaves);
    if (form == 0) {
      auto f = exact ? f8_few_rows_kernel<T, 1, true, false> : f8_few_rows_kernel<T, 1, false, false>;
      hipLaunchKernelGGL(f, columns, threads, 0, st, x, (size_t)x_stride, (uint32_t)k, nullptr, nullptr, s, d_codes, d_scales, out);
      return check_launch();
    }
    uint8_t *codes = static_cast<uint8_t*>(d_ws), *scales = codes + padded(rows) * kb * kBlock;
    hipLaunchKernelGGL(f8_rows_kernel<T>, dim3((unsigned)((rows + 15) / 16 * kb)), dim3(256), 0, st, x, (size_t)x_stride, (uint32_t)rows, (uint32_t)k, kb,
                       reinterpret_cast<uint2*>(codes), scales, s.scale_pitch);
    if (int e = check_launch()) return e;
    if (form <= 64) {
      auto few = [&](auto f) {
        hipLaunchKernelGGL(f, columns, threads, 0, st, nullptr, 0, (uint32_t)k, codes, scales, s, d_codes, d_scales, out);
        return check_launch();
      };
      if (exact) return form == 32 ? few(f8_few_rows_kernel<F32, 2, true, true>) : few(f8_few_rows_kernel<F32, 4, true, true>);
      return form == 32 ? few(f8_few_rows_kernel<F32, 2, false, true>) : few(f8_few_rows_kernel<F32, 4, false, true>);
    }
    auto launch = [&](auto f, uint32_t tm, uint32_t tn, uint32_t threads) {
      s.tiles_m = (uint32_t)((rows + tm - 1) / tm), s.tiles_n = (uint32_t)((n + tn - 1) / tn);
      const uint32_t count = s.tiles_m * s.tiles_n;
      hipLaunchKernelGGL(f, dim3(tm + tn > 256 && goes_on(kb, exact) && count > kOnWorkgroups ? kOnWorkgroups : count), dim3(threads), 0, st, codes, scales, d_codes, d_scales, s, out);
      return check_launch();
    };
    if (exact) {
      if (form == 256) return launch(f8_product_kernel<256, 256, 2, 2, true>, 256, 256, 256);
      if (form == 192) return launch(f8_product_kernel<256, 192, 2, 2, true>, 256, 192, 256);
      return launch(f8_product_kernel<128, 128, 2, 2, true>, 128, 128, 256);
    }
    if (form == 256) return launch(f8_product_kernel<256, 256, 2, 2, false>, 256, 256, 256);
    if (form == 192) return launch(f8_product_kernel<256, 192, 2, 2, false>, 256, 192, 256);
    return launch(f8_product_kernel<128, 128, 2, 2, false>, 128, 128, 256);
  });
}
