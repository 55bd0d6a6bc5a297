// wgrad_kernels.hip -- the gradients of a linear layer's weight and bias from the 8-bit checkpoint of its input:
//
//   dW[n][k] = sum over m of dY[m][n] x^[m][k],   db[n] = sum over m of dY[m][n],   x^ = code * 2^e
//
// x^ is one bf16 exactly (seven bits and a power of two), so a bf16 dY takes one matrix instruction per product and nothing is
// rounded before the fp32 sums.  An fp32 dY is cut into three bf16 of eight bits each, exactly: three matrix instructions of the
// 16-bit rate instead of one of the fp32 rate, which is a sixteenth of it.  An fp16 dY meets x^ as fp16, which is exact where
// the checkpoint was made from fp16.
//
// Both operands run along m, memory's slow direction, and a matrix instruction wants eight consecutive m of one row or column
// in a lane.  dY goes to LDS as it lies in memory and the codes as the 16-bit values that they stand for, and both are read
// by the transposing LDS reads of this chip.  (The first form turned them round in registers, in pieces of 2 x 8 values loaded
// two at a time: 16384 x 4096 x 1024 bf16 2084 us.)
//
// What bounds it: the matrix instructions, at the clock that they leave.  16384 x 4096 x 1024 bf16: 136 us and 12 for the sum
// of four splits, 930 TFLOP/s in all, where torch's product of the same bf16 matrices takes 180-195 us; the matrix units are
// busy 54 % of the time that a compute unit is, at 2.05 of 2.4 GHz.  The rest is issue: 100 vector instructions and 56 LDS
// instructions to 32 matrix instructions in a wavefront's stage.  fp32 of that size 390 us (353 TFLOP/s; torch's fp32
// product 950).  8192 x 8192 x 2048 bf16 262 us, 1050 TFLOP/s (torch 248).
//
// Measured and not kept: four wavefronts to a 256 x 256 tile (4096^3 fp16 163 : 149 us; a wavefront alone on its SIMD issues
// one instruction in four cycles, and a stage has 400 of them), an order of instructions given to the compiler group by group
// (four patterns, +-3 %), db as a product with ones (its sums did not fit the registers beside the tile: 268 us, half of it
// moves between register files), the two wavefronts of a SIMD held half a step apart by barriers (4096^3 bf16 155 : 159-168).
#include <hip/hip_runtime.h>
#include "../../include/cswap_hip.h"
#include "../../include/cswap_test_hooks.h"
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
};
template <> struct Feed<F32> {
  typedef BF16 type;
  static constexpr int parts = 3;
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

// eight m of one column for each lane, from two transposing reads of four
__device__ inline uint4 read_turned(const uint16_t* at, int four_rows)
{
  const s4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)(at));
  const s4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)(at + four_rows));
  const uint2 x = __builtin_bit_cast(uint2, lo), y = __builtin_bit_cast(uint2, hi);
  return make_uint4(x.x, x.y, y.x, y.y);
}

// A workgroup of 2 x WK wavefronts makes a TN x TK tile of dW from one split of the rows, BK rows (a stage) at a time.  A
// product of 32 x 32 x 16 takes 0.75 fragments from LDS in a tile of 256 x 256, 1 in one of 128 x 256, 1.25 in a narrow one of
// 64 x 256 and 1.5 in one of 128 x 128, and the small ones read either operand twice as often from the caches; of the large and
// middle ones one fits a compute unit (128 KB of LDS for two stages), of the others two, and more of them there are where dW is
// small.
//
// The tile of a stage lies in LDS as it does in memory, m by m, in chunks of 16 bytes whose order within a row depends on m: the
// transposing reads take four rows at once, which have to lie in different banks.  a_at and b_at are the places of value
// (m, column) of either operand, in 16-bit units.
template <typename T, int TN, int TK, int BK> struct GradTile {
  static constexpr int P = Feed<T>::parts;
  static constexpr int kAPlane = BK * TN, kStage = P * kAPlane + BK * TK;
  static __device__ inline int a_at(int m, int col)
  {
    // in a tile of 64 columns two rows take all banks: of four, two differ in the order
    return m * TN + 8 * ((col >> 3) ^ (TN == 64 ? (m & 2) << 1 : (m & 3) << 2)) + (col & 7);
  }
  static __device__ inline int b_at(int m, int col)
  {
    // pieces of 16 codes leave a lane as two chunks: those of all pieces first, then those of the others, so that neighbouring
    // lanes write neighbouring chunks
    const int piece = col >> 4, h = (col >> 3) & 1;
    return P * kAPlane + m * TK + 8 * (h * (TK / 16) + (piece ^ (2 * (m & 3)) ^ (TK == 256 ? 8 * h : 0))) + (col & 7);
  }
};

// Which tile and split a workgroup has.  Workgroups go to the eight XCDs in turn, each of which has a cache of its own: an XCD gets
// neighbouring tiles of one split, up to 16 along k (whose operand is the smaller one) before the next row of tiles.
struct TilePlace {
  uint32_t tn, tk, split;
};
__device__ inline TilePlace tile_place(uint32_t id, uint32_t count, const GradShape& s)
{
  const uint32_t each = count / 8, more = count % 8, xcd = id % 8;
  uint32_t at = xcd * each + min(xcd, more) + id / 8;
  const uint32_t tiles = s.tiles_n * s.tiles_k, split = at / tiles;
  at -= split * tiles;
  const uint32_t column = at / (16 * s.tiles_n), width = min(16u, s.tiles_k - 16 * column);
  at -= column * 16 * s.tiles_n;
  return {at / width, 16 * column + at % width, split};
}

// The same address in all lanes, for the compiler: loads then take it from scalar registers and 32-bit offsets from the lanes.
typedef const __attribute__((address_space(1))) char* global_bytes;
typedef const __attribute__((address_space(1))) u4_any* global_u4;
typedef const __attribute__((address_space(1))) uint8_t* global_u1;
__device__ inline global_bytes uniform(const char* p)
{
  const uint64_t v = reinterpret_cast<uint64_t>(p);
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)v), hi = __builtin_amdgcn_readfirstlane((uint32_t)(v >> 32));
  return (global_bytes)((uint64_t)hi << 32 | lo);
}

__device__ char spare[1024 + 16];  // 256 columns of fp32, and 16 bytes from the last of them on

template <typename T, int TN, int TK, int BK, int WK>
__global__ __launch_bounds__(128 * WK, TN * TK == 128 * 128 && WK == 4 ? 4 : 2) void weight_grad_kernel(
    const typename T::value* __restrict__ dy, const int8_t* __restrict__ codes, const uint8_t* __restrict__ scales, GradShape s,
    void* __restrict__ dw, void* __restrict__ db, int out_dtype)
{
  typedef GradTile<T, TN, TK, BK> Tile;
  typedef typename Feed<T>::type M;
  typedef typename T::value V;
  constexpr int P = Feed<T>::parts, W = T::bytes / 2;               // 16-byte words of a chunk of dY
  constexpr int NT = 128 * WK, FN = TN / 64, FK = TK / (32 * WK);  // threads; 32 x 32 pieces of a wavefront's part
  constexpr int kSteps = BK / 16;                                   // matrix instructions' depth
  constexpr int kAChunks = TN / 8, kARows = NT / kAChunks, kALoads = BK / kARows;
  constexpr int kBPieces = TK / 16, kBRows = NT / kBPieces, kBLoads = BK / kBRows;
  __shared__ __attribute__((aligned(16))) uint16_t lds[2][Tile::kStage];

  const TilePlace at = tile_place(blockIdx.x, gridDim.x, s);
  const uint32_t tk = at.tk, tn = at.tn, split = at.split;
  const uint32_t n0 = tn * TN, k0 = tk * TK;
  const uint32_t from = split * s.step_rows, to = min(s.rows, from + s.step_rows);
  const uint32_t stages = (to - from + BK - 1) / BK;
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;

  // A stage is plain if all of its loads are in the tensors: columns behind a row's last one read what lies there, which goes
  // into columns of the product that nobody stores.  Rows that are not there have to be zeros in both operands; the stages from
  // the first one that is not plain on (the last rows of the tensors) are loaded chunk by chunk as far as they are there.
  const size_t dy_end = (size_t)(s.rows - 1) * s.dy_stride + s.n;
  uint32_t plain = stages;
  while (plain > 0) {
    const uint32_t end = from + plain * BK;
    if (end <= to && (size_t)(end - 1) * s.dy_stride + n0 + TN <= dy_end &&
        (size_t)(end - 1) * s.code_pitch + k0 + TK <= (size_t)s.rows * s.code_pitch)
      break;
    --plain;
  }
  // The loop asks for a plain stage in every turn, the last one again where there is no other; without any it reads
  // a spare array, and what it reads is not used.
  const size_t dy_stride = plain ? s.dy_stride : 0, code_pitch = plain ? s.code_pitch : 0, scale_pitch = plain ? s.scale_pitch : 0;
  const char* const dy_from = plain ? reinterpret_cast<const char*>(dy + (size_t)from * s.dy_stride + n0) : spare;
  const char* const codes_from = plain ? reinterpret_cast<const char*>(codes) + (size_t)from * s.code_pitch + k0 : spare;
  const char* const scales_from = plain ? reinterpret_cast<const char*>(scales) + (size_t)from * s.scale_pitch + k0 / kGroup : spare;

  // staging: this thread's column chunk and first row of either operand
  const int a_chunk = tid % kAChunks, a_row = tid / kAChunks, b_piece = tid % kBPieces, b_row = tid / kBPieces;
  const uint32_t a_off = ((uint32_t)a_row * (uint32_t)dy_stride + 8 * a_chunk) * (uint32_t)sizeof(V);
  const uint32_t b_off = (uint32_t)b_row * (uint32_t)code_pitch + 16 * b_piece;
  const uint32_t c_off = (uint32_t)b_row * (uint32_t)scale_pitch + b_piece / 2;
  u4_any a_raw[kALoads][W], b_raw[kBLoads];
  uint32_t b_scale[kBLoads];
  auto load_a = [&](uint32_t st, int i) {
    const global_bytes base = uniform(dy_from + (size_t)(st * BK + i * kARows) * dy_stride * sizeof(V));
#pragma unroll
    for (int h = 0; h < W; ++h) a_raw[i][h] = *(global_u4)(base + a_off + 16 * h);
  };
  auto load_b = [&](uint32_t st, int i) {
    b_raw[i] = *(global_u4)(uniform(codes_from + (size_t)(st * BK + i * kBRows) * code_pitch) + b_off);
    b_scale[i] = *(global_u1)(uniform(scales_from + (size_t)(st * BK + i * kBRows) * scale_pitch) + c_off);
  };
  auto store_a = [&](uint16_t* buf, int i) {
    uint16_t* at = buf + Tile::a_at(a_row + i * kARows, 8 * a_chunk);
    if constexpr (P == 3) {
      float v[8];
      uint4 w[3];
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = __uint_as_float(a_raw[i][0][e]), v[4 + e] = __uint_as_float(a_raw[i][1][e]);
      split3(v, w);
#pragma unroll
      for (int p = 0; p < 3; ++p) *reinterpret_cast<uint4*>(at + p * Tile::kAPlane) = w[p];
    } else {
      *reinterpret_cast<uint4*>(at) = make_uint4(a_raw[i][0][0], a_raw[i][0][1], a_raw[i][0][2], a_raw[i][0][3]);
    }
  };
  auto store_b = [&](uint16_t* buf, int i) {
    const float unit = unit_of(b_scale[i]);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float v[8];
      decode_chunk(make_uint2(b_raw[i][2 * h], b_raw[i][2 * h + 1]), unit, v);
      *reinterpret_cast<uint4*>(buf + Tile::b_at(b_row + i * kBRows, 16 * b_piece + 8 * h)) =
          make_uint4(to_pair<M>(v[0], v[1]), to_pair<M>(v[2], v[3]), to_pair<M>(v[4], v[5]), to_pair<M>(v[6], v[7]));
    }
  };

  // db: the columns of dY, each stage's added up by one of the workgroups that have them
  float b_sum[8] = {};
  auto add_columns = [&] {
#pragma unroll
    for (int i = 0; i < kALoads; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e)
        b_sum[e] += T::bytes == 4 ? __uint_as_float(a_raw[i][(e / 4) % W][e % 4])
                                  : to_float<T>((V)(uint16_t)(a_raw[i][0][e / 2] >> (16 * (e & 1))));
  };

  // A stage that is not plain: every chunk that is there, and zeros.
  auto load_guarded = [&](uint32_t m0) {
    const uint32_t a_col = n0 + 8 * a_chunk, b_col = k0 + 16 * b_piece;
    const int valid = a_col + 8 <= s.n ? 8 : a_col < s.n ? (int)(s.n - a_col) : 0;
#pragma unroll
    for (int i = 0; i < kALoads; ++i) {
      const uint32_t m = m0 + a_row + i * kARows;
      load_raw<T>(dy + (size_t)m * s.dy_stride + a_col, m < to ? valid : 0, a_raw[i]);
    }
#pragma unroll
    for (int i = 0; i < kBLoads; ++i) {
      const uint32_t m = m0 + b_row + i * kBRows;
      b_raw[i] = (u4_any){0, 0, 0, 0}, b_scale[i] = 1;
      if (m < to && b_col < s.code_pitch) {
        b_raw[i] = *reinterpret_cast<const u4_any*>(codes + (size_t)m * s.code_pitch + b_col);
        b_scale[i] = scales[(size_t)m * s.scale_pitch + b_col / kGroup];
      }
    }
  };

  // reading: a lane supplies the address of four values of row 8 (lane / 32) + (lane % 16) / 4 and gets column lane % 32
  const int m_lane = 8 * (lane >> 5) + ((lane & 15) >> 2), c_lane = 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
  int a_at[FN], b_at[FK];
#pragma unroll
  for (int i = 0; i < FN; ++i) a_at[i] = Tile::a_at(m_lane, ((wave / WK) * FN + i) * 32 + c_lane);
#pragma unroll
  for (int j = 0; j < FK; ++j) b_at[j] = Tile::b_at(m_lane, ((wave % WK) * FK + j) * 32 + c_lane);

  f16v acc[FN][FK] = {};
  static_assert(kSteps % 2 == 0, "a stage begins with the first of either pair of fragments");
  uint4 a[2][FN], b[2][FK];
  auto read_a = [&](const uint16_t* buf, int c, int p, uint4* to_a) {
#pragma unroll
    for (int i = 0; i < FN; ++i) to_a[i] = read_turned(buf + p * Tile::kAPlane + a_at[i] + c * 16 * TN, 4 * TN);
  };
  auto read_b = [&](const uint16_t* buf, int c, uint4* to_b) {
#pragma unroll
    for (int j = 0; j < FK; ++j) to_b[j] = read_turned(buf + b_at[j] + c * 16 * TK, 4 * TK);
  };

  auto load = [&](uint32_t st) {
#pragma unroll
    for (int i = 0; i < kALoads; ++i) load_a(st, i);
#pragma unroll
    for (int i = 0; i < kBLoads; ++i) load_b(st, i);
  };
  // out_dtype: the results themselves leave; else (-1) what this split has of them
  auto my_turn = [&](uint32_t st) { return db && (out_dtype < 0 ? st % s.tiles_k == tk : tk == 0); };
  const uint32_t last = plain ? plain - 1 : 0;

  auto store = [&](uint16_t* buf) {
#pragma unroll
    for (int i = 0; i < kALoads; ++i) store_a(buf, i);
#pragma unroll
    for (int i = 0; i < kBLoads; ++i) store_b(buf, i);
  };
  if (stages) {
    if (plain) load(0);
    else load_guarded(from);
    if (my_turn(0)) add_columns();
    store(lds[0]);
  }
  load(min(1u, last));
  __syncthreads();
  read_b(lds[0], 0, b[0]);
  read_a(lds[0], 0, P - 1, a[0]);
  // One stage's products a turn.  Meanwhile the next stage goes from registers to LDS and the one after that is asked for; the
  // fragments of a step are read while the step before multiplies, those of a stage's first step, behind the barrier, beside
  // the last products of the stage before.
  for (uint32_t st = 0; st < stages; ++st) {
    const uint16_t* buf = lds[st & 1];
    uint16_t* next = lds[(st + 1) & 1];
    const uint32_t after = min(st + 2, last);
    if (st + 1 < plain && my_turn(st + 1)) add_columns();
    constexpr int kParts = kSteps * P;
#pragma unroll
    for (int part = 0; part < kParts; ++part) {
      const int c = part / P, q = part % P, at = part & 1;
#pragma unroll
      for (int i = 0; i < kALoads; ++i)
        if (i * kParts / kALoads == part) {
          store_a(next, i);
          load_a(after, i);
        }
#pragma unroll
      for (int i = 0; i < kBLoads; ++i)
        if (i * kParts / kBLoads == part) {
          store_b(next, i);
          load_b(after, i);
        }
      if (q + 1 < P) {
        read_a(buf, c, P - 2 - q, a[at ^ 1]);
      } else if (c + 1 < kSteps) {
        read_b(buf, c + 1, b[(c + 1) & 1]);
        read_a(buf, c + 1, P - 1, a[at ^ 1]);
      } else {
        if (st + 1 < stages && st + 1 >= plain) {
          load_guarded(from + (st + 1) * BK);
          if (my_turn(st + 1)) add_columns();
          __syncthreads();  // the turn has left something there
          store(next);
        }
        __syncthreads();
        read_b(next, 0, b[0]);
        read_a(next, 0, P - 1, a[0]);
      }
#pragma unroll
      for (int i = 0; i < FN; ++i)
#pragma unroll
        for (int j = 0; j < FK; ++j) acc[i][j] = mma(M(), a[at][i], b[c & 1][j], acc[i][j]);
    }
  }

  auto leave = [&](auto t, void* to) {
    typedef decltype(t) O;
    typename O::value* out = static_cast<typename O::value*>(to);
#pragma unroll
    for (int i = 0; i < FN; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const uint32_t n = n0 + ((wave / WK) * FN + i) * 32 + 8 * (r / 4) + 4 * (lane >> 5) + r % 4;
        if (n >= s.n) continue;
#pragma unroll
        for (int j = 0; j < FK; ++j) {
          const uint32_t k = k0 + ((wave % WK) * FK + j) * 32 + (lane & 31);
          if (k < s.k) out[(size_t)n * s.k + k] = from_float<O>(acc[i][j][r]);
        }
      }
  };
  if (out_dtype < 0)
    leave(F32(), static_cast<float*>(dw) + (size_t)split * s.n * s.k);
  else if (out_dtype == CSWAP_DT_F32)
    leave(F32(), dw);
  else if (out_dtype == CSWAP_DT_BF16)
    leave(BF16(), dw);
  else
    leave(F16(), dw);
  if (db && (out_dtype < 0 || tk == 0)) {
    float* sums = reinterpret_cast<float*>(lds[0]);                 // [kARows][TN]
    static_assert(sizeof(lds) >= sizeof(float) * kARows * TN, "room for the columns' sums");
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 8; ++e) sums[a_row * TN + 8 * a_chunk + e] = b_sum[e];
    __syncthreads();
    if (tid < TN && n0 + tid < s.n) {
      float v = 0.0f;
      for (int r = 0; r < kARows; ++r) v += sums[r * TN + tid];
      const uint32_t n = n0 + tid;
      if (out_dtype < 0)
        static_cast<float*>(db)[(size_t)(split * s.tiles_k + tk) * s.n + n] = v;
      else if (out_dtype == CSWAP_DT_F32)
        static_cast<float*>(db)[n] = v;
      else if (out_dtype == CSWAP_DT_BF16)
        static_cast<uint16_t*>(db)[n] = from_float<BF16>(v);
      else
        static_cast<uint16_t*>(db)[n] = from_float<F16>(v);
    }
  }
}

// out[i] = sum over `parts` of part[.][i], rounded once: dW from its splits, and behind it db.  Of few splits a thread sums four
// values; of many, which a small dW has, eight lanes sum one.
struct GradSums {
  const float *dw, *db;
  size_t dw_count, dw_groups;  // workgroups that sum dW
  uint32_t dw_parts, db_parts, n;
};
constexpr uint32_t kFewSplits = 16;

// 32 values a workgroup, eight lanes to a value
template <typename O> __device__ inline void sum_by_eight(const float* part, uint32_t parts, size_t count, size_t group,
                                                          typename O::value* out)
{
  __shared__ float sum[8][32];
  const uint32_t lane = threadIdx.x & 31, seg = threadIdx.x >> 5;
  const size_t i = group * 32 + lane;
  float v = 0.0f;
  if (i < count) {
#pragma unroll 8
    for (uint32_t p = seg; p < parts; p += 8) v += part[(size_t)p * count + i];
  }
  sum[seg][lane] = v;
  __syncthreads();
  if (seg == 0 && i < count) {
#pragma unroll
    for (int k = 1; k < 8; ++k) v += sum[k][lane];
    out[i] = from_float<O>(v);
  }
}

template <typename O> __global__ __launch_bounds__(256) void weight_grad_reduce_kernel(GradSums s, typename O::value* __restrict__ dw,
                                                                                       typename O::value* __restrict__ db)
{
  if (blockIdx.x >= s.dw_groups) {
    sum_by_eight<O>(s.db, s.db_parts, s.n, blockIdx.x - s.dw_groups, db);
  } else if (s.dw_parts > kFewSplits) {
    sum_by_eight<O>(s.dw, s.dw_parts, s.dw_count, blockIdx.x, dw);
  } else {
    const size_t at = ((size_t)blockIdx.x * 256 + threadIdx.x) * 4;
    if (at + 4 <= s.dw_count) {
      float v[4] = {};
#pragma unroll 4
      for (uint32_t p = 0; p < s.dw_parts; ++p) {
        const u4_any w = *reinterpret_cast<const u4_any*>(s.dw + (size_t)p * s.dw_count + at);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] += __uint_as_float(w[i]);
      }
      if constexpr (O::bytes == 4)
        *reinterpret_cast<u4_any*>(dw + at) =
            (u4_any){__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])};
      else
        *reinterpret_cast<u2_any*>(dw + at) = (u2_any){to_pair<O>(v[0], v[1]), to_pair<O>(v[2], v[3])};
    } else {
      for (size_t i = at; i < s.dw_count; ++i) {
        float v = 0.0f;
        for (uint32_t p = 0; p < s.dw_parts; ++p) v += s.dw[(size_t)p * s.dw_count + i];
        dw[i] = from_float<O>(v);
      }
    }
  }
}

// ---------------------------------------------------------------- launches
constexpr size_t kMaxGradSide = (size_t)1 << 20;    // features on either side
constexpr size_t kMaxGradStride = (size_t)1 << 24;  // a workgroup's offsets within 32 rows are 32 bits

// Tiles of dW: n x k features.  The narrow ones are for an fp32 dY of few columns, whose three products of those that are not there
// cost the most: in us, narrow : others, 32768 x 8 x 2048 37 : 55, 32768 x 64 x 4096 72 : 102, 8192 x 64 x 768 19.1 : 20.3, but
// 32768 x 320 x 256 37 : 33; bf16 32768 x 64 x 4096 50.5 : 51.9, 8192 x 64 x 2048 23.8 : 18.6.
enum GradForm { kSmallTile, kMiddleTile, kLargeTile, kNarrowTile, kGradForms };
constexpr size_t kTileN[kGradForms] = {128, 128, 256, 64}, kTileK[kGradForms] = {128, 256, 256, 256};

static bool narrow_fits(int dtype, size_t n, size_t k) { return dtype == CSWAP_DT_F32 && n <= 64 && k > 128; }

struct GradPlan {
  int form;
  unsigned tiles_n, tiles_k, splits;
  uint32_t step_rows;
};

// Tiles and splits with the least estimated time.  Measured on 256 compute units, in us: a workgroup takes `stage` for 64 rows, a
// compute unit with two workgroups of the small or narrow tiles `pair` for 64 rows of both; `fixed` is the rest of a launch; splits cost
// the sums' launch (5) and their bytes there and back at 5.5 TB/s.  What it decides between, small : middle : large tiles in us,
// each with its best splits.  bf16: 512 x 2048 x 2048 14 : 18 : 33, 8192 x 768 x 768 28.5 : 28.6 : 36, 8192 x 1024 x 1024 39.7 : 37.6 :
// 43, 8192 x 2048 x 2048 102 : 91 : 86, 32768 x 4096 x 1024 371 : 328 : 273, 2048 x 4096 x 4096 92 : 84 : 71; fp32: 8192 x 768 x 768
// 52 : 42 : 50, 2048 x 2048 x 2048 68 : 61 : 70, 8192 x 4096 x 1024 222 : 184 : 180, 32768 x 768 x 4096 677 : 561 : 514.  Small tiles with
// one : two workgroups a compute unit, bf16: 2048 x 2048 x 2048 (not split : in two) 36.6 : 40.9, 32768 x 768 x 768 77 : 66.
static double grad_estimate(int form, bool f32, size_t tiles, size_t splits, size_t step, size_t n, size_t k)
{
  constexpr double kFixed[kGradForms] = {8.0, 9.5, 11.0, 8.0};
  constexpr double kStage[2][kGradForms] = {{0.77, 1.05, 1.65}, {1.9, 2.35, 4.4, 1.75}};
  constexpr double kPair[2][kGradForms] = {{1.2, 1.05, 1.65}, {3.2, 2.35, 4.4, 3.0}};
  const bool two = form == kSmallTile || form == kNarrowTile;
  const size_t groups = tiles * splits, at_once = two ? 512 : 256, rest = groups % at_once;
  const double units = (double)step / 64, stage = kStage[f32][form], both = kPair[f32][form];
  double t = kFixed[form] + (double)(groups / at_once) * units * both;
  if (rest) t += units * (rest > 256 ? both : stage);
  if (splits > 1) t += 5.0 + (double)(splits * n * k) * 8.0 / 5.5e6;
  return t;
}

static GradPlan grad_plan(int dtype, size_t rows, size_t n, size_t k)
{
  GradPlan best = {};
  double least = 0.0;
  for (int form = 0; form < kGradForms; ++form) {
    if (form == kNarrowTile && !narrow_fits(dtype, n, k)) continue;
    const size_t tiles_n = (n + kTileN[form] - 1) / kTileN[form], tiles_k = (k + kTileK[form] - 1) / kTileK[form];
    const size_t tiles = tiles_n * tiles_k;
    // every number of splits up to 16, then an eighth more each time: the estimate is not finer, and a call takes this long
    for (size_t want = 1; want == 1 || (want <= 512 && want * tiles <= 1024 && want * 64 <= rows); want += want < 16 ? 1 : want / 8) {
      const size_t step = rows ? ((rows + want - 1) / want + 63) / 64 * 64 : 64, splits = rows ? (rows + step - 1) / step : 1;
      const double t = grad_estimate(form, dtype == CSWAP_DT_F32, tiles, splits, step, n, k);
      if (best.splits == 0 || t < least) {
        least = t;
        best = {form, (unsigned)tiles_n, (unsigned)tiles_k, (unsigned)splits, (uint32_t)step};
      }
    }
  }
  return best;
}

static size_t bias_parts(const GradPlan& p) { return (size_t)p.splits * p.tiles_k; }

// Sums of the splits; none where the tiles leave as results.
static size_t grad_room(const GradPlan& p, size_t n, size_t k)
{
  return p.splits == 1 ? 0 : ((size_t)p.splits * n * k + bias_parts(p) * n) * sizeof(float);
}

}  // namespace q8
}  // namespace cswap

using namespace cswap;
using namespace cswap::q8;

static bool grad_sizes(size_t rows, size_t n, size_t k)
{
  return n && k && n <= kMaxGradSide && k <= kMaxGradSide && rows < ((size_t)1 << 31);
}

extern "C" int cswap_test_weight_grad_plan(int dtype, size_t rows, size_t n, size_t k)
{
  const GradPlan p = grad_plan(dtype, rows, n, k);
  return (int)p.splits + 1000 * p.form;
}

extern "C" size_t cswap_q8_weight_grad_workspace_bytes(int dtype, size_t rows, size_t n, size_t k)
{
  if (!dtype_known(dtype) || !grad_sizes(rows, n, k)) return 0;
  return grad_room(grad_plan(dtype, rows, n, k), n, k);
}

extern "C" int cswap_q8_weight_grad(const void* d_dy, int dtype, size_t rows, size_t n, ptrdiff_t dy_stride, const int8_t* d_codes,
                                    const uint8_t* d_scales, size_t k, void* d_dw, void* d_db, int out_dtype, void* d_ws,
                                    size_t ws_bytes, cswap_stream_t stream)
{
  ptrdiff_t unused = 0;
  if (int e = check_rows(rows, n, &dy_stride)) return e;
  if (int e = check_rows(rows, k, &unused)) return e;
  if (!dtype_known(dtype) || !dtype_known(out_dtype)) return CSWAP_E_ARG;
  if (!grad_sizes(rows, n, k) || (size_t)dy_stride > kMaxGradStride) return CSWAP_E_UNSUPPORTED;
  if (!value_ptr(d_dw, out_dtype) || (d_db && !value_ptr(d_db, out_dtype))) return CSWAP_E_ARG;
  if (rows && (!value_ptr(d_dy, dtype) || !checkpoint_ptrs(d_codes, d_scales))) return CSWAP_E_ARG;
  const GradPlan p = grad_plan(dtype, rows, n, k);
  const size_t room = grad_room(p, n, k);
  if (room && !value_ptr(d_ws, CSWAP_DT_F32)) return CSWAP_E_ARG;
  if (ws_bytes < room) return CSWAP_E_NOMEM;
  const GradShape s = {(uint32_t)rows, (uint32_t)n, (uint32_t)k, (uint32_t)groups_of(k), p.step_rows, p.tiles_n, p.tiles_k,
                       (size_t)dy_stride, pitch_of(k)};
  const bool direct = p.splits == 1;
  float* part = static_cast<float*>(d_ws);
  float* part_b = part + (size_t)p.splits * n * k;
  hipStream_t st = static_cast<hipStream_t>(stream);
  const auto launch = [&](auto t) {
    typedef decltype(t) T;
    // stages of 32 rows in fp32, whose three planes need the room; a small tile's codes are then too few for eight wavefronts
    constexpr int BK = T::bytes == 4 ? 32 : 64, kSmall = T::bytes == 4 ? 2 : 4;
    auto kernel = p.form == kLargeTile    ? weight_grad_kernel<T, 256, 256, BK, 4>
                  : p.form == kMiddleTile ? weight_grad_kernel<T, 128, 256, BK, 4>
                                          : weight_grad_kernel<T, 128, 128, BK, kSmall>;
    unsigned threads = p.form == kSmallTile ? 128 * kSmall : 512;
    if constexpr (T::bytes == 4)
      if (p.form == kNarrowTile) kernel = weight_grad_kernel<T, 64, 256, BK, 2>, threads = 256;
    hipLaunchKernelGGL(kernel, dim3(p.tiles_n * p.tiles_k * p.splits), dim3(threads), 0, st,
                       static_cast<const typename T::value*>(d_dy), d_codes, d_scales, s, direct ? d_dw : part,
                       !d_db ? nullptr : direct ? d_db : part_b, direct ? out_dtype : -1);
    return check_launch();
  };
  if (int e = dtype == CSWAP_DT_F32 ? launch(F32()) : dtype == CSWAP_DT_BF16 ? launch(BF16()) : launch(F16())) return e;
  if (direct) return CSWAP_OK;
  const size_t dw_groups = p.splits > kFewSplits ? (n * k + 31) / 32 : (n * k + 1023) / 1024;
  const GradSums sums = {part, part_b, n * k, dw_groups, p.splits, (uint32_t)bias_parts(p), (uint32_t)n};
  const auto reduce = [&](auto t) {
    typedef decltype(t) O;
    hipLaunchKernelGGL(weight_grad_reduce_kernel<O>, dim3((unsigned)(dw_groups + (d_db ? (n + 31) / 32 : 0))), dim3(256), 0, st, sums,
                       static_cast<typename O::value*>(d_dw), static_cast<typename O::value*>(d_db));
    return check_launch();
  };
  return out_dtype == CSWAP_DT_F32 ? reduce(F32()) : out_dtype == CSWAP_DT_BF16 ? reduce(BF16()) : reduce(F16());
}
