// group_norm_kernels.hip -- group norm with an activation function for images that lie in memory channels last, forward and backward.
// A sample is a matrix of positions x channels, a group some neighbouring channels of all positions of a sample.
//
//   forward   mu, r = 1 / sqrt(var + eps) of a sample's group, h = (x - mu) r, z = h g + b, y = f(z)
//   backward  h as above from the 8-bit checkpoint of x (or from x), dz = dy f'(z), u = dz g,
//             dx = r (u - mean(u) - h mean(u h)), dg = sum over samples and positions of dz h, db = sum of dz
//
// Memory bounds both.  A group's sums take all positions of a sample, so either direction goes over its tensors twice: the first pass
// leaves sums of tiles of positions (so that there are workgroups enough where samples are few), the second joins a sample's tiles and
// writes; what it reads again comes from the memory-side cache.  Where a sample is a workgroup's work, both passes are one launch.
//
// Variances: a thread sums differences from the first value that it meets in each channel.  That value is one of those that it sums over, so what
// cancels is at most as many times the result as there are values (a few hundred roundings at the very worst, one or two as a rule);
// threads and tiles are joined by their means and squares about them.  All sums are fp32, in a fixed order: the same call gives the same bits.
//
// Launch by launch (traced, tensors that are in no cache): 128 x 64 x 64 images of 64 channels, fp32, GELU: sums and checkpoint 43 us, writing 50,
// backward 53 and 58: 4.0, 5.4, 3.2 and 5.2 TB/s of what each goes over; the four in a row 196 us, 910 MB at 4.6 TB/s (606 MB are needed
// once).  16 x 64 x 64 of 256, bf16, SiLU: 18, 16, 20 and 19 us, where SiLU's slope alone is 7 us of vector instructions in each backward
// stage.  A workgroup's sums through LDS take 3 us of each first stage, during which nothing is loaded.
// Measured and not kept: a tile's rows strewn over its sample (+5 to +10 %), the next rows asked for before these are worked on (+-3 %), 1024 to
// 4096 tiles instead of 512 (+-3 %, the second backward stage +20 % with the shares' sums), 8 rows of 16-bit values under way in the backward pass.
#include <hip/hip_runtime.h>
#include "../../include/cswap_hip.h"
#include "common.h"
#include "q8_act.h"
#include "q8_block.h"
#include "q8_params.h"

namespace cswap {
namespace q8 {

constexpr uint32_t kMaxChannels = 4096;
constexpr uint32_t kMaxGroups = 2048;
constexpr size_t kMaxSamples = (size_t)1 << 22;  // a launch has fewer than 2^32 threads
constexpr int NT = 512;  // threads of a workgroup: a chunk of every channel
// A workgroup's NT threads are `lanes` rows of `width` chunks; a tile is `tile_rows` positions of a sample.
struct GroupShape {
  uint32_t samples, positions, channels, groups, per_group;
  uint32_t width, lanes, tiles, tile_rows;
  uint32_t code_chunks;
  RowDivisor by_width, by_group;
  size_t x_stride, y_stride;
  float eps;
};

struct Pass {
  uint32_t sample, tile, rows;  // rows: of the tile
  uint32_t lane, chunk;         // of the thread; lane >= shape.lanes: none
  int valid;
  uint32_t count;   // rows of the thread
  size_t row;       // its first one in the tensor; of a thread without rows the tile's
  uint32_t column;  // its first channel; of a thread without channels 0
};

__device__ inline Pass pass_of(const GroupShape& s, uint32_t item)
{
  Pass p;
  p.sample = item / s.tiles, p.tile = item - p.sample * s.tiles;
  const uint32_t at = p.tile * s.tile_rows;
  p.rows = min(s.tile_rows, s.positions - at);
  p.lane = divide(threadIdx.x, s.by_width);
  p.chunk = threadIdx.x - p.lane * s.width;
  const bool here = p.lane < s.lanes;
  p.valid = here ? valid_at(p.chunk * kChunk, s.channels) : 0;
  p.count = here && p.lane < p.rows ? (p.rows - p.lane + s.lanes - 1) / s.lanes : 0;
  p.row = (size_t)p.sample * s.positions + at + (p.count ? p.lane : 0);
  p.column = p.valid ? p.chunk * kChunk : 0;
  return p;
}

// LDS of a workgroup: a chunk of each thread; sums of channels where several threads have one; sums of groups, twice; gamma (backward).
struct GroupRoom {
  static __host__ __device__ size_t chunks() { return (size_t)NT * kChunk; }
  static __host__ __device__ size_t channels() { return (size_t)NT * kChunk / 2 + kChunk; }
  static size_t bytes(const GroupShape& s, bool gamma) { return (chunks() + channels() + 2 * (size_t)s.groups + (gamma ? s.channels : 0)) * sizeof(float); }
};

// v + v of lane ^ N of a wavefront
template <int N> __device__ inline float add_lane(float v)
{
  const int u = __builtin_bit_cast(int, v);
  if constexpr (N == 1) return v + __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(u, 0xb1, 0xf, 0xf, true));
  else if constexpr (N == 2) return v + __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(u, 0x4e, 0xf, 0xf, true));
  else if constexpr (N == 4) return v + __builtin_bit_cast(float, __builtin_amdgcn_ds_swizzle(u, 0x101f));
  else if constexpr (N == 8) return v + __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(u, 0x128, 0xf, 0xf, true));  // turned by 8 in 16
  else {
    const auto p = N == 16 ? __builtin_amdgcn_permlane16_swap((unsigned)u, (unsigned)u, false, false)
                           : __builtin_amdgcn_permlane32_swap((unsigned)u, (unsigned)u, false, false);
    return __uint_as_float(p[0]) + __uint_as_float(p[1]);
  }
}

// Sums over the threads that have a channel, for all channels: where they are.  Every thread runs this.  Where a wavefront's lanes are
// whole rows of a power of two of chunks they add up by exchanges first, which leaves a row for each wavefront.
__device__ inline const float* sum_channels(const float given[8], const GroupShape& s, float* room)
{
  float v[8];
#pragma unroll
  for (int i = 0; i < kChunk; ++i) v[i] = given[i];
  const bool whole = s.width <= 32 && (s.width & (s.width - 1)) == 0;
  if (whole) {
#pragma unroll
    for (int i = 0; i < kChunk; ++i) {
      v[i] = add_lane<32>(v[i]);
      if (s.width <= 16) v[i] = add_lane<16>(v[i]);
      if (s.width <= 8) v[i] = add_lane<8>(v[i]);
      if (s.width <= 4) v[i] = add_lane<4>(v[i]);
      if (s.width <= 2) v[i] = add_lane<2>(v[i]);
      if (s.width <= 1) v[i] = add_lane<1>(v[i]);
    }
  }
  __syncthreads();  // whoever reads the room has done so
  const uint32_t pitch = s.width * kChunk, rows = whole ? NT / 64 : s.lanes;
  if (!whole || (threadIdx.x & 63) < s.width) {
    float4* to = reinterpret_cast<float4*>(room + (whole ? (threadIdx.x >> 6) * pitch + (threadIdx.x & 63) * kChunk : threadIdx.x * kChunk));
    to[0] = make_float4(v[0], v[1], v[2], v[3]), to[1] = make_float4(v[4], v[5], v[6], v[7]);
  }
  __syncthreads();
  if (rows == 1) return room;
  float* sums = room + GroupRoom::chunks();
  for (uint32_t c = threadIdx.x; c < s.channels; c += NT) {
    float sum = 0.0f;
    uint32_t r = 0;
    for (; r + 4 <= rows; r += 4) {
      const float a = room[r * pitch + c], b = room[(r + 1) * pitch + c], d = room[(r + 2) * pitch + c], e = room[(r + 3) * pitch + c];
      sum += (a + b) + (d + e);
    }
    for (; r < rows; ++r) sum += room[r * pitch + c];
    sums[c] = sum;
  }
  __syncthreads();
  return sums;
}

__device__ inline float sum_of_eight(float x)
{
  x += __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, x), 0xb1, 0xf, 0xf, true));   // lane ^ 1
  x += __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, x), 0x4e, 0xf, 0xf, true));   // lane ^ 2
  x += __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, x), 0x141, 0xf, 0xf, true));  // 7 - lane
  return x;
}

// sum over a group's channels of term(c), eight lanes to a group; to(group, sum) in one of them.
template <typename Term, typename To> __device__ inline void sum_groups(const GroupShape& s, Term&& term, To&& to)
{
  for (uint32_t j = threadIdx.x; j < s.groups * 8; j += NT) {
    const uint32_t g = j / 8, first = g * s.per_group;
    float sum = 0.0f;
    for (uint32_t c = j % 8; c < s.per_group; c += 8) sum += term(first + c);
    sum = sum_of_eight(sum);
    if (j % 8 == 0) to(g, sum);
  }
}

// The groups of a thread's channels: the first one's, and how many channels are left in it.
struct GroupPlace {
  uint32_t group, left;
};
__device__ inline GroupPlace group_place(const GroupShape& s, const Pass& p)
{
  const uint32_t c = min(p.chunk * kChunk, s.channels - 1), g = divide(c, s.by_group);
  return {g, s.per_group - (c - g * s.per_group)};
}

// What a thread has of its channels' groups; of channels behind the last, what the last has.
__device__ inline void spread(const GroupShape& s, GroupPlace at, const float* by_group, float v[8])
{
#pragma unroll
  for (int i = 0; i < kChunk; ++i) {
    v[i] = by_group[at.group];
    if (--at.left == 0) at.group = min(at.group + 1, s.groups - 1), at.left = s.per_group;
  }
}

// take(number of a tile, its pair) over eight lanes' share of a group's tiles, eight loads under way.
template <typename Take> __device__ inline void for_tiles(const GroupShape& s, const float2* from, uint32_t lane, Take&& take)
{
  for (uint32_t t0 = lane; t0 < s.tiles; t0 += 64) {
    float2 v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = from[min(t0 + 8 * k, s.tiles - 1)];
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (t0 + 8 * k < s.tiles) take(t0 + 8 * k, v[k]);
  }
}

// Rows of a thread from number `from` on as they lie in memory, ROWS of them at once.  A kernel asks for its first ones before anything
// else, as what follows waits for memory, too.  WHOLE: channels are whole chunks.  Then every lane loads, the last row again where
// it has no more and the tile's first where it has none: a branch for each row and for each value of a last chunk makes three times the code
// (and takes as long, +-3 %).  Shapes that are not whole have one form for all activation functions.
template <typename T, bool WHOLE, int ROWS> struct RowBatch {
  u4_any raw[ROWS][T::bytes / 2];
  __device__ inline void load(const GroupShape& s, const Pass& p, const typename T::value* x, size_t stride, uint32_t from)
  {
    const uint32_t last = p.count ? p.count - 1 : 0;
#pragma unroll
    for (int k = 0; k < ROWS; ++k) {
      if (WHOLE) load_raw<T>(x + (p.row + min(from + k, last) * s.lanes) * stride + p.column, kChunk, raw[k]);
      else load_raw<T>(x + (p.row + (from + k) * s.lanes) * stride + p.column, from + k < p.count ? p.valid : 0, raw[k]);
    }
  }
  __device__ inline void value(int k, float v[8]) const { widen<T>(raw[k], v); }
};

// The same of x or its checkpoint.
template <typename T, bool WHOLE, bool HELD, int ROWS> struct HeldBatch : RowBatch<T, WHOLE, ROWS> {
  __device__ inline void load(const GroupShape& s, const Pass& p, const typename T::value* x, const uint2*, const uint8_t*, uint32_t from)
  {
    RowBatch<T, WHOLE, ROWS>::load(s, p, x, s.x_stride, from);
  }
  __device__ inline void minus(int k, const float mu[8], float v[8]) const
  {
    this->value(k, v);
#pragma unroll
    for (int i = 0; i < kChunk; ++i) v[i] -= mu[i];
  }
};
template <typename T, bool WHOLE, int ROWS> struct HeldBatch<T, WHOLE, true, ROWS> {
  uint2 q[ROWS];
  uint32_t scale[ROWS];
  __device__ inline void load(const GroupShape& s, const Pass& p, const typename T::value*, const uint2* codes, const uint8_t* scales, uint32_t from)
  {
    const uint32_t last = p.count ? p.count - 1 : 0;
#pragma unroll
    for (int k = 0; k < ROWS; ++k) {
      const size_t at = (p.row + min(from + k, last) * s.lanes) * s.code_chunks + p.column / kChunk;
      q[k] = codes[at], scale[k] = scales[at / kChunksPerGroup];
    }
  }
  // x - mu: a code's value is a product without rounding, so this rounds once
  __device__ inline void minus(int k, const float mu[8], float v[8]) const
  {
    const float unit = unit_of(scale[k]);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[i] = __builtin_fmaf(code_value(q[k].x, i), unit, -mu[i]);
      v[4 + i] = __builtin_fmaf(code_value(q[k].y, i), unit, -mu[4 + i]);
    }
  }
};

// An activation function that is known at the launch, for shapes that are rare.
struct AnyAct {
  int kind;
  template <typename T> __device__ inline float value(float x) const
  {
    return kind == CSWAP_ACT_GELU ? Gelu::value<T>(x) : kind == CSWAP_ACT_GELU_TANH ? GeluTanh::value<T>(x) : kind == CSWAP_ACT_SILU ? Silu::value<T>(x) : x;
  }
  template <typename T> __device__ inline float slope(float x) const
  {
    return kind == CSWAP_ACT_GELU ? Gelu::slope<T>(x) : kind == CSWAP_ACT_GELU_TANH ? GeluTanh::slope<T>(x) : kind == CSWAP_ACT_SILU ? Silu::slope<T>(x) : 1.0f;
  }
};
template <typename A> struct IsWhole {
  static constexpr bool value = true;
};
template <> struct IsWhole<AnyAct> {
  static constexpr bool value = false;
};

template <typename A> struct FirstStage {
  typedef Identity type;
};
template <> struct FirstStage<AnyAct> {
  typedef AnyAct type;
};

enum Stage { kSums = 0, kWrite = 1, kBoth = 2 };

// part[sample][group][tile]: mean and sum of squares about it of a group's values in a tile.
template <typename T, typename A, bool HOLD, int STAGE>
__global__ __launch_bounds__(NT) void group_norm_forward_kernel(const typename T::value* __restrict__ x, GroupShape s, A act, Params gamma, Params beta,
                                                                typename T::value* __restrict__ y, float* __restrict__ mean,
                                                                float* __restrict__ rstd, uint2* __restrict__ codes,
                                                                uint8_t* __restrict__ scales, float2* __restrict__ part)
{
  extern __shared__ float room[];
  float* const group_mean = room + GroupRoom::chunks() + GroupRoom::channels();
  float* const group_rstd = group_mean + s.groups;
  const Pass p = pass_of(s, STAGE == kWrite ? gridDim.x - 1 - blockIdx.x : blockIdx.x);  // what was read last is read first
  const GroupPlace place = group_place(s, p);
  constexpr int kRows = T::bytes == 4 ? 4 : 8;  // 128 bytes of a lane under way
  constexpr bool kWhole = IsWhole<A>::value;
  RowBatch<T, kWhole, kRows> batch;
  batch.load(s, p, x, s.x_stride, 0);
  auto each_row = [&](auto&& each) {
    for (uint32_t from = 0;;) {
#pragma unroll
      for (int k = 0; k < kRows; ++k) {
        float v[8];
        batch.value(k, v);
        if (from + k < p.count) each(p.row + (from + k) * s.lanes, v);
      }
      from += kRows;
      if (from >= p.count) break;
      batch.load(s, p, x, s.x_stride, from);
    }
  };
  float k[8], b[8];
  if (STAGE != kSums) {
    load_params(gamma, p.chunk * kChunk, p.valid, 1.0f, k);
    load_params(beta, p.chunk * kChunk, p.valid, 0.0f, b);
  }
  if (STAGE != kWrite) {
    float first[8], sum[8], squares[8];
#pragma unroll
    for (int i = 0; i < kChunk; ++i) sum[i] = squares[i] = 0.0f;
    widen<T>(batch.raw[0], first);
    each_row([&](size_t row, float v[8]) {
      if (HOLD) {  // the lanes of a quad have the same rows
        if (kWhole && !p.valid) {
#pragma unroll
          for (int i = 0; i < kChunk; ++i) v[i] = 0.0f;
        }
        uint32_t scale;
        const uint2 q = encode_chunk(v, quad_max_bits(v), &scale);
        const size_t at = row * s.code_chunks + p.chunk;
        codes[at] = q;
        if ((p.chunk & (kChunksPerGroup - 1)) == 0) scales[at / kChunksPerGroup] = (uint8_t)scale;
      }
#pragma unroll
      for (int i = 0; i < kChunk; ++i) {
        const float d = v[i] - first[i];
        sum[i] += d;
        squares[i] = __builtin_fmaf(d, d, squares[i]);
      }
    });
    if (STAGE == kBoth) batch.load(s, p, x, s.x_stride, 0);
    const float count = (float)p.count, inverse = p.count ? 1.0f / count : 0.0f;
#pragma unroll
    for (int i = 0; i < kChunk; ++i) {
      const float m = sum[i] * inverse;
      squares[i] = larger(__builtin_fmaf(-m, sum[i], squares[i]), 0.0f);
      first[i] += m;  // the thread's mean
      sum[i] = first[i] * count;
    }
    const float* sums = sum_channels(sum, s, room);
    const float inverse_all = 1.0f / ((float)p.rows * (float)s.per_group);
    sum_groups(s, [&](uint32_t c) { return sums[c]; }, [&](uint32_t g, float v) { group_mean[g] = v * inverse_all; });
    __syncthreads();
    spread(s, place, group_mean, sum);
#pragma unroll
    for (int i = 0; i < kChunk; ++i) {
      const float d = first[i] - sum[i];
      squares[i] = p.count ? __builtin_fmaf(count * d, d, squares[i]) : 0.0f;
    }
    sums = sum_channels(squares, s, room);
    sum_groups(s, [&](uint32_t c) { return sums[c]; }, [&](uint32_t g, float v) {
      if (STAGE == kSums) part[((size_t)p.sample * s.groups + g) * s.tiles + p.tile] = make_float2(group_mean[g], v);
      else group_rstd[g] = 1.0f / __builtin_sqrtf(v * inverse_all + s.eps);
    });
    if (STAGE == kSums) return;
  } else {
    // join the tiles: their means about the first one's
    for (uint32_t j = threadIdx.x; j < s.groups * 8; j += NT) {
      const uint32_t g = j / 8;
      const float2* from = part + ((size_t)p.sample * s.groups + g) * s.tiles;
      const float shift = from[0].x;
      float a = 0.0f, b = 0.0f, m2 = 0.0f;
      for_tiles(s, from, j % 8, [&](uint32_t t, float2 v) {
        const float rows = (float)min(s.tile_rows, s.positions - t * s.tile_rows), d = v.x - shift;
        a = __builtin_fmaf(rows, d, a), b = __builtin_fmaf(rows * d, d, b), m2 += v.y;
      });
      a = sum_of_eight(a), b = sum_of_eight(b), m2 = sum_of_eight(m2);
      if (j % 8 == 0) {
        const float inverse = 1.0f / (float)s.positions, off = a * inverse, cg = (float)s.per_group;
        group_mean[g] = shift + off;
        group_rstd[g] = 1.0f / __builtin_sqrtf(larger(__builtin_fmaf(m2, 1.0f / cg, __builtin_fmaf(-off, a, b)), 0.0f) * inverse + s.eps);
      }
    }
  }
  __syncthreads();
  if (p.tile == 0)
    for (uint32_t g = threadIdx.x; g < s.groups; g += NT) {
      mean[(size_t)p.sample * s.groups + g] = group_mean[g];
      rstd[(size_t)p.sample * s.groups + g] = group_rstd[g];
    }
  float mu[8], r[8];
  spread(s, place, group_mean, mu);
  spread(s, place, group_rstd, r);
#pragma unroll
  for (int i = 0; i < kChunk; ++i) k[i] *= r[i];
  each_row([&](size_t row, float v[8]) {
#pragma unroll
    for (int i = 0; i < kChunk; ++i) v[i] = act.template value<T>(__builtin_fmaf(v[i] - mu[i], k[i], b[i]));
    if (!kWhole || p.valid) store_chunk<T>(y + row * s.y_stride + p.column, kWhole ? kChunk : p.valid, v);
  });
}

struct BackShape {
  size_t dy_stride, dx_stride;
};

// share[item][0 = gamma, 1 = beta][channels]: an item's sums for the parameters' gradients; part[sample][group][tile]: those of u and u h.
// In the second stage workgroups behind the tiles' sum the shares.  With d = x - mu, a = r g: z = d a + b, the sums for gamma are r times those
// of dz d, and dx = dz a - (r^2 mean(u h) d + r mean(u)), so that a value takes six instructions besides its conversions and the slope.
template <typename T, typename A, bool HELD, int STAGE>
__global__ __launch_bounds__(NT) void group_norm_backward_kernel(A act, const typename T::value* __restrict__ dy, const typename T::value* __restrict__ x,
                                                                 const uint2* __restrict__ codes, const uint8_t* __restrict__ scales,
                                                                 GroupShape s, BackShape b, const float* __restrict__ mean,
                                                                 const float* __restrict__ rstd, Params gamma, Params beta,
                                                                 typename T::value* __restrict__ dx, float2* __restrict__ part,
                                                                 float* __restrict__ share, GradParams grads)
{
  extern __shared__ float room[];
  const uint32_t items = s.samples * s.tiles;
  if (STAGE == kWrite && blockIdx.x >= items) {
    sum_shares<NT / 32>(share, items, s.channels, blockIdx.x - items, grads, room);
    return;
  }
  float* const s1 = room + GroupRoom::chunks() + GroupRoom::channels();
  float *const s2 = s1 + s.groups, *const by_channel = s2 + s.groups;
  const uint32_t item = STAGE == kWrite ? items - 1 - blockIdx.x : blockIdx.x;
  const Pass p = pass_of(s, item);
  const GroupPlace place = group_place(s, p);
  constexpr int kRows = T::bytes == 4 && !HELD ? 2 : 4;
  constexpr bool kWhole = IsWhole<A>::value;
  RowBatch<T, kWhole, kRows> above;
  HeldBatch<T, kWhole, HELD, kRows> held;
  auto load = [&](uint32_t from) {
    above.load(s, p, dy, b.dy_stride, from);
    held.load(s, p, x, codes, scales, from);
  };
  load(0);
  float mu[8], r[8], a[8], beta_of[8];
  spread(s, place, mean + (size_t)p.sample * s.groups, mu);
  spread(s, place, rstd + (size_t)p.sample * s.groups, r);
  load_params(gamma, p.chunk * kChunk, p.valid, 1.0f, a);
  load_params(beta, p.chunk * kChunk, p.valid, 0.0f, beta_of);
  if (STAGE != kWrite && threadIdx.x < s.width) {
#pragma unroll
    for (int i = 0; i < kChunk; ++i)
      if (i < p.valid) by_channel[p.chunk * kChunk + i] = a[i];
  }
#pragma unroll
  for (int i = 0; i < kChunk; ++i) a[i] *= r[i];
  // each(row, dz, x - mu) for every row of the thread
  auto each_row = [&](auto&& each) {
    for (uint32_t from = 0;;) {
#pragma unroll
      for (int k = 0; k < kRows; ++k) {
        float u[8], v[8];
        above.value(k, u);
        held.minus(k, mu, v);
#pragma unroll
        for (int i = 0; i < kChunk; ++i) u[i] *= act.template slope<T>(__builtin_fmaf(v[i], a[i], beta_of[i]));
        if (from + k < p.count) each(p.row + (from + k) * s.lanes, u, v);
      }
      from += kRows;
      if (from >= p.count) break;
      load(from);
    }
  };
  const float inverse = 1.0f / ((float)s.positions * (float)s.per_group);
  if (STAGE != kWrite) {
    float dg[8], db[8];
#pragma unroll
    for (int i = 0; i < kChunk; ++i) dg[i] = db[i] = 0.0f;
    each_row([&](size_t, float u[8], float v[8]) {
#pragma unroll
      for (int i = 0; i < kChunk; ++i) dg[i] = __builtin_fmaf(u[i], v[i], dg[i]), db[i] += u[i];
    });
    if (STAGE == kBoth) load(0);
#pragma unroll
    for (int i = 0; i < kChunk; ++i) {
      dg[i] *= r[i];
      if (HELD && !kWhole && i >= p.valid) dg[i] = db[i] = 0.0f;  // a group of NaN reaches behind a row's end
    }
    // sums of the channels for the parameters, and, each times its gamma, of the groups
    auto finish = [&](const float v[8], int which, float* group_sum) {
      const float* sums = sum_channels(v, s, room);
      if (share) {
        float* to = share + ((size_t)item * 2 + which) * s.channels;
        for (uint32_t c = threadIdx.x; c < s.channels; c += NT) to[c] = sums[c];
      }
      sum_groups(s, [&](uint32_t c) { return sums[c] * by_channel[c]; }, [&](uint32_t at, float sum) { group_sum[at] = sum; });
    };
    finish(dg, 0, s2);
    finish(db, 1, s1);
    __syncthreads();
    if (STAGE == kSums) {
      for (uint32_t at = threadIdx.x; at < s.groups; at += NT)
        part[((size_t)p.sample * s.groups + at) * s.tiles + p.tile] = make_float2(s1[at], s2[at]);
      return;
    }
    for (uint32_t at = threadIdx.x; at < s.groups; at += NT) s1[at] *= inverse, s2[at] *= inverse;
  } else {
    for (uint32_t j = threadIdx.x; j < s.groups * 8; j += NT) {
      const float2* from = part + ((size_t)p.sample * s.groups + j / 8) * s.tiles;
      float sum1 = 0.0f, sum2 = 0.0f;
      for_tiles(s, from, j % 8, [&](uint32_t, float2 v) { sum1 += v.x, sum2 += v.y; });
      sum1 = sum_of_eight(sum1), sum2 = sum_of_eight(sum2);
      if (j % 8 == 0) s1[j / 8] = sum1 * inverse, s2[j / 8] = sum2 * inverse;
    }
  }
  __syncthreads();
  float m1[8], m2[8];
  spread(s, place, s1, m1);
  spread(s, place, s2, m2);
#pragma unroll
  for (int i = 0; i < kChunk; ++i) m1[i] *= r[i], m2[i] *= r[i] * r[i];
  each_row([&](size_t row, float u[8], float v[8]) {
#pragma unroll
    for (int i = 0; i < kChunk; ++i) u[i] = __builtin_fmaf(u[i], a[i], -__builtin_fmaf(v[i], m2[i], m1[i]));
    if (!kWhole || p.valid) store_chunk<T>(dx + row * b.dx_stride + p.column, kWhole ? kChunk : p.valid, u);
  });
}

// The parameters' gradients where the backward pass was one launch.
__global__ __launch_bounds__(1024) void group_norm_reduce_kernel(const float* __restrict__ share, uint32_t shares, uint32_t channels, GradParams grads)
{
  __shared__ float sum[32 * 33];
  sum_shares<32>(share, shares, channels, blockIdx.x, grads, sum);
}

__global__ void group_norm_zero_kernel(uint32_t channels, GradParams grads)
{
  const uint32_t i = blockIdx.x * blockDim.x + threadIdx.x;
  if (i < channels) grads.store(true, i, 0.0f), grads.store(false, i, 0.0f);
}

// ---------------------------------------------------------------- launches
constexpr uint32_t kWantedTiles = 512;   // workgroups of a launch: two to a compute unit
constexpr uint32_t kLeastRows = 8;  // of a thread in a tile, unless a sample has fewer

// Tiles go by the shape alone, so that forward, backward and the workspace agree whatever a call's type.
static int group_shape(size_t samples, size_t positions, size_t channels, size_t groups, bool quads, GroupShape* s)
{
  if (channels == 0 || positions == 0 || groups == 0 || channels % groups) return CSWAP_E_ARG;
  if (channels > kMaxChannels || groups > kMaxGroups || samples > kMaxSamples || positions >= ((size_t)1 << 31) ||
      (samples && positions > (((size_t)1 << 31) - 1) / samples))
    return CSWAP_E_UNSUPPORTED;
  const uint32_t nt = NT;
  s->samples = (uint32_t)samples, s->positions = (uint32_t)positions, s->channels = (uint32_t)channels, s->groups = (uint32_t)groups;
  s->per_group = (uint32_t)(channels / groups);
  s->code_chunks = (uint32_t)(pitch_of(channels) / kChunk);
  s->width = quads ? s->code_chunks : (uint32_t)((channels + kChunk - 1) / kChunk);
  s->lanes = nt / s->width;
  s->by_width = row_divisor(s->width), s->by_group = row_divisor(s->per_group);
  // by whole quads of chunks in any case, so that tiles do not depend on `quads`
  const uint32_t least = nt / s->code_chunks * kLeastRows, most = (s->positions + least - 1) / least;
  uint32_t tiles = samples ? (kWantedTiles + s->samples - 1) / s->samples : 1;
  if (tiles > most) tiles = most;
  s->tile_rows = (s->positions + tiles - 1) / tiles;
  s->tiles = (s->positions + s->tile_rows - 1) / s->tile_rows;
  return CSWAP_OK;
}

template <typename Fn> static int with_act(int act, bool whole, Fn&& fn)
{
  if (!whole) return fn(AnyAct{act});
  switch (act) {
    case CSWAP_ACT_GELU: return fn(Gelu());
    case CSWAP_ACT_GELU_TANH: return fn(GeluTanh());
    case CSWAP_ACT_SILU: return fn(Silu());
    default: return fn(Identity());
  }
}

static bool act_ok(int act) { return act == CSWAP_ACT_NONE || (act >= CSWAP_ACT_GELU && act <= CSWAP_ACT_SILU); }

static size_t part_bytes(const GroupShape& s) { return s.tiles > 1 ? (size_t)s.samples * s.groups * s.tiles * sizeof(float2) : 0; }

}  // namespace q8
}  // namespace cswap

using namespace cswap;
using namespace cswap::q8;

extern "C" size_t cswap_group_norm_workspace_bytes(size_t samples, size_t positions, size_t channels, size_t groups, int backward)
{
  GroupShape s;
  if (group_shape(samples, positions, channels, groups, true, &s) || samples == 0) return 0;
  return part_bytes(s) + (backward ? (size_t)s.samples * s.tiles * 2 * s.channels * sizeof(float) : 0);
}

extern "C" int cswap_group_norm_forward(int act, const void* d_x, int dtype, size_t samples, size_t positions, size_t channels, size_t groups,
                                        ptrdiff_t x_stride, const void* d_gamma, const void* d_beta, int param_dtype, float eps, void* d_y,
                                        ptrdiff_t y_stride, float* d_mean, float* d_rstd, int8_t* d_codes, uint8_t* d_scales, void* d_ws,
                                        size_t ws_bytes, cswap_stream_t stream)
{
  GroupShape s;
  const bool hold = d_codes || d_scales;
  if (int e = group_shape(samples, positions, channels, groups, hold, &s)) return e;
  if (int e = check_rows(samples * positions, channels, &x_stride)) return e;
  if (int e = check_rows(samples * positions, channels, &y_stride)) return e;
  if (!act_ok(act) || !dtype_known(dtype) || !dtype_known(param_dtype) || !(eps >= 0.0f)) return CSWAP_E_ARG;
  if (samples == 0) return CSWAP_OK;
  if (!value_ptr(d_x, dtype) || !value_ptr(d_y, dtype) || !value_ptr(d_mean, CSWAP_DT_F32) || !value_ptr(d_rstd, CSWAP_DT_F32))
    return CSWAP_E_ARG;
  if ((d_gamma && !value_ptr(d_gamma, param_dtype)) || (d_beta && !value_ptr(d_beta, param_dtype))) return CSWAP_E_ARG;
  if (hold && !checkpoint_ptrs(d_codes, d_scales)) return CSWAP_E_ARG;
  const size_t need = part_bytes(s);
  if (need && (!d_ws || reinterpret_cast<uintptr_t>(d_ws) % 8)) return CSWAP_E_ARG;
  if (ws_bytes < need) return CSWAP_E_NOMEM;
  s.x_stride = (size_t)x_stride, s.y_stride = (size_t)y_stride, s.eps = eps;
  const Params g = {d_gamma, param_dtype}, b = {d_beta, param_dtype};
  hipStream_t st = static_cast<hipStream_t>(stream);
  return with_type(dtype, [&](auto t) {
    typedef decltype(t) T;
    return with_act(act, s.channels % kChunk == 0, [&](auto f) {
      typedef decltype(f) A;
      auto launch = [&](auto k, auto a) {
        hipLaunchKernelGGL(k, dim3(s.samples * s.tiles), dim3(NT), GroupRoom::bytes(s, false), st, static_cast<const typename T::value*>(d_x), s, a, g, b,
                           static_cast<typename T::value*>(d_y), d_mean, d_rstd, reinterpret_cast<uint2*>(d_codes), d_scales,
                           static_cast<float2*>(d_ws));
        return check_launch();
      };
      if (s.tiles == 1) return hold ? launch(group_norm_forward_kernel<T, A, true, kBoth>, f) : launch(group_norm_forward_kernel<T, A, false, kBoth>, f);
      // the first stage needs no activation
      typedef typename FirstStage<A>::type B;
      const B none = {};
      if (int e = hold ? launch(group_norm_forward_kernel<T, B, true, kSums>, none) : launch(group_norm_forward_kernel<T, B, false, kSums>, none)) return e;
      return launch(group_norm_forward_kernel<T, A, false, kWrite>, f);
    });
  });
}

extern "C" int cswap_group_norm_backward(int act, const void* d_dy, int dtype, size_t samples, size_t positions, size_t channels, size_t groups,
                                         ptrdiff_t dy_stride, const void* d_x, ptrdiff_t x_stride, const int8_t* d_codes,
                                         const uint8_t* d_scales, const float* d_mean, const float* d_rstd, const void* d_gamma,
                                         const void* d_beta, int param_dtype, void* d_dx, ptrdiff_t dx_stride, void* d_dgamma, void* d_dbeta,
                                         void* d_ws, size_t ws_bytes, cswap_stream_t stream)
{
  GroupShape s;
  if (int e = group_shape(samples, positions, channels, groups, false, &s)) return e;
  if (int e = check_rows(samples * positions, channels, &dy_stride)) return e;
  if (int e = check_rows(samples * positions, channels, &x_stride)) return e;
  if (int e = check_rows(samples * positions, channels, &dx_stride)) return e;
  if (!act_ok(act) || !dtype_known(dtype) || !dtype_known(param_dtype)) return CSWAP_E_ARG;
  if ((d_gamma && !value_ptr(d_gamma, param_dtype)) || (d_beta && !value_ptr(d_beta, param_dtype)) ||
      (d_dgamma && !value_ptr(d_dgamma, param_dtype)) || (d_dbeta && !value_ptr(d_dbeta, param_dtype)))
    return CSWAP_E_ARG;
  const GradParams grads = {d_dgamma, d_dbeta, param_dtype};
  const bool reduce = d_dgamma || d_dbeta;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (samples == 0) {
    if (!reduce) return CSWAP_OK;
    hipLaunchKernelGGL(group_norm_zero_kernel, dim3((s.channels + 255) / 256), dim3(256), 0, st, s.channels, grads);
    return check_launch();
  }
  const bool held = d_codes || d_scales;
  if (!value_ptr(d_dy, dtype) || !value_ptr(d_dx, dtype) || !value_ptr(d_mean, CSWAP_DT_F32) || !value_ptr(d_rstd, CSWAP_DT_F32)) return CSWAP_E_ARG;
  if (held ? (d_x || !checkpoint_ptrs(d_codes, d_scales)) : !value_ptr(d_x, dtype)) return CSWAP_E_ARG;
  const size_t first = part_bytes(s), need = first + (reduce ? (size_t)s.samples * s.tiles * 2 * s.channels * sizeof(float) : 0);
  if (need && (!d_ws || reinterpret_cast<uintptr_t>(d_ws) % 8)) return CSWAP_E_ARG;
  if (ws_bytes < need) return CSWAP_E_NOMEM;
  s.x_stride = (size_t)x_stride, s.eps = 0.0f;
  const BackShape strides = {(size_t)dy_stride, (size_t)dx_stride};
  float* share = reduce ? reinterpret_cast<float*>(static_cast<char*>(d_ws) + first) : nullptr;
  const Params g = {d_gamma, param_dtype}, b = {d_beta, param_dtype};
  const uint32_t items = s.samples * s.tiles, columns = (2 * s.channels + 31) / 32;
  const int e = with_type(dtype, [&](auto t) {
    typedef decltype(t) T;
    return with_act(act, s.channels % kChunk == 0, [&](auto f) {
      typedef decltype(f) A;
      auto launch = [&](auto k, uint32_t grid) {
        hipLaunchKernelGGL(k, dim3(grid), dim3(NT), GroupRoom::bytes(s, true), st, f, static_cast<const typename T::value*>(d_dy),
                           static_cast<const typename T::value*>(d_x), reinterpret_cast<const uint2*>(d_codes), d_scales, s, strides, d_mean,
                           d_rstd, g, b, static_cast<typename T::value*>(d_dx), static_cast<float2*>(d_ws), share, grads);
        return check_launch();
      };
      if (s.tiles == 1) return held ? launch(group_norm_backward_kernel<T, A, true, kBoth>, items) : launch(group_norm_backward_kernel<T, A, false, kBoth>, items);
      if (int r = held ? launch(group_norm_backward_kernel<T, A, true, kSums>, items) : launch(group_norm_backward_kernel<T, A, false, kSums>, items)) return r;
      const uint32_t grid = items + (reduce ? columns : 0);
      return held ? launch(group_norm_backward_kernel<T, A, true, kWrite>, grid) : launch(group_norm_backward_kernel<T, A, false, kWrite>, grid);
    });
  });
  if (e || s.tiles > 1 || !reduce) return e;
  hipLaunchKernelGGL(group_norm_reduce_kernel, dim3(columns), dim3(1024), 0, st, share, items, s.channels, grads);
  return check_launch();
}
