// adamw_kernels.hip -- one AdamW step over many tensors at once, the moments held in 8 bits or in fp32.
//
//   m' = b1 m + (1 - b1) g,   v' = b2 v + (1 - b2) g^2                                   (t: the step, from 1)
//   p' = (1 - lr wd) p - lr / (1 - b1^t) m' / (sqrt(v') / sqrt(1 - b2^t) + eps)
//
// Moments in 8 bits.  32 consecutive values of a tensor share 2^e, e = max(floor(log2 max|x|) - 6, -126), as the byte e + 127 (255, with
// codes of 0: a NaN or an infinity among them).  A value's magnitude y = |x| / 2^e is held by the exponent and three bits of y + T, and
// stands for that sum less T: T = 2^-8 for m, whose eighth bit is the sign, T = 2^-24 for v.  So a value keeps a relative precision of
// 1/16 to 1/8 of the least bit over 15 powers of two of m and 31 of v (m goes with the root of v), and fades out evenly below; eight bits
// spread evenly, as those of an activation, would make v 0 where g is a tenth of its neighbours', and m / sqrt(v) with it arbitrary.
//
// Rounding to nearest would hold v for ever: b2 = 0.999 moves it by a thousandth a step, codes are 1/8 to 1/16 apart.  What is cut off is
// carried up where it and an offset u make a whole, u = (i A + t B) mod 2^32 for m and (i B + t A) mod 2^32 for v (i: the element's
// number in its tensor), A and B 2^32 over the plastic number and over its square: over the steps the offsets of an element, and in a
// step those of its neighbours, fill [0, 2^32) as evenly as any (M. Roberts, "The unreasonable effectiveness of quasirandom sequences").
// After 6000 steps on gradients N(0, 1) of many scales v is 17 % off what fp32 makes of it (one standard deviation; 2 % low in the mean),
// on gradients that are 0 in 98 of 100 steps 12 % (5 % low); with random offsets 20 and 24 %; to nearest it is 75 % low, and three times too large.
// The update itself uses m' and v' as they are before they are rounded.  Where v's code becomes 0 m's does, too: m / eps is no step.
//
// A code hangs on its value's last bits, so m' and v' are rounded after each product and each sum, to the same bits whoever computes them
// (the build contracts nothing); what only the parameter sees goes through v_sqrt_f32 and v_rcp_f32, one unit off in the last place each.
//
// Memory bounds it: bf16 with moments in 8 bits 10.1 bytes a value, fp32 with fp32 moments 28.  Traced: 101.8 M bf16 values in 130 tensors, moments in
// 8 bits, two launches of 99 us and one of 7 (5.0 TB/s; a copy reaches 5.1), 51.4 M fp32 values with fp32 moments 260 and 10 (5.3 TB/s), the moments as fp32 values 111
// a launch (4.5 TB/s).  The tensors of a launch are in its
// arguments (so that it needs no table in device memory, which a
// capture or a second call could find changed), a workgroup finds its tensor by halving.
#include <hip/hip_runtime.h>
#include <math.h>
#include "../../include/cswap_hip.h"
#include "common.h"
#include "q8_block.h"

namespace cswap {
namespace q8 {

constexpr uint32_t kOffsetA = 0xC13FA9A9u, kOffsetB = 0x91E10DA5u;
constexpr uint32_t kNearest = 0x80000000u;  // the offset that rounds to nearest

// What a step's values go through; `step` alone is no factor.
struct StepFactors {
  float b1, one_minus_b1, b2, one_minus_b2, root, eps, decay, rate;  // root: 1 / sqrt(1 - b2^t), rate: lr / (1 - b1^t)
  uint32_t step;
};

struct StepTensor {
  void* param;
  const void* grad;
  uint8_t *m, *v;  // 8 bits: codes of whole groups, then their scales; else fp32 values
  float* master;   // NULL: none
  size_t n;
};

constexpr int kStepThreads = 256, kTensors = 64;
struct StepTable {  // 4 KB of arguments in all, with the rest
  StepTensor t[kTensors];
  uint32_t first[kTensors];  // workgroup
  uint8_t dtype[kTensors];
  uint32_t count;
};

// The last tensor that begins at or before the workgroup; a tensor without workgroups begins where the next one does.
template <typename Table> __device__ inline uint32_t tensor_of(const Table& table, uint32_t group)
{
  uint32_t lo = 0, hi = table.count;
  while (hi - lo > 1) {
    const uint32_t mid = (lo + hi) / 2;
    if (table.first[mid] <= group) lo = mid;
    else hi = mid;
  }
  return lo;
}

template <bool SIGNED> struct MomentCode {
  static constexpr uint32_t exponent = SIGNED ? 119 : 103;                  // of T
  static constexpr uint32_t base = exponent << 23;
  static __device__ inline float least() { return __uint_as_float(base); }
};

template <bool SIGNED> __device__ inline void decode_moment(uint2 q, float unit, float x[8])
{
#pragma unroll
  for (int i = 0; i < kChunk; ++i) {
    const uint32_t w = i < 4 ? q.x : q.y, c = (w >> (8 * (i & 3))) & (SIGNED ? 0x7fu : 0xffu);
    const float y = (__uint_as_float((c << 20) + MomentCode<SIGNED>::base) - MomentCode<SIGNED>::least()) * unit;
    x[i] = SIGNED ? __uint_as_float(__float_as_uint(y) | ((w << (24 - 8 * (i & 3))) & 0x80000000u)) : y;
  }
}

// The words whose top bytes are the codes.  (bits(y + T) << 4) + (u >> 8) - (bits(T) << 4) has the code there: the exponent's bits above
// the eighth fall off, and the last term is a byte that the shift brings in.
template <bool SIGNED> __device__ inline void moment_words(const float x[8], uint32_t max_bits, uint32_t u, uint32_t step, uint32_t* scale, uint32_t t[8])
{
  const int exponent = (int)(max_bits >> 23), b = max(exponent - 6, 1);
  *scale = exponent == 255 ? 255u : (uint32_t)b;
  const float inverse = __uint_as_float((uint32_t)(254 - b) << 23);
  constexpr uint32_t kTop = (0u - (MomentCode<SIGNED>::base >> 20)) & 0xffu;
#pragma unroll
  for (int i = 0; i < kChunk; ++i) {
    const float y = __builtin_fmaf(__builtin_fabsf(x[i]), inverse, MomentCode<SIGNED>::least());  // the product is exact
    t[i] = (__float_as_uint(y) << 4) + __builtin_amdgcn_alignbit(kTop, u, 8);
    u += step;
  }
}

__device__ inline uint2 top_bytes(const uint32_t t[8])
{
  // v_perm_b32 numbers the bytes of its second operand 0 to 3 and those of its first 4 to 7
  uint2 q;
  q.x = __builtin_amdgcn_perm(__builtin_amdgcn_perm(t[3], t[2], 0x07030c0cu), __builtin_amdgcn_perm(t[1], t[0], 0x0c0c0703u), 0x07060100u);
  q.y = __builtin_amdgcn_perm(__builtin_amdgcn_perm(t[7], t[6], 0x07030c0cu), __builtin_amdgcn_perm(t[5], t[4], 0x0c0c0703u), 0x07060100u);
  return q;
}

// Both moments of a chunk; all four lanes of a quad have to run this.
__device__ inline void store_moments(const float m[8], const float v[8], uint32_t um, uint32_t sm, uint32_t uv, uint32_t sv, uint8_t* m_at,
                                     uint8_t* v_at, size_t chunk, size_t groups)
{
  uint32_t tm[8], tv[8], m_scale, v_scale;
  moment_words<true>(m, quad_max_bits(m), um, sm, &m_scale, tm);
  moment_words<false>(v, quad_max_bits(v), uv, sv, &v_scale, tv);
#pragma unroll
  for (int i = 0; i < kChunk; ++i) {
    tm[i] |= __float_as_uint(m[i]) & 0x80000000u;
    if (tv[i] < 0x01000000u) tm[i] = 0;
  }
  uint2 qm = top_bytes(tm), qv = top_bytes(tv);
  if (m_scale == 255u || v_scale == 255u) qm = {0u, 0u};
  if (v_scale == 255u) qv = {0u, 0u};
  reinterpret_cast<uint2*>(m_at)[chunk] = qm;
  reinterpret_cast<uint2*>(v_at)[chunk] = qv;
  if ((chunk & (kChunksPerGroup - 1)) == 0) {
    m_at[groups * kGroup + chunk / kChunksPerGroup] = (uint8_t)m_scale;
    v_at[groups * kGroup + chunk / kChunksPerGroup] = (uint8_t)v_scale;
  }
}

// v_sqrt_f32 takes a subnormal for 0.  Its root, below 2^-63, is nothing beside an eps of 2^25 times as much; with a smaller eps, which m
// would be divided by alone, such v are brought up by 2^64 first (five instructions a value: 3 us more a launch of 99).
__device__ inline bool roots_matter(const StepFactors& f) { return f.eps < 0x1p-38f * f.root; }
__device__ inline float root_of(float v, bool matter)
{
  if (!matter) return __builtin_amdgcn_sqrtf(v);
  const bool low = v < 0x1p-126f;
  return __builtin_amdgcn_ldexpf(__builtin_amdgcn_sqrtf(__builtin_amdgcn_ldexpf(v, low ? 64 : 0)), low ? -32 : 0);
}

template <typename T, bool SMALL> __device__ inline void step_chunk(const StepTensor& t, size_t chunk, size_t groups, const StepFactors& f)
{
  typedef typename T::value Value;
  const size_t at = chunk * kChunk;
  const int valid = at + kChunk <= t.n ? kChunk : at < t.n ? (int)(t.n - at) : 0;
  float p[8], g[8], m[8], v[8];
  load_chunk<T>(static_cast<const Value*>(t.grad) + at, valid, g);
  if (t.master) load_chunk<F32>(t.master + at, valid, p);
  else load_chunk<T>(static_cast<const Value*>(t.param) + at, valid, p);
  if (SMALL) {
    const uint2 qm = reinterpret_cast<const uint2*>(t.m)[chunk], qv = reinterpret_cast<const uint2*>(t.v)[chunk];
    const size_t scale = groups * kGroup + chunk / kChunksPerGroup;
    const float m_unit = unit_of(t.m[scale]), v_unit = unit_of(t.v[scale]);
    decode_moment<true>(qm, m_unit, m);
    decode_moment<false>(qv, v_unit, v);
  } else {
    load_chunk<F32>(reinterpret_cast<const float*>(t.m) + at, valid, m);
    load_chunk<F32>(reinterpret_cast<const float*>(t.v) + at, valid, v);
  }
  const bool matter = roots_matter(f);
#pragma unroll
  for (int i = 0; i < kChunk; ++i) {
    m[i] = m[i] * f.b1 + g[i] * f.one_minus_b1;
    v[i] = v[i] * f.b2 + (g[i] * g[i]) * f.one_minus_b2;
    const float d = __builtin_fmaf(root_of(v[i], matter), f.root, f.eps);
    p[i] = __builtin_fmaf(-f.rate, m[i] * __builtin_amdgcn_rcpf(d), p[i] * f.decay);
  }
  if (t.master) store_chunk<F32>(t.master + at, valid, p);
  store_chunk<T>(static_cast<Value*>(t.param) + at, valid, p);
  if (SMALL) {
    if (valid < kChunk) {  // a group of NaN reaches behind the last value
#pragma unroll
      for (int i = 0; i < kChunk; ++i) m[i] = i < valid ? m[i] : 0.0f, v[i] = i < valid ? v[i] : 0.0f;
    }
    const uint32_t i0 = (uint32_t)at;
    store_moments(m, v, i0 * kOffsetA + f.step * kOffsetB, kOffsetA, i0 * kOffsetB + f.step * kOffsetA, kOffsetB, t.m, t.v, chunk, groups);
  } else {
    store_chunk<F32>(reinterpret_cast<float*>(t.m) + at, valid, m);
    store_chunk<F32>(reinterpret_cast<float*>(t.v) + at, valid, v);
  }
}

template <bool SMALL>
__global__ __launch_bounds__(kStepThreads) void adamw_step_kernel(StepTable table, StepFactors given, const StepFactors* __restrict__ factors)
{
  const StepFactors f = factors ? *factors : given;
  const uint32_t k = tensor_of(table, blockIdx.x);
  const StepTensor& t = table.t[k];
  const size_t groups = (t.n + kGroup - 1) / kGroup, chunk = (size_t)(blockIdx.x - table.first[k]) * kStepThreads + threadIdx.x;
  if (chunk >= groups * kChunksPerGroup) return;  // a quad leaves as a whole
  switch (table.dtype[k]) {
    case CSWAP_DT_F32: return step_chunk<F32, SMALL>(t, chunk, groups, f);
    case CSWAP_DT_BF16: return step_chunk<BF16, SMALL>(t, chunk, groups, f);
    default: return step_chunk<F16, SMALL>(t, chunk, groups, f);
  }
}

struct MomentTensor {
  float *m, *v;        // values
  uint8_t *m8, *v8;
  size_t n;
};
struct MomentTable {
  MomentTensor t[kTensors];
  uint32_t first[kTensors];
  uint32_t count;
};

template <bool PACK> __global__ __launch_bounds__(kStepThreads) void adamw_moments_kernel(MomentTable table)
{
  const uint32_t k = tensor_of(table, blockIdx.x);
  const MomentTensor& t = table.t[k];
  const size_t groups = (t.n + kGroup - 1) / kGroup, chunk = (size_t)(blockIdx.x - table.first[k]) * kStepThreads + threadIdx.x;
  if (chunk >= groups * kChunksPerGroup) return;
  const size_t at = chunk * kChunk, scale = groups * kGroup + chunk / kChunksPerGroup;
  const int valid = at + kChunk <= t.n ? kChunk : at < t.n ? (int)(t.n - at) : 0;
  float m[8], v[8];
  if (PACK) {
    load_chunk<F32>(t.m + at, valid, m);
    load_chunk<F32>(t.v + at, valid, v);
    store_moments(m, v, kNearest, 0, kNearest, 0, t.m8, t.v8, chunk, groups);
  } else {
    decode_moment<true>(reinterpret_cast<const uint2*>(t.m8)[chunk], unit_of(t.m8[scale]), m);
    decode_moment<false>(reinterpret_cast<const uint2*>(t.v8)[chunk], unit_of(t.v8[scale]), v);
    store_chunk<F32>(t.m + at, valid, m);
    store_chunk<F32>(t.v + at, valid, v);
  }
}

static __host__ __device__ StepFactors factors_of(double lr, double b1, double b2, double eps, double decay, long long step)
{
  StepFactors f;
  f.b1 = (float)b1, f.one_minus_b1 = (float)(1.0 - b1), f.b2 = (float)b2, f.one_minus_b2 = (float)(1.0 - b2);
  f.root = (float)(1.0 / sqrt(1.0 - pow(b2, (double)step))), f.eps = (float)eps;
  f.decay = (float)(1.0 - lr * decay), f.rate = (float)(lr / (1.0 - pow(b1, (double)step)));
  f.step = (uint32_t)step;
  return f;
}

// The next step's factors, for launches behind this one on the stream.
__global__ void adamw_begin_kernel(long long* step, const float* lr, double given, double b1, double b2, double eps, double decay, StepFactors* out)
{
  const long long t = *step + 1;
  *step = t;
  *out = factors_of(lr ? (double)*lr : given, b1, b2, eps, decay, t);
}

static bool options_fit(const cswap_adamw_options* o)
{
  return o && o->lr >= 0.0 && o->lr < 1e30 && o->beta1 >= 0.0 && o->beta1 < 1.0 && o->beta2 >= 0.0 && o->beta2 < 1.0 && o->eps >= 1e-30 &&
         o->eps < 1e30 && o->weight_decay >= 0.0 && o->weight_decay < 1e30;
}

constexpr size_t kMostValues = kMaxChunks * kChunk - kGroup;  // of a tensor: chunk numbers are 31 bits

constexpr uint64_t kMostGroups = (1u << 24) - 1;          // of a launch: 2^32 threads

// Launches of up to kTensors tensors; `take` puts number i of the caller's into a place of the table and says how many values it has.
template <typename Table, typename Take, typename Launch> static int for_tables(size_t count, Take&& take, Launch&& launch)
{
  Table table;
  table.count = 0;
  uint64_t groups = 0;
  for (size_t i = 0; i <= count; ++i) {
    if (i < count) {
      const size_t n = take(i, table, table.count);
      if (n) {
        const uint64_t more = ((n + kGroup - 1) / kGroup * kChunksPerGroup + kStepThreads - 1) / kStepThreads;
        if (table.count == 0 || groups + more <= kMostGroups) {
          table.first[table.count++] = (uint32_t)groups;
          groups += more;
          if (table.count < kTensors) continue;
        } else {
          --i;  // first in the next launch
        }
      } else {
        continue;
      }
    }
    if (table.count == 0) continue;
    launch(table, dim3((unsigned)groups));
    if (int e = check_launch()) return e;
    table.count = 0, groups = 0;
  }
  return CSWAP_OK;
}

static int check_tensors(const cswap_adamw_tensor* t, size_t count, int bits)
{
  if (bits != 8 && bits != 32) return CSWAP_E_ARG;
  if (count && !t) return CSWAP_E_ARG;
  for (size_t i = 0; i < count; ++i) {
    if (!dtype_known(t[i].dtype)) return CSWAP_E_ARG;
    if (t[i].n == 0) continue;
    if (t[i].n > kMostValues) return CSWAP_E_UNSUPPORTED;
    if (!value_ptr(t[i].param, t[i].dtype) || !value_ptr(t[i].grad, t[i].dtype)) return CSWAP_E_ARG;
    if (t[i].master && !value_ptr(t[i].master, CSWAP_DT_F32)) return CSWAP_E_ARG;
    const uintptr_t align = bits == 8 ? 8 : 4;
    if (!t[i].exp_avg || !t[i].exp_avg_sq || reinterpret_cast<uintptr_t>(t[i].exp_avg) % align || reinterpret_cast<uintptr_t>(t[i].exp_avg_sq) % align)
      return CSWAP_E_ARG;
  }
  return CSWAP_OK;
}

static int step_all(const cswap_adamw_tensor* tensors, size_t count, int bits, const StepFactors& given, const StepFactors* factors, hipStream_t st)
{
  return for_tables<StepTable>(
      count,
      [&](size_t i, StepTable& table, uint32_t at) {
        const cswap_adamw_tensor& t = tensors[i];
        table.t[at] = {t.param, t.grad, static_cast<uint8_t*>(t.exp_avg), static_cast<uint8_t*>(t.exp_avg_sq), t.master, t.n};
        table.dtype[at] = (uint8_t)t.dtype;
        return t.n;
      },
      [&](const StepTable& table, dim3 grid) {
        hipLaunchKernelGGL(bits == 8 ? adamw_step_kernel<true> : adamw_step_kernel<false>, grid, dim3(kStepThreads), 0, st, table, given, factors);
      });
}

template <bool PACK> static int moments_all(const cswap_adamw_moments* tensors, size_t count, hipStream_t st)
{
  if (count && !tensors) return CSWAP_E_ARG;
  for (size_t i = 0; i < count; ++i) {
    const cswap_adamw_moments& t = tensors[i];
    if (t.n == 0) continue;
    if (t.n > kMostValues) return CSWAP_E_UNSUPPORTED;
    if (!value_ptr(t.exp_avg, CSWAP_DT_F32) || !value_ptr(t.exp_avg_sq, CSWAP_DT_F32) || !t.exp_avg8 || !t.exp_avg_sq8 ||
        reinterpret_cast<uintptr_t>(t.exp_avg8) % 8 || reinterpret_cast<uintptr_t>(t.exp_avg_sq8) % 8)
      return CSWAP_E_ARG;
  }
  return for_tables<MomentTable>(
      count,
      [&](size_t i, MomentTable& table, uint32_t at) {
        const cswap_adamw_moments& t = tensors[i];
        table.t[at] = {t.exp_avg, t.exp_avg_sq, t.exp_avg8, t.exp_avg_sq8, t.n};
        return t.n;
      },
      [&](const MomentTable& table, dim3 grid) {
        hipLaunchKernelGGL(adamw_moments_kernel<PACK>, grid, dim3(kStepThreads), 0, st, table);
      });
}

}  // namespace q8
}  // namespace cswap

using namespace cswap;
using namespace cswap::q8;

extern "C" size_t cswap_adamw_moment_bytes(size_t n) { return groups_of(n) * (kGroup + 1); }

extern "C" size_t cswap_adamw_factors_bytes(void) { return sizeof(StepFactors); }

extern "C" int cswap_adamw_step(const cswap_adamw_tensor* tensors, size_t count, int bits, const cswap_adamw_options* options,
                                long long step, cswap_stream_t stream)
{
  if (int e = check_tensors(tensors, count, bits)) return e;
  if (!options_fit(options) || step < 1) return CSWAP_E_ARG;
  const StepFactors f = factors_of(options->lr, options->beta1, options->beta2, options->eps, options->weight_decay, step);
  return step_all(tensors, count, bits, f, nullptr, static_cast<hipStream_t>(stream));
}

extern "C" int cswap_adamw_step_counted(const cswap_adamw_tensor* tensors, size_t count, int bits, const cswap_adamw_options* options,
                                        long long* d_step, const float* d_lr, void* d_factors, cswap_stream_t stream)
{
  if (int e = check_tensors(tensors, count, bits)) return e;
  if (!options_fit(options) || !d_step || reinterpret_cast<uintptr_t>(d_step) % 8 || (d_lr && !value_ptr(d_lr, CSWAP_DT_F32)) ||
      !value_ptr(d_factors, CSWAP_DT_F32))
    return CSWAP_E_ARG;
  hipStream_t st = static_cast<hipStream_t>(stream);
  hipLaunchKernelGGL(adamw_begin_kernel, dim3(1), dim3(1), 0, st, d_step, d_lr, options->lr, options->beta1, options->beta2, options->eps,
                     options->weight_decay, static_cast<StepFactors*>(d_factors));
  if (int e = check_launch()) return e;
  return step_all(tensors, count, bits, StepFactors(), static_cast<const StepFactors*>(d_factors), st);
}

extern "C" int cswap_adamw_pack(const cswap_adamw_moments* tensors, size_t count, cswap_stream_t stream)
{
  return moments_all<true>(tensors, count, static_cast<hipStream_t>(stream));
}

extern "C" int cswap_adamw_unpack(const cswap_adamw_moments* tensors, size_t count, cswap_stream_t stream)
{
  return moments_all<false>(tensors, count, static_cast<hipStream_t>(stream));
}
