// AdamW over many tensors in one launch, moments in 32 or in 8 bits.
//
//   g' = g * grad_scale;  m = b1 m + (1 - b1) g';  v = b2 v + (1 - b2) g'^2
//   w  = w (1 - lr wd) - (lr / (1 - b1^t)) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// w is the fp32 parameter, or the fp32 master of a 16-bit parameter, which then receives w rounded
// to nearest.  Every operation is one correctly rounded fp32 operation in the order written here
// (no contraction, see the Makefile), so a host restatement in the same order gives the same bits.
//
// 8-bit moments.  256 consecutive entries of a tensor share one power of two: the fp32 exponent
// field E of the largest finite |x| among them (one byte).  |x| times 2^(top - E) is an fp32 number
// whose bits, cut to exponent and three bits of mantissa (>> 20), are the code: a float with the
// subnormals of fp32 itself, no table and no division.  m: sign and 4 + 3 bits (top 14), v: 5 + 3
// bits (top 30); the all-ones code is a value that was not finite.
// Rounding is stochastic: b2 = 0.999 moves v by 0.1 % a step and the codes are 6 to 12 % apart, so
// rounding to nearest would hold v where it is for ever; rounding up with the probability that the
// remainder stands for keeps the expected value exact.  The bits come from a hash of (seed, step,
// tensor, entry), so a step can be repeated.  A positive v never becomes zero: the step m / eps that
// would follow is unbounded.
//
// Bound: HBM.  Everything is read and written once, in 16-byte accesses (4 bytes of codes) that pass the caches
// by: nothing is used again before the next step, and 92 M fp32 weights take 432 us (6.0 TB/s) that way, 478
// through the caches.  Codes stay in the caches (8-bit step of 226 M bf16 weights and a decode 930 us, 994 past
// them).  A thread takes four entries at a time, a workgroup 1024 or, with the longer 8-bit arithmetic, 2048
// (bf16 / 8 bits 624 us, 5.8 TB/s, 674 with 1024; fp32 / 32 bits 432 with 1024, 460 with 2048).
#include <algorithm>
#include <cmath>

#include "pp_device.h"
#include "pp_lowp.h"

namespace {

constexpr int kBlk = 256;  // entries that share an exponent: one wave x 4

struct AdamWDescs {
  void* p[PP_OPT_MAX_TENSORS];
  const void* g[PP_OPT_MAX_TENSORS];
  float* w[PP_OPT_MAX_TENSORS];
  void* m[PP_OPT_MAX_TENSORS];
  void* v[PP_OPT_MAX_TENSORS];
  uint8_t* me[PP_OPT_MAX_TENSORS];
  uint8_t* ve[PP_OPT_MAX_TENSORS];
  const int64_t* step[PP_OPT_MAX_TENSORS];  // device counter, or NULL: number, c1, c2 from the host
  int64_t n[PP_OPT_MAX_TENSORS];
  int first[PP_OPT_MAX_TENSORS + 1];        // first workgroup of each tensor
  uint32_t number[PP_OPT_MAX_TENSORS];
  uint32_t wide;                            // bit t: four entries of every list of tensor t are one access
  float c1[PP_OPT_MAX_TENSORS];             // lr / (1 - b1^t)
  float c2[PP_OPT_MAX_TENSORS];             // 1 / sqrt(1 - b2^t)
};
struct AdamWArgs {
  float b1, nb1, b2, nb2, eps, decay;
  double lr, beta1, beta2;
  uint32_t seed, index;
  const float* grad_scale;
  int count;
};

__host__ __device__ inline uint32_t mix32(uint32_t x) {
  x ^= x >> 16;
  x *= 0x9E3779B9u;
  x ^= x >> 15;
  x *= 0xD1B54A33u;
  return x ^ (x >> 16);
}

// b^t by repeated squaring: the same on host and device
__host__ __device__ inline double int_power(double b, int64_t t) {
  double r = 1.0;
  for (; t > 0; t >>= 1, b *= b)
    if (t & 1) r *= b;
  return r;
}

__device__ __forceinline__ float wave_max_nonneg(float v) {
  v = pp_dpp_max<0x128>(v);
  v = pp_dpp_max<0x124>(v);
  v = pp_dpp_max<0x122>(v);
  v = pp_dpp_max<0x121>(v);
  return fmaxf(fmaxf(pp_readlane_f(v, 0), pp_readlane_f(v, 16)),
               fmaxf(pp_readlane_f(v, 32), pp_readlane_f(v, 48)));
}

// the value of a code: fp32 bits (exponent, 3 bits of mantissa) << 20, times 2^(E - top)
template <int TOP, bool SIGNED>
__device__ __forceinline__ float decode8(uint32_t code, int E) {
  const uint32_t mag = SIGNED ? (code & 127u) : code;
  float x = ldexpf(__uint_as_float(mag << 20), E - TOP);
  if (mag == (SIGNED ? 127u : 255u)) x = __uint_as_float(0x7fc00000u);
  return SIGNED && (code & 128u) ? -x : x;
}

__device__ __forceinline__ float finite_size(float x) {
  const float a = fabsf(x);
  return a < __uint_as_float(0x7f800000u) ? a : 0.0f;  // (false for NaN)
}

template <int TOP, bool SIGNED>
__device__ __forceinline__ uint32_t encode8(float x, int E, uint32_t byte) {
  const float a = fabsf(x);
  uint32_t code = (__float_as_uint(ldexpf(a, TOP - E)) + (byte << 12) + 2048u) >> 20;
  if (!SIGNED && a > 0.0f) code = code > 1u ? code : 1u;
  if (!(a < __uint_as_float(0x7f800000u))) code = SIGNED ? 127u : 255u;
  if (SIGNED) code |= (__float_as_uint(x) >> 24) & 128u;
  return code;
}

// T: element type of p and g;  EIGHT: moments in 8 bits
template <typename T, bool EIGHT>
__global__ __launch_bounds__(256) void pp_adamw_kernel(AdamWDescs d, AdamWArgs a, int per_block) {
  int t = 0;
  for (int i = 1; i < a.count; ++i) t += (int)blockIdx.x >= d.first[i];
  const int64_t n = d.n[t];
  T* __restrict__ p = static_cast<T*>(d.p[t]);
  const T* __restrict__ g = static_cast<const T*>(d.g[t]);
  float* __restrict__ w = d.w[t];
  float c1 = d.c1[t], c2 = d.c2[t];
  uint32_t number = d.number[t];
  if (d.step[t]) {
    const int64_t s = *d.step[t];
    c1 = (float)(a.lr / (1.0 - int_power(a.beta1, s)));
    c2 = (float)(1.0 / sqrt(1.0 - int_power(a.beta2, s)));
    number = (uint32_t)s;
  }
  const float gs = a.grad_scale ? *a.grad_scale : 1.0f;
  const uint32_t key = EIGHT ? mix32(mix32(mix32(number) ^ a.seed) + a.index + (uint32_t)t) : 0u;
  const int64_t first = (int64_t)((int)blockIdx.x - d.first[t]) * per_block;
  const bool wide = d.wide >> t & 1;
  void* __restrict__ mp = d.m[t];
  void* __restrict__ vp = d.v[t];
  typedef PPElems<T, 4> ET;
  typedef PPElems<float, 4> EF;
  typedef PPElems<uint8_t, 4> E8;
  for (int it = 0; it < per_block; it += 1024) {
    const int64_t e0 = first + it + (int64_t)threadIdx.x * 4;
    if (first + it + (threadIdx.x & ~63) * 4 >= n) return;  // the whole wave is behind the end
    float gv[4], wv[4], mv[4], vv[4];
    uint32_t mc[4], vc[4];
    int Em = 0, Ev = 0;
    if (EIGHT) {
      Em = d.me[t][e0 / kBlk];
      Ev = d.ve[t][e0 / kBlk];
    }
    const bool whole = wide && e0 + 4 <= n;
    if (whole) {
      const typename ET::raw gr = ET::take(g + e0);
      const typename EF::raw wr = EF::take(w + e0);
      if (EIGHT) {
        const uint32_t mr = E8::load(static_cast<const uint8_t*>(mp) + e0);
        const uint32_t vr = E8::load(static_cast<const uint8_t*>(vp) + e0);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          mc[j] = mr >> (8 * j) & 255u;
          vc[j] = vr >> (8 * j) & 255u;
        }
      } else {
        const typename EF::raw mr = EF::take(static_cast<const float*>(mp) + e0);
        const typename EF::raw vr = EF::take(static_cast<const float*>(vp) + e0);
        EF::get(mr, mv);
        EF::get(vr, vv);
      }
      ET::get(gr, gv);
      EF::get(wr, wv);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int64_t e = e0 + j;
        const bool live = e < n;
        gv[j] = live ? (float)g[e] : 0.0f;
        wv[j] = live ? w[e] : 0.0f;
        if (EIGHT) {
          mc[j] = live ? static_cast<const uint8_t*>(mp)[e] : 0u;
          vc[j] = live ? static_cast<const uint8_t*>(vp)[e] : 0u;
        } else {
          mv[j] = live ? static_cast<const float*>(mp)[e] : 0.0f;
          vv[j] = live ? static_cast<const float*>(vp)[e] : 0.0f;
        }
      }
    }
    float tm = 0.0f, tv = 0.0f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (EIGHT) {
        mv[j] = decode8<14, true>(mc[j], Em);
        vv[j] = decode8<30, false>(vc[j], Ev);
      }
      const float gg = gv[j] * gs;
      mv[j] = mv[j] * a.b1 + gg * a.nb1;
      vv[j] = vv[j] * a.b2 + (gg * gg) * a.nb2;
      wv[j] = wv[j] * a.decay - (mv[j] / (sqrtf(vv[j]) * c2 + a.eps)) * c1;
      if (EIGHT) {
        tm = fmaxf(tm, finite_size(mv[j]));
        tv = fmaxf(tv, finite_size(vv[j]));
      }
    }
    if (EIGHT) {
      Em = (int)(__float_as_uint(wave_max_nonneg(tm)) >> 23);
      Ev = (int)(__float_as_uint(wave_max_nonneg(tv)) >> 23);
      const uint32_t q = key + 2u * (uint32_t)(e0 >> 2);
      const uint32_t bm = mix32(q), bv = mix32(q + 1u);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        mc[j] = encode8<14, true>(mv[j], Em, (bm >> (8 * j)) & 255u);
        vc[j] = encode8<30, false>(vv[j], Ev, (bv >> (8 * j)) & 255u);
      }
      if ((threadIdx.x & 63) == 0) {
        d.me[t][e0 / kBlk] = (uint8_t)Em;
        d.ve[t][e0 / kBlk] = (uint8_t)Ev;
      }
    }
    if (whole) {
      EF::stream(w + e0, EF::put(wv));
      if (sizeof(T) == 2) ET::stream(p + e0, ET::put(wv));
      if (EIGHT) {
        E8::store(static_cast<uint8_t*>(mp) + e0, mc[0] | mc[1] << 8 | mc[2] << 16 | mc[3] << 24);
        E8::store(static_cast<uint8_t*>(vp) + e0, vc[0] | vc[1] << 8 | vc[2] << 16 | vc[3] << 24);
      } else {
        EF::stream(static_cast<float*>(mp) + e0, EF::put(mv));
        EF::stream(static_cast<float*>(vp) + e0, EF::put(vv));
      }
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int64_t e = e0 + j;
        if (e >= n) break;
        w[e] = wv[j];
        if (sizeof(T) == 2) p[e] = (T)wv[j];
        if (EIGHT) {
          static_cast<uint8_t*>(mp)[e] = (uint8_t)mc[j];
          static_cast<uint8_t*>(vp)[e] = (uint8_t)vc[j];
        } else {
          static_cast<float*>(mp)[e] = mv[j];
          static_cast<float*>(vp)[e] = vv[j];
        }
      }
    }
  }
}

// Eight codes a thread: 8 bytes in, 16 or 32 out.
template <typename O, bool SIGNED>
__global__ __launch_bounds__(256) void pp_decode_moment_kernel(const uint8_t* __restrict__ code,
                                                               const uint8_t* __restrict__ exps,
                                                               O* __restrict__ out, int64_t n, int wide) {
  constexpr int kPer = 16 / sizeof(O);  // entries of a store
  const int64_t e0 = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 8;
  if (e0 >= n) return;
  const int E = exps[e0 / kBlk];
  if (wide && e0 + 8 <= n) {
    const typename PPRaw<8>::type c = PPElems<uint8_t, 8>::load(code + e0);
#pragma unroll
    for (int i = 0; i < 8; i += kPer) {
      float x[kPer];
#pragma unroll
      for (int j = 0; j < kPer; ++j)
        x[j] = decode8<SIGNED ? 14 : 30, SIGNED>(c[(i + j) / 4] >> (8 * (j & 3)) & 255u, E);
      PPElems<O, kPer>::stream(out + e0 + i, PPElems<O, kPer>::put(x));
    }
    return;
  }
  for (int64_t e = e0; e < n && e < e0 + 8; ++e) out[e] = (O)decode8<SIGNED ? 14 : 30, SIGNED>(code[e], E);
}

struct StepCounters {
  int64_t* at[PP_OPT_MAX_TENSORS];
};
__global__ void pp_count_step_kernel(StepCounters c, int count) {
  if ((int)threadIdx.x < count) *c.at[threadIdx.x] += 1;
}

}  // namespace

hipError_t pp_launch_count_step(int count, int64_t* const* step, hipStream_t st) {
  StepCounters c;
  for (int i = 0; i < count; ++i) c.at[i] = step[i];
  hipLaunchKernelGGL(pp_count_step_kernel, dim3(1), dim3(64), 0, st, c, count);
  return hipGetLastError();
}

hipError_t pp_launch_adamw(int count, int dtype, int bits, void* const* p, const void* const* g,
                           float* const* master, void* const* m, void* const* v,
                           uint8_t* const* m_exp, uint8_t* const* v_exp, const int64_t* numel,
                           const int64_t* step, const int64_t* const* step_dev, double lr,
                           double beta1, double beta2, double eps, double wd,
                           const float* grad_scale, uint32_t seed, uint32_t index, hipStream_t st) {
  AdamWDescs d;
  AdamWArgs a;
  a.b1 = (float)beta1; a.nb1 = (float)(1.0 - beta1);
  a.b2 = (float)beta2; a.nb2 = (float)(1.0 - beta2);
  a.eps = (float)eps; a.decay = (float)(1.0 - lr * wd);
  a.lr = lr; a.beta1 = beta1; a.beta2 = beta2;
  a.seed = seed; a.index = index; a.grad_scale = grad_scale; a.count = count;
  const int per_block = bits == 8 ? 2048 : 1024;
  int64_t blocks = 0;
  d.wide = 0;
  for (int t = 0; t < count; ++t) {
    d.p[t] = p[t]; d.g[t] = g[t]; d.m[t] = m[t]; d.v[t] = v[t];
    d.w[t] = dtype == PP_F32 ? static_cast<float*>(p[t]) : master[t];
    d.me[t] = bits == 8 ? m_exp[t] : nullptr;
    d.ve[t] = bits == 8 ? v_exp[t] : nullptr;
    d.step[t] = step_dev ? step_dev[t] : nullptr;
    d.n[t] = numel[t];
    const int64_t s = d.step[t] ? 1 : step[t];
    d.number[t] = (uint32_t)s;
    d.c1[t] = (float)(lr / (1.0 - int_power(beta1, s)));
    d.c2[t] = (float)(1.0 / std::sqrt(1.0 - int_power(beta2, s)));
    const size_t es = dtype == PP_F32 ? 4 : 2, ms = bits / 8;
    if ((((size_t)p[t] | (size_t)g[t]) % (4 * es) | (size_t)d.w[t] % 16 | ((size_t)m[t] | (size_t)v[t]) % (4 * ms)) == 0)
      d.wide |= 1u << t;
    d.first[t] = (int)blocks;
    blocks += (numel[t] + per_block - 1) / per_block;
  }
  d.first[count] = (int)blocks;
  if (blocks >= (1LL << 24)) return hipErrorInvalidValue;  // 2^32 threads
  const dim3 grid((unsigned)blocks), block(256);
#define PP_ADAMW(T)                                                                             \
  do {                                                                                          \
    if (bits == 8)                                                                              \
      hipLaunchKernelGGL((pp_adamw_kernel<T, true>), grid, block, 0, st, d, a, per_block);      \
    else                                                                                        \
      hipLaunchKernelGGL((pp_adamw_kernel<T, false>), grid, block, 0, st, d, a, per_block);     \
  } while (0)
  if (dtype == PP_F32) PP_ADAMW(float);
  else if (dtype == PP_BF16) PP_ADAMW(pp_bf16);
  else PP_ADAMW(pp_f16);
  return hipGetLastError();
}

hipError_t pp_launch_decode_moment(const uint8_t* code, const uint8_t* exps, void* out, int dtype,
                                   int is_signed, int64_t n, hipStream_t st) {
  const int64_t blocks = (n + 2047) / 2048;
  if (blocks >= (1LL << 24)) return hipErrorInvalidValue;
  const int wide = (size_t)code % 8 == 0 && (size_t)out % 16 == 0;
  const dim3 grid((unsigned)blocks), block(256);
#define PP_DECODE(T)                                                                             \
  do {                                                                                           \
    if (is_signed)                                                                               \
      hipLaunchKernelGGL((pp_decode_moment_kernel<T, true>), grid, block, 0, st, code, exps,     \
                         static_cast<T*>(out), n, wide);                                               \
    else                                                                                         \
      hipLaunchKernelGGL((pp_decode_moment_kernel<T, false>), grid, block, 0, st, code, exps,    \
                         static_cast<T*>(out), n, wide);                                               \
  } while (0)
  if (dtype == PP_F32) PP_DECODE(float);
  else if (dtype == PP_BF16) PP_DECODE(pp_bf16);
  else PP_DECODE(pp_f16);
  return hipGetLastError();
}
