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
// remainder stands for keeps the expected value.  An entry has 8 random bits for that, so the probability is a
// multiple of 1/256, and what is under 1/512 of a unit is rounded away: a code has 8 to 16 units, so a step has to move
// the moment by 2^-12 of it at least.  At b2 = 0.999 v falls by b2^n to a few per cent, and rests while g^2 stays within
// 12 to 24 % of it; with b above 1 - 2^-12 it would stand still, and is refused.  (More random bits: two more hashes for every
// four entries, in a step that the vector units bound, and other codes for the same seed.)  The bits come from a
// hash of (seed, step, tensor, entry), so a step can be repeated.  A positive v never becomes zero: the step
// m / eps that would follow is unbounded.
//
// Bound: HBM.  Everything is read and written once, in 16-byte accesses (4 bytes of codes) that pass the caches
// by: nothing is used again before the next step, and 92 M fp32 weights take 432 us (6.0 TB/s) that way, 478
// through the caches.  A thread takes four entries at a time, a workgroup 1024 or, with the longer 8-bit
// arithmetic, 2048 (fp32 / 32 bits 432 with 1024, 460 with 2048; 226 M at 8 bits with both decodes 854 with 2048, 914 with 4096).
// With 8 bits the vector units are as busy as the memory (75 instructions an entry, and steps on end lower the
// clock: 226 M bf16 weights 530 us the first, 600 to 650 the later): hence one path for ordinary waves, without the
// cases of numbers that are not finite or tiny, and integer maxima over the lanes (5 M bf16 weights 31 -> 27 us,
// 57 M fp32 189 -> 170, 226 M bf16 698 -> 650).
#include <algorithm>
#include <cmath>
#include <type_traits>

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

template <int CTRL>
__device__ __forceinline__ uint32_t dpp_max(uint32_t v) {
  return max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, CTRL, 0xf, 0xf, true));
}
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
  v = dpp_max<0x128>(v);
  v = dpp_max<0x124>(v);
  v = dpp_max<0x122>(v);
  v = dpp_max<0x121>(v);
  const uint32_t a = max((uint32_t)__builtin_amdgcn_readlane((int)v, 0), (uint32_t)__builtin_amdgcn_readlane((int)v, 16));
  const uint32_t b = max((uint32_t)__builtin_amdgcn_readlane((int)v, 32), (uint32_t)__builtin_amdgcn_readlane((int)v, 48));
  return max(a, b);
}

constexpr uint32_t kInfinity = 0x7f800000u;
__device__ __forceinline__ uint32_t size_of(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// the value of a code that is finite: fp32 bits (sign, exponent, 3 bits of mantissa) << 20, times 2^(E - top)
template <int TOP, bool SIGNED>
__device__ __forceinline__ float decode_finite(uint32_t code, int E) {
  const uint32_t bits = SIGNED ? (code & 127u) << 20 | (code & 128u) << 24 : code << 20;
  return ldexpf(__uint_as_float(bits), E - TOP);
}
template <int TOP, bool SIGNED>
__device__ __forceinline__ float decode8(uint32_t code, int E) {
  const bool finite = (SIGNED ? code & 127u : code) != (SIGNED ? 127u : 255u);
  const uint32_t nan = 0x7fc00000u | (SIGNED ? (code & 128u) << 24 : 0u);
  return finite ? decode_finite<TOP, SIGNED>(code, E) : __uint_as_float(nan);
}
// bits in the bytes of m's and v's codes that are not finite
__device__ __forceinline__ uint32_t not_finite(uint32_t mr, uint32_t vr) {
  return (((mr & 0x7f7f7f7fu) + 0x01010101u) | (((vr & 0x7f7f7f7fu) + 0x01010101u) & vr)) & 0x80808080u;
}

template <int TOP, bool SIGNED, bool PLAIN>
__device__ __forceinline__ uint32_t encode8(float x, int E, uint32_t byte) {
  const uint32_t a = size_of(x);
  uint32_t code = (__float_as_uint(ldexpf(__uint_as_float(a), TOP - E)) + (byte << 12) + 2048u) >> 20;
  if (!SIGNED) code = max(code, min(a, 1u));
  if (!PLAIN && a >= kInfinity) code = SIGNED ? 127u : 255u;
  if (SIGNED) code |= (__float_as_uint(x) >> 24) & 128u;
  return code;
}

// Square root of 0 or of x >= 2^-96, correctly rounded: the instruction is off by at most one step, and the sign
// of x - s (s -+ step) tells on which side of the halfway point to either neighbour x lies (Tuckerman's test).
__device__ __forceinline__ float sqrt_plain(float x) {
  const float s = __builtin_amdgcn_sqrtf(x);
  const float less = __uint_as_float(__float_as_uint(s) - 1u), more = __uint_as_float(__float_as_uint(s) + 1u);
  float r = fmaf(-less, s, x) <= 0.0f ? less : s;
  return fmaf(-more, s, x) > 0.0f ? more : r;
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
    uint32_t mr = 0, vr = 0;  // codes
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
        mr = E8::take(static_cast<const uint8_t*>(mp) + e0);
        vr = E8::take(static_cast<const uint8_t*>(vp) + e0);
      } else {
        const typename EF::raw m4 = EF::take(static_cast<const float*>(mp) + e0);
        const typename EF::raw v4 = EF::take(static_cast<const float*>(vp) + e0);
        EF::get(m4, mv);
        EF::get(v4, vv);
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
          mr |= live ? (uint32_t)static_cast<const uint8_t*>(mp)[e] << (8 * j) : 0u;
          vr |= live ? (uint32_t)static_cast<const uint8_t*>(vp)[e] << (8 * j) : 0u;
        } else {
          mv[j] = live ? static_cast<const float*>(mp)[e] : 0.0f;
          vv[j] = live ? static_cast<const float*>(vp)[e] : 0.0f;
        }
      }
    }
    if (EIGHT) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        mv[j] = decode_finite<14, true>(mr >> (8 * j) & 255u, Em);
        vv[j] = decode_finite<30, false>(vr >> (8 * j) & 255u, Ev);
      }
      if (__any(not_finite(mr, vr) != 0u)) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          mv[j] = decode8<14, true>(mr >> (8 * j) & 255u, Em);
          vv[j] = decode8<30, false>(vr >> (8 * j) & 255u, Ev);
        }
      }
    }
    uint32_t most = 0u, least = ~0u;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float gg = gv[j] * gs;
      mv[j] = mv[j] * a.b1 + gg * a.nb1;
      vv[j] = vv[j] * a.b2 + (gg * gg) * a.nb2;
      most = max(most, max(size_of(mv[j]), __float_as_uint(vv[j])));  // (a NaN may be negative: larger still)
      least = min(least, __float_as_uint(vv[j]) - 1u);                // (0 does not count)
    }
    // what is left, once for numbers that are all finite and not tiny, as they nearly always are
    auto finish = [&](auto plain) {
      constexpr bool PLAIN = decltype(plain)::value;
      uint32_t tm = 0u, tv = 0u;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float s = PLAIN ? sqrt_plain(vv[j]) : sqrtf(vv[j]);
        wv[j] = wv[j] * a.decay - (mv[j] / (s * c2 + a.eps)) * c1;
        const uint32_t sm = size_of(mv[j]), sv = size_of(vv[j]);
        tm = max(tm, PLAIN || sm < kInfinity ? sm : 0u);
        tv = max(tv, PLAIN || sv < kInfinity ? sv : 0u);
      }
      if (EIGHT) {
        Em = (int)(wave_max(tm) >> 23);
        Ev = (int)(wave_max(tv) >> 23);
        const uint32_t q = key + 2u * (uint32_t)(e0 >> 2);
        const uint32_t bm = mix32(q), bv = mix32(q + 1u);
        mr = vr = 0u;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          mr |= encode8<14, true, PLAIN>(mv[j], Em, (bm >> (8 * j)) & 255u) << (8 * j);
          vr |= encode8<30, false, PLAIN>(vv[j], Ev, (bv >> (8 * j)) & 255u) << (8 * j);
        }
      }
    };
    if (EIGHT && !__any(most >= kInfinity || least < 0x0f7fffffu))
      finish(std::true_type());
    else
      finish(std::false_type());
    if (EIGHT && (threadIdx.x & 63) == 0) {
      d.me[t][e0 / kBlk] = (uint8_t)Em;
      d.ve[t][e0 / kBlk] = (uint8_t)Ev;
    }
    if (whole) {
      EF::stream(w + e0, EF::put(wv));
      if (sizeof(T) == 2) ET::stream(p + e0, ET::put(wv));
      if (EIGHT) {
        E8::stream(static_cast<uint8_t*>(mp) + e0, mr);
        E8::stream(static_cast<uint8_t*>(vp) + e0, vr);
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
          static_cast<uint8_t*>(mp)[e] = (uint8_t)(mr >> (8 * j));
          static_cast<uint8_t*>(vp)[e] = (uint8_t)(vr >> (8 * j));
        } else {
          static_cast<float*>(mp)[e] = mv[j];
          static_cast<float*>(vp)[e] = vv[j];
        }
      }
    }
  }
}

// Both are ready before what follows: two stores that fill a line between them then leave together.
template <typename R>
__device__ __forceinline__ void keep_both(R& a, R& b) { asm volatile("" : "+v"(a), "+v"(b)); }

// Eight codes a thread and turn, 8 bytes in, 16 or 32 out; the loads of all TURNS are in flight together, and a
// wave's values lie together.
template <typename O, bool SIGNED, int TURNS>
__global__ __launch_bounds__(256) void pp_decode_moment_kernel(const uint8_t* __restrict__ code,
                                                               const uint8_t* __restrict__ exps,
                                                               O* __restrict__ out, int64_t n, int wide) {
  constexpr int kPer = 16 / sizeof(O);  // entries of a store
  typedef PPElems<O, kPer> EO;
  const int64_t first = (((int64_t)blockIdx.x * 256 + (threadIdx.x & ~63)) * TURNS + (threadIdx.x & 63)) * 8;
  typename PPRaw<8>::type c[TURNS];
  int E[TURNS];
#pragma unroll
  for (int k = 0; k < TURNS; ++k) {
    const int64_t e0 = first + k * 512;
    E[k] = e0 < n ? exps[e0 / kBlk] : 0;
    if (wide && e0 + 8 <= n) c[k] = PPElems<uint8_t, 8>::load(code + e0);
  }
#pragma unroll
  for (int k = 0; k < TURNS; ++k) {
    const int64_t e0 = first + k * 512;
    if (wide && e0 + 8 <= n) {
      typename EO::raw r[8 / kPer];
#pragma unroll
      for (int i = 0; i < 8; i += kPer) {
        float x[kPer];
#pragma unroll
        for (int j = 0; j < kPer; ++j)
          x[j] = decode8<SIGNED ? 14 : 30, SIGNED>(c[k][(i + j) / 4] >> (8 * (j & 3)) & 255u, E[k]);
        r[i / kPer] = EO::put(x);
      }
      if (kPer < 8) keep_both(r[0], r[8 / kPer - 1]);
#pragma unroll
      for (int i = 0; i < 8; i += kPer) EO::stream(out + e0 + i, r[i / kPer]);
    } else {
      for (int64_t e = e0; e < n && e < e0 + 8; ++e) out[e] = (O)decode8<SIGNED ? 14 : 30, SIGNED>(code[e], E[k]);
    }
  }
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

// To 16 bits four turns a thread hide the latency of the small loads once there is work for all (226 M codes 125 us, 151
// with one; 100000 codes 3.8 us, 2.7 with one); to fp32 the stores alone keep the memory busy (226 M codes 215 us,
// 265 with four).
constexpr int64_t kManyCodes = 1 << 23;
template <typename O>
static void run_decode(const uint8_t* code, const uint8_t* exps, void* out, int is_signed, int64_t n, hipStream_t st) {
  const int wide = (size_t)code % 8 == 0 && (size_t)out % 16 == 0;
  constexpr int kMost = sizeof(O) == 2 ? 4 : 1;
  const int turns = n >= kManyCodes ? kMost : 1, part = turns * 2048;
  const dim3 grid((unsigned)((n + part - 1) / part)), block(256);
#define PP_DECODE(SIGNED, TURNS)                                                                   \
  hipLaunchKernelGGL((pp_decode_moment_kernel<O, SIGNED, TURNS>), grid, block, 0, st, code, exps, \
                     static_cast<O*>(out), n, wide)
  if (is_signed && turns > 1) PP_DECODE(true, kMost);
  else if (is_signed) PP_DECODE(true, 1);
  else if (turns > 1) PP_DECODE(false, kMost);
  else PP_DECODE(false, 1);
#undef PP_DECODE
}

hipError_t pp_launch_decode_moment(const uint8_t* code, const uint8_t* exps, void* out, int dtype,
                                   int is_signed, int64_t n, hipStream_t st) {
  if (dtype == PP_F32) run_decode<float>(code, exps, out, is_signed, n, st);
  else if (dtype == PP_BF16) run_decode<pp_bf16>(code, exps, out, is_signed, n, st);
  else run_decode<pp_f16>(code, exps, out, is_signed, n, st);
  return hipGetLastError();
}
