// Gated linear recurrence, forward and backward, and its single-token step.
//
//   a_t = sigmoid(f_t);   h_t = a_t h_{t-1} + (1 - a_t) z_t
//
// per channel, z and f [b][l][d] in fp32, bf16 or fp16, the state in fp32.  reset[b][t] != 0 drops
// the state before step t (h_{t-1} := 0: a new document); steps from lengths[b] on do not exist
// (y = 0, gradients 0, nothing read), the state stays as it is.  Backward, with e_t = dL/dh_t:
//
//   e_t = gy_t + u_t;  u_{t-1} = a_t e_t  (0 at a reset; u = gh_last behind the last step)
//   gz_t = e_t (1 - a_t);   gf_t = e_t a_t (1 - a_t) (h_{t-1} - z_t);   gh0 = a_0 e_0
//
// With x = e^-f: a = 1 / (1 + x) and 1 - a = x a, so neither gate loses its small end to cancellation, and
// h_t = a_t h_{t-1} + (x a_t) z_t.  (z + a (h - z) needs no 1 - a, but takes the input's share from a rounded a: nothing
// of it is left from f = 17 on.)  What a itself leaves of a long memory stays: fp32 [2, 16384, 64] from an empty state, f
// normal around 8, 12, 16: the state is off by 1.4e-6, 9.9e-6, 4e-5 of itself, as in elementary fp32 operations (3e-6, 1.2e-5, 4e-5).
//
// Split of the length.  A step is linear in the state, so a stretch of steps is h_out = P h_in + H
// with P the product of its a and H its result from 0.  A wave takes kSteps steps x 64 V channels:
// it loads them once (16 loads of each input in flight), keeps gates and candidates in registers,
// computes (P, H), and, once h_in is known, walks the steps again from registers.  The waves of a
// workgroup are consecutive stretches, joined through LDS; the workgroups of a row (chunks) are
// joined through global memory: each publishes its (P, H) as soon as it has it, then looks back for
// the nearest chunk whose final state is known and applies the (P, H) of those in between, in
// order -- the same fma of each chunk whoever applies it, so results do not depend on timing.  (The single-pass
// scan with decoupled look-back of Merrill and Garland, 2016, for the composition of affine maps.)
//   Waiting is safe: a workgroup draws its chunk from a counter, chunks in the order of the chain,
// so it waits only for workgroups that are running already and that publish before they wait.
//   The published words carry their own readiness (all ones = not yet, the fill before the launch),
// read and written with device-scope atomics; no other data travels between workgroups, so no fence
// (on this chip a release would write back an XCD's L2) is needed.
//   A reset makes P = -0.0, which no product of gates is: it cuts even a state that is NaN.
// The forward of a training step keeps h at the start of every kSteps steps in fp32 (the states in
// between are recomputed from it; y, rounded to 16 bits, would not do for the differences).
//
// Bound: forward 3 and backward 5 values an entry through HBM, each once.  Measured (MI355X, bf16):
// [8, 2048, 2048] forward 50 us (4.2 TB/s with the kept states), backward 74 us (4.6); [1, 100003, 640] 103
// and 148 us.  The rest is the shape of a workgroup: 16 waves of 113 registers are all that a CU holds, so
// its loads, its walks and its waits follow one another.  Counter and look-back are 5 to 10 %, the gates
// nothing (measured without them).  Rows of few channels share waves (folds).
#include <algorithm>

#include "pp_device.h"
#include "pp_lowp.h"

namespace {

constexpr int kSteps = PP_RECURRENCE_STEPS;  // steps of a wave, and between two kept states
constexpr int kMostWaves = 16;               // waves (stretches) of a workgroup
constexpr uint32_t kNotYet = 0xffffffffu;

struct RecArgs {
  int64_t zb, zl, fb, fl, gb, gl;  // strides in elements of z, f and gy over batch and time
  int b, l, d;
  int nchunk, ngroup;  // chunks of a row, groups of 64 V channels (of one row, or folded: of all)
  int chunk;           // steps of a chunk
  int chains;
  const float* h0;
  const int32_t* lengths;
  const uint8_t* reset;
  uint32_t* ticket;
  unsigned long long* part;  // [chain][chunk][64 V]: (P, H) of a chunk
  uint32_t* done;            // [chain][chunk][64 V]: state behind it
};

// e^-f (infinity where f is far below 0)
template <bool EXACT>
__device__ __forceinline__ float gate_exp(float f) {
  const float hi = f * -1.44269502f;
  const float x = __builtin_amdgcn_exp2f(hi);
  if (!EXACT) return x;
  // the rounding of f log2(e) is made good: matters for |f| >> 1 in fp32
  const float lo = fmaf(f, -1.92596299e-8f, fmaf(f, -1.44269502f, -hi));
  return fabsf(hi) < 126.0f ? fmaf(x * 0.693147182f, lo, x) : x;
}
// a and 1 - a, each to its own digits: 1 - a = x a, where x is held below what makes a zero of a (a NaN stays one)
template <bool EXACT>
__device__ __forceinline__ void both_gates(float f, float& a, float& r) {
  const float x = __builtin_elementwise_minimum(gate_exp<EXACT>(f), 0x1p126f);
  a = __builtin_amdgcn_rcpf(1.0f + x);
  r = x * a;
}
// Both gates in one register for later walks: the smaller of the two, its sign telling which it is
// (1 - a for f >= 0, -a else); the other is 1 minus it.
template <bool EXACT>
__device__ __forceinline__ float gate_code(float f) {
  const float x = gate_exp<EXACT>(fabsf(f));
  return copysignf(x * __builtin_amdgcn_rcpf(1.0f + x), f);
}
__device__ __forceinline__ void gates(float q, float& a, float& r) {
  const float small = fabsf(q), big = 1.0f - small;
  const bool neg = __float_as_int(q) < 0;  // (also -0.0, a closed gate)
  a = neg ? small : big;
  r = neg ? big : small;
}

// Holds a value in this very form: without it the compiler keeps what the value was made from, or
// both gates of an earlier walk, in registers of their own, at the cost of half the resident waves.
__device__ __forceinline__ void keep(float& x) { asm volatile("" : "+v"(x)); }
template <int V>
__device__ __forceinline__ void keep_all(float (&q)[kSteps][V]) {
#pragma unroll
  for (int j = 0; j < kSteps; ++j)
#pragma unroll
    for (int v = 0; v < V; ++v) keep(q[j][v]);
}

// state behind a stretch (P, H) from the state before it
__device__ __forceinline__ float through(float P, float H, float h) {
  return __float_as_uint(P) == 0x80000000u ? H : fmaf(P, h, H);
}

__device__ __forceinline__ uint32_t word_of(float x) {
  return x != x ? 0x7fc00000u : __float_as_uint(x);  // one NaN: never kNotYet
}

// The state behind chunk `last` of a chain that begins with chunk `first` (which publishes its state
// without waiting); one wave, V channels a lane, kWindow chunks looked at together.
template <int kWindow, int V>
__device__ __forceinline__ void look_back(const RecArgs& p, int64_t chain, int first, int last,
                                          float (&h)[V]) {
  const uint32_t lane = threadIdx.x & 63;
  const uint32_t* done = p.done + chain * p.nchunk * (64 * V);
  const unsigned long long* part = p.part + chain * p.nchunk * (64 * V);
  int k = last;
  for (bool found = false; !found;) {  // the nearest chunk whose state is known
    uint32_t w[kWindow][V];
#pragma unroll
    for (int j = 0; j < kWindow; ++j)
#pragma unroll
      for (int v = 0; v < V; ++v)
        w[j][v] = __hip_atomic_load(done + (int64_t)max(k - j, first) * (64 * V) + v * 64 + lane, __ATOMIC_RELAXED,
                                    __HIP_MEMORY_SCOPE_AGENT);
#pragma unroll
    for (int j = 0; j < kWindow; ++j) {
      if (found) continue;
      bool ready = true;
#pragma unroll
      for (int v = 0; v < V; ++v) ready = ready && w[j][v] != kNotYet;
      if (__all(ready)) {
        found = true;
        k = max(k - j, first);
#pragma unroll
        for (int v = 0; v < V; ++v) h[v] = __uint_as_float(w[j][v]);
      }
    }
    if (!found) {
      if (k - kWindow < first) {  // not even the first: wait and start again from the near end
        __builtin_amdgcn_s_sleep(2);
        k = last;
      } else {
        k -= kWindow;
      }
    }
  }
  while (k < last) {  // ... and on from there, chunk by chunk
    const int n = min(kWindow, last - k);
    unsigned long long w[kWindow][V];
#pragma unroll
    for (int j = 0; j < kWindow; ++j)
#pragma unroll
      for (int v = 0; v < V; ++v)
        w[j][v] = __hip_atomic_load(part + (int64_t)min(k + 1 + j, last) * (64 * V) + v * 64 + lane,
                                    __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    int used = 0;
#pragma unroll
    for (int j = 0; j < kWindow; ++j) {
      bool ready = j < n && used == j;
#pragma unroll
      for (int v = 0; v < V; ++v) ready = ready && (uint32_t)w[j][v] != kNotYet;
      if (__all(ready)) {
        used = j + 1;
#pragma unroll
        for (int v = 0; v < V; ++v)
          h[v] = through(__uint_as_float((uint32_t)w[j][v]), __uint_as_float((uint32_t)(w[j][v] >> 32)), h[v]);
      }
    }
    k += used;
    if (!used) __builtin_amdgcn_s_sleep(1);
  }
}

template <int V>
__device__ __forceinline__ void publish_part(const RecArgs& p, int64_t chain, int c, const float (&P)[V],
                                             const float (&H)[V]) {
  unsigned long long* at = p.part + (chain * p.nchunk + c) * (64 * V) + (threadIdx.x & 63);
#pragma unroll
  for (int v = 0; v < V; ++v)
    __hip_atomic_store(at + v * 64, (unsigned long long)word_of(P[v]) | (unsigned long long)word_of(H[v]) << 32,
                       __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
template <int V>
__device__ __forceinline__ void publish_done(const RecArgs& p, int64_t chain, int c, const float (&h)[V]) {
  uint32_t* at = p.done + (chain * p.nchunk + c) * (64 * V) + (threadIdx.x & 63);
#pragma unroll
  for (int v = 0; v < V; ++v)
    __hip_atomic_store(at + v * 64, word_of(h[v]), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

__global__ __launch_bounds__(256) void pp_rec_fill_kernel(uint32_t* __restrict__ ws, int64_t words) {
  const int64_t i = (int64_t)blockIdx.x * 1024 + threadIdx.x;
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (i + j * 256 < words) ws[i + j * 256] = i + j * 256 < 4 ? 0u : kNotYet;  // the counter, then the rest
}

// One wave joins the (P, H) of the stretches from, from + step, ... (`waves` of them) into (P, H) of the chunk
// and leaves in the place of each what lies before it.  Four are read ahead: one after the other, each LDS
// access costs its latency, 1 us a chunk (bf16 [1, 100003, 640] forward 103 instead of 92 us).
template <int V>
__device__ __forceinline__ void join_parts(float2 (&part)[kMostWaves][V][64], int waves, int from, int step,
                                           float (&P)[V], float (&H)[V]) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    P[v] = 1.0f;
    H[v] = 0.0f;
  }
  for (int i = 0; i < waves; i += 4) {
    float2 s[4][V];
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int v = 0; v < V; ++v) s[k][v] = part[from + min(i + k, waves - 1) * step][v][lane];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (i + k >= waves) break;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        part[from + (i + k) * step][v][lane] = make_float2(P[v], H[v]);
        H[v] = through(s[k][v].x, s[k][v].y, H[v]);
        P[v] = __float_as_uint(s[k][v].x) == 0x80000000u ? s[k][v].x : P[v] * s[k][v].x;
      }
    }
  }
}

// bits j: step t0 + j starts a document
__device__ __forceinline__ uint32_t reset_bits(const uint8_t* reset, int64_t row, int t0, int n) {
  if (!reset) return 0u;
  const int lane = threadIdx.x & 63;
  const bool on = lane < n && reset[row + t0 + lane] != 0;
  return (uint32_t)__ballot(on);
}

// The same for one lane's row.
__device__ __forceinline__ uint32_t own_reset_bits(const uint8_t* reset, int64_t at, int n) {
  uint32_t bits = 0u;
  if (reset)
    for (int j = 0; j < n; ++j) bits |= (reset[at + j] != 0 ? 1u : 0u) << j;
  return bits;
}

template <bool FOLD>
__device__ __forceinline__ uint32_t cuts(const RecArgs& p, int b, int t0, int n) {
  if (FOLD) return own_reset_bits(p.reset, (int64_t)b * p.l + t0, n);
  return n > 0 ? reset_bits(p.reset, (int64_t)b * p.l, t0, n) : 0u;
}

// this workgroup's chunk (counted along the chain), channel group and row
__device__ __forceinline__ void draw_tile(const RecArgs& p, int* shared, int& c, int& g, int& b) {
  int id = blockIdx.x;
  if (p.nchunk > 1) {
    if (threadIdx.x == 0) *shared = (int)atomicAdd(p.ticket, 1u);
    __syncthreads();
    id = __builtin_amdgcn_readfirstlane(*shared);
  }
  c = id / p.chains;
  b = (id % p.chains) / p.ngroup;
  g = id % p.ngroup;
}

// The walks over the steps of a stretch.  FAST: all steps exist and none drops the state, which is
// nearly always so; the general form costs twice the scalar and vector instructions, and either
// kernel issues for half of its time.  fr, zr, gr: rows as they came; addresses advance by a row.
template <bool FAST, typename T, int V>
__device__ __forceinline__ void load_rows(typename PPElems<T, V>::raw (&fr)[kSteps], const T* fp, int64_t fl,
                                          typename PPElems<T, V>::raw (&zr)[kSteps], const T* zp, int64_t zl,
                                          uint32_t ch, int n) {
#pragma unroll
  for (int j = 0; j < kSteps; ++j) {
    fr[j] = PPElems<T, V>::load_any(fp + ch);
    zr[j] = PPElems<T, V>::load_any(zp + ch);
    if (FAST || j + 1 < n) {  // behind the last: the last again
      fp += fl;
      zp += zl;
    }
  }
}

// hl, pl of each step: the state from 0 at the start of the stretch, the product of its a until then.
template <bool FAST, typename T, int V>
__device__ __forceinline__ void first_walk(const T* zp, int64_t zl, const T* fp, int64_t fl, uint32_t ch, int n,
                                           uint32_t cut, float (&hl)[kSteps][V], float (&pl)[kSteps][V],
                                           float (&P)[V], float (&H)[V]) {
  typedef PPElems<T, V> E;
  typename E::raw fr[kSteps], zr[kSteps];
  load_rows<FAST, T, V>(fr, fp, fl, zr, zp, zl, ch, n);
#pragma unroll
  for (int j = 0; j < kSteps; ++j) {
    float fv[V], zv[V];
    E::get(fr[j], fv);
    E::get(zr[j], zv);
    if (FAST || j < n) {
#pragma unroll
      for (int v = 0; v < V; ++v) {
        float a, r;
        both_gates<sizeof(T) == 4>(fv[v], a, r);
        if (!FAST && (cut >> j & 1)) {
          P[v] = -0.0f;
          H[v] = 0.0f;
        }
        H[v] = fmaf(a, H[v], r * zv[v]);
        P[v] *= a;
      }
    }
#pragma unroll
    for (int v = 0; v < V; ++v) {
      hl[j][v] = H[v];
      pl[j][v] = P[v];
    }
  }
}

// (folded rows are a few bytes long: the cache joins a lane's to lines)
template <bool FOLD, typename T, int V>
__device__ __forceinline__ void put_row(T* at, const float (&x)[V]) {
  if (FOLD)
    PPElems<T, V>::store(at, PPElems<T, V>::put(x));
  else
    PPElems<T, V>::stream_any(at, PPElems<T, V>::put(x));
}

// y of each step from the state h that enters the stretch.
template <bool FAST, bool FOLD, typename T, int V>
__device__ __forceinline__ void second_walk(T* yp, int d, uint32_t ch, int n, int rows,
                                            const float (&hl)[kSteps][V], const float (&pl)[kSteps][V],
                                            const float (&h)[V]) {
#pragma unroll
  for (int j = 0; j < kSteps; ++j) {
    float out[V];
#pragma unroll
    for (int v = 0; v < V; ++v)
      out[v] = FAST ? fmaf(pl[j][v], h[v], hl[j][v]) : j < n ? through(pl[j][v], hl[j][v], h[v]) : 0.0f;
    if (FAST || j < rows) put_row<FOLD, T, V>(yp + ch, out);
    yp += d;
  }
}

// q, gap of each step: its gates and h_{t-1} - z_t; gr: gy; (P, G) of the stretch, backwards.
template <bool FAST, typename T, int V>
__device__ __forceinline__ void first_walk_back(const T* zp, int64_t zl, const T* fp, int64_t fl, const T* gp,
                                                int64_t gl, uint32_t ch, int n, uint32_t cut, float (&h)[V],
                                                float (&q)[kSteps][V], float (&gap)[kSteps][V],
                                                typename PPElems<T, V>::raw (&gr)[kSteps], float (&P)[V],
                                                float (&G)[V]) {
  typedef PPElems<T, V> E;
  typename E::raw fr[kSteps], zr[kSteps];
  load_rows<FAST, T, V>(fr, fp, fl, zr, zp, zl, ch, n);
#pragma unroll
  for (int j = 0; j < kSteps; ++j) {
    gr[j] = E::load_any(gp + ch);
    if (FAST || j + 1 < n) gp += gl;
  }
#pragma unroll
  for (int j = 0; j < kSteps; ++j) {
    float fv[V], zv[V];
    E::get(fr[j], fv);
    E::get(zr[j], zv);
#pragma unroll
    for (int v = 0; v < V; ++v) {
      q[j][v] = gate_code<sizeof(T) == 4>(fv[v]);
      float a, r;
      gates(q[j][v], a, r);
      if (!FAST && (cut >> j & 1)) h[v] = 0.0f;
      gap[j][v] = h[v] - zv[v];
      h[v] = fmaf(a, h[v], r * zv[v]);
      keep(q[j][v]);
      keep(gap[j][v]);
    }
  }
#pragma unroll
  for (int j = kSteps - 1; j >= 0; --j) {
    if (!FAST && j >= n) continue;
    float gv[V];
    E::get(gr[j], gv);
#pragma unroll
    for (int v = 0; v < V; ++v) {
      float a, r;
      gates(q[j][v], a, r);
      G[v] = a * (gv[v] + G[v]);
      P[v] *= a;
      if (!FAST && (cut >> j & 1)) {
        P[v] = -0.0f;
        G[v] = 0.0f;
      }
    }
  }
}

// gz, gf of each step from the gradient u that arrives behind the stretch; u then leaves in front of it.
template <bool FAST, bool FOLD, typename T, int V>
__device__ __forceinline__ void second_walk_back(T* gzp, T* gfp, int d, uint32_t ch, int n, int rows,
                                                 uint32_t cut, const float (&q)[kSteps][V],
                                                 const float (&gap)[kSteps][V],
                                                 const typename PPElems<T, V>::raw (&gr)[kSteps],
                                                 float (&u)[V]) {
  typedef PPElems<T, V> E;
  gzp += (int64_t)(kSteps - 1) * d;
  gfp += (int64_t)(kSteps - 1) * d;
#pragma unroll
  for (int j = kSteps - 1; j >= 0; --j) {
    float oz[V], of[V];
#pragma unroll
    for (int v = 0; v < V; ++v) oz[v] = of[v] = 0.0f;
    if (FAST || j < n) {
      float gv[V];
      E::get(gr[j], gv);
#pragma unroll
      for (int v = 0; v < V; ++v) {
        float a, r;
        gates(q[j][v], a, r);
        const float e = gv[v] + u[v];
        u[v] = a * e;
        oz[v] = e * r;
        of[v] = (u[v] * r) * gap[j][v];
        if (!FAST && (cut >> j & 1)) u[v] = 0.0f;
      }
    }
    if (FAST || j < rows) {
      put_row<FOLD, T, V>(gzp + ch, oz);
      put_row<FOLD, T, V>(gfp + ch, of);
    }
    gzp -= d;
    gfp -= d;
  }
}

// Zeros where a sequence has ended.  (A workgroup that has nothing else to do leaves with them at once: fp16 [16,
// 1531, 1536] with lengths 0 .. 1531 40 us, 44 by way of the walks.)
template <typename T, int V>
__device__ __forceinline__ void zero_rows(T* p, int d, uint32_t ch, int rows) {
  typename PPElems<T, V>::raw zero = {};
  for (int j = 0; j < rows; ++j) PPElems<T, V>::stream_any(p + (int64_t)j * d + ch, zero);
}

// What a lane works on.  FOLD: rows of fewer channels than half a wave share it, a lane's row is its own; a
// sequence that has ended is then a stretch with P = 1, H = 0, and every chain is as long as the tensors.
template <int V, bool FOLD>
struct Place {
  int b;        // row
  uint32_t ch;  // first channel
  bool live;    // (a lane without channels reads the last ones and writes nothing)
  __device__ __forceinline__ Place(const RecArgs& p, int g, int row) {
    const int want = (g * 64 + (int)(threadIdx.x & 63)) * V;
    if (FOLD) {
      live = want < p.b * p.d;
      const int i = min(want, p.b * p.d - 1);
      b = i / p.d;
      ch = i % p.d;
    } else {
      live = want < p.d;
      b = row;
      ch = min(want, p.d - V);  // (an odd last channel is taken with the one before, by two lanes alike)
    }
  }
};

template <typename T, int V, bool FOLD>
__global__ __launch_bounds__(64 * kMostWaves, 4) void pp_rec_fwd_kernel(const T* __restrict__ z,
                                                                 const T* __restrict__ f,
                                                                 T* __restrict__ y,
                                                                 float* __restrict__ h_last,
                                                                 float* __restrict__ starts, RecArgs p) {
  __shared__ float2 part[kMostWaves][V][64];
  __shared__ float carry[V][64];
  __shared__ int drawn;
  int c, g, row;
  draw_tile(p, &drawn, c, g, row);
  const int lane = threadIdx.x & 63, waves = blockDim.x >> 6;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Place<V, FOLD> place(p, g, row);
  const int b = place.b;
  const uint32_t ch = place.ch;
  const bool live = place.live;
  const int own = p.lengths ? max(0, min(p.l, p.lengths[b])) : p.l;  // steps of the row
  const int len = FOLD ? p.l : own;                                   // steps of the chain
  const int t0 = c * p.chunk + wave * kSteps;
  const int n = max(0, min(kSteps, own - t0));        // steps of this wave that exist
  const int rows = max(0, min(kSteps, p.l - t0));     // rows of y to write
  const int64_t chain = FOLD ? g : (int64_t)b * p.ngroup + g;
  const int64_t row0 = (int64_t)b * p.l + t0;
  if (c > 0 && c * p.chunk >= len) {  // (all of the workgroup, and nobody waits for it)
    if (live) zero_rows<T, V>(y + row0 * p.d, p.d, ch, rows);
    return;
  }

  float hl[kSteps][V] = {}, pl[kSteps][V] = {};
  float P[V], H[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    P[v] = 1.0f;
    H[v] = 0.0f;
  }
  const uint32_t cut = cuts<FOLD>(p, b, t0, n);
  const bool fast = n == kSteps && cut == 0;
  const bool straight = FOLD ? __all(fast || n == 0) : fast;  // (the same way for all lanes of a wave)
  if (n > 0) {
    const T* zp = z + b * p.zb + t0 * p.zl;  // (the same for all lanes: scalar addresses)
    const T* fp = f + b * p.fb + t0 * p.fl;
    if (straight)
      first_walk<true, T, V>(zp, p.zl, fp, p.fl, ch, n, cut, hl, pl, P, H);
    else
      first_walk<false, T, V>(zp, p.zl, fp, p.fl, ch, n, cut, hl, pl, P, H);
  }
#pragma unroll
  for (int v = 0; v < V; ++v) part[wave][v][lane] = make_float2(P[v], H[v]);
  __syncthreads();
  const bool alone = p.nchunk == 1;
  if (wave == 0) {  // the state before this chunk
    float h[V];
    if (c == 0) {
#pragma unroll
      for (int v = 0; v < V; ++v) h[v] = p.h0 && live ? p.h0[(int64_t)b * p.d + ch + v] : 0.0f;
    }
    float CP[V], CH[V];
    join_parts<V>(part, waves, 0, 1, CP, CH);
    if (!alone && len > 0) {
      const bool more = (c + 1) * p.chunk < len;  // someone waits for it
      if (c > 0) {
        if (more) publish_part<V>(p, chain, c, CP, CH);
        look_back<8, V>(p, chain, 0, c - 1, h);
      }
      if (more) {
        float out[V];
#pragma unroll
        for (int v = 0; v < V; ++v) out[v] = through(CP[v], CH[v], h[v]);
        publish_done<V>(p, chain, c, out);
      }
    }
#pragma unroll
    for (int v = 0; v < V; ++v) carry[v][lane] = h[v];
  }
  __syncthreads();
  float h[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const float2 before = part[wave][v][lane];
    h[v] = through(before.x, before.y, carry[v][lane]);
  }
  if (!live) return;
  if (starts && n > 0) {
    float* at = starts + ((int64_t)b * ((p.l + kSteps - 1) / kSteps) + t0 / kSteps) * p.d;
#pragma unroll
    for (int v = 0; v < V; ++v) at[ch + v] = h[v];
  }
  T* yp = y + row0 * p.d;
  if (fast)
    second_walk<true, FOLD, T, V>(yp, p.d, ch, n, rows, hl, pl, h);
  else
    second_walk<false, FOLD, T, V>(yp, p.d, ch, n, rows, hl, pl, h);
  if (FOLD ? rows > 0 && t0 + rows == p.l : (n > 0 && t0 + n == len) || (len == 0 && c == 0 && wave == 0)) {
#pragma unroll
    for (int v = 0; v < V; ++v) h_last[(int64_t)b * p.d + ch + v] = through(P[v], H[v], h[v]);
  }
}

// Chunks are counted from the end of the (allocated) row: chunk c of the chain is row chunk
// nchunk - 1 - c; those behind the end of a shorter row only write zeros.
template <typename T, int V, bool FOLD>
__global__ __launch_bounds__(64 * kMostWaves, 4) void pp_rec_bwd_kernel(
    const T* __restrict__ z, const T* __restrict__ f, const float* __restrict__ starts,
    const T* __restrict__ gy, const float* __restrict__ gh, T* __restrict__ gz, T* __restrict__ gf,
    float* __restrict__ gh0, RecArgs p) {
  typedef PPElems<T, V> E;
  __shared__ float2 part[kMostWaves][V][64];
  __shared__ float carry[V][64];
  __shared__ int drawn;
  int c, g, row;
  draw_tile(p, &drawn, c, g, row);
  const int lane = threadIdx.x & 63, waves = blockDim.x >> 6;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Place<V, FOLD> place(p, g, row);
  const int b = place.b;
  const uint32_t ch = place.ch;
  const bool live = place.live;
  const int own = p.lengths ? max(0, min(p.l, p.lengths[b])) : p.l;
  const int len = FOLD ? p.l : own;
  const int chunk0 = (p.nchunk - 1 - c) * p.chunk;  // first step of the chunk
  const int t0 = chunk0 + wave * kSteps;
  const int n = max(0, min(kSteps, own - t0));
  const int rows = max(0, min(kSteps, p.l - t0));
  const int64_t chain = FOLD ? g : (int64_t)b * p.ngroup + g;
  const int64_t row0 = (int64_t)b * p.l + t0;
  if (chunk0 > 0 && chunk0 >= len) {
    if (live) {
      zero_rows<T, V>(gz + row0 * p.d, p.d, ch, rows);
      zero_rows<T, V>(gf + row0 * p.d, p.d, ch, rows);
    }
    return;
  }

  float q[kSteps][V], gap[kSteps][V];  // gates, h_{t-1} - z_t
  typename E::raw gr[kSteps];
  float P[V], G[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    P[v] = 1.0f;
    G[v] = 0.0f;
  }
  const uint32_t cut = cuts<FOLD>(p, b, t0, n);
  const bool fast = n == kSteps && cut == 0;
  const bool straight = FOLD ? __all(fast || n == 0) : fast;
  if (n > 0) {
    const T* zp = z + b * p.zb + t0 * p.zl;  // (the same for all lanes: scalar addresses)
    const T* fp = f + b * p.fb + t0 * p.fl;
    const T* gp = gy + b * p.gb + t0 * p.gl;
    const float* sp = starts + ((int64_t)b * ((p.l + kSteps - 1) / kSteps) + t0 / kSteps) * p.d;
    float h[V];
#pragma unroll
    for (int v = 0; v < V; ++v) h[v] = sp[ch + v];
    if (straight)
      first_walk_back<true, T, V>(zp, p.zl, fp, p.fl, gp, p.gl, ch, n, cut, h, q, gap, gr, P, G);
    else
      first_walk_back<false, T, V>(zp, p.zl, fp, p.fl, gp, p.gl, ch, n, cut, h, q, gap, gr, P, G);
  }
#pragma unroll
  for (int v = 0; v < V; ++v) part[wave][v][lane] = make_float2(P[v], G[v]);
  __syncthreads();
  if (wave == 0) {  // the gradient that arrives behind this chunk
    float u[V];
    const int first = p.nchunk - (len + p.chunk - 1) / p.chunk;  // the chain's chunk with the last step
    if (c <= first) {
#pragma unroll
      for (int v = 0; v < V; ++v) u[v] = gh && live ? gh[(int64_t)b * p.d + ch + v] : 0.0f;
    }
    float CP[V], CG[V];
    join_parts<V>(part, waves, waves - 1, -1, CP, CG);
    if (chunk0 < len && p.nchunk > 1) {
      const bool more = chunk0 > 0;
      if (c > first) {
        if (more) publish_part<V>(p, chain, c, CP, CG);
        look_back<4, V>(p, chain, first, c - 1, u);
      }
      if (more) {
        float out[V];
#pragma unroll
        for (int v = 0; v < V; ++v) out[v] = through(CP[v], CG[v], u[v]);
        publish_done<V>(p, chain, c, out);
      }
    }
#pragma unroll
    for (int v = 0; v < V; ++v) carry[v][lane] = u[v];
  }
  __syncthreads();
  float u[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const float2 behind = part[wave][v][lane];
    u[v] = through(behind.x, behind.y, carry[v][lane]);
  }
  if (!live) return;
  keep_all<V>(q);
  T* gzp = gz + row0 * p.d;
  T* gfp = gf + row0 * p.d;
  if (fast)
    second_walk_back<true, FOLD, T, V>(gzp, gfp, p.d, ch, n, rows, cut, q, gap, gr, u);
  else
    second_walk_back<false, FOLD, T, V>(gzp, gfp, p.d, ch, n, rows, cut, q, gap, gr, u);
  if (gh0 && chunk0 == 0 && wave == 0) {
#pragma unroll
    for (int v = 0; v < V; ++v) gh0[(int64_t)b * p.d + ch + v] = u[v];
  }
}

template <typename T, int V>
__global__ __launch_bounds__(256) void pp_rec_step_kernel(const T* __restrict__ z, int64_t zb,
                                                          const T* __restrict__ f, int64_t fb,
                                                          float* __restrict__ h, int64_t hb,
                                                          T* __restrict__ y, int b, int d) {
  typedef PPElems<T, V> E;
  typedef PPElems<float, V> EH;
  const int wide = d / V;  // (V divides d)
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= (int64_t)b * wide) return;
  const int64_t row = i / wide;
  const int ch = (int)(i % wide) * V;
  float zv[V], fv[V], hv[V];
  E::get(E::load(z + row * zb + ch), zv);
  E::get(E::load(f + row * fb + ch), fv);
  EH::get(EH::load(h + row * hb + ch), hv);
#pragma unroll
  for (int v = 0; v < V; ++v) {
    float a, r;
    gates(gate_code<sizeof(T) == 4>(fv[v]), a, r);
    hv[v] = fmaf(a, hv[v], r * zv[v]);
  }
  EH::store(h + row * hb + ch, EH::put(hv));
  E::store(y + row * d + ch, E::put(hv));
}

// V elements from every address that `strides` steps away from `at` are one aligned access
bool fits(int v, size_t size, std::initializer_list<const void*> at, std::initializer_list<int64_t> strides) {
  for (const void* q : at)
    if ((size_t)q % (v * size)) return false;
  for (int64_t s : strides)
    if (s % v) return false;
  return true;
}

// groups of 64 v channels: of a row, or of all rows together where they share waves
int groups(int b, int d, int v, bool fold) { return (int)(((fold ? (int64_t)b * d : d) + 64 * v - 1) / (64 * v)); }

// A short row is one chunk, others are cut into chunks of kMostWaves stretches: with half of that the
// long chains wait twice as often (bf16 [1, 100003, 640] forward + backward 289 against 241 us, fp32
// [4, 1024, 2048] 75 against 64), and where nothing waits little is gained ([2, 8192, 2048] 129, 131).
void plan(RecArgs& p, int v, bool fold, void* ws) {
  p.ngroup = groups(p.b, p.d, v, fold);
  p.chains = fold ? p.ngroup : p.ngroup * p.b;
  p.chunk = kSteps * std::min(kMostWaves, (p.l + kSteps - 1) / kSteps);
  p.nchunk = (p.l + p.chunk - 1) / p.chunk;
  p.ticket = static_cast<uint32_t*>(ws);
  const int64_t n = (int64_t)p.chains * p.nchunk * 64 * v;
  p.part = reinterpret_cast<unsigned long long*>(p.ticket + 4);
  p.done = reinterpret_cast<uint32_t*>(p.part + n);
}

void fill(const RecArgs& p, int v, hipStream_t st) {
  if (p.nchunk == 1) return;
  const int64_t words = 4 + (int64_t)p.chains * p.nchunk * 64 * v * 3;
  hipLaunchKernelGGL(pp_rec_fill_kernel, dim3((unsigned)((words + 1023) / 1024)), dim3(256), 0, st,
                     p.ticket, words);
}

// Two channels a lane, 4 bytes an access, in 16-bit types where that fills the lanes (fp32 has not the registers:
// it spills), and where a wave for every 64 channels and 16 steps would be more than 16 for each of 256 CUs: more
// and smaller waves win until then (bf16 forward + backward, one against two channels: [8, 2000, 256], 4000 waves,
// 30 and 32 us, [10, 2000, 256], 5000 waves, 39 and 34, [1, 100003, 640] 302 and 241; [1, 100003, 64] 96 and 119).
// Pairs start at any element: odd rows too ([8, 2048, 2047] 162 us, 198 by single elements).
bool pairs(int dtype, int b, int l, int d) {
  return dtype != PP_F32 && d > 64 &&
         (int64_t)b * ((d + 63) / 64) * ((l + kSteps - 1) / kSteps) > 16 * 256;
}

// Rows of up to 32 channels share waves where a wave a row would be more than 16 for each of 256 CUs and shared waves
// are still enough to hide the loads of single rows (us, bf16 forward + backward, shared and a wave a row: [457, 131072,
// 1] 1377 and 11798, [256, 5000, 16] 103 and 287, [256, 5000, 32] 185 and 295, [64, 2000, 4], 500 waves, 34 and 43;
// [300, 300, 3], 285 waves, 48 and 45, [128, 1000, 2], 252 waves, 58 and 42).
bool folds(int b, int l, int d) {
  const int64_t stretches = (l + kSteps - 1) / kSteps;
  return d <= 32 && b * stretches > 16 * 256 && ((int64_t)b * d + 63) / 64 * stretches >= 384;
}

template <typename T, int V, bool FOLD>
void run_fwd(const void* z, const void* f, void* y, float* h_last, float* starts, RecArgs p, void* ws,
             hipStream_t st) {
  plan(p, V, FOLD, ws);
  fill(p, V, st);
  hipLaunchKernelGGL((pp_rec_fwd_kernel<T, V, FOLD>), dim3((unsigned)p.nchunk * p.chains),
                     dim3(4 * p.chunk), 0, st, static_cast<const T*>(z), static_cast<const T*>(f),
                     static_cast<T*>(y), h_last, starts, p);
}
template <typename T, int V, bool FOLD>
void run_bwd(const void* z, const void* f, const float* starts, const void* gy, const float* gh,
             void* gz, void* gf, float* gh0, RecArgs p, void* ws, hipStream_t st) {
  plan(p, V, FOLD, ws);
  fill(p, V, st);
  hipLaunchKernelGGL((pp_rec_bwd_kernel<T, V, FOLD>), dim3((unsigned)p.nchunk * p.chains),
                     dim3(4 * p.chunk), 0, st, static_cast<const T*>(z), static_cast<const T*>(f),
                     starts, static_cast<const T*>(gy), gh, static_cast<T*>(gz), static_cast<T*>(gf),
                     gh0, p);
}
template <typename T, int V>
void run_step(const void* z, int64_t zb, const void* f, int64_t fb, float* h, int64_t hb, void* y, int b,
              int d, hipStream_t st) {
  const int64_t n = (int64_t)b * (d / V);
  hipLaunchKernelGGL((pp_rec_step_kernel<T, V>), dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st,
                     static_cast<const T*>(z), zb, static_cast<const T*>(f), fb, h, hb,
                     static_cast<T*>(y), b, d);
}

}  // namespace

#define PP_REC_TYPES(CALL)                    \
  do {                                        \
    if (dtype == PP_F32) CALL(float);         \
    else if (dtype == PP_BF16) CALL(pp_bf16); \
    else CALL(pp_f16);                        \
    return hipGetLastError();                 \
  } while (0)

size_t pp_rec_workspace_bytes(int b, int l, int d) {
  if (l <= kMostWaves * kSteps) return 0;
  const size_t chunk = kMostWaves * kSteps, nchunk = ((size_t)l + chunk - 1) / chunk;
  // (without the type: room for two channels a lane)
  const size_t lanes = folds(b, l, d) ? 64 * (size_t)groups(b, d, 1, true) : 128 * (size_t)groups(b, d, 2, false) * b;
  return 16 + lanes * nchunk * 12;
}

hipError_t pp_launch_rec_fwd(const void* z, int64_t zb, int64_t zl, const void* f, int64_t fb,
                             int64_t fl, int dtype, const float* h0, const int32_t* lengths,
                             const uint8_t* reset, void* y, float* h_last, float* starts, void* ws,
                             int b, int l, int d, hipStream_t st) {
  const RecArgs p = {zb, zl, fb, fl, 0, 0, b, l, d, 0, 0, 0, 0, h0, lengths, reset, nullptr, nullptr, nullptr};
  const bool two = pairs(dtype, b, l, d);
#define PP_CALL(T)                                                                      \
  do {                                                                                  \
    if (folds(b, l, d))                                                                 \
      run_fwd<T, 1, true>(z, f, y, h_last, starts, p, ws, st);                          \
    else if (sizeof(T) == 2 && two)                                                     \
      run_fwd<T, sizeof(T) == 2 ? 2 : 1, false>(z, f, y, h_last, starts, p, ws, st);    \
    else                                                                                \
      run_fwd<T, 1, false>(z, f, y, h_last, starts, p, ws, st);                         \
  } while (0)
  PP_REC_TYPES(PP_CALL);
#undef PP_CALL
}

hipError_t pp_launch_rec_bwd(const void* z, int64_t zb, int64_t zl, const void* f, int64_t fb,
                             int64_t fl, int dtype, const int32_t* lengths, const uint8_t* reset,
                             const float* starts, const void* gy, int64_t gb, int64_t gl,
                             const float* gh_last, void* gz, void* gf, float* gh0, void* ws, int b,
                             int l, int d, hipStream_t st) {
  const RecArgs p = {zb, zl, fb, fl, gb, gl, b, l, d, 0, 0, 0, 0, nullptr, lengths, reset, nullptr, nullptr, nullptr};
  const bool two = pairs(dtype, b, l, d);
#define PP_CALL(T)                                                           \
  do {                                                                       \
    if (folds(b, l, d))                                                      \
      run_bwd<T, 1, true>(z, f, starts, gy, gh_last, gz, gf, gh0, p, ws, st); \
    else if (sizeof(T) == 2 && two)                                          \
      run_bwd<T, sizeof(T) == 2 ? 2 : 1, false>(z, f, starts, gy, gh_last, gz, gf, gh0, p, ws, st); \
    else                                                                     \
      run_bwd<T, 1, false>(z, f, starts, gy, gh_last, gz, gf, gh0, p, ws, st); \
  } while (0)
  PP_REC_TYPES(PP_CALL);
#undef PP_CALL
}

hipError_t pp_launch_rec_step(const void* z, int64_t zb, const void* f, int64_t fb, int dtype,
                              float* h, int64_t hb, void* y, int b, int d, hipStream_t st) {
  const size_t s = dtype == PP_F32 ? 4 : 2;
  const bool two = fits(2, s, {z, f, y}, {zb, fb, (int64_t)d}) && fits(2, 4, {h}, {hb});
#define PP_CALL(T)                                       \
  do {                                                   \
    if (two)                                             \
      run_step<T, 2>(z, zb, f, fb, h, hb, y, b, d, st);  \
    else                                                 \
      run_step<T, 1>(z, zb, f, fb, h, hb, y, b, d, st);  \
  } while (0)
  PP_REC_TYPES(PP_CALL);
#undef PP_CALL
}
