// Token log-probabilities and the clipped policy loss with a KL term, from logits.
//
//   lp = logits[token] - logsumexp(logits);  rho = exp(lp - old)
//   term = -min(rho A, clip(rho, 1 - low, 1 + high) A) + beta (exp(ref - lp) - (ref - lp) - 1)
//   loss = sum_t w_t term_t,  w = mask / #tokens  or  mask / (#tokens of the sequence * #sequences)
//   dloss/dlogits = c (onehot(token) - softmax),  c = w (-A rho [not clipped] + beta (1 - exp(ref - lp)))
//
// The sum of exp(x - max) is taken in fp32 a lane and in 64 bits over the lanes; lp = (x - max) - log sum
// and its differences to old and ref are formed in 64 bits (a few operations a row: the log is that of the
// mantissa in fp32, and the exponent times log 2), since a ratio is the exponential of a small difference of
// numbers around -10, whose fp32 spacing alone would be 1e-6 of it.  The backward keeps (max, sum) in fp32.
// A masked token's logits, token, old, ref and advantage are not read; its gradient row is zeros.
//
// Bound: the logits are read once and the gradient written once.  A row that fits is therefore held
// in registers, as it came, between the statistics and the gradient (pp_policy_fused_kernel: a wave or
// 256 to 1024 threads a row, up to 16 vectors of 16 bytes a thread); a longer one is read twice
// (pp_row_terms_kernel, then pp_row_grad_kernel, which are also the score and the backward alone).
// Rows start anywhere: up to 7 elements before the first 16-byte boundary and behind the last are
// taken one by one ("edge"), all others as aligned vectors.
// Measured (MI355X, bf16): training [16, 384, 50021], 58 % of the tokens counting, 199 us (4.9 TB/s), [4, 1500,
// 131072] 454 us (5.1), in registers against 303 and 594 read twice; score [8, 511, 32000] 27 us (5.5).  Between
// load and store a row needs two exponentials an entry, which is 40 % of the time and hides only behind
// the other rows of the CU: two at up to 65536 entries, one above.
#include <algorithm>
#include <cmath>

#include "pp_device.h"
#include "pp_lowp.h"

namespace {

constexpr float kLog2e = 1.44269502f, kLog2eAbove = 1.44269514f, kLn2 = 0.693147182f, kLn2Rest = -1.90465421e-9f;

struct PolArgs {
  const int64_t* tokens;
  const uint8_t* mask;
  int64_t lb, lt, gb, gt;  // strides of the logits and of their gradient over batch and time
  int first, rows, t, v;   // of this launch: rows first .. rows - 1
  __device__ __forceinline__ int64_t logits_at(int row) const { return (row / t) * lb + (row % t) * lt; }
  __device__ __forceinline__ int64_t grad_at(int row) const { return (row / t) * gb + (row % t) * gt; }
};
struct PolTerms {
  const float* old;
  const float* adv;
  const float* ref;
  int64_t ab, at;       // strides of adv
  float beta;
  double low, high;          // 1 - clip_low, 1 + clip_high
  double log_low, log_high;  // their logarithms (NaN of a negative: no ratio is below)
  const float* weight;  // of a token, by sequence; NULL: `every`
  float every;
  double* loss;         // [padded rows]: weighted
  float* figures;       // [2][padded rows]: weighted kl, clipped
  int padded;
};

// Vectors and edge elements of a row at x.
template <typename T>
struct Span {
  static constexpr int kVec = 16 / sizeof(T);
  int head, vecs, edge;
  __device__ __forceinline__ Span(const T* x, int v) {
    const int off = (int)((size_t)x & 15) / (int)sizeof(T);
    head = min(v, off ? kVec - off : 0);
    vecs = (v - head) / kVec;
    edge = v - vecs * kVec;  // head and tail
  }
  // element number of edge i < edge
  __device__ __forceinline__ int edge_at(int i) const { return i < head ? i : i + vecs * kVec; }
};

// e^d, off by up to 2^-24 |d| of itself (the product is rounded, and log2(e) too).
__device__ __forceinline__ float exp_of(float d, float log2e = kLog2e) { return __builtin_amdgcn_exp2f(d * log2e); }
// In a sum over classes the products' roundings cancel, that of log2(e) does not (sums of normal logits were off by 6e-8 of
// themselves, all to one side).  So a sixth of the lanes take the next number above: 10 of 64 of them bring the mean
// of all to log2(e) within 5e-10 of it, at no instruction a class.
__device__ __forceinline__ float lane_log2e() {
  return (0x0820820820820820ull >> (threadIdx.x & 63)) & 1 ? kLog2eAbove : kLog2e;  // lanes 5, 11, ... 59
}
// The same to 2 units of its own size: an fp32 gradient has a value for each class.
__device__ __forceinline__ float exp_digits(float d) {
  d = __builtin_elementwise_maximum(d, -200.0f);  // (0 from there on; a NaN stays one)
  const float hi = d * kLog2e, x = __builtin_amdgcn_exp2f(hi);
  return fmaf(x, fmaf(-hi, kLn2Rest, fmaf(-hi, kLn2, d)), x);
}

// What a lane has seen: the max, and the sum of exp(x - max), brought to a new max by one factor a vector.
struct Running {
  float max = -3.40282347e38f, sum = 0.0f;  // (finite, so that -inf - max is -inf and not NaN)
  const float log2e = lane_log2e();
  template <int N>
  __device__ __forceinline__ void add(const float (&e)[N]) {
    float top = max;
#pragma unroll
    for (int j = 0; j < N; ++j) top = fmaxf(top, e[j]);
    sum *= exp_of(max - top, log2e);
    max = top;
#pragma unroll
    for (int j = 0; j < N; ++j) sum += exp_of(e[j] - top, log2e);
  }
  __device__ __forceinline__ void add(float e) {
    const float one[1] = {e};
    add(one);
  }
};

// The same of the THREADS lanes that share a row, the sum in 64 bits over the lanes.  One exchange through
// LDS: each wave its pair, then as many neighbouring lanes as there are waves join those.
struct MaxSum {
  float max;
  double sum;
};
__device__ __forceinline__ float wave_max(float v) {
  v = pp_dpp_max<0x128>(v);
  v = pp_dpp_max<0x124>(v);
  v = pp_dpp_max<0x122>(v);
  v = pp_dpp_max<0x121>(v);
  return fmaxf(fmaxf(pp_readlane_f(v, 0), pp_readlane_f(v, 16)), fmaxf(pp_readlane_f(v, 32), pp_readlane_f(v, 48)));
}
template <int THREADS>
__device__ __forceinline__ MaxSum join_lanes(const Running& run, MaxSum* red) {
  MaxSum r;
  r.max = wave_max(run.max);
  float v = run.sum * exp_digits(run.max - r.max);
  v = pp_dpp_add<0x128>(v);
  v = pp_dpp_add<0x124>(v);
  v = pp_dpp_add<0x122>(v);
  v = pp_dpp_add<0x121>(v);
  r.sum = ((double)pp_readlane_f(v, 0) + (double)pp_readlane_f(v, 16)) +
          ((double)pp_readlane_f(v, 32) + (double)pp_readlane_f(v, 48));
  if (THREADS > 64) {
    constexpr int kWaves = THREADS / 64;
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = r;
    __syncthreads();
    const MaxSum mine = red[threadIdx.x % kWaves];
    r.max = wave_max(mine.max);
    r.sum = mine.sum * (double)exp_digits(mine.max - r.max);
#pragma unroll
    for (int o = kWaves / 2; o; o >>= 1) r.sum += __shfl_xor(r.sum, o);
  }
  return r;
}

// log of a sum: exponent and mantissa apart, the mantissa between sqrt(1/2) and sqrt(2), so that nothing cancels where the
// sum is near 1 (a certain token: 0 for 1, and never less)
__device__ __forceinline__ double log_of(double sum) {
  const float f = (float)sum;
  const float low = (float)((sum - (double)f) / sum);  // what fp32 rounds off (NaN for 0 and infinity)
  int e = __builtin_amdgcn_frexp_expf(f);
  float m = __builtin_amdgcn_frexp_mantf(f);
  if (m < 0.707106781f) {
    m *= 2.0f;
    e -= 1;
  }
  const double l = (double)e * 0.69314718055994531 + (double)logf(m);
  return low == low ? l + (double)low : l;
}

// A row's max, the sum of exp(x - max) and its log.
struct RowStats {
  float max, sum;
  double log_sum;
  __device__ __forceinline__ explicit RowStats(const MaxSum& r) : max(r.max), sum((float)r.sum), log_sum(log_of(r.sum)) {}
  // (the sum, not its log: a share from a log around 10 that is rounded to fp32 would be off by 8 such roundings)
  __device__ __forceinline__ float2 kept() const { return make_float2(max, sum); }
  __device__ __forceinline__ double lp(float x) const { return ((double)x - (double)max) - log_sum; }
};

// The token's logit; NaN where there is no such class: the loss says so.
template <typename T>
__device__ __forceinline__ float token_logit(const T* __restrict__ x, int64_t token, int v) {
  return token >= 0 && token < v ? (float)x[token] : __uint_as_float(0x7fc00000u);
}

// The terms of one token; returns the gradient's coefficient.
__device__ __forceinline__ float policy_terms(const PolArgs& p, const PolTerms& q, int row, double lp,
                                              bool writer) {
  const int b = row / p.t, t = row % p.t;
  const float w = q.weight ? q.weight[b] : q.every, adv = q.adv[b * q.ab + t * q.at];
  const double step = lp - (double)q.old[row];
  const float rho = expf((float)step);
  // (in 64 bits: a ratio of fp32 lies on a border that it is beyond by half a unit)
  const bool clipped = adv >= 0.0f ? step > q.log_high : step < q.log_low;
  float c = clipped ? 0.0f : -adv * rho, kl = 0.0f;
  float loss = c;  // (of a clipped token: without its ratio)
  if (q.ref) {
    const float delta = (float)((double)q.ref[row] - lp), grow = expm1f(delta);
    kl = grow - delta;
    loss += q.beta * kl;
    c -= q.beta * grow;
  }
  if (writer) {
    // Ratios are rounded by chance; a border is the same for all the tokens it holds, and advantages repeat: their product in
    // 64 bits, or all would be off alike, by 2e-8 of it, which a loss shows where its terms cancel.
    double term = (double)(loss * w);
    if (clipped) term -= (adv >= 0.0f ? q.high : q.low) * (double)adv * (double)w;
    q.loss[row] = term;
    q.figures[row] = kl * w;
    q.figures[q.padded + row] = clipped ? w : 0.0f;
  }
  return c * w;
}
__device__ __forceinline__ void no_terms(const PolTerms& q, int row) {
  q.loss[row] = 0.0;
  q.figures[row] = q.figures[q.padded + row] = 0.0f;
}

template <typename T, int THREADS>
__device__ __forceinline__ void zero_row(T* __restrict__ g, int v, int tid) {
  typedef PPElems<T, Span<T>::kVec> E;
  const Span<T> s(g, v);
  typename E::raw zero = {};
  for (int i = tid; i < s.vecs; i += THREADS) E::stream(g + s.head + (int64_t)i * s.kVec, zero);
  if (tid < s.edge) g[s.edge_at(tid)] = (T)0.0f;
}

// The statistics of a row by one pass over it, kAhead vectors in flight.
template <typename T, int THREADS>
__device__ __forceinline__ RowStats stream_stats(const T* __restrict__ x, int v, int tid, MaxSum* red) {
  constexpr int kVec = Span<T>::kVec, kAhead = 4;
  typedef PPElems<T, kVec> E;
  const Span<T> s(x, v);
  const T* body = x + s.head;
  Running run;
  int i = tid;
  for (; i + (kAhead - 1) * THREADS < s.vecs; i += kAhead * THREADS) {
    typename E::raw r[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) r[k] = E::take(body + (int64_t)(i + k * THREADS) * kVec);
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      float e[kVec];
      E::get(r[k], e);
      run.add(e);
    }
  }
  for (; i < s.vecs; i += THREADS) {
    float e[kVec];
    E::get(E::take(body + (int64_t)i * kVec), e);
    run.add(e);
  }
  if (tid < s.edge) run.add((float)x[s.edge_at(tid)]);
  return RowStats(join_lanes<THREADS>(run, red));
}

// stats and lp, or stats, terms and coef, of each row.  THREADS lanes a row, 256 a workgroup.
template <typename T, int THREADS, bool POLICY>
__global__ __launch_bounds__(256) void pp_row_terms_kernel(const T* __restrict__ logits, PolArgs p,
                                                           PolTerms q, float2* __restrict__ stats,
                                                           float* __restrict__ out) {
  __shared__ MaxSum red[4];
  const int tid = threadIdx.x % THREADS;
  const int row = p.first + blockIdx.x * (256 / THREADS) + threadIdx.x / THREADS;
  if (row >= p.rows) return;
  if (p.mask && !p.mask[row]) {
    if (tid == 0) {
      if (stats) stats[row] = make_float2(0.0f, 0.0f);
      if (out) out[row] = 0.0f;
      if (POLICY) no_terms(q, row);
    }
    return;
  }
  const T* x = logits + p.logits_at(row);
  const RowStats st = stream_stats<T, THREADS>(x, p.v, tid, red);
  if (tid == 0) {
    const double lp = st.lp(token_logit(x, p.tokens[row], p.v));
    if (stats) stats[row] = st.kept();
    if (POLICY) {
      const float c = policy_terms(p, q, row, lp, true);
      if (out) out[row] = c;
    } else {
      out[row] = (float)lp;
    }
  }
}

// exp(x - max) for a gradient in T: fp32 keeps the digits, 16 bits have no room for them.  That costs fp32 up to 2 %
// ([8, 512, v]: v = 4000 37.4 -> 38.1 us, 9001 65.5 -> 65.6, 50021 333 -> 337, 65536 405 -> 410).  In the sums it would
// cost another 2 to 4 %, there in 16 bits 2 to 30 %: lane_log2e instead.
template <typename T>
__device__ __forceinline__ float share_of(float d) {
  return sizeof(T) == 4 ? exp_digits(d) : exp_of(d);
}

// One vector of the gradient: k exp(x - max), and c more at the token.
template <typename T>
__device__ __forceinline__ typename PPElems<T, Span<T>::kVec>::raw grad_vec(
    const typename PPElems<T, Span<T>::kVec>::raw& r, float m, float k, float c, int token_in) {
  constexpr int kVec = Span<T>::kVec;
  typedef PPElems<T, kVec> E;
  float e[kVec];
  E::get(r, e);
#pragma unroll
  for (int j = 0; j < kVec; ++j) e[j] = k * share_of<T>(e[j] - m);
  if ((unsigned)token_in < (unsigned)kVec) {
#pragma unroll
    for (int j = 0; j < kVec; ++j) e[j] += j == token_in ? c : 0.0f;
  }
  return E::put(e);
}

// grad = gout * coef * (onehot - softmax).  done_if_one: the gradient for gout = 1 is in `grad`
// already (the forward of the loss wrote it), so that only another gout needs the work; it starts
// from the logits again, since scaling the stored 16-bit values would round twice and would not
// bring back what underflowed at gout = 1 (a loss scaled for fp16).
template <typename T, int THREADS>
__global__ __launch_bounds__(256) void pp_row_grad_kernel(const T* __restrict__ logits, PolArgs p,
                                                          const float2* __restrict__ stats,
                                                          const float* __restrict__ coef,
                                                          const float* __restrict__ gout,
                                                          int done_if_one, T* __restrict__ grad) {
  constexpr int kVec = Span<T>::kVec;
  typedef PPElems<T, kVec> E;
  const float go = gout ? *gout : 1.0f;
  if (done_if_one && go == 1.0f) return;
  const int tid = threadIdx.x % THREADS;
  for (int row = blockIdx.x * (256 / THREADS) + threadIdx.x / THREADS; row < p.rows;
       row += gridDim.x * (256 / THREADS)) {
    const T* x = logits + p.logits_at(row);
    T* g = grad + p.grad_at(row);
    if (p.mask && !p.mask[row]) {
      zero_row<T, THREADS>(g, p.v, tid);
      continue;
    }
    const float c = coef[row] * go;
    const float2 st = stats[row];
    const float k = -c / st.y;
    const int64_t tok = p.tokens[row];
    const int token = tok >= 0 && tok < p.v ? (int)tok : -1 - kVec;
    const Span<T> s(x, p.v);
    for (int i = tid; i < s.vecs; i += THREADS) {
      const int64_t e = s.head + (int64_t)i * kVec;
      E::stream(g + e, grad_vec<T>(E::take(x + e), st.x, k, c, token - (int)e));
    }
    if (tid < s.edge) {
      const int e = s.edge_at(tid);
      g[e] = (T)(k * share_of<T>((float)x[e] - st.x) + (e == token ? c : 0.0f));
    }
  }
}

template <typename T>
__device__ __forceinline__ typename PPElems<T, Span<T>::kVec>::raw minus_infinity() {
  float e[Span<T>::kVec];
#pragma unroll
  for (int j = 0; j < Span<T>::kVec; ++j) e[j] = -INFINITY;
  return PPElems<T, Span<T>::kVec>::put(e);
}

// Holds the row as it came: without this the compiler keeps its fp32 values, and then their
// exponentials, from one walk to the next, in two to four times the registers.
template <typename R, int NV>
__device__ __forceinline__ void keep_raw(R (&r)[NV]) {
#pragma unroll
  for (int i = 0; i < NV; ++i) asm volatile("" : "+v"(r[i]));
}

// Statistics, terms and gradient of a row that NV vectors a thread hold.  Up to 8 of them leave room for
// 8 waves a SIMD (64 registers): without that bound [16, 384, 50021] takes 242 instead of 211 us.
template <typename T, int THREADS, int NV>
__global__ __launch_bounds__(THREADS < 256 ? 256 : THREADS, NV <= 8 ? 8 : 4) void pp_policy_fused_kernel(
    const T* __restrict__ logits, PolArgs p, PolTerms q, float2* __restrict__ stats,
    float* __restrict__ coef, T* __restrict__ grad) {
  constexpr int kVec = Span<T>::kVec, kRows = THREADS < 256 ? 256 / THREADS : 1;
  typedef PPElems<T, kVec> E;
  __shared__ MaxSum red[THREADS / 64];
  const int tid = threadIdx.x % THREADS;
  const int row = p.first + blockIdx.x * kRows + threadIdx.x / THREADS;
  if (row >= p.rows) return;
  const T* x = logits + p.logits_at(row);
  T* g = grad ? grad + p.grad_at(row) : nullptr;
  if (p.mask && !p.mask[row]) {
    if (tid == 0) {
      if (stats) stats[row] = make_float2(0.0f, 0.0f);
      if (coef) coef[row] = 0.0f;
      no_terms(q, row);
    }
    if (g) zero_row<T, THREADS>(g, p.v, tid);
    return;
  }
  const Span<T> s(x, p.v);
  typename E::raw r[NV];  // (-inf where the row has ended: no share in the sum)
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int n = i * THREADS + tid;
    r[i] = minus_infinity<T>();
    if (n < s.vecs) r[i] = E::take(x + s.head + (int64_t)n * kVec);
  }
  float edge = -INFINITY;
  if (tid < s.edge) edge = (float)x[s.edge_at(tid)];
  const int64_t tok = p.tokens[row];
  const float xt = token_logit(x, tok, p.v);
  // (no max of the whole row first: with that exchange before the sums' own [4, 1500, 131072] takes 474, not 452
  // us, [16, 384, 50021] 209, not 211)
  Running run;
  if (tid < s.edge) run.add(edge);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    if (i * THREADS < s.vecs) {  // (the same for all lanes)
      float e[kVec];
      E::get(r[i], e);
      run.add(e);
    }
  }
  keep_raw(r);
  const RowStats st(join_lanes<THREADS>(run, red));
  const float c = policy_terms(p, q, row, st.lp(xt), tid == 0);
  if (tid == 0) {
    if (stats) stats[row] = st.kept();
    if (coef) coef[row] = c;
  }
  if (!g) return;
  const float k = -c / st.sum;
  const int token = tok >= 0 && tok < p.v ? (int)tok : -1 - kVec;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int n = i * THREADS + tid;
    if (n < s.vecs) {
      const int e = s.head + n * kVec;
      E::stream(g + e, grad_vec<T>(r[i], st.max, k, c, token - e));
    }
  }
  if (tid < s.edge) {
    const int e = s.edge_at(tid);
    g[e] = (T)(k * share_of<T>(edge - st.max) + (e == token ? c : 0.0f));
  }
}

// The weight of a token of each sequence; one workgroup.
__global__ __launch_bounds__(1024) void pp_policy_weight_kernel(const uint8_t* __restrict__ mask,
                                                                int b, int t, int by_sequence,
                                                                float* __restrict__ w) {
  __shared__ int total, filled;
  if (threadIdx.x == 0) total = filled = 0;
  __syncthreads();
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  if (by_sequence) {
    for (int s = wave; s < b; s += 16) {
      int n = 0;
#pragma unroll 4
      for (int i = lane; i < t; i += 64) n += mask[(int64_t)s * t + i] != 0;
      for (int o = 32; o; o >>= 1) n += __shfl_xor(n, o);
      if (lane == 0) {
        if (n) atomicAdd(&filled, 1);
        w[s] = (float)n;
      }
    }
  } else {
    int n = 0;
#pragma unroll 8
    for (int i = threadIdx.x; i < b * t; i += 1024) n += mask[i] != 0;
    for (int o = 32; o; o >>= 1) n += __shfl_xor(n, o);
    if (lane == 0) atomicAdd(&total, n);
  }
  __syncthreads();
  for (int s = threadIdx.x; s < b; s += 1024) {
    if (by_sequence) {
      const float n = w[s];
      w[s] = n == 0.0f ? 0.0f : 1.0f / n / (float)filled;
    } else {
      w[s] = total ? 1.0f / (float)total : 0.0f;
    }
  }
}

// 16 bytes of a list of terms, as one number of 64 bits
__device__ __forceinline__ double sum_of(const double2& x) { return x.x + x.y; }
__device__ __forceinline__ double sum_of(const float4& x) { return ((double)x.x + (double)x.y) + ((double)x.z + (double)x.w); }
template <typename V, typename T>
__device__ __forceinline__ double sum_list(const T* x, int rows) {
  constexpr int kVec = sizeof(V) / sizeof(T);
  const V* v = reinterpret_cast<const V*>(x);  // (lists begin at multiples of 16 bytes)
  double s = 0.0;
#pragma unroll 16
  for (int i = threadIdx.x; i < rows / kVec; i += 1024) s += sum_of(v[i]);
  if ((int)threadIdx.x < rows % kVec) s += (double)x[rows - rows % kVec + threadIdx.x];
  return s;
}

// Sum of each of the three lists, in 64 bits and in a fixed order.
__global__ __launch_bounds__(1024) void pp_policy_finish_kernel(const double* __restrict__ loss,
                                                                const float* __restrict__ figures,
                                                                int rows, int padded,
                                                                float* __restrict__ out) {
  __shared__ double red[16];
  double s = blockIdx.x == 0 ? sum_list<double2>(loss, rows)
                             : sum_list<float4>(figures + (int64_t)(blockIdx.x - 1) * padded, rows);
  for (int o = 32; o; o >>= 1) s += __shfl_xor(s, o);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
#pragma unroll
    for (int i = 1; i < 16; ++i) s += red[i];
    out[blockIdx.x] = (float)s;
  }
}

constexpr int kWaveRow = 4096;     // bytes up to which a row is one wave's
constexpr int kWorkgroups = 8192;  // of the gradient kernel, which strides over the rows

// A launch takes fewer than 2^32 threads: the rows in slices, `kernel(p, rows)` for each.
constexpr int kSlice = 1 << 20;
template <typename F>
void in_slices(PolArgs p, F kernel) {
  const int rows = p.rows;
  for (p.first = 0; p.first < rows; p.first += kSlice) {
    p.rows = std::min(rows - p.first, kSlice) + p.first;
    kernel(p, p.rows - p.first);
  }
}

template <typename T, bool POLICY>
void run_terms(const T* logits, const PolArgs& all, const PolTerms& q, float2* stats, float* out,
               hipStream_t st) {
  in_slices(all, [&](const PolArgs& p, int rows) {
    if ((int64_t)p.v * (int64_t)sizeof(T) <= kWaveRow)
      hipLaunchKernelGGL((pp_row_terms_kernel<T, 64, POLICY>), dim3((rows + 3) / 4), dim3(256), 0, st,
                         logits, p, q, stats, out);
    else
      hipLaunchKernelGGL((pp_row_terms_kernel<T, 256, POLICY>), dim3(rows), dim3(256), 0, st, logits, p,
                         q, stats, out);
  });
}

template <typename T>
void run_grad(const T* logits, const PolArgs& p, const float2* stats, const float* coef,
              const float* gout, int done_if_one, T* grad, hipStream_t st) {
  if ((int64_t)p.v * (int64_t)sizeof(T) <= kWaveRow)
    hipLaunchKernelGGL((pp_row_grad_kernel<T, 64>), dim3(std::min((p.rows + 3) / 4, kWorkgroups)), dim3(256), 0,
                       st, logits, p, stats, coef, gout, done_if_one, grad);
  else
    hipLaunchKernelGGL((pp_row_grad_kernel<T, 256>), dim3(std::min(p.rows, kWorkgroups)), dim3(256), 0, st,
                       logits, p, stats, coef, gout, done_if_one, grad);
}

template <typename T, int THREADS, int NV>
bool try_fused(const T* logits, const PolArgs& all, const PolTerms& q, float2* stats, float* coef, T* grad,
               hipStream_t st) {
  if (all.v > THREADS * NV * Span<T>::kVec) return false;
  constexpr int kRows = THREADS < 256 ? 256 / THREADS : 1;
  in_slices(all, [&](const PolArgs& p, int rows) {
    hipLaunchKernelGGL((pp_policy_fused_kernel<T, THREADS, NV>), dim3((rows + kRows - 1) / kRows),
                       dim3(THREADS < 256 ? 256 : THREADS), 0, st, logits, p, q, stats, coef, grad);
  });
  return true;
}

template <typename T>
void run_policy(const T* logits, const PolArgs& p, const PolTerms& q, float2* stats, float* coef, T* grad,
                hipStream_t st) {
  // The least threads that hold the row in 8 vectors, so that many rows share a CU (bf16 [8, 512, 20001] with 8 of
  // 512 threads 75 us, with 4 of 1024 87; [8, 512, 12000] with 8 of 256 50, with 4 of 512 55); 16 vectors where
  // 1024 threads are not enough.  Without a gradient too: the loss has the same bits whether one follows or not.
  if (try_fused<T, 64, 1>(logits, p, q, stats, coef, grad, st) ||
      try_fused<T, 64, 2>(logits, p, q, stats, coef, grad, st) ||
      try_fused<T, 64, 4>(logits, p, q, stats, coef, grad, st) ||
      try_fused<T, 256, 2>(logits, p, q, stats, coef, grad, st) ||
      try_fused<T, 256, 4>(logits, p, q, stats, coef, grad, st) ||
      try_fused<T, 256, 8>(logits, p, q, stats, coef, grad, st) ||
      try_fused<T, 512, 8>(logits, p, q, stats, coef, grad, st) ||
      try_fused<T, 1024, 8>(logits, p, q, stats, coef, grad, st) ||
      try_fused<T, 1024, 16>(logits, p, q, stats, coef, grad, st))
    return;
  run_terms<T, true>(logits, p, q, stats, coef, st);
  if (grad) run_grad<T>(logits, p, stats, coef, nullptr, 0, grad, st);
}

}  // namespace

#define PP_POL_TYPES(CALL)                    \
  do {                                        \
    if (dtype == PP_F32) CALL(float);         \
    else if (dtype == PP_BF16) CALL(pp_bf16); \
    else CALL(pp_f16);                        \
  } while (0)

hipError_t pp_launch_token_lp(const void* logits, int64_t lb, int64_t lt, int dtype,
                              const int64_t* tokens, const uint8_t* mask, float* lp, float* stats,
                              int b, int t, int v, hipStream_t st) {
  const PolArgs p = {tokens, mask, lb, lt, 0, 0, 0, b * t, t, v};
  const PolTerms q = {};
#define PP_CALL(T) \
  run_terms<T, false>(static_cast<const T*>(logits), p, q, reinterpret_cast<float2*>(stats), lp, st)
  PP_POL_TYPES(PP_CALL);
#undef PP_CALL
  return hipGetLastError();
}

hipError_t pp_launch_token_lp_bwd(const void* logits, int64_t lb, int64_t lt, int dtype,
                                  const int64_t* tokens, const uint8_t* mask, const float* stats,
                                  const float* coef, const float* gout, int done_if_one, void* grad,
                                  int64_t gb, int64_t gt, int b, int t, int v, hipStream_t st) {
  const PolArgs p = {tokens, mask, lb, lt, gb, gt, 0, b * t, t, v};
#define PP_CALL(T)                                                                                     \
  run_grad<T>(static_cast<const T*>(logits), p, reinterpret_cast<const float2*>(stats), coef, gout,    \
              done_if_one, static_cast<T*>(grad), st)
  PP_POL_TYPES(PP_CALL);
#undef PP_CALL
  return hipGetLastError();
}

static int padded_rows(int b, int t) { return (b * t + 3) & ~3; }

size_t pp_policy_workspace_bytes(int b, int t) {
  return (((size_t)b + 3) & ~(size_t)3) * sizeof(float) +
         (size_t)padded_rows(b, t) * (sizeof(double) + 2 * sizeof(float));
}

hipError_t pp_launch_policy(const void* logits, int64_t lb, int64_t lt, int dtype,
                            const int64_t* tokens, const uint8_t* mask, const float* old,
                            const float* adv, int64_t ab, int64_t at, const float* ref, float low,
                            float high, float beta, int by_sequence, float* out, float* stats,
                            float* coef, void* grad, int64_t gb, int64_t gt, void* ws, int b, int t, int v,
                            hipStream_t st) {
  const PolArgs p = {tokens, mask, lb, lt, gb, gt, 0, b * t, t, v};
  float* weight = static_cast<float*>(ws);
  // (without a mask both means are the mean over all tokens)
  const int padded = padded_rows(b, t);
  double* loss = reinterpret_cast<double*>(weight + ((b + 3) & ~3));
  const PolTerms q = {old, adv, ref, ab, at, beta, 1.0 - (double)low, 1.0 + (double)high, std::log1p(-(double)low),
                      std::log1p((double)high), mask ? weight : nullptr, 1.0f / ((float)b * (float)t), loss,
                      reinterpret_cast<float*>(loss + padded), padded};
  if (mask)
    hipLaunchKernelGGL(pp_policy_weight_kernel, dim3(1), dim3(1024), 0, st, mask, b, t, by_sequence,
                       weight);
#define PP_CALL(T)                                                                                      \
  run_policy<T>(static_cast<const T*>(logits), p, q, reinterpret_cast<float2*>(stats), coef,            \
                static_cast<T*>(grad), st)
  PP_POL_TYPES(PP_CALL);
#undef PP_CALL
  hipLaunchKernelGGL(pp_policy_finish_kernel, dim3(3), dim3(1024), 0, st, q.loss, q.figures, p.rows, q.padded, out);
  return hipGetLastError();
}
