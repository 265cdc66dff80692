// Token log-probabilities and the clipped policy loss with a KL term, from logits.
//
//   lp = logits[token] - logsumexp(logits);  rho = exp(lp - old)
//   term = -min(rho A, clip(rho, 1 - low, 1 + high) A) + beta (exp(ref - lp) - (ref - lp) - 1)
//   loss = sum_t w_t term_t,  w = mask / #tokens  or  mask / (#tokens of the sequence * #sequences)
//   dloss/dlogits = c (onehot(token) - softmax),  c = w (-A rho [not clipped] + beta (1 - exp(ref - lp)))
//
// Row statistics are kept as (max, log of the sum of exp(x - max)) in fp32: lp = (x - max) - log sum
// is a difference of small numbers, where x - logsumexp would lose the digits of a large max.
// A masked token's logits, token, old, ref and advantage are not read; its gradient row is zeros.
#include <algorithm>

#include "pp_device.h"
#include "pp_lowp.h"

namespace {

struct PolArgs {
  const int64_t* tokens;
  const uint8_t* mask;
  int64_t lb, lt;  // strides of the logits (and of their gradient) over batch and time
  int rows, t, v;
};
struct PolTerms {
  const float* old;
  const float* adv;
  const float* ref;
  int64_t ab, at;  // strides of adv
  float low, high, beta;
};

__device__ __forceinline__ float block_max(float v, float* red) {
  for (int o = 32; o; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  float r = red[0];
  for (int i = 1; i < (int)blockDim.x / 64; ++i) r = fmaxf(r, red[i]);
  __syncthreads();
  return r;
}
__device__ __forceinline__ float block_sum(float v, float* red) {
  for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  float r = 0.0f;
  for (int i = 0; i < (int)blockDim.x / 64; ++i) r += red[i];
  __syncthreads();
  return r;
}

// (max, log sum) of a row
template <typename T>
__device__ __forceinline__ float2 row_stats(const T* __restrict__ x, int v, float* red) {
  float m = -INFINITY;
  for (int i = threadIdx.x; i < v; i += blockDim.x) m = fmaxf(m, (float)x[i]);
  m = block_max(m, red);
  float s = 0.0f;
  for (int i = threadIdx.x; i < v; i += blockDim.x) s += expf((float)x[i] - m);
  s = block_sum(s, red);
  return make_float2(m, logf(s));
}

template <typename T>
__device__ __forceinline__ float token_lp(const T* __restrict__ x, int64_t token, int v, float2 st) {
  if (token < 0 || token >= v) return NAN;  // no such class: the loss says so
  return ((float)x[token] - st.x) - st.y;
}

template <typename T>
__device__ __forceinline__ void write_grad(const T* __restrict__ x, T* __restrict__ g, int64_t token,
                                           int v, float2 st, float c) {
  for (int i = threadIdx.x; i < v; i += blockDim.x) {
    float q = 0.0f;
    if (c != 0.0f) q = c * ((i == token ? 1.0f : 0.0f) - expf(((float)x[i] - st.x) - st.y));
    g[i] = (T)q;
  }
}

template <typename T>
__global__ __launch_bounds__(256) void pp_token_lp_kernel(const T* __restrict__ logits, PolArgs p,
                                                          float* __restrict__ lp,
                                                          float2* __restrict__ stats) {
  __shared__ float red[4];
  const int row = blockIdx.x;
  if (p.mask && !p.mask[row]) {
    if (threadIdx.x == 0) {
      lp[row] = 0.0f;
      if (stats) stats[row] = make_float2(0.0f, 0.0f);
    }
    return;
  }
  const T* x = logits + (row / p.t) * p.lb + (row % p.t) * p.lt;
  const float2 st = row_stats(x, p.v, red);
  if (threadIdx.x == 0) {
    lp[row] = token_lp(x, p.tokens[row], p.v, st);
    if (stats) stats[row] = st;
  }
}

// grad = gout * coef * (onehot - softmax).  done_if_one: the gradient for gout = 1 is in `grad`
// already (the forward of the loss wrote it), so that only another gout needs the work; it starts
// from the logits again, since scaling the stored 16-bit values would round twice and would not
// bring back what underflowed at gout = 1 (a loss scaled for fp16).
template <typename T>
__global__ __launch_bounds__(256) void pp_token_lp_bwd_kernel(
    const T* __restrict__ logits, PolArgs p, const float2* __restrict__ stats,
    const float* __restrict__ coef, const float* __restrict__ gout, int done_if_one,
    T* __restrict__ grad) {
  const float go = gout ? *gout : 1.0f;
  if (done_if_one && go == 1.0f) return;
  for (int row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const int64_t at = (row / p.t) * p.lb + (row % p.t) * p.lt;
    const float c = p.mask && !p.mask[row] ? 0.0f : coef[row] * go;
    write_grad(logits + at, grad + at, p.tokens[row], p.v, stats[row], c);
  }
}

// the weight of a token of each sequence; one workgroup
__global__ __launch_bounds__(1024) void pp_policy_weight_kernel(const uint8_t* __restrict__ mask,
                                                                int b, int t, int by_sequence,
                                                                float* __restrict__ w) {
  __shared__ int total, filled;
  if (threadIdx.x == 0) total = filled = 0;
  __syncthreads();
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  for (int s = wave; s < b; s += 16) {
    int n = 0;
    for (int i = lane; i < t; i += 64) n += mask ? mask[(int64_t)s * t + i] != 0 : 1;
    for (int o = 32; o; o >>= 1) n += __shfl_xor(n, o);
    if (lane == 0) {
      atomicAdd(&total, n);
      if (n) atomicAdd(&filled, 1);
      w[s] = (float)n;
    }
  }
  __syncthreads();
  for (int s = threadIdx.x; s < b; s += 1024) {
    const float n = w[s];
    w[s] = n == 0.0f ? 0.0f : by_sequence ? 1.0f / n / (float)filled : 1.0f / (float)total;
  }
}

template <typename T>
__global__ __launch_bounds__(256) void pp_policy_kernel(const T* __restrict__ logits, PolArgs p,
                                                        PolTerms q, const float* __restrict__ weight,
                                                        float2* __restrict__ stats,
                                                        float* __restrict__ coef,
                                                        float* __restrict__ terms,
                                                        T* __restrict__ grad) {
  __shared__ float red[4];
  const int row = blockIdx.x, b = row / p.t, t = row % p.t;
  const int64_t at = b * p.lb + t * p.lt;
  float c = 0.0f, loss = 0.0f, kl = 0.0f, cut = 0.0f;
  float2 st = make_float2(0.0f, 0.0f);
  int64_t token = 0;
  if (!p.mask || p.mask[row]) {
    const T* x = logits + at;
    token = p.tokens[row];
    st = row_stats(x, p.v, red);
    const float lp = token_lp(x, token, p.v, st);
    const float w = weight[b], adv = q.adv[b * q.ab + t * q.at];
    const float rho = expf(lp - q.old[row]);
    const float border = adv >= 0.0f ? 1.0f + q.high : 1.0f - q.low;
    const bool clipped = adv >= 0.0f ? rho > border : rho < border;
    loss = -(clipped ? border : rho) * adv;
    c = clipped ? 0.0f : -adv * rho;
    if (q.ref) {
      const float delta = q.ref[row] - lp, grow = expm1f(delta);
      kl = grow - delta;
      loss += q.beta * kl;
      c -= q.beta * grow;
    }
    c *= w;
    loss *= w;
    kl *= w;
    cut = clipped ? w : 0.0f;
  }
  if (threadIdx.x == 0) {
    terms[row] = loss;
    terms[p.rows + row] = kl;
    terms[2 * (int64_t)p.rows + row] = cut;
    if (stats) {
      stats[row] = st;
      coef[row] = c;
    }
  }
  if (grad) write_grad(logits + at, grad + at, token, p.v, st, c);
}

__global__ __launch_bounds__(1024) void pp_policy_finish_kernel(const float* __restrict__ terms,
                                                                int rows, float* __restrict__ out) {
  __shared__ double red[16];
  const float* x = terms + (int64_t)blockIdx.x * rows;
  double s = 0.0;
  for (int i = threadIdx.x; i < rows; i += 1024) s += (double)x[i];
  for (int o = 32; o; o >>= 1) s += __shfl_xor(s, o);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < 16; ++i) s += red[i];
    out[blockIdx.x] = (float)s;
  }
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
  const PolArgs p = {tokens, mask, lb, lt, b * t, t, v};
#define PP_CALL(T)                                                                               \
  hipLaunchKernelGGL((pp_token_lp_kernel<T>), dim3(p.rows), dim3(256), 0, st,                    \
                     static_cast<const T*>(logits), p, lp, reinterpret_cast<float2*>(stats))
  PP_POL_TYPES(PP_CALL);
#undef PP_CALL
  return hipGetLastError();
}

hipError_t pp_launch_token_lp_bwd(const void* logits, int64_t lb, int64_t lt, int dtype,
                                  const int64_t* tokens, const uint8_t* mask, const float* stats,
                                  const float* coef, const float* gout, int done_if_one, void* grad,
                                  int b, int t, int v, hipStream_t st) {
  const PolArgs p = {tokens, mask, lb, lt, b * t, t, v};
  const int grid = std::min(p.rows, 4096);
#define PP_CALL(T)                                                                               \
  hipLaunchKernelGGL((pp_token_lp_bwd_kernel<T>), dim3(grid), dim3(256), 0, st,                  \
                     static_cast<const T*>(logits), p, reinterpret_cast<const float2*>(stats),   \
                     coef, gout, done_if_one, static_cast<T*>(grad))
  PP_POL_TYPES(PP_CALL);
#undef PP_CALL
  return hipGetLastError();
}

size_t pp_policy_workspace_bytes(int b, int t) {
  return ((size_t)b + 3 * (size_t)b * t) * sizeof(float);
}

hipError_t pp_launch_policy(const void* logits, int64_t lb, int64_t lt, int dtype,
                            const int64_t* tokens, const uint8_t* mask, const float* old,
                            const float* adv, int64_t ab, int64_t at, const float* ref, float low,
                            float high, float beta, int by_sequence, float* out, float* stats,
                            float* coef, void* grad, void* ws, int b, int t, int v, hipStream_t st) {
  const PolArgs p = {tokens, mask, lb, lt, b * t, t, v};
  const PolTerms q = {old, adv, ref, ab, at, low, high, beta};
  float* weight = static_cast<float*>(ws);
  float* terms = weight + b;
  hipLaunchKernelGGL(pp_policy_weight_kernel, dim3(1), dim3(1024), 0, st, mask, b, t, by_sequence,
                     weight);
#define PP_CALL(T)                                                                                \
  hipLaunchKernelGGL((pp_policy_kernel<T>), dim3(p.rows), dim3(256), 0, st,                       \
                     static_cast<const T*>(logits), p, q, weight, reinterpret_cast<float2*>(stats), \
                     coef, terms, static_cast<T*>(grad))
  PP_POL_TYPES(PP_CALL);
#undef PP_CALL
  hipLaunchKernelGGL(pp_policy_finish_kernel, dim3(3), dim3(1024), 0, st, terms, p.rows, out);
  return hipGetLastError();
}
