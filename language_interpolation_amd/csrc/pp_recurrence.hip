// Gated linear recurrence, forward and backward, and its single-token step.
//
//   a_t = sigmoid(f_t);   h_t = a_t h_{t-1} + (1 - a_t) z_t = z_t + a_t (h_{t-1} - z_t)
//
// per channel, z and f [b][l][d] in fp32, bf16 or fp16, the state in fp32.  reset[b][t] != 0 drops
// the state before step t (h_{t-1} := 0: a new document); steps from lengths[b] on do not exist
// (y = 0, gradients 0, nothing read), the state stays as it is.  Backward, with e_t = dL/dh_t:
//
//   e_t = gy_t + a_{t+1} e_{t+1}  (a := 0 at a reset, gh_last arrives behind the last step)
//   gz_t = e_t (1 - a_t);   gf_t = e_t a_t (1 - a_t) (h_{t-1} - z_t);   gh0 = a_0 e_0
//
// 1 - a is computed as sigmoid(-f), so neither gate loses its small end to cancellation.
// The forward of a training step keeps h at the start of every kSteps steps in fp32 (the states
// in between are recomputed from it; y, rounded to 16 bits, would not do for the differences).
#include <algorithm>

#include "pp_device.h"
#include "pp_lowp.h"

namespace {

constexpr int kSteps = PP_RECURRENCE_STEPS;  // steps between two kept states

struct RecArgs {
  int64_t zb, zl, fb, fl, gb, gl;  // strides in elements of z, f and gy over batch and time
  int b, l, d;
  const float* h0;
  const int32_t* lengths;
  const uint8_t* reset;
};

__device__ __forceinline__ void gates(float f, float& a, float& r) {
  const float x = expf(-fabsf(f));  // in (0, 1]: neither gate overflows
  const float big = 1.0f / (1.0f + x), small = x * big;
  a = f >= 0.0f ? big : small;
  r = f >= 0.0f ? small : big;
}

template <typename T>
__global__ __launch_bounds__(64) void pp_rec_fwd_kernel(const T* __restrict__ z,
                                                        const T* __restrict__ f, T* __restrict__ y,
                                                        float* __restrict__ h_last,
                                                        float* __restrict__ starts, RecArgs p) {
  const int ch = blockIdx.x * 64 + threadIdx.x, b = blockIdx.y;
  if (ch >= p.d) return;
  const int len = p.lengths ? max(0, min(p.l, p.lengths[b])) : p.l;
  const int nchunk = (p.l + kSteps - 1) / kSteps;
  float h = p.h0 ? p.h0[(int64_t)b * p.d + ch] : 0.0f;
  for (int t = 0; t < p.l; ++t) {
    if (starts && t % kSteps == 0) starts[((int64_t)b * nchunk + t / kSteps) * p.d + ch] = h;
    float out = 0.0f;
    if (t < len) {
      float a, r;
      gates((float)f[b * p.fb + t * p.fl + ch], a, r);
      if (p.reset && p.reset[(int64_t)b * p.l + t]) h = 0.0f;
      h = fmaf(a, h, r * (float)z[b * p.zb + t * p.zl + ch]);
      out = h;
    }
    y[((int64_t)b * p.l + t) * p.d + ch] = (T)out;
  }
  h_last[(int64_t)b * p.d + ch] = h;
}

template <typename T>
__global__ __launch_bounds__(64) void pp_rec_bwd_kernel(
    const T* __restrict__ z, const T* __restrict__ f, const float* __restrict__ starts,
    const T* __restrict__ gy, const float* __restrict__ gh, T* __restrict__ gz, T* __restrict__ gf,
    float* __restrict__ gh0, RecArgs p) {
  const int ch = blockIdx.x * 64 + threadIdx.x, b = blockIdx.y;
  if (ch >= p.d) return;
  const int len = p.lengths ? max(0, min(p.l, p.lengths[b])) : p.l;
  const int nchunk = (p.l + kSteps - 1) / kSteps;
  float u = gh ? gh[(int64_t)b * p.d + ch] : 0.0f;  // a_{t+1} e_{t+1}
  for (int c = nchunk - 1; c >= 0; --c) {
    const int t0 = c * kSteps;
    float prev[kSteps];
    float h = starts[((int64_t)b * nchunk + c) * p.d + ch];
#pragma unroll
    for (int j = 0; j < kSteps; ++j) {
      const int t = t0 + j;
      prev[j] = 0.0f;
      if (t < len) {
        float a, r;
        gates((float)f[b * p.fb + t * p.fl + ch], a, r);
        if (p.reset && p.reset[(int64_t)b * p.l + t]) h = 0.0f;
        prev[j] = h;
        h = fmaf(a, h, r * (float)z[b * p.zb + t * p.zl + ch]);
      }
    }
#pragma unroll
    for (int j = kSteps - 1; j >= 0; --j) {
      const int t = t0 + j;
      if (t >= p.l) continue;
      const int64_t at = ((int64_t)b * p.l + t) * p.d + ch;
      float oz = 0.0f, of = 0.0f;
      if (t < len) {
        float a, r;
        gates((float)f[b * p.fb + t * p.fl + ch], a, r);
        const float e = (float)gy[b * p.gb + t * p.gl + ch] + u;
        oz = e * r;
        of = e * (a * r) * (prev[j] - (float)z[b * p.zb + t * p.zl + ch]);
        u = p.reset && p.reset[(int64_t)b * p.l + t] ? 0.0f : a * e;
      }
      gz[at] = (T)oz;
      gf[at] = (T)of;
    }
  }
  if (gh0) gh0[(int64_t)b * p.d + ch] = u;
}

template <typename T>
__global__ __launch_bounds__(256) void pp_rec_step_kernel(const T* __restrict__ z, int64_t zb,
                                                          const T* __restrict__ f, int64_t fb,
                                                          float* __restrict__ h, int64_t hb,
                                                          T* __restrict__ y, int b, int d) {
  const int ch = blockIdx.x * 256 + threadIdx.x, row = blockIdx.y;
  if (ch >= d) return;
  float a, r;
  gates((float)f[row * fb + ch], a, r);
  const float n = fmaf(a, h[row * hb + ch], r * (float)z[row * zb + ch]);
  h[row * hb + ch] = n;
  y[(int64_t)row * d + ch] = (T)n;
}

}  // namespace

#define PP_REC_TYPES(CALL)                 \
  do {                                     \
    if (dtype == PP_F32) CALL(float);      \
    else if (dtype == PP_BF16) CALL(pp_bf16); \
    else CALL(pp_f16);                     \
    return hipGetLastError();              \
  } while (0)

size_t pp_rec_workspace_bytes(int b, int l, int d) { return 0; }

hipError_t pp_launch_rec_fwd(const void* z, int64_t zb, int64_t zl, const void* f, int64_t fb,
                             int64_t fl, int dtype, const float* h0, const int32_t* lengths,
                             const uint8_t* reset, void* y, float* h_last, float* starts, void* ws,
                             int b, int l, int d, hipStream_t st) {
  const RecArgs p = {zb, zl, fb, fl, 0, 0, b, l, d, h0, lengths, reset};
#define PP_CALL(T)                                                                             \
  hipLaunchKernelGGL((pp_rec_fwd_kernel<T>), dim3((d + 63) / 64, b), dim3(64), 0, st,          \
                     static_cast<const T*>(z), static_cast<const T*>(f), static_cast<T*>(y),   \
                     h_last, starts, p)
  PP_REC_TYPES(PP_CALL);
#undef PP_CALL
}

hipError_t pp_launch_rec_bwd(const void* z, int64_t zb, int64_t zl, const void* f, int64_t fb,
                             int64_t fl, int dtype, const int32_t* lengths, const uint8_t* reset,
                             const float* starts, const void* gy, int64_t gb, int64_t gl,
                             const float* gh_last, void* gz, void* gf, float* gh0, void* ws, int b,
                             int l, int d, hipStream_t st) {
  const RecArgs p = {zb, zl, fb, fl, gb, gl, b, l, d, nullptr, lengths, reset};
#define PP_CALL(T)                                                                              \
  hipLaunchKernelGGL((pp_rec_bwd_kernel<T>), dim3((d + 63) / 64, b), dim3(64), 0, st,           \
                     static_cast<const T*>(z), static_cast<const T*>(f), starts,                \
                     static_cast<const T*>(gy), gh_last, static_cast<T*>(gz),                   \
                     static_cast<T*>(gf), gh0, p)
  PP_REC_TYPES(PP_CALL);
#undef PP_CALL
}

hipError_t pp_launch_rec_step(const void* z, int64_t zb, const void* f, int64_t fb, int dtype,
                              float* h, int64_t hb, void* y, int b, int d, hipStream_t st) {
#define PP_CALL(T)                                                                              \
  hipLaunchKernelGGL((pp_rec_step_kernel<T>), dim3((d + 255) / 256, b), dim3(256), 0, st,       \
                     static_cast<const T*>(z), zb, static_cast<const T*>(f), fb, h, hb,         \
                     static_cast<T*>(y), b, d)
  PP_REC_TYPES(PP_CALL);
#undef PP_CALL
}
