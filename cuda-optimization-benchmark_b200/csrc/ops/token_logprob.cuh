// Log-probability of each position's token and the entropy of its distribution, from logits.
//
// Per row of V logits x, with i running over the vocabulary, inv = 1 / temperature, m = max x:
//   d_i = (x_i - m) * inv,  S = sum exp(d_i),  U = sum exp(d_i) d_i
//   log_prob = d_token - log S,   entropy = log S - U / S
// d is taken from the difference to the maximum before it is scaled, so logits of any size (the
// type's lowest value among them) neither overflow nor lose digits; a logit of -inf has probability
// 0 and adds 0 to U.  stats keeps (m, log S, entropy) per row for the backward:
//   p_i = exp(d_i - log S)
//   grad_x_i = inv * (g_lp * ([i = token] - p_i) - g_ent * p_i * (d_i - log S + entropy))
// A negative token masks its row: outputs and gradient 0, the logits not read.  A token >= V makes
// the row's log_prob (and its gradient) NaN.
#pragma once

#include "../common/dtype.cuh"

namespace b200 {
namespace lp {

constexpr int kThreads = 256;

// Running (max, sum, weighted sum) of a part of a row.
struct Acc {
  float m, s, u;
};

__device__ __forceinline__ Acc empty_acc() { return Acc{-INFINITY, 0.0f, 0.0f}; }

// acc with its maximum moved to m >= acc.m.
__device__ __forceinline__ void rebase(Acc& a, float m, float inv) {
  if (a.m == m) return;
  if (a.s == 0.0f || a.m == -INFINITY) {  // nothing finite yet
    a.m = m;
    return;
  }
  const float delta = (a.m - m) * inv;  // < 0, -inf when the old part vanishes beside the new maximum
  const float scale = expf(delta);
  a.u = scale == 0.0f ? 0.0f : (a.u + delta * a.s) * scale;
  a.s *= scale;
  a.m = m;
}

__device__ __forceinline__ void merge(Acc& a, Acc b, float inv) {
  const float m = fmaxf(a.m, b.m);
  rebase(a, m, inv);
  rebase(b, m, inv);
  a.s += b.s;
  a.u += b.u;
}

__device__ __forceinline__ void add(Acc& a, float x, float inv) {
  if (x == -INFINITY) return;
  if (x > a.m) rebase(a, x, inv);
  const float d = (x - a.m) * inv;
  const float e = expf(d);
  a.s += e;
  if (e > 0.0f) a.u += e * d;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) forward_kernel(const T* __restrict__ x, int64_t xb, int64_t xt,
                                                           const int64_t* __restrict__ token, int64_t kb, int64_t kt,
                                                           int64_t Tn, int64_t V, float inv,
                                                           float* __restrict__ log_prob, float* __restrict__ entropy,
                                                           float* __restrict__ stats) {
  pdl_begin();
  const int64_t r = blockIdx.x, b = r / Tn, t = r - b * Tn;
  const int64_t tok = token[b * kb + t * kt];
  if (tok < 0) {
    if (threadIdx.x == 0) {
      log_prob[r] = 0.0f;
      if (entropy) entropy[r] = 0.0f;
      if (stats)
        for (int k = 0; k < 3; ++k) stats[3 * r + k] = 0.0f;
    }
    return;
  }
  const T* row = x + b * xb + t * xt;
  Acc a = empty_acc();
  for (int64_t i = threadIdx.x; i < V; i += kThreads) add(a, to_f32(row[i]), inv);
  __shared__ Acc part[kThreads];
  part[threadIdx.x] = a;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < kThreads; ++i) merge(a, part[i], inv);
    const float log_s = logf(a.s);
    const float ent = log_s - a.u / a.s;
    log_prob[r] = tok < V ? (to_f32(row[tok]) - a.m) * inv - log_s : NAN;
    if (entropy) entropy[r] = ent;
    if (stats) {
      stats[3 * r] = a.m;
      stats[3 * r + 1] = log_s;
      stats[3 * r + 2] = ent;
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) backward_kernel(const T* __restrict__ x, int64_t xb, int64_t xt,
                                                            const int64_t* __restrict__ token, int64_t kb, int64_t kt,
                                                            const float* __restrict__ stats,
                                                            const float* __restrict__ g_lp,
                                                            const float* __restrict__ g_ent, int64_t Tn, int64_t V,
                                                            float inv, T* __restrict__ grad) {
  pdl_begin();
  const int64_t r = blockIdx.x, b = r / Tn, t = r - b * Tn;
  const int64_t tok = token[b * kb + t * kt];
  const T* row = x + b * xb + t * xt;
  T* out = grad + r * V;
  if (tok < 0) {
    for (int64_t i = threadIdx.x; i < V; i += kThreads) out[i] = from_f32<T>(0.0f);
    return;
  }
  const float m = stats[3 * r], log_s = stats[3 * r + 1], ent = stats[3 * r + 2];
  const float gl = tok < V ? g_lp[r] : NAN, ge = g_ent ? g_ent[r] : 0.0f;
  for (int64_t i = threadIdx.x; i < V; i += kThreads) {
    const float l = (to_f32(row[i]) - m) * inv - log_s;
    const float p = expf(l);
    float g = (i == tok ? gl : 0.0f) - gl * p;
    if (p > 0.0f) g -= ge * p * (l + ent);
    out[i] = from_f32<T>(g * inv);
  }
}

inline bool temperature_ok(double temperature) { return temperature > 0.0 && temperature < INFINITY; }

// strides (host array): logits (batch, time), token (batch, time), in elements.
inline int forward(const void* logits, int dtype, const int64_t* strides, const int64_t* token, int32_t B, int32_t T,
                   int32_t V, double temperature, float* log_prob, float* entropy, float* stats,
                   cudaStream_t stream) {
  if (B < 0 || T < 0 || V < 1 || !dtype_ok(dtype) || strides == nullptr || !temperature_ok(temperature))
    return kInvalidArgument;
  const int64_t rows = int64_t(B) * T;
  if (rows == 0) return kOk;
  if (logits == nullptr || token == nullptr || log_prob == nullptr || rows > 0x7fffffff) return kInvalidArgument;
  return with_dtype(dtype, [&](auto e) {
    using E = decltype(e);
    return launch_pdl(forward_kernel<E>, dim3(unsigned(rows)), dim3(kThreads), 0, stream,
                      static_cast<const E*>(logits), strides[0], strides[1], token, strides[2], strides[3], int64_t(T),
                      int64_t(V), float(1.0 / temperature), log_prob, entropy, stats);
  });
}

inline int backward(const void* logits, int dtype, const int64_t* strides, const int64_t* token, const float* stats,
                    const float* grad_log_prob, const float* grad_entropy, int32_t B, int32_t T, int32_t V,
                    double temperature, void* grad_logits, cudaStream_t stream) {
  if (B < 0 || T < 0 || V < 1 || !dtype_ok(dtype) || strides == nullptr || !temperature_ok(temperature))
    return kInvalidArgument;
  const int64_t rows = int64_t(B) * T;
  if (rows == 0) return kOk;
  if (logits == nullptr || token == nullptr || stats == nullptr || grad_log_prob == nullptr ||
      grad_logits == nullptr || rows > 0x7fffffff)
    return kInvalidArgument;
  return with_dtype(dtype, [&](auto e) {
    using E = decltype(e);
    return launch_pdl(backward_kernel<E>, dim3(unsigned(rows)), dim3(kThreads), 0, stream,
                      static_cast<const E*>(logits), strides[0], strides[1], token, strides[2], strides[3], stats,
                      grad_log_prob, grad_entropy, int64_t(T), int64_t(V), float(1.0 / temperature),
                      static_cast<E*>(grad_logits));
  });
}

}  // namespace lp
}  // namespace b200
