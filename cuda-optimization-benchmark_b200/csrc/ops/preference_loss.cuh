// Preference loss over pairs of answers (a chosen and a rejected one), with its gradients.
//
// Per pair, with s the sum over the answer's masked tokens of log_prob - ref_log_prob (of log_prob
// alone without a reference), divided by the tokens' number when `average`:
//   reward_chosen = beta s_c,  reward_rejected = beta s_r,  z = beta (s_c - s_r) - margin
//     sigmoid: loss = -(1 - e) log sigmoid(z) - e log sigmoid(-z)   (e: label smoothing)
//     hinge:   loss = max(0, 1 - z)
//     ipo:     loss = (z / beta - 1 / (2 beta))^2
// out = mean over the pairs of the loss, of [reward_chosen > reward_rejected] and of reward_chosen -
// reward_rejected.  Every masked token of an answer has the gradient +-beta dloss/dz / B (/ its
// answer's tokens when `average`).  An answer without tokens has s = 0.
// The sums are in fp64: their difference, a small part of them, is what the loss sees.
#pragma once

#include "../common/dtype.cuh"
#include "../common/workspace.cuh"

namespace b200 {
namespace pref {

enum Form : int { kSigmoid = 0, kHinge = 1, kIpo = 2 };

constexpr int kThreads = 256;
constexpr int kOutputs = 3;

struct Side {
  const float *lp, *ref;
  const uint8_t* mask;
  int64_t lp_s, ref_s, mask_s;  // row strides
  int T;
  float *reward, *grad;
};

struct Params {
  Side side[2];  // chosen, rejected
  int B;
  double beta, smoothing, margin;
  int form;
  bool average;
  float* out;
};

__device__ __forceinline__ double softplus(double v) { return fmax(v, 0.0) + log1p(exp(-fabs(v))); }
__device__ __forceinline__ double sigmoid(double v) { return 1.0 / (1.0 + exp(-v)); }

__device__ __forceinline__ double pair_loss(const Params& p, double z, double& dz) {
  if (p.form == kSigmoid) {
    dz = p.smoothing - sigmoid(-z);
    return (1.0 - p.smoothing) * softplus(-z) + p.smoothing * softplus(z);
  }
  if (p.form == kHinge) {
    dz = z < 1.0 ? -1.0 : 0.0;
    return z >= 1.0 ? 0.0 : 1.0 - z;  // NaN stays NaN
  }
  const double u = (z - 0.5) / p.beta;
  dz = 2.0 * u / p.beta;
  return u * u;
}

struct PairOut {
  double loss, win, gap;
};

__global__ void __launch_bounds__(kThreads) pair_kernel(Params p, PairOut* __restrict__ pairs) {
  pdl_begin();
  const int64_t b = blockIdx.x;
  __shared__ double part[kThreads];
  __shared__ unsigned cnt[kThreads];
  __shared__ float slope[2];
  double s[2];
  unsigned n[2];
  for (int k = 0; k < 2; ++k) {
    const Side& d = p.side[k];
    double a = 0.0;
    unsigned c = 0;
    for (int64_t t = threadIdx.x; t < d.T; t += kThreads) {
      if (d.mask != nullptr && d.mask[b * d.mask_s + t] == 0) continue;
      a += double(d.lp[b * d.lp_s + t]) - (d.ref ? double(d.ref[b * d.ref_s + t]) : 0.0);
      ++c;
    }
    part[threadIdx.x] = a;
    cnt[threadIdx.x] = c;
    __syncthreads();
    if (threadIdx.x == 0) {
      for (int i = 1; i < kThreads; ++i) a += part[i], c += cnt[i];
      s[k] = a;
      n[k] = c;
    }
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    double inv[2] = {1.0, 1.0};
    for (int k = 0; k < 2; ++k)
      if (p.average) inv[k] = 1.0 / (n[k] > 0 ? n[k] : 1), s[k] *= inv[k];
    const double rc = p.beta * s[0], rr = p.beta * s[1];
    double dz;
    const double loss = pair_loss(p, p.beta * (s[0] - s[1]) - p.margin, dz);
    pairs[b] = PairOut{loss, s[0] > s[1] ? 1.0 : 0.0, p.beta * (s[0] - s[1])};
    p.side[0].reward[b] = float(rc);
    p.side[1].reward[b] = float(rr);
    slope[0] = float(p.beta * dz * inv[0] / p.B);
    slope[1] = float(-p.beta * dz * inv[1] / p.B);
  }
  __syncthreads();
  for (int k = 0; k < 2; ++k) {
    const Side& d = p.side[k];
    if (d.grad == nullptr) continue;
    for (int64_t t = threadIdx.x; t < d.T; t += kThreads)
      d.grad[b * d.T + t] = d.mask != nullptr && d.mask[b * d.mask_s + t] == 0 ? 0.0f : slope[k];
  }
}

__global__ void finish_kernel(Params p, const PairOut* __restrict__ pairs) {
  pdl_begin();
  PairOut a = {};
  for (int b = 0; b < p.B; ++b) a.loss += pairs[b].loss, a.win += pairs[b].win, a.gap += pairs[b].gap;
  p.out[0] = float(a.loss / p.B);
  p.out[1] = float(a.win / p.B);
  p.out[2] = float(a.gap / p.B);
}

inline int64_t workspace_bytes(int32_t B) { return int64_t(256 + align256(size_t(B) * sizeof(PairOut))); }

// strides (host array): rows of chosen, rejected, ref_chosen, ref_rejected, chosen_mask, rejected_mask.
inline int run(const float* chosen, const float* rejected, const float* ref_chosen, const float* ref_rejected,
               const uint8_t* chosen_mask, const uint8_t* rejected_mask, const int64_t* strides, int32_t B, int32_t Tc,
               int32_t Tr, double beta, int form, double smoothing, double margin, int average, float* out,
               float* reward_chosen, float* reward_rejected, float* grad_chosen, float* grad_rejected, void* ws,
               int64_t ws_bytes, cudaStream_t stream) {
  if (B < 0 || Tc < 0 || Tr < 0 || out == nullptr || strides == nullptr) return kInvalidArgument;
  if (!(beta > 0.0) || form < kSigmoid || form > kIpo || !(smoothing >= 0.0 && smoothing <= 0.5))
    return kInvalidArgument;
  if (form != kSigmoid && smoothing != 0.0) return kInvalidArgument;
  if ((ref_chosen == nullptr) != (ref_rejected == nullptr) && Tc > 0 && Tr > 0) return kInvalidArgument;
  if (B == 0) return cudaMemsetAsync(out, 0, kOutputs * sizeof(float), stream) == cudaSuccess ? kOk : kCudaError;
  if ((Tc > 0 && chosen == nullptr) || (Tr > 0 && rejected == nullptr) || reward_chosen == nullptr ||
      reward_rejected == nullptr)
    return kInvalidArgument;
  if (ws == nullptr || ws_bytes < workspace_bytes(B)) return kWorkspaceTooSmall;
  Params p;
  p.side[0] = Side{chosen, ref_chosen, chosen_mask, strides[0], strides[2], strides[4], Tc, reward_chosen, grad_chosen};
  p.side[1] =
      Side{rejected, ref_rejected, rejected_mask, strides[1], strides[3], strides[5], Tr, reward_rejected, grad_rejected};
  p.B = B, p.beta = beta, p.smoothing = smoothing, p.margin = margin, p.form = form, p.average = average != 0;
  p.out = out;
  PairOut* pairs = reinterpret_cast<PairOut*>(static_cast<char*>(ws) + 256);
  int st = launch_pdl(pair_kernel, dim3(B), dim3(kThreads), 0, stream, p, pairs);
  if (st == kOk) st = launch_pdl(finish_kernel, dim3(1), dim3(1), 0, stream, p, static_cast<const PairOut*>(pairs));
  return st;
}

}  // namespace pref
}  // namespace b200
