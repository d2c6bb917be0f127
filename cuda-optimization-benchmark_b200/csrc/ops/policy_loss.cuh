// Clipped policy loss with a KL term and an entropy term over masked token log-probs [B, T], with its
// gradients.
//
// Per token with mask m (all tokens without a mask), d = cur - old, r = exp(d), advantage A:
//   gain = min(r A, clip(r, 1 - clip_low, 1 + clip_high) A);  with a dual clip c > 1 and A < 0: max(gain, c A)
//   kl (q = ref - cur):  k1 = -q,  k2 = q^2 / 2,  k3 = exp(q) - q - 1
//   loss = sum w (-gain + kl_coef kl - entropy_coef entropy),  w = scale m * {
//     token_mean: 1 / sum m;  sequence_mean: 1 / (non-empty rows * tokens of the row);  sum: 1 }
//   d loss / d cur     = w (-[not clipped] r A + kl_coef dkl),  dkl = 1, -q, 1 - exp(q)
//   d loss / d entropy = -w entropy_coef
// old, ref and A are constants.  Outputs: loss, its three parts (policy, kl, entropy; unscaled by their
// coefficients), and over the masked-in tokens the clip fraction (r outside the clip range), the mean of
// exp(d) - 1 - d, the largest r and the mean r.  Without tokens every output and gradient is 0.
//
// A token is clipped or not by a step in its gradient, so the comparison is exact: cur - old as an
// unrounded pair of floats (s, e) against log(1 + clip_high) and log(1 - clip_low) as pairs.
#pragma once

#include "../common/dtype.cuh"
#include "../common/workspace.cuh"

namespace b200 {
namespace policy {

enum KlForm : int { kK1 = 0, kK2 = 1, kK3 = 2 };
enum Reduction : int { kTokenMean = 0, kSequenceMean = 1, kSum = 2 };

constexpr int kOutputs = 8;
constexpr int kThreads = 256;

// A threshold as the nearest float and the remainder.
struct Pair {
  float hi, lo;
};

inline Pair make_pair_of(double v) {
  const float hi = float(v);
  return Pair{hi, hi == hi && hi - hi == 0.0f ? float(v - double(hi)) : 0.0f};
}

// a - b without rounding as s + e (Knuth's two-sum).
__device__ __forceinline__ void two_diff(float a, float b, float& s, float& e) {
  s = __fsub_rn(a, b);
  const float bb = __fsub_rn(s, a);
  e = __fsub_rn(__fsub_rn(a, __fsub_rn(s, bb)), __fadd_rn(b, bb));
}
__device__ __forceinline__ bool above(float s, float e, Pair p) { return s > p.hi || (s == p.hi && e > p.lo); }
__device__ __forceinline__ bool below(float s, float e, Pair p) { return s < p.hi || (s == p.hi && e < p.lo); }

// exp(q) - 1 - q without the cancellation near 0: its Taylor series up to q^8 / 8! for |q| < 1/4
// (the next term is below 2^-24 of the value), the plain difference beyond.
__device__ __forceinline__ float exp_minus_1_minus(float q) {
  if (fabsf(q) >= 0.25f) return expm1f(q) - q;
  float p = 1.0f / 40320.0f;
  p = fmaf(p, q, 1.0f / 5040.0f);
  p = fmaf(p, q, 1.0f / 720.0f);
  p = fmaf(p, q, 1.0f / 120.0f);
  p = fmaf(p, q, 1.0f / 24.0f);
  p = fmaf(p, q, 1.0f / 6.0f);
  p = fmaf(p, q, 0.5f);
  return q * q * p;
}

struct Params {
  const float *cur, *old, *adv, *ref, *ent;
  const uint8_t* mask;
  int64_t cur_s, old_s, adv_s, adv_e, ref_s, ent_s, mask_s;  // row strides; adv_e: 1, or 0 for one per row
  int B, T;
  Pair log_high, log_low, log_dual;
  float high, low, dual;  // 1 + clip_high, 1 - clip_low, c (0: off)
  float kl_coef, ent_coef;
  int kl_form, reduction;
  double scale, kl_coef_d, ent_coef_d;
  float *grad, *grad_ent, *out;
};

struct Token {
  float pg, kl, d_cur, ratio, diff;
  bool outside;
};

__device__ __forceinline__ float kl_term(int form, float q, float& dkl) {
  if (form == kK1) {
    dkl = 1.0f;
    return -q;
  }
  if (form == kK2) {
    dkl = -q;
    return 0.5f * q * q;
  }
  dkl = -expm1f(q);
  return exp_minus_1_minus(q);
}

__device__ __forceinline__ Token token_loss(const Params& p, float cur, float old, float adv, float ref) {
  Token k;
  float s, e;
  two_diff(cur, old, s, e);
  const bool hi = above(s, e, p.log_high), lo = below(s, e, p.log_low);
  k.ratio = expf(s);
  k.diff = exp_minus_1_minus(s);
  k.outside = hi || lo;
  const bool dual = p.dual > 0.0f && adv < 0.0f && above(s, e, p.log_dual);
  const bool clipped = (adv > 0.0f && hi) || (adv < 0.0f && lo) || dual || adv == 0.0f;
  const float held = dual ? p.dual : hi ? p.high : lo ? p.low : k.ratio;
  k.pg = adv == 0.0f ? 0.0f : clipped ? -held * adv : -k.ratio * adv;
  k.d_cur = clipped ? 0.0f : -k.ratio * adv;
  k.kl = 0.0f;
  if (p.ref != nullptr) {
    float dkl;
    k.kl = kl_term(p.kl_form, __fsub_rn(ref, cur), dkl);
    k.d_cur = fmaf(p.kl_coef, dkl, k.d_cur);
  }
  return k;
}

// Sums over tokens: weighted policy, kl and entropy terms; counts; diagnostics.
struct Sums {
  double pg, kl, ent, diff, ratio, outside;
  float max_ratio;
};

struct Norm {
  double tokens, rows;
};

__device__ __forceinline__ double weight(const Params& p, double tokens, double rows, int row_count) {
  if (p.reduction == kTokenMean) return p.scale / (tokens > 0 ? tokens : 1.0);
  if (p.reduction == kSequenceMean) return p.scale / ((rows > 0 ? rows : 1.0) * double(row_count > 0 ? row_count : 1));
  return p.scale;
}

__global__ void __launch_bounds__(kThreads) count_kernel(Params p, int* __restrict__ counts) {
  pdl_begin();
  const int b = blockIdx.x;
  unsigned n = 0;
  for (int t = threadIdx.x; t < p.T; t += kThreads) n += p.mask == nullptr || p.mask[b * p.mask_s + t] != 0;
  __shared__ unsigned part[kThreads / 32];
  n = warp_sum_u32(n);
  if (threadIdx.x % 32 == 0) part[threadIdx.x / 32] = n;
  __syncthreads();
  if (threadIdx.x == 0) {
    unsigned s = 0;
    for (int i = 0; i < kThreads / 32; ++i) s += part[i];
    counts[b] = int(s);
  }
}

__global__ void norm_kernel(Params p, const int* __restrict__ counts, Norm* norm) {
  pdl_begin();
  double tokens = 0.0, rows = 0.0;
  for (int b = threadIdx.x; b < p.B; b += 32) {
    tokens += counts[b];
    rows += counts[b] > 0;
  }
  tokens = warp_sum(tokens);
  rows = warp_sum(rows);
  if (threadIdx.x == 0) *norm = Norm{tokens, rows};
}

__global__ void __launch_bounds__(kThreads) token_kernel(Params p, const int* __restrict__ counts,
                                                         const Norm* __restrict__ norm, Sums* __restrict__ sums) {
  pdl_begin();
  const int64_t b = blockIdx.x;
  const double w = weight(p, norm->tokens, norm->rows, counts[b]);
  const float wf = float(w);
  Sums a = {};
  for (int64_t t = threadIdx.x; t < p.T; t += kThreads) {
    const bool m = p.mask == nullptr || p.mask[b * p.mask_s + t] != 0;
    float g = 0.0f, ge = 0.0f;
    if (m) {
      const float cur = p.cur[b * p.cur_s + t];
      const Token k = token_loss(p, cur, p.old[b * p.old_s + t], p.adv[b * p.adv_s + t * p.adv_e],
                                 p.ref ? p.ref[b * p.ref_s + t] : 0.0f);
      a.pg += k.pg;
      a.kl += k.kl;
      if (p.ent) a.ent += p.ent[b * p.ent_s + t];
      a.diff += k.diff;
      a.ratio += k.ratio;
      a.outside += k.outside;
      a.max_ratio = fmaxf(a.max_ratio, k.ratio);
      g = k.d_cur * wf;
      ge = float(-w * p.ent_coef_d);
    }
    if (p.grad) p.grad[b * p.T + t] = g;
    if (p.grad_ent) p.grad_ent[b * p.T + t] = ge;
  }
  __shared__ Sums part[kThreads];
  part[threadIdx.x] = a;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < kThreads; ++i) {
      a.pg += part[i].pg;
      a.kl += part[i].kl;
      a.ent += part[i].ent;
      a.diff += part[i].diff;
      a.ratio += part[i].ratio;
      a.outside += part[i].outside;
      a.max_ratio = fmaxf(a.max_ratio, part[i].max_ratio);
    }
    a.pg *= w;
    a.kl *= w;
    a.ent *= w;
    sums[b] = a;
  }
}

__global__ void finish_kernel(Params p, const Norm* __restrict__ norm, const Sums* __restrict__ sums) {
  pdl_begin();
  Sums a = {};
  for (int b = 0; b < p.B; ++b) {
    a.pg += sums[b].pg;
    a.kl += sums[b].kl;
    a.ent += sums[b].ent;
    a.diff += sums[b].diff;
    a.ratio += sums[b].ratio;
    a.outside += sums[b].outside;
    a.max_ratio = fmaxf(a.max_ratio, sums[b].max_ratio);
  }
  const double n = norm->tokens > 0 ? norm->tokens : 1.0;
  p.out[0] = float(a.pg + p.kl_coef_d * a.kl - p.ent_coef_d * a.ent);
  p.out[1] = float(a.pg);
  p.out[2] = float(a.kl);
  p.out[3] = float(a.ent);
  p.out[4] = float(a.outside / n);
  p.out[5] = float(a.diff / n);
  p.out[6] = a.max_ratio;
  p.out[7] = float(a.ratio / n);
}

inline int64_t workspace_bytes(int32_t B, int32_t) {
  return int64_t(256 + align256(size_t(B) * sizeof(int)) + align256(size_t(B) * sizeof(Sums)));
}

// strides (host array): rows of log_prob, old, advantage, its elements (0 or 1), ref, entropy, mask.
inline int run(const float* cur, const float* old, const float* adv, const float* ref, const float* ent,
               const uint8_t* mask, const int64_t* strides, int32_t B, int32_t T, double clip_low, double clip_high,
               double dual_clip, double kl_coef, int kl_form, double ent_coef, int reduction, double scale, float* out,
               float* grad, float* grad_ent, void* ws, int64_t ws_bytes, cudaStream_t stream) {
  if (B < 0 || T < 0 || out == nullptr || strides == nullptr) return kInvalidArgument;
  if (!(clip_low >= 0.0 && clip_low < 1.0) || !(clip_high >= 0.0) || !(dual_clip == 0.0 || dual_clip > 1.0))
    return kInvalidArgument;
  if (kl_form < kK1 || kl_form > kK3 || reduction < kTokenMean || reduction > kSum) return kInvalidArgument;
  if (strides[3] != 0 && strides[3] != 1) return kInvalidArgument;
  if (B == 0 || T == 0)
    return cudaMemsetAsync(out, 0, kOutputs * sizeof(float), stream) == cudaSuccess ? kOk : kCudaError;
  if (cur == nullptr || old == nullptr || adv == nullptr || (grad_ent != nullptr && ent == nullptr))
    return kInvalidArgument;
  if (ws == nullptr || ws_bytes < workspace_bytes(B, T)) return kWorkspaceTooSmall;
  Params p;
  p.cur = cur, p.old = old, p.adv = adv, p.ref = ref, p.ent = ent, p.mask = mask;
  p.cur_s = strides[0], p.old_s = strides[1], p.adv_s = strides[2], p.adv_e = strides[3];
  p.ref_s = strides[4], p.ent_s = strides[5], p.mask_s = strides[6];
  p.B = B, p.T = T;
  p.log_high = make_pair_of(log1p(clip_high)), p.log_low = make_pair_of(log1p(-clip_low));
  p.log_dual = make_pair_of(dual_clip > 0.0 ? log(dual_clip) : 0.0);
  p.high = float(1.0 + clip_high), p.low = float(1.0 - clip_low), p.dual = float(dual_clip);
  p.kl_coef = float(kl_coef), p.ent_coef = float(ent_coef), p.kl_form = kl_form, p.reduction = reduction;
  p.scale = scale, p.kl_coef_d = kl_coef, p.ent_coef_d = ent_coef;
  p.grad = grad, p.grad_ent = grad_ent, p.out = out;
  char* w = static_cast<char*>(ws);
  Norm* norm = reinterpret_cast<Norm*>(w + 64);
  int* counts = reinterpret_cast<int*>(w + 256);
  Sums* sums = reinterpret_cast<Sums*>(w + 256 + align256(size_t(B) * sizeof(int)));
  int st = launch_pdl(count_kernel, dim3(B), dim3(kThreads), 0, stream, p, counts);
  if (st == kOk) st = launch_pdl(norm_kernel, dim3(1), dim3(32), 0, stream, p, static_cast<const int*>(counts), norm);
  if (st == kOk)
    st = launch_pdl(token_kernel, dim3(B), dim3(kThreads), 0, stream, p, static_cast<const int*>(counts),
                    static_cast<const Norm*>(norm), sums);
  if (st == kOk)
    st = launch_pdl(finish_kernel, dim3(1), dim3(1), 0, stream, p, static_cast<const Norm*>(norm),
                    static_cast<const Sums*>(sums));
  return st;
}

}  // namespace policy
}  // namespace b200
