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

#include <math.h>

#include "../common/vec.cuh"
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

// exp(q) - 1 - q without the cancellation near 0: its Taylor series up to q^12 / 12! for |q| <= 1 (the next
// term is below 2^-31 of the value), the difference beyond, where it costs at most some bits of expm1's.
__device__ __forceinline__ float exp_minus_1_minus(float q) {
  if (fabsf(q) > 1.0f) return expm1f(q) - q;
  float p = 1.0f / 479001600.0f;
  p = fmaf(p, q, 1.0f / 39916800.0f);
  p = fmaf(p, q, 1.0f / 3628800.0f);
  p = fmaf(p, q, 1.0f / 362880.0f);
  p = fmaf(p, q, 1.0f / 40320.0f);
  p = fmaf(p, q, 1.0f / 5040.0f);
  p = fmaf(p, q, 1.0f / 720.0f);
  p = fmaf(p, q, 1.0f / 120.0f);
  p = fmaf(p, q, 1.0f / 24.0f);
  p = fmaf(p, q, 1.0f / 6.0f);
  p = fmaf(p, q, 0.5f);
  return q * q * p;
}

// i / d for i < 2^31 by a multiplication (d >= 1).
struct FastDiv {
  unsigned d, mul, shift;
  __device__ __forceinline__ unsigned div(unsigned i) const { return d == 1u ? i : __umulhi(i, mul) >> shift; }
};
inline FastDiv fast_div(unsigned d) {
  unsigned l = 0;
  while ((uint64_t(1) << l) < d) ++l;  // 2^(l-1) < d <= 2^l
  return FastDiv{d, unsigned(((uint64_t(1) << (31 + l)) + d - 1) / d), l > 0 ? l - 1 : 0u};
}

struct Params {
  const float *cur, *old, *adv, *ref, *ent;
  const uint8_t* mask;
  int64_t cur_s, old_s, adv_s, ref_s, ent_s, mask_s;  // row strides
  int B, T;
  unsigned n;      // B * T
  FastDiv by_T;
  bool dense;      // every stream's row stride is T: a token has one offset in all of them
  bool vec;        // four consecutive tokens are one aligned vector of every stream
  bool adv_rows;   // one advantage per row
  bool need_row;   // a token's row is needed
  Pair log_high, log_low, log_dual;
  float high, low, dual;  // 1 + clip_high, 1 - clip_low, c (0: off)
  float kl_coef, ent_coef;
  int kl_form, reduction;
  double scale, kl_coef_d, ent_coef_d;
  float *grad, *grad_ent, *out;
};

// Weighted sums of the policy, kl and entropy terms; over the masked tokens the sums of exp(d) - 1 - d and of
// r, the largest r, and the counts of tokens and of those outside the clip range.
struct Sums {
  double pg, kl, ent, diff, ratio;
  float max_ratio;
  unsigned outside, tokens;
};

// The workspace's control words: zero before the first call, and again after each.
struct Ctl {
  unsigned done, rows;
  unsigned long long tokens;
};

__device__ __forceinline__ float token_weight(const Params& p, unsigned long long tokens, unsigned rows, int row_tokens) {
  if (p.reduction == kTokenMean) return float(p.scale / double(tokens > 0 ? tokens : 1ull));
  if (p.reduction == kSequenceMean)
    return float(p.scale / (double(rows > 0 ? rows : 1u) * double(row_tokens > 0 ? row_tokens : 1)));
  return float(p.scale);
}

// The tokens of one lane as they are read: kPer consecutive ones (p.vec), or kPer a warp's width apart.  What
// masked-out tokens hold is read with the others and not used.
constexpr int kPer = 4;

struct Raw {
  float cur[kPer], old[kPer], adv[kPer], ref[kPer], ent[kPer];
  unsigned row[kPer];
  unsigned on;  // bit j: token j counts
};

__device__ __forceinline__ void load4(const float* p, int64_t at, float (&f)[kPer]) {
  const float4 v = ld_stream_f4(p + at);
  f[0] = v.x, f[1] = v.y, f[2] = v.z, f[3] = v.w;
}

// First token and distance between the tokens of a lane, in stretch u of `threads` * kPer tokens.
template <bool kVec>
__device__ __forceinline__ unsigned first_token(unsigned u, unsigned threads) {
  const unsigned at = u * threads * kPer;
  return kVec ? at + threadIdx.x * kPer : at + threadIdx.x / 32 * (32 * kPer) + threadIdx.x % 32;
}
template <bool kVec>
__device__ __forceinline__ unsigned token_of(unsigned first, int j) {
  return kVec ? first + j : first + j * 32;
}

template <bool kVec>
__device__ __forceinline__ void load_tokens(const Params& p, unsigned first, Raw& r) {
  r.on = 0u;
#pragma unroll
  for (int j = 0; j < kPer; ++j) r.cur[j] = r.old[j] = r.adv[j] = r.ref[j] = r.ent[j] = 0.0f, r.row[j] = 0u;
  if (kVec && first + kPer <= p.n) {
    unsigned t = first;
    if (p.need_row) {
      if (p.T % kPer == 0) {
        r.row[0] = p.by_T.div(first);
        t = first - r.row[0] * unsigned(p.T);
        r.row[1] = r.row[2] = r.row[3] = r.row[0];
      } else {
#pragma unroll
        for (int j = 0; j < kPer; ++j) r.row[j] = p.by_T.div(first + j);
      }
    }
    const int64_t b = r.row[0];
    const auto at = [&](int64_t stride) { return p.dense ? int64_t(first) : b * stride + t; };
    uint32_t m = 0x01010101u;
    if (p.mask != nullptr) m = __vminu4(*reinterpret_cast<const uint32_t*>(p.mask + at(p.mask_s)), 0x01010101u);
    load4(p.cur, at(p.cur_s), r.cur);
    load4(p.old, at(p.old_s), r.old);
    if (p.adv_rows) {
#pragma unroll
      for (int j = 0; j < kPer; ++j) r.adv[j] = p.adv[int64_t(r.row[j]) * p.adv_s];
    } else {
      load4(p.adv, at(p.adv_s), r.adv);
    }
    if (p.ref != nullptr) load4(p.ref, at(p.ref_s), r.ref);
    if (p.ent != nullptr) load4(p.ent, at(p.ent_s), r.ent);
    r.on = (m * 0x10204080u) >> 28;  // bit 8 j of m to bit j
  } else {
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const unsigned i = token_of<kVec>(first, j);
      if (i >= p.n) continue;
      unsigned t = i;
      if (p.need_row) {
        r.row[j] = p.by_T.div(i);
        t = i - r.row[j] * unsigned(p.T);
      }
      const int64_t b = r.row[j];
      const auto at = [&](int64_t stride) { return p.dense ? int64_t(i) : b * stride + t; };
      if (p.mask == nullptr || p.mask[at(p.mask_s)] != 0) r.on |= 1u << j;
      r.cur[j] = ld_stream_f1(p.cur + at(p.cur_s));
      r.old[j] = ld_stream_f1(p.old + at(p.old_s));
      r.adv[j] = p.adv_rows ? p.adv[b * p.adv_s] : ld_stream_f1(p.adv + at(p.adv_s));
      if (p.ref != nullptr) r.ref[j] = ld_stream_f1(p.ref + at(p.ref_s));
      if (p.ent != nullptr) r.ent[j] = ld_stream_f1(p.ent + at(p.ent_s));
    }
  }
}

// What a token adds: policy, kl and entropy terms weighted with w, exp(d) - 1 - d, r; and its gradient.
struct Terms {
  float pg, kl, ent, diff, ratio;
};

__device__ __forceinline__ float take_token(const Params& p, const Raw& r, int j, float w, Sums& a, Terms& k) {
  k = Terms{0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
  if (((r.on >> j) & 1u) == 0u) return 0.0f;
  const float cur = r.cur[j], adv = r.adv[j];
  const float s = __fsub_rn(cur, r.old[j]);
  bool hi = s > p.log_high.hi, lo = s < p.log_low.hi;
  bool dual = adv < 0.0f && s > p.log_dual.hi;
  if (s == p.log_high.hi || s == p.log_low.hi || s == p.log_dual.hi) {  // the rounding decides: look at it
    float d, e;
    two_diff(cur, r.old[j], d, e);
    hi = above(s, e, p.log_high);
    lo = below(s, e, p.log_low);
    dual = adv < 0.0f && above(s, e, p.log_dual);
  }
  k.ratio = exp2_approx(s * 1.4426950408889634f);
  k.diff = exp_minus_1_minus(s);
  const bool clipped = (adv > 0.0f && hi) || (adv < 0.0f && lo) || dual || adv == 0.0f;
  const float held = dual ? p.dual : hi ? p.high : p.low;
  const float pg = adv == 0.0f ? 0.0f : (clipped ? held : k.ratio) * -adv;
  float g = clipped ? 0.0f : pg;
  if (p.ref != nullptr) {
    const float q = __fsub_rn(r.ref[j], cur);
    float dkl;
    if (p.kl_form == kK1) {
      k.kl = -q, dkl = 1.0f;
    } else if (p.kl_form == kK2) {
      k.kl = 0.5f * q * q, dkl = -q;
    } else {
      k.kl = exp_minus_1_minus(q), dkl = -(q + k.kl);  // 1 - exp(q)
    }
    g = fmaf(p.kl_coef, dkl, g);
    k.kl *= w;
  }
  k.pg = pg * w;
  k.ent = r.ent[j] * w;
  a.max_ratio = fmaxf(a.max_ratio, k.ratio);
  a.outside += hi || lo;
  return g * w;
}

// The tokens of one lane: their terms are added in fp32 in a tree and then to the running sums in fp64, their
// gradients are written.  w: each token's weight.
template <bool kVec>
__device__ __forceinline__ void take_tokens(const Params& p, unsigned first, const Raw& r, const float (&w)[kPer],
                                            Sums& a) {
  Terms k[kPer];
  float g[kPer], ge[kPer];
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    g[j] = take_token(p, r, j, w[j], a, k[j]);
    ge[j] = ((r.on >> j) & 1u) != 0u ? -w[j] * p.ent_coef : 0.0f;
  }
  a.tokens += __popc(r.on);
  a.pg += double((k[0].pg + k[1].pg) + (k[2].pg + k[3].pg));
  if (p.ref != nullptr) a.kl += double((k[0].kl + k[1].kl) + (k[2].kl + k[3].kl));
  if (p.ent != nullptr) a.ent += double((k[0].ent + k[1].ent) + (k[2].ent + k[3].ent));
  a.diff += double((k[0].diff + k[1].diff) + (k[2].diff + k[3].diff));
  a.ratio += double((k[0].ratio + k[1].ratio) + (k[2].ratio + k[3].ratio));
  if (kVec && first + kPer <= p.n) {
    if (p.grad) st_stream_f4(p.grad + first, make_float4(g[0], g[1], g[2], g[3]));
    if (p.grad_ent) st_stream_f4(p.grad_ent + first, make_float4(ge[0], ge[1], ge[2], ge[3]));
  } else {
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const unsigned i = token_of<kVec>(first, j);
      if (i >= p.n) continue;
      if (p.grad) p.grad[i] = g[j];
      if (p.grad_ent) p.grad_ent[i] = ge[j];
    }
  }
}

// The warp's sums, in a fixed order; lane 0 has them all.
__device__ __forceinline__ void sum_warp(Sums& a) {
  a.pg = warp_sum(a.pg);
  a.kl = warp_sum(a.kl);
  a.ent = warp_sum(a.ent);
  a.diff = warp_sum(a.diff);
  a.ratio = warp_sum(a.ratio);
  a.max_ratio = warp_max(a.max_ratio);
  a.outside = warp_sum_u32(a.outside);
  a.tokens = warp_sum_u32(a.tokens);
}
template <int kW>
__device__ __forceinline__ void sum_block(Sums& a) {
  __shared__ Sums part[kW];
  const unsigned lane = threadIdx.x % 32, w = threadIdx.x / 32;
  sum_warp(a);
  __syncthreads();
  if (lane == 0) part[w] = a;
  __syncthreads();
  if (w == 0) {
    a = lane < kW ? part[lane] : Sums{};
    sum_warp(a);
  }
}

// tokens: fp64 holds the counts' sum of any size.
__device__ __forceinline__ void write_outputs(const Params& p, const Sums& a, double tokens, double outside) {
  const double n = tokens > 0 ? tokens : 1.0;
  p.out[0] = float(a.pg + p.kl_coef_d * a.kl - p.ent_coef_d * a.ent);
  p.out[1] = float(a.pg);
  p.out[2] = float(a.kl);
  p.out[3] = float(a.ent);
  p.out[4] = float(outside / n);
  p.out[5] = float(a.diff / n);
  p.out[6] = a.max_ratio;
  p.out[7] = float(a.ratio / n);
}

// --------------------------------------------------------------------------- few tokens: one CTA
constexpr int kSmallThreads = 1024;
constexpr unsigned kSmallTokens = kPer * kSmallThreads;
constexpr int kSmallRows = 2048;

template <bool kVec>
__global__ void __launch_bounds__(kSmallThreads) small_kernel(const __grid_constant__ Params p) {
  __shared__ int row_tokens[kSmallRows];
  __shared__ unsigned total, rows;
  const bool per_row = p.reduction == kSequenceMean;
  if (per_row)
    for (int b = threadIdx.x; b < p.B; b += kSmallThreads) row_tokens[b] = 0;
  if (threadIdx.x == 0) total = rows = 0u;
  pdl_begin();
  __syncthreads();
  Raw r;
  const unsigned first = first_token<kVec>(0u, kSmallThreads);
  load_tokens<kVec>(p, first, r);
  const unsigned on = warp_sum_u32(__popc(r.on));
  if (threadIdx.x % 32 == 0 && on > 0) atomicAdd(&total, on);
  if (per_row) {
#pragma unroll
    for (int j = 0; j < kPer; ++j)
      if ((r.on >> j) & 1u) atomicAdd(&row_tokens[r.row[j]], 1);
  }
  __syncthreads();
  if (per_row) {
    for (int b = threadIdx.x; b < p.B; b += kSmallThreads)
      if (row_tokens[b] > 0) atomicAdd(&rows, 1u);
    __syncthreads();
  }
  Sums a = {};
  float w[kPer];
#pragma unroll
  for (int j = 0; j < kPer; ++j)
    w[j] = per_row || j == 0 ? token_weight(p, total, rows, per_row ? row_tokens[r.row[j]] : 0) : w[0];
  take_tokens<kVec>(p, first, r, w, a);
  sum_block<kSmallThreads / 32>(a);
  if (threadIdx.x == 0) write_outputs(p, a, double(a.tokens), double(a.outside));
}

// ------------------------------------------------------------------- many tokens: counts, then terms
// Counts of the masked tokens, in all (token mean) or per row (sequence mean): rows cut into stretches, a warp
// each.  Whole-number atomics, so the order does not matter.
constexpr int kStretch = 4096;

__global__ void __launch_bounds__(kThreads) count_kernel(const Params p, unsigned stretches, Ctl* ctl, int* counts) {
  pdl_begin();
  const unsigned lane = threadIdx.x % 32;
  const uint64_t warps = uint64_t(gridDim.x) * (kThreads / 32);
  unsigned long long tokens = 0;
  unsigned rows = 0;
  for (uint64_t u = uint64_t(blockIdx.x) * (kThreads / 32) + threadIdx.x / 32; u < uint64_t(p.B) * stretches; u += warps) {
    const int64_t b = int64_t(u / stretches);
    const int t0 = int(u - uint64_t(b) * stretches) * kStretch;
    const int len = min(kStretch, p.T - t0);
    const uint8_t* m = p.mask + b * p.mask_s + t0;
    const int head = min(len, int((16 - (reinterpret_cast<uintptr_t>(m) & 15u)) & 15u));
    const int vecs = (len - head) / 16, tail = head + vecs * 16;
    unsigned c = 0;
    if (int(lane) < head) c += m[lane] != 0;
    if (tail + int(lane) < len) c += m[tail + lane] != 0;
    const uint4* v = reinterpret_cast<const uint4*>(m + head);
#pragma unroll 4
    for (int i = lane; i < vecs; i += 32) {
      const uint4 x = __ldg(v + i);
      c += __popc(__vminu4(x.x, 0x01010101u)) + __popc(__vminu4(x.y, 0x01010101u)) +
           __popc(__vminu4(x.z, 0x01010101u)) + __popc(__vminu4(x.w, 0x01010101u));
    }
    c = warp_sum_u32(c);
    if (lane == 0 && c > 0) {
      if (p.reduction == kSequenceMean)
        rows += atomicAdd(&counts[b], int(c)) == 0;  // the add that finds an empty row counts it
      tokens += c;
    }
  }
  __shared__ unsigned long long s_tokens;
  __shared__ unsigned s_rows;
  if (threadIdx.x == 0) s_tokens = 0ull, s_rows = 0u;
  __syncthreads();
  if (lane == 0 && tokens > 0) {
    atomicAdd(&s_tokens, tokens);
    atomicAdd(&s_rows, rows);
  }
  __syncthreads();
  if (threadIdx.x == 0 && s_tokens > 0) {
    atomicAdd(&ctl->tokens, s_tokens);
    if (s_rows > 0) atomicAdd(&ctl->rows, s_rows);
  }
}

// Bytes of all streams' L2 prefetch, at most: lines prefetched beyond it would be evicted before their use.
constexpr int64_t kPrefetchBytes = 48 << 20;

// A CTA takes stretches of kThreads * kPer tokens, grid-stride.  counted: count_kernel ran before; while it does,
// this kernel brings its first stretches into L2 (their own reads wait for it).
template <bool kVec>
__global__ void __launch_bounds__(kThreads, 4) token_kernel(const __grid_constant__ Params p, bool counted,
                                                            unsigned prefetch, Ctl* ctl, int* counts, Sums* sums) {
  constexpr unsigned kUnit = kThreads * kPer;
  const unsigned units = (p.n + kUnit - 1) / kUnit;
  if (counted && p.dense) {
    const float* streams[5] = {p.cur, p.old, p.adv_rows ? nullptr : p.adv, p.ref, p.ent};
    for (unsigned u = blockIdx.x, k = 0; u < units && k < prefetch; u += gridDim.x, ++k) {
      const unsigned at = u * kUnit + threadIdx.x * 32;  // a 128-byte line per thread
      if (threadIdx.x < kUnit / 32 && at < p.n)
#pragma unroll
        for (int s = 0; s < 5; ++s)
          if (streams[s] != nullptr) asm volatile("prefetch.global.L2 [%0];" ::"l"(streams[s] + at));
    }
  }
  pdl_begin();
  const bool per_row = p.reduction == kSequenceMean;
  const unsigned rows = counted ? ld_cg_u32(&ctl->rows) : unsigned(p.B);
  const unsigned long long tokens =
      counted ? *reinterpret_cast<volatile unsigned long long*>(&ctl->tokens) : (unsigned long long)(p.n);
  float w[kPer];
#pragma unroll
  for (int j = 0; j < kPer; ++j) w[j] = j == 0 ? token_weight(p, tokens, rows, p.T) : w[0];
  Sums a = {};
  for (unsigned u = blockIdx.x; u < units; u += gridDim.x) {
    const unsigned first = first_token<kVec>(u, kThreads);
    Raw r;
    load_tokens<kVec>(p, first, r);
    if (per_row && counted) {
#pragma unroll
      for (int j = 0; j < kPer; ++j)
        w[j] = kVec && j > 0 && r.row[j] == r.row[j - 1] ? w[j - 1] : token_weight(p, tokens, rows, counts[r.row[j]]);
    }
    take_tokens<kVec>(p, first, r, w, a);
  }
  sum_block<kThreads / 32>(a);
  if (threadIdx.x == 0) sums[blockIdx.x] = a;
  if (!elect_last_cta(&ctl->done)) return;
  a = Sums{};
  double all = 0.0, out = 0.0;
  for (unsigned i = threadIdx.x; i < gridDim.x; i += kThreads) {
    const Sums& s = sums[i];
    a.pg += __ldcg(&s.pg);
    a.kl += __ldcg(&s.kl);
    a.ent += __ldcg(&s.ent);
    a.diff += __ldcg(&s.diff);
    a.ratio += __ldcg(&s.ratio);
    a.max_ratio = fmaxf(a.max_ratio, __ldcg(&s.max_ratio));
    a.outside += __ldcg(&s.outside);
    a.tokens += __ldcg(&s.tokens);
  }
  sum_block<kThreads / 32>(a);
  if (threadIdx.x == 0) {
    all = double(a.tokens), out = double(a.outside);
    write_outputs(p, a, all, out);
    ctl->tokens = 0ull;
    ctl->rows = 0u;
  }
  if (per_row && counted)
    for (int b = threadIdx.x; b < p.B; b += kThreads) counts[b] = 0;
}

// ------------------------------------------------------------------------------------ host side
constexpr int kMaxCtas = 2048;
constexpr size_t kSumsBytes = kMaxCtas * sizeof(Sums);

inline int64_t workspace_bytes(int32_t B, int32_t T) {
  if (int64_t(B) * T <= kSmallTokens && B <= kSmallRows) return 0;
  return int64_t(256 + kSumsBytes + align256(size_t(B) * sizeof(int)));
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
  for (int i = 0; i < 7; ++i)
    if (strides[i] < 0) return kInvalidArgument;
  if (strides[3] > 1) return kInvalidArgument;
  if (B == 0 || T == 0)
    return cudaMemsetAsync(out, 0, kOutputs * sizeof(float), stream) == cudaSuccess ? kOk : kCudaError;
  if (cur == nullptr || old == nullptr || adv == nullptr || (grad_ent != nullptr && ent == nullptr))
    return kInvalidArgument;
  const int64_t n = int64_t(B) * T;
  if (n > 0x7fffffff - 2 * int64_t(kSmallTokens)) return kUnsupported;  // token indexes are 31 bits
  const int64_t need = workspace_bytes(B, T);
  if (need > 0 && (ws == nullptr || ws_bytes < need)) return kWorkspaceTooSmall;
  if (need > 0 && !aligned16(ws)) return kInvalidArgument;
  Params p = {};
  p.cur = cur, p.old = old, p.adv = adv, p.ref = ref, p.ent = ent, p.mask = mask;
  p.cur_s = strides[0], p.old_s = strides[1], p.adv_s = strides[2], p.adv_rows = strides[3] == 0;
  p.ref_s = strides[4], p.ent_s = strides[5], p.mask_s = strides[6];
  p.B = B, p.T = T, p.n = unsigned(n), p.by_T = fast_div(unsigned(T));
  const auto dense = [&](const void* q, int64_t s) { return q == nullptr || s == T || B == 1; };
  p.dense = dense(cur, p.cur_s) && dense(old, p.old_s) && (p.adv_rows || dense(adv, p.adv_s)) && dense(ref, p.ref_s) &&
            dense(ent, p.ent_s) && dense(mask, p.mask_s);
  p.need_row = !p.dense || p.adv_rows || reduction == kSequenceMean;
  p.log_high = make_pair_of(log1p(clip_high)), p.log_low = make_pair_of(log1p(-clip_low));
  p.log_dual = make_pair_of(dual_clip > 0.0 ? log(dual_clip) : double(NAN));  // NaN: no difference is it
  p.high = float(1.0 + clip_high), p.low = float(1.0 - clip_low), p.dual = float(dual_clip);
  p.kl_coef = float(kl_coef), p.ent_coef = float(ent_coef), p.kl_form = kl_form, p.reduction = reduction;
  p.scale = scale, p.kl_coef_d = kl_coef, p.ent_coef_d = ent_coef;
  p.grad = grad, p.grad_ent = grad_ent, p.out = out;
  const auto aligned = [&](const void* q, int64_t s) {
    return q == nullptr || (aligned16(q) && (p.dense || (T % kPer == 0 && s % kPer == 0)));
  };
  p.vec = aligned(cur, p.cur_s) && aligned(old, p.old_s) && (p.adv_rows || aligned(adv, p.adv_s)) &&
          aligned(ref, p.ref_s) && aligned(ent, p.ent_s) && aligned(grad, T) && aligned(grad_ent, T) &&
          (mask == nullptr || (reinterpret_cast<uintptr_t>(mask) % kPer == 0 &&
                               (p.dense || (T % kPer == 0 && p.mask_s % kPer == 0))));
  if (need == 0)
    return launch_pdl(p.vec ? small_kernel<true> : small_kernel<false>, dim3(1), dim3(kSmallThreads), 0, stream, p);

  char* w = static_cast<char*>(ws);
  Ctl* ctl = reinterpret_cast<Ctl*>(w);
  Sums* sums = reinterpret_cast<Sums*>(w + 256);
  int* counts = reinterpret_cast<int*>(w + 256 + kSumsBytes);
  const bool counted = mask != nullptr && reduction != kSum;
  if (counted) {
    const unsigned stretches = unsigned((int64_t(T) + kStretch - 1) / kStretch);
    const int64_t warps = int64_t(B) * stretches;
    const int64_t want = (warps + kThreads / 32 - 1) / (kThreads / 32), most = int64_t(sm_count()) * 4;
    const int st = launch_pdl(count_kernel, dim3(unsigned(want < most ? want : most)), dim3(kThreads), 0, stream, p,
                              stretches, ctl, counts);
    if (st != kOk) return st;
  }
  const int64_t units = (n + kThreads * kPer - 1) / (kThreads * kPer);
  int64_t ctas = int64_t(sm_count()) * resident_ctas_per_sm(token_kernel<true>, kThreads, 0);
  if (ctas > kMaxCtas) ctas = kMaxCtas;
  if (ctas > units) ctas = units;
  const int streams = 2 + !p.adv_rows + (ref != nullptr) + (ent != nullptr);
  const int64_t unit_bytes = int64_t(kThreads) * kPer * 4 * streams;
  const unsigned prefetch = unsigned(kPrefetchBytes / (unit_bytes * ctas));
  return launch_pdl(p.vec ? token_kernel<true> : token_kernel<false>, dim3(unsigned(ctas)), dim3(kThreads), 0, stream, p, counted, prefetch, ctl, counts,
                    sums);
}

}  // namespace policy
}  // namespace b200
