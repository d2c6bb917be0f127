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
// What bounds it: memory for many tokens (25 bytes a token with all streams), a launch's latency for few.  The weights
// of the means need the number of tokens first, so a small kernel counts the mask (a byte a token) and the main one,
// whose loads run ahead meanwhile, follows it; up to kSmallTokens tokens and kSmallRows rows one CTA does both in one
// launch.  Measured: 16 x 256 tokens 4.6 us; 61 x 4099 11.3 us; 4096 x 1000 with an entropy 21.9 us (4.7 TB/s), 19.2
// us (5.3 TB/s) without the counting (sum).  Loads through registers, without the bulk copies, took 30 us.  With a
// reference and k3 instructions are the bound (25 us).
//
// A token is clipped or not by a step in its gradient, so the comparison is exact: cur - old as an
// unrounded pair of floats (s, e) against log(1 + clip_high) and log(1 - clip_low) as pairs.
#pragma once

#include <math.h>

#include "../common/bulk.cuh"
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

// exp(q) - 1 - q without the cancellation near 0: the Taylor series up to q^12 / 12!, for |q| <= 1 (the next
// term is below 2^-31 of the value).
__device__ __forceinline__ float2 exp_tail(float2 q) {
  float2 p = splat2(1.0f / 479001600.0f);
  p = fma2(p, q, splat2(1.0f / 39916800.0f));
  p = fma2(p, q, splat2(1.0f / 3628800.0f));
  p = fma2(p, q, splat2(1.0f / 362880.0f));
  p = fma2(p, q, splat2(1.0f / 40320.0f));
  p = fma2(p, q, splat2(1.0f / 5040.0f));
  p = fma2(p, q, splat2(1.0f / 720.0f));
  p = fma2(p, q, splat2(1.0f / 120.0f));
  p = fma2(p, q, splat2(1.0f / 24.0f));
  p = fma2(p, q, splat2(1.0f / 6.0f));
  p = fma2(p, q, splat2(0.5f));
  return mul2(mul2(q, q), p);
}
// The same for kPer values of any size: beyond 1 the difference itself, which costs at most some bits of expm1's.
__device__ __forceinline__ void exp_minus_1_minus(const float (&q)[4], float (&r)[4]) {
  const float2 a = exp_tail(make_float2(q[0], q[1])), b = exp_tail(make_float2(q[2], q[3]));
  r[0] = a.x, r[1] = a.y, r[2] = b.x, r[3] = b.y;
  if (fmaxf(fmaxf(fabsf(q[0]), fabsf(q[1])), fmaxf(fabsf(q[2]), fabsf(q[3]))) > 1.0f) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (fabsf(q[j]) > 1.0f) r[j] = expm1f(q[j]) - q[j];
  }
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
  float mid, half, band;  // the clip range of d is mid +- half; within band of its borders the pairs decide
  float high, low, dual;  // 1 + clip_high, 1 - clip_low, c (infinite: off)
  float kl_coef, ent_coef;
  int kl_form, reduction;
  float scale;
  double kl_coef_d, ent_coef_d;
  float *grad, *grad_ent, *out;
};

// Weighted sums of the policy, kl and entropy terms; over the tokens that count the sum of exp(d) - 1 - d, the
// largest d, their number and that of those outside the clip range; the sum of r over all tokens seen, r = 1 at
// those that do not count, and the number of these.
struct Sums {
  double pg, kl, ent, diff, ratio;
  float max_d;
  unsigned outside, tokens, skipped;
};
__device__ __forceinline__ Sums no_sums() { return Sums{0.0, 0.0, 0.0, 0.0, 0.0, -INFINITY, 0u, 0u, 0u}; }

// The workspace's control words: zero before the first call, and again after each.
struct Ctl {
  unsigned done, rows;
  unsigned long long tokens;
};

// The weight of a token: three roundings at most.
__device__ __forceinline__ float token_weight(const Params& p, unsigned long long tokens, unsigned rows, int row_tokens) {
  if (p.reduction == kTokenMean) return __fdiv_rn(p.scale, float(tokens > 0 ? tokens : 1ull));
  if (p.reduction == kSequenceMean)
    return __fdiv_rn(p.scale, float(rows > 0 ? rows : 1u) * float(row_tokens > 0 ? row_tokens : 1));
  return p.scale;
}

// The tokens of one lane as they are read: kPer consecutive ones (p.vec), or kPer a warp's width apart.  What
// masked-out tokens hold is read with the others and not used.
constexpr int kPer = 4;

struct Raw {
  float cur[kPer], old[kPer], adv[kPer], ref[kPer], ent[kPer];
  unsigned row[kPer];
  uint32_t on;  // byte j: 0xff where token j counts, else 0
};
__device__ __forceinline__ uint32_t count_word(uint32_t mask_bytes) { return __vminu4(mask_bytes, 0x01010101u) * 0xffu; }
// All bits set where token j counts, else none.
template <int j>
__device__ __forceinline__ uint32_t bits_of(uint32_t on) {
  return __byte_perm(on, 0u, j * 0x1111u);
}
__device__ __forceinline__ float keep(float v, uint32_t bits) { return __uint_as_float(__float_as_uint(v) & bits); }

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
    r.on = p.mask == nullptr ? ~0u : count_word(*reinterpret_cast<const uint32_t*>(p.mask + at(p.mask_s)));
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
      if (p.mask == nullptr || p.mask[at(p.mask_s)] != 0) r.on |= 0xffu << (8 * j);
      r.cur[j] = ld_stream_f1(p.cur + at(p.cur_s));
      r.old[j] = ld_stream_f1(p.old + at(p.old_s));
      r.adv[j] = p.adv_rows ? p.adv[b * p.adv_s] : ld_stream_f1(p.adv + at(p.adv_s));
      if (p.ref != nullptr) r.ref[j] = ld_stream_f1(p.ref + at(p.ref_s));
      if (p.ent != nullptr) r.ent[j] = ld_stream_f1(p.ent + at(p.ent_s));
    }
  }
}

__device__ __forceinline__ float sum4(const float (&v)[kPer]) {
  const float2 s = add2(make_float2(v[0], v[1]), make_float2(v[2], v[3]));
  return s.x + s.y;
}

__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// Four tokens of one lane: their terms are added in fp32 in a tree and then to the running sums in fp64; g and ge
// are their gradients.  weight: each token's.  Instructions are what this costs, so a masked-out token is not
// branched around: its values are cleared by bits, d = 0 and A = 0, and it adds r = 1 alone.
//   With e = d - mid, d is outside the clip range where |e| > half, and its gradient is cut there where A e > 0
//   (A > 0 is held at 1 + clip_high, A < 0 at 1 - clip_low).
__device__ __forceinline__ void take_tokens(const Params& p, const Raw& r, const float (&weight)[kPer], Sums& a,
                                            float (&g)[kPer], float (&ge)[kPer]) {
  const uint32_t bits[kPer] = {bits_of<0>(r.on), bits_of<1>(r.on), bits_of<2>(r.on), bits_of<3>(r.on)};
  float s[kPer], A[kPer], e[kPer];
  bool close = false;
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const float d = __fsub_rn(r.cur[j], r.old[j]);
    A[j] = keep(r.adv[j], bits[j]);
    s[j] = keep(d, bits[j]);
    a.max_d = fmaxf(a.max_d, __uint_as_float(__float_as_uint(d) | ~bits[j]));  // a NaN does not count
    e[j] = s[j] - p.mid;
    close |= fabsf(fabsf(e[j]) - p.half) <= p.band;
  }
  if (close) {  // roundings decide: e from the exact differences
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      float d, rest;
      two_diff(r.cur[j], r.old[j], d, rest);
      if (bits[j] != 0u)
        e[j] = above(d, rest, p.log_high) ? INFINITY : below(d, rest, p.log_low) ? -INFINITY : 0.0f;
    }
  }
  float ratio[kPer], diff[kPer], pg[kPer];
#pragma unroll
  for (int j = 0; j < kPer; j += 2) {
    const float2 z = mul2(make_float2(s[j], s[j + 1]), splat2(1.4426950408889634f));
    ratio[j] = exp2_approx(z.x), ratio[j + 1] = exp2_approx(z.y);
  }
  exp_minus_1_minus(s, diff);
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    // (A = 0 times an infinite e is NaN and not above 0.)
    const bool out = fabsf(e[j]) > p.half, held = out && A[j] * e[j] > 0.0f;
    // A ratio beyond fp32 is held at its largest value, so that A = 0 adds 0.
    const float v = held ? (A[j] > 0.0f ? p.high : p.low) : min_nan(ratio[j], 3.402823466e38f);
    pg[j] = v * (-A[j] * weight[j]);
    g[j] = held ? 0.0f : pg[j];
    if (out) a.outside += 1u;
  }
  if (p.dual < INFINITY) {
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      float d, rest;
      two_diff(r.cur[j], r.old[j], d, rest);
      if (A[j] < 0.0f && above(d, rest, p.log_dual)) {
        pg[j] = p.dual * (-A[j] * weight[j]);
        g[j] = 0.0f;
      }
    }
  }
  const unsigned n = __popc(r.on) / 8;
  a.tokens += n;
  a.skipped += kPer - n;
  a.pg += double(sum4(pg));
  a.diff += double(sum4(diff));
  a.ratio += double(sum4(ratio));
  if (p.ref != nullptr) {
    float q[kPer], kl[kPer], dkl[kPer];
#pragma unroll
    for (int j = 0; j < kPer; ++j) q[j] = keep(__fsub_rn(r.ref[j], r.cur[j]), bits[j]);
    if (p.kl_form == kK1) {
#pragma unroll
      for (int j = 0; j < kPer; ++j) kl[j] = -q[j], dkl[j] = keep(1.0f, bits[j]);
    } else if (p.kl_form == kK2) {
#pragma unroll
      for (int j = 0; j < kPer; ++j) kl[j] = 0.5f * q[j] * q[j], dkl[j] = -q[j];
    } else {
      exp_minus_1_minus(q, kl);
#pragma unroll
      for (int j = 0; j < kPer; ++j) dkl[j] = -(q[j] + kl[j]);  // 1 - exp(q)
    }
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      g[j] = fmaf(p.kl_coef * weight[j], dkl[j], g[j]);
      kl[j] *= weight[j];
    }
    a.kl += double(sum4(kl));
  }
  if (p.ent != nullptr) {
    float h[kPer];
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      h[j] = keep(r.ent[j] * weight[j], bits[j]);
      ge[j] = keep(-p.ent_coef * weight[j], bits[j]);
    }
    a.ent += double(sum4(h));
  } else {
#pragma unroll
    for (int j = 0; j < kPer; ++j) ge[j] = 0.0f;
  }
}

template <bool kVec>
__device__ __forceinline__ void write_tokens(const Params& p, unsigned first, const float (&g)[kPer],
                                             const float (&ge)[kPer]) {
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
  a.max_d = warp_max(a.max_d);
  a.outside = warp_sum_u32(a.outside);
  a.tokens = warp_sum_u32(a.tokens);
  a.skipped = warp_sum_u32(a.skipped);
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
    a = lane < kW ? part[lane] : no_sums();
    sum_warp(a);
  }
}

__device__ __forceinline__ void write_outputs(const Params& p, const Sums& a) {
  const double inv = 1.0 / double(a.tokens > 0u ? a.tokens : 1u);
  p.out[0] = float(a.pg + p.kl_coef_d * a.kl - p.ent_coef_d * a.ent);
  p.out[1] = float(a.pg);
  p.out[2] = float(a.kl);
  p.out[3] = float(a.ent);
  p.out[4] = float(double(a.outside) * inv);
  p.out[5] = float(a.diff * inv);
  p.out[6] = a.tokens > 0u ? exp2_approx(a.max_d * 1.4426950408889634f) : 0.0f;
  p.out[7] = float((a.ratio - double(a.skipped)) * inv);
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
  const unsigned on = warp_sum_u32(__popc(r.on) / 8);
  if (threadIdx.x % 32 == 0 && on > 0) atomicAdd(&total, on);
  if (per_row) {
#pragma unroll
    for (int j = 0; j < kPer; ++j)
      if ((r.on >> (8 * j)) & 1u) atomicAdd(&row_tokens[r.row[j]], 1);
  }
  __syncthreads();
  if (per_row) {
    for (int b = threadIdx.x; b < p.B; b += kSmallThreads)
      if (row_tokens[b] > 0) atomicAdd(&rows, 1u);
    __syncthreads();
  }
  Sums a = no_sums();
  float w[kPer];
#pragma unroll
  for (int j = 0; j < kPer; ++j)
    w[j] = per_row || j == 0 ? token_weight(p, total, rows, per_row ? row_tokens[r.row[j]] : 0) : w[0];
  float g[kPer], ge[kPer];
  take_tokens(p, r, w, a, g, ge);
  write_tokens<kVec>(p, first, g, ge);
  sum_block<kSmallThreads / 32>(a);
  if (threadIdx.x == 0) write_outputs(p, a);
}

// ------------------------------------------------------------------- many tokens: counts, then terms
// Counts of the masked tokens, in all (token mean) or per row (sequence mean): rows cut into stretches, a warp
// each.  Whole-number atomics, so the order does not matter.
constexpr int kStretch = 1024;

__device__ __forceinline__ unsigned ones16(const uint4& x) {
  return __popc(__vminu4(x.x, 0x01010101u)) + __popc(__vminu4(x.y, 0x01010101u)) + __popc(__vminu4(x.z, 0x01010101u)) +
         __popc(__vminu4(x.w, 0x01010101u));
}

// Adds the CTA's numbers to the control words.
__device__ __forceinline__ void add_counts(Ctl* ctl, unsigned tokens, unsigned rows) {
  __shared__ unsigned part[2][kThreads / 32];
  tokens = warp_sum_u32(tokens);
  rows = warp_sum_u32(rows);
  if (threadIdx.x % 32 == 0) part[0][threadIdx.x / 32] = tokens, part[1][threadIdx.x / 32] = rows;
  __syncthreads();
  if (threadIdx.x < 32) {
    const bool in = threadIdx.x < kThreads / 32;
    tokens = warp_sum_u32(in ? part[0][threadIdx.x] : 0u);
    rows = warp_sum_u32(in ? part[1][threadIdx.x] : 0u);
    if (threadIdx.x == 0) {
      if (tokens > 0) atomicAdd(&ctl->tokens, (unsigned long long)(tokens));
      if (rows > 0) atomicAdd(&ctl->rows, rows);
    }
  }
}

__global__ void __launch_bounds__(kThreads) count_rows_kernel(const __grid_constant__ Params p, unsigned stretches,
                                                              Ctl* ctl, int* counts) {
  pdl_begin();
  const unsigned lane = threadIdx.x % 32;
  const uint64_t warps = uint64_t(gridDim.x) * (kThreads / 32);
  unsigned tokens = 0, rows = 0;
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
    for (int i = lane; i < vecs; i += 32) c += ones16(__ldg(v + i));
    c = warp_sum_u32(c);
    if (lane == 0 && c > 0) {
      if (p.reduction == kSequenceMean)
        rows += atomicAdd(&counts[b], int(c)) == 0;  // the add that finds an empty row counts it
      tokens += c;
    }
  }
  add_counts(ctl, tokens, rows);
}

// All tokens of a dense mask on a 16-byte boundary.
__global__ void __launch_bounds__(kThreads) count_all_kernel(const uint8_t* __restrict__ mask, unsigned n, Ctl* ctl) {
  pdl_begin();
  const uint4* v = reinterpret_cast<const uint4*>(mask);
  const unsigned vecs = n / 16, threads = gridDim.x * kThreads, id = blockIdx.x * kThreads + threadIdx.x;
  unsigned c = 0;
  for (unsigned i = id; i < vecs; i += 4 * threads) {
    uint4 x[4];
#pragma unroll
    for (unsigned k = 0; k < 4; ++k)
      x[k] = i + k * threads < vecs ? __ldg(v + i + k * threads) : make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int k = 0; k < 4; ++k) c += ones16(x[k]);
  }
  if (id < n - vecs * 16) c += mask[vecs * 16 + id] != 0;
  add_counts(ctl, c, 0u);
}

// What the counts say, for every CTA of a kernel behind a count kernel.
struct Counts {
  unsigned long long tokens;
  unsigned rows;
};
__device__ __forceinline__ Counts read_counts(const Params& p, bool counted, Ctl* ctl) {
  if (!counted) return Counts{(unsigned long long)(p.n), unsigned(p.B)};
  return Counts{*reinterpret_cast<volatile unsigned long long*>(&ctl->tokens), ld_cg_u32(&ctl->rows)};
}

// The end of a kernel of many CTAs: each writes its sums, the last adds them up in their order, writes the
// outputs and leaves the workspace as it was.
__device__ __forceinline__ void finish(const Params& p, Sums& a, bool counted, Ctl* ctl, int* counts, Sums* sums) {
  sum_block<kThreads / 32>(a);
  if (threadIdx.x == 0) sums[blockIdx.x] = a;
  if (!elect_last_cta(&ctl->done)) return;
  a = no_sums();
  for (unsigned i = threadIdx.x; i < gridDim.x; i += kThreads) {
    const Sums& s = sums[i];
    a.pg += __ldcg(&s.pg);
    a.kl += __ldcg(&s.kl);
    a.ent += __ldcg(&s.ent);
    a.diff += __ldcg(&s.diff);
    a.ratio += __ldcg(&s.ratio);
    a.max_d = fmaxf(a.max_d, __ldcg(&s.max_d));
    a.outside += __ldcg(&s.outside);
    a.tokens += __ldcg(&s.tokens);
    a.skipped += __ldcg(&s.skipped);
  }
  sum_block<kThreads / 32>(a);
  if (threadIdx.x == 0) {
    write_outputs(p, a);
    ctl->tokens = 0ull;
    ctl->rows = 0u;
  }
  if (p.reduction == kSequenceMean && counted)
    for (int b = threadIdx.x; b < p.B; b += kThreads) counts[b] = 0;
}

// Any layout: a CTA takes stretches of kThreads * kPer tokens, grid-stride, through registers.
template <bool kVec>
__global__ void __launch_bounds__(kThreads) token_kernel(const __grid_constant__ Params p, bool counted, Ctl* ctl,
                                                         int* counts, Sums* sums) {
  constexpr unsigned kStretchTokens = kThreads * kPer;
  const unsigned units = (p.n + kStretchTokens - 1) / kStretchTokens;
  pdl_begin();
  const bool per_row = p.reduction == kSequenceMean;
  const Counts c = read_counts(p, counted, ctl);
  float w[kPer];
#pragma unroll
  for (int j = 0; j < kPer; ++j) w[j] = j == 0 ? token_weight(p, c.tokens, c.rows, p.T) : w[0];
  Sums a = no_sums();
  for (unsigned u = blockIdx.x; u < units; u += gridDim.x) {
    const unsigned first = first_token<kVec>(u, kThreads);
    Raw r;
    load_tokens<kVec>(p, first, r);
    if (per_row && counted) {
#pragma unroll
      for (int j = 0; j < kPer; ++j) w[j] = token_weight(p, c.tokens, c.rows, counts[r.row[j]]);
    }
    float g[kPer], ge[kPer];
    take_tokens(p, r, w, a, g, ge);
    write_tokens<kVec>(p, first, g, ge);
  }
  finish(p, a, counted, ctl, counts, sums);
}

// Dense streams on 16-byte boundaries: stretches of kUnit tokens arrive in shared memory by bulk copies, kStages
// ahead, so that loads never wait for arithmetic.  A thread has four consecutive tokens of a stretch.  What is left of
// less than a stretch goes through registers.
// Measured with inputs and outputs out of L2, 4096 x 1000 tokens with an entropy (the same with reduction sum, and 16384 x
// 1000 of that): 24.9 us (22.4, 67.0: 6.1 TB/s); with three stages 24.5 (23.4, 75.4), with two of 2048 tokens 26.6 (24.4,
// 76.7), with four CTAs per SM, whose 64 registers spill, 29.3 (25.9, 73.4).
// Behind a count kernel the copies start before the counts are there: every CTA of that lets this kernel
// start only after it has itself waited for the kernels before it, so the inputs are complete.
constexpr int kStages = 2;
constexpr unsigned kUnit = kThreads * kPer;
constexpr unsigned kStreamBytes = kUnit * 4u;

struct Streams {
  const float* p[5];  // cur, old, adv, ref, ent; null: not there
  int slot[5];        // its place in a stage
  int n;              // streams that are there
};

__global__ void __launch_bounds__(kThreads, 3) dense_kernel(const __grid_constant__ Params p,
                                                            const __grid_constant__ Streams st, bool counted, Ctl* ctl,
                                                            int* counts, Sums* sums) {
  extern __shared__ __align__(128) char smem[];
  __shared__ uint64_t full[kStages];
  const unsigned whole = p.n / kUnit;
  const unsigned stage_bytes = unsigned(st.n) * kStreamBytes + (p.mask != nullptr ? kUnit : 0u);
  if (threadIdx.x == 0) {
    for (int k = 0; k < kStages; ++k) mbar_init(&full[k], 1);
    fence_barrier_init();
  }
  __syncthreads();
  if (!counted) pdl_begin();
  const auto fetch = [&](unsigned u, unsigned stage) {  // thread 0
    if (u >= whole) return;
    char* dst = smem + stage * stage_bytes;
    mbar_arrive_expect_tx(&full[stage], stage_bytes);
#pragma unroll
    for (int s = 0; s < 5; ++s)
      if (st.p[s] != nullptr)
        bulk_g2s(dst + st.slot[s] * kStreamBytes, st.p[s] + size_t(u) * kUnit, kStreamBytes, &full[stage]);
    if (p.mask != nullptr) bulk_g2s(dst + st.n * kStreamBytes, p.mask + size_t(u) * kUnit, kUnit, &full[stage]);
  };
  if (threadIdx.x == 0)
    for (unsigned k = 0; k < unsigned(kStages); ++k) fetch(blockIdx.x + k * gridDim.x, k);
  if (counted) pdl_begin();
  const bool per_row = p.reduction == kSequenceMean;
  const Counts c = read_counts(p, counted, ctl);
  float w[kPer];
#pragma unroll
  for (int j = 0; j < kPer; ++j) w[j] = j == 0 ? token_weight(p, c.tokens, c.rows, p.T) : w[0];
  Sums a = no_sums();
  unsigned stage = 0, parity = 0;
  for (unsigned u = blockIdx.x; u < whole; u += gridDim.x) {
    mbar_wait(&full[stage], parity);
    const char* base = smem + stage * stage_bytes;
    const unsigned at = threadIdx.x, first = u * kUnit + at * kPer;
    Raw r;
    const auto take4 = [&](int s, float (&f)[kPer]) {
      const float4 v = *reinterpret_cast<const float4*>(base + st.slot[s] * kStreamBytes + at * (kPer * 4));
      f[0] = v.x, f[1] = v.y, f[2] = v.z, f[3] = v.w;
    };
    if (p.need_row) {
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        const bool again = j > 0 && p.T % kPer == 0;  // the first token's row
        const unsigned row = again ? r.row[0] : p.by_T.div(first + j);
        r.row[j] = row;
        if (per_row && counted) w[j] = again ? w[0] : token_weight(p, c.tokens, c.rows, counts[row]);
        if (p.adv_rows) r.adv[j] = again ? r.adv[0] : p.adv[int64_t(row) * p.adv_s];
      }
    }
    take4(0, r.cur);
    take4(1, r.old);
    if (!p.adv_rows) take4(2, r.adv);
    if (p.ref != nullptr) take4(3, r.ref);
    if (p.ent != nullptr) take4(4, r.ent);
    r.on = p.mask == nullptr
               ? ~0u
               : count_word(*reinterpret_cast<const uint32_t*>(base + st.n * kStreamBytes + at * kPer));
    float g[kPer], ge[kPer];
    take_tokens(p, r, w, a, g, ge);
    write_tokens<true>(p, first, g, ge);
    __syncthreads();  // the stage is read
    if (threadIdx.x == 0) fetch(u + kStages * gridDim.x, stage);
    if (++stage == unsigned(kStages)) stage = 0, parity ^= 1u;
  }
  if (blockIdx.x == gridDim.x - 1 && whole * kUnit < p.n) {
    const unsigned first = whole * kUnit + threadIdx.x * kPer;
    Raw r;
    load_tokens<true>(p, first, r);
    if (per_row && counted) {
#pragma unroll
      for (int j = 0; j < kPer; ++j) w[j] = token_weight(p, c.tokens, c.rows, counts[r.row[j]]);
    }
    float g[kPer], ge[kPer];
    take_tokens(p, r, w, a, g, ge);
    write_tokens<true>(p, first, g, ge);
  }
  finish(p, a, counted, ctl, counts, sums);
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
  if (!(clip_low >= 0.0 && clip_low < 1.0) || !(clip_high >= 0.0 && clip_high < INFINITY) || !(dual_clip == 0.0 || dual_clip > 1.0))
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
  {
    // d - mid and half carry some roundings relative to the borders' sizes: band covers them.
    const double H = log1p(clip_high), L = log1p(-clip_low);
    p.mid = float((H + L) / 2), p.half = float((H - L) / 2);
    p.band = float((fabs(H) + fabs(L)) * 1e-6) + 1e-30f;
  }
  p.high = float(1.0 + clip_high), p.low = float(1.0 - clip_low), p.dual = dual_clip > 0.0 ? float(dual_clip) : INFINITY;
  p.kl_coef = float(kl_coef), p.ent_coef = float(ent_coef), p.kl_form = kl_form, p.reduction = reduction;
  p.scale = float(scale), p.kl_coef_d = kl_coef, p.ent_coef_d = ent_coef;
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
    int st;
    if (reduction == kTokenMean && (p.mask_s == T || B == 1) && aligned16(mask)) {
      const int64_t want = (n / 16 + 4 * kThreads - 1) / (4 * kThreads), most = int64_t(sm_count()) * 2;
      st = launch_pdl(count_all_kernel, dim3(unsigned(want < 1 ? 1 : want < most ? want : most)), dim3(kThreads), 0,
                      stream, mask, p.n, ctl);
    } else {
      const unsigned stretches = unsigned((int64_t(T) + kStretch - 1) / kStretch);
      const int64_t warps = int64_t(B) * stretches;
      const int64_t want = (warps + kThreads / 32 - 1) / (kThreads / 32), most = int64_t(sm_count()) * 4;
      st = launch_pdl(count_rows_kernel, dim3(unsigned(want < most ? want : most)), dim3(kThreads), 0, stream, p,
                      stretches, ctl, counts);
    }
    if (st != kOk) return st;
  }
  const auto grid = [&](int per_sm, unsigned stretch) {
    const int64_t units = (n + stretch - 1) / stretch;
    const int64_t most = int64_t(sm_count()) * per_sm;
    return unsigned(most < units ? (most < kMaxCtas ? most : kMaxCtas) : (units < kMaxCtas ? units : kMaxCtas));
  };
  if (p.dense && p.vec && (mask == nullptr || aligned16(mask))) {
    Streams st = {};
    const float* all[5] = {cur, old, p.adv_rows ? nullptr : adv, ref, ent};
    for (int s = 0; s < 5; ++s) {
      st.p[s] = all[s];
      if (all[s] != nullptr) st.slot[s] = st.n++;
    }
    const int smem = kStages * int(unsigned(st.n) * kStreamBytes + (mask != nullptr ? kUnit : 0u));
    if (!ensure_dyn_smem(dense_kernel, smem)) return kCudaError;
    return launch_pdl(dense_kernel, dim3(grid(resident_ctas_per_sm(dense_kernel, kThreads, size_t(smem)), kUnit)),
                      dim3(kThreads), size_t(smem), stream, p, st, counted, ctl, counts, sums);
  }
  const auto kernel = p.vec ? token_kernel<true> : token_kernel<false>;
  return launch_pdl(kernel, dim3(grid(resident_ctas_per_sm(kernel, kThreads, 0), kThreads * kPer)), dim3(kThreads), 0, stream, p, counted,
                    ctl, counts, sums);
}

}  // namespace policy
}  // namespace b200
