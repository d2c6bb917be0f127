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
//
// What bounds it: memory for many tokens, and for few the latency of a launch with its reductions.  One kernel does it
// all: the pair's slope is known as soon as its CTAs have met, and the gradients, constant along an answer, are
// written then.  Measured: 4 pairs of 700 and 523 tokens 6.7 us; 512 pairs of 8192 tokens with references and masks 20.1 us
// (5.4 TB/s); 2 pairs of 131072 tokens 17 us.
#pragma once

#include "../common/bulk.cuh"
#include "../common/dtype.cuh"
#include "../common/workspace.cuh"

namespace b200 {
namespace pref {

enum Form : int { kSigmoid = 0, kHinge = 1, kIpo = 2 };

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
  double beta, smoothing, margin, inv_B, inv_beta;
  int form;
  bool average;
  float* out;
};

// The derivative of the loss of margin z.
__device__ __forceinline__ double pair_slope(const Params& p, double z) {
  if (p.form == kSigmoid) {
    const double e = exp(-fabs(z)), inv = 1.0 / (1.0 + e);
    return z != z ? z : p.smoothing - (z >= 0.0 ? e * inv : inv);  // e - sigmoid(-z)
  }
  if (p.form == kHinge) return z < 1.0 ? -1.0 : 0.0;
  return 2.0 * (z - 0.5) * p.inv_beta * p.inv_beta;
}

// The loss of margin z.
__device__ __forceinline__ double pair_loss(const Params& p, double z) {
  if (p.form == kSigmoid) {
    const double tail = log1p(exp(-fabs(z)));  // softplus(z) = max(z, 0) + tail
    return (1.0 - p.smoothing) * (fmax(-z, 0.0) + tail) + p.smoothing * (fmax(z, 0.0) + tail);
  }
  if (p.form == kHinge) return z >= 1.0 ? 0.0 : 1.0 - z;  // NaN stays NaN
  const double u = (z - 0.5) * p.inv_beta;
  return u * u;
}

struct PairOut {
  double loss, win, gap;
};

// An answer's sum and number of tokens.
struct Part {
  double s;
  unsigned n;
};

// The workspace's control words: zero before the first call, and again after each.
struct Ctl {
  unsigned done;
};

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxCluster = 8;
constexpr int kVecs = 2;      // vectors of four tokens of a lane in flight, log-probs and references
constexpr int kPer = 4 * kVecs;

__device__ __forceinline__ double gap_of(float x, float r, bool on) {
  return on ? double(x) - double(r) : 0.0;
}

__device__ __forceinline__ unsigned ld_u8(const uint8_t* p) {
  unsigned v;
  asm volatile("ld.global.u8 %0, [%1];" : "=r"(v) : "l"(p));
  return v;
}
__device__ __forceinline__ uint32_t ld_u32(const uint8_t* p) {
  uint32_t v;
  asm volatile("ld.global.u32 %0, [%1];" : "=r"(v) : "l"(p));
  return v;
}

// One answer's row and a CTA's stretch of it.
struct Row {
  const float *lp, *ref;  // ref and mask may be null
  const uint8_t* mask;
  float* grad;
  int t0, t1;  // the stretch
  int v0, v1;  // of it, the part that is whole vectors of four tokens in every stream (v0 = v1: none)
};

// Rows start anywhere (every row of an odd length does), but where all streams are off their 16-byte (the mask: 4-byte)
// boundaries by the same number of tokens, vectors begin after the same few tokens in all of them.
__device__ __forceinline__ Row row_of(const Side& d, int64_t b, unsigned part, unsigned parts) {
  Row r;
  r.lp = d.lp + b * d.lp_s;
  r.ref = d.ref == nullptr ? nullptr : d.ref + b * d.ref_s;
  r.mask = d.mask == nullptr ? nullptr : d.mask + b * d.mask_s;
  r.grad = d.grad == nullptr ? nullptr : d.grad + b * d.T;
  const auto off = [](const float* p) { return unsigned(reinterpret_cast<uintptr_t>(p) >> 2) & 3u; };
  const unsigned o = off(r.lp);
  const bool same = (r.ref == nullptr || off(r.ref) == o) && (r.grad == nullptr || off(r.grad) == o) &&
                    (r.mask == nullptr || (unsigned(reinterpret_cast<uintptr_t>(r.mask)) & 3u) == o);
  const int head = min(d.T, int((4u - o) & 3u));
  const int per = int((unsigned(d.T - head) + 4 * parts - 1) / (4 * parts)) * 4;
  r.t0 = part == 0 ? 0 : int(min(int64_t(d.T), head + int64_t(per) * part));
  r.t1 = int(min(int64_t(d.T), head + int64_t(per) * (part + 1)));
  r.v0 = part == 0 ? head : r.t0;
  r.v1 = same ? r.v0 + ((r.t1 - r.v0) & ~3) : r.v0;
  return r;
}

// The stretch's sum and count.  What masked-out tokens hold is read with the others and not used.
__device__ __forceinline__ Part sum_stretch(const Row& d) {
  double s = 0.0;
  unsigned n = 0;
  for (int t = d.v0 + int(threadIdx.x) * 4; t < d.v1; t += kPer * kThreads) {
    float4 x[kVecs], r[kVecs];
    uint32_t on[kVecs];
#pragma unroll
    for (int k = 0; k < kVecs; ++k) {
      const int at = t + k * 4 * kThreads;
      const bool in = at < d.v1;
      x[k] = in ? ld_stream_f4(d.lp + at) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      r[k] = in && d.ref != nullptr ? ld_stream_f4(d.ref + at) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      on[k] = !in ? 0u : d.mask == nullptr ? 0x01010101u : ld_u32(d.mask + at);
    }
#pragma unroll
    for (int k = 0; k < kVecs; ++k) {
      s += (gap_of(x[k].x, r[k].x, on[k] & 0xffu) + gap_of(x[k].y, r[k].y, on[k] & 0xff00u)) +
           (gap_of(x[k].z, r[k].z, on[k] & 0xff0000u) + gap_of(x[k].w, r[k].w, on[k] & 0xff000000u));
      n += __popc(__vminu4(on[k], 0x01010101u));
    }
  }
  // The rest: the tokens before and behind the vectors, or, without vectors, all of them.
  const int before = d.v0 - d.t0, rest = before + d.t1 - d.v1;
  for (int i = threadIdx.x; i < rest; i += kPer * kThreads) {
    float x[kPer], r[kPer];
    unsigned on[kPer];
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      const int q = i + k * kThreads, at = q < before ? d.t0 + q : d.v1 + q - before;
      const bool in = q < rest;
      x[k] = in ? ld_stream_f1(d.lp + at) : 0.0f;
      r[k] = in && d.ref != nullptr ? ld_stream_f1(d.ref + at) : 0.0f;
      on[k] = !in ? 0u : d.mask == nullptr ? 1u : ld_u8(d.mask + at);
    }
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      s += gap_of(x[k], r[k], on[k] != 0u);
      n += on[k] != 0u;
    }
  }
  return Part{s, n};
}

__device__ __forceinline__ void write_stretch(const Row& d, float slope) {
  if (d.grad == nullptr) return;
  for (int t = d.v0 + int(threadIdx.x) * 4; t < d.v1; t += kPer * kThreads) {
    uint32_t on[kVecs];
#pragma unroll
    for (int k = 0; k < kVecs; ++k) {
      const int at = t + k * 4 * kThreads;
      on[k] = at < d.v1 && d.mask != nullptr ? ld_u32(d.mask + at) : ~0u;
    }
#pragma unroll
    for (int k = 0; k < kVecs; ++k) {
      const int at = t + k * 4 * kThreads;
      if (at < d.v1)
        st_stream_f4(d.grad + at, make_float4(on[k] & 0xffu ? slope : 0.0f, on[k] & 0xff00u ? slope : 0.0f,
                                              on[k] & 0xff0000u ? slope : 0.0f, on[k] & 0xff000000u ? slope : 0.0f));
    }
  }
  const int before = d.v0 - d.t0, rest = before + d.t1 - d.v1;
  for (int i = threadIdx.x; i < rest; i += kPer * kThreads) {
    unsigned on[kPer];
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      const int q = i + k * kThreads, at = q < before ? d.t0 + q : d.v1 + q - before;
      on[k] = q >= rest ? 0u : d.mask == nullptr ? 1u : ld_u8(d.mask + at);
    }
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      const int q = i + k * kThreads, at = q < before ? d.t0 + q : d.v1 + q - before;
      if (q < rest) d.grad[at] = on[k] != 0u ? slope : 0.0f;
    }
  }
}

// A cluster of `parts` CTAs per pair, each on a stretch of both answers: the CTAs exchange their sums through
// shared memory, every one forms the pair's slope from all of them in the same order and writes its
// stretch of the gradients.  The last CTA of the grid adds up the pairs in their order.
__global__ void __launch_bounds__(kThreads) pair_kernel(const __grid_constant__ Params p, unsigned parts, Ctl* ctl,
                                                        PairOut* pairs) {
  __shared__ Part warp_part[2][kWarps];
  __shared__ Part cta_part[2][kMaxCluster];
  __shared__ bool last;
  __shared__ double total[3][kWarps];
  const unsigned lane = threadIdx.x % 32, w = threadIdx.x / 32;
  const unsigned part = blockIdx.x % parts;
  const int64_t b = blockIdx.x / parts;
  pdl_begin();
  // Every CTA of the cluster runs before any of them writes to another (waited for below).
  if (parts > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  Row row[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    row[k] = row_of(p.side[k], b, part, parts);
    Part a = sum_stretch(row[k]);
    a.s = warp_sum(a.s);
    a.n = warp_sum_u32(a.n);
    if (lane == 0) warp_part[k][w] = a;
  }
  if (parts > 1) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
  __syncthreads();
  if (w < 2) {  // warp k: answer k
    Part a = lane < kWarps ? warp_part[w][lane] : Part{0.0, 0u};
    a.s = warp_sum(a.s);
    a.n = warp_sum_u32(a.n);
    if (lane < parts) {  // into CTA `lane`'s cta_part[w][part]
      if (parts == 1) {
        cta_part[w][0] = a;
      } else {
        uint32_t dst;
        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;"
                     : "=r"(dst)
                     : "r"(smem_addr(&cta_part[w][part])), "r"(lane));
        asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(dst), "d"(a.s) : "memory");
        asm volatile("st.shared::cluster.u32 [%0 + 8], %1;" ::"r"(dst), "r"(a.n) : "memory");
      }
    }
  }
  if (parts > 1) {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  } else {
    __syncthreads();
  }
  // Every thread forms the pair's slopes, so that no one waits for another to; one of them goes on to the loss while
  // the rest write gradients.
  double s[2], inv[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    Part a = cta_part[k][0];
    for (unsigned i = 1; i < parts; ++i) a.s += cta_part[k][i].s, a.n += cta_part[k][i].n;
    inv[k] = p.average ? 1.0 / double(a.n > 0 ? a.n : 1u) : 1.0;
    s[k] = a.s * inv[k];
  }
  const double gap = p.beta * (s[0] - s[1]), slope = p.beta * pair_slope(p, gap - p.margin) * p.inv_B;
  if (part == 0 && threadIdx.x == kThreads - 1) {
    pairs[b] = PairOut{pair_loss(p, gap - p.margin), s[0] > s[1] ? 1.0 : 0.0, gap};
    p.side[0].reward[b] = float(p.beta * s[0]);
    p.side[1].reward[b] = float(p.beta * s[1]);
    __threadfence();
    last = atomicAdd(&ctl->done, 1u) == unsigned(p.B) - 1u;
  }
  write_stretch(row[0], float(slope * inv[0]));
  write_stretch(row[1], float(-slope * inv[1]));
  if (part != 0) return;
  __syncthreads();
  if (!last) return;
  __threadfence();
  if (threadIdx.x == 0) ctl->done = 0u;
  double a[3] = {0.0, 0.0, 0.0};
  for (int i = threadIdx.x; i < p.B; i += kThreads) {
    a[0] += __ldcg(&pairs[i].loss);
    a[1] += __ldcg(&pairs[i].win);
    a[2] += __ldcg(&pairs[i].gap);
  }
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    a[k] = warp_sum(a[k]);
    if (lane == 0) total[k][w] = a[k];
  }
  __syncthreads();
  if (w == 0) {
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      const double s = warp_sum(lane < kWarps ? total[k][lane] : 0.0);
      if (lane == 0) p.out[k] = float(s * p.inv_B);
    }
  }
}

inline int64_t workspace_bytes(int32_t B) { return int64_t(256 + align256(size_t(B) * sizeof(PairOut))); }

// CTAs per pair: doubled while two CTAs per SM hold them all and none has fewer than 4096 tokens.  Measured with 1, 2, 4 and
// 8 CTAs per pair: 16 pairs of 2 x 16384 tokens 16.0, 12.0, 9.7 and 9.1 us, 64 of 2 x 4096 9.2, 8.9, 9.1 and 10.2, 256
// of 2 x 2048 8.3, 11.1, 14.0 and 20.6; a pair of 2 x 512 takes 6.4 us with one and 6.8 with two.  CTAs of 1024 threads
// took 1 to 3 us more than these of 256 up to 2 pairs of 2 x 32768 tokens, and twice the time for many pairs (2 pairs of 2 x
// 131072, 14 us against 17, are what they were good for).
inline unsigned cluster_of(int64_t pairs, int64_t tokens) {
  unsigned c = 1;
  while (c < unsigned(kMaxCluster) && pairs * 2 * c <= 2 * sm_count() && tokens / (2 * c) >= 4096) c *= 2;
  return c;
}

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
  for (int i = 0; i < 6; ++i)
    if (strides[i] < 0) return kInvalidArgument;
  if (B == 0) return cudaMemsetAsync(out, 0, kOutputs * sizeof(float), stream) == cudaSuccess ? kOk : kCudaError;
  if ((Tc > 0 && chosen == nullptr) || (Tr > 0 && rejected == nullptr) || reward_chosen == nullptr ||
      reward_rejected == nullptr)
    return kInvalidArgument;
  // Token indexes run in ints, up to a round of the CTA past the end.
  if (Tc > 0x7fffffff - 2 * kPer * kThreads || Tr > 0x7fffffff - 2 * kPer * kThreads) return kUnsupported;
  if (ws == nullptr || ws_bytes < workspace_bytes(B)) return kWorkspaceTooSmall;
  if (!aligned16(ws)) return kInvalidArgument;
  Params p;
  p.side[0] = Side{chosen, ref_chosen, chosen_mask, strides[0], strides[2], strides[4], Tc, reward_chosen, grad_chosen};
  p.side[1] =
      Side{rejected, ref_rejected, rejected_mask, strides[1], strides[3], strides[5], Tr, reward_rejected, grad_rejected};
  p.B = B, p.inv_B = 1.0 / B, p.inv_beta = 1.0 / beta, p.beta = beta, p.smoothing = smoothing, p.margin = margin, p.form = form, p.average = average != 0;
  p.out = out;
  const unsigned parts = cluster_of(B, int64_t(Tc) + Tr);
  if (int64_t(B) * parts > 0x7fffffff) return kUnsupported;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(B) * parts);
  cfg.blockDim = dim3(kThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = parts;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = parts > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, pair_kernel, p, parts, static_cast<Ctl*>(ws),
                            reinterpret_cast<PairOut*>(static_cast<char*>(ws) + 256)) == cudaSuccess
             ? kOk
             : kCudaError;
}

}  // namespace pref
}  // namespace b200
