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
//
// What bounds it: memory.  The forward reads each logit once, with a running maximum: a thread keeps (m, S, U)
// of the 16-byte vectors it has seen and rescales S and U when its maximum grows.  exp is one ex2 an
// element (16 a clock and SM, against some 12 bf16 logits a clock that HBM delivers: the forward runs close
// to both limits), everything else is packed two to an instruction.  The backward reads the logits once
// more and writes the gradient.
//
// Split: a warp per row where there are many rows for their length (warps_take), else a CTA per row (the backward: per
// piece of one), and in the forward, with few long rows, a cluster of up to 8 CTAs per row, each on a stretch of it, whose
// partial results meet in the first CTA's shared memory.
//
// Measured, bf16, forward and backward (a plain copy runs at 6.56 TB/s on the same GPU):
//   16 rows of 32768 (forward): 3.0 us (the smallest calls take 1.9);
//   4096 rows of 131072: 150 us and 335 us (6.4 TB/s, counting the rows that are masked, which only the backward
//   writes);
//   2044 rows of 50001: 36 us (5.7 TB/s) and 78 us (5.2 TB/s; 63 us at 50000, where rows are on 16 bytes);
//   37888 rows of 512: 19 us each (2 and 4 TB/s): a warp's row is then two vectors a lane, and the reductions over
//   the warp take longer than its loads.
#pragma once

#include <math.h>

#include "../common/bulk.cuh"
#include "../common/vec.cuh"

namespace b200 {
namespace lp {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kUnroll = 4;          // vectors in flight per thread
constexpr int kMaxCluster = 8;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
// Below this, 2^z is 0 in fp32: z is held above it so that 0 * z stays 0 (z = -inf at masked logits).
constexpr float kLowZ = -200.0f;

// (max, sum of 2^z, sum of 2^z z) of a part of a row, z = (x - m) * c2, c2 = inv * log2(e).
struct Acc {
  float m, s, u;
};

__device__ __forceinline__ Acc empty_acc() { return Acc{-INFINITY, 0.0f, 0.0f}; }

// a with its maximum moved to m >= a.m.
__device__ __forceinline__ void rebase(Acc& a, float m, float c2) {
  if (a.m == m) return;
  if (a.m > -INFINITY) {
    const float dz = (a.m - m) * c2;  // < 0, -inf where the old part vanishes beside the new maximum
    const float scale = exp2_approx(dz);
    a.u = (a.u + max_nan(dz, kLowZ) * a.s) * scale;
    a.s *= scale;
  }
  a.m = m;
}

__device__ __forceinline__ Acc shuffle(const Acc& a, int o) {
  return Acc{__shfl_xor_sync(0xffffffffu, a.m, o), __shfl_xor_sync(0xffffffffu, a.s, o),
             __shfl_xor_sync(0xffffffffu, a.u, o)};
}

__device__ __forceinline__ void merge(Acc& a, Acc b, float c2) {
  const float m = fmaxf(a.m, b.m);
  rebase(a, m, c2);
  rebase(b, m, c2);
  a.s += b.s;
  a.u += b.u;
}

// The warp's maximum is agreed on first, so each lane rescales once.
__device__ __forceinline__ void merge_warp(Acc& a, float c2) {
  rebase(a, warp_max(a.m), c2);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    a.s += __shfl_xor_sync(0xffffffffu, a.s, o);
    a.u += __shfl_xor_sync(0xffffffffu, a.u, o);
  }
}

template <bool kEnt>
__device__ __forceinline__ void add_one(Acc& a, float x, float c2) {
  if (x > a.m) rebase(a, x, c2);
  const float z = max_nan((x - (a.m > -INFINITY ? a.m : 0.0f)) * c2, kLowZ);
  const float e = exp2_approx(z);
  a.s += e;
  if (kEnt) a.u = fmaf(e, z, a.u);
}

// A running row part: packed sums over pairs of elements, in kSets sets: one where many threads share a row
// (registers are occupancy there), two where a warp has a row for itself (shorter chains of additions).
template <int kSets>
struct Run {
  float m;
  float2 s[kSets], u[kSets];
};
template <int kSets>
__device__ __forceinline__ void start_run(Run<kSets>& r, const Acc& a) {
  r.m = a.m;
#pragma unroll
  for (int k = 0; k < kSets; ++k) {
    r.s[k] = make_float2(k == 0 ? a.s : 0.0f, 0.0f);
    r.u[k] = make_float2(k == 0 ? a.u : 0.0f, 0.0f);
  }
}
template <int kSets>
__device__ __forceinline__ Acc total(const Run<kSets>& r) {
  float2 s = r.s[0], u = r.u[0];
#pragma unroll
  for (int k = 1; k < kSets; ++k) s = add2(s, r.s[k]), u = add2(u, r.u[k]);
  return Acc{r.m, s.x + s.y, u.x + u.y};
}

// kN vectors, of which the first n are there.
template <typename T, bool kEnt, int kN, int kSets>
__device__ __forceinline__ void add_vectors(Run<kSets>& r, const uint4 (&v)[kN], int n, float c2) {
  float top = -INFINITY;
#pragma unroll
  for (int k = 0; k < kN; ++k)
    if (k < n) top = fmaxf(top, max16<T>(v[k]));
  if (top > r.m) {
    Acc a = total(r);
    rebase(a, top, c2);
    start_run(r, a);
  }
  const float2 neg = splat2(r.m > -INFINITY ? -r.m : 0.0f), c = splat2(c2);
#pragma unroll
  for (int k = 0; k < kN; ++k) {
    if (k >= n) continue;
    float2 f[Vec16<T>::kPairs];
    unpack16<T>(v[k], f);
#pragma unroll
    for (int j = 0; j < Vec16<T>::kPairs; ++j) {
      float2 z = mul2(add2(f[j], neg), c);
      if (kEnt) z = make_float2(max_nan(z.x, kLowZ), max_nan(z.y, kLowZ));
      const float2 e = make_float2(exp2_approx(z.x), exp2_approx(z.y));
      const int set = j % kSets;
      r.s[set] = add2(r.s[set], e);
      if (kEnt) r.u[set] = fma2(e, z, r.u[set]);
    }
  }
}

// Elements of a row at p before the first 16-byte boundary.
template <typename T>
__device__ __forceinline__ int64_t head_elems(const T* p, int64_t V) {
  const int64_t h = int64_t((16 - (reinterpret_cast<uintptr_t>(p) & 15u)) & 15u) / int64_t(sizeof(T));
  return h < V ? h : V;
}

// Part `part` of `parts` of a row, by `kN` threads of which this is number `tid`.
template <typename T, bool kEnt, int kN>
__device__ __forceinline__ Acc row_part(const T* row, int64_t V, unsigned part, unsigned parts, int tid, float c2) {
  constexpr int kE = Vec16<T>::kElems;
  const int64_t head = head_elems(row, V), nv = (V - head) / kE;
  const unsigned per = (unsigned(nv) + parts - 1) / parts;
  const int64_t v0 = int64_t(per) * part, v1 = min(nv, v0 + per);
  const uint4* vec = reinterpret_cast<const uint4*>(row + head);
  // The elements before and behind the vectors, loaded first so that their wait overlaps the vectors'.
  const int64_t rest = head + nv * kE + tid;
  const bool has_head = part == 0 && tid < head, has_rest = part == 0 && rest < V;
  const float x_head = has_head ? to_f32(row[tid]) : 0.0f, x_rest = has_rest ? to_f32(row[rest]) : 0.0f;
  Run<kN == 32 ? 2 : 1> r;
  start_run(r, empty_acc());
  int64_t i = v0 + tid;
  for (; i + (kUnroll - 1) * kN < v1; i += kUnroll * kN) {
    uint4 v[kUnroll];
#pragma unroll
    for (int k = 0; k < kUnroll; ++k) v[k] = ld_stream_u4(vec + i + k * kN);
    add_vectors<T, kEnt>(r, v, kUnroll, c2);
  }
  if (i < v1) {
    uint4 v[kUnroll - 1];
    const int n = int((v1 - i + kN - 1) / kN);
#pragma unroll
    for (int k = 0; k < kUnroll - 1; ++k) v[k] = k < n ? ld_stream_u4(vec + i + k * kN) : make_uint4(0, 0, 0, 0);
    add_vectors<T, kEnt>(r, v, n, c2);
  }
  Acc a = total(r);
  if (has_head) add_one<kEnt>(a, x_head, c2);
  if (has_rest) add_one<kEnt>(a, x_rest, c2);
  return a;
}

struct Out {
  float *log_prob, *entropy, *stats;
};

// x_tok: the token's logit (NaN for a token that is not one).
template <bool kEnt>
__device__ __forceinline__ void write_row(const Out& o, int64_t r, const Acc& a, float x_tok, float inv) {
  const float log_s = logf(a.s);
  const float ent = kEnt ? log_s - kLn2 * (a.u / a.s) : NAN;  // not computed: no gradient of it either
  o.log_prob[r] = (x_tok - a.m) * inv - log_s;
  if (o.entropy) o.entropy[r] = ent;
  if (o.stats) {
    o.stats[3 * r] = a.m;
    o.stats[3 * r + 1] = log_s;
    o.stats[3 * r + 2] = ent;
  }
}
__device__ __forceinline__ void write_masked(const Out& o, int64_t r) {
  o.log_prob[r] = 0.0f;
  if (o.entropy) o.entropy[r] = 0.0f;
  if (o.stats)
    for (int k = 0; k < 3; ++k) o.stats[3 * r + k] = 0.0f;
}

struct Rows {
  int64_t xb, xt, kb, kt;  // element strides of logits and token over (batch, time)
  unsigned T;
  unsigned rows;
  int64_t V;
};

template <typename T>
__device__ __forceinline__ float token_logit(const T* row, int64_t tok, int64_t V) {
  return tok < V ? to_f32(row[tok]) : NAN;
}

// kWarpRows: a warp per row.  Otherwise gridDim.x / rows CTAs, one cluster, per row.
template <typename T, bool kEnt, bool kWarpRows>
__global__ void __launch_bounds__(kThreads) forward_kernel(const T* __restrict__ x, const int64_t* __restrict__ token,
                                                           Rows q, float inv, unsigned parts, Out out) {
  pdl_begin();
  const unsigned lane = threadIdx.x % 32, w = threadIdx.x / 32;
  const float c2 = inv * kLog2e;
  const unsigned part = kWarpRows ? 0u : blockIdx.x % parts;
  const unsigned r = kWarpRows ? blockIdx.x * kWarps + w : blockIdx.x / parts;
  if (kWarpRows && r >= q.rows) return;
  const unsigned b = r / q.T, t = r - b * q.T;
  const int64_t tok = token[b * q.kb + t * q.kt];
  if (tok < 0) {  // the whole cluster leaves: no barrier is waited at
    if (part == 0 && (kWarpRows ? lane == 0 : threadIdx.x == 0)) write_masked(out, r);
    return;
  }
  // Every CTA of the cluster runs before any of them writes to another (waited for below).
  if (!kWarpRows && parts > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  const T* row = x + b * q.xb + t * q.xt;
  const bool owner = part == 0 && (kWarpRows ? lane == 0 : threadIdx.x == 0);
  const float x_tok = owner ? token_logit(row, tok, q.V) : 0.0f;
  Acc a = row_part<T, kEnt, kWarpRows ? 32 : kThreads>(row, q.V, part, parts, kWarpRows ? lane : threadIdx.x, c2);
  merge_warp(a, c2);
  if (!kWarpRows) {
    __shared__ Acc warps[kWarps];
    __shared__ Acc ctas[kMaxCluster];
    if (lane == 0) warps[w] = a;
    if (parts > 1) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
    __syncthreads();
    if (w == 0) {
      a = lane < kWarps ? warps[lane] : empty_acc();
      merge_warp(a, c2);
      if (parts > 1 && lane == 0) {  // into the first CTA's ctas[part]
        uint32_t dst;
        asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(dst) : "r"(smem_addr(&ctas[part])));
        asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(dst), "f"(a.m) : "memory");
        asm volatile("st.shared::cluster.f32 [%0 + 4], %1;" ::"r"(dst), "f"(a.s) : "memory");
        asm volatile("st.shared::cluster.f32 [%0 + 8], %1;" ::"r"(dst), "f"(a.u) : "memory");
      }
    }
    if (parts > 1) {
      asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
      asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
      if (part != 0 || w != 0) return;
      a = lane < parts ? ctas[lane] : empty_acc();
      merge_warp(a, c2);
    }
  }
  if (owner) write_row<kEnt>(out, r, a, x_tok, inv);
}

// ------------------------------------------------------------------------------------ backward
struct Grad {
  const float *stats, *g_lp, *g_ent;
};

// grad_x = k_p p + k_e p z', z' = log2 p:  k_p = -inv (g_lp + g_ent entropy), k_e = -inv g_ent ln 2; the token's
// logit also gets inv g_lp.
struct Coef {
  float m, log_s2, k_p, k_e, k_tok;
};

template <bool kEnt>
__device__ __forceinline__ float2 grad_pair(float2 f, const Coef& k, float c2) {
  float2 z = fma2(add2(f, splat2(-k.m)), splat2(c2), splat2(-k.log_s2));
  if (kEnt) z = make_float2(max_nan(z.x, kLowZ), max_nan(z.y, kLowZ));
  const float2 p = make_float2(exp2_approx(z.x), exp2_approx(z.y));
  return mul2(p, kEnt ? fma2(splat2(k.k_e), z, splat2(k.k_p)) : splat2(k.k_p));
}
template <typename T, bool kEnt>
__device__ __forceinline__ T grad_one(float x, bool is_token, const Coef& k, float c2) {
  const float2 g = grad_pair<kEnt>(splat2(x), k, c2);
  return from_f32<T>(is_token ? g.x + k.k_tok : g.x);
}

template <typename T, bool kEnt>
__device__ __forceinline__ uint4 grad_vector(const uint4& v, int64_t first, int64_t tok, const Coef& k, float c2) {
  float2 f[Vec16<T>::kPairs];
  unpack16<T>(v, f);
#pragma unroll
  for (int j = 0; j < Vec16<T>::kPairs; ++j) f[j] = grad_pair<kEnt>(f[j], k, c2);
  const int64_t at = tok - first;
  if (at >= 0 && at < Vec16<T>::kElems) {
#pragma unroll
    for (int j = 0; j < Vec16<T>::kPairs; ++j) {
      if (at == 2 * j) f[j].x += k.k_tok;
      if (at == 2 * j + 1) f[j].y += k.k_tok;
    }
  }
  return pack16<T>(f);
}

// The 16 bytes at byte offset `off` (1 .. 15) of the 32 bytes (a, b).
__device__ __forceinline__ uint4 shifted(const uint4& a, const uint4& b, unsigned off) {
  uint4 lo = a;
  uint32_t next = b.x;
  if (off >= 12u) {
    lo = make_uint4(a.w, b.x, b.y, b.z), next = b.w;
  } else if (off >= 8u) {
    lo = make_uint4(a.z, a.w, b.x, b.y), next = b.z;
  } else if (off >= 4u) {
    lo = make_uint4(a.y, a.z, a.w, b.x), next = b.y;
  }
  const unsigned bits = (off & 3u) * 8u;
  return make_uint4(__funnelshift_r(lo.x, lo.y, bits), __funnelshift_r(lo.y, lo.z, bits),
                    __funnelshift_r(lo.z, lo.w, bits), __funnelshift_r(lo.w, next, bits));
}

// Rows cut into equal pieces of at most kPieceVecs vectors, a CTA (a warp of it for short rows) each.
constexpr int kPieceVecs = kThreads * kUnroll;

// Occupancy, measured at 4096 rows of 131072 bf16 logits: 6 CTAs per SM 335 us, 4 CTAs 384 us (4096 logits a
// row, warps: 5 CTAs 328 us, 6 CTAs, which spill, 352 us).
template <typename T, bool kEnt, bool kWarpRows>
__global__ void __launch_bounds__(kThreads, kWarpRows ? 5 : 6) backward_kernel(const T* x, const int64_t* __restrict__ token, Rows q,
                                                            float inv, unsigned pieces, Grad g, T* out) {
  pdl_begin();
  constexpr int kE = Vec16<T>::kElems;
  constexpr int kN = kWarpRows ? 32 : kThreads;
  const unsigned lane = threadIdx.x % 32;
  const int tid = kWarpRows ? int(lane) : int(threadIdx.x);
  const unsigned piece = kWarpRows ? 0u : blockIdx.x % pieces;
  const unsigned r = kWarpRows ? blockIdx.x * kWarps + threadIdx.x / 32 : blockIdx.x / pieces;
  if (kWarpRows && r >= q.rows) return;
  const unsigned b = r / q.T, t = r - b * q.T;
  const int64_t V = q.V;
  const int64_t tok = token[b * q.kb + t * q.kt];
  const T* row = x + b * q.xb + t * q.xt;
  T* dst = out + int64_t(r) * V;

  // The output's vectors; delta: bytes by which the input lies behind a 16-byte boundary there.  Where delta
  // is not 0 a vector is put together from two aligned ones, both inside the row.
  int64_t head = head_elems(dst, V);
  const unsigned delta = unsigned(reinterpret_cast<uintptr_t>(row + head) & 15u);
  if (delta != 0 && head * int64_t(sizeof(T)) < delta) head = head + kE < V ? head + kE : V;
  int64_t nv = (V - head) / kE;
  if (delta != 0 && nv > 0) {
    const int64_t room = (V - head) * int64_t(sizeof(T)) + delta;  // bytes from the first aligned block to the end
    nv = min(nv, room / 16 - 1);  // at least 0: room is above 16
  }
  const unsigned per = (unsigned(nv) + pieces - 1) / pieces;
  const int64_t v0 = int64_t(per) * piece, v1 = min(nv, v0 + per);
  const char* src = reinterpret_cast<const char*>(row + head) - delta;
  uint4* vec = reinterpret_cast<uint4*>(dst + head);
  const int64_t tail = head + nv * kE;

  if (tok < 0) {
    for (int64_t i = v0 + tid; i < v1; i += kN) vec[i] = make_uint4(0, 0, 0, 0);
    if (piece == 0) {
      for (int64_t i = tid; i < head; i += kN) dst[i] = from_f32<T>(0.0f);
      for (int64_t i = tail + tid; i < V; i += kN) dst[i] = from_f32<T>(0.0f);
    }
    return;
  }
  const float c2 = inv * kLog2e;
  Coef k;
  {
    const float gl = tok < V ? g.g_lp[r] : NAN, ge = kEnt ? g.g_ent[r] : 0.0f;
    k.m = g.stats[3 * int64_t(r)];
    k.log_s2 = g.stats[3 * int64_t(r) + 1] * kLog2e;
    k.k_p = -inv * (kEnt ? fmaf(ge, g.stats[3 * int64_t(r) + 2], gl) : gl);
    k.k_e = -inv * ge * kLn2;
    k.k_tok = inv * gl;
  }
  if (delta == 0) {
    for (int64_t i = v0 + tid; i < v1; i += kUnroll * kN) {
      uint4 v[kUnroll];
#pragma unroll
      for (int j = 0; j < kUnroll; ++j)
        if (i + j * kN < v1) v[j] = ld_once_u4(src + 16 * (i + j * kN));
#pragma unroll
      for (int j = 0; j < kUnroll; ++j) {
        const int64_t at = i + j * kN;
        if (at < v1) st_stream_u4(vec + at, grad_vector<T, kEnt>(v[j], head + at * kE, tok, k, c2));
      }
    }
  } else {
    // A lane's second block is the next lane's first, so whole warps go round together.
    for (int64_t i = v0 + tid; i - lane < v1; i += 2 * kN) {
      uint4 v[2], last[2];  // last: lane 31's second block
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int64_t at = i + j * kN;
        v[j] = at <= v1 ? ld_stream_u4(src + 16 * at) : make_uint4(0, 0, 0, 0);
        last[j] = lane == 31 && at < v1 ? ld_stream_u4(src + 16 * (at + 1)) : make_uint4(0, 0, 0, 0);
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        uint4 n;
        n.x = __shfl_down_sync(0xffffffffu, v[j].x, 1);
        n.y = __shfl_down_sync(0xffffffffu, v[j].y, 1);
        n.z = __shfl_down_sync(0xffffffffu, v[j].z, 1);
        n.w = __shfl_down_sync(0xffffffffu, v[j].w, 1);
        const int64_t at = i + j * kN;
        const uint4 x4 = shifted(v[j], lane == 31 ? last[j] : n, delta);
        if (at < v1) st_stream_u4(vec + at, grad_vector<T, kEnt>(x4, head + at * kE, tok, k, c2));
      }
    }
  }
  if (piece == 0) {
    for (int64_t i = tid; i < head; i += kN) dst[i] = grad_one<T, kEnt>(to_f32(row[i]), i == tok, k, c2);
    for (int64_t i = tail + tid; i < V; i += kN) dst[i] = grad_one<T, kEnt>(to_f32(row[i]), i == tok, k, c2);
  }
}

// ------------------------------------------------------------------------------------ host side
// 1 / temperature, and that times log2(e), are ordinary fp32 numbers.
inline bool temperature_ok(double temperature) { return temperature >= 1e-30 && temperature <= 1e30; }

inline int check(const void* logits, int dtype, const int64_t* strides, const int64_t* token, int32_t B, int32_t T,
                 int32_t V, double temperature) {
  if (B < 0 || T < 0 || V < 1 || !dtype_ok(dtype) || strides == nullptr || !temperature_ok(temperature))
    return kInvalidArgument;
  for (int i = 0; i < 4; ++i)
    if (strides[i] < 0) return kInvalidArgument;
  const int64_t rows = int64_t(B) * T;
  if (rows == 0) return kOk;
  if (logits == nullptr || token == nullptr || rows > 0x7fffffff) return kInvalidArgument;
  return -1;  // proceed
}

inline Rows rows_of(const int64_t* s, int32_t B, int32_t T, int32_t V) {
  return Rows{s[0], s[1], s[2], s[3], unsigned(T), unsigned(int64_t(B) * T), V};
}

template <typename F>
inline int with_flag(bool flag, F&& f) {
  return flag ? f(std::true_type{}) : f(std::false_type{});
}

// Whether a warp takes a row alone: the time of one row grows with its length then, while many warps share the GPU, and a
// CTA has its reductions to pay for, so it takes the more rows the longer they are.  The factor is where both are alike;
// measured, us, warp and CTA per row, bf16:
//   forward  V 512: 256 rows 2.5 and 3.0, 9472 rows 6.2 and 24;  V 2048: 256 rows 3.2 and 3.2, 9472 rows 9.8 and 28;
//            V 6000: 592 rows 6.4 and 4.9, 2368 rows 8.2 and 10.1, 37888 rows 87 and 136;
//            V 12000: 1184 rows 9.6 and 8.2, 37888 rows 141 and 188;  V 24000: 2368 rows 28 and 23, 37888 rows 266 and 293
//   backward V 512: 256 rows 2.2 and 2.7;  V 2048: 256 rows 3.7 and 2.5, 9472 rows 12.5 and 30;
//            V 6000: 2368 rows 11.5 and 11.6, 37888 rows 150 and 162;  V 12000: 9472 rows 81 and 78, 37888 rows 298 and 345
constexpr int64_t kForwardRows = 32768, kBackwardRows = 8192;
constexpr int64_t kWarpRowV = 32768;  // the longest row that was measured
inline bool warps_take(int64_t rows, int64_t V, int64_t factor) { return V <= kWarpRowV && rows * factor >= V * V; }

// CTAs per row: 1 once two CTAs per SM have a row each, else enough for that, but no CTA with fewer than
// 8192 logits: joining a cluster costs more than it saves there (64 rows of 50001 bf16 logits: 5.2 us with
// 4 CTAs a row, 6.2 us with 8; 2044 rows: 37 us with one, 42 us with 2, 56 us with 4).
inline unsigned cluster_of(int64_t rows, int64_t V) {
  unsigned c = 1;
  while (c < unsigned(kMaxCluster) && rows * c < 2 * sm_count() && V / (2 * c) >= 8192) c *= 2;
  return c;
}

// strides (host array): logits (batch, time), token (batch, time), in elements.
inline int forward(const void* logits, int dtype, const int64_t* strides, const int64_t* token, int32_t B, int32_t T,
                   int32_t V, double temperature, float* log_prob, float* entropy, float* stats,
                   cudaStream_t stream) {
  const int st = check(logits, dtype, strides, token, B, T, V, temperature);
  if (st >= 0) return st;
  if (log_prob == nullptr) return kInvalidArgument;
  const Rows q = rows_of(strides, B, T, V);
  const bool warp_rows = warps_take(q.rows, V, kForwardRows);
  const unsigned parts = warp_rows ? 1u : cluster_of(q.rows, V);
  const int64_t grid = warp_rows ? (int64_t(q.rows) + kWarps - 1) / kWarps : int64_t(q.rows) * parts;
  if (grid > 0x7fffffff) return kInvalidArgument;
  const Out out{log_prob, entropy, stats};
  return with_dtype(dtype, [&](auto e) {
    using E = decltype(e);
    return with_flag(entropy != nullptr, [&](auto ent) {
      return with_flag(warp_rows, [&](auto wr) {
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(unsigned(grid));
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
        return cudaLaunchKernelEx(&cfg, forward_kernel<E, decltype(ent)::value, decltype(wr)::value>,
                                  static_cast<const E*>(logits), token, q, float(1.0 / temperature), parts,
                                  out) == cudaSuccess
                   ? int(kOk)
                   : int(kCudaError);
      });
    });
  });
}

// grad_logits [B, T, V] may be the logits' own memory (then these are contiguous): every thread reads an
// element before it writes it, and no other reads it.
inline int backward(const void* logits, int dtype, const int64_t* strides, const int64_t* token, const float* stats,
                    const float* grad_log_prob, const float* grad_entropy, int32_t B, int32_t T, int32_t V,
                    double temperature, void* grad_logits, cudaStream_t stream) {
  const int st = check(logits, dtype, strides, token, B, T, V, temperature);
  if (st >= 0) return st;
  if (stats == nullptr || grad_log_prob == nullptr || grad_logits == nullptr) return kInvalidArgument;
  const Rows q = rows_of(strides, B, T, V);
  const bool warp_rows = warps_take(q.rows, V, kBackwardRows);
  const int64_t vecs = (int64_t(V) * dtype_size(dtype) + 15) / 16;
  const unsigned pieces = warp_rows ? 1u : unsigned((vecs + kPieceVecs - 1) / kPieceVecs);
  const int64_t grid = warp_rows ? (int64_t(q.rows) + kWarps - 1) / kWarps : int64_t(q.rows) * pieces;
  if (grid > 0x7fffffff) return kInvalidArgument;
  const Grad g{stats, grad_log_prob, grad_entropy};
  return with_dtype(dtype, [&](auto e) {
    using E = decltype(e);
    return with_flag(grad_entropy != nullptr, [&](auto ent) {
      return with_flag(warp_rows, [&](auto wr) {
        return launch_pdl(backward_kernel<E, decltype(ent)::value, decltype(wr)::value>, dim3(unsigned(grid)),
                          dim3(kThreads), 0, stream, static_cast<const E*>(logits), token, q, float(1.0 / temperature),
                          pieces, g, static_cast<E*>(grad_logits));
      });
    });
  });
}

}  // namespace lp
}  // namespace b200
