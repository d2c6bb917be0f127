// Gated linear recurrence: T steps, B*H independent channels, state in fp32.
//
//   h[b,t,c] = a[b,t,c] * h[b,t-1,c] + v[b,t,c],   h[b,-1,c] = state[b,c] (0 without a state)
//     decay form:    a = gate,           v = x
//     sigmoid form:  a = sigmoid(gate),  v = (1 - a) * x
//   reset[b,t] != 0 drops h[b,t-1] (the first step of a packed document).
// Backward, with g[T] = 0 and a[t+1] = 0 where reset[t+1]:
//   g[t] = grad_h[t] + a[t+1] * g[t+1]      (grad_h[T-1] also takes grad_final)
//     decay:    grad_x = g,            grad_gate = g * h[t-1]
//     sigmoid:  grad_x = (1 - a) * g,  grad_gate = g * (h[t-1] - x) * a * (1 - a)
//   grad_state = a[0] * g[0]            (h[t-1] and grad_state are 0 over a reset)
#pragma once

#include <type_traits>

#include "../common/dtype.cuh"

namespace b200 {
namespace linrec {

enum Form : int { kDecay = 0, kSigmoid = 1 };

constexpr int kTile = 128;  // time steps per checkpoint

struct Strides {  // in elements; the channel axis is contiguous
  int64_t b, t;
};

__host__ __device__ inline int64_t tiles(int64_t T) { return (T + kTile - 1) / kTile; }

// a and 1 - a of the sigmoid form, each with a relative error of a few ulp: 1 - a is not formed by
// subtraction, so gates far from 0 keep the digits of both.
__device__ __forceinline__ void sigmoid_pair(float gate, float& a, float& na) {
  const float e = __expf(-fabsf(gate));  // in [0, 1]
  const float r = __fdividef(1.0f, 1.0f + e), er = e * r;
  a = gate >= 0.0f ? r : er;
  na = gate >= 0.0f ? er : r;
  if (gate != gate) a = na = gate;
}

template <int kForm>
__device__ __forceinline__ void coeffs(float gate, float x, float& a, float& v) {
  if (kForm == kDecay) {
    a = gate;
    v = x;
  } else {
    float na;
    sigmoid_pair(gate, a, na);
    v = na * x;
  }
}

template <typename T, int kForm>
__global__ void __launch_bounds__(128) forward_kernel(const T* __restrict__ gate, Strides gs, const T* __restrict__ x,
                                                      Strides xs, const float* __restrict__ state,
                                                      const uint8_t* __restrict__ reset, Strides rs, int64_t BH, int H,
                                                      int64_t Tn, T* __restrict__ h, Strides hs,
                                                      float* __restrict__ final_state, float* __restrict__ ckpt) {
  pdl_begin();
  const int64_t n = int64_t(blockIdx.x) * blockDim.x + threadIdx.x;
  if (n >= BH) return;
  const int64_t b = n / H, c = n - b * H;
  float s = state ? state[n] : 0.0f;
  for (int64_t t = 0; t < Tn; ++t) {
    if (ckpt != nullptr && t % kTile == 0) ckpt[(b * tiles(Tn) + t / kTile) * H + c] = s;
    float a, v;
    coeffs<kForm>(to_f32(gate[b * gs.b + t * gs.t + c]), to_f32(x[b * xs.b + t * xs.t + c]), a, v);
    if (reset != nullptr && reset[b * rs.b + t * rs.t]) s = 0.0f;
    s = fmaf(a, s, v);
    h[b * hs.b + t * hs.t + c] = from_f32<T>(s);
  }
  if (final_state != nullptr) final_state[n] = s;
}

template <typename T, int kForm>
__global__ void __launch_bounds__(128) backward_kernel(const T* __restrict__ gate, Strides gs, const T* __restrict__ x,
                                                       Strides xs, const float* __restrict__ ckpt,
                                                       const uint8_t* __restrict__ reset, Strides rs,
                                                       const T* __restrict__ grad_h, Strides ds,
                                                       const float* __restrict__ grad_final, int64_t BH, int H,
                                                       int64_t Tn, T* __restrict__ grad_gate, Strides ggs,
                                                       T* __restrict__ grad_x, Strides gxs,
                                                       float* __restrict__ grad_state) {
  pdl_begin();
  const int64_t n = int64_t(blockIdx.x) * blockDim.x + threadIdx.x;
  if (n >= BH) return;
  const int64_t b = n / H, c = n - b * H;
  float carry = grad_final ? grad_final[n] : 0.0f;  // a[t+1] g[t+1]
  float prev[kTile];
  for (int64_t k = tiles(Tn) - 1; k >= 0; --k) {
    const int64_t t0 = k * kTile;
    const int len = int(Tn - t0 < kTile ? Tn - t0 : kTile);
    float s = ckpt[(b * tiles(Tn) + k) * H + c];
    for (int i = 0; i < len; ++i) {
      const int64_t t = t0 + i;
      float a, v;
      coeffs<kForm>(to_f32(gate[b * gs.b + t * gs.t + c]), to_f32(x[b * xs.b + t * xs.t + c]), a, v);
      if (reset != nullptr && reset[b * rs.b + t * rs.t]) s = 0.0f;
      prev[i] = s;
      s = fmaf(a, s, v);
    }
    for (int i = len - 1; i >= 0; --i) {
      const int64_t t = t0 + i;
      const float xv = to_f32(x[b * xs.b + t * xs.t + c]);
      float a = to_f32(gate[b * gs.b + t * gs.t + c]), na = 1.0f;
      if (kForm == kSigmoid) sigmoid_pair(a, a, na);
      const float g = to_f32(grad_h[b * ds.b + t * ds.t + c]) + carry;
      const float gg = kForm == kDecay ? g * prev[i] : g * (prev[i] - xv) * a * na;
      const float gx = na * g;
      grad_gate[b * ggs.b + t * ggs.t + c] = from_f32<T>(gg);
      grad_x[b * gxs.b + t * gxs.t + c] = from_f32<T>(gx);
      carry = reset != nullptr && reset[b * rs.b + t * rs.t] ? 0.0f : a * g;
    }
  }
  if (grad_state != nullptr) grad_state[n] = carry;
}

// One token per row.  Rows that name the same slot are consecutive tokens of one sequence, in row
// order: the first of them walks them all.  Rows whose slot is outside [0, n_slots) are skipped.
template <typename T, int kForm>
__global__ void __launch_bounds__(128) step_kernel(const T* __restrict__ gate, int64_t gsb, const T* __restrict__ x,
                                                   int64_t xsb, const float* state, float* state_out,
                                                   const int32_t* __restrict__ slots, int n_slots, int B, int H,
                                                   T* __restrict__ h, int64_t hsb) {
  pdl_begin();
  const int64_t n = int64_t(blockIdx.x) * blockDim.x + threadIdx.x;
  if (n >= int64_t(B) * H) return;
  const int b = int(n / H);
  const int64_t c = n - int64_t(b) * H;
  const int slot = slots != nullptr ? slots[b] : b;
  if (slot < 0 || slot >= n_slots) return;
  if (slots != nullptr)
    for (int j = 0; j < b; ++j)
      if (slots[j] == slot) return;
  float s = state[int64_t(slot) * H + c];
  for (int j = b; j < B; ++j) {
    if (j != b && (slots == nullptr || slots[j] != slot)) continue;
    float a, v;
    coeffs<kForm>(to_f32(gate[j * gsb + c]), to_f32(x[j * xsb + c]), a, v);
    s = fmaf(a, s, v);
    h[j * hsb + c] = from_f32<T>(s);
  }
  state_out[int64_t(slot) * H + c] = s;
}

inline bool grid_ok(int64_t blocks) { return blocks > 0 && blocks <= 0x7fffffff; }

inline int64_t checkpoint_count(int64_t B, int64_t T, int64_t H) { return B * tiles(T) * H; }

inline size_t workspace_bytes(int32_t, int32_t, int32_t) { return 0; }

template <typename F>
inline int with_form(int form, F&& f) {
  if (form == kDecay) return f(std::integral_constant<int, kDecay>{});
  if (form == kSigmoid) return f(std::integral_constant<int, kSigmoid>{});
  return kInvalidArgument;
}

// strides (host array): gate, x, h, reset, each as (batch, time).
inline int forward(const void* gate, const void* x, int dtype, int form, const int64_t* strides, const float* state,
                   const uint8_t* reset, int32_t B, int32_t T, int32_t H, void* h, float* final_state, float* ckpt,
                   void*, size_t, cudaStream_t stream) {
  if (B < 0 || T < 0 || H < 0 || !dtype_ok(dtype) || strides == nullptr) return kInvalidArgument;
  const int64_t BH = int64_t(B) * H;
  if (BH == 0) return kOk;
  if (T > 0 && (gate == nullptr || x == nullptr || h == nullptr)) return kInvalidArgument;
  const Strides gs{strides[0], strides[1]}, xs{strides[2], strides[3]}, hs{strides[4], strides[5]},
      rs{strides[6], strides[7]};
  const int64_t blocks = (BH + 127) / 128;
  if (!grid_ok(blocks)) return kInvalidArgument;
  return with_dtype(dtype, [&](auto e) {
    using E = decltype(e);
    return with_form(form, [&](auto f) {
      return launch_pdl(forward_kernel<E, f.value>, dim3(unsigned(blocks)), dim3(128), 0, stream,
                        static_cast<const E*>(gate), gs, static_cast<const E*>(x), xs, state, reset, rs, BH, H,
                        int64_t(T), static_cast<E*>(h), hs, final_state, ckpt);
    });
  });
}

// strides (host array): gate, x, grad_h, grad_gate, grad_x, reset, each as (batch, time).
inline int backward(const void* gate, const void* x, int dtype, int form, const int64_t* strides, const float* ckpt,
                    const uint8_t* reset, const void* grad_h, const float* grad_final, int32_t B, int32_t T, int32_t H,
                    void* grad_gate, void* grad_x, float* grad_state, void*, size_t, cudaStream_t stream) {
  if (B < 0 || T < 0 || H < 0 || !dtype_ok(dtype) || strides == nullptr) return kInvalidArgument;
  const int64_t BH = int64_t(B) * H;
  if (BH == 0) return kOk;
  if (T > 0 && (gate == nullptr || x == nullptr || ckpt == nullptr || grad_h == nullptr || grad_gate == nullptr ||
                grad_x == nullptr))
    return kInvalidArgument;
  const Strides gs{strides[0], strides[1]}, xs{strides[2], strides[3]}, ds{strides[4], strides[5]},
      ggs{strides[6], strides[7]}, gxs{strides[8], strides[9]}, rs{strides[10], strides[11]};
  const int64_t blocks = (BH + 127) / 128;
  if (!grid_ok(blocks)) return kInvalidArgument;
  return with_dtype(dtype, [&](auto e) {
    using E = decltype(e);
    return with_form(form, [&](auto f) {
      return launch_pdl(backward_kernel<E, f.value>, dim3(unsigned(blocks)), dim3(128), 0, stream,
                        static_cast<const E*>(gate), gs, static_cast<const E*>(x), xs, ckpt, reset, rs,
                        static_cast<const E*>(grad_h), ds, grad_final, BH, H, int64_t(T), static_cast<E*>(grad_gate),
                        ggs, static_cast<E*>(grad_x), gxs, grad_state);
    });
  });
}

// strides (host array): row strides of gate, x and h.
inline int step(const void* gate, const void* x, int dtype, int form, const int64_t* strides, const float* state,
                float* state_out, const int32_t* slots, int32_t n_slots, int32_t B, int32_t H, void* h,
                cudaStream_t stream) {
  if (B < 0 || H < 0 || n_slots < 0 || !dtype_ok(dtype) || strides == nullptr) return kInvalidArgument;
  if (slots == nullptr && n_slots < B) return kInvalidArgument;
  if (B == 0 || H == 0 || n_slots == 0) return kOk;
  if (gate == nullptr || x == nullptr || h == nullptr || state == nullptr || state_out == nullptr)
    return kInvalidArgument;
  const int64_t blocks = (int64_t(B) * H + 127) / 128;
  if (!grid_ok(blocks)) return kInvalidArgument;
  return with_dtype(dtype, [&](auto e) {
    using E = decltype(e);
    return with_form(form, [&](auto f) {
      return launch_pdl(step_kernel<E, f.value>, dim3(unsigned(blocks)), dim3(128), 0, stream,
                        static_cast<const E*>(gate), strides[0], static_cast<const E*>(x), strides[1], state, state_out,
                        slots, n_slots, B, H, static_cast<E*>(h), strides[2]);
    });
  });
}

}  // namespace linrec
}  // namespace b200
