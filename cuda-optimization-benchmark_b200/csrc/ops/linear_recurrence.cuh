// Gated linear recurrence: T steps, B*H independent channels, state in fp32.
//
//   h[b,t,c] = a[b,t,c] * h[b,t-1,c] + v[b,t,c],   h[b,-1,c] = state[b,c] (0 without a state)
//     decay form:    a = gate,           v = x
//     sigmoid form:  a = sigmoid(gate),  v = (1 - a) * x
//   reset[b,t] != 0 drops h[b,t-1] (the first step of a packed document).
// Backward: the gradient carried back, c[t] = a[t] g[t] (0 over a reset), c[T] = grad_final:
//   g[t] = grad_h[t] + c[t+1]
//     decay:    grad_x = g,            grad_gate = g * h[t-1]
//     sigmoid:  grad_x = (1 - a) * g,  grad_gate = g * (h[t-1] - x) * a * (1 - a)
//   grad_state = c[0]
//
// Both directions are scans of maps y -> A y + b along time (forward: A = a, b = v; backward: A = a,
// b = a * grad_h), whose composition is associative, so time is split as well as the channels.
// What bounds them is memory: forward 3 elements a step and channel, backward 5.
//
// A tile is kTile = 128 steps of one group of channels, 128 bytes wide (64 channels of 16 bits, 32 of
// 32): each of 8 warps takes 16 steps, each lane 4 bytes of channels, so every load and store of a warp is a
// full line.  CTAs are persistent and take tiles in time order from a ticket counter: while one tile
// is worked on, the next one's rows arrive in the other shared-memory buffer (cp.async), so the loads
// never pause.  A tile is read once:
//   1. each warp composes its 16 steps into one map per channel;
//   2. the 8 maps meet in shared memory; the tile's map goes out as a record in global memory;
//   3. the state coming into the tile is formed from the records of the tiles before it;
//   4. each warp runs its 16 steps again from its own incoming state and writes them.
// Records: `span` consecutive tiles form a block.  A tile that ends a block publishes the state (or
// carried gradient) itself, the others their map; a tile takes the state at its block's start and the maps
// of the block's tiles before it, in order.  So the association is fixed by the sizes alone and
// results are the same bits whatever the timing.  Each record word travels with the launch's epoch (LL
// records), so reader and writer need no fence, and a tile waits only for tiles with smaller tickets, which
// running CTAs hold: the wait always ends, also when two calls share the GPU.
// Small spans keep the records few, large ones keep the chain of dependent states short: the span is
// about the number of tiles of one channel group that are worked on at once.
#pragma once

#include <type_traits>

#include "../common/bulk.cuh"
#include "../common/dtype.cuh"
#include "../common/ll.cuh"

namespace b200 {
namespace linrec {

enum Form : int { kDecay = 0, kSigmoid = 1 };

constexpr int kWarps = 8;
constexpr int kSteps = 16;               // time steps per warp and tile
constexpr int kTile = kWarps * kSteps;   // time steps per tile (and per checkpoint)
constexpr int kThreads = kWarps * 32;
constexpr int kRowBytes = 128;           // bytes of a tile's row
constexpr int kBufBytes = kTile * kRowBytes;
constexpr int kMaxSpan = 16;
constexpr size_t kCtlBytes = 256;

struct Strides {  // in elements; the channel axis is contiguous
  int64_t b, t;
};

// Control words of the workspace: zero before the first launch, and ready for the next after each.
struct Ctl {
  unsigned ticket, done, epoch;
};

__host__ __device__ inline int64_t tiles(int64_t T) { return (T + kTile - 1) / kTile; }

// ------------------------------------------------------------------------- per-element arithmetic
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

// The channels of one lane: 4 bytes of a row.
template <typename T>
struct Lane;
template <>
struct Lane<float> {
  static constexpr int kVec = 1;
  static __device__ __forceinline__ void unpack(uint32_t u, float (&f)[1]) { f[0] = __uint_as_float(u); }
  static __device__ __forceinline__ uint32_t pack(const float (&f)[1]) { return __float_as_uint(f[0]); }
};
template <>
struct Lane<__nv_bfloat16> {
  static constexpr int kVec = 2;
  static __device__ __forceinline__ void unpack(uint32_t u, float (&f)[2]) {
    f[0] = __uint_as_float(u << 16);
    f[1] = __uint_as_float(u & 0xffff0000u);
  }
  static __device__ __forceinline__ uint32_t pack(const float (&f)[2]) {
    const __nv_bfloat162 p = __floats2bfloat162_rn(f[0], f[1]);
    return *reinterpret_cast<const uint32_t*>(&p);
  }
};
template <>
struct Lane<__half> {
  static constexpr int kVec = 2;
  static __device__ __forceinline__ void unpack(uint32_t u, float (&f)[2]) {
    const float2 p = __half22float2(*reinterpret_cast<const __half2*>(&u));
    f[0] = p.x;
    f[1] = p.y;
  }
  static __device__ __forceinline__ uint32_t pack(const float (&f)[2]) {
    const __half2 p = __floats2half2_rn(f[0], f[1]);
    return *reinterpret_cast<const uint32_t*>(&p);
  }
};

// ---------------------------------------------------------------------------------- moving rows
template <int kBytes>
__device__ __forceinline__ void cp_async(char* dst, const char* src, int bytes) {
  if (kBytes == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_addr(dst)), "l"(src), "r"(bytes)
                 : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %3, %2;" ::"r"(smem_addr(dst)), "l"(src), "r"(bytes),
                 "n"(kBytes)
                 : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
__device__ __forceinline__ void cp_wait_all() { asm volatile("cp.async.wait_group 0;" ::: "memory"); }

template <int kBytes>
__device__ __forceinline__ void copy_rows_by(char* dst, const char* src, int64_t pitch, int rows, int width) {
  constexpr int kPer = kRowBytes / kBytes;
  const int off = int(threadIdx.x % kPer) * kBytes;
  const int left = width - off;
  if (left <= 0) return;
  for (int r = int(threadIdx.x) / kPer; r < rows; r += kThreads / kPer)
    cp_async<kBytes>(dst + r * kRowBytes + off, src + r * pitch + off, left < kBytes ? left : kBytes);
}

// `rows` rows of `width` bytes (at most 128), pitch bytes apart, into a tile buffer.  `granule` bytes
// divide the source address and the pitch; 2-byte granules (16-bit rows at odd elements) go through
// registers, which cp.async cannot copy.
__device__ __forceinline__ void copy_rows(char* dst, const char* src, int64_t pitch, int rows, int width,
                                          int granule) {
  if (granule == 16)
    copy_rows_by<16>(dst, src, pitch, rows, width);
  else if (granule == 8)
    copy_rows_by<8>(dst, src, pitch, rows, width);
  else if (granule == 4)
    copy_rows_by<4>(dst, src, pitch, rows, width);
  else
    for (int r = int(threadIdx.x) / 64, o = int(threadIdx.x % 64) * 2; r < rows; r += kThreads / 64)
      if (o < width)
        *reinterpret_cast<uint16_t*>(dst + r * kRowBytes + o) =
            *reinterpret_cast<const uint16_t*>(src + r * pitch + o);
}

// ------------------------------------------------------------------------------- tiles and records
struct Grid {
  int64_t T;
  int H;
  unsigned groups, chains, n_tiles, total;  // chains = B * groups; total = chains * n_tiles
  unsigned span;
  Ctl* ctl;          // null when a row is one tile: no tile waits for another, CTAs take tiles in turn
  ulonglong2* recs;  // [n_tiles, B, H]
};

struct Tile {
  unsigned k;       // position in the order of the scan
  unsigned b, group;
};

__device__ __forceinline__ Tile tile_of(const Grid& g, unsigned ticket) {
  Tile t;
  t.k = ticket / g.chains;
  const unsigned chain = ticket - t.k * g.chains;
  t.b = chain / g.groups;
  t.group = chain - t.b * g.groups;
  return t;
}

// Shared memory beside the tile buffers.
template <int kVec>
struct Shared {
  float2 map[kWarps][32 * kVec];         // the warps' maps (scan direction)
  float2 fwd[kWarps][32 * kVec];         // the warps' forward maps (backward kernel)
  float2 look[kMaxSpan][32 * kVec];      // records of the tiles before this one
  unsigned look_cut[kMaxSpan];
  unsigned cut[kWarps], fwd_cut[kWarps];  // the warp's steps hold a reset: its map does not see what comes in
  unsigned ticket[2];
};

// map applied to y; a map with a cut drops y, whatever it holds.
__device__ __forceinline__ float apply(float2 m, bool cut, float y) { return cut ? m.y : fmaf(m.x, y, m.y); }

// Publish a record for this lane's channels: tag = epoch * 2 + cut.
template <int kVec>
__device__ __forceinline__ void publish(const Grid& g, const Tile& t, int64_t B, int c, const float2 (&m)[kVec],
                                        unsigned tag) {
  ulonglong2* r = g.recs + (int64_t(t.k) * B + t.b) * g.H + c;
#pragma unroll
  for (int v = 0; v < kVec; ++v)
    if (c + v < g.H)
      ll_store2<LLScope::kGpu>(r + v, ll_word(__float_as_uint(m[v].x), tag), ll_word(__float_as_uint(m[v].y), tag));
}

// What comes into tile t from the tiles before it, for this lane's channels: y on entry is the value
// before tile 0.  Every thread of the CTA calls it.
template <int kVec>
__device__ __forceinline__ void incoming(const Grid& g, const Tile& t, int64_t B, int c, unsigned epoch,
                                         Shared<kVec>& sh, float (&y)[kVec]) {
  if (t.k == 0) return;
  const unsigned q = t.k % g.span;                    // tiles of the block before this one
  const unsigned n = q + (t.k >= g.span ? 1u : 0u);   // their maps, and the state at the block's start
  const unsigned lane = threadIdx.x % 32, w = threadIdx.x / 32;
  const unsigned first = t.k - n;
  unsigned long long t0 = 0;
  for (unsigned i = w; i < n; i += kWarps) {
    const ulonglong2* r = g.recs + (int64_t(first + i) * B + t.b) * g.H + c;
    unsigned cut = 0;
#pragma unroll
    for (int v = 0; v < kVec; ++v) {
      if (c + v >= g.H) continue;
      ulonglong2 x = ll_load2<LLScope::kGpu>(r + v);
      for (unsigned spin = 1; unsigned(x.x >> 33) != epoch || unsigned(x.y >> 33) != epoch; ++spin) {
        if ((spin & 63u) == 0) {
          if (t0 == 0) t0 = global_ns();
          else if (global_ns() - t0 > kWaitLimitNs) {
            atomicOr(&g_b200_fault, kFaultWaitTimeout);
            break;
          }
        }
        x = ll_load2<LLScope::kGpu>(r + v);
      }
      sh.look[i][lane * kVec + v] = make_float2(__uint_as_float(unsigned(x.x)), __uint_as_float(unsigned(x.y)));
      cut |= unsigned(x.x >> 32) & 1u;
    }
    cut = __any_sync(0xffffffffu, cut);
    if (lane == 0) sh.look_cut[i] = cut;
  }
  __syncthreads();
  for (unsigned i = 0; i < n; ++i) {
    const bool cut = sh.look_cut[i] != 0;
#pragma unroll
    for (int v = 0; v < kVec; ++v) y[v] = apply(sh.look[i][lane * kVec + v], cut, y[v]);
  }
}

// Publish this tile's record once the tile's map is known (and, where it ends a block, once what comes in
// is): called twice by the last warp, before incoming() with ends = false and after it with ends = true.
__device__ __forceinline__ bool ends_block(const Grid& g, unsigned k) { return k % g.span == g.span - 1; }

// Ends the launch's use of the workspace: the last CTA to leave makes it ready for the next launch.
__device__ __forceinline__ void leave(const Grid& g, unsigned epoch) {
  if (g.ctl == nullptr || threadIdx.x != 0) return;
  __threadfence();
  if (atomicAdd(&g.ctl->done, 1u) == gridDim.x - 1) {
    g.ctl->ticket = 0;
    g.ctl->done = 0;
    g.ctl->epoch = epoch;
    __threadfence();
  }
}

__device__ __forceinline__ unsigned next_ticket(const Grid& g, unsigned last) {
  return g.ctl != nullptr ? atomicAdd(&g.ctl->ticket, 1u) : last + gridDim.x;
}

// The launch's epoch: 31 bits, never 0 (a zero-filled record belongs to no launch).
__device__ __forceinline__ unsigned launch_epoch(const Grid& g) {
  if (g.ctl == nullptr) return 1u;
  const unsigned e = (ld_cg_u32(&g.ctl->epoch) + 1u) & 0x7fffffffu;
  return e == 0u ? 1u : e;
}

// The resets of one warp's steps as bits (bit i: step i of the warp).
struct Resets {
  const uint8_t* p;
  Strides s;
  __device__ __forceinline__ uint8_t load(unsigned b, int64_t t, int64_t T) const {
    return p != nullptr && threadIdx.x % 32 < kSteps && t < T ? p[int64_t(b) * s.b + t * s.t] : uint8_t(0);
  }
};

// ------------------------------------------------------------------------------------- forward
template <typename T>
struct Forward {
  Grid g;
  const T *gate, *x;
  Strides gs, xs, hs;
  const float* state;
  Resets reset;
  int64_t B;
  T* h;
  float *final_state, *ckpt;
  int granule;     // bytes that divide every row's address in gate and x
  bool wide;       // h rows take 4-byte stores
};

template <typename T, int kForm>
__global__ void __launch_bounds__(kThreads, 2) forward_kernel(const Forward<T> p) {
  constexpr int kVec = Lane<T>::kVec, kGroup = 32 * kVec;
  extern __shared__ __align__(128) char smem[];
  __shared__ Shared<kVec> sh;
  const unsigned lane = threadIdx.x % 32, w = threadIdx.x / 32;
  pdl_begin();
  const unsigned epoch = launch_epoch(p.g);

  const auto prefetch = [&](unsigned ticket, int buf) {
    if (ticket < p.g.total) {
      const Tile t = tile_of(p.g, ticket);
      const int64_t t0 = int64_t(t.k) * kTile;
      const int rows = int(p.g.T - t0 < kTile ? p.g.T - t0 : kTile);
      const int c0 = int(t.group) * kGroup;
      const int width = min(kGroup, p.g.H - c0) * int(sizeof(T));
      char* dst = smem + buf * 2 * kBufBytes;
      copy_rows(dst, reinterpret_cast<const char*>(p.gate + t.b * p.gs.b + t0 * p.gs.t + c0),
                p.gs.t * int64_t(sizeof(T)), rows, width, p.granule);
      copy_rows(dst + kBufBytes, reinterpret_cast<const char*>(p.x + t.b * p.xs.b + t0 * p.xs.t + c0),
                p.xs.t * int64_t(sizeof(T)), rows, width, p.granule);
    }
    cp_commit();
  };
  const auto load_reset = [&](unsigned ticket) {
    if (ticket >= p.g.total) return uint8_t(0);
    const Tile t = tile_of(p.g, ticket);
    return p.reset.load(t.b, int64_t(t.k) * kTile + w * kSteps + lane, p.g.T);
  };

  if (threadIdx.x == 0) sh.ticket[0] = p.g.ctl != nullptr ? atomicAdd(&p.g.ctl->ticket, 1u) : blockIdx.x;
  __syncthreads();
  unsigned ticket = sh.ticket[0];
  prefetch(ticket, 0);
  uint8_t reset_byte = load_reset(ticket);
  for (int buf = 0; ticket < p.g.total; buf ^= 1) {
    if (threadIdx.x == 0) sh.ticket[1] = next_ticket(p.g, ticket);
    cp_wait_all();
    const unsigned resets = __ballot_sync(0xffffffffu, reset_byte != 0);
    __syncthreads();  // this tile's rows and the next ticket are here; the other buffer is free
    const unsigned next = sh.ticket[1];
    prefetch(next, buf ^ 1);
    reset_byte = load_reset(next);

    const Tile t = tile_of(p.g, ticket);
    const int64_t t0 = int64_t(t.k) * kTile + w * kSteps;  // this warp's first step
    const int n = int(p.g.T - t0 < kSteps ? (p.g.T > t0 ? p.g.T - t0 : 0) : kSteps);
    const int c = int(t.group) * kGroup + int(lane) * kVec;
    const char* row = smem + buf * 2 * kBufBytes + w * kSteps * kRowBytes + lane * 4;

    // 1. The warp's steps as one map per channel; a and v stay in registers for step 4.
    float a[kSteps][kVec], u[kSteps][kVec];
    float2 m[kVec];
#pragma unroll
    for (int v = 0; v < kVec; ++v) m[v] = make_float2(1.0f, 0.0f);
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      if (i >= n) break;
      float gt[kVec], xv[kVec];
      Lane<T>::unpack(*reinterpret_cast<const uint32_t*>(row + i * kRowBytes), gt);
      Lane<T>::unpack(*reinterpret_cast<const uint32_t*>(row + kBufBytes + i * kRowBytes), xv);
      const bool cut = (resets >> i) & 1u;
#pragma unroll
      for (int v = 0; v < kVec; ++v) {
        coeffs<kForm>(gt[v], xv[v], a[i][v], u[i][v]);
        m[v].y = cut ? u[i][v] : fmaf(a[i][v], m[v].y, u[i][v]);
        m[v].x *= a[i][v];
      }
    }
#pragma unroll
    for (int v = 0; v < kVec; ++v) sh.map[w][lane * kVec + v] = m[v];
    if (lane == 0) sh.cut[w] = resets != 0;
    __syncthreads();

    // 2. The tile's map, by the last warp; a tile that ends a block publishes its state in step 3.
    const bool ends = ends_block(p.g, t.k), more = t.k + 1 < p.g.n_tiles;
    bool tile_cut = false;
    if (w == kWarps - 1 && more) {
#pragma unroll
      for (int v = 0; v < kVec; ++v) m[v] = make_float2(1.0f, 0.0f);
      for (int j = 0; j < kWarps; ++j) {
        const bool cut = sh.cut[j] != 0;
        tile_cut |= cut;
#pragma unroll
        for (int v = 0; v < kVec; ++v) {
          const float2 s = sh.map[j][lane * kVec + v];
          m[v] = make_float2(s.x * m[v].x, apply(s, cut, m[v].y));
        }
      }
      if (!ends) publish<kVec>(p.g, t, p.B, c, m, epoch * 2u + (tile_cut ? 1u : 0u));
    }

    // 3. The state that comes in.
    float y[kVec];
#pragma unroll
    for (int v = 0; v < kVec; ++v)
      y[v] = p.state != nullptr && t.k < p.g.span && c + v < p.g.H ? p.state[int64_t(t.b) * p.g.H + c + v] : 0.0f;
    incoming<kVec>(p.g, t, p.B, c, epoch, sh, y);
    if (w == kWarps - 1 && more && ends) {
#pragma unroll
      for (int v = 0; v < kVec; ++v) m[v] = make_float2(0.0f, apply(m[v], tile_cut, y[v]));
      publish<kVec>(p.g, t, p.B, c, m, epoch * 2u + 1u);
    }
    if (w == 0 && p.ckpt != nullptr) {
#pragma unroll
      for (int v = 0; v < kVec; ++v)
        if (c + v < p.g.H) p.ckpt[(int64_t(t.b) * p.g.n_tiles + t.k) * p.g.H + c + v] = y[v];
    }
    for (unsigned j = 0; j < w; ++j) {
      const bool cut = sh.cut[j] != 0;
#pragma unroll
      for (int v = 0; v < kVec; ++v) y[v] = apply(sh.map[j][lane * kVec + v], cut, y[v]);
    }

    // 4. The steps from there.
    T* out = p.h + t.b * p.hs.b + t0 * p.hs.t + c;
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      if (i >= n) break;
      const bool cut = (resets >> i) & 1u;
#pragma unroll
      for (int v = 0; v < kVec; ++v) y[v] = cut ? u[i][v] : fmaf(a[i][v], y[v], u[i][v]);
      if (p.wide) {
        if (c < p.g.H) *reinterpret_cast<uint32_t*>(out) = Lane<T>::pack(y);
      } else {
#pragma unroll
        for (int v = 0; v < kVec; ++v)
          if (c + v < p.g.H) out[v] = from_f32<T>(y[v]);
      }
      out += p.hs.t;
    }
    if (p.final_state != nullptr && n > 0 && t0 + n == p.g.T) {
#pragma unroll
      for (int v = 0; v < kVec; ++v)
        if (c + v < p.g.H) p.final_state[int64_t(t.b) * p.g.H + c + v] = y[v];
    }
    ticket = next;
  }
  leave(p.g, epoch);
}

// ------------------------------------------------------------------------------------ backward
template <typename T>
struct Backward {
  Grid g;
  const T *gate, *x, *dh;
  Strides gs, xs, ds, ggs, gxs;
  const float *ckpt, *grad_final;
  Resets reset;
  int64_t B;
  T *grad_gate, *grad_x;
  float* grad_state;
  int granule;
  bool wide;
};

// A pair (a, 1 - a) in one word: the smaller of the two, negative when it is 1 - a.  The other is 1 minus it,
// which keeps its digits since the smaller is at most 1/2.
__device__ __forceinline__ float pack_pair(float a, float na) { return a <= na ? a : -na; }
__device__ __forceinline__ void unpack_pair(float s, float& a, float& na) {
  const float t = 1.0f - fabsf(s);
  const bool neg = __float_as_int(s) < 0;
  a = neg ? t : s;
  na = neg ? -s : t;
}

// Tiles run from the last to the first (position k is time tile n_tiles - 1 - k).  The states h[t-1] of a
// tile are formed again from its checkpoint.
template <typename T, int kForm>
__global__ void __launch_bounds__(kThreads, 2) backward_kernel(const Backward<T> p) {
  constexpr int kVec = Lane<T>::kVec, kGroup = 32 * kVec;
  extern __shared__ __align__(128) char smem[];
  __shared__ Shared<kVec> sh;
  const unsigned lane = threadIdx.x % 32, w = threadIdx.x / 32;
  pdl_begin();
  const unsigned epoch = launch_epoch(p.g);

  const auto prefetch = [&](unsigned ticket, int buf) {
    if (ticket < p.g.total) {
      const Tile t = tile_of(p.g, ticket);
      const int64_t t0 = int64_t(p.g.n_tiles - 1 - t.k) * kTile;
      const int rows = int(p.g.T - t0 < kTile ? p.g.T - t0 : kTile);
      const int c0 = int(t.group) * kGroup;
      const int width = min(kGroup, p.g.H - c0) * int(sizeof(T));
      char* dst = smem + buf * 3 * kBufBytes;
      copy_rows(dst, reinterpret_cast<const char*>(p.gate + t.b * p.gs.b + t0 * p.gs.t + c0),
                p.gs.t * int64_t(sizeof(T)), rows, width, p.granule);
      copy_rows(dst + kBufBytes, reinterpret_cast<const char*>(p.x + t.b * p.xs.b + t0 * p.xs.t + c0),
                p.xs.t * int64_t(sizeof(T)), rows, width, p.granule);
      copy_rows(dst + 2 * kBufBytes, reinterpret_cast<const char*>(p.dh + t.b * p.ds.b + t0 * p.ds.t + c0),
                p.ds.t * int64_t(sizeof(T)), rows, width, p.granule);
    }
    cp_commit();
  };
  const auto load_reset = [&](unsigned ticket) {
    if (ticket >= p.g.total) return uint8_t(0);
    const Tile t = tile_of(p.g, ticket);
    return p.reset.load(t.b, int64_t(p.g.n_tiles - 1 - t.k) * kTile + w * kSteps + lane, p.g.T);
  };

  if (threadIdx.x == 0) sh.ticket[0] = p.g.ctl != nullptr ? atomicAdd(&p.g.ctl->ticket, 1u) : blockIdx.x;
  __syncthreads();
  unsigned ticket = sh.ticket[0];
  prefetch(ticket, 0);
  uint8_t reset_byte = load_reset(ticket);
  for (int buf = 0; ticket < p.g.total; buf ^= 1) {
    if (threadIdx.x == 0) sh.ticket[1] = next_ticket(p.g, ticket);
    const Tile t = tile_of(p.g, ticket);
    const unsigned kt = p.g.n_tiles - 1 - t.k;  // the time tile
    const int64_t t0 = int64_t(kt) * kTile + w * kSteps;
    const int n = int(p.g.T - t0 < kSteps ? (p.g.T > t0 ? p.g.T - t0 : 0) : kSteps);
    const int c = int(t.group) * kGroup + int(lane) * kVec;
    float s[kVec];  // the state before the tile
#pragma unroll
    for (int v = 0; v < kVec; ++v)
      s[v] = c + v < p.g.H ? p.ckpt[(int64_t(t.b) * p.g.n_tiles + kt) * p.g.H + c + v] : 0.0f;
    cp_wait_all();
    const unsigned resets = __ballot_sync(0xffffffffu, reset_byte != 0);
    __syncthreads();
    const unsigned next = sh.ticket[1];
    prefetch(next, buf ^ 1);
    reset_byte = load_reset(next);
    const char* row = smem + buf * 3 * kBufBytes + w * kSteps * kRowBytes + lane * 4;

    // 1. The warp's forward and backward maps.  ap: a (decay: read again instead), or the pair (a, 1 - a).
    float ap[kSteps][kVec];
    float2 f[kVec], m[kVec];
#pragma unroll
    for (int v = 0; v < kVec; ++v) f[v] = m[v] = make_float2(1.0f, 0.0f);
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      if (i >= n) break;
      float gt[kVec], xv[kVec];
      Lane<T>::unpack(*reinterpret_cast<const uint32_t*>(row + i * kRowBytes), gt);
      Lane<T>::unpack(*reinterpret_cast<const uint32_t*>(row + kBufBytes + i * kRowBytes), xv);
      const bool cut = (resets >> i) & 1u;
#pragma unroll
      for (int v = 0; v < kVec; ++v) {
        float a = gt[v], na = 1.0f;
        if (kForm == kSigmoid) sigmoid_pair(gt[v], a, na);
        ap[i][v] = kForm == kSigmoid ? pack_pair(a, na) : a;
        const float u = na * xv[v];
        f[v].y = cut ? u : fmaf(a, f[v].y, u);
        f[v].x *= a;
      }
    }
#pragma unroll
    for (int i = kSteps - 1; i >= 0; --i) {
      if (i >= n) continue;
      float dv[kVec];
      Lane<T>::unpack(*reinterpret_cast<const uint32_t*>(row + 2 * kBufBytes + i * kRowBytes), dv);
      const bool cut = (resets >> i) & 1u;
#pragma unroll
      for (int v = 0; v < kVec; ++v) {
        float a = ap[i][v], na;
        if (kForm == kSigmoid) unpack_pair(ap[i][v], a, na);
        m[v].y = cut ? 0.0f : a * (dv[v] + m[v].y);
        m[v].x *= a;
      }
    }
#pragma unroll
    for (int v = 0; v < kVec; ++v) {
      sh.map[w][lane * kVec + v] = m[v];
      sh.fwd[w][lane * kVec + v] = f[v];
    }
    if (lane == 0) sh.cut[w] = resets != 0;
    __syncthreads();

    // 2. The tile's map (from its last warp back), by warp 0, which holds the last of it.
    const bool ends = ends_block(p.g, t.k), more = t.k + 1 < p.g.n_tiles;
    bool tile_cut = false;
    if (w == 0 && more) {
#pragma unroll
      for (int v = 0; v < kVec; ++v) m[v] = make_float2(1.0f, 0.0f);
      for (int j = kWarps - 1; j >= 0; --j) {
        const bool cut = sh.cut[j] != 0;
        tile_cut |= cut;
#pragma unroll
        for (int v = 0; v < kVec; ++v) {
          const float2 q = sh.map[j][lane * kVec + v];
          m[v] = make_float2(q.x * m[v].x, apply(q, cut, m[v].y));
        }
      }
      if (!ends) publish<kVec>(p.g, t, p.B, c, m, epoch * 2u + (tile_cut ? 1u : 0u));
    }

    // The states before each step, from the checkpoint.
    for (unsigned j = 0; j < w; ++j) {
      const bool cut = sh.cut[j] != 0;
#pragma unroll
      for (int v = 0; v < kVec; ++v) s[v] = apply(sh.fwd[j][lane * kVec + v], cut, s[v]);
    }
    float prev[kSteps][kVec];
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      if (i >= n) break;
      float xv[kVec];
      Lane<T>::unpack(*reinterpret_cast<const uint32_t*>(row + kBufBytes + i * kRowBytes), xv);
      const bool cut = (resets >> i) & 1u;
#pragma unroll
      for (int v = 0; v < kVec; ++v) {
        float a = ap[i][v], na = 1.0f;
        if (kForm == kSigmoid) unpack_pair(ap[i][v], a, na);
        prev[i][v] = cut ? 0.0f : s[v];
        const float u = na * xv[v];
        s[v] = cut ? u : fmaf(a, s[v], u);
      }
    }

    // 3. The gradient that comes in.
    float y[kVec];
#pragma unroll
    for (int v = 0; v < kVec; ++v)
      y[v] = p.grad_final != nullptr && t.k < p.g.span && c + v < p.g.H ? p.grad_final[int64_t(t.b) * p.g.H + c + v]
                                                                          : 0.0f;
    incoming<kVec>(p.g, t, p.B, c, epoch, sh, y);
    if (w == 0 && more && ends) {
#pragma unroll
      for (int v = 0; v < kVec; ++v) m[v] = make_float2(0.0f, apply(m[v], tile_cut, y[v]));
      publish<kVec>(p.g, t, p.B, c, m, epoch * 2u + 1u);
    }
    for (int j = kWarps - 1; j > int(w); --j) {
      const bool cut = sh.cut[j] != 0;
#pragma unroll
      for (int v = 0; v < kVec; ++v) y[v] = apply(sh.map[j][lane * kVec + v], cut, y[v]);
    }

    // 4. The steps from there, backwards.
    T* og = p.grad_gate + t.b * p.ggs.b + t0 * p.ggs.t + c;
    T* ox = p.grad_x + t.b * p.gxs.b + t0 * p.gxs.t + c;
#pragma unroll
    for (int i = kSteps - 1; i >= 0; --i) {
      if (i >= n) continue;
      float xv[kVec], dv[kVec], gg[kVec], gx[kVec];
      Lane<T>::unpack(*reinterpret_cast<const uint32_t*>(row + kBufBytes + i * kRowBytes), xv);
      Lane<T>::unpack(*reinterpret_cast<const uint32_t*>(row + 2 * kBufBytes + i * kRowBytes), dv);
      const bool cut = (resets >> i) & 1u;
#pragma unroll
      for (int v = 0; v < kVec; ++v) {
        float a = ap[i][v], na = 1.0f;
        if (kForm == kSigmoid) unpack_pair(ap[i][v], a, na);
        const float g = dv[v] + y[v];
        gx[v] = na * g;
        gg[v] = kForm == kSigmoid ? g * (prev[i][v] - xv[v]) * (a * na) : g * prev[i][v];
        y[v] = cut ? 0.0f : a * g;
      }
      T *pg = og + i * p.ggs.t, *px = ox + i * p.gxs.t;
      if (p.wide) {
        if (c < p.g.H) {
          *reinterpret_cast<uint32_t*>(pg) = Lane<T>::pack(gg);
          *reinterpret_cast<uint32_t*>(px) = Lane<T>::pack(gx);
        }
      } else {
#pragma unroll
        for (int v = 0; v < kVec; ++v)
          if (c + v < p.g.H) pg[v] = from_f32<T>(gg[v]), px[v] = from_f32<T>(gx[v]);
      }
    }
    if (p.grad_state != nullptr && t0 == 0) {
#pragma unroll
      for (int v = 0; v < kVec; ++v)
        if (c + v < p.g.H) p.grad_state[int64_t(t.b) * p.g.H + c + v] = y[v];
    }
    ticket = next;
  }
  leave(p.g, epoch);
}

// T = 0: what comes in goes out.
__global__ void __launch_bounds__(256) copy_state_kernel(const float* __restrict__ in, int64_t n,
                                                         float* __restrict__ out) {
  pdl_begin();
  const int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x;
  if (i < n) out[i] = in != nullptr ? in[i] : 0.0f;
}

inline int copy_state(const float* in, int64_t n, float* out, cudaStream_t stream) {
  if (out == nullptr) return kOk;
  return launch_pdl(copy_state_kernel, dim3(unsigned((n + 255) / 256)), dim3(256), 0, stream, in, n, out);
}

// ---------------------------------------------------------------------------------------- step
// One token per row, a CTA per row and stretch of channels.  Rows that name the same slot are
// consecutive tokens of one sequence, in row order: the first of them walks them all.  Rows whose slot
// is outside [0, n_slots) are skipped.
constexpr int kStepThreads = 128;

template <typename T, int kForm>
__global__ void __launch_bounds__(kStepThreads) step_kernel(const T* __restrict__ gate, int64_t gsb,
                                                            const T* __restrict__ x, int64_t xsb, const float* state,
                                                            float* state_out, const int32_t* __restrict__ slots,
                                                            int n_slots, int B, int H, int blocks, T* __restrict__ h,
                                                            int64_t hsb) {
  pdl_begin();
  const int b = int(blockIdx.x) / blocks;
  const int c = (int(blockIdx.x) - b * blocks) * kStepThreads + int(threadIdx.x);
  const int slot = slots != nullptr ? slots[b] : b;
  if (slot < 0 || slot >= n_slots) return;
  bool again = false;  // a later row has the same slot
  if (slots != nullptr) {
    bool before = false;
    for (int j = threadIdx.x; j < B; j += kStepThreads) {
      const bool same = slots[j] == slot;
      before |= same && j < b;
      again |= same && j > b;
    }
    if (__syncthreads_or(before)) return;
    again = __syncthreads_or(again);
  }
  if (c >= H) return;
  float s = state[int64_t(slot) * H + c];
  for (int j = b; j < B; ++j) {
    if (j != b && slots[j] != slot) continue;
    float a, v;
    coeffs<kForm>(to_f32(gate[j * gsb + c]), to_f32(x[j * xsb + c]), a, v);
    s = fmaf(a, s, v);
    h[j * hsb + c] = from_f32<T>(s);
    if (!again) break;
  }
  state_out[int64_t(slot) * H + c] = s;
}

// ------------------------------------------------------------------------------------ host side
inline int64_t checkpoint_count(int64_t B, int64_t T, int64_t H) { return B * tiles(T) * H; }

inline int64_t workspace_bytes(int64_t B, int64_t T, int64_t H) {
  return tiles(T) <= 1 ? 0 : int64_t(kCtlBytes) + checkpoint_count(B, T, H) * int64_t(sizeof(ulonglong2));
}

template <typename F>
inline int with_form(int form, F&& f) {
  if (form == kDecay) return f(std::integral_constant<int, kDecay>{});
  if (form == kSigmoid) return f(std::integral_constant<int, kSigmoid>{});
  return kInvalidArgument;
}

// Channel indexes are ints up to the end of the last, partly empty group.
inline bool channels_ok(int64_t H) { return H <= 0x7fffffff - kThreads; }

// The largest of 16, 8, 4, 2 bytes that divides every given address and stride.
struct Granule {
  uint64_t bits = 0;
  void add(const void* p, Strides s, int64_t size) {
    bits |= uint64_t(reinterpret_cast<uintptr_t>(p)) | uint64_t(s.b * size) | uint64_t(s.t * size);
  }
  int bytes() const { return bits % 16 == 0 ? 16 : bits % 8 == 0 ? 8 : bits % 4 == 0 ? 4 : 2; }
};

// Fills the scan geometry and the grid size; kernel is the instantiation to launch.
template <typename Kernel>
inline int plan(Kernel kernel, int smem, int vec, int64_t B, int64_t T, int64_t H, void* ws, int64_t ws_bytes, Grid* g,
                unsigned* ctas) {
  const int64_t groups = (H + 32 * vec - 1) / (32 * vec), n = tiles(T);
  if (groups > 0x7fffffff / B || n > 0x7fffffff / (B * groups)) return kInvalidArgument;
  g->T = T, g->H = int(H), g->groups = unsigned(groups), g->chains = unsigned(B * groups);
  g->n_tiles = unsigned(n), g->total = unsigned(B * groups * n);
  g->ctl = nullptr, g->recs = nullptr;
  if (n > 1) {
    if (ws == nullptr || ws_bytes < workspace_bytes(B, T, H)) return kWorkspaceTooSmall;
    if (!aligned16(ws)) return kInvalidArgument;
    g->ctl = static_cast<Ctl*>(ws);
    g->recs = reinterpret_cast<ulonglong2*>(static_cast<char*>(ws) + kCtlBytes);
  }
  if (!ensure_dyn_smem(kernel, smem)) return kCudaError;
  const unsigned resident = unsigned(sm_count() * resident_ctas_per_sm(kernel, kThreads, size_t(smem)));
  *ctas = resident < g->total ? resident : g->total;
  // Tiles of one chain that are worked on at once, rounded up to a power of two.
  unsigned span = 1;
  while (span < kMaxSpan && span * g->chains < resident) span *= 2;
  g->span = span;
  return kOk;
}

inline bool strides_ok(const int64_t* s, int n) {
  for (int i = 0; i < n; ++i)
    if (s[i] < 0) return false;
  return true;
}

// strides (host array): gate, x, h, reset, each as (batch, time).
inline int forward(const void* gate, const void* x, int dtype, int form, const int64_t* strides, const float* state,
                   const uint8_t* reset, int32_t B, int32_t T, int32_t H, void* h, float* final_state, float* ckpt,
                   void* ws, int64_t ws_bytes, cudaStream_t stream) {
  if (B < 0 || T < 0 || H < 0 || !dtype_ok(dtype) || (form != kDecay && form != kSigmoid) || strides == nullptr ||
      !strides_ok(strides, 8))
    return kInvalidArgument;
  const int64_t BH = int64_t(B) * H;
  if (BH == 0) return kOk;
  if (!channels_ok(H)) return kUnsupported;
  if (T == 0) return copy_state(state, BH, final_state, stream);
  if (gate == nullptr || x == nullptr || h == nullptr) return kInvalidArgument;
  return with_dtype(dtype, [&](auto e) {
    using E = decltype(e);
    return with_form(form, [&](auto f) {
      Forward<E> p;
      p.gate = static_cast<const E*>(gate), p.x = static_cast<const E*>(x), p.h = static_cast<E*>(h);
      p.gs = Strides{strides[0], strides[1]}, p.xs = Strides{strides[2], strides[3]};
      p.hs = Strides{strides[4], strides[5]};
      p.reset = Resets{reset, Strides{strides[6], strides[7]}};
      p.state = state, p.B = B, p.final_state = final_state, p.ckpt = ckpt;
      Granule in, out;
      in.add(gate, p.gs, sizeof(E)), in.add(x, p.xs, sizeof(E)), out.add(h, p.hs, sizeof(E));
      p.granule = in.bytes();
      p.wide = out.bytes() >= 4 && H % Lane<E>::kVec == 0;
      constexpr int kSmem = 4 * kBufBytes;
      const auto kernel = forward_kernel<E, f.value>;
      unsigned ctas = 0;
      const int st = plan(kernel, kSmem, Lane<E>::kVec, B, T, H, ws, ws_bytes, &p.g, &ctas);
      return st != kOk ? st : launch_pdl(kernel, dim3(ctas), dim3(kThreads), kSmem, stream, p);
    });
  });
}

// strides (host array): gate, x, grad_h, grad_gate, grad_x, reset, each as (batch, time).
inline int backward(const void* gate, const void* x, int dtype, int form, const int64_t* strides, const float* ckpt,
                    const uint8_t* reset, const void* grad_h, const float* grad_final, int32_t B, int32_t T, int32_t H,
                    void* grad_gate, void* grad_x, float* grad_state, void* ws, int64_t ws_bytes,
                    cudaStream_t stream) {
  if (B < 0 || T < 0 || H < 0 || !dtype_ok(dtype) || (form != kDecay && form != kSigmoid) || strides == nullptr ||
      !strides_ok(strides, 12))
    return kInvalidArgument;
  const int64_t BH = int64_t(B) * H;
  if (BH == 0) return kOk;
  if (!channels_ok(H)) return kUnsupported;
  if (T == 0) return copy_state(grad_final, BH, grad_state, stream);
  if (gate == nullptr || x == nullptr || ckpt == nullptr || grad_h == nullptr || grad_gate == nullptr ||
      grad_x == nullptr)
    return kInvalidArgument;
  return with_dtype(dtype, [&](auto e) {
    using E = decltype(e);
    return with_form(form, [&](auto f) {
      Backward<E> p;
      p.gate = static_cast<const E*>(gate), p.x = static_cast<const E*>(x), p.dh = static_cast<const E*>(grad_h);
      p.grad_gate = static_cast<E*>(grad_gate), p.grad_x = static_cast<E*>(grad_x);
      p.gs = Strides{strides[0], strides[1]}, p.xs = Strides{strides[2], strides[3]};
      p.ds = Strides{strides[4], strides[5]}, p.ggs = Strides{strides[6], strides[7]};
      p.gxs = Strides{strides[8], strides[9]};
      p.reset = Resets{reset, Strides{strides[10], strides[11]}};
      p.ckpt = ckpt, p.grad_final = grad_final, p.B = B, p.grad_state = grad_state;
      Granule in, out;
      in.add(gate, p.gs, sizeof(E)), in.add(x, p.xs, sizeof(E)), in.add(grad_h, p.ds, sizeof(E));
      out.add(grad_gate, p.ggs, sizeof(E)), out.add(grad_x, p.gxs, sizeof(E));
      p.granule = in.bytes();
      p.wide = out.bytes() >= 4 && H % Lane<E>::kVec == 0;
      constexpr int kSmem = 6 * kBufBytes;
      const auto kernel = backward_kernel<E, f.value>;
      unsigned ctas = 0;
      const int st = plan(kernel, kSmem, Lane<E>::kVec, B, T, H, ws, ws_bytes, &p.g, &ctas);
      return st != kOk ? st : launch_pdl(kernel, dim3(ctas), dim3(kThreads), kSmem, stream, p);
    });
  });
}

// strides (host array): row strides of gate, x and h.
inline int step(const void* gate, const void* x, int dtype, int form, const int64_t* strides, const float* state,
                float* state_out, const int32_t* slots, int32_t n_slots, int32_t B, int32_t H, void* h,
                cudaStream_t stream) {
  if (B < 0 || H < 0 || n_slots < 0 || !dtype_ok(dtype) || (form != kDecay && form != kSigmoid) ||
      strides == nullptr || !strides_ok(strides, 3))
    return kInvalidArgument;
  if (slots == nullptr && n_slots < B) return kInvalidArgument;
  if (B == 0 || H == 0 || n_slots == 0) return kOk;
  if (!channels_ok(H)) return kUnsupported;
  if (gate == nullptr || x == nullptr || h == nullptr || state == nullptr || state_out == nullptr)
    return kInvalidArgument;
  const int64_t per_row = (int64_t(H) + kStepThreads - 1) / kStepThreads;
  if (per_row > 0x7fffffff / B) return kInvalidArgument;
  return with_dtype(dtype, [&](auto e) {
    using E = decltype(e);
    return with_form(form, [&](auto f) {
      return launch_pdl(step_kernel<E, f.value>, dim3(unsigned(per_row * B)), dim3(kStepThreads), 0, stream,
                        static_cast<const E*>(gate), strides[0], static_cast<const E*>(x), strides[1], state, state_out,
                        slots, n_slots, B, H, int(per_row), static_cast<E*>(h), strides[2]);
    });
  });
}

}  // namespace linrec
}  // namespace b200
