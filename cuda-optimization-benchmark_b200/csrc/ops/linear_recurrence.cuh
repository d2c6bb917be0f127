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
// full line.  CTAs are persistent and take tiles in time order from a ticket counter.  A tile is read once:
//   1. each warp composes its 16 steps into one map per channel;
//   2. the 8 maps meet in shared memory; the tile's map goes out as a record in global memory;
//   3. the state coming into the tile is formed from the records of the tiles before it;
//   4. each warp runs its 16 steps again from its own incoming state and writes them.
// Behind step 1 one warp, the clerk, finds the CTA's next tile and starts its loads into the other buffer (one
// tensor load per input; where rows are not on 16 bytes every warp copies its own): after step 1, since a
// tile's time is a chain of waits that all 8 warps share, and there the other warps wait anyway.
// Records: `span` consecutive tiles form a block.  A tile that ends a block publishes the state (or
// carried gradient) itself, the others their map; a tile takes the state at its block's start and the maps
// of the block's tiles before it, in order.  So the association is fixed by the sizes alone and
// results are the same bits whatever the timing.  Each record word travels with the launch's epoch (LL
// records), so reader and writer need no fence, and a tile waits only for tiles with smaller tickets, which
// running CTAs hold: the wait always ends, also when two calls share the GPU.
// Small spans keep the records few, large ones keep the chain of dependent states short: the span is
// about the number of tiles of one channel group that are worked on at once, 16 at most (one sequence of 65536 steps,
// 1024 channels of 16 bits: 196 us with spans up to 4, 162 up to 8, 150 up to 16).
//
// Measured, forward and backward (a plain copy runs at 6.56 TB/s on the same GPU), B = 8, T = 4096, H = 2048:
//   bf16 sigmoid 86 us (4.7 TB/s) and 130 us (5.2 TB/s), bf16 decay 74 and 116 us;
//   fp32 sigmoid 127 us (6.3 TB/s) and 211 us (6.4 TB/s).
// So fp32 is bound by memory.  With 16 bits the same bytes carry twice the elements: 21 and 37 instructions an element
// leave a warp of the 16 on an SM issuing in 45 to 50 % of the cycles, and what it waits for is its own arithmetic
// and the three barriers of a tile.  Tried without gain: a ninth warp that only serves tickets, loads and records (96
// registers a thread are left, which spill), three tickets held ahead, shorter unrolled loops.
// One long sequence (1 x 65539 x 1024 fp32: 154 us, 5.2 TB/s) is also bound by the chain of records.
// Rows off 16 bytes go through copies of 8, 4 or 2 bytes: 123 us and 255 us at H = 2044, and
// 254 and 636 us at odd H, where each element is moved to its place on its way in and out.
#pragma once

#include <type_traits>

#include "../common/bulk.cuh"
#include "../common/dtype.cuh"
#include "../common/ll.cuh"
#include "../common/tcgen05.cuh"

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
constexpr int kClerk = 5;                // the warp that takes the tickets (none of those with other extra work)
constexpr size_t kCtlBytes = 256;

struct Strides {  // in elements; the channel axis is contiguous
  int64_t b, t;
};

// Control words of the workspace: zero before the first launch, and ready for the next after each.
struct Ctl {
  unsigned ticket, epoch;  // tickets taken in this launch, epoch of the one before
};

__host__ __device__ inline int64_t tiles(int64_t T) { return (T + kTile - 1) / kTile; }

// --------------------------------------------------------------------------- the lane's channels
// A lane holds 4 bytes of a row: one fp32 channel (float), or two 16-bit ones (float2, whose products and
// sums are packed two to an instruction; instruction issue is the next bound after memory).
__device__ __forceinline__ float vset(float, float a) { return a; }
__device__ __forceinline__ float2 vset(float2, float a) { return make_float2(a, a); }
__device__ __forceinline__ float vmul(float a, float b) { return a * b; }
__device__ __forceinline__ float2 vmul(float2 a, float2 b) { return __fmul2_rn(a, b); }
__device__ __forceinline__ float vadd(float a, float b) { return a + b; }
__device__ __forceinline__ float2 vadd(float2 a, float2 b) { return __fadd2_rn(a, b); }
__device__ __forceinline__ float vfma(float a, float b, float c) { return fmaf(a, b, c); }
__device__ __forceinline__ float2 vfma(float2 a, float2 b, float2 c) { return __ffma2_rn(a, b, c); }
__device__ __forceinline__ float vsub(float a, float b) { return a - b; }
__device__ __forceinline__ float2 vsub(float2 a, float2 b) { return __ffma2_rn(b, make_float2(-1.0f, -1.0f), a); }

__device__ __forceinline__ float ex2(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float rcp(float v) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}

constexpr float kLog2e = 1.4426950408889634f;

// The gate clamped at -87 from below (NaN kept): exp(87) is still finite in fp32, and sigmoid(-87), about
// 2^-125.5, is as good as 0.
constexpr float kLowGate = -87.0f;
__device__ __forceinline__ float clamp_gate(float g) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(g), "f"(kLowGate));
  return r;
}

// a = sigmoid(gate) and 1 - a, each with a relative error of a few ulp: with e = exp(-gate) they are
// 1 / (1 + e) and e / (1 + e), and neither is formed by subtraction, so gates far from 0 keep the digits of
// both.  gate >= kLowGate.
__device__ __forceinline__ void sigmoid_pair(float gate, float& a, float& na) {
  const float e = ex2(gate * -kLog2e);
  a = rcp(1.0f + e);
  na = e * a;
}
__device__ __forceinline__ void sigmoid_pair(float2 gate, float2& a, float2& na) {
  const float2 z = vmul(gate, vset(gate, -kLog2e));
  const float2 e = make_float2(ex2(z.x), ex2(z.y));
  const float2 d = vadd(e, vset(e, 1.0f));
  a = make_float2(rcp(d.x), rcp(d.y));
  na = vmul(e, a);
}

template <typename T>
struct Lane;
template <>
struct Lane<float> {
  using V = float;
  static constexpr int kVec = 1;
  static __device__ __forceinline__ V unpack(uint32_t u) { return __uint_as_float(u); }
  static __device__ __forceinline__ V unpack_gate(uint32_t u) { return clamp_gate(__uint_as_float(u)); }
  static __device__ __forceinline__ uint32_t pack(V f) { return __float_as_uint(f); }
};
template <>
struct Lane<__nv_bfloat16> {
  using V = float2;
  static constexpr int kVec = 2;
  static __device__ __forceinline__ V unpack(uint32_t u) {
    return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
  }
  static __device__ __forceinline__ V unpack_gate(uint32_t u) {
    const __nv_bfloat162 g = __hmax2_nan(*reinterpret_cast<const __nv_bfloat162*>(&u),
                                         __floats2bfloat162_rn(kLowGate, kLowGate));
    return unpack(*reinterpret_cast<const uint32_t*>(&g));
  }
  static __device__ __forceinline__ uint32_t pack(V f) {
    const __nv_bfloat162 p = __floats2bfloat162_rn(f.x, f.y);
    return *reinterpret_cast<const uint32_t*>(&p);
  }
};
template <>
struct Lane<__half> {
  using V = float2;
  static constexpr int kVec = 2;
  static __device__ __forceinline__ V unpack(uint32_t u) {
    return __half22float2(*reinterpret_cast<const __half2*>(&u));
  }
  static __device__ __forceinline__ V unpack_gate(uint32_t u) {
    return __half22float2(__hmax2_nan(*reinterpret_cast<const __half2*>(&u), __floats2half2_rn(kLowGate, kLowGate)));
  }
  static __device__ __forceinline__ uint32_t pack(V f) {
    const __half2 p = __floats2half2_rn(f.x, f.y);
    return *reinterpret_cast<const uint32_t*>(&p);
  }
};

// The lane's fp32 values at p (channel c of H) in a row of fp32, 0 past the last channel.
__device__ __forceinline__ void load_row(const float* p, int c, int H, float& y) { y = c < H ? p[0] : 0.0f; }
__device__ __forceinline__ void load_row(const float* p, int c, int H, float2& y) {
  y.x = c < H ? p[0] : 0.0f;
  y.y = c + 1 < H ? p[1] : 0.0f;
}
__device__ __forceinline__ void store_row(float* p, int c, int H, float y) {
  if (c < H) p[0] = y;
}
__device__ __forceinline__ void store_row(float* p, int c, int H, float2 y) {
  if (c < H) p[0] = y.x;
  if (c + 1 < H) p[1] = y.y;
}
// One row of an output (whole warps).  wide: rows are aligned to 4 bytes and hold whole lanes.  Otherwise 16-bit
// rows may start between two words: each lane then writes the word of its left neighbour's second and its own
// first channel, and the ends are written alone.
template <typename T>
__device__ __forceinline__ void store_out(T* p, int c, int H, bool wide, typename Lane<T>::V y) {
  const uint32_t u = Lane<T>::pack(y);
  if (wide || sizeof(T) == 4) {
    if (c < H) *reinterpret_cast<uint32_t*>(p) = u;
    return;
  }
  const unsigned lane = threadIdx.x % 32;
  uint16_t* q = reinterpret_cast<uint16_t*>(p);
  const bool off = (reinterpret_cast<uintptr_t>(p) & 2u) != 0;  // the same in all lanes
  const uint32_t left = __shfl_up_sync(0xffffffffu, u, 1);
  if (off) {
    if (lane > 0 && c < H) *reinterpret_cast<uint32_t*>(q - 1) = __byte_perm(left, u, 0x5432);
    if (lane > 0 && c == H) q[-1] = uint16_t(left >> 16);
    if (lane == 0 && c < H) q[0] = uint16_t(u);
    if (lane == 31 && c + 1 < H) q[1] = uint16_t(u >> 16);
  } else {
    if (c + 1 < H) *reinterpret_cast<uint32_t*>(q) = u;
    else if (c < H) q[0] = uint16_t(u);
  }
}

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
  const int lane = int(threadIdx.x % 32), off = lane % kPer * kBytes;
  const int left = width - off;
  if (left <= 0) return;
#pragma unroll
  for (int i = 0; i < kSteps * kPer / 32; ++i) {
    const int r = i * (32 / kPer) + lane / kPer;
    if (r < rows) cp_async<kBytes>(dst + r * kRowBytes + off, src + r * pitch + off, left < kBytes ? left : kBytes);
  }
}

// A warp's `rows` rows of `width` bytes (at most 128), pitch bytes apart, into its part of a tile buffer.
// `granule` bytes divide the source address and the pitch.  Rows of 16-bit elements off 4 bytes are copied
// with the 4-byte word that their first element lies in, the word behind the row's 32 goes to more[r], and
// align_rows() shifts them.
__device__ __forceinline__ void copy_rows(char* dst, uint32_t* more, const char* src, int64_t pitch, int rows,
                                          int width, int granule) {
  const int lane = int(threadIdx.x % 32);
  if (granule == 16) {
    copy_rows_by<16>(dst, src, pitch, rows, width);
  } else if (granule == 8) {
    copy_rows_by<8>(dst, src, pitch, rows, width);
  } else if (granule == 4) {
    copy_rows_by<4>(dst, src, pitch, rows, width);
  } else {
#pragma unroll 4
    for (int r = 0; r < rows; ++r) {
      const char* s = src + r * pitch;
      const int off = int(reinterpret_cast<uintptr_t>(s) & 2u), left = width + off - lane * 4;
      if (left > 0) cp_async<4>(dst + r * kRowBytes + lane * 4, s - off + lane * 4, left < 4 ? left : 4);
    }
    if (lane < rows) {
      const char* s = src + lane * pitch;
      const int off = int(reinterpret_cast<uintptr_t>(s) & 2u), left = width + off - kRowBytes;
      if (left > 0) cp_async<4>(reinterpret_cast<char*>(more + lane), s - off + kRowBytes, left);
    }
  }
}

// Rows copied from an address off 4 bytes, shifted to their place (the warp's own rows).
__device__ __forceinline__ void align_rows(char* dst, const uint32_t* more, const char* src, int64_t pitch, int rows) {
  const int lane = int(threadIdx.x % 32);
#pragma unroll 4
  for (int r = 0; r < rows; ++r) {
    if ((reinterpret_cast<uintptr_t>(src + r * pitch) & 2u) == 0) continue;
    uint32_t* row = reinterpret_cast<uint32_t*>(dst + r * kRowBytes);
    const uint32_t lo = row[lane];
    uint32_t hi = __shfl_down_sync(0xffffffffu, lo, 1);
    if (lane == 31) hi = more[r];
    __syncwarp();
    row[lane] = __funnelshift_r(lo, hi, 16);
  }
  __syncwarp();
}

// ------------------------------------------------------------------------------- tiles and records
struct Grid {
  int64_t T;
  int H;
  unsigned groups, chains, n_tiles, total;  // chains = B * groups; total = chains * n_tiles
  unsigned span;
  bool one;          // every CTA takes one ticket: there are as many as tiles
  Ctl* ctl;          // null when a row is one tile: no tile waits for another, CTAs take tiles in turn
  ulonglong2* recs;  // [n_tiles, B, H]
  bool back;         // the scan runs from the last tile to the first
};

struct __align__(16) Tile {
  unsigned k;  // position in the order of the scan
  unsigned b, group;
  unsigned live;  // 0: the ticket lies past the last tile
};
// The tile's first step.
__device__ __forceinline__ int64_t first_step(const Grid& g, const Tile& t) {
  return int64_t(g.back ? g.n_tiles - 1 - t.k : t.k) * kTile;
}

__device__ __forceinline__ Tile tile_of(const Grid& g, unsigned ticket) {
  Tile t;
  t.k = ticket / g.chains;
  const unsigned chain = ticket - t.k * g.chains;
  t.b = chain / g.groups;
  t.group = chain - t.b * g.groups;
  t.live = ticket < g.total;
  return t;
}

// A map y -> x y + b of the lane's channels.
template <typename V>
struct __align__(2 * sizeof(V)) Map {
  V x, b;
};

// Shared memory beside the tile buffers; kLook: records that it holds at once.
template <typename V, bool kBack, int kLook>
struct Shared {
  Map<V> map[kWarps][32];        // the warps' maps (scan direction)
  V fwd[kBack ? kWarps - 1 : 1][32];  // the warps' forward offsets (backward kernel; the factor is map.x)
  Map<V> look[kLook][32];        // records of the tiles before this one
  unsigned look_cut[kLook];
  uint64_t cut;                  // byte w: warp w's steps hold a reset, its map does not see what comes in
  Tile tile[2];                  // of the CTA's tiles in turn
  uint64_t full[2];              // the tile buffers' loads have landed (tensor loads)
  unsigned epoch;                // the launch's
};

// The map applied to y; a map with a cut drops y, whatever it holds.
template <typename V>
__device__ __forceinline__ V apply(const Map<V>& m, bool cut, V y) {
  return cut ? m.b : vfma(m.x, y, m.b);
}

__device__ __forceinline__ void put_record(ulonglong2* r, float x, float b, unsigned tag) {
  ll_store2<LLScope::kGpu>(r, ll_word(__float_as_uint(x), tag), ll_word(__float_as_uint(b), tag));
}
// Publish a record for this lane's channels: tag = epoch * 2 + cut.
__device__ __forceinline__ void publish(const Grid& g, const Tile& t, int64_t B, int c, const Map<float>& m,
                                        unsigned tag) {
  if (c < g.H) put_record(g.recs + (int64_t(t.k) * B + t.b) * g.H + c, m.x, m.b, tag);
}
__device__ __forceinline__ void publish(const Grid& g, const Tile& t, int64_t B, int c, const Map<float2>& m,
                                        unsigned tag) {
  ulonglong2* r = g.recs + (int64_t(t.k) * B + t.b) * g.H + c;
  if (c < g.H) put_record(r, m.x.x, m.b.x, tag);
  if (c + 1 < g.H) put_record(r + 1, m.x.y, m.b.y, tag);
}

// A record of this epoch: waits (at most kWaitLimitNs) until its writer has published it.
__device__ __forceinline__ ulonglong2 wait_record(const ulonglong2* r, ulonglong2 x, unsigned epoch) {
  unsigned long long t0 = 0;
  for (unsigned spin = 1; unsigned(x.x >> 33) != epoch || unsigned(x.y >> 33) != epoch; ++spin) {
    if ((spin & 63u) == 0) {
      if (t0 == 0) {
        t0 = global_ns();
      } else if (global_ns() - t0 > kWaitLimitNs) {
        atomicOr(&g_b200_fault, kFaultWaitTimeout);
        break;
      }
    }
    x = ll_load2<LLScope::kGpu>(r);
  }
  return x;
}
__device__ __forceinline__ float low_float(unsigned long long v) { return __uint_as_float(unsigned(v)); }

// This lane's records as they are now.
template <int kVec>
struct Record {
  ulonglong2 x[kVec];
};
template <int kVec>
__device__ __forceinline__ Record<kVec> peek_record(const ulonglong2* r, int c, int H) {
  Record<kVec> q;
#pragma unroll
  for (int v = 0; v < kVec; ++v) q.x[v] = c + v < H ? ll_load2<LLScope::kGpu>(r + v) : make_ulonglong2(0ull, 0ull);
  return q;
}
// The same once they are there; cut: their writer's steps held a reset.
__device__ __forceinline__ void take_record(const ulonglong2* r, const Record<1>& q, int c, int H, unsigned epoch,
                                            Map<float>& m, unsigned& cut) {
  m = Map<float>{1.0f, 0.0f};
  cut = 0;
  if (c >= H) return;
  const ulonglong2 x = wait_record(r, q.x[0], epoch);
  m = Map<float>{low_float(x.x), low_float(x.y)};
  cut = unsigned(x.x >> 32) & 1u;
}
__device__ __forceinline__ void take_record(const ulonglong2* r, const Record<2>& q, int c, int H, unsigned epoch,
                                            Map<float2>& m, unsigned& cut) {
  m = Map<float2>{make_float2(1.0f, 1.0f), make_float2(0.0f, 0.0f)};
  cut = 0;
  if (c >= H) return;
  const ulonglong2 x = wait_record(r, q.x[0], epoch);
  const ulonglong2 y = c + 1 < H ? wait_record(r + 1, q.x[1], epoch) : x;
  m = Map<float2>{make_float2(low_float(x.x), low_float(y.x)), make_float2(low_float(x.y), low_float(y.y))};
  cut = unsigned(x.x >> 32) & 1u;
}

// The records of the tiles before tile t that what comes into it is formed from: n of them, the first (if the block
// is not the row's first) the state at the block's start, then the maps of the block's tiles before t.
struct Before {
  const ulonglong2* first;  // of this lane's channels
  int64_t step;
  unsigned n;
};
__device__ __forceinline__ Before records_before(const Grid& g, const Tile& t, int64_t B, int c) {
  const unsigned n = (t.k & (g.span - 1)) + (t.k >= g.span ? 1u : 0u);
  const int64_t step = B * g.H;
  return Before{g.recs + int64_t(t.k - n) * step + int64_t(t.b) * g.H + c, step, n};
}

// What comes into the tile, for this lane's channels: y on entry is the value before tile 0.  Warp w brings
// record w of every kWarps, kLook of them at a time.  Every thread of the CTA calls it.
template <int kVec, typename V, bool kBack, int kLook>
__device__ __forceinline__ void incoming(const Before& f, int c, int H, unsigned epoch, Shared<V, kBack, kLook>& sh,
                                         V& y) {
  static_assert(kLook % kWarps == 0 && kMaxSpan % kLook == 0, "");
  if (f.n == 0) return;
  const unsigned lane = threadIdx.x % 32, w = threadIdx.x / 32;
#pragma unroll 1
  for (unsigned from = 0; from < (kLook < kMaxSpan ? f.n : 1u); from += kLook) {
    if (from != 0) __syncthreads();  // the records before are used
    const unsigned n = kLook < kMaxSpan && f.n - from > kLook ? kLook : f.n - from;
    for (unsigned i = w; i < n; i += kWarps) {
      const ulonglong2* r = f.first + (from + i) * f.step;
      unsigned cut;
      Map<V> m;
      take_record(r, peek_record<kVec>(r, c, H), c, H, epoch, m, cut);
      sh.look[i][lane] = m;
      cut = __any_sync(0xffffffffu, cut);
      if (lane == 0) sh.look_cut[i] = cut;
    }
    __syncthreads();
    for (unsigned i = 0; i < n; ++i) y = apply(sh.look[i][lane], sh.look_cut[i] != 0, y);
  }
}

// The maps of the warps before warp w in the scan's direction, composed.
template <bool kUp, typename V>
__device__ __forceinline__ Map<V> before_warp(const Map<V> (&map)[kWarps][32], uint64_t cuts, unsigned w, bool& cut) {
  const unsigned lane = threadIdx.x % 32;
  Map<V> p{vset(V{}, 1.0f), vset(V{}, 0.0f)};
  cut = false;
#pragma unroll
  for (int i = 0; i < kWarps - 1; ++i) {
    const unsigned j = kUp ? i : kWarps - 1 - i;
    if (kUp ? j >= w : j <= w) break;
    const Map<V> m = map[j][lane];
    if (cuts == 0) {
      p = Map<V>{vmul(m.x, p.x), vfma(m.x, p.b, m.b)};
    } else {
      const bool now = ((cuts >> (8 * j)) & 1u) != 0u;
      cut = cut || now;
      p = Map<V>{vmul(m.x, p.x), apply(m, now, p.b)};
    }
  }
  return p;
}

__device__ __forceinline__ bool ends_block(const Grid& g, unsigned k) { return (k & (g.span - 1)) == g.span - 1; }

// Tickets, by the clerk.  The first comes with the launch's epoch: 31 bits, never 0 (a zero-filled record belongs to no
// launch).
__device__ __forceinline__ unsigned first_ticket(const Grid& g, unsigned& epoch) {
  epoch = 1u;
  if (g.ctl == nullptr) return blockIdx.x;
  unsigned before;  // read before this CTA's ticket is counted
  asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(before) : "l"(&g.ctl->epoch) : "memory");
  const unsigned e = (before + 1u) & 0x7fffffffu;
  epoch = e == 0u ? 1u : e;
  return atomicAdd(&g.ctl->ticket, 1u);
}
// The next one; where every CTA takes one only, a ticket past the last tile.
__device__ __forceinline__ unsigned next_ticket(const Grid& g, unsigned last) {
  if (g.ctl == nullptr) return last + gridDim.x;
  return g.one ? g.total : atomicAdd(&g.ctl->ticket, 1u);
}
// A CTA stops at its first ticket past the last tile, so every launch takes the same number of them, and who has the last
// leaves the workspace ready for the next launch.
__device__ __forceinline__ void settle(const Grid& g, unsigned ticket, unsigned epoch) {
  if (g.ctl != nullptr && ticket == (g.one ? g.total : g.total + gridDim.x) - 1u) {
    __threadfence();
    g.ctl->ticket = 0;
    g.ctl->epoch = epoch;
  }
}

// The resets of one warp's steps as bits (bit i: step i of the warp).
struct Resets {
  const uint8_t* p;
  Strides s;
  __device__ __forceinline__ uint8_t load(unsigned b, int64_t t, int64_t T) const {
    return p != nullptr && threadIdx.x % 32 < kSteps && t < T ? p[int64_t(b) * s.b + t * s.t] : uint8_t(0);
  }
};

// An input of the scan: rows of T at p, and the tensor map over [B, T, H] that loads a tile at once where
// `tma` (16-byte rows); `swap`: the map's second axis is the batch and its third the time.
template <typename T>
struct __align__(64) Input {
  CUtensorMap map;
  const T* p;
  Strides s;
  int swap;
};

// One tensor load of a tile (one thread).
template <typename T>
__device__ __forceinline__ void load_tile(const Input<T>& in, char* dst, const Tile& t, int64_t t0, uint64_t* bar) {
  const int c0 = int(t.group) * (kRowBytes / int(sizeof(T))), a = int(t0), b = int(t.b);
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::
          "r"(smem_addr(dst)),
      "l"(&in.map), "r"(c0), "r"(in.swap ? b : a), "r"(in.swap ? a : b), "r"(smem_addr(bar))
      : "memory");
}

// A warp's own rows of an input, by copies (every lane).
template <typename T>
__device__ __forceinline__ const char* warp_rows(const Input<T>& in, const Tile& t, int64_t t0) {
  return reinterpret_cast<const char*>(in.p + t.b * in.s.b + t0 * in.s.t + int64_t(t.group) * (kRowBytes / int(sizeof(T))));
}
template <typename T>
__device__ __forceinline__ void copy_tile(const Input<T>& in, char* dst, uint32_t* more, const Tile& t, int64_t t0,
                                          const Grid& g, int granule) {
  constexpr int kGroup = kRowBytes / int(sizeof(T));
  const int rows = int(g.T - t0 < kSteps ? g.T - t0 : kSteps);
  if (rows > 0)
    copy_rows(dst, more, warp_rows(in, t, t0), in.s.t * int64_t(sizeof(T)), rows,
              min(kGroup, g.H - int(t.group) * kGroup) * int(sizeof(T)), granule);
}
template <typename T>
__device__ __forceinline__ void align_tile(const Input<T>& in, char* dst, const uint32_t* more, const Tile& t,
                                           int64_t t0, const Grid& g) {
  const int rows = int(g.T - t0 < kSteps ? g.T - t0 : kSteps);
  if (rows > 0) align_rows(dst, more, warp_rows(in, t, t0), in.s.t * int64_t(sizeof(T)), rows);
}

// Dynamic shared memory: kIn inputs in two buffers, and the words behind the rows of unaligned copies.
constexpr int kMoreWords = kTile;
template <int kIn>
constexpr int smem_bytes(int granule) {
  return 2 * kIn * (kBufBytes + (granule == 2 ? kMoreWords * 4 : 0));
}
template <int kIn>
__device__ __forceinline__ char* buffer(char* smem, unsigned buf, int in) {
  return smem + (buf * kIn + in) * kBufBytes;
}
template <int kIn>
__device__ __forceinline__ uint32_t* more_of(char* smem, unsigned buf, int in) {
  return reinterpret_cast<uint32_t*>(smem + 2 * kIn * kBufBytes) + (buf * kIn + in) * kMoreWords;
}

// ------------------------------------------------------------------------------------- forward
template <typename T>
struct Forward {
  Input<T> gate, x;
  Grid g;
  Strides hs;
  const float* state;
  Resets reset;
  int64_t B;
  T* h;
  float *final_state, *ckpt;
  int granule;     // bytes that divide every row's address in gate and x
  bool tma, wide;  // tiles come by tensor loads; h rows take 4-byte stores
};

// Step 1 of the warp: a and v = u of its n steps, and their map.  kAny: fewer steps than kSteps, or resets.
// (In the decay form a and u are the inputs themselves, which step 4 reads again instead.)
template <typename T, int kForm, bool kAny, typename V>
__device__ __forceinline__ void forward_map(const char* row, unsigned resets, int n, V (&a)[kSteps], V (&u)[kSteps],
                                            Map<V>& m) {
  m = Map<V>{vset(V{}, 1.0f), vset(V{}, 0.0f)};
#pragma unroll
  for (int i = 0; i < kSteps; ++i) {
    if (kAny && i >= n) break;
    const uint32_t gt = *reinterpret_cast<const uint32_t*>(row + i * kRowBytes);
    const V xv = Lane<T>::unpack(*reinterpret_cast<const uint32_t*>(row + kBufBytes + i * kRowBytes));
    V ai, ui;
    if (kForm == kDecay) {
      ai = Lane<T>::unpack(gt);
      ui = xv;
    } else {
      V na;
      sigmoid_pair(Lane<T>::unpack_gate(gt), ai, na);
      ui = vmul(na, xv);
      a[i] = ai;
      u[i] = ui;
    }
    if (kAny && ((resets >> i) & 1u)) m = Map<V>{vset(V{}, 0.0f), vset(V{}, 0.0f)};
    m.b = vfma(ai, m.b, ui);
    m.x = vmul(m.x, ai);
  }
}

// Step 4: the warp's steps from its incoming state y, written to out.  !kAny: kSteps steps without resets,
// 4-byte stores.
template <typename T, int kForm, bool kAny, typename V>
__device__ __forceinline__ void forward_steps(const char* row, const V (&a)[kSteps], const V (&u)[kSteps],
                                              unsigned resets, int n, int c, int H, bool wide, T* out, int64_t pitch,
                                              V& y) {
#pragma unroll
  for (int i = 0; i < kSteps; ++i) {
    if (kAny && i >= n) break;
    if (kAny && ((resets >> i) & 1u)) y = vset(V{}, 0.0f);
    if (kForm == kDecay)
      y = vfma(Lane<T>::unpack(*reinterpret_cast<const uint32_t*>(row + i * kRowBytes)), y,
               Lane<T>::unpack(*reinterpret_cast<const uint32_t*>(row + kBufBytes + i * kRowBytes)));
    else
      y = vfma(a[i], y, u[i]);
    store_out<T>(out, c, H, !kAny || wide, y);
    out += pitch;
  }
}

// CTAs per SM: three, except in the sigmoid form of 16 bits, whose a and v of two channels take 128 registers a thread.
// Measured with two and with three: 1 x 65539 x 1024 fp32 177 and 154 us; decay, bf16: B = 8, T = 4096, H = 2048 76.3 and
// 73.7 us, B = 1, T = 65536, H = 1024 150 and 122 us (three need the records' buffer of two-channel lanes halved).  Sigmoid,
// bf16, three with a and v formed again in step 4: 93.8 us instead of 85.6, and 141 instead of 157 for the long
// sequence; with 6 of the 16 kept in registers 88.5 and 142.
template <typename T, int kForm>
constexpr bool kThreeCtas = sizeof(T) == 4 || kForm == kDecay;

template <typename T, int kForm>
__global__ void __launch_bounds__(kThreads, (kThreeCtas<T, kForm> ? 3 : 2)) forward_kernel(const __grid_constant__ Forward<T> p) {
  using V = typename Lane<T>::V;
  constexpr int kVec = Lane<T>::kVec, kIn = 2;
  extern __shared__ __align__(128) char smem[];
  __shared__ Shared<V, false, kThreeCtas<T, kForm> && kVec == 2 ? kWarps : kMaxSpan> sh;
  const unsigned lane = threadIdx.x % 32, w = threadIdx.x / 32;
  pdl_begin();
  // A tile's loads: tensor loads by one thread, or this warp's own rows.
  const auto load_all = [&](const Tile& t, unsigned buf) {
    if (!t.live) return;
    mbar_arrive_expect_tx(&sh.full[buf], kIn * kBufBytes);
    load_tile(p.gate, buffer<kIn>(smem, buf, 0), t, first_step(p.g, t), &sh.full[buf]);
    load_tile(p.x, buffer<kIn>(smem, buf, 1), t, first_step(p.g, t), &sh.full[buf]);
  };
  uint8_t reset_byte = 0;
  const auto fetch_own = [&](const Tile& t, unsigned buf) {
    if (!t.live) return;
    const int64_t t0 = first_step(p.g, t) + w * kSteps;
    reset_byte = p.reset.load(t.b, t0 + lane, p.g.T);
    if (!p.tma) {
      copy_tile(p.gate, buffer<kIn>(smem, buf, 0) + w * kSteps * kRowBytes, more_of<kIn>(smem, buf, 0) + w * kSteps, t,
                t0, p.g, p.granule);
      copy_tile(p.x, buffer<kIn>(smem, buf, 1) + w * kSteps * kRowBytes, more_of<kIn>(smem, buf, 1) + w * kSteps, t,
                t0, p.g, p.granule);
      cp_commit();
    }
  };
  const bool own = !p.tma || p.reset.p != nullptr;  // every warp fetches something itself

  const bool clerk = threadIdx.x == kClerk * 32;
  unsigned ahead = 0;
  if (clerk) {
    mbar_init(&sh.full[0], 1);
    mbar_init(&sh.full[1], 1);
    fence_barrier_init();
    unsigned e;
    ahead = first_ticket(p.g, e);
    sh.tile[0] = tile_of(p.g, ahead);
    if (p.tma) load_all(sh.tile[0], 0);
    sh.epoch = e;
    settle(p.g, ahead, e);
  }
  __syncthreads();
  const unsigned epoch = sh.epoch;
  if (own) fetch_own(sh.tile[0], 0);
  for (unsigned it = 0;; ++it) {
    const unsigned buf = it & 1u;
    if (it > 0) __syncthreads();  // the tile before is done: its buffer and the maps are free
    const Tile t = sh.tile[buf];
    if (!t.live) break;
    const int64_t t0 = first_step(p.g, t) + w * kSteps;            // this warp's first step
    const int n = int(p.g.T - t0 < kSteps ? p.g.T - t0 : kSteps);  // its steps (0 or less: none)
    const int c = (int(t.group) * 32 + int(lane)) * kVec;
    const int64_t state_at = int64_t(t.b) * p.g.H + c;
    char* rows = buffer<kIn>(smem, buf, 0) + w * kSteps * kRowBytes;
    if (p.tma) {
      mbar_wait(&sh.full[buf], (it >> 1) & 1u);
    } else {
      cp_wait_all();
      __syncwarp();
      if (p.granule == 2) {
        align_tile(p.gate, rows, more_of<kIn>(smem, buf, 0) + w * kSteps, t, t0, p.g);
        align_tile(p.x, rows + kBufBytes, more_of<kIn>(smem, buf, 1) + w * kSteps, t, t0, p.g);
      }
    }
    // The next ticket, once the rows are there: by then every CTA has its first.
    if (clerk) ahead = next_ticket(p.g, ahead);
    const unsigned resets = own ? __ballot_sync(0xffffffffu, reset_byte != 0) : 0u;
    const char* row = rows + lane * 4;

    // 1. The warp's steps as one map per channel; a and v stay in registers for step 4.
    V a[kSteps], u[kSteps];  // (decay: not used)
    Map<V> m;
    const bool plain = resets == 0 && n >= kSteps;
    if (plain)
      forward_map<T, kForm, false>(row, 0u, kSteps, a, u, m);
    else
      forward_map<T, kForm, true>(row, resets, n, a, u, m);
    sh.map[w][lane] = m;
    if (lane == 0) reinterpret_cast<uint8_t*>(&sh.cut)[w] = resets != 0;
    if (own && clerk) sh.tile[buf ^ 1] = tile_of(p.g, ahead);  // all warps need it at once
    __syncthreads();
    if (own) {
      fetch_own(sh.tile[buf ^ 1], buf ^ 1);
      if (p.tma && clerk) load_all(sh.tile[buf ^ 1], buf ^ 1);
    } else if (clerk) {
      sh.tile[buf ^ 1] = tile_of(p.g, ahead);
      load_all(sh.tile[buf ^ 1], buf ^ 1);
    }
    const uint64_t cuts = sh.cut;
    bool pre_cut;
    const Map<V> pre = before_warp<true>(sh.map, cuts, w, pre_cut);

    // 2. The tile's map, by the last warp; a tile that ends a block publishes its state in step 3.
    const bool ends = ends_block(p.g, t.k), more = t.k + 1 < p.g.n_tiles;
    if (w == kWarps - 1 && more) {
      m = Map<V>{vmul(m.x, pre.x), apply(m, resets != 0, pre.b)};
      if (!ends) publish(p.g, t, p.B, c, m, epoch * 2u + (cuts != 0 ? 1u : 0u));
    }

    // 3. The state that comes in.
    V y = vset(V{}, 0.0f);
    if (p.state != nullptr && t.k < p.g.span) load_row(p.state + state_at, c, p.g.H, y);
    incoming<kVec>(records_before(p.g, t, p.B, c), c, p.g.H, epoch, sh, y);
    if (w == kWarps - 1 && more && ends)
      publish(p.g, t, p.B, c, Map<V>{vset(V{}, 0.0f), apply(m, cuts != 0, y)}, epoch * 2u + 1u);
    if (w == 0 && p.ckpt != nullptr)
      store_row(p.ckpt + (int64_t(t.b) * p.g.n_tiles + t.k) * p.g.H + c, c, p.g.H, y);
    y = apply(pre, pre_cut, y);

    // 4. The steps from there.
    T* out = p.h + t.b * p.hs.b + t0 * p.hs.t + c;
    if (plain && p.wide)
      forward_steps<T, kForm, false>(row, a, u, 0u, kSteps, c, p.g.H, p.wide, out, p.hs.t, y);
    else
      forward_steps<T, kForm, true>(row, a, u, resets, n, c, p.g.H, p.wide, out, p.hs.t, y);
    if (p.final_state != nullptr && n > 0 && t0 + n == p.g.T) store_row(p.final_state + state_at, c, p.g.H, y);
  }
  if (clerk) settle(p.g, ahead, epoch);
}

// ------------------------------------------------------------------------------------ backward
template <typename T>
struct Backward {
  Input<T> gate, x, dh;
  Grid g;
  Strides ggs, gxs;
  const float *ckpt, *grad_final;
  Resets reset;
  int64_t B;
  T *grad_gate, *grad_x;
  float* grad_state;
  int granule;
  bool tma, wide;
};

constexpr int kHalf = kSteps / 2;

// What step 1 leaves of a warp's steps: a and 1 - a (decay: a alone), the state after the first half as a map of
// the state before it, and the forward offset and the backward map of them all.
template <typename V>
struct Steps {
  V a[kSteps], na[kSteps];
  Map<V> half, m;
  V f;
};

// In the order of time the backward map of steps 0 .. i is c -> P_i c + sum_j P_j grad_h[j], P_i the product of
// a up to step i, so it needs no second pass and its factor is the forward map's.
template <typename T, int kForm, bool kAny, typename V>
__device__ __forceinline__ void backward_map(const char* row, unsigned resets, int n, Steps<V>& q) {
  q.f = vset(V{}, 0.0f);
  q.m = q.half = Map<V>{vset(V{}, 1.0f), vset(V{}, 0.0f)};
  bool cut = false;
#pragma unroll
  for (int i = 0; i < kSteps; ++i) {
    if (kAny && i >= n) break;
    const uint32_t gt = *reinterpret_cast<const uint32_t*>(row + i * kRowBytes);
    V u = Lane<T>::unpack(*reinterpret_cast<const uint32_t*>(row + kBufBytes + i * kRowBytes));
    const V dv = Lane<T>::unpack(*reinterpret_cast<const uint32_t*>(row + 2 * kBufBytes + i * kRowBytes));
    if (kForm == kDecay) {
      q.a[i] = Lane<T>::unpack(gt);
    } else {
      sigmoid_pair(Lane<T>::unpack_gate(gt), q.a[i], q.na[i]);
      u = vmul(q.na[i], u);
    }
    if (kAny && ((resets >> i) & 1u)) {
      q.f = vset(V{}, 0.0f);
      cut = true;  // what lies behind a reset reaches no step before it
    }
    q.f = vfma(q.a[i], q.f, u);
    q.m.x = vmul(q.m.x, q.a[i]);
    if (!kAny || !cut) q.m.b = vfma(q.m.x, dv, q.m.b);
    if (i == kHalf - 1) q.half = Map<V>{q.m.x, q.f};
  }
}

// Step 4 for half the warp's steps, kFrom .. kFrom + kHalf - 1: the states before them, from the state s before the
// first, turned into what multiplies g in grad_gate (h[t-1], or (h[t-1] - x) a (1 - a)), then the steps
// backwards from the gradient y that comes in.  Half at a time keeps these factors in few registers.
template <typename T, int kForm, bool kAny, int kFrom, typename V>
__device__ __forceinline__ void backward_steps(const char* row, unsigned resets, int n, const Steps<V>& q, V s, int c,
                                               int H, bool wide, T* og, int64_t gpitch, T* ox, int64_t xpitch, V& y) {
  V d[kHalf];
#pragma unroll
  for (int k = 0; k < kHalf; ++k) {
    const int i = kFrom + k;
    if (kAny && i >= n) break;
    const V xv = Lane<T>::unpack(*reinterpret_cast<const uint32_t*>(row + kBufBytes + i * kRowBytes));
    if (kAny && ((resets >> i) & 1u)) s = vset(V{}, 0.0f);
    if (kForm == kDecay) {
      d[k] = s;
      s = vfma(q.a[i], s, xv);
    } else {
      d[k] = vmul(vsub(s, xv), vmul(q.a[i], q.na[i]));
      s = vfma(q.a[i], s, vmul(q.na[i], xv));
    }
  }
  og += (kFrom + kHalf - 1) * gpitch;
  ox += (kFrom + kHalf - 1) * xpitch;
#pragma unroll
  for (int k = kHalf - 1; k >= 0; --k) {
    const int i = kFrom + k;
    if (!kAny || i < n) {
      const V dv = Lane<T>::unpack(*reinterpret_cast<const uint32_t*>(row + 2 * kBufBytes + i * kRowBytes));
      const V g = vadd(dv, y);
      store_out<T>(og, c, H, !kAny || wide, vmul(g, d[k]));
      store_out<T>(ox, c, H, !kAny || wide, kForm == kDecay ? g : vmul(q.na[i], g));
      y = vmul(q.a[i], g);
      if (kAny && ((resets >> i) & 1u)) y = vset(V{}, 0.0f);
    }
    og -= gpitch;
    ox -= xpitch;
  }
}

// Tiles run from the last to the first (position k is time tile n_tiles - 1 - k).  The states h[t-1] of a
// tile are formed again from its checkpoint.
template <typename T, int kForm>
__global__ void __launch_bounds__(kThreads, 2) backward_kernel(const __grid_constant__ Backward<T> p) {
  using V = typename Lane<T>::V;
  constexpr int kVec = Lane<T>::kVec, kIn = 3;
  extern __shared__ __align__(128) char smem[];
  __shared__ Shared<V, true, kMaxSpan> sh;
  const unsigned lane = threadIdx.x % 32, w = threadIdx.x / 32;
  pdl_begin();
  // A tile's loads: tensor loads by one thread, or this warp's own rows.
  const auto load_all = [&](const Tile& t, unsigned buf) {
    if (!t.live) return;
    mbar_arrive_expect_tx(&sh.full[buf], kIn * kBufBytes);
    load_tile(p.gate, buffer<kIn>(smem, buf, 0), t, first_step(p.g, t), &sh.full[buf]);
    load_tile(p.x, buffer<kIn>(smem, buf, 1), t, first_step(p.g, t), &sh.full[buf]);
    load_tile(p.dh, buffer<kIn>(smem, buf, 2), t, first_step(p.g, t), &sh.full[buf]);
  };
  uint8_t reset_byte = 0;
  const auto fetch_own = [&](const Tile& t, unsigned buf) {
    if (!t.live) return;
    const int64_t t0 = first_step(p.g, t) + w * kSteps;
    reset_byte = p.reset.load(t.b, t0 + lane, p.g.T);
    if (!p.tma) {
      copy_tile(p.gate, buffer<kIn>(smem, buf, 0) + w * kSteps * kRowBytes, more_of<kIn>(smem, buf, 0) + w * kSteps, t,
                t0, p.g, p.granule);
      copy_tile(p.x, buffer<kIn>(smem, buf, 1) + w * kSteps * kRowBytes, more_of<kIn>(smem, buf, 1) + w * kSteps, t,
                t0, p.g, p.granule);
      copy_tile(p.dh, buffer<kIn>(smem, buf, 2) + w * kSteps * kRowBytes, more_of<kIn>(smem, buf, 2) + w * kSteps, t,
                t0, p.g, p.granule);
      cp_commit();
    }
  };
  const bool own = !p.tma || p.reset.p != nullptr;  // every warp fetches something itself

  const bool clerk = threadIdx.x == kClerk * 32;
  unsigned ahead = 0;
  if (clerk) {
    mbar_init(&sh.full[0], 1);
    mbar_init(&sh.full[1], 1);
    fence_barrier_init();
    unsigned e;
    ahead = first_ticket(p.g, e);
    sh.tile[0] = tile_of(p.g, ahead);
    if (p.tma) load_all(sh.tile[0], 0);
    sh.epoch = e;
    settle(p.g, ahead, e);
  }
  __syncthreads();
  const unsigned epoch = sh.epoch;
  if (own) fetch_own(sh.tile[0], 0);
  for (unsigned it = 0;; ++it) {
    const unsigned buf = it & 1u;
    if (it > 0) __syncthreads();  // the tile before is done: its buffer and the maps are free
    const Tile t = sh.tile[buf];
    if (!t.live) break;
    const unsigned kt = p.g.n_tiles - 1 - t.k;  // the time tile
    const int64_t t0 = first_step(p.g, t) + w * kSteps;
    const int n = int(p.g.T - t0 < kSteps ? p.g.T - t0 : kSteps);
    const int c = (int(t.group) * 32 + int(lane)) * kVec;
    const int64_t state_at = int64_t(t.b) * p.g.H + c;
    V s;  // the state before the tile
    load_row(p.ckpt + (int64_t(t.b) * p.g.n_tiles + kt) * p.g.H + c, c, p.g.H, s);
    char* rows = buffer<kIn>(smem, buf, 0) + w * kSteps * kRowBytes;
    if (p.tma) {
      mbar_wait(&sh.full[buf], (it >> 1) & 1u);
    } else {
      cp_wait_all();
      __syncwarp();
      if (p.granule == 2) {
        align_tile(p.gate, rows, more_of<kIn>(smem, buf, 0) + w * kSteps, t, t0, p.g);
        align_tile(p.x, rows + kBufBytes, more_of<kIn>(smem, buf, 1) + w * kSteps, t, t0, p.g);
        align_tile(p.dh, rows + 2 * kBufBytes, more_of<kIn>(smem, buf, 2) + w * kSteps, t, t0, p.g);
      }
    }
    // The next ticket, once the rows are there: by then every CTA has its first.
    if (clerk) ahead = next_ticket(p.g, ahead);
    const unsigned resets = own ? __ballot_sync(0xffffffffu, reset_byte != 0) : 0u;
    const char* row = rows + lane * 4;

    // 1. The warp's forward and backward maps.
    Steps<V> q;
    const bool plain = resets == 0 && n >= kSteps;
    if (plain)
      backward_map<T, kForm, false>(row, 0u, kSteps, q);
    else
      backward_map<T, kForm, true>(row, resets, n, q);
    sh.map[w][lane] = q.m;
    if (w < kWarps - 1) sh.fwd[w][lane] = q.f;  // (no warp comes after the last)
    if (lane == 0) reinterpret_cast<uint8_t*>(&sh.cut)[w] = resets != 0;
    if (own && clerk) sh.tile[buf ^ 1] = tile_of(p.g, ahead);  // all warps need it at once
    __syncthreads();
    if (own) {
      fetch_own(sh.tile[buf ^ 1], buf ^ 1);
      if (p.tma && clerk) load_all(sh.tile[buf ^ 1], buf ^ 1);
    } else if (clerk) {
      sh.tile[buf ^ 1] = tile_of(p.g, ahead);
      load_all(sh.tile[buf ^ 1], buf ^ 1);
    }
    const uint64_t cuts = sh.cut;
    bool pre_cut;
    const Map<V> pre = before_warp<false>(sh.map, cuts, w, pre_cut);

    // 2. The tile's map (from its last warp back), by warp 0, which holds the last of it.
    const bool ends = ends_block(p.g, t.k), more = t.k + 1 < p.g.n_tiles;
    Map<V> m;
    if (w == 0 && more) {
      m = Map<V>{vmul(q.m.x, pre.x), apply(q.m, resets != 0, pre.b)};
      if (!ends) publish(p.g, t, p.B, c, m, epoch * 2u + (cuts != 0 ? 1u : 0u));
    }

    // The state before the warp's steps, from the checkpoint, and in their middle.
#pragma unroll
    for (int j = 0; j < kWarps - 1; ++j) {
      if (j >= int(w)) break;
      const V x = sh.map[j][lane].x, f = sh.fwd[j][lane];
      s = cuts == 0 ? vfma(x, s, f) : apply(Map<V>{x, f}, ((cuts >> (8 * j)) & 1u) != 0u, s);
    }
    const V mid = apply(q.half, (resets & ((1u << kHalf) - 1u)) != 0u, s);

    // 3. The gradient that comes in.
    V y = vset(V{}, 0.0f);
    if (p.grad_final != nullptr && t.k < p.g.span) load_row(p.grad_final + state_at, c, p.g.H, y);
    incoming<kVec>(records_before(p.g, t, p.B, c), c, p.g.H, epoch, sh, y);
    if (w == 0 && more && ends)
      publish(p.g, t, p.B, c, Map<V>{vset(V{}, 0.0f), apply(m, cuts != 0, y)}, epoch * 2u + 1u);
    y = apply(pre, pre_cut, y);

    // 4. The steps from there, backwards.
    T* og = p.grad_gate + t.b * p.ggs.b + t0 * p.ggs.t + c;
    T* ox = p.grad_x + t.b * p.gxs.b + t0 * p.gxs.t + c;
    if (plain && p.wide) {
      backward_steps<T, kForm, false, kHalf>(row, 0u, kSteps, q, mid, c, p.g.H, true, og, p.ggs.t, ox, p.gxs.t, y);
      backward_steps<T, kForm, false, 0>(row, 0u, kSteps, q, s, c, p.g.H, true, og, p.ggs.t, ox, p.gxs.t, y);
    } else {
      backward_steps<T, kForm, true, kHalf>(row, resets, n, q, mid, c, p.g.H, p.wide, og, p.ggs.t, ox, p.gxs.t, y);
      backward_steps<T, kForm, true, 0>(row, resets, n, q, s, c, p.g.H, p.wide, og, p.ggs.t, ox, p.gxs.t, y);
    }
    if (p.grad_state != nullptr && t0 == 0) store_row(p.grad_state + state_at, c, p.g.H, y);
  }
  if (clerk) settle(p.g, ahead, epoch);
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
    float a = to_f32(gate[j * gsb + c]), v = to_f32(x[j * xsb + c]);
    if (kForm == kSigmoid) {
      float na;
      sigmoid_pair(clamp_gate(a), a, na);
      v = na * v;
    }
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
  g->one = *ctas == g->total;
  // Tiles of one chain that are worked on at once, rounded up to a power of two.
  unsigned span = 1;
  while (span < kMaxSpan && span * g->chains < resident) span *= 2;
  g->span = span;
  return kOk;
}

// The tensor map of an input over [B, T, H], boxes of kTile steps of one channel group.  false: the layout
// does not take one (rows off 16 bytes, shared rows, strides that are no multiples of one another).
template <typename T>
inline bool make_input_map(Input<T>* in, int64_t B, int64_t Tn, int64_t H) {
  const int64_t size = sizeof(T);
  int64_t st = in->s.t * size, sb = in->s.b * size;
  const int64_t row = (H * size + 15) / 16 * 16;
  in->swap = B > 1 && Tn > 1 && sb < st;
  if (Tn == 1) st = B == 1 ? row : sb;  // an axis of one step has no stride of its own
  if (B == 1) sb = st * Tn;
  const int64_t s1 = in->swap ? sb : st, s2 = in->swap ? st : sb;
  if (!aligned16(in->p) || s1 <= 0 || s1 % 16 != 0 || s2 % s1 != 0 || s2 >= (int64_t(1) << 40)) return false;
  const auto fn = tc::encode_fn();
  if (fn == nullptr) return false;
  const cuuint64_t dims[3] = {cuuint64_t(H), cuuint64_t(in->swap ? B : Tn), cuuint64_t(in->swap ? Tn : B)};
  const cuuint64_t strides[2] = {cuuint64_t(s1), cuuint64_t(s2)};
  const cuuint32_t box[3] = {cuuint32_t(kRowBytes / size), cuuint32_t(in->swap ? 1 : kTile),
                             cuuint32_t(in->swap ? kTile : 1)};
  const cuuint32_t step[3] = {1, 1, 1};
  const CUtensorMapDataType type = size == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_UINT16;
  return fn(&in->map, type, 3, const_cast<T*>(in->p), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
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
      p.gate.p = static_cast<const E*>(gate), p.x.p = static_cast<const E*>(x), p.h = static_cast<E*>(h);
      p.gate.s = Strides{strides[0], strides[1]}, p.x.s = Strides{strides[2], strides[3]};
      p.hs = Strides{strides[4], strides[5]};
      p.reset = Resets{reset, Strides{strides[6], strides[7]}};
      p.state = state, p.B = B, p.final_state = final_state, p.ckpt = ckpt;
      Granule in, out;
      in.add(gate, p.gate.s, sizeof(E)), in.add(x, p.x.s, sizeof(E)), out.add(h, p.hs, sizeof(E));
      p.tma = make_input_map(&p.gate, B, T, H) && make_input_map(&p.x, B, T, H);
      p.granule = in.bytes();
      p.wide = out.bytes() >= 4 && H % Lane<E>::kVec == 0;
      const int smem = smem_bytes<2>(p.granule);
      p.g.back = false;
      const auto kernel = forward_kernel<E, f.value>;
      unsigned ctas = 0;
      const int st = plan(kernel, smem, Lane<E>::kVec, B, T, H, ws, ws_bytes, &p.g, &ctas);
      return st != kOk ? st : launch_pdl(kernel, dim3(ctas), dim3(kThreads), size_t(smem), stream, p);
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
      p.gate.p = static_cast<const E*>(gate), p.x.p = static_cast<const E*>(x), p.dh.p = static_cast<const E*>(grad_h);
      p.grad_gate = static_cast<E*>(grad_gate), p.grad_x = static_cast<E*>(grad_x);
      p.gate.s = Strides{strides[0], strides[1]}, p.x.s = Strides{strides[2], strides[3]};
      p.dh.s = Strides{strides[4], strides[5]}, p.ggs = Strides{strides[6], strides[7]};
      p.gxs = Strides{strides[8], strides[9]};
      p.reset = Resets{reset, Strides{strides[10], strides[11]}};
      p.ckpt = ckpt, p.grad_final = grad_final, p.B = B, p.grad_state = grad_state;
      Granule in, out;
      in.add(gate, p.gate.s, sizeof(E)), in.add(x, p.x.s, sizeof(E)), in.add(grad_h, p.dh.s, sizeof(E));
      p.tma = make_input_map(&p.gate, B, T, H) && make_input_map(&p.x, B, T, H) && make_input_map(&p.dh, B, T, H);
      out.add(grad_gate, p.ggs, sizeof(E)), out.add(grad_x, p.gxs, sizeof(E));
      p.granule = in.bytes();
      p.wide = out.bytes() >= 4 && H % Lane<E>::kVec == 0;
      const int smem = smem_bytes<3>(p.granule);
      p.g.back = true;
      const auto kernel = backward_kernel<E, f.value>;
      unsigned ctas = 0;
      const int st = plan(kernel, smem, Lane<E>::kVec, B, T, H, ws, ws_bytes, &p.g, &ctas);
      return st != kOk ? st : launch_pdl(kernel, dim3(ctas), dim3(kThreads), size_t(smem), stream, p);
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
