// Selective state space scan: definitions shared by its kernels.
//
//   d_t = softplus(dt_t + bias)  (or dt_t + bias),   h_t = exp(d_t A) h_{t-1} + d_t x_t B_t,   y_t = C_t h_t + D x_t,  times SiLU(z_t)
// for every channel, with N states h and A [C][N], and with B_t, C_t [N] shared by a group's channels; a start at token t puts
// h_{t-1} = 0.
//
// What bounds it from below is exponentials: one per state, channel and token, 16 per SM and clock, where memory would allow twice as
// many at N = 16 (16 x 2048 tokens of 1536 channels, 8.05e8 states: 179 us, 224 us with those of steps and gates; 1115 MB of a training
// step 170 us).  What bounds it now is all of issue slots, exponentials and shared-memory reads together: 73 instructions per token and
// 16 channels forward (57 % of issue slots, 60 % of exponentials on average, a sixth more on SMs with three blocks of 2.6), 214
// backward.  A thread holds SEL_EACH states of two neighbouring channels (of one where N <= 8); NP / SEL_EACH lanes share a channel.
// Four warps of a block scan; four others (SEL_THREADS each) do what is done once per token and channel: they copy tiles of SEL_TILE
// tokens ahead (cp.async), turn them into (step, step times x) pairs in float32 in shared memory a tile before the scan, and write the
// results a tile behind it, so that the two kinds of work hide one another's latency.  One barrier of the block per tile.
#pragma once

#include "ttt_kernels.h"
#include "ttt_vec.cuh"

namespace ttt {

constexpr int SEL_THREADS = 128;  // of each kind
constexpr int SEL_STAGES = 3;     // tiles of inputs in shared memory
constexpr int SEL_EACH = 4;  // states per thread

template <int NP>
struct SelShape {
  static constexpr int SL = NP / SEL_EACH;         // lanes that share a channel
  static constexpr int CL = 32 / SL;               // lanes with channels of their own
  static constexpr int CC = SL >= 4 ? 2 : 1;       // channels of a thread
  static constexpr int WARP_CH = CL * CC;
  static constexpr int CH = WARP_CH * (SEL_THREADS / 32);  // of a block: 128, 64, 64, 32, 16
  static constexpr int PAIRS = CH / 2;
  static constexpr int ROWS = SEL_THREADS / PAIRS;         // tokens that the block's threads cover, pair by pair
  static constexpr int SHARES = SL * CH;           // floats of a token's results as the scanning lanes have them
};

// The lanes' shares of a token's results in shared memory: lane sl's of the pair (or, CC = 1, the channel) of channels `e` at e SL + sl
// pairs (floats), lanes of a pair in an order by which sixteen neighbouring pairs lie in different banks.
template <int NP>
__device__ __forceinline__ int share_at(int e, int sl) {
  using S = SelShape<NP>;
  if constexpr (S::CC == 1) return e * S::SL + sl;
  else return 2 * (e * S::SL + (sl ^ (e / (16 / S::SL) & (S::SL - 1))));
}
// a pair's sum over its lanes
template <int NP>
__device__ __forceinline__ F2 sum_shares(const float* row, int pr) {
  using S = SelShape<NP>;
  F2 v = f2(0.f);
#pragma unroll 4
  for (int l = 0; l < S::SL; ++l) {
    if constexpr (S::CC == 2) v = f2add(v, *reinterpret_cast<const float2*>(row + share_at<NP>(pr, l)));
    else v = f2add(v, f2(row[share_at<NP>(2 * pr, l)], row[share_at<NP>(2 * pr + 1, l)]));
  }
  return v;
}

// The decay exp(d A), A times log2 e.  ex2.approx errs low by up to 2.7e-8 on average between -0.06 and 0 (measured), where decays of
// long memories lie: thousands of them in a product lean that way.  An exponent greater by 2.2e-8 leaves 1e-8 of it, and 1 for a step
// of zero (measured); error of a state after 8192 tokens: tests/test_selective_scan_gpu.py.
__device__ __forceinline__ F2 decay_of(F2 A, F2 d) { return ex2(f2fma(A, d, f2(2.2e-8f))); }
__device__ __forceinline__ F2 decay_of(F2 A, float d) { return decay_of(A, f2(d)); }

// A rate times log2 e, at least -2^100: a rate of -inf keeps nothing over steps from 2^-93 (1e-28) on, and all over a step of zero, where 0
// times -inf would be a NaN (the places behind the last token are such steps); a rate times a state's gradient stays finite, so that softplus's
// slope of zero there makes zero of it.  A comparison per step instead would cost the backward 1 to 11 % where there are starts.
__device__ __forceinline__ float rate_of(float a) { return a * LOG2E < -0x1p100f ? -0x1p100f : a * LOG2E; }

// log(1 + exp(v)) = max(v, 0) + log(1 + e), e = exp(-|v|) in (0, 1].  log(1 + e) / e is a polynomial of degree 8, fitted on [0, 1] for
// the least largest relative error (3.0e-8): accurate relative to small steps too, which a logarithm of 1 + e is not, and without a
// quotient, whose place among the exponentials it would take.  Two channels at once; a NaN stays one.
__device__ __forceinline__ F2 softplus_of(F2 v) {
  const F2 e = f2(ex2(-LOG2E * fabsf(v.x)), ex2(-LOG2E * fabsf(v.y)));
  F2 r = f2fma(e, f2(0.005232690833508968f), f2(-0.029505228623747826f));
  r = f2fma(e, r, f2(0.07822594791650772f));
  r = f2fma(e, r, f2(-0.13663245737552643f));
  r = f2fma(e, r, f2(0.19106008112430573f));
  r = f2fma(e, r, f2(-0.2484298199415207f));
  r = f2fma(e, r, f2(0.3331909775733948f));
  r = f2fma(e, r, f2(-0.4999949336051941f));
  r = f2fma(e, r, f2(0.9999999403953552f));
  return f2fma(e, r, f2(v.x < 0.f ? 0.f : v.x, v.y < 0.f ? 0.f : v.y));
}

__device__ __forceinline__ void copy_async16(void* dst, const void* src, bool live) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(live ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy_async4(void* dst, const void* src, bool live) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(live ? 4 : 0) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// the block's threads that do not scan
__device__ __forceinline__ void helpers_sync() { asm volatile("bar.sync 1, %0;" ::"n"(SEL_THREADS) : "memory"); }
__device__ __forceinline__ void copy_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// rows [t0, t0 + SEL_TILE) of `have` elements, at most WIDE, into dst [SEL_TILE][WIDE]; zeros beyond T and `have`.  bytes: 16, 4, or an
// element's size, what addresses, strides and `have` are multiples of; by elements, AHEAD are on their way at a time.
template <typename T, int WIDE, int AHEAD>
__device__ __forceinline__ void copy_rows(int tid, T* dst, const T* src, int64_t stride, int64_t t0, int64_t t_end, int have, int bytes) {
  constexpr int V16 = 16 / sizeof(T);
  if (WIDE >= V16 && bytes == 16) {
    constexpr int V = WIDE >= V16 ? V16 : 1, PER = WIDE / V;
    for (int i = tid; i < SEL_TILE * PER; i += SEL_THREADS) {
      const int r = i / PER, e = (i - r * PER) * V;
      const bool live = t0 + r < t_end && e < have;
      copy_async16(dst + r * WIDE + e, live ? src + (t0 + r) * stride + e : src, live);
    }
  } else if (bytes >= 4) {
    constexpr int V = 4 / sizeof(T), PER = WIDE / V;
    for (int i = tid; i < SEL_TILE * PER; i += SEL_THREADS) {
      const int r = i / PER, e = (i - r * PER) * V;
      const bool live = t0 + r < t_end && e < have;
      copy_async4(dst + r * WIDE + e, live ? src + (t0 + r) * stride + e : src, live);
    }
  } else {
    constexpr int MOST = (SEL_TILE * WIDE + SEL_THREADS - 1) / SEL_THREADS, PER = MOST < AHEAD ? MOST : AHEAD;
    for (int i0 = tid; i0 < SEL_TILE * WIDE; i0 += PER * SEL_THREADS) {
      T v[PER];
#pragma unroll
      for (int k = 0; k < PER; ++k) {
        const int i = i0 + k * SEL_THREADS, r = i / WIDE, e = i - r * WIDE;
        v[k] = T(0.f);
        if (i < SEL_TILE * WIDE && t0 + r < t_end && e < have) v[k] = src[(t0 + r) * stride + e];
      }
#pragma unroll
      for (int k = 0; k < PER; ++k)
        if (i0 + k * SEL_THREADS < SEL_TILE * WIDE) dst[i0 + k * SEL_THREADS] = v[k];
    }
  }
}

// Two neighbouring channels of a row, from shared memory and to global memory (whole: both exist and lie on a pair's address)
__device__ __forceinline__ float2 pair_of(const float* p) { return *reinterpret_cast<const float2*>(p); }
__device__ __forceinline__ float2 pair_of(const __nv_bfloat16* p) {
  const uint32_t v = *reinterpret_cast<const uint32_t*>(p);
  return make_float2(bf16_lo(v), bf16_hi(v));
}
template <typename T>
__device__ __forceinline__ void put_pair(T* p, float2 v, int have, bool whole) {
  if (whole) {
    if constexpr (sizeof(T) == 4) *reinterpret_cast<float2*>(p) = v;
    else *reinterpret_cast<uint32_t*>(p) = pack_bf16(v.x, v.y);
  } else {
    if (have > 0) st_from_float<T>(p, 0, v.x);
    if (have > 1) st_from_float<T>(p, 1, v.y);
  }
}

// v[i] summed over the LANES lanes that differ in the lane bits STRIDE, 2 STRIDE, ...; the lane with number k among them gets v[k]
// (COUNT = LANES), or v[k COUNT / LANES ...] in v[0 ...] (COUNT > LANES), or the one that k's high bits name (COUNT < LANES).
template <int COUNT, int LANES, int STRIDE>
__device__ __forceinline__ void sum_and_deal(float (&v)[COUNT], int lane) {
  constexpr int STEPS = LANES == 1 ? 0 : LANES == 2 ? 1 : LANES == 4 ? 2 : LANES == 8 ? 3 : LANES == 16 ? 4 : 5;
  int n = COUNT, o = LANES / 2;
#pragma unroll
  for (int k = 0; k < STEPS; ++k) {
    const bool up = (lane & (o * STRIDE)) != 0;
    if (n > 1) {
#pragma unroll
      for (int i = 0; i < COUNT / 2; ++i)
        if (i < n / 2) {
          const float send = up ? v[i] : v[i + n / 2], keep = up ? v[i + n / 2] : v[i];
          v[i] = keep + __shfl_xor_sync(0xffffffffu, send, o * STRIDE);
        }
      n /= 2;
    } else {
      v[0] += __shfl_xor_sync(0xffffffffu, v[0], o * STRIDE);
    }
    o /= 2;
  }
}

// Where a block stands: batch row, group, its channels, its segment of the tokens
template <int NP>
struct SelPlace {
  using S = SelShape<NP>;
  int64_t b;
  int g, block, seg, c0, have;  // have: channels of the block that exist
  int64_t t_lo, t_hi;           // tokens of the segment
  // blocks of `segments` segments, from `first` on
  __device__ __forceinline__ SelPlace(const SelParams& p, int first, int segments) {
    const int each = p.C / p.G, blocks = (each + S::CH - 1) / S::CH;
    int64_t i = blockIdx.x;
    block = (int)(i % blocks), i /= blocks;
    g = (int)(i % p.G), i /= p.G;
    seg = first + (int)(i % segments), b = i / segments;
    c0 = g * each + block * S::CH;
    have = min(S::CH, each - block * S::CH);
    t_lo = (int64_t)seg * p.seg_tiles * SEL_TILE;
    t_hi = min(p.T, t_lo + (int64_t)p.seg_tiles * SEL_TILE);
  }
};

// Rates of a thread's channels (times log2 e), and what is read and written as [C][N] or [C][NP] rows
template <int NP>
struct SelLane {
  using S = SelShape<NP>;
  int lane, sl, ch;  // ch: the first of the thread's channels, in the block
  __device__ __forceinline__ SelLane() {
    lane = threadIdx.x & 31;
    sl = lane & (S::SL - 1);
    ch = (threadIdx.x >> 5) * S::WARP_CH + (lane / S::SL) * S::CC;
  }
  // rates, as rate_of gives them
  __device__ __forceinline__ void load_rates(F2 (&A)[S::CC][2], const float* rows, int n, int have) const {
    load(A, rows, n, have);
#pragma unroll
    for (int k = 0; k < S::CC; ++k)
#pragma unroll
      for (int i = 0; i < 2; ++i) A[k][i] = f2(rate_of(A[k][i].x), rate_of(A[k][i].y));
  }
  // row of `n` states (N in memory) of channel c0 + ch + k, zeros beyond
  __device__ __forceinline__ void load(F2 (&v)[S::CC][2], const float* rows, int n, int have) const {
#pragma unroll
    for (int k = 0; k < S::CC; ++k) {
      float e[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) e[i] = rows != nullptr && ch + k < have && 4 * sl + i < n ? rows[(int64_t)(ch + k) * n + 4 * sl + i] : 0.f;
      v[k][0] = f2(e[0], e[1]), v[k][1] = f2(e[2], e[3]);
    }
  }
  __device__ __forceinline__ void store(const F2 (&v)[S::CC][2], float* rows, int n, int have) const {
#pragma unroll
    for (int k = 0; k < S::CC; ++k) {
      if (ch + k >= have) continue;
      float* at = rows + (int64_t)(ch + k) * n + 4 * sl;
      if (n == NP) {
        *reinterpret_cast<float4*>(at) = make_float4(v[k][0].x, v[k][0].y, v[k][1].x, v[k][1].y);
      } else {
        if (4 * sl < n) at[0] = v[k][0].x;
        if (4 * sl + 1 < n) at[1] = v[k][0].y;
        if (4 * sl + 2 < n) at[2] = v[k][1].x;
        if (4 * sl + 3 < n) at[3] = v[k][1].y;
      }
    }
  }
  // [C][NP] rows
  __device__ __forceinline__ void load_padded(F2 (&v)[S::CC][2], const float* rows, int have) const {
#pragma unroll
    for (int k = 0; k < S::CC; ++k) {
      float4 e = make_float4(0.f, 0.f, 0.f, 0.f);
      if (ch + k < have) e = *reinterpret_cast<const float4*>(rows + (int64_t)(ch + k) * NP + 4 * sl);
      v[k][0] = f2(e.x, e.y), v[k][1] = f2(e.z, e.w);
    }
  }
};

}  // namespace ttt
