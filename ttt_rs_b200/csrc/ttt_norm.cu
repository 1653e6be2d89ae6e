// Group norm with channels last, [B,T,C], forward and backward, with an activation or a gate.
//
//   n = (x - mean) / sqrt(var + eps) over a group of c = C / G neighbouring channels, of one token or of a whole sequence
//   u = n w + b;    y = act(u), or u act(gate)
// Gradients, with du = dy act'(u) or dy act(gate), p = du w and means over the group:
//   dx = (p - mean(p) - n mean(p n)) / sqrt(var + eps),  dw = sum du n,  db = sum du,  dgate = dy u act'(gate)
// Variances are sums of squares of differences from the mean, never differences of sums.
//
// Memory-bound.
//   A token's groups: eight channels per thread, a group to a power of two of lanes (several warps where it has more than 256
//   channels), everything in registers between one read and one write, but for what spills: nothing in the gradient of bf16 vectors with
//   SiLU, 80 bytes per thread with another activation, 84 of float32 vectors, 128 of float32 pairs, 496 (bf16) and 708 (float32) channel by
//   channel, whose eight places per thread have a weight, a bias and two sums each.  A thread keeps its channels from token to token, so that
//   weights and their gradients stay in registers; the backward's blocks leave a row of sums each, joined in a fixed order.  bf16, 65536
//   tokens of 24 heads of 64 channels with gate: 117 us (5.2 TB/s, 0.79 of a copy), gradient 212 us (4.7 TB/s, 0.72; with two tokens at a
//   time, which two instead of three blocks per SM have room for, 250 us); SiLU known when the kernel is built: 151 and 455 us before that.
//   One group of 1536 channels: 252 and 533 us, the barriers of the block's sums.
//   A sequence's groups: a pass for the statistics (backward: for every channel's sums of du and du n) and one that applies them,
//   which reads x again, from L2 where the tensors fit.  Chunks of tokens leave (mean, sum of squares) pairs that every block of the
//   second pass joins in the same order.  16 x 4096 x 512: 20 + 28 us, gradient 39 + 5 + 38 + 3 us (135 MB in and out 2.8 TB/s forward).
#include "ttt_kernels.h"
#include "ttt_vec.cuh"

namespace ttt {

constexpr int NORM_THREADS = 256;
constexpr int NORM_FWD_RESIDENT = 4, NORM_BWD_RESIDENT = 3, NORM_SEQ_RESIDENT = 3;  // blocks of 256 threads per SM that registers are bounded for
constexpr int NORM_EACH = 8;  // channels per thread, a token's groups
constexpr int NORM_WIDE = NORM_TOKEN_CHANNELS / NORM_EACH;  // threads at most, of groups that several warps share

// What a kernel knows of the call when it is built: everything at run time, SiLU without a gate, or a gate with SiLU
enum : int { NORM_GENERAL = 0, NORM_SILU = 1, NORM_GATED_SILU = 2 };
template <int MODE>
__device__ __forceinline__ bool norm_gated(const NormParams& p) {
  return MODE == NORM_GATED_SILU || (MODE == NORM_GENERAL && p.gate != nullptr);
}
template <int MODE>
__device__ __forceinline__ int norm_act(const NormParams& p) {
  return MODE == NORM_GENERAL ? p.act : ACT_SILU;
}
// A place among the tokens, walked in steps: its offsets in x, the gate and the result's gradient
struct NormWalk {
  uint32_t t;  // of its sequence
  int64_t x, gate, gy;
  __device__ __forceinline__ NormWalk(const NormParams& p, int64_t token) {
    const int64_t b = token / p.T;
    t = (uint32_t)(token - b * p.T);
    x = b * p.xs[0] + t * p.xs[1];
    gate = b * p.gates[0] + t * p.gates[1];
    gy = b * p.gys[0] + t * p.gys[1];
  }
  __device__ __forceinline__ void step(const NormParams& p, uint32_t by) {
    t += by;
    x += by * p.xs[1];
    gate += by * p.gates[1];
    gy += by * p.gys[1];
    if (t >= (uint32_t)p.T) {
      const uint32_t rows = t / (uint32_t)p.T;
      t -= rows * (uint32_t)p.T;
      x += rows * (p.xs[0] - p.T * p.xs[1]);
      gate += rows * (p.gates[0] - p.T * p.gates[1]);
      gy += rows * (p.gys[0] - p.T * p.gys[1]);
    }
  }
};

// Sums over the lanes of a group.  WIDE: over its warps too, through shared memory; all threads of the block take part, and the sums
// go round four places, so that one barrier each is enough.
template <bool WIDE>
struct NormSum;
template <>
struct NormSum<false> {
  __device__ __forceinline__ float operator()(float v, int lanes) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
      if (o < lanes) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
  }
};
template <>
struct NormSum<true> {
  float* red;  // [4][warps]
  int turn = 0;
  __device__ __forceinline__ float operator()(float v, int lanes) {
    constexpr int WARPS = NORM_WIDE / 32;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    const int warp = threadIdx.x >> 5, warps = lanes >> 5, first = warp & ~(warps - 1);
    float* at = red + (turn++ & 3) * WARPS;
    if ((threadIdx.x & 31) == 0) at[warp] = v;
    __syncthreads();
    v = 0.f;
#pragma unroll
    for (int k = 0; k < WARPS; ++k)
      if (k < warps) v += at[first + k];
    return v;
  }
};
template <bool WIDE>
__device__ __forceinline__ NormSum<WIDE> norm_sum() {
  if constexpr (WIDE) {
    __shared__ float red[4 * NORM_WIDE / 32];
    return {red};
  } else {
    return {};
  }
}

template <typename T, int V>
struct NormLane {  // a thread's channels
  static constexpr int NV = NORM_EACH / V, P = Chan<T, V>::P;
  int c0;           // first channel of the group
  int at[NV];       // channels of the group: V from each on, or -1
  F2 w[NV][P], b[NV][P];
  __device__ __forceinline__ void set(const NormParams& p, int g, int l, bool live) {
    c0 = g * p.c;
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      const int e = (n * p.lanes + l) * V;
      at[n] = live && e < p.c ? e : -1;
#pragma unroll
      for (int k = 0; k < P; ++k) w[n][k] = f2(1.f), b[n][k] = f2(0.f);
      if (at[n] >= 0) {
        Chan<T, V> r;
        if (p.w != nullptr) r.load(static_cast<const T*>(p.w) + c0 + at[n]), r.unpack(w[n]);
        if (p.bias != nullptr) r.load(static_cast<const T*>(p.bias) + c0 + at[n]), r.unpack(b[n]);
      }
    }
  }
};

// difference from the mean and 1 / sqrt(var + eps) of a thread's channels (d: the channels on entry)
template <typename T, int V, bool WIDE>
__device__ __forceinline__ float norm_stats(F2 (&d)[NormLane<T, V>::NV][NormLane<T, V>::P], const NormLane<T, V>& me, const NormParams& p,
                                            NormSum<WIDE>& sum) {
  using L = NormLane<T, V>;
  F2 s = f2(0.f);
#pragma unroll
  for (int n = 0; n < L::NV; ++n)
#pragma unroll
    for (int k = 0; k < L::P; ++k) s = f2add(s, d[n][k]);
  const float mean = sum(f2hsum(s), p.lanes) * p.inv_c;
  F2 q = f2(0.f);
#pragma unroll
  for (int n = 0; n < L::NV; ++n)
#pragma unroll
    for (int k = 0; k < L::P; ++k) {
      d[n][k] = me.at[n] < 0 ? f2(0.f) : f2(d[n][k].x - mean, V > 1 ? d[n][k].y - mean : 0.f);
      q = f2fma(d[n][k], d[n][k], q);
    }
  return rsqrtf(sum(f2hsum(q), p.lanes) * p.inv_c + p.eps);
}

template <typename T, int V, bool WIDE, int MODE>
__global__ void __launch_bounds__(WIDE ? NORM_WIDE : NORM_THREADS, WIDE ? NORM_FWD_RESIDENT / 2 : NORM_FWD_RESIDENT) ttt_norm_token_kernel(const NormParams p) {
  using Ch = Chan<T, V>;
  using L = NormLane<T, V>;
  constexpr int NV = L::NV, P = L::P, AHEAD = V == 1 || sizeof(T) == 4 ? 1 : 2;
  NormSum<WIDE> sum = norm_sum<WIDE>();
  const int row = threadIdx.x / p.cols, col = threadIdx.x - row * p.cols, gcol = (int)blockIdx.y * p.cols + col;
  const int g = gcol / p.lanes, l = gcol & (p.lanes - 1), act = norm_act<MODE>(p);
  const bool live = row < p.rows && g < p.G, gated = norm_gated<MODE>(p);
  L me;
  me.set(p, g, l, live);
  const T* x = static_cast<const T*>(p.x) + me.c0;
  const T* gate = static_cast<const T*>(p.gate) + me.c0;
  const uint32_t step = gridDim.x * p.rows;
  int64_t token = (int64_t)blockIdx.x * p.rows + row;
  T* y = static_cast<T*>(p.y) + token * p.C + me.c0;
  NormWalk at(p, token);
  for (int64_t base = (int64_t)blockIdx.x * p.rows; base < p.tokens; base += (int64_t)step * AHEAD) {
    Ch in[AHEAD][NV], gt[AHEAD][NV];
    bool has[AHEAD];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      has[u] = live && token < p.tokens;
#pragma unroll
      for (int n = 0; n < NV; ++n) {
        in[u][n].zero();
        gt[u][n].zero();
        if (has[u] && me.at[n] >= 0) {
          in[u][n].load(x + at.x + me.at[n]);
          if (gated) gt[u][n].load(gate + at.gate + me.at[n]);
        }
      }
      token += step;
      at.step(p, step);
    }
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      if (u > 0 && base + (int64_t)u * step >= p.tokens) break;  // (the whole block)
      F2 d[NV][P];
#pragma unroll
      for (int n = 0; n < NV; ++n) in[u][n].unpack(d[n]);
      const float r = norm_stats<T, V, WIDE>(d, me, p, sum);
#pragma unroll
      for (int n = 0; n < NV; ++n) {
        F2 e[P];
        gt[u][n].unpack(e);
#pragma unroll
        for (int k = 0; k < P; ++k) {
          const F2 v = f2fma(f2mul(d[n][k], f2(r)), me.w[n][k], me.b[n][k]);
          if (gated) d[n][k] = f2mul(v, f2(act_of(e[k].x, act), act_of(e[k].y, act)));
          else d[n][k] = f2(act_of(v.x, act), act_of(v.y, act));
        }
        if (has[u] && me.at[n] >= 0) {
          Ch out;
          out.pack(d[n]);
          out.store(y + me.at[n]);
        }
      }
      y += (int64_t)step * p.C;
    }
  }
}

template <typename T, int V, bool WIDE, int MODE>
__global__ void __launch_bounds__(WIDE ? NORM_WIDE : NORM_THREADS, WIDE ? 1 : NORM_BWD_RESIDENT) ttt_norm_token_bwd_kernel(const NormParams p) {
  using Ch = Chan<T, V>;
  using L = NormLane<T, V>;
  constexpr int NV = L::NV, P = L::P, AHEAD = 1;
  NormSum<WIDE> sum = norm_sum<WIDE>();
  const int row = threadIdx.x / p.cols, col = threadIdx.x - row * p.cols, gcol = (int)blockIdx.y * p.cols + col;
  const int g = gcol / p.lanes, l = gcol & (p.lanes - 1), act = norm_act<MODE>(p);
  const bool live = row < p.rows && g < p.G, gated = norm_gated<MODE>(p);
  L me;
  me.set(p, g, l, live);
  const T* x = static_cast<const T*>(p.x) + me.c0;
  const T* gate = static_cast<const T*>(p.gate) + me.c0;
  const T* gy = static_cast<const T*>(p.gy) + me.c0;
  const uint32_t step = gridDim.x * p.rows;
  int64_t token = (int64_t)blockIdx.x * p.rows + row, to = token * p.C + me.c0;
  T* gx = static_cast<T*>(p.gx);
  T* ggate = static_cast<T*>(p.ggate);
  NormWalk at(p, token);
  F2 dw[NV][P], db[NV][P];
#pragma unroll
  for (int n = 0; n < NV; ++n)
#pragma unroll
    for (int k = 0; k < P; ++k) dw[n][k] = db[n][k] = f2(0.f);
  for (int64_t base = (int64_t)blockIdx.x * p.rows; base < p.tokens; base += (int64_t)step * AHEAD) {
    Ch in[AHEAD][NV], gt[AHEAD][NV], gr[AHEAD][NV];
    bool has[AHEAD];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      has[u] = live && token < p.tokens;
#pragma unroll
      for (int n = 0; n < NV; ++n) {
        in[u][n].zero();
        gt[u][n].zero();
        gr[u][n].zero();
        if (has[u] && me.at[n] >= 0) {
          in[u][n].load(x + at.x + me.at[n]);
          gr[u][n].load(gy + at.gy + me.at[n]);
          if (gated) gt[u][n].load(gate + at.gate + me.at[n]);
        }
      }
      token += step;
      at.step(p, step);
    }
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      if (u > 0 && base + (int64_t)u * step >= p.tokens) break;  // (the whole block)
      F2 d[NV][P];
#pragma unroll
      for (int n = 0; n < NV; ++n) in[u][n].unpack(d[n]);
      const float stat = norm_stats<T, V, WIDE>(d, me, p, sum), r = has[u] ? stat : 0.f;  // (no token: 1 / sqrt(0 + eps) may be infinite)
      F2 q[NV][P], s1 = f2(0.f), s2 = f2(0.f);
#pragma unroll
      for (int n = 0; n < NV; ++n) {
        F2 e[P], du[P], dg[P];
        gr[u][n].unpack(du);
        gt[u][n].unpack(e);
#pragma unroll
        for (int k = 0; k < P; ++k) {
          d[n][k] = f2mul(d[n][k], f2(r));  // n
          const F2 v = f2fma(d[n][k], me.w[n][k], me.b[n][k]);
          F2 a, slope;
          if (gated) {
            a.x = act_and_slope(e[k].x, act, slope.x);
            a.y = act_and_slope(e[k].y, act, slope.y);
            dg[k] = f2mul(f2mul(du[k], v), slope);
            du[k] = f2mul(du[k], a);
          } else {
            act_and_slope(v.x, act, slope.x);
            act_and_slope(v.y, act, slope.y);
            du[k] = f2mul(du[k], slope);
          }
          dw[n][k] = f2fma(du[k], d[n][k], dw[n][k]);
          db[n][k] = f2add(db[n][k], du[k]);
          q[n][k] = f2mul(du[k], me.w[n][k]);
          s1 = f2add(s1, q[n][k]);
          s2 = f2fma(q[n][k], d[n][k], s2);
        }
        if (gated && has[u] && me.at[n] >= 0) {
          Ch out;
          out.pack(dg);
          out.store(ggate + to + me.at[n]);
        }
      }
      const float m1 = sum(f2hsum(s1), p.lanes) * p.inv_c, m2 = sum(f2hsum(s2), p.lanes) * p.inv_c;
#pragma unroll
      for (int n = 0; n < NV; ++n) {
#pragma unroll
        for (int k = 0; k < P; ++k) q[n][k] = f2mul(f2fma(d[n][k], f2(-m2), f2add(q[n][k], f2(-m1))), f2(r));
        if (has[u] && me.at[n] >= 0) {
          Ch out;
          out.pack(q[n]);
          out.store(gx + to + me.at[n]);
        }
      }
      to += (int64_t)step * p.C;
    }
  }
  if (p.partials == nullptr) return;
  // this block's sums for the weights, over its rows in their order: [2][C]
  extern __shared__ float norm_smem[];  // [2][rows][cols][8]; rows == 1: not used
  float* out = p.partials + (int64_t)blockIdx.x * 2 * p.C;
#pragma unroll
  for (int n = 0; n < NV; ++n)
#pragma unroll
    for (int k = 0; k < P; ++k)
#pragma unroll
      for (int h = 0; h < (V > 1 ? 2 : 1); ++h) {
        const float a = h ? dw[n][k].y : dw[n][k].x, b = h ? db[n][k].y : db[n][k].x;
        const int e = n * V + 2 * k + h;
        if (p.rows > 1) {
          if (row < p.rows) {
            norm_smem[(row * p.cols + col) * NORM_EACH + e] = a;
            norm_smem[((p.rows + row) * p.cols + col) * NORM_EACH + e] = b;
          }
        } else if (me.at[n] >= 0) {
          out[me.c0 + me.at[n] + 2 * k + h] = a;
          out[p.C + me.c0 + me.at[n] + 2 * k + h] = b;
        }
      }
  if (p.rows == 1) return;
  __syncthreads();
  if (row != 0 || !live) return;
#pragma unroll
  for (int n = 0; n < NV; ++n)
    if (me.at[n] >= 0)
#pragma unroll
      for (int e = 0; e < V; ++e)
#pragma unroll
        for (int m = 0; m < 2; ++m) {
          float v = 0.f;
          for (int q = 0; q < p.rows; ++q) v += norm_smem[((m * p.rows + q) * p.cols + col) * NORM_EACH + n * V + e];
          out[m * p.C + me.c0 + me.at[n] + e] = v;
        }
}

// rows of partial sums [rows][2][C] (of du n and du) -> weight's and bias's gradients, in a fixed order
template <typename T>
__global__ void __launch_bounds__(ROWS_THREADS) ttt_norm_reduce_kernel(const float* partials, int64_t rows, int C, T* gw, T* gb) {
  int64_t col;
  float v;
  if (!sum_of_rows(partials, rows, 2 * C, 2 * C, blockIdx.x, &col, &v)) return;
  if (col < C) {
    if (gw != nullptr) st_from_float<T>(gw, col, v);
  } else if (gb != nullptr) {
    st_from_float<T>(gb, col - C, v);
  }
}

// ---- whole sequences -----------------------------------------------------------------------------------------------
// Numbers seen so far: how many, their mean, the sum of squares of differences from it.  Joined as by Chan, Golub and LeVeque
// (1979), which does not cancel.
struct Moments {
  float n, mean, m2;
  __device__ __forceinline__ void join(float bn, float bmean, float bm2) {
    const float all = n + bn, d = bmean - mean, f = all > 0.f ? __fdividef(bn, all) : 0.f;
    mean = fmaf(d, f, mean);
    m2 += bm2 + d * d * n * f;
    n = all;
  }
  __device__ __forceinline__ void join_lanes(int lanes) {  // over a power of two of neighbouring lanes
    for (int o = 1; o < lanes; o <<= 1) {
      const float bn = __shfl_xor_sync(0xffffffffu, n, o), bm = __shfl_xor_sync(0xffffffffu, mean, o), b2 = __shfl_xor_sync(0xffffffffu, m2, o);
      // (both lanes join in the same order, so that both have the same)
      const bool second = (threadIdx.x & o) != 0;
      Moments lo = second ? Moments{bn, bm, b2} : *this;
      lo.join(second ? n : bn, second ? mean : bm, second ? m2 : b2);
      *this = lo;
    }
  }
};
// threads for each of a block's groups: a power of two, all groups at once
__device__ __forceinline__ int threads_per_group(int groups) {
  int w = 32;
  while (w > 1 && w * groups > NORM_THREADS) w >>= 1;
  return w;
}

// Where a block of the sequence kernels stands.  blockIdx.x: row of the batch and chunk of tokens; blockIdx.y: groups, or a part of
// a group's channels.
struct SeqPlace {
  int64_t b, t_lo, t_hi;
  int chunk, g0, groups, span;  // groups [g0, g0 + groups) or part `span` of group g0
  int row, c;                   // this thread's row and first channel, c < 0: none
  __device__ __forceinline__ SeqPlace(const NormParams& p, int V) {
    b = blockIdx.x / p.chunks;
    chunk = (int)(blockIdx.x - b * p.chunks);
    t_lo = (int64_t)chunk * p.chunk;
    t_hi = min(t_lo + p.chunk, p.T);
    row = threadIdx.x / p.cols;
    const int col = threadIdx.x - row * p.cols, vectors = p.c / V;
    if (p.spans == 1) {
      g0 = (int)blockIdx.y * p.per_block;
      groups = min(p.per_block, p.G - g0);
      span = 0;
      c = row < p.rows && col < groups * vectors ? g0 * p.c + col * V : -1;
    } else {
      g0 = (int)blockIdx.y / p.spans;
      groups = 1;
      span = (int)blockIdx.y - g0 * p.spans;
      const int v = span * p.cols + col;
      c = row < p.rows && v < vectors ? g0 * p.c + v * V : -1;
    }
  }
};

template <typename T, int V>
__global__ void __launch_bounds__(NORM_THREADS, NORM_SEQ_RESIDENT) ttt_norm_seq_stats_kernel(const NormParams p) {
  using Ch = Chan<T, V>;
  constexpr int P = Ch::P, AHEAD = 4;
  __shared__ float sm[3][NORM_THREADS];
  const SeqPlace at(p, V);
  Moments me{0.f, 0.f, 0.f};
  if (at.c >= 0) {
    const T* x = static_cast<const T*>(p.x) + at.b * p.xs[0] + at.c;
    for (int64_t t = at.t_lo + at.row; t < at.t_hi; t += (int64_t)AHEAD * p.rows) {
      Ch in[AHEAD];
      int have = 0;
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) {
        in[u].zero();
        if (t + (int64_t)u * p.rows < at.t_hi) in[u].load(x + (t + (int64_t)u * p.rows) * p.xs[1]), ++have;
      }
      F2 v[AHEAD][P], s = f2(0.f), q = f2(0.f);
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) {
        in[u].unpack(v[u]);
#pragma unroll
        for (int k = 0; k < P; ++k) s = f2add(s, v[u][k]);
      }
      const float n = (float)(have * V), mean = f2hsum(s) / n;
#pragma unroll
      for (int u = 0; u < AHEAD; ++u)
        if (u < have)
#pragma unroll
          for (int k = 0; k < P; ++k) {
            const F2 d = f2(v[u][k].x - mean, V > 1 ? v[u][k].y - mean : 0.f);
            q = f2fma(d, d, q);
          }
      me.join(n, mean, f2hsum(q));
    }
  }
  sm[0][threadIdx.x] = me.n, sm[1][threadIdx.x] = me.mean, sm[2][threadIdx.x] = me.m2;
  __syncthreads();
  const int per_group = p.spans == 1 ? p.c / V : p.cols, entries = per_group * p.rows;
  const int w = threads_per_group(at.groups), k = threadIdx.x / w, lane = threadIdx.x & (w - 1);
  Moments m{0.f, 0.f, 0.f};
  if (k < at.groups)
    for (int e = lane; e < entries; e += w) {
      const int r = e / per_group, i = r * p.cols + k * per_group + (e - r * per_group);
      m.join(sm[0][i], sm[1][i], sm[2][i]);
    }
  m.join_lanes(w);
  if (k < at.groups && lane == 0) {
    float* out = p.moments + (((at.b * p.G + at.g0 + k) * p.chunks + at.chunk) * p.spans + at.span) * 3;
    out[0] = m.n, out[1] = m.mean, out[2] = m.m2;
  }
}

template <typename T, int V, int MODE>
__global__ void __launch_bounds__(NORM_THREADS, NORM_SEQ_RESIDENT) ttt_norm_seq_apply_kernel(const NormParams p) {
  using Ch = Chan<T, V>;
  constexpr int P = Ch::P, AHEAD = 4;
  __shared__ float stat[NORM_THREADS][2];
  const SeqPlace at(p, V);
  const bool gated = norm_gated<MODE>(p);
  const int act = norm_act<MODE>(p);
  {
    const int w = threads_per_group(at.groups), k = threadIdx.x / w, lane = threadIdx.x & (w - 1);
    Moments all{0.f, 0.f, 0.f};
    if (k < at.groups) {
      const float* m = p.moments + (at.b * p.G + at.g0 + k) * p.chunks * p.spans * 3;
#pragma unroll 4
      for (int e = lane; e < p.chunks * p.spans; e += w) all.join(m[3 * e], m[3 * e + 1], m[3 * e + 2]);
    }
    all.join_lanes(w);
    if (k < at.groups && lane == 0) {
      stat[k][0] = all.mean;
      stat[k][1] = rsqrtf(all.m2 / all.n + p.eps);
      if (p.stats != nullptr && at.chunk == 0 && at.span == 0) {
        p.stats[(at.b * p.G + at.g0 + k) * 2] = stat[k][0];
        p.stats[(at.b * p.G + at.g0 + k) * 2 + 1] = stat[k][1];
      }
    }
  }
  __syncthreads();
  if (at.c < 0) return;
  const int k0 = at.c / p.c - at.g0;
  const float mean = stat[k0][0], r = stat[k0][1];
  F2 w[P], b[P];
#pragma unroll
  for (int k = 0; k < P; ++k) w[k] = f2(1.f), b[k] = f2(0.f);
  Ch raw;
  if (p.w != nullptr) raw.load(static_cast<const T*>(p.w) + at.c), raw.unpack(w);
  if (p.bias != nullptr) raw.load(static_cast<const T*>(p.bias) + at.c), raw.unpack(b);
  const T* x = static_cast<const T*>(p.x) + at.b * p.xs[0] + at.c;
  const T* gate = static_cast<const T*>(p.gate) + at.b * p.gates[0] + at.c;
  T* y = static_cast<T*>(p.y) + at.b * p.T * p.C + at.c;
  for (int64_t t = at.t_lo + at.row; t < at.t_hi; t += (int64_t)AHEAD * p.rows) {
    Ch in[AHEAD], gt[AHEAD];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      gt[u].zero();
      if (t + (int64_t)u * p.rows < at.t_hi) {
        in[u].load(x + (t + (int64_t)u * p.rows) * p.xs[1]);
        if (gated) gt[u].load(gate + (t + (int64_t)u * p.rows) * p.gates[1]);
      }
    }
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      if (t + (int64_t)u * p.rows >= at.t_hi) break;
      F2 v[P], e[P];
      in[u].unpack(v);
      gt[u].unpack(e);
#pragma unroll
      for (int k = 0; k < P; ++k) {
        v[k] = f2fma(f2mul(f2add(v[k], f2(-mean)), f2(r)), w[k], b[k]);
        if (gated) v[k] = f2mul(v[k], f2(act_of(e[k].x, act), act_of(e[k].y, act)));
        else v[k] = f2(act_of(v[k].x, act), act_of(v[k].y, act));
      }
      Ch out;
      out.pack(v);
      out.store(y + (t + (int64_t)u * p.rows) * p.C);
    }
  }
}

// du and n of a thread's channels of one token, and the gate's gradient
template <int P>
__device__ __forceinline__ void norm_du(bool gated, int act, F2 (&n)[P], F2 (&du)[P], const F2 (&e)[P], F2 (&dg)[P], float mean, float r,
                                        const F2 (&w)[P], const F2 (&b)[P]) {
#pragma unroll
  for (int k = 0; k < P; ++k) {
    n[k] = f2mul(f2add(n[k], f2(-mean)), f2(r));
    const F2 v = f2fma(n[k], w[k], b[k]);
    F2 a, slope;
    if (gated) {
      a.x = act_and_slope(e[k].x, act, slope.x);
      a.y = act_and_slope(e[k].y, act, slope.y);
      dg[k] = f2mul(f2mul(du[k], v), slope);
      du[k] = f2mul(du[k], a);
    } else {
      act_and_slope(v.x, act, slope.x);
      act_and_slope(v.y, act, slope.y);
      du[k] = f2mul(du[k], slope);
    }
  }
}

// APPLY false: every channel's sums of du and du n over the chunk.  true: the gradients of x and the gate.
template <typename T, int V, bool APPLY, int MODE>
__global__ void __launch_bounds__(NORM_THREADS, NORM_SEQ_RESIDENT) ttt_norm_seq_bwd_kernel(const NormParams p) {
  using Ch = Chan<T, V>;
  constexpr int P = Ch::P, AHEAD = 2;
  __shared__ float mean_of[NORM_THREADS][2];
  extern __shared__ float norm_smem[];  // APPLY false: [2][rows][cols][V]
  const SeqPlace at(p, V);
  const bool gated = norm_gated<MODE>(p);
  const int act = norm_act<MODE>(p);
  if constexpr (APPLY) {  // the groups' means of p and p n, from the channels' sums
    const float inv = 1.f / ((float)p.c * (float)p.T);
    const int w = threads_per_group(at.groups), k = threadIdx.x / w, lane = threadIdx.x & (w - 1);
    float m1 = 0.f, m2 = 0.f;
    if (k < at.groups) {
      const int c0 = (at.g0 + k) * p.c;
      const float* s = p.sums + at.b * 2 * p.C + c0;
#pragma unroll 4
      for (int c = lane; c < p.c; c += w) {
        const float wt = p.w != nullptr ? ld_as_float<T>(p.w, c0 + c) : 1.f;
        m2 = fmaf(wt, s[c], m2);
        m1 = fmaf(wt, s[p.C + c], m1);
      }
    }
    for (int o = 1; o < w; o <<= 1) {
      m1 += __shfl_xor_sync(0xffffffffu, m1, o);
      m2 += __shfl_xor_sync(0xffffffffu, m2, o);
    }
    if (k < at.groups && lane == 0) mean_of[k][0] = m1 * inv, mean_of[k][1] = m2 * inv;
    __syncthreads();
  }
  F2 s1[P], s2[P];
#pragma unroll
  for (int k = 0; k < P; ++k) s1[k] = s2[k] = f2(0.f);
  if (at.c >= 0) {
    const int g = at.c / p.c;
    const float mean = p.stats[(at.b * p.G + g) * 2], r = p.stats[(at.b * p.G + g) * 2 + 1];
    const float m1 = APPLY ? mean_of[g - at.g0][0] : 0.f, m2 = APPLY ? mean_of[g - at.g0][1] : 0.f;
    F2 w[P], b[P];
#pragma unroll
    for (int k = 0; k < P; ++k) w[k] = f2(1.f), b[k] = f2(0.f);
    Ch raw;
    if (p.w != nullptr) raw.load(static_cast<const T*>(p.w) + at.c), raw.unpack(w);
    if (p.bias != nullptr) raw.load(static_cast<const T*>(p.bias) + at.c), raw.unpack(b);
    const T* x = static_cast<const T*>(p.x) + at.b * p.xs[0] + at.c;
    const T* gate = static_cast<const T*>(p.gate) + at.b * p.gates[0] + at.c;
    const T* gy = static_cast<const T*>(p.gy) + at.b * p.gys[0] + at.c;
    T* gx = static_cast<T*>(p.gx) + at.b * p.T * p.C + at.c;
    T* ggate = static_cast<T*>(p.ggate) + at.b * p.T * p.C + at.c;
    for (int64_t t = at.t_lo + at.row; t < at.t_hi; t += (int64_t)AHEAD * p.rows) {
      Ch in[AHEAD], gt[AHEAD], gr[AHEAD];
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) {
        const int64_t tu = t + (int64_t)u * p.rows;
        gt[u].zero();
        if (tu < at.t_hi) {
          in[u].load(x + tu * p.xs[1]);
          gr[u].load(gy + tu * p.gys[1]);
          if (gated) gt[u].load(gate + tu * p.gates[1]);
        }
      }
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) {
        const int64_t tu = t + (int64_t)u * p.rows;
        if (tu >= at.t_hi) break;
        F2 n[P], du[P], e[P], dg[P];
        in[u].unpack(n);
        gr[u].unpack(du);
        gt[u].unpack(e);
        norm_du<P>(gated, act, n, du, e, dg, mean, r, w, b);
        if constexpr (APPLY) {
          Ch out;
#pragma unroll
          for (int k = 0; k < P; ++k) du[k] = f2mul(f2fma(n[k], f2(-m2), f2fma(du[k], w[k], f2(-m1))), f2(r));
          out.pack(du);
          out.store(gx + tu * p.C);
          if (gated) {
            out.pack(dg);
            out.store(ggate + tu * p.C);
          }
        } else {
#pragma unroll
          for (int k = 0; k < P; ++k) {
            s1[k] = f2add(s1[k], du[k]);
            s2[k] = f2fma(du[k], n[k], s2[k]);
          }
        }
      }
    }
  }
  if constexpr (!APPLY) {
    const int width = p.cols * V, col = threadIdx.x - at.row * p.cols;
    if (at.row < p.rows)
#pragma unroll
      for (int k = 0; k < P; ++k)
#pragma unroll
        for (int h = 0; h < (V > 1 ? 2 : 1); ++h) {
          norm_smem[at.row * width + col * V + 2 * k + h] = h ? s1[k].y : s1[k].x;
          norm_smem[(p.rows + at.row) * width + col * V + 2 * k + h] = h ? s2[k].y : s2[k].x;
        }
    __syncthreads();
    // [2][C] per chunk: du n first, as the weight's gradient stands before the bias's
    float* out = p.partials + (int64_t)blockIdx.x * 2 * p.C;
    const int first = p.spans == 1 ? at.g0 * p.c : at.g0 * p.c + at.span * width;
    const int have = p.spans == 1 ? at.groups * p.c : min(width, p.c - at.span * width);
    for (int e = threadIdx.x; e < 2 * have; e += NORM_THREADS) {
      const int m = e / have, c = e - m * have;
      float v = 0.f;
      for (int q = 0; q < p.rows; ++q) v += norm_smem[(m * p.rows + q) * width + c];
      out[(1 - m) * p.C + first + c] = v;
    }
  }
}

// the chunks' sums [B][chunks][2][C] -> [B][2][C]
__global__ void __launch_bounds__(ROWS_THREADS) ttt_norm_seq_sums_kernel(const float* partials, float* sums, int chunks, int C, int column_blocks) {
  const int64_t b = blockIdx.x / column_blocks;
  int64_t col;
  float v;
  if (!sum_of_rows(partials + b * chunks * 2 * C, chunks, 2 * C, 2 * C, blockIdx.x - b * column_blocks, &col, &v)) return;
  sums[b * 2 * C + col] = v;
}

// ---- launches --------------------------------------------------------------------------------------------------------
struct NormCut {
  int lanes, cols, rows, y, threads;      // a token's groups
  int per_block, spans, chunks;           // sequences
  int64_t chunk, x;
};
static NormCut norm_token_cut(int64_t tokens, int G, int c, bool bwd) {
  NormCut k{};
  k.lanes = 1;
  while (k.lanes * NORM_EACH < c) k.lanes *= 2;
  const int64_t total = (int64_t)G * k.lanes;
  const int64_t blocks = (total + NORM_THREADS - 1) / NORM_THREADS;
  const int64_t share = (total + blocks - 1) / blocks;
  k.cols = (int)((share + k.lanes - 1) / k.lanes) * k.lanes;
  k.rows = k.cols < NORM_THREADS ? NORM_THREADS / k.cols : 1;
  k.threads = (k.cols * k.rows + 31) / 32 * 32;
  k.y = (int)((total + k.cols - 1) / k.cols);
  const bool wide = k.lanes > 32;
  const int regs = !bwd ? 65536 / (NORM_THREADS * NORM_FWD_RESIDENT) : wide ? 65536 / NORM_WIDE : 65536 / (NORM_THREADS * NORM_BWD_RESIDENT);
  const int64_t resident = 65536 / (regs * k.threads);
  const int64_t need = (tokens + k.rows - 1) / k.rows, wanted = 148 * resident / k.y, most = wanted > 1 ? wanted : 1;
  k.x = need < most ? need : most;
  return k;
}
static NormCut norm_seq_cut(int64_t B, int64_t T, int G, int c, int V) {
  NormCut k{};
  const int vectors = c / V;
  if (vectors <= NORM_THREADS) {
    const int fit = NORM_THREADS / vectors, blocks = (G + fit - 1) / fit;
    k.spans = 1;
    k.per_block = (G + blocks - 1) / blocks;
    k.cols = k.per_block * vectors;
    k.rows = NORM_THREADS / k.cols;
    k.y = blocks;
  } else {
    k.spans = (vectors + NORM_THREADS - 1) / NORM_THREADS;
    k.per_block = 1;
    k.cols = NORM_THREADS;
    k.rows = 1;
    k.y = G * k.spans;
  }
  int64_t chunks = 148 * NORM_SEQ_RESIDENT / (B * k.y);
  if (chunks < 1) chunks = 1;
  const int64_t most = (T + 4 * k.rows - 1) / (4 * k.rows);  // (four tokens per thread at least)
  if (chunks > most) chunks = most;
  k.chunk = (T + chunks - 1) / chunks;
  k.chunks = (int)((T + k.chunk - 1) / k.chunk);
  k.x = B * k.chunks;
  return k;
}
static int norm_widths(int es, int c, int (&v)[3]) {  // the vector widths that a group of c channels allows; which runs depends on addresses
  int n = 0;
  for (int V : {16 / es, 2, 1})
    if (c % V == 0) v[n++] = V;
  return n;
}
size_t norm_forward_floats(int64_t B, int64_t T, int C, int G, bool sequence, int es) {
  if (!sequence) return 0;
  size_t most = 0;
  int v[3];
  for (int i = norm_widths(es, C / G, v); i-- > 0;) {
    const NormCut k = norm_seq_cut(B, T, G, C / G, v[i]);
    const size_t n = (size_t)B * G * k.chunks * k.spans * 3;
    if (n > most) most = n;
  }
  return most;
}
size_t norm_backward_floats(int64_t B, int64_t T, int C, int G, bool sequence, int es) {
  if (!sequence) return (size_t)norm_token_cut(B * T, G, C / G, true).x * 2 * C;
  size_t most = 0;
  int v[3];
  for (int i = norm_widths(es, C / G, v); i-- > 0;) {
    const NormCut k = norm_seq_cut(B, T, G, C / G, v[i]);
    const size_t n = (size_t)B * (k.chunks + 1) * 2 * C;
    if (n > most) most = n;
  }
  return most;
}

template <typename T>
static cudaError_t reduce(const NormParams& p, const float* partials, int64_t rows, cudaStream_t st) {
  ttt_norm_reduce_kernel<T><<<(2 * p.C + 31) / 32, ROWS_THREADS, 0, st>>>(partials, rows, p.C, static_cast<T*>(p.gw), static_cast<T*>(p.gb));
  return cudaGetLastError();
}
// (the wide vectors' kernels know a SiLU when they are built; the others, and what is rare, ask at run time)
template <typename T, int V, bool WIDE>
static cudaError_t token_mode(const NormParams& p, const NormCut& k, bool bwd, size_t smem, cudaStream_t st) {
  void (*kernel)(NormParams) = bwd ? ttt_norm_token_bwd_kernel<T, V, WIDE, NORM_GENERAL> : ttt_norm_token_kernel<T, V, WIDE, NORM_GENERAL>;
  if constexpr (V * sizeof(T) == 16 && !WIDE) {
    if (p.act == ACT_SILU && p.gate != nullptr) kernel = bwd ? ttt_norm_token_bwd_kernel<T, V, WIDE, NORM_GATED_SILU> : ttt_norm_token_kernel<T, V, WIDE, NORM_GATED_SILU>;
    else if (p.act == ACT_SILU) kernel = bwd ? ttt_norm_token_bwd_kernel<T, V, WIDE, NORM_SILU> : ttt_norm_token_kernel<T, V, WIDE, NORM_SILU>;
  }
  kernel<<<dim3((unsigned)k.x, k.y), k.threads, smem, st>>>(p);
  return cudaGetLastError();
}
template <typename T, int V>
static cudaError_t launch_token(NormParams p, bool bwd, cudaStream_t st) {
  const NormCut k = norm_token_cut(p.tokens, p.G, p.c, bwd);
  p.lanes = k.lanes, p.cols = k.cols, p.rows = k.rows;
  const size_t smem = bwd && k.rows > 1 ? sizeof(float) * 2 * k.rows * k.cols * NORM_EACH : 0;
  const cudaError_t e = k.lanes > 32 ? token_mode<T, V, true>(p, k, bwd, smem, st) : token_mode<T, V, false>(p, k, bwd, smem, st);
  return e != cudaSuccess || !bwd || p.partials == nullptr ? e : reduce<T>(p, p.partials, k.x, st);
}
template <typename T, int V, int MODE>
static cudaError_t launch_seq(NormParams p, bool bwd, cudaStream_t st) {
  const NormCut k = norm_seq_cut(p.B, p.T, p.G, p.c, V);
  p.cols = k.cols, p.rows = k.rows, p.per_block = k.per_block, p.spans = k.spans, p.chunks = k.chunks, p.chunk = k.chunk;
  const dim3 grid((unsigned)k.x, k.y);
  cudaError_t e;
  if (!bwd) {
    ttt_norm_seq_stats_kernel<T, V><<<grid, NORM_THREADS, 0, st>>>(p);
    if ((e = cudaGetLastError()) != cudaSuccess) return e;
    ttt_norm_seq_apply_kernel<T, V, MODE><<<grid, NORM_THREADS, 0, st>>>(p);
    return cudaGetLastError();
  }
  p.sums = p.partials + (size_t)k.x * 2 * p.C;
  ttt_norm_seq_bwd_kernel<T, V, false, MODE><<<grid, NORM_THREADS, sizeof(float) * 2 * k.rows * k.cols * V, st>>>(p);
  if ((e = cudaGetLastError()) != cudaSuccess) return e;
  const int column_blocks = (2 * p.C + 31) / 32;
  ttt_norm_seq_sums_kernel<<<(unsigned)(p.B * column_blocks), ROWS_THREADS, 0, st>>>(p.partials, p.sums, k.chunks, p.C, column_blocks);
  if ((e = cudaGetLastError()) != cudaSuccess) return e;
  ttt_norm_seq_bwd_kernel<T, V, true, MODE><<<grid, NORM_THREADS, 0, st>>>(p);
  if ((e = cudaGetLastError()) != cudaSuccess) return e;
  return p.gw == nullptr && p.gb == nullptr ? cudaSuccess : reduce<T>(p, p.sums, p.B, st);
}
template <typename T, int V>
static cudaError_t launch_v(const NormParams& p, bool sequence, bool bwd, cudaStream_t st) {
  if (!sequence) return launch_token<T, V>(p, bwd, st);
  if constexpr (V * sizeof(T) == 16) {
    if (p.act == ACT_SILU) return p.gate != nullptr ? launch_seq<T, V, NORM_GATED_SILU>(p, bwd, st) : launch_seq<T, V, NORM_SILU>(p, bwd, st);
  }
  return launch_seq<T, V, NORM_GENERAL>(p, bwd, st);
}
// V: the widest vector that the group's channels and all addresses allow (16 bytes, 2 channels or 1)
cudaError_t launch_norm(int dtype, const NormParams& p, int V, bool sequence, bool bwd, cudaStream_t st) {
  if (dtype == 1)
    return V == 8 ? launch_v<__nv_bfloat16, 8>(p, sequence, bwd, st) : V == 2 ? launch_v<__nv_bfloat16, 2>(p, sequence, bwd, st)
                                                                              : launch_v<__nv_bfloat16, 1>(p, sequence, bwd, st);
  return V == 4 ? launch_v<float, 4>(p, sequence, bwd, st) : V == 2 ? launch_v<float, 2>(p, sequence, bwd, st) : launch_v<float, 1>(p, sequence, bwd, st);
}

}  // namespace ttt
