// Causal depthwise convolution of 2 to 4 taps over [B,T,C], channels last, with bias and SiLU, forward and backward.
//
//   v_t = bias + sum_j w_j x_{t-K+1+j},  y_t = v_t or SiLU(v_t)
// Inputs before the row are the carried state's (or zeros); a start at token t hides everything before t from t on.  The new state
// is the last K - 1 inputs, as they are visible behind the last token.  With g_t = dy_t act'(v_t):
//   dx_s = sum_j w_j g_{s+K-1-j} over the tokens that saw s (+ the new state's gradient),  dw_j = sum_t g_t x_{t-K+1+j},  db = sum_t g_t
//
// Memory-bound.  A thread holds V neighbouring channels (16 bytes; backward 8 bytes: its sums for the weights are registers) and
// walks a strip of tokens with the last K - 1 inputs in registers, CONV_AHEAD tokens on their way at a time; the tokens before a
// strip (and behind it, for dx) are read again, from L2.  A start empties the registers of the inputs, and the sums of dx know the
// last start's place.
#include "ttt_kernels.h"
#include "ttt_vec.cuh"

namespace ttt {

constexpr int CONV_THREADS = 256;
constexpr int CONV_AHEAD = 8;      // forward: tokens on their way
constexpr int CONV_BWD_AHEAD = 4;  // backward
constexpr int64_t NO_START = -(1ll << 40);

// V channels of row t of a sequence; rows before the first are the state's, rows from T on zeros
template <typename T, int V, int K>
__device__ __forceinline__ void conv_row(Chan<T, V>& r, const ConvParams& p, const T* x, const T* state, int64_t t) {
  if (t >= 0 && t < p.T) r.load(x + t * p.xs[1]);
  else if (t < 0 && state != nullptr) r.load(state + (t + K - 1) * p.C);
  else r.zero();
}

template <typename T, int V, int K>
struct ConvWeights {
  static constexpr int P = Chan<T, V>::P;
  F2 w[K][P];
  F2 bias[P];
  __device__ __forceinline__ void load(const ConvParams& p, int c) {
    float e[K * V];
    const T* at = static_cast<const T*>(p.w) + (int64_t)c * K;
#pragma unroll
    for (int i = 0; i < K * V; ++i) e[i] = ld_as_float<T>(at, i);
#pragma unroll
    for (int k = 0; k < P; ++k) {
#pragma unroll
      for (int j = 0; j < K; ++j) w[j][k] = f2(e[2 * k * K + j], 2 * k + 1 < V ? e[(2 * k + 1 < V ? 2 * k + 1 : 0) * K + j] : 0.f);
      bias[k] = f2(0.f);
      if (p.bias != nullptr) bias[k] = f2(ld_as_float<T>(p.bias, c + 2 * k), 2 * k + 1 < V ? ld_as_float<T>(p.bias, c + 2 * k + 1) : 0.f);
    }
  }
};

template <typename T, int V, int K>
__global__ void __launch_bounds__(CONV_THREADS) ttt_conv_kernel(const ConvParams p) {
  using Ch = Chan<T, V>;
  constexpr int P = Ch::P;
  const int lane = threadIdx.x & ((1 << p.lanes_log) - 1);
  const int64_t strip = (int64_t)blockIdx.x * (CONV_THREADS >> p.lanes_log) + (threadIdx.x >> p.lanes_log);
  const int c = ((int)blockIdx.y * (1 << p.lanes_log) + lane) * V;
  if (c >= p.C || strip >= p.B * p.strips) return;
  const int64_t b = strip / p.strips, t0 = (strip - b * p.strips) * p.strip, t1 = min(t0 + p.strip, p.T);
  ConvWeights<T, V, K> w;
  w.load(p, c);
  const T* x = static_cast<const T*>(p.x) + b * p.xs[0] + c;
  const T* state = p.state != nullptr ? static_cast<const T*>(p.state) + b * (K - 1) * p.C + c : nullptr;
  const uint8_t* starts = p.starts != nullptr ? p.starts + b * p.T : nullptr;
  T* y = static_cast<T*>(p.y) + b * p.T * p.C + c;
  F2 h[K - 1][P];  // h[i]: token t - (K - 1) + i
  {
    Ch r[K - 1];
#pragma unroll
    for (int i = 0; i < K - 1; ++i) conv_row<T, V, K>(r[i], p, x, state, t0 - (K - 1) + i);
#pragma unroll
    for (int i = 0; i < K - 1; ++i) r[i].unpack(h[i]);
    if (starts != nullptr) {  // a start hides what lies before it
#pragma unroll
      for (int i = 1; i < K - 1; ++i) {
        const int64_t t = t0 - (K - 1) + i;
        if (t >= 0 && starts[t]) {
#pragma unroll
          for (int e = 0; e < i; ++e)
#pragma unroll
            for (int k = 0; k < P; ++k) h[e][k] = f2(0.f);
        }
      }
    }
  }
  for (int64_t at = t0; at < t1; at += CONV_AHEAD) {
    Ch in[CONV_AHEAD];
    uint8_t first[CONV_AHEAD];
#pragma unroll
    for (int u = 0; u < CONV_AHEAD; ++u) {
      first[u] = 0;
      if (at + u < t1) {
        in[u].load(x + (at + u) * p.xs[1]);
        if (starts != nullptr) first[u] = starts[at + u];
      }
    }
#pragma unroll
    for (int u = 0; u < CONV_AHEAD; ++u) {
      if (at + u >= t1) break;
      if (first[u]) {
#pragma unroll
        for (int i = 0; i < K - 1; ++i)
#pragma unroll
          for (int k = 0; k < P; ++k) h[i][k] = f2(0.f);
      }
      F2 now[P], v[P];
      in[u].unpack(now);
#pragma unroll
      for (int k = 0; k < P; ++k) {
        v[k] = f2fma(now[k], w.w[K - 1][k], w.bias[k]);
#pragma unroll
        for (int i = 0; i < K - 1; ++i) v[k] = f2fma(h[i][k], w.w[i][k], v[k]);
#pragma unroll
        for (int i = 0; i < K - 2; ++i) h[i][k] = h[i + 1][k];
        h[K - 2][k] = now[k];
        if (p.act == ACT_SILU) v[k] = f2(act_of(v[k].x, ACT_SILU), act_of(v[k].y, ACT_SILU));
      }
      Ch out;
      out.pack(v);
      out.store(y + (at + u) * p.C);
    }
  }
  // The thread of the first tokens, the only one that has read the given state, writes the new one: they may be the same tensor.
  // (Behind a short row a part of the given state is still visible: read it all before writing.)
  if (t0 == 0) {
    Ch r[K - 1];
#pragma unroll
    for (int i = 0; i < K - 1; ++i) conv_row<T, V, K>(r[i], p, x, state, p.T - (K - 1) + i);
    if (starts != nullptr) {
#pragma unroll
      for (int i = 0; i < K - 1; ++i) {
        const int64_t t = p.T - (K - 1) + i;
        if (t >= 0 && starts[t]) {
#pragma unroll
          for (int e = 0; e < i; ++e) r[e].zero();
        }
      }
    }
    T* out = static_cast<T*>(p.state_out) + b * (K - 1) * p.C + c;
#pragma unroll
    for (int i = 0; i < K - 1; ++i) r[i].store(out + (int64_t)i * p.C);
  }
}

// Blocks walk strips with a stride and leave one row of sums for the weights and the bias each: [K + 1][C].
template <typename T, int V, int K>
__global__ void __launch_bounds__(CONV_THREADS) ttt_conv_bwd_kernel(const ConvParams p) {
  using Ch = Chan<T, V>;
  constexpr int P = Ch::P;
  const int lanes = 1 << p.lanes_log, rows = CONV_THREADS >> p.lanes_log;
  const int lane = threadIdx.x & (lanes - 1), row = threadIdx.x >> p.lanes_log;
  const int c = ((int)blockIdx.y * lanes + lane) * V;
  const bool live = c < p.C;
  F2 dw[K + 1][P];
#pragma unroll
  for (int j = 0; j <= K; ++j)
#pragma unroll
    for (int k = 0; k < P; ++k) dw[j][k] = f2(0.f);
  if (live) {
    ConvWeights<T, V, K> w;
    w.load(p, c);
    for (int64_t strip = (int64_t)blockIdx.x * rows + row; strip < p.B * p.strips; strip += (int64_t)gridDim.x * rows) {
      const int64_t b = strip / p.strips, t0 = (strip - b * p.strips) * p.strip, t1 = min(t0 + p.strip, p.T);
      const int64_t s_lo = t0 == 0 ? -(K - 1) : t0;  // the first strip's gradients begin with the state's
      const T* x = static_cast<const T*>(p.x) + b * p.xs[0] + c;
      const T* g = static_cast<const T*>(p.gy) + b * p.gs[0] + c;
      const T* state = p.state != nullptr ? static_cast<const T*>(p.state) + b * (K - 1) * p.C + c : nullptr;
      const T* gstate_out = p.gstate_out != nullptr ? static_cast<const T*>(p.gstate_out) + b * (K - 1) * p.C + c : nullptr;
      const uint8_t* starts = p.starts != nullptr ? p.starts + b * p.T : nullptr;
      T* gx = static_cast<T*>(p.gx) + b * p.T * p.C + c;
      T* gstate = p.gstate != nullptr ? static_cast<T*>(p.gstate) + b * (K - 1) * p.C + c : nullptr;
      F2 h[K - 1][P], acc[K - 1][P];  // acc[i]: gradient of token t - (K - 1) + i so far
      int64_t last = NO_START;
      {
        Ch r[K - 1];
#pragma unroll
        for (int i = 0; i < K - 1; ++i) conv_row<T, V, K>(r[i], p, x, state, t0 - (K - 1) + i);
#pragma unroll
        for (int i = 0; i < K - 1; ++i) {
          r[i].unpack(h[i]);
#pragma unroll
          for (int k = 0; k < P; ++k) acc[i][k] = f2(0.f);
        }
        if (starts != nullptr) {
#pragma unroll
          for (int i = 1; i < K - 1; ++i) {
            const int64_t t = t0 - (K - 1) + i;
            if (t >= 0 && starts[t]) {
              last = t;
#pragma unroll
              for (int e = 0; e < i; ++e)
#pragma unroll
                for (int k = 0; k < P; ++k) h[e][k] = f2(0.f);
            }
          }
        }
      }
      // token t completes the gradient of token t - (K - 1)
      for (int64_t at = t0; at < t1 + K - 1; at += CONV_BWD_AHEAD) {
        Ch in[CONV_BWD_AHEAD], grad[CONV_BWD_AHEAD];
        uint8_t first[CONV_BWD_AHEAD];
#pragma unroll
        for (int u = 0; u < CONV_BWD_AHEAD; ++u) {
          const int64_t t = at + u;
          first[u] = 0;
          in[u].zero();
          grad[u].zero();
          if (t < t1 + K - 1 && t < p.T) {
            in[u].load(x + t * p.xs[1]);
            grad[u].load(g + t * p.gs[1]);
            if (starts != nullptr) first[u] = starts[t];
          }
        }
#pragma unroll
        for (int u = 0; u < CONV_BWD_AHEAD; ++u) {
          const int64_t t = at + u;
          if (t >= t1 + K - 1) break;
          if (first[u]) {
            last = t;
#pragma unroll
            for (int i = 0; i < K - 1; ++i)
#pragma unroll
              for (int k = 0; k < P; ++k) h[i][k] = f2(0.f);
          }
          F2 now[P], gv[P], whole[P];
          in[u].unpack(now);
          grad[u].unpack(gv);
          const bool counts = t < t1;  // (the tokens behind the strip are another's for the weights)
#pragma unroll
          for (int k = 0; k < P; ++k) {
            if (p.act == ACT_SILU) {
              F2 v = f2fma(now[k], w.w[K - 1][k], w.bias[k]), slope;
#pragma unroll
              for (int i = 0; i < K - 1; ++i) v = f2fma(h[i][k], w.w[i][k], v);
              act_and_slope(v.x, ACT_SILU, slope.x);
              act_and_slope(v.y, ACT_SILU, slope.y);
              gv[k] = t < p.T ? f2mul(gv[k], slope) : f2(0.f);
            }
            if (counts) {
#pragma unroll
              for (int i = 0; i < K - 1; ++i) dw[i][k] = f2fma(gv[k], h[i][k], dw[i][k]);
              dw[K - 1][k] = f2fma(gv[k], now[k], dw[K - 1][k]);
              dw[K][k] = f2add(dw[K][k], gv[k]);
            }
#pragma unroll
            for (int i = 0; i < K - 1; ++i)
              if (t - (K - 1) + i >= last) acc[i][k] = f2fma(gv[k], w.w[i][k], acc[i][k]);
            whole[k] = acc[0][k];
#pragma unroll
            for (int i = 0; i < K - 2; ++i) acc[i][k] = acc[i + 1][k], h[i][k] = h[i + 1][k];
            acc[K - 2][k] = f2mul(gv[k], w.w[K - 1][k]);
            h[K - 2][k] = now[k];
          }
          const int64_t s = t - (K - 1);
          if (s < s_lo) continue;
          if (gstate_out != nullptr && s >= p.T - (K - 1) && s >= last) {
            Ch r;
            F2 e[P];
            r.load(gstate_out + (s - (p.T - (K - 1))) * p.C);
            r.unpack(e);
#pragma unroll
            for (int k = 0; k < P; ++k) whole[k] = f2add(whole[k], e[k]);
          }
          Ch out;
          out.pack(whole);
          if (s >= 0) out.store(gx + s * p.C);
          else if (gstate != nullptr) out.store(gstate + (s + K - 1) * p.C);
        }
      }
    }
  }
  if (p.partials == nullptr) return;
  extern __shared__ float conv_smem[];  // [rows][K + 1][lanes * V]: the block's sum in a fixed order
  const int width = lanes * V;
#pragma unroll
  for (int j = 0; j <= K; ++j)
#pragma unroll
    for (int k = 0; k < P; ++k) {
      float* at = conv_smem + ((row * (K + 1) + j) * width + lane * V + 2 * k);
      at[0] = dw[j][k].x;
      if (2 * k + 1 < V) at[1] = dw[j][k].y;
    }
  __syncthreads();
  for (int e = threadIdx.x; e < (K + 1) * width; e += CONV_THREADS) {
    float v = 0.f;
    for (int r = 0; r < rows; ++r) v += conv_smem[r * (K + 1) * width + e];
    const int j = e / width, ch = (int)blockIdx.y * width + (e - j * width);
    if (ch < p.C) p.partials[((int64_t)blockIdx.x * (K + 1) + j) * p.C + ch] = v;
  }
}

// rows of partial sums [rows][n] -> out: a block per 32 columns, 8 shares of the rows, in a fixed order
template <typename T>
__global__ void __launch_bounds__(256) ttt_conv_reduce_kernel(const float* partials, int rows, int C, int K, T* gw, T* gbias) {
  __shared__ float part[8][33];
  const int col = (int)blockIdx.x * 32 + (threadIdx.x & 31), share = threadIdx.x >> 5, n = (K + 1) * C;
  float v = 0.f;
  if (col < n)
    for (int r = share; r < rows; r += 8) v += partials[(int64_t)r * n + col];
  part[share][threadIdx.x & 31] = v;
  __syncthreads();
  if (share != 0 || col >= n) return;
#pragma unroll
  for (int k = 1; k < 8; ++k) v += part[k][threadIdx.x & 31];
  const int j = col / C, c = col - j * C;
  if (j < K) {
    if (gw != nullptr) st_from_float<T>(gw, (size_t)c * K + j, v);
  } else if (gbias != nullptr) {
    st_from_float<T>(gbias, c, v);
  }
}

// Strips of 16 tokens (forward) or 32 (backward) where the threads then fill the card, shorter ones where not: a strip's neighbours
// cost K - 1 rows more.
struct ConvCut {
  int lanes_log, strip, y;
  int64_t strips, x;
};
static ConvCut conv_cut(int64_t B, int64_t T, int C, int V, int strip) {
  ConvCut k{};
  const int vectors = (C + V - 1) / V;
  while (k.lanes_log < 5 && (1 << k.lanes_log) < vectors) ++k.lanes_log;
  k.y = (vectors + (1 << k.lanes_log) - 1) >> k.lanes_log;
  const int64_t wide = (int64_t)k.y << k.lanes_log;
  while (strip > 4 && B * ((T + strip - 1) / strip) * wide < 148 * 1024) strip /= 2;
  k.strip = strip;
  k.strips = (T + strip - 1) / strip;
  const int per_block = CONV_THREADS >> k.lanes_log;
  k.x = (B * k.strips + per_block - 1) / per_block;
  return k;
}
static int64_t conv_bwd_blocks(const ConvCut& k) {
  const int64_t most = 148 * 4 / k.y > 1 ? 148 * 4 / k.y : 1;
  return k.x < most ? k.x : most;
}
template <typename T>
static constexpr int conv_width(bool vec, bool bwd) {
  return !vec ? 1 : bwd ? 4 : 16 / (int)sizeof(T);
}
size_t conv_partial_floats(int64_t B, int64_t T, int C, int K) {  // for either width
  size_t most = 0;
  for (int V : {1, 4}) {
    const size_t n = (size_t)conv_bwd_blocks(conv_cut(B, T, C, V, 32)) * (K + 1) * C;
    if (n > most) most = n;
  }
  return most;
}

template <typename T, int V, int K>
static cudaError_t launch_fwd(ConvParams p, cudaStream_t st) {
  const ConvCut k = conv_cut(p.B, p.T, p.C, V, 16);
  p.lanes_log = k.lanes_log, p.strip = k.strip, p.strips = k.strips;
  ttt_conv_kernel<T, V, K><<<dim3((unsigned)k.x, k.y), CONV_THREADS, 0, st>>>(p);
  return cudaGetLastError();
}
template <typename T, int V, int K>
static cudaError_t launch_bwd(ConvParams p, cudaStream_t st) {
  const ConvCut k = conv_cut(p.B, p.T, p.C, V, 32);
  p.lanes_log = k.lanes_log, p.strip = k.strip, p.strips = k.strips;
  const int64_t blocks = conv_bwd_blocks(k);
  const size_t smem = sizeof(float) * CONV_THREADS * V * (K + 1);
  ttt_conv_bwd_kernel<T, V, K><<<dim3((unsigned)blocks, k.y), CONV_THREADS, smem, st>>>(p);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess || p.partials == nullptr) return e;
  ttt_conv_reduce_kernel<T><<<((K + 1) * p.C + 31) / 32, 256, 0, st>>>(p.partials, (int)blocks, p.C, K, static_cast<T*>(p.gw),
                                                                      static_cast<T*>(p.gbias));
  return cudaGetLastError();
}
template <typename T, int V>
static cudaError_t launch_k(const ConvParams& p, int taps, cudaStream_t st) {
  switch (taps) {
    case 2: return launch_fwd<T, V, 2>(p, st);
    case 3: return launch_fwd<T, V, 3>(p, st);
    default: return launch_fwd<T, V, 4>(p, st);
  }
}
template <typename T, int V>
static cudaError_t launch_bwd_k(const ConvParams& p, int taps, cudaStream_t st) {
  switch (taps) {
    case 2: return launch_bwd<T, V, 2>(p, st);
    case 3: return launch_bwd<T, V, 3>(p, st);
    default: return launch_bwd<T, V, 4>(p, st);
  }
}
cudaError_t launch_conv(int dtype, const ConvParams& p, int taps, bool vec, cudaStream_t st) {
  if (dtype == 1) return vec ? launch_k<__nv_bfloat16, 8>(p, taps, st) : launch_k<__nv_bfloat16, 1>(p, taps, st);
  return vec ? launch_k<float, 4>(p, taps, st) : launch_k<float, 1>(p, taps, st);
}
cudaError_t launch_conv_bwd(int dtype, const ConvParams& p, int taps, bool vec, cudaStream_t st) {
  if (dtype == 1) return vec ? launch_bwd_k<__nv_bfloat16, 4>(p, taps, st) : launch_bwd_k<__nv_bfloat16, 1>(p, taps, st);
  return vec ? launch_bwd_k<float, 4>(p, taps, st) : launch_bwd_k<float, 1>(p, taps, st);
}

}  // namespace ttt
