// Causal depthwise convolution of 2 to 4 taps over [B,T,C], channels last, with bias and SiLU, forward and backward.
//
//   v_t = bias + sum_j w_j x_{t-K+1+j},  y_t = v_t or SiLU(v_t)
// Inputs before the row are the carried state's (or zeros); a start at token t hides everything before t from t on.  The new state
// is the last K - 1 inputs, as they are visible behind the last token.  With g_t = dy_t act'(v_t):
//   dx_s = sum_j w_j g_{s+K-1-j} over the tokens that saw s (+ the new state's gradient),  dw_j = sum_t g_t x_{t-K+1+j},  db = sum_t g_t
//
// Memory-bound by its bytes, held back by latency with few warps and by instructions.  A thread holds four neighbouring channels (two of bf16, or one,
// where rows are off a vector's address) and walks a strip of tokens with the last K - 1 inputs in registers and the next few tokens on their way; the
// tokens before a strip (and behind it, for dx) are read again, from L2.  Whole groups of tokens inside a strip go without checks.  A
// start empties the registers of the inputs, and the sums of dx know the last start's place; without starts, kernels know of none.
// bf16, 65536 tokens of 1536 channels, 4 taps, SiLU: 94 us forward (4.3 TB/s, 0.65 of a copy), 167 us backward (3.6 TB/s, 0.55).  Eight
// channels per thread took so many registers that a quarter of the threads fitted: 208 us forward.  Strips of 64 tokens: 115 us for 100
// at that stage; without the next tokens on their way 230 us for 207 backward; with checks at every token 207 us for 168.  15 of 64 warps
// are active, 46 and 53 % of issue slots used; of the 128 registers that two backward blocks leave a thread, 4 taps of bf16 spill: 184 bytes
// written and 268 read per thread with SiLU (104 / 100 without, 202 / 332 with starts; float32 36 to 84 / 80 to 156; 3 taps 16 / 32).
#include <type_traits>

#include "ttt_kernels.h"
#include "ttt_vec.cuh"

namespace ttt {

constexpr int CONV_THREADS = 256;
constexpr int CONV_FWD_RESIDENT = 2, CONV_BWD_RESIDENT = 2;  // blocks per SM that registers are bounded for
template <typename T>
__host__ __device__ constexpr int conv_ahead(bool bwd) {  // tokens on their way at a time
  return bwd && sizeof(T) == 4 ? 2 : 4;
}

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
    if constexpr (V > 1) {  // (as aligned as the rows)
#pragma unroll
      for (int i = 0; i < K; ++i) {
        Chan<T, V> r;
        F2 v[P];
        r.load(at + i * V);
        r.unpack(v);
#pragma unroll
        for (int k = 0; k < P; ++k) e[i * V + 2 * k] = v[k].x, e[i * V + 2 * k + 1] = v[k].y;
      }
    } else {
#pragma unroll
      for (int i = 0; i < K; ++i) e[i] = ld_as_float<T>(at, i);
    }
#pragma unroll
    for (int k = 0; k < P; ++k) {
#pragma unroll
      for (int j = 0; j < K; ++j) w[j][k] = f2(e[2 * k * K + j], 2 * k + 1 < V ? e[(2 * k + 1 < V ? 2 * k + 1 : 0) * K + j] : 0.f);
      bias[k] = f2(0.f);
      if (p.bias != nullptr) bias[k] = f2(ld_as_float<T>(p.bias, c + 2 * k), 2 * k + 1 < V ? ld_as_float<T>(p.bias, c + 2 * k + 1) : 0.f);
    }
  }
};

// The K - 1 inputs before token t0 of a sequence, as they are visible there; `last`: the last start among them, from t0 on
template <typename T, int V, int K, bool MARKS>
__device__ __forceinline__ void conv_before(F2 (&h)[K - 1][Chan<T, V>::P], int& last, const ConvParams& p, const T* x, const T* state,
                                            const uint8_t* starts, int64_t t0) {
  constexpr int P = Chan<T, V>::P;
  Chan<T, V> r[K - 1];
#pragma unroll
  for (int i = 0; i < K - 1; ++i) conv_row<T, V, K>(r[i], p, x, state, t0 - (K - 1) + i);
#pragma unroll
  for (int i = 0; i < K - 1; ++i) r[i].unpack(h[i]);
  if constexpr (MARKS) {  // a start hides what lies before it
#pragma unroll
    for (int i = 0; i < K - 1; ++i) {
      const int64_t t = t0 - (K - 1) + i;
      if (t >= 0 && starts[t]) {
        last = i - (K - 1);
#pragma unroll
        for (int e = 0; e < i; ++e)
#pragma unroll
          for (int k = 0; k < P; ++k) h[e][k] = f2(0.f);
      }
    }
  }
}

// Blocks walk strips with a stride: the weights are read once.  MARKS: there are starts.
template <typename T, int V, int K, bool ACT, bool MARKS>
__global__ void __launch_bounds__(CONV_THREADS, CONV_FWD_RESIDENT) ttt_conv_kernel(const ConvParams p) {
  using Ch = Chan<T, V>;
  constexpr int P = Ch::P, AHEAD = conv_ahead<T>(false);
  const int lane = threadIdx.x & ((1 << p.lanes_log) - 1), rows = CONV_THREADS >> p.lanes_log;
  const int c = ((int)blockIdx.y * (1 << p.lanes_log) + lane) * V;
  if (c >= p.C) return;
  ConvWeights<T, V, K> w;
  w.load(p, c);
  for (int64_t strip = (int64_t)blockIdx.x * rows + (threadIdx.x >> p.lanes_log); strip < p.B * p.strips; strip += (int64_t)gridDim.x * rows) {
    const int64_t b = strip / p.strips, t0 = (strip - b * p.strips) * p.strip;
    const int n = (int)min((int64_t)p.strip, p.T - t0);
    const T* x = static_cast<const T*>(p.x) + b * p.xs[0] + c;
    const T* state = p.state != nullptr ? static_cast<const T*>(p.state) + b * (K - 1) * p.C + c : nullptr;
    const uint8_t* starts = MARKS ? p.starts + b * p.T : nullptr;
    F2 h[K - 1][P];  // h[i]: token t - (K - 1) + i
    int last = 0;
    conv_before<T, V, K, MARKS>(h, last, p, x, state, starts, t0);
    const T* in_at = x + t0 * p.xs[1];
    T* y = static_cast<T*>(p.y) + (b * p.T + t0) * p.C + c;
    Ch next[AHEAD];  // the tokens behind those that are worked on: on their way meanwhile
    [[maybe_unused]] uint8_t next_first[AHEAD];
    auto fetch = [&](int at) {
      if (at + AHEAD <= n) {
#pragma unroll
        for (int u = 0; u < AHEAD; ++u, in_at += p.xs[1]) {
          next[u].load(in_at);
          if constexpr (MARKS) next_first[u] = starts[t0 + at + u];
        }
      } else {
#pragma unroll
        for (int u = 0; u < AHEAD; ++u, in_at += p.xs[1])
          if (at + u < n) {
            next[u].load(in_at);
            if constexpr (MARKS) next_first[u] = starts[t0 + at + u];
          }
      }
    };
    auto some = [&](int at, auto all) {  // AHEAD tokens, or as many as are left
      Ch in[AHEAD];
      [[maybe_unused]] uint8_t first[AHEAD];
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) {
        in[u] = next[u];
        if constexpr (MARKS) first[u] = next_first[u];
      }
      fetch(at + AHEAD);
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) {
        if (!decltype(all)::value && at + u >= n) break;
        if (MARKS && first[u]) {
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
          if constexpr (ACT) v[k] = f2(act_of(v[k].x, ACT_SILU), act_of(v[k].y, ACT_SILU));
        }
        Ch out;
        out.pack(v);
        out.store(y);
        y += p.C;
      }
    };
    fetch(0);
    int at = 0;
    for (; at + AHEAD <= n; at += AHEAD) some(at, std::true_type{});
    if (at < n) some(at, std::false_type{});
    // The thread of the first tokens, the only one that has read the given state, writes the new one: they may be the same tensor.
    // (Behind a short row a part of the given state is still visible: read it all before writing.)
    if (t0 == 0) {
      Ch r[K - 1];
#pragma unroll
      for (int i = 0; i < K - 1; ++i) conv_row<T, V, K>(r[i], p, x, state, p.T - (K - 1) + i);
      if constexpr (MARKS) {
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
}

// Blocks walk strips with a stride and leave one row of sums for the weights and the bias each: [K + 1][C].
template <typename T, int V, int K, bool ACT, bool MARKS>
__global__ void __launch_bounds__(CONV_THREADS, CONV_BWD_RESIDENT) ttt_conv_bwd_kernel(const ConvParams p) {
  using Ch = Chan<T, V>;
  constexpr int P = Ch::P, AHEAD = conv_ahead<T>(true);
  const int lanes = 1 << p.lanes_log, rows = CONV_THREADS >> p.lanes_log;
  const int lane = threadIdx.x & (lanes - 1), row = threadIdx.x >> p.lanes_log;
  const int c = ((int)blockIdx.y * lanes + lane) * V;
  F2 dw[K + 1][P];
#pragma unroll
  for (int j = 0; j <= K; ++j)
#pragma unroll
    for (int k = 0; k < P; ++k) dw[j][k] = f2(0.f);
  if (c < p.C) {
    ConvWeights<T, V, K> w;
    w.load(p, c);
    for (int64_t strip = (int64_t)blockIdx.x * rows + row; strip < p.B * p.strips; strip += (int64_t)gridDim.x * rows) {
      // tokens and gradients count from the strip's first token
      const int64_t b = strip / p.strips, t0 = (strip - b * p.strips) * p.strip;
      const int n = (int)min((int64_t)p.strip, p.T - t0);
      const int n_read = (int)min((int64_t)(p.strip + K - 1), p.T - t0);      // tokens that add to this strip's gradients
      const int s_lo = t0 == 0 ? -(K - 1) : 0;                                // the first strip's begin with the state's
      const int s_tail = (int)min(p.T - (K - 1) - t0, (int64_t)1 << 30);      // from here on the new state's gradient is added
      const T* x = static_cast<const T*>(p.x) + b * p.xs[0] + c;
      const T* state = p.state != nullptr ? static_cast<const T*>(p.state) + b * (K - 1) * p.C + c : nullptr;
      const T* gstate_out = p.gstate_out != nullptr ? static_cast<const T*>(p.gstate_out) + b * (K - 1) * p.C + c : nullptr;
      const uint8_t* starts = MARKS ? p.starts + b * p.T : nullptr;
      F2 h[K - 1][P], acc[K - 1][P];  // acc[i]: gradient of token t - (K - 1) + i so far
      int last = -(1 << 30);
      conv_before<T, V, K, MARKS>(h, last, p, x, state, starts, t0);
#pragma unroll
      for (int i = 0; i < K - 1; ++i)
#pragma unroll
        for (int k = 0; k < P; ++k) acc[i][k] = f2(0.f);
      const T* in_at = x + t0 * p.xs[1];
      const T* g_at = static_cast<const T*>(p.gy) + b * p.gs[0] + t0 * p.gs[1] + c;
      T* gx = static_cast<T*>(p.gx) + (b * p.T + t0 - (K - 1)) * p.C + c;  // token t completes the gradient of token t - (K - 1)
      Ch next[AHEAD], next_grad[AHEAD];  // the tokens behind those that are worked on: on their way meanwhile
      [[maybe_unused]] uint8_t next_first[AHEAD];
      auto fetch = [&](int at) {
        if (at + AHEAD <= n_read) {
#pragma unroll
          for (int u = 0; u < AHEAD; ++u, in_at += p.xs[1], g_at += p.gs[1]) {
            next[u].load(in_at);
            next_grad[u].load(g_at);
            if constexpr (MARKS) next_first[u] = starts[t0 + at + u];
          }
        } else {
#pragma unroll
          for (int u = 0; u < AHEAD; ++u, in_at += p.xs[1], g_at += p.gs[1]) {
            next[u].zero();  // (no gradient: nothing is added)
            next_grad[u].zero();
            if constexpr (MARKS) next_first[u] = 0;
            if (at + u < n_read) {
              next[u].load(in_at);
              next_grad[u].load(g_at);
              if constexpr (MARKS) next_first[u] = starts[t0 + at + u];
            }
          }
        }
      };
      auto some = [&](int at, auto all) {  // AHEAD tokens; all: of the strip, each, and at least K - 1 of it before them
        Ch in[AHEAD], grad[AHEAD];
        [[maybe_unused]] uint8_t first[AHEAD];
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
          in[u] = next[u], grad[u] = next_grad[u];
          if constexpr (MARKS) first[u] = next_first[u];
        }
        fetch(at + AHEAD);
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
          const int t = at + u;
          if (!decltype(all)::value && t >= n + K - 1) break;
          if (MARKS && first[u]) {
            last = t;
#pragma unroll
            for (int i = 0; i < K - 1; ++i)
#pragma unroll
              for (int k = 0; k < P; ++k) h[i][k] = f2(0.f);
          }
          F2 now[P], gv[P], whole[P];
          in[u].unpack(now);
          grad[u].unpack(gv);
#pragma unroll
          for (int k = 0; k < P; ++k) {
            if constexpr (ACT) {
              F2 v = f2fma(now[k], w.w[K - 1][k], w.bias[k]), slope;
#pragma unroll
              for (int i = 0; i < K - 1; ++i) v = f2fma(h[i][k], w.w[i][k], v);
              act_and_slope(v.x, ACT_SILU, slope.x);
              act_and_slope(v.y, ACT_SILU, slope.y);
              if (decltype(all)::value || t < n_read) gv[k] = f2mul(gv[k], slope);
            }
            if (decltype(all)::value || t < n) {  // (the tokens behind the strip are another's for the weights)
#pragma unroll
              for (int i = 0; i < K - 1; ++i) dw[i][k] = f2fma(gv[k], h[i][k], dw[i][k]);
              dw[K - 1][k] = f2fma(gv[k], now[k], dw[K - 1][k]);
              dw[K][k] = f2add(dw[K][k], gv[k]);
            }
#pragma unroll
            for (int i = 0; i < K - 1; ++i)
              if (!MARKS || t - (K - 1) + i >= last) acc[i][k] = f2fma(gv[k], w.w[i][k], acc[i][k]);
            whole[k] = acc[0][k];
#pragma unroll
            for (int i = 0; i < K - 2; ++i) acc[i][k] = acc[i + 1][k], h[i][k] = h[i + 1][k];
            acc[K - 2][k] = f2mul(gv[k], w.w[K - 1][k]);
            h[K - 2][k] = now[k];
          }
          const int s = t - (K - 1);
          if (decltype(all)::value || s >= s_lo) {
            if (!decltype(all)::value && gstate_out != nullptr && s >= s_tail && (!MARKS || s >= last)) {
              Ch r;
              F2 e[P];
              r.load(gstate_out + (int64_t)(s - s_tail) * p.C);
              r.unpack(e);
#pragma unroll
              for (int k = 0; k < P; ++k) whole[k] = f2add(whole[k], e[k]);
            }
            Ch out;
            out.pack(whole);
            if (decltype(all)::value || t0 + s >= 0) out.store(gx);
            else if (p.gstate != nullptr) out.store(static_cast<T*>(p.gstate) + (b * (K - 1) + s + K - 1) * p.C + c);
          }
          gx += p.C;
        }
      };
      fetch(0);
      int at = 0;
      for (; at < K - 1; at += AHEAD) some(at, std::false_type{});
      for (; at + AHEAD <= n; at += AHEAD) some(at, std::true_type{});
      for (; at < n + K - 1; at += AHEAD) some(at, std::false_type{});
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

// the blocks' sums [rows][K + 1][C] -> gradients of the weight [C][K] and the bias
template <typename T>
__global__ void __launch_bounds__(ROWS_THREADS) ttt_conv_reduce_kernel(const float* partials, int rows, int C, int K, T* gw, T* gbias) {
  int64_t col;
  float v;
  const int64_t n = (int64_t)(K + 1) * C;
  if (!sum_of_rows(partials, rows, n, n, blockIdx.x, &col, &v)) return;
  const int j = (int)(col / C), c = (int)(col - (int64_t)j * C);
  if (j < K) {
    if (gw != nullptr) st_from_float<T>(gw, (size_t)c * K + j, v);
  } else if (gbias != nullptr) {
    st_from_float<T>(gbias, c, v);
  }
}

// Strips of 32 tokens where the threads then fill the card, shorter ones where not: a strip's neighbours cost K - 1 rows more.  Blocks
// that are resident walk all strips.
struct ConvCut {
  int lanes_log, strip, y;
  int64_t strips, x;
};
static ConvCut conv_cut(int64_t B, int64_t T, int C, int V, bool bwd) {
  ConvCut k{};
  const int vectors = (C + V - 1) / V, resident = bwd ? CONV_BWD_RESIDENT : CONV_FWD_RESIDENT;
  while (k.lanes_log < 5 && (1 << k.lanes_log) < vectors) ++k.lanes_log;
  k.y = (vectors + (1 << k.lanes_log) - 1) >> k.lanes_log;
  const int64_t wide = (int64_t)k.y << k.lanes_log, fill = (int64_t)148 * resident * CONV_THREADS;
  int strip = 32;
  while (strip > 4 && B * ((T + strip - 1) / strip) * wide < fill) strip /= 2;
  k.strip = strip;
  k.strips = (T + strip - 1) / strip;
  const int per_block = CONV_THREADS >> k.lanes_log;
  const int64_t need = (B * k.strips + per_block - 1) / per_block, most = 148 * resident / k.y > 1 ? 148 * resident / k.y : 1;
  k.x = need < most ? need : most;
  return k;
}
size_t conv_partial_floats(int64_t B, int64_t T, int C, int K) {  // for any width
  size_t most = 0;
  for (int V : {1, 2, 4}) {
    const size_t n = (size_t)conv_cut(B, T, C, V, true).x * (K + 1) * C;
    if (n > most) most = n;
  }
  return most;
}

template <typename T, int V, int K, bool ACT, bool MARKS>
static cudaError_t launch_one(ConvParams p, bool bwd, cudaStream_t st) {
  const ConvCut k = conv_cut(p.B, p.T, p.C, V, bwd);
  p.lanes_log = k.lanes_log, p.strip = k.strip, p.strips = k.strips;
  const dim3 grid((unsigned)k.x, k.y);
  if (!bwd) {
    ttt_conv_kernel<T, V, K, ACT, MARKS><<<grid, CONV_THREADS, 0, st>>>(p);
    return cudaGetLastError();
  }
  const size_t smem = sizeof(float) * CONV_THREADS * V * (K + 1);
  ttt_conv_bwd_kernel<T, V, K, ACT, MARKS><<<grid, CONV_THREADS, smem, st>>>(p);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess || p.partials == nullptr) return e;
  ttt_conv_reduce_kernel<T><<<((K + 1) * p.C + 31) / 32, ROWS_THREADS, 0, st>>>(p.partials, (int)k.x, p.C, K, static_cast<T*>(p.gw),
                                                                               static_cast<T*>(p.gbias));
  return cudaGetLastError();
}
template <typename T, int V, int K>
static cudaError_t launch_kind(const ConvParams& p, bool bwd, cudaStream_t st) {
  if (p.starts != nullptr) return p.act == ACT_SILU ? launch_one<T, V, K, true, true>(p, bwd, st) : launch_one<T, V, K, false, true>(p, bwd, st);
  return p.act == ACT_SILU ? launch_one<T, V, K, true, false>(p, bwd, st) : launch_one<T, V, K, false, false>(p, bwd, st);
}
template <typename T, int V>
static cudaError_t launch_k(const ConvParams& p, int taps, bool bwd, cudaStream_t st) {
  switch (taps) {
    case 2: return launch_kind<T, V, 2>(p, bwd, st);
    case 3: return launch_kind<T, V, 3>(p, bwd, st);
    default: return launch_kind<T, V, 4>(p, bwd, st);
  }
}
cudaError_t launch_conv(int dtype, const ConvParams& p, int taps, int V, bool bwd, cudaStream_t st) {
  if (dtype == 1)
    return V == 4 ? launch_k<__nv_bfloat16, 4>(p, taps, bwd, st) : V == 2 ? launch_k<__nv_bfloat16, 2>(p, taps, bwd, st)
                                                                          : launch_k<__nv_bfloat16, 1>(p, taps, bwd, st);
  return V == 4 ? launch_k<float, 4>(p, taps, bwd, st) : launch_k<float, 1>(p, taps, bwd, st);
}

}  // namespace ttt
