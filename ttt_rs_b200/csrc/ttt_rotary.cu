// Rotary positions, and the root-mean-square norm of every head's query and key with the rotation in the same pass.
//
//   n = x / sqrt(mean(x^2) + eps) * w            (norm; w [F] for queries, another for keys)
//   (a, b) -> size (a cos - b sin, b cos + a sin)   for pairs p < rotary_dim / 2 of a row; angle = position * freq_p
// with neighbouring features (2p, 2p + 1) or the two halves of the rotated part (p, p + rotary_dim / 2) as pairs; features from
// rotary_dim on are left as they are.  Gradients: the rotation back by the same angle; with u the gradient of n,
//   dx = r (w u - x r^2 mean(w u x)),   dw = sum over rows of u x r,      r = 1 / sqrt(mean(x^2) + eps)
//
// Angles are integers: a frequency is held in turns per position as a 64-bit fraction, so position * frequency modulo one turn
// is one 64-bit product, exact to 2^-33 of a turn at any position, where a float32 angle of position 10^6 would be off by 0.03.
//
// Memory-bound: 16 bytes per lane and row both ways.  A group of lanes that covers a row owns one token: it makes the token's
// sines and cosines once and walks the heads of queries and keys with them, a few rows in flight.  Rows of a token's heads are
// neighbours in [B,T,H,F], rows of neighbouring tokens (the other groups of the warp) in [B,H,T,F]: whole lines in both.
#include "ttt_kernels.h"
#include "ttt_common.cuh"

namespace ttt {

constexpr int ROT_THREADS = 256;
constexpr int ROT_ROWS = 4;  // rows in flight

// V pairs of a row, NU times per lane (stride: the group).  V = 4: vectors of 4 or 8 elements; V = 1: any alignment.
template <typename T, int V>
struct PairIo;
template <typename T>
struct PairIo<T, 1> {
  T a, b;
  __device__ __forceinline__ void load(const T* p, int i, int j) { a = p[i], b = p[j]; }
  __device__ __forceinline__ void unpack(float (&x)[1], float (&y)[1]) const { x[0] = (float)a, y[0] = (float)b; }
  static __device__ __forceinline__ void store(T* p, int i, int j, const float (&x)[1], const float (&y)[1]) {
    p[i] = (T)x[0];
    p[j] = (T)y[0];
  }
};
template <>
struct PairIo<float, 4> {
  float4 a, b;
  __device__ __forceinline__ void load(const float* p, int i, int j) {
    a = *reinterpret_cast<const float4*>(p + i);
    b = *reinterpret_cast<const float4*>(p + j);
  }
  __device__ __forceinline__ void unpack(float (&x)[4], float (&y)[4]) const {
    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, y[0] = b.x, y[1] = b.y, y[2] = b.z, y[3] = b.w;
  }
  static __device__ __forceinline__ void store(float* p, int i, int j, const float (&x)[4], const float (&y)[4]) {
    *reinterpret_cast<float4*>(p + i) = make_float4(x[0], x[1], x[2], x[3]);
    *reinterpret_cast<float4*>(p + j) = make_float4(y[0], y[1], y[2], y[3]);
  }
};
template <>
struct PairIo<__nv_bfloat16, 4> {
  uint2 a, b;
  __device__ __forceinline__ void load(const __nv_bfloat16* p, int i, int j) {
    if (j == i + 4) {
      const uint4 v = *reinterpret_cast<const uint4*>(p + i);
      a = make_uint2(v.x, v.y);
      b = make_uint2(v.z, v.w);
    } else {
      a = *reinterpret_cast<const uint2*>(p + i);
      b = *reinterpret_cast<const uint2*>(p + j);
    }
  }
  __device__ __forceinline__ void unpack(float (&x)[4], float (&y)[4]) const {
    x[0] = bf16_lo(a.x), x[1] = bf16_hi(a.x), x[2] = bf16_lo(a.y), x[3] = bf16_hi(a.y);
    y[0] = bf16_lo(b.x), y[1] = bf16_hi(b.x), y[2] = bf16_lo(b.y), y[3] = bf16_hi(b.y);
  }
  static __device__ __forceinline__ void store(__nv_bfloat16* p, int i, int j, const float (&x)[4], const float (&y)[4]) {
    const uint2 a = make_uint2(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3])), b = make_uint2(pack_bf16(y[0], y[1]), pack_bf16(y[2], y[3]));
    if (j == i + 4) {
      *reinterpret_cast<uint4*>(p + i) = make_uint4(a.x, a.y, b.x, b.y);
    } else {
      *reinterpret_cast<uint2*>(p + i) = a;
      *reinterpret_cast<uint2*>(p + j) = b;
    }
  }
};

// Where the elements of a lane's unit lie in the row, and which of them belong to a pair: with x = elements at i.., y = at j..,
// pairs are (x[k], y[k]) if `split` (halves) and (x[0], x[1]), (x[2], x[3]), (y[0], y[1]), .. if not (V = 1: (x, y) always)
template <int V, bool HALF>
struct Unit {
  int i, j, pair;  // pair: first pair, or -1: not rotated
  bool live;
  __device__ __forceinline__ Unit(int u, int F, int r) {
    live = 2 * V * u < F;
    const bool rotated = 2 * V * u < r;
    pair = rotated ? V * u : -1;
    if (HALF && rotated) {
      i = V * u;
      j = r / 2 + V * u;
    } else {
      i = 2 * V * u;
      j = i + V;
    }
  }
};
template <int V, bool HALF>
__device__ __forceinline__ void rotate(float (&x)[V], float (&y)[V], const float (&c)[V], const float (&s)[V]) {
  if constexpr (HALF || V == 1) {
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const float a = x[k], b = y[k];
      x[k] = a * c[k] - b * s[k];
      y[k] = b * c[k] + a * s[k];
    }
  } else {
#pragma unroll
    for (int k = 0; k < V; k += 2) {
      const float a = x[k], b = x[k + 1], d = y[k], e = y[k + 1];
      x[k] = a * c[k / 2] - b * s[k / 2];
      x[k + 1] = b * c[k / 2] + a * s[k / 2];
      y[k] = d * c[V / 2 + k / 2] - e * s[V / 2 + k / 2];
      y[k + 1] = e * c[V / 2 + k / 2] + d * s[V / 2 + k / 2];
    }
  }
}
template <int V>
__device__ __forceinline__ void sines(float (&c)[V], float (&s)[V], const RotaryParams& p, int64_t pos, int pair) {
#pragma unroll
  for (int k = 0; k < V; ++k) {
    c[k] = 1.f;
    s[k] = 0.f;
    if (pair >= 0) {
      const uint64_t turn = (uint64_t)pos * p.turns[pair + k];
      sincospif((float)(int32_t)(turn >> 32) * 0x1p-31f, &s[k], &c[k]);
      c[k] *= p.size;
      s[k] *= p.sign * p.size;
    }
  }
}
__device__ __forceinline__ int64_t position(const RotaryParams& p, int64_t token, int T) {
  const int64_t b = token / T, t = token - b * T;
  int64_t pos = p.positions != nullptr ? p.positions[b * p.pos_stride + t] : p.start + t;
  if (p.wrap > 0) {
    pos %= p.wrap;
    if (pos < 0) pos += p.wrap;
  }
  return pos;
}
__device__ __forceinline__ float group_sum(float v, int lanes) {
  for (int o = lanes >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// NORM: the norm before the rotation.  BWD (with NORM): its gradient.
template <typename T, int V, int NU, bool HALF, bool NORM, bool BWD>
__global__ void __launch_bounds__(ROT_THREADS) ttt_rotary_kernel(const RotaryParams p) {
  const int lanes = p.lanes, tid = threadIdx.x, sub = tid & (lanes - 1), groups = ROT_THREADS / lanes;
  const int rows = p.heads[0] + p.heads[1];
  const int r_lo = (int)blockIdx.y * p.rows_each, r_hi = min(rows, r_lo + p.rows_each);
  const float inv_f = 1.f / p.F;
  float wgt[NORM ? 2 : 1][NU][2 * V], dw[BWD ? 2 : 1][NU][2 * V];
  if constexpr (NORM) {
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int n = 0; n < NU; ++n) {
        const Unit<V, HALF> u(sub + lanes * n, p.F, p.rdim);
#pragma unroll
        for (int k = 0; k < V; ++k) {
          wgt[m][n][k] = u.live && p.w[m] != nullptr ? ld_as_float<T>(p.w[m], u.i + k) : 1.f;
          wgt[m][n][V + k] = u.live && p.w[m] != nullptr ? ld_as_float<T>(p.w[m], u.j + k) : 1.f;
        }
      }
  }
  if constexpr (BWD) {
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int n = 0; n < NU; ++n)
#pragma unroll
        for (int k = 0; k < 2 * V; ++k) dw[m][n][k] = 0.f;
  }
  // whole groups of a warp take part in its shuffles to the end: a group without a token works on the last one and stores nothing
  for (int64_t first = (int64_t)blockIdx.x * groups; first < p.tokens; first += (int64_t)gridDim.x * groups) {
    const bool has = first + tid / lanes < p.tokens;
    const int64_t token = has ? first + tid / lanes : p.tokens - 1;
    const int64_t b = token / p.T, t = token - b * p.T;
    float c[NU][V], s[NU][V];
    const int64_t pos = p.rdim > 0 ? position(p, token, p.T) : 0;
#pragma unroll
    for (int n = 0; n < NU; ++n) sines<V>(c[n], s[n], p, pos, Unit<V, HALF>(sub + lanes * n, p.F, p.rdim).pair);
    for (int row0 = r_lo; row0 < r_hi; row0 += ROT_ROWS) {
      PairIo<T, V> in[ROT_ROWS][NU], grad[BWD ? ROT_ROWS : 1][NU];
#pragma unroll
      for (int q = 0; q < ROT_ROWS; ++q) {
        const int row = min(row0 + q, r_hi - 1), m = row >= p.heads[0], h = row - (m ? p.heads[0] : 0);
        const T* src = static_cast<const T*>(p.x[m]) + (b * p.xs[m][0] + h * p.xs[m][1] + t * p.xs[m][2]);
#pragma unroll
        for (int n = 0; n < NU; ++n) {
          const Unit<V, HALF> u(sub + lanes * n, p.F, p.rdim);
          if (u.live) in[q][n].load(src, u.i, u.j);
        }
        if constexpr (BWD) {
          const T* g = static_cast<const T*>(p.g[m]) + (b * p.gs[m][0] + h * p.gs[m][1] + t * p.gs[m][2]);
#pragma unroll
          for (int n = 0; n < NU; ++n) {
            const Unit<V, HALF> u(sub + lanes * n, p.F, p.rdim);
            if (u.live) grad[q][n].load(g, u.i, u.j);
          }
        }
      }
#pragma unroll
      for (int q = 0; q < ROT_ROWS; ++q) {
        if (row0 + q >= r_hi) break;
        const int row = row0 + q, m = row >= p.heads[0], h = row - (m ? p.heads[0] : 0);
        T* dst = static_cast<T*>(p.y[m]) + (b * p.ys[m][0] + h * p.ys[m][1] + t * p.ys[m][2]);
        float x[NU][V], y[NU][V];
        float sq = 0.f;
#pragma unroll
        for (int n = 0; n < NU; ++n) {
          const Unit<V, HALF> u(sub + lanes * n, p.F, p.rdim);
          if (u.live) in[q][n].unpack(x[n], y[n]);
#pragma unroll
          for (int k = 0; k < V; ++k) {
            if (!u.live) x[n][k] = y[n][k] = 0.f;
            if (NORM) sq = fmaf(x[n][k], x[n][k], fmaf(y[n][k], y[n][k], sq));
          }
        }
        float r = 1.f;
        if constexpr (NORM) r = rsqrtf(group_sum(sq, lanes) * inv_f + p.eps);
        if constexpr (!BWD) {
#pragma unroll
          for (int n = 0; n < NU; ++n) {
            const Unit<V, HALF> u(sub + lanes * n, p.F, p.rdim);
            if constexpr (NORM) {
#pragma unroll
              for (int k = 0; k < V; ++k) {
                x[n][k] *= r * (m ? wgt[1][n][k] : wgt[0][n][k]);
                y[n][k] *= r * (m ? wgt[1][n][V + k] : wgt[0][n][V + k]);
              }
            }
            rotate<V, HALF>(x[n], y[n], c[n], s[n]);
            if (u.live && has) PairIo<T, V>::store(dst, u.i, u.j, x[n], y[n]);
          }
        } else {
          float gx[NU][V], gy[NU][V], dot = 0.f;
#pragma unroll
          for (int n = 0; n < NU; ++n) {
            const Unit<V, HALF> u(sub + lanes * n, p.F, p.rdim);
            if (u.live) grad[q][n].unpack(gx[n], gy[n]);
#pragma unroll
            for (int k = 0; k < V; ++k)
              if (!u.live) gx[n][k] = gy[n][k] = 0.f;
            rotate<V, HALF>(gx[n], gy[n], c[n], s[n]);
#pragma unroll
            for (int k = 0; k < V; ++k) {
              const float ax = gx[n][k] * x[n][k] * r, ay = gy[n][k] * y[n][k] * r;
              if (has) {
                dw[0][n][k] += m ? 0.f : ax;
                dw[0][n][V + k] += m ? 0.f : ay;
                dw[1][n][k] += m ? ax : 0.f;
                dw[1][n][V + k] += m ? ay : 0.f;
              }
              gx[n][k] *= m ? wgt[1][n][k] : wgt[0][n][k];
              gy[n][k] *= m ? wgt[1][n][V + k] : wgt[0][n][V + k];
              dot = fmaf(gx[n][k], x[n][k], fmaf(gy[n][k], y[n][k], dot));
            }
          }
          const float f = group_sum(dot, lanes) * inv_f * r * r * r;
#pragma unroll
          for (int n = 0; n < NU; ++n) {
            const Unit<V, HALF> u(sub + lanes * n, p.F, p.rdim);
#pragma unroll
            for (int k = 0; k < V; ++k) {
              gx[n][k] = r * gx[n][k] - f * x[n][k];
              gy[n][k] = r * gy[n][k] - f * y[n][k];
            }
            if (u.live && has) PairIo<T, V>::store(dst, u.i, u.j, gx[n], gy[n]);
          }
        }
      }
    }
  }
  if constexpr (BWD) {  // this block's share of the weights' gradients, in a fixed order: groups of a warp, warps, blocks
    if (p.partials == nullptr) return;
    extern __shared__ float rot_smem[];  // [warps][2][F]
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int n = 0; n < NU; ++n) {
        const Unit<V, HALF> u(sub + lanes * n, p.F, p.rdim);
#pragma unroll
        for (int k = 0; k < 2 * V; ++k) {
          float v = dw[m][n][k];
          for (int o = lanes; o < 32; o <<= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
          if (u.live && (tid & 31) < lanes) rot_smem[((tid >> 5) * 2 + m) * p.F + (k < V ? u.i + k : u.j + k - V)] = v;
        }
      }
    __syncthreads();
    float* out = p.partials + ((size_t)blockIdx.y * gridDim.x + blockIdx.x) * 2 * p.F;
    for (int e = tid; e < 2 * p.F; e += ROT_THREADS) {
      float v = 0.f;
#pragma unroll
      for (int k = 0; k < ROT_THREADS / 32; ++k) v += rot_smem[k * 2 * p.F + e];
      out[e] = v;
    }
  }
}

// The blocks' shares to the gradients of both weights: a warp per column, lanes over the blocks
template <typename T>
__global__ void __launch_bounds__(256) ttt_rotary_reduce_kernel(const float* partials, int blocks, int F, T* dq, T* dk) {
  const int col = (int)blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (col >= 2 * F) return;
  float v = 0.f;
  for (int k = lane; k < blocks; k += 32) v += partials[(size_t)k * 2 * F + col];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if (lane != 0) return;
  T* out = col < F ? dq : dk;
  if (out != nullptr) st_from_float<T>(out, col < F ? col : col - F, v);
}

// Blocks: tokens of groups of lanes, and the rows of a token in as many shares as it takes to fill the card
struct RotaryGrid {
  int x, y, rows_each, lanes;
};
static RotaryGrid rotary_grid(int64_t tokens, int rows, int F, bool vec, bool bwd) {
  RotaryGrid g;
  const int units = vec ? F / 8 : F / 2;
  g.lanes = 1;
  while (g.lanes < units && g.lanes < 32) g.lanes *= 2;
  const int groups = ROT_THREADS / g.lanes;
  const int64_t blocks = (tokens + groups - 1) / groups;
  constexpr int FILL = 148 * 8;
  int64_t shares = (FILL + blocks - 1) / blocks;
  const int most = (rows + ROT_ROWS - 1) / ROT_ROWS;
  if (shares > most) shares = most;
  g.rows_each = (int)((rows + shares - 1) / shares);
  g.y = (rows + g.rows_each - 1) / g.rows_each;
  int64_t x = blocks;
  const int64_t cap = bwd ? (FILL + g.y - 1) / g.y : (int64_t)1 << 30;
  if (x > cap) x = cap;
  g.x = (int)x;
  return g;
}
size_t rotary_partial_floats(int64_t tokens, int rows, int F) {
  size_t most = 0;
  for (bool vec : {false, true}) {  // (which of them runs depends on addresses)
    if (vec && F % 8 != 0) continue;
    const RotaryGrid g = rotary_grid(tokens, rows, F, vec, true);
    const size_t n = (size_t)g.x * g.y * 2 * F;
    if (n > most) most = n;
  }
  return most;
}

template <typename T, int V, int NU, bool HALF>
static cudaError_t launch_rot(RotaryParams p, bool norm, bool bwd, cudaStream_t st) {
  const RotaryGrid g = rotary_grid(p.tokens, p.heads[0] + p.heads[1], p.F, V == 4, bwd);
  p.rows_each = g.rows_each;
  p.lanes = g.lanes;
  const dim3 grid(g.x, g.y);
  const size_t smem = bwd ? (ROT_THREADS / 32) * 2 * p.F * sizeof(float) : 0;
  if (!norm) ttt_rotary_kernel<T, V, NU, HALF, false, false><<<grid, ROT_THREADS, 0, st>>>(p);
  else if (!bwd) ttt_rotary_kernel<T, V, NU, HALF, true, false><<<grid, ROT_THREADS, 0, st>>>(p);
  else ttt_rotary_kernel<T, V, NU, HALF, true, true><<<grid, ROT_THREADS, smem, st>>>(p);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess || !bwd || p.partials == nullptr) return e;
  ttt_rotary_reduce_kernel<T><<<(2 * p.F + 7) / 8, 256, 0, st>>>(p.partials, g.x * g.y, p.F, static_cast<T*>(p.dw[0]),
                                                                static_cast<T*>(p.dw[1]));
  return cudaGetLastError();
}
template <typename T>
static cudaError_t launch_rot_t(const RotaryParams& p, bool vec, bool half, bool norm, bool bwd, cudaStream_t st) {
  if (vec) return half ? launch_rot<T, 4, 1, true>(p, norm, bwd, st) : launch_rot<T, 4, 1, false>(p, norm, bwd, st);
  return half ? launch_rot<T, 1, 4, true>(p, norm, bwd, st) : launch_rot<T, 1, 4, false>(p, norm, bwd, st);
}
cudaError_t launch_rotary(int dtype, const RotaryParams& p, bool vec, bool half, bool norm, bool bwd, cudaStream_t st) {
  return dtype == 1 ? launch_rot_t<__nv_bfloat16>(p, vec, half, norm, bwd, st) : launch_rot_t<float>(p, vec, half, norm, bwd, st);
}

}  // namespace ttt
