// Rotary positions, and the root-mean-square norm of every head's query and key with the rotation in the same pass.
//
//   n = x / sqrt(mean(x^2) + eps) * w            (norm; w [F] for queries, another for keys)
//   (a, b) -> size (a cos - b sin, b cos + a sin)   for pairs p < rotary_dim / 2 of a row; angle = position * freq_p
// with neighbouring features (2p, 2p + 1) or the two halves of the rotated part (p, p + rotary_dim / 2) as pairs; features from
// rotary_dim on are left as they are.  Gradients: the rotation back by the same angle; with u the gradient of n,
//   dx = r (w u - x r^2 mean(w u x)),   dw = sum over rows of u x r,      r = 1 / sqrt(mean(x^2) + eps)
//
// Angles are integers: a frequency is held in turns per position as a 64-bit fraction, so position * frequency modulo one turn
// is one 64-bit product, exact at any position, where a float32 angle of position 10^6 would be off by 0.03.  What is off is the
// float32 that the sine takes, by 2^-26 of a turn at most (half a last place near half a turn), and the table, made of frequencies of 53
// bits: about 2^-55 of a turn per position for the fastest pair, 2^-24 at position 2^31.
//
// Memory-bound: 16 bytes per lane and row both ways.  A group of lanes that covers a row owns one token: it makes the token's
// sines and cosines once and walks the heads of queries and keys with them, a few rows in flight.  Rows of a token's heads are
// neighbours in [B,T,H,F], rows of neighbouring tokens (the other groups of the warp) in [B,H,T,F]: whole lines in both.  bf16,
// F = 64: rotation of 32768 tokens of 32 rows 45 us (6.0 TB/s, 0.91 of a copy), norm and rotation of 65536 tokens of 24 rows 72 us, its
// gradient 108 us (5.6 TB/s both, 0.85); float32 calls of the latter sizes 131 and 201 us (0.94 and 0.92), though the gradient's registers
// leave one block per SM.  Rows off the 16 bytes, and rotated parts that are no multiple of 8, go feature by feature with a warp per row,
// in instances that spill: bf16, 32768 tokens of 16 + 16 rows of 80 features, 20 of them rotated against 24, the call: norm and rotation
// 301 to 393 us against 90 to 96, its gradient 850 to 968 against 145 to 152; rotation alone (16 rows) 94 to 123 against 39 to 45.
#include <type_traits>

#include "ttt_kernels.h"
#include "ttt_common.cuh"

namespace ttt {

constexpr int ROT_THREADS = 256;
constexpr int ROT_ROWS = 4;  // rows in flight

constexpr int rotary_resident(bool f32, bool norm, bool bwd) {  // blocks per SM that the kernels' registers are bounded for
  return bwd ? (f32 ? 1 : 2) : f32 ? (norm ? 2 : 3) : norm ? 3 : 4;
}
// A unit is V pairs of a row, NU of them per lane (a group's lanes apart): x[k] and y[k] are the two features of pair k (V = 4: of
// two pairs (x[0], x[1]) and (y[0], y[1]) side by side in registers, for the packed float32 operations).  Features behind the rotated
// part come in units too, as pairs that are not turned.  V = 4 takes 16 bytes at a time, V = 1 single features at any address.
template <int V, bool HALF>
struct Unit {
  int i, j, pair;  // elements of the row: V from i on and V from j on; first pair, or -1: not rotated
  bool live;
  __device__ __forceinline__ Unit(int u, int F, int r) {
    live = 2 * V * u < F;
    const bool rotated = 2 * V * u < r;
    pair = rotated ? V * u : -1;
    i = HALF && rotated ? V * u : 2 * V * u;
    j = HALF && rotated ? r / 2 + V * u : i + V;
  }
};
template <typename T, int V, bool HALF>
struct Pairs;
template <typename T, bool HALF>
struct Pairs<T, 1, HALF> {
  T a, b;
  __device__ __forceinline__ void load(const T* p, const Unit<1, HALF>& u) { a = p[u.i], b = p[u.j]; }
  __device__ __forceinline__ void unpack(F2 (&x)[1], F2 (&y)[1]) const { x[0] = f2((float)a, 0.f), y[0] = f2((float)b, 0.f); }
  static __device__ __forceinline__ void store(T* p, const Unit<1, HALF>& u, const F2 (&x)[1], const F2 (&y)[1]) {
    p[u.i] = (T)x[0].x;
    p[u.j] = (T)y[0].x;
  }
};
template <bool HALF>
struct Pairs<float, 4, HALF> {
  float4 a, b;
  __device__ __forceinline__ void load(const float* p, const Unit<4, HALF>& u) {
    a = *reinterpret_cast<const float4*>(p + u.i);
    b = *reinterpret_cast<const float4*>(p + u.j);
  }
  __device__ __forceinline__ void unpack(F2 (&x)[2], F2 (&y)[2]) const {
    if constexpr (HALF) x[0] = f2(a.x, a.y), x[1] = f2(a.z, a.w), y[0] = f2(b.x, b.y), y[1] = f2(b.z, b.w);
    else x[0] = f2(a.x, a.z), y[0] = f2(a.y, a.w), x[1] = f2(b.x, b.z), y[1] = f2(b.y, b.w);
  }
  static __device__ __forceinline__ void store(float* p, const Unit<4, HALF>& u, const F2 (&x)[2], const F2 (&y)[2]) {
    float4 a, b;
    if constexpr (HALF) a = make_float4(x[0].x, x[0].y, x[1].x, x[1].y), b = make_float4(y[0].x, y[0].y, y[1].x, y[1].y);
    else a = make_float4(x[0].x, y[0].x, x[0].y, y[0].y), b = make_float4(x[1].x, y[1].x, x[1].y, y[1].y);
    *reinterpret_cast<float4*>(p + u.i) = a;
    *reinterpret_cast<float4*>(p + u.j) = b;
  }
};
template <bool HALF>
struct Pairs<__nv_bfloat16, 4, HALF> {
  uint2 a, b;
  __device__ __forceinline__ void load(const __nv_bfloat16* p, const Unit<4, HALF>& u) {
    if constexpr (HALF) {
      a = *reinterpret_cast<const uint2*>(p + u.i);
      b = *reinterpret_cast<const uint2*>(p + u.j);
    } else {
      const uint4 v = *reinterpret_cast<const uint4*>(p + u.i);
      a = make_uint2(v.x, v.y);
      b = make_uint2(v.z, v.w);
    }
  }
  __device__ __forceinline__ void unpack(F2 (&x)[2], F2 (&y)[2]) const {
    if constexpr (HALF) {
      x[0] = f2(bf16_lo(a.x), bf16_hi(a.x)), x[1] = f2(bf16_lo(a.y), bf16_hi(a.y));
      y[0] = f2(bf16_lo(b.x), bf16_hi(b.x)), y[1] = f2(bf16_lo(b.y), bf16_hi(b.y));
    } else {
      x[0] = f2(bf16_lo(a.x), bf16_lo(a.y)), y[0] = f2(bf16_hi(a.x), bf16_hi(a.y));
      x[1] = f2(bf16_lo(b.x), bf16_lo(b.y)), y[1] = f2(bf16_hi(b.x), bf16_hi(b.y));
    }
  }
  static __device__ __forceinline__ void store(__nv_bfloat16* p, const Unit<4, HALF>& u, const F2 (&x)[2], const F2 (&y)[2]) {
    if constexpr (HALF) {
      *reinterpret_cast<uint2*>(p + u.i) = make_uint2(pack_bf16(x[0].x, x[0].y), pack_bf16(x[1].x, x[1].y));
      *reinterpret_cast<uint2*>(p + u.j) = make_uint2(pack_bf16(y[0].x, y[0].y), pack_bf16(y[1].x, y[1].y));
    } else {
      *reinterpret_cast<uint4*>(p + u.i) = make_uint4(pack_bf16(x[0].x, y[0].x), pack_bf16(x[0].y, y[0].y), pack_bf16(x[1].x, y[1].x),
                                                      pack_bf16(x[1].y, y[1].y));
    }
  }
};

__device__ __forceinline__ int64_t position(const RotaryParams& p, int64_t b, int64_t t) {
  int64_t pos = p.positions != nullptr ? p.positions[b * p.pos_stride + t] : p.start + t;
  if (p.wrap > 0) {
    pos %= p.wrap;
    if (pos < 0) pos += p.wrap;
  }
  return pos;
}
__device__ __forceinline__ float2 turn(const RotaryParams& p, int64_t pos, int pair) {  // cosine and sine, of the results' size
  const uint64_t t = (uint64_t)pos * p.turns[pair];
  float c, s;
  sincospif((float)(int32_t)(t >> 32) * 0x1p-31f, &s, &c);
  return make_float2(c * p.size, s * p.sign * p.size);
}
template <int LANES>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// NORM: the norm before the rotation.  BWD (with NORM): its gradient.
template <typename T, int V, int NU, int LANES, bool HALF, bool NORM, bool BWD>
__global__ void __launch_bounds__(ROT_THREADS, rotary_resident(sizeof(T) == 4, NORM, BWD))
    ttt_rotary_kernel(const RotaryParams p) {
  constexpr int H = V == 1 ? 1 : V / 2;  // pairs of pairs
  using Io = Pairs<T, V, HALF>;
  using Un = Unit<V, HALF>;
  constexpr int groups = ROT_THREADS / LANES;
  const int tid = threadIdx.x, sub = tid & (LANES - 1);
  const int r_lo = (int)blockIdx.y * p.rows_each, r_hi = min(p.heads[0] + p.heads[1], r_lo + p.rows_each);
  const float inv_f = 1.f / p.F;
  F2 wx[NORM ? 2 : 1][NU][H], wy[NORM ? 2 : 1][NU][H], dx[BWD ? 2 : 1][NU][H], dy[BWD ? 2 : 1][NU][H];
  if constexpr (NORM) {
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int n = 0; n < NU; ++n) {
        const Un u(sub + LANES * n, p.F, p.rdim);
#pragma unroll
        for (int k = 0; k < H; ++k) wx[m][n][k] = wy[m][n][k] = f2(1.f);
        if (u.live && p.w[m] != nullptr) {
          if constexpr (V == 1) {
            wx[m][n][0].x = ld_as_float<T>(p.w[m], u.i);
            wy[m][n][0].x = ld_as_float<T>(p.w[m], u.j);
          } else {
            float e[8];
#pragma unroll
            for (int k = 0; k < 4; ++k) e[k] = ld_as_float<T>(p.w[m], u.i + k), e[4 + k] = ld_as_float<T>(p.w[m], u.j + k);
            if constexpr (HALF) {
              wx[m][n][0] = f2(e[0], e[1]), wx[m][n][H - 1] = f2(e[2], e[3]), wy[m][n][0] = f2(e[4], e[5]), wy[m][n][H - 1] = f2(e[6], e[7]);
            } else {
              wx[m][n][0] = f2(e[0], e[2]), wy[m][n][0] = f2(e[1], e[3]), wx[m][n][H - 1] = f2(e[4], e[6]), wy[m][n][H - 1] = f2(e[5], e[7]);
            }
          }
        }
      }
  }
  if constexpr (BWD) {
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int n = 0; n < NU; ++n)
#pragma unroll
        for (int k = 0; k < H; ++k) dx[m][n][k] = dy[m][n][k] = f2(0.f);
  }
  // whole groups of a warp take part in its shuffles to the end: a group without a token works on the last one and stores nothing
  for (int64_t first = (int64_t)blockIdx.x * groups; first < p.tokens; first += (int64_t)gridDim.x * groups) {
    const bool has = first + tid / LANES < p.tokens;
    const int64_t token = has ? first + tid / LANES : p.tokens - 1;
    const int64_t b = token / p.T, t = token - b * p.T;
    F2 c[NU][H], s[NU][H];
    const int64_t pos = p.rdim > 0 ? position(p, b, t) : 0;
#pragma unroll
    for (int n = 0; n < NU; ++n) {
      const Un u(sub + LANES * n, p.F, p.rdim);
#pragma unroll
      for (int k = 0; k < H; ++k) {
        c[n][k] = f2(1.f);
        s[n][k] = f2(0.f);
        if (u.pair >= 0) {
          const float2 e = turn(p, pos, u.pair + 2 * k), f = V == 1 ? e : turn(p, pos, u.pair + 2 * k + 1);
          c[n][k] = f2(e.x, f.x);
          s[n][k] = f2(e.y, f.y);
        }
      }
    }
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      const int off = m ? p.heads[0] : 0, h_lo = max(r_lo - off, 0), h_hi = min(r_hi - off, p.heads[m]);
      if (h_lo >= h_hi) continue;
      const T* src = static_cast<const T*>(p.x[m]) + (b * p.xs[m][0] + h_lo * p.xs[m][1] + t * p.xs[m][2]);
      const T* grd = BWD ? static_cast<const T*>(p.g[m]) + (b * p.gs[m][0] + h_lo * p.gs[m][1] + t * p.gs[m][2]) : nullptr;
      T* dst = static_cast<T*>(p.y[m]) + (b * p.ys[m][0] + h_lo * p.ys[m][1] + t * p.ys[m][2]);
      auto rows = [&](auto count) {  // so many rows, all of them on their way before the first is worked on
        constexpr int ROWS = decltype(count)::value;
        Io in[ROWS][NU];
        [[maybe_unused]] Io grad[BWD ? ROWS : 1][NU];
#pragma unroll
        for (int q = 0; q < ROWS; ++q) {
#pragma unroll
          for (int n = 0; n < NU; ++n) {
            const Un u(sub + LANES * n, p.F, p.rdim);
            if (u.live) in[q][n].load(src, u);
            if constexpr (BWD) {
              if (u.live) grad[q][n].load(grd, u);
            }
          }
          src += p.xs[m][1];
          if constexpr (BWD) grd += p.gs[m][1];
        }
#pragma unroll
        for (int q = 0; q < ROWS; ++q) {
          {
            F2 x[NU][H], y[NU][H], sq = f2(0.f);
#pragma unroll
            for (int n = 0; n < NU; ++n) {
              const Un u(sub + LANES * n, p.F, p.rdim);
#pragma unroll
              for (int k = 0; k < H; ++k) x[n][k] = y[n][k] = f2(0.f);
              if (u.live) in[q][n].unpack(x[n], y[n]);
              if constexpr (NORM) {
#pragma unroll
                for (int k = 0; k < H; ++k) sq = f2fma(x[n][k], x[n][k], f2fma(y[n][k], y[n][k], sq));
              }
            }
            [[maybe_unused]] float r = 1.f;
            if constexpr (NORM) r = rsqrtf(group_sum<LANES>(f2hsum(sq)) * inv_f + p.eps);
            if constexpr (!BWD) {
#pragma unroll
              for (int n = 0; n < NU; ++n) {
                const Un u(sub + LANES * n, p.F, p.rdim);
#pragma unroll
                for (int k = 0; k < H; ++k) {
                  if constexpr (NORM) {
                    x[n][k] = f2mul(x[n][k], f2mul(wx[m][n][k], f2(r)));
                    y[n][k] = f2mul(y[n][k], f2mul(wy[m][n][k], f2(r)));
                  }
                  const F2 a = f2fma(x[n][k], c[n][k], f2neg(f2mul(y[n][k], s[n][k])));
                  y[n][k] = f2fma(y[n][k], c[n][k], f2mul(x[n][k], s[n][k]));
                  x[n][k] = a;
                }
                if (u.live && has) Io::store(dst, u, x[n], y[n]);
              }
            } else {
              F2 gx[NU][H], gy[NU][H], dot = f2(0.f);
#pragma unroll
              for (int n = 0; n < NU; ++n) {
                const Un u(sub + LANES * n, p.F, p.rdim);
#pragma unroll
                for (int k = 0; k < H; ++k) gx[n][k] = gy[n][k] = f2(0.f);
                if (u.live && has) grad[q][n].unpack(gx[n], gy[n]);
#pragma unroll
                for (int k = 0; k < H; ++k) {
                  const F2 a = f2fma(gx[n][k], c[n][k], f2neg(f2mul(gy[n][k], s[n][k])));
                  const F2 e = f2fma(gy[n][k], c[n][k], f2mul(gx[n][k], s[n][k]));
                  const F2 px = f2mul(a, x[n][k]), py = f2mul(e, y[n][k]);
                  dx[m][n][k] = f2fma(px, f2(r), dx[m][n][k]);
                  dy[m][n][k] = f2fma(py, f2(r), dy[m][n][k]);
                  dot = f2fma(px, wx[m][n][k], f2fma(py, wy[m][n][k], dot));
                  gx[n][k] = f2mul(a, wx[m][n][k]);
                  gy[n][k] = f2mul(e, wy[m][n][k]);
                }
              }
              const float f = -group_sum<LANES>(f2hsum(dot)) * inv_f * r * r * r;
#pragma unroll
              for (int n = 0; n < NU; ++n) {
                const Un u(sub + LANES * n, p.F, p.rdim);
#pragma unroll
                for (int k = 0; k < H; ++k) {
                  gx[n][k] = f2fma(gx[n][k], f2(r), f2mul(x[n][k], f2(f)));
                  gy[n][k] = f2fma(gy[n][k], f2(r), f2mul(y[n][k], f2(f)));
                }
                if (u.live && has) Io::store(dst, u, gx[n], gy[n]);
              }
            }
          }
          dst += p.ys[m][1];
        }
      };
      int h = h_lo;
      for (; h + ROT_ROWS <= h_hi; h += ROT_ROWS) rows(std::integral_constant<int, ROT_ROWS>{});
      for (; h < h_hi; ++h) rows(std::integral_constant<int, 1>{});
    }
  }
  if constexpr (BWD) {  // this block's share of the weights' gradients, in a fixed order: groups of a warp, warps, blocks
    if (p.partials == nullptr) return;
    extern __shared__ float rot_smem[];  // [warps][2][F]
    auto put = [&](int m, int at, float v, bool live) {
#pragma unroll
      for (int o = LANES; o < 32; o <<= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
      if (live && (tid & 31) < LANES) rot_smem[((tid >> 5) * 2 + m) * p.F + at] = v;
    };
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int n = 0; n < NU; ++n) {
        const Un u(sub + LANES * n, p.F, p.rdim);
        if constexpr (V == 1) {
          put(m, u.i, dx[m][n][0].x, u.live);
          put(m, u.j, dy[m][n][0].x, u.live);
        } else {
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            put(m, HALF ? u.i + 2 * k : (k ? u.j : u.i), dx[m][n][k].x, u.live);
            put(m, HALF ? u.i + 2 * k + 1 : (k ? u.j : u.i) + 2, dx[m][n][k].y, u.live);
            put(m, HALF ? u.j + 2 * k : (k ? u.j : u.i) + 1, dy[m][n][k].x, u.live);
            put(m, HALF ? u.j + 2 * k + 1 : (k ? u.j : u.i) + 3, dy[m][n][k].y, u.live);
          }
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

// Lanes of a row: with vectors a lane per 8 features, else the whole warp
static int rotary_lanes(int F, bool vec) {
  if (!vec || F > 128) return 32;
  return F > 64 ? 16 : F > 32 ? 8 : 4;
}
// Blocks of tokens (x) and shares of a token's rows (y).  More shares than one where the tokens do not fill the card, or where the
// last round of blocks would run half empty: a share costs its rows and, for the sines, about ROT_SETUP more, and the rounds
// count.  (32768 tokens of 32 rows: 2 shares in 3.5 rounds
// 57.8 us, 4 in 6.9 rounds 52.9, before the loads of a row went out at once.)  The gradient's blocks are no more than are
// resident, since each leaves a row of partial sums.
constexpr int ROT_SETUP = 4;
struct RotaryGrid {
  int x, y, rows_each;
};
static RotaryGrid rotary_grid(int64_t tokens, int rows, int F, bool vec, int resident, bool bwd) {
  RotaryGrid g{};
  const int groups = ROT_THREADS / rotary_lanes(F, vec);
  const int64_t blocks = (tokens + groups - 1) / groups, most = 148 * resident;
  int64_t least = -1;
  for (int each = rows; each >= 1; each = each > ROT_ROWS ? (each - 1) / ROT_ROWS * ROT_ROWS : each > 1 ? 1 : 0) {
    const int64_t shares = (rows + each - 1) / each;
    if (bwd && shares > most) break;
    const int64_t cost = (blocks * shares + most - 1) / most * (each + ROT_SETUP);
    if (least >= 0 && cost >= least) continue;
    least = cost;
    g.rows_each = each;
    g.y = (int)shares;
  }
  const int64_t cap = bwd ? most / g.y : (int64_t)1 << 30;
  g.x = (int)(blocks < cap ? blocks : cap);
  return g;
}
size_t rotary_partial_floats(int64_t tokens, int rows, int F, bool f32) {
  size_t most = 0;
  for (bool vec : {false, true}) {  // (which of them runs depends on addresses)
    if (vec && F % 8 != 0) continue;
    const RotaryGrid g = rotary_grid(tokens, rows, F, vec, rotary_resident(f32, true, true), true);
    const size_t n = (size_t)g.x * g.y * 2 * F;
    if (n > most) most = n;
  }
  return most;
}

template <typename T, int V, int NU, int LANES, bool HALF>
static cudaError_t launch_rot(RotaryParams p, bool norm, bool bwd, cudaStream_t st) {
  const RotaryGrid g = rotary_grid(p.tokens, p.heads[0] + p.heads[1], p.F, V == 4, rotary_resident(sizeof(T) == 4, norm, bwd), bwd);
  p.rows_each = g.rows_each;
  const dim3 grid(g.x, g.y);
  const size_t smem = bwd ? (ROT_THREADS / 32) * 2 * p.F * sizeof(float) : 0;
  if (!norm) ttt_rotary_kernel<T, V, NU, LANES, HALF, false, false><<<grid, ROT_THREADS, 0, st>>>(p);
  else if (!bwd) ttt_rotary_kernel<T, V, NU, LANES, HALF, true, false><<<grid, ROT_THREADS, 0, st>>>(p);
  else ttt_rotary_kernel<T, V, NU, LANES, HALF, true, true><<<grid, ROT_THREADS, smem, st>>>(p);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess || !bwd || p.partials == nullptr) return e;
  ttt_rotary_reduce_kernel<T><<<(2 * p.F + 7) / 8, 256, 0, st>>>(p.partials, g.x * g.y, p.F, static_cast<T*>(p.dw[0]),
                                                                static_cast<T*>(p.dw[1]));
  return cudaGetLastError();
}
template <typename T, bool HALF>
static cudaError_t launch_rot_t(const RotaryParams& p, bool vec, bool norm, bool bwd, cudaStream_t st) {
  if (!vec) return launch_rot<T, 1, 4, 32, HALF>(p, norm, bwd, st);
  switch (rotary_lanes(p.F, true)) {
    case 4: return launch_rot<T, 4, 1, 4, HALF>(p, norm, bwd, st);
    case 8: return launch_rot<T, 4, 1, 8, HALF>(p, norm, bwd, st);
    case 16: return launch_rot<T, 4, 1, 16, HALF>(p, norm, bwd, st);
    default: return launch_rot<T, 4, 1, 32, HALF>(p, norm, bwd, st);
  }
}
cudaError_t launch_rotary(int dtype, const RotaryParams& p, bool vec, bool half, bool norm, bool bwd, cudaStream_t st) {
  if (half) return dtype == 1 ? launch_rot_t<__nv_bfloat16, true>(p, vec, norm, bwd, st) : launch_rot_t<float, true>(p, vec, norm, bwd, st);
  return dtype == 1 ? launch_rot_t<__nv_bfloat16, false>(p, vec, norm, bwd, st) : launch_rot_t<float, false>(p, vec, norm, bwd, st);
}

}  // namespace ttt
