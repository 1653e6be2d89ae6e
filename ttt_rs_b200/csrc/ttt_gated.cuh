// Building blocks of the gated linear recurrence's kernels (ttt_gated_fwd.cu, ttt_gated_bwd.cu).
//
//   W_t = a_t W_{t-1} + beta_t k_t^T v_t,   o_t = q_t W_t,   a_t = exp(g_t)          (W is F x F, per (batch, head) stream)
//
// Tokens are taken in chunks of GC = 64.  With G_i = sum of g over the chunk up to and including token i and W the state
// before the chunk,
//   o_i  = e^{G_i} q_i W + sum_{j <= i} e^{G_i - G_j} beta_j (q_i . k_j) v_j
//   W'   = e^{G_end} W + sum_j (e^{G_end - G_j} beta_j k_j)^T v_j
// so everything but one product per chunk is a matrix product of 64-row tiles, and no exponent is ever positive for g <= 0:
// decays are formed as exponentials of differences, never as quotients.  The sums G are taken in 64 bits and carried as two
// floats, because a decay of zero (g = -inf: a new sequence begins) counts as one of 2^-160 (zero in float32), after which G is
// large and its differences would keep few digits.
//
// Operands.  bf16 inputs go to the tensor cores as they are.  What a float32 result depends on (the state, the gradients of the
// gates) must not be rounded to bf16 on the way: the state and the scaled keys enter products as two bf16 planes (16 bits of
// mantissa: 2^-17 of a term at most).  float32 inputs are carried as three planes throughout, as in the other float32 kernels.
#pragma once

#include "ttt_common.cuh"

namespace ttt {

constexpr int GC = 64;            // tokens per chunk
constexpr int GATED_WARPS = 4;    // warps that share the rows of a chunk, 16 each
constexpr float GATED_ZERO = -160.f;  // log2 of a decay that is zero

template <>
__device__ __forceinline__ Pk<2> split_pack<2>(float x, float y) {
  Pk<2> r;
  r.p[0] = pack_bf16(x, y);
  r.p[1] = pack_bf16(x - bf16_lo(r.p[0]), y - bf16_hi(r.p[0]));
  return r;
}

// A bf16 tile of rows of F elements (128 or 64 bytes) in the swizzle of TMA: rows 0..63, any multiple of 8 columns
template <int F>
struct GTile {
  static constexpr uint32_t ROW = F * 2, BYTES = GC * ROW, STATE_BYTES = F * ROW;
  static __device__ __forceinline__ uint32_t off(int row, int col) {
    const int x = F == 64 ? (row & 7) : ((row >> 1) & 3);
    return (uint32_t)(row * (int)ROW + (((col >> 3) ^ x) << 4) + ((col & 7) << 1));
  }
  // lane addresses of ldmatrix.x4; row0 and col0 multiples of 8
  // A operand [16 rows of the product][16 of its K], stored [row][k]
  static __device__ __forceinline__ uint32_t a_mk(int lane, int row0, int k0) {
    return off(row0 + (lane & 7) + ((lane >> 3) & 1) * 8, k0 + (lane >> 4) * 8);
  }
  // the same operand stored [k][row] (with .trans)
  static __device__ __forceinline__ uint32_t a_km(int lane, int row0, int k0) {
    return off(k0 + (lane & 7) + (lane >> 4) * 8, row0 + ((lane >> 3) & 1) * 8);
  }
  // B operand, two tiles of 8 of the product's columns, stored [n][k]
  static __device__ __forceinline__ uint32_t b_nk(int lane, int n0, int k0) {
    return off(n0 + (lane & 7) + (lane >> 4) * 8, k0 + ((lane >> 3) & 1) * 8);
  }
  // the same stored [k][n] (with .trans)
  static __device__ __forceinline__ uint32_t b_kn(int lane, int n0, int k0) {
    return off(k0 + (lane & 7) + ((lane >> 3) & 1) * 8, n0 + (lane >> 4) * 8);
  }
};

// c0 += a . b[0..1], c1 += a . b[2..3]: the products of planes whose weight is at least 2^-16 of the leading one
template <int NA, int NB>
__device__ __forceinline__ void mma_planes(float (&c0)[4], float (&c1)[4], const Pk<NA> (&a)[4], const Pk<NB> (&b)[4]) {
  if constexpr (NA == 3 && NB == 3) {
    const Pk<3> b0[2] = {b[0], b[1]}, b1[2] = {b[2], b[3]};
    mma_np2<3>(c0, a, b0, c1, a, b1);
  } else {
    static_assert(NA * NB <= 2, "planes");
#pragma unroll
    for (int i = NA * NB - 1; i >= 0; --i) {  // the small plane first
      const int pa = NA == 2 ? i : 0, pb = NB == 2 ? i : 0;
      mma_bf16(c0, a[0].p[pa], a[1].p[pa], a[2].p[pa], a[3].p[pa], b[0].p[pb], b[1].p[pb]);
      mma_bf16(c1, a[0].p[pa], a[1].p[pa], a[2].p[pa], a[3].p[pa], b[2].p[pb], b[3].p[pb]);
    }
  }
}

template <int NP>
__device__ __forceinline__ float pk_lo(const Pk<NP>& v) {
  float s = 0.f;
#pragma unroll
  for (int i = NP - 1; i >= 0; --i) s += bf16_lo(v.p[i]);
  return s;
}
template <int NP>
__device__ __forceinline__ float pk_hi(const Pk<NP>& v) {
  float s = 0.f;
#pragma unroll
  for (int i = NP - 1; i >= 0; --i) s += bf16_hi(v.p[i]);
  return s;
}
// an A fragment (lane 4g + t: columns 2t, 2t+1 in [0], [1]; 2t+8, 2t+9 in [2], [3]) with its columns scaled
template <int NO, int NI>
__device__ __forceinline__ void scale_a_cols(Pk<NO> (&o)[4], const Pk<NI> (&a)[4], float2 lo, float2 hi) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 s = i < 2 ? lo : hi;
    o[i] = split_pack<NO>(pk_lo(a[i]) * s.x, pk_hi(a[i]) * s.y);
  }
}

// The gates of a chunk, for all warps of a block
struct ChunkGates {
  float hi[GC], lo[GC];  // G_i in units of log2, in two floats
  float from[GC];        // e^{G_i}: what is left at token i of the state before the chunk
  float to[GC];          // e^{G_end - G_i}: what is left of token i after the chunk
  float beta[GC];
  float all;             // e^{G_end}
  float pad[3];
};
__device__ __forceinline__ float gated_decay(const ChunkGates& s, int i, int j) {  // e^{G_i - G_j}
  return exp2f((s.hi[i] - s.hi[j]) + (s.lo[i] - s.lo[j]));
}
// One warp; lane l brings tokens 2l and 2l + 1 of the chunk.  Tokens behind the sequence: g = 0, beta = 0.
__device__ __forceinline__ void make_chunk_gates(ChunkGates& s, int lane, float2 g, float2 beta) {
  auto log2_of = [](float x) {
    const double v = (double)x * 1.4426950408889634;
    return v < (double)GATED_ZERO ? (double)GATED_ZERO : v;  // (a NaN stays one)
  };
  const double g0 = log2_of(g.x), g1 = log2_of(g.y);
  double sum = g0 + g1;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const double up = __shfl_up_sync(0xffffffffu, sum, o);
    if (lane >= o) sum += up;
  }
  const double end = __shfl_sync(0xffffffffu, sum, 31), G0 = sum - g1, G1 = sum;
  const float h0 = (float)G0, h1 = (float)G1;
  *reinterpret_cast<float2*>(&s.hi[2 * lane]) = make_float2(h0, h1);
  *reinterpret_cast<float2*>(&s.lo[2 * lane]) = make_float2((float)(G0 - h0), (float)(G1 - h1));
  *reinterpret_cast<float2*>(&s.from[2 * lane]) = make_float2(exp2f((float)G0), exp2f((float)G1));
  *reinterpret_cast<float2*>(&s.to[2 * lane]) = make_float2(exp2f((float)(end - G0)), exp2f((float)(end - G1)));
  *reinterpret_cast<float2*>(&s.beta[2 * lane]) = beta;
  if (lane == 0) s.all = exp2f((float)end);
}
// what lane `lane` brings for the chunk that starts at token t0
__device__ __forceinline__ float2 load_gates(const float* x, int t0, int T, int lane, float none) {
  const int t = t0 + 2 * lane;
  float2 v = make_float2(0.f, 0.f);
  if (t < T) v.x = x != nullptr ? x[t] : none;
  if (t + 1 < T) v.y = x != nullptr ? x[t + 1] : none;
  return v;
}

// Four registers of the four lanes of a quad, turned: lane t gets register t of lanes 0..3, in their order
__device__ __forceinline__ void quad_transpose(uint32_t (&r)[4], int lane) {
  const bool odd = lane & 1, high = lane & 2;
#pragma unroll
  for (int k = 0; k < 4; k += 2) {
    const uint32_t got = __shfl_xor_sync(0xffffffffu, odd ? r[k] : r[k + 1], 1);
    if (odd) r[k] = got;
    else r[k + 1] = got;
  }
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const uint32_t got = __shfl_xor_sync(0xffffffffu, high ? r[k] : r[k + 2], 2);
    if (high) r[k] = got;
    else r[k + 2] = got;
  }
}
// Accumulators of 16 rows x F columns to global rows base[row * F], rows below `rows`.  bf16: 64 contiguous bytes per row and
// store (four lanes of 16), float32: 32.
template <typename T, int F>
__device__ __forceinline__ void store_rows(T* base, int row0, int rows, const float (&c)[F / 8][4], int lane) {
  const int g = lane >> 2, t = lane & 3;
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const int row = row0 + g + 8 * half;
    if constexpr (sizeof(T) == 2) {
#pragma unroll
      for (int n = 0; n < F / 8; n += 4) {
        uint32_t r[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) r[k] = pack_bf16(c[n + k][2 * half], c[n + k][2 * half + 1]);
        quad_transpose(r, lane);
        if (row < rows) *reinterpret_cast<uint4*>(base + (size_t)row * F + 8 * (n + t)) = make_uint4(r[0], r[1], r[2], r[3]);
      }
    } else if (row < rows) {
#pragma unroll
      for (int n = 0; n < F / 8; ++n)
        *reinterpret_cast<float2*>(base + (size_t)row * F + 8 * n + 2 * t) = make_float2(c[n][2 * half], c[n][2 * half + 1]);
    }
  }
}

// float32 rows as TMA lays them ([rows][F], no swizzle) -> three planes of bf16 tiles
template <int F>
__device__ __forceinline__ void split_rows(uint32_t planes, uint32_t plane_stride, const float* src, int rows, int tid, int threads) {
  constexpr int Q = F / 4;
  for (int e = tid; e < rows * Q; e += threads) {
    const int row = e / Q, col = 4 * (e - row * Q);
    const float4 v = *reinterpret_cast<const float4*>(src + 4 * e);
    const Pk<3> a = split_pack<3>(v.x, v.y), b = split_pack<3>(v.z, v.w);
#pragma unroll
    for (int i = 0; i < 3; ++i)
      asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(planes + i * plane_stride + GTile<F>::off(row, col)), "r"(a.p[i]),
                   "r"(b.p[i])
                   : "memory");
  }
}
__device__ __forceinline__ void st_shared_b32(uint32_t addr, uint32_t v) {
  asm volatile("st.shared.b32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}
__device__ __forceinline__ uint32_t ld_shared_b32(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(addr));
  return v;
}

// 4-D TMA load: features, tokens, heads, batch
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* tm, int y, int z, int w, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
      "l"(tm), "r"(0), "r"(y), "r"(z), "r"(w), "r"(bar)
      : "memory");
}

// How the F x F state lies in the registers of four warps: warp w holds rows 16 (w % SLABS).. and the columns of its part
template <int F>
struct StateShare {
  static constexpr int SLABS = F / 16, PARTS = GATED_WARPS / SLABS, COLS = F / PARTS, NT = COLS / 8;
};

// A warp's share of the state (rows row0.., columns col0..) as NP bf16 planes in the tile layout: to shared memory (planes
// STATE_BYTES apart) and, where `image` is given, the same bytes to global memory.
template <int F, int NP>
__device__ __forceinline__ void put_state(const float (&w)[StateShare<F>::NT][4], int row0, int col0, uint32_t smem, uint8_t* image,
                                          int lane) {
  using S = StateShare<F>;
  const int g = lane >> 2, t = lane & 3;
  auto put = [&](uint32_t (&r)[4], int plane, int row, int col) {
    quad_transpose(r, lane);
    const uint32_t at = plane * GTile<F>::STATE_BYTES + GTile<F>::off(row, col);
    if (smem != 0)
      asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(smem + at), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]) : "memory");
    if (image != nullptr) *reinterpret_cast<uint4*>(image + at) = make_uint4(r[0], r[1], r[2], r[3]);
  };
  if constexpr (S::NT % 4 == 0) {
#pragma unroll
    for (int half = 0; half < 2; ++half)
#pragma unroll
      for (int n = 0; n < S::NT; n += 4) {
        Pk<NP> v[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = split_pack<NP>(w[n + k][2 * half], w[n + k][2 * half + 1]);
#pragma unroll
        for (int i = 0; i < NP; ++i) {
          uint32_t r[4] = {v[0].p[i], v[1].p[i], v[2].p[i], v[3].p[i]};
          put(r, i, row0 + g + 8 * half, col0 + 8 * (n + t));
        }
      }
  } else {
    static_assert(S::NT == 2, "two tiles of eight columns");
    Pk<NP> v[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = split_pack<NP>(w[k & 1][k & 2], w[k & 1][(k & 2) + 1]);
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      uint32_t r[4] = {v[0].p[i], v[1].p[i], v[2].p[i], v[3].p[i]};
      put(r, i, row0 + g + 8 * (t >> 1), col0 + 8 * (t & 1));
    }
  }
}
// The same share to and from a float32 matrix [F][F]
template <int F>
__device__ __forceinline__ void store_state(float* m, const float (&w)[StateShare<F>::NT][4], int row0, int col0, int lane) {
#pragma unroll
  for (int n = 0; n < StateShare<F>::NT; ++n)
#pragma unroll
    for (int half = 0; half < 2; ++half)
      *reinterpret_cast<float2*>(m + (size_t)(row0 + (lane >> 2) + 8 * half) * F + col0 + 8 * n + 2 * (lane & 3)) =
          make_float2(w[n][2 * half], w[n][2 * half + 1]);
}
template <int F>
__device__ __forceinline__ void load_state(float (&w)[StateShare<F>::NT][4], const float* m, int row0, int col0, int lane) {
#pragma unroll
  for (int n = 0; n < StateShare<F>::NT; ++n)
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      float2 v = make_float2(0.f, 0.f);
      if (m != nullptr)
        v = *reinterpret_cast<const float2*>(m + (size_t)(row0 + (lane >> 2) + 8 * half) * F + col0 + 8 * n + 2 * (lane & 3));
      w[n][2 * half] = v.x;
      w[n][2 * half + 1] = v.y;
    }
}

}  // namespace ttt
