// Vectors of V neighbouring channels between memory (T: float or bf16) and float32 pairs in registers.
#pragma once

#include "ttt_common.cuh"
#include "ttt_kernels.h"

namespace ttt {

template <int BYTES>
struct Word;
template <>
struct Word<2> {
  using type = uint16_t;
};
template <>
struct Word<4> {
  using type = uint32_t;
};
template <>
struct Word<8> {
  using type = uint2;
};
template <>
struct Word<16> {
  using type = uint4;
};

// V channels as they lie in memory (16 bytes at most) and as float32 pairs; V = 1 leaves the second half of its pair at 0.
template <typename T, int V>
struct Chan {
  static constexpr int P = (V + 1) / 2;
  using W = typename Word<V * (int)sizeof(T)>::type;
  W w;
  __device__ __forceinline__ void load(const T* p) { w = *reinterpret_cast<const W*>(p); }
  __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<W*>(p) = w; }
  __device__ __forceinline__ void zero() { w = W{}; }
  __device__ __forceinline__ void unpack(F2 (&x)[P]) const {
    if constexpr (sizeof(T) == 4) {
      if constexpr (V == 4) x[0] = f2(__uint_as_float(w.x), __uint_as_float(w.y)), x[1] = f2(__uint_as_float(w.z), __uint_as_float(w.w));
      else if constexpr (V == 2) x[0] = f2(__uint_as_float(w.x), __uint_as_float(w.y));
      else x[0] = f2(__uint_as_float(w), 0.f);
    } else {
      if constexpr (V == 8) {
        x[0] = f2(bf16_lo(w.x), bf16_hi(w.x)), x[1] = f2(bf16_lo(w.y), bf16_hi(w.y));
        x[2] = f2(bf16_lo(w.z), bf16_hi(w.z)), x[3] = f2(bf16_lo(w.w), bf16_hi(w.w));
      } else if constexpr (V == 4) x[0] = f2(bf16_lo(w.x), bf16_hi(w.x)), x[1] = f2(bf16_lo(w.y), bf16_hi(w.y));
      else if constexpr (V == 2) x[0] = f2(bf16_lo(w), bf16_hi(w));
      else x[0] = f2(bf16_lo((uint32_t)w), 0.f);
    }
  }
  __device__ __forceinline__ void pack(const F2 (&x)[P]) {
    if constexpr (sizeof(T) == 4) {
      if constexpr (V == 4) w = make_uint4(__float_as_uint(x[0].x), __float_as_uint(x[0].y), __float_as_uint(x[1].x), __float_as_uint(x[1].y));
      else if constexpr (V == 2) w = make_uint2(__float_as_uint(x[0].x), __float_as_uint(x[0].y));
      else w = __float_as_uint(x[0].x);
    } else {
      if constexpr (V == 8) w = make_uint4(pack_bf16(x[0].x, x[0].y), pack_bf16(x[1].x, x[1].y), pack_bf16(x[2].x, x[2].y), pack_bf16(x[3].x, x[3].y));
      else if constexpr (V == 4) w = make_uint2(pack_bf16(x[0].x, x[0].y), pack_bf16(x[1].x, x[1].y));
      else if constexpr (V == 2) w = pack_bf16(x[0].x, x[0].y);
      else w = (uint16_t)(pack_bf16(x[0].x, 0.f) & 0xffffu);
    }
  }
};

// 2^x and 1 / x, approximate (2 and 1 units in the last place), results below 2^-126 as zero
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ F2 ex2(F2 x) { return f2(ex2(x.x), ex2(x.y)); }
__device__ __forceinline__ float rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

// Activations and their derivatives.  (1 + exp(-v) that overflows has a reciprocal of 0, as the limit is.)
__device__ __forceinline__ float sigmoid_of(float v) { return rcp(1.f + ex2(-LOG2E * v)); }
__device__ __forceinline__ float act_of(float v, int act) {
  if (act == ACT_SILU) return v * sigmoid_of(v);
  if (act == ACT_GELU) {
    // v sigmoid(2u): no difference of nearly equal numbers in the negative tail
    const float u = 0.7978845608028654f * v * fmaf(0.044715f * v, v, 1.f);
    return v * sigmoid_of(2.f * u);
  }
  return v;
}
// act(v), and its derivative in `slope`
__device__ __forceinline__ float act_and_slope(float v, int act, float& slope) {
  if (act == ACT_SILU) {
    const float s = sigmoid_of(v), y = v * s;
    slope = fmaf(y, 1.f - s, s);
    return y;
  }
  if (act == ACT_GELU) {
    const float u = 0.7978845608028654f * v * fmaf(0.044715f * v, v, 1.f), s = sigmoid_of(2.f * u), y = v * s;
    // s + 2 k y (1 - s) (1 + 3 c v v), from the left: where v v is beyond float32, y (1 - s) is 0 and must meet no infinity
    const float t = y * (1.f - s);
    slope = fmaf(6.f * 0.044715f * 0.7978845608028654f, t * v * v, fmaf(2.f * 0.7978845608028654f, t, s));
    return y;
  }
  slope = 1.f;
  return v;
}


// Sums over rows [rows][pitch] of blocks' shares, in a fixed order: a block of ROWS_THREADS per 32 columns, a warp per 32nd row.  True in
// the thread that has column *col's sum.
constexpr int ROWS_THREADS = 1024;
__device__ __forceinline__ bool sum_of_rows(const float* partials, int64_t rows, int64_t pitch, int64_t columns, int64_t block, int64_t* col, float* sum) {
  __shared__ float part[ROWS_THREADS / 32][33];
  const int lane = threadIdx.x & 31, share = threadIdx.x >> 5;
  *col = block * 32 + lane;
  float v = 0.f;
  if (*col < columns) {
    const float* at = partials + *col;
#pragma unroll 4
    for (int64_t r = share; r < rows; r += ROWS_THREADS / 32) v += at[r * pitch];
  }
  part[share][lane] = v;
  __syncthreads();
  if (share != 0 || *col >= columns) return false;
#pragma unroll
  for (int k = 1; k < ROWS_THREADS / 32; ++k) v += part[k][lane];
  *sum = v;
  return true;
}

}  // namespace ttt
