// Gated linear recurrence, a step of 1 to 16 tokens against the resident state (definitions: ttt_gated.cuh): token-by-token
// generation.  Bound by reading and writing the float32 state once (32 KB per stream of 64 features), or by the launch:
// 2048 streams 13 us (5.2 TB/s, 0.8 of a copy), 96 streams 4 us.
//
// A CTA of four warps per stream.  Every thread holds four columns of the state's rows kg, kg + GROUPS, ...; a token is a
// multiply-add per element for the state and one for the output, whose partial sums over the rows meet once, behind the last
// token, so that the tokens follow one another without a barrier.
#include "ttt_kernels.h"
#include "ttt_common.cuh"

namespace ttt {

constexpr int GS_THREADS = 128, GS_TOKENS = 16;

template <typename T, int F>
__global__ void __launch_bounds__(GS_THREADS) ttt_gated_step_kernel(const GatedStepParams p) {
  constexpr int QUADS = F / 4, GROUPS = GS_THREADS / QUADS, ROWS = F / GROUPS;
  __shared__ float qs[GS_TOKENS][F], ks[GS_TOKENS][F], vs[GS_TOKENS][F], ga[GS_TOKENS];
  __shared__ float4 part[GS_TOKENS][GS_THREADS / 32][QUADS];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, quad = tid % QUADS, kg = tid / QUADS;
  const long stream = blockIdx.x;
  const long b = stream / p.H, h = stream - b * p.H;
  float4 w[ROWS];
  const float4* src = reinterpret_cast<const float4*>(p.w) + stream * (F * QUADS);
#pragma unroll
  for (int r = 0; r < ROWS; ++r) w[r] = p.w != nullptr ? src[(kg + GROUPS * r) * QUADS + quad] : make_float4(0.f, 0.f, 0.f, 0.f);
  for (int e = tid; e < p.R * F; e += GS_THREADS) {
    const int t = e / F, f = e - t * F;
    const float beta = p.beta != nullptr ? p.beta[stream * p.R + t] : 1.f;
    qs[t][f] = ld_as_float<T>(p.q, (size_t)(b * p.sq[0] + h * p.sq[1] + t * p.sq[2] + f));
    ks[t][f] = beta * ld_as_float<T>(p.k, (size_t)(b * p.sk[0] + h * p.sk[1] + t * p.sk[2] + f));
    vs[t][f] = ld_as_float<T>(p.v, (size_t)(b * p.sv[0] + h * p.sv[1] + t * p.sv[2] + f));
  }
  if (tid < p.R) ga[tid] = expf(p.g[stream * p.R + tid]);
  __syncthreads();
  for (int t = 0; t < p.R; ++t) {
    const float a = ga[t];
    const float4 v = *reinterpret_cast<const float4*>(&vs[t][4 * quad]);
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      const float k = ks[t][kg + GROUPS * r], q = qs[t][kg + GROUPS * r];
      w[r] = make_float4(fmaf(k, v.x, a * w[r].x), fmaf(k, v.y, a * w[r].y), fmaf(k, v.z, a * w[r].z), fmaf(k, v.w, a * w[r].w));
      o = make_float4(fmaf(q, w[r].x, o.x), fmaf(q, w[r].y, o.y), fmaf(q, w[r].z, o.z), fmaf(q, w[r].w, o.w));
    }
#pragma unroll
    for (int x = QUADS; x < 32; x <<= 1) {
      o.x += __shfl_xor_sync(0xffffffffu, o.x, x);
      o.y += __shfl_xor_sync(0xffffffffu, o.y, x);
      o.z += __shfl_xor_sync(0xffffffffu, o.z, x);
      o.w += __shfl_xor_sync(0xffffffffu, o.w, x);
    }
    if (lane < QUADS) part[t][warp][quad] = o;
  }
  float4* dst = reinterpret_cast<float4*>(p.w_out) + stream * (F * QUADS);
#pragma unroll
  for (int r = 0; r < ROWS; ++r) dst[(kg + GROUPS * r) * QUADS + quad] = w[r];
  __syncthreads();
  for (int e = tid; e < p.R * F; e += GS_THREADS) {
    const int t = e / F, f = e - t * F;
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < GS_THREADS / 32; ++k) s += reinterpret_cast<const float*>(&part[t][k][0])[f];
    st_from_float<T>(p.out, (size_t)stream * p.R * F + e, s);
  }
}

cudaError_t launch_gated_step(int dtype, int F, const GatedStepParams& p, int nstreams, cudaStream_t st) {
  if (F == 64 && dtype == 1) ttt_gated_step_kernel<__nv_bfloat16, 64><<<nstreams, GS_THREADS, 0, st>>>(p);
  else if (F == 64) ttt_gated_step_kernel<float, 64><<<nstreams, GS_THREADS, 0, st>>>(p);
  else if (dtype == 1) ttt_gated_step_kernel<__nv_bfloat16, 32><<<nstreams, GS_THREADS, 0, st>>>(p);
  else ttt_gated_step_kernel<float, 32><<<nstreams, GS_THREADS, 0, st>>>(p);
  return cudaGetLastError();
}

}  // namespace ttt
