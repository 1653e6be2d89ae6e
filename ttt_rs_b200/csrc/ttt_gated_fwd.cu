// Gated linear recurrence, forward (the mathematics and its chunked form: ttt_gated.cuh).
//
// One CTA of four warps per stream (or per segment of one) walks its chunks; warp w owns 16 queries of the chunk and 16 rows of
// the float32 state, both in accumulator layout.  Per chunk, for each block of 16 tokens: their keys against the queries at or
// behind them, the decayed products as the A operand of the product with their values, and the same values, still in registers,
// under the transposed and scaled keys for the state.  The state goes to shared memory once per chunk as the operand of the next
// chunk's q W (double-buffered: one barrier per chunk); the next two chunks are on their way meanwhile (TMA, rows behind the
// sequence read as zeros).
//
// Few streams are cut into segments: a first launch leaves every segment's own state (as if it began with none) and its decay, a
// second one joins them along the sequence, and the third is this kernel with a CTA per segment.
#include "ttt_kernels.h"
#include "ttt_gated.cuh"
#include "ttt_stage.cuh"

namespace ttt {

constexpr int GF_THREADS = 32 * GATED_WARPS;

// STATE: only the state at the end of the segment is wanted (REV: of the gradient's walk, from the last token to the first)
template <typename T, int F, bool STATE>
struct GatedFwdSmem {
  static constexpr bool BF = sizeof(T) == 2;
  static constexpr int NP = BF ? 1 : 3, NIN = STATE ? 2 : 3;
  static constexpr uint32_t PLANE = GTile<F>::BYTES, TILE = NP * PLANE;
  static constexpr uint32_t RAW = GC * F * 4;                                 // float32 rows as they arrive
  static constexpr uint32_t STAGES = BF ? 2 : 1;
  static constexpr uint32_t TILES = 0, RAWS = TILES + STAGES * NIN * TILE;
  static constexpr uint32_t W = RAWS + (BF ? 0 : NIN * RAW);
  static constexpr uint32_t GATES = W + (STATE ? 0 : 2 * NP * GTile<F>::STATE_BYTES);
  static constexpr uint32_t BAR = GATES + 2 * sizeof(ChunkGates), BYTES = BAR + 16 + 1024;  // (1024: the base is aligned by hand)
};

template <typename T, int F, bool SAVE, bool STATE, bool REV>
__global__ void __launch_bounds__(GF_THREADS, sizeof(T) == 2 ? 3 : 1)
    ttt_gated_fwd_kernel(const __grid_constant__ GatedMaps maps, const GatedParams p) {
  using SM = GatedFwdSmem<T, F, STATE>;
  using SH = StateShare<F>;
  constexpr bool BF = SM::BF;
  constexpr int NP = SM::NP, NS = BF ? 2 : 3;  // planes of inputs, of scaled keys
  constexpr int KS = F / 16;
  extern __shared__ uint8_t gated_smem[];
  const uint32_t raw = smem_u32(gated_smem), base = (raw + 1023) & ~1023u;
  uint8_t* const mem = gated_smem + (base - raw);
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5, g = lane >> 2, t4 = lane & 3;
  const int stream = blockIdx.x / p.nseg, seg = blockIdx.x - stream * p.nseg;
  const int c_lo = seg * p.seg_chunks, c_hi = min(p.NC, c_lo + p.seg_chunks), n = c_hi - c_lo;
  const int h = stream % p.H, b = stream / p.H;
  if (STATE && seg == (REV ? 0 : p.nseg - 1)) return;  // nothing follows it
  const uint32_t bar = base + SM::BAR;
  if (tid == 0) {
    mbar_init(bar, 1);
    mbar_init(bar + 8, 1);
    fence_mbar_init();
  }
  __syncthreads();
  auto chunk_of = [&](int i) { return REV ? c_hi - 1 - i : c_lo + i; };
  auto fetch = [&](int i) {  // thread 0
    const int slot = BF ? i & 1 : 0;
    const uint32_t at = bar + 8 * slot, dst = base + (BF ? SM::TILES + slot * SM::NIN * SM::TILE : SM::RAWS);
    constexpr uint32_t bytes = BF ? SM::TILE : SM::RAW;
    mbar_expect_tx(at, SM::NIN * bytes);
#pragma unroll
    for (int m = 0; m < SM::NIN; ++m) tma_load_4d(dst + m * bytes, &maps.m[(STATE ? 1 : 0) + m], chunk_of(i) * GC, h, b, at);
  };
  if (tid == 0) {
    fetch(0);
    if (BF && n > 1) fetch(1);
  }
  const float* gp = p.g + (size_t)stream * p.T;
  const float* bp = p.beta != nullptr ? p.beta + (size_t)stream * p.T : nullptr;
  ChunkGates* const gates = reinterpret_cast<ChunkGates*>(mem + SM::GATES);
  // the gates of walk step i by warp i % 4, a step ahead
  auto make_gates = [&](int i) {
    const int t0 = chunk_of(i) * GC;
    make_chunk_gates(gates[i & 1], lane, load_gates(gp, t0, p.T, lane, 0.f), load_gates(bp, t0, p.T, lane, 1.f));
  };
  if (w == 0) make_gates(0);

  // this warp's share of the state
  const int row0 = 16 * (w % SH::SLABS), part = w / SH::SLABS, col0 = part * SH::COLS;
  float W[SH::NT][4];
  {
    const float* w0 = nullptr;
    if (!STATE) w0 = seg > 0 ? p.seg_state + ((size_t)stream * p.nseg + seg) * F * F : p.w0 != nullptr ? p.w0 + (size_t)stream * F * F : nullptr;
    load_state<F>(W, w0, row0, col0, lane);
  }
  float total = 1.f;  // what is left of the state before the segment after it
  uint8_t* const saved = SAVE ? p.saved + (size_t)stream * p.NC * F * F * 4 : nullptr;
  auto publish = [&](int i) {  // the state before walk step i: operand of its q W, and what the backward reads back
    if constexpr (!STATE) {
      const uint32_t dst = base + SM::W + (i & 1) * NP * GTile<F>::STATE_BYTES;
      put_state<F, NP>(W, row0, col0, dst, lane);
      if (SAVE && i < n) put_fragments<F>(reinterpret_cast<float4*>(saved + (size_t)(c_lo + i) * F * F * 4), W, w, lane);
    }
  };
  publish(0);
  __syncthreads();
  const uint32_t low = GTile<F>::low(lane), high = GTile<F>::high(lane);

  for (int i = 0; i < n; ++i) {
    const int slot = BF ? i & 1 : 0, t0 = chunk_of(i) * GC;
    const bool ahead = w == ((i + 1) & 3) && i + 1 < n;
    float2 g_next, b_next;
    if (ahead) {
      g_next = load_gates(gp, chunk_of(i + 1) * GC, p.T, lane, 0.f);
      b_next = load_gates(bp, chunk_of(i + 1) * GC, p.T, lane, 1.f);
    }
    if (!mbar_wait_bounded(bar + 8 * slot, (BF ? i >> 1 : i) & 1)) {
      if (tid == 0) report_timeout(p.status, 20, (uint32_t)i);
      return;
    }
    const uint32_t tiles = base + SM::TILES + slot * SM::NIN * SM::TILE;
    if constexpr (!BF) {
#pragma unroll
      for (int m = 0; m < SM::NIN; ++m)
        split_rows<F>(tiles + m * SM::TILE, SM::PLANE, reinterpret_cast<const float*>(mem + SM::RAWS + m * SM::RAW), GC, tid, GF_THREADS);
      __syncthreads();
      if (tid == 0 && i + 1 < n) fetch(i + 1);
    }
    const uint32_t tq = tiles, tk = tiles + (STATE ? 0 : SM::TILE), tv = tk + SM::TILE;
    const ChunkGates& cg = gates[i & 1];

    float o[STATE ? 1 : F / 8][4];
    Pk<NP> q[STATE ? 1 : KS][4];
    if constexpr (!STATE) {
      // q_i W, from the start of this warp's block on
      const uint32_t tw = base + SM::W + (i & 1) * NP * GTile<F>::STATE_BYTES;
#pragma unroll
      for (int k = 0; k < KS; ++k) ldsm_np<NP>(q[k], (tq + 16 * w * GTile<F>::ROW + low) ^ (k << 5), SM::PLANE, false);
#pragma unroll
      for (int k = 0; k < F / 8; ++k) o[k][0] = o[k][1] = o[k][2] = o[k][3] = 0.f;
#pragma unroll
      for (int k = 0; k < KS; ++k)
#pragma unroll
        for (int m = 0; m < KS; ++m) {
          Pk<NP> f[4];
          ldsm_np<NP>(f, (tw + 16 * k * GTile<F>::ROW + low) ^ (m << 5), GTile<F>::STATE_BYTES, true);
          mma_planes<NP, NP>(o[2 * m], o[2 * m + 1], q[k], f);
        }
      const float first = cg.starts[w];
#pragma unroll
      for (int k = 0; k < F / 8; ++k) scale_rows(o[k], first, first);
    }
    const float all = cg.all;
    total *= all;
#pragma unroll
    for (int k = 0; k < SH::NT; ++k) scale_rows(W[k], all, all);

#pragma unroll 1
    for (int jt = 0; jt < GC / 16; ++jt) {
      const int j0 = 16 * jt + 2 * t4;
      // queries of this warp against the keys of the block, decayed, as an operand of the inputs' planes
      Pk<NP> a[4];
      const bool here = !STATE && jt <= w;
      if constexpr (!STATE) {
        if (here) {
          float s0[4] = {}, s1[4] = {};
#pragma unroll
          for (int k = 0; k < KS; ++k) {
            Pk<NP> f[4];
            ldsm_np<NP>(f, (tk + 16 * jt * GTile<F>::ROW + high) ^ (k << 5), SM::PLANE, false);
            mma_planes<NP, NP>(s0, s1, q[k], f);
          }
          if (jt < w) {
            const F2 between = f2(cg.blocks[jt][w - 1]);
            scale_cols(s0, f2mul(ld2(&cg.out_b[j0]), between));
            scale_cols(s1, f2mul(ld2(&cg.out_b[j0 + 8]), between));
          } else {
            // what came from before the block, to each of its tokens; then the block itself
            const float ra = cg.into[16 * w + g], rb = cg.into[16 * w + g + 8];
#pragma unroll
            for (int k = 0; k < F / 8; ++k) scale_rows(o[k], ra, rb);
            float d[2][4];
            block_decays<true>(d, cg, w, g, t4);
            const float2 b0 = ld2(&cg.beta[j0]), b1 = ld2(&cg.beta[j0 + 8]);
#pragma unroll
            for (int half = 0; half < 2; ++half) {  // (a select, not a product: what is not there may be infinite)
              s0[2 * half] = d[half][0] > 0.f ? s0[2 * half] * (d[half][0] * b0.x) : 0.f;
              s0[2 * half + 1] = d[half][1] > 0.f ? s0[2 * half + 1] * (d[half][1] * b0.y) : 0.f;
              s1[2 * half] = d[half][2] > 0.f ? s1[2 * half] * (d[half][2] * b1.x) : 0.f;
              s1[2 * half + 1] = d[half][3] > 0.f ? s1[2 * half + 1] * (d[half][3] * b1.y) : 0.f;
            }
          }
          as_operand<NP>(a, s0, s1);
        }
      }
      // keys of the block, transposed: rows of the state
      Pk<NS> kt[4];
      {
        Pk<NP> f[4];
        ldsm_np<NP>(f, (tk + 16 * jt * GTile<F>::ROW + high) ^ (row0 << 1), SM::PLANE, true);
        const float* scale = REV ? cg.from : cg.end_b;  // (REV: what is left at the token of the state before the chunk)
        scale_a_cols<NS, NP>(kt, f, ld2(scale + j0), ld2(scale + j0 + 8));
      }
#pragma unroll
      for (int m = 0; m < KS; ++m) {
        const bool mine = SH::PARTS == 1 || m == part;
        if (!mine && !here) continue;
        Pk<NP> f[4];
        ldsm_np<NP>(f, (tv + 16 * jt * GTile<F>::ROW + low) ^ (m << 5), SM::PLANE, true);
        if constexpr (!STATE) {
          if (here) mma_planes<NP, NP>(o[2 * m], o[2 * m + 1], a, f);
        }
        if (mine) {
          const int at = SH::PARTS == 1 ? 2 * m : 0;
          mma_planes<NS, NP>(W[at], W[at + 1], kt, f);
        }
      }
    }
    if constexpr (!STATE)
      store_rows<T, F>(static_cast<T*>(p.out) + ((size_t)stream * p.T + t0) * F, 16 * w, p.T - t0, o, lane);
    if (i + 1 < n) publish(i + 1);
    if (ahead) make_chunk_gates(gates[(i + 1) & 1], lane, g_next, b_next);
    __syncthreads();  // the tiles and this chunk's state and gates are free, the next one's are there
    if (BF && tid == 0 && i + 2 < n) fetch(i + 2);
  }
  if constexpr (STATE) {
    store_state<F>(p.seg_state + ((size_t)stream * p.nseg + seg) * F * F, W, row0, col0, lane);
    if (tid == 0) p.seg_decay[(size_t)stream * p.nseg + seg] = total;
  } else if (seg == p.nseg - 1) {
    store_state<F>(p.w_out + (size_t)stream * F * F, W, row0, col0, lane);
  }
}

// The segments' own states to the states before them, along the sequence (REV: gradients, from the last segment to the first):
// state[s] <- W_s, W_{s+1} = decay[s] W_s + own[s].  Every thread carries one float4 of a stream's state.
template <int F, bool REV>
__global__ void __launch_bounds__(256) ttt_gated_join_kernel(const GatedParams p) {
  constexpr int Q = F * F / 4;
  const long e = (long)blockIdx.x * 256 + threadIdx.x;
  if (e >= (long)p.nstreams * Q) return;
  const long stream = e / Q;
  const int at = (int)(e - stream * Q);
  float4* s = reinterpret_cast<float4*>(p.seg_state) + stream * p.nseg * Q + at;
  const float* d = p.seg_decay + stream * p.nseg;
  float4 w = make_float4(0.f, 0.f, 0.f, 0.f);
  if (p.w0 != nullptr) w = reinterpret_cast<const float4*>(p.w0)[stream * Q + at];
  for (int k = 0; k < p.nseg; ++k) {
    const int i = REV ? p.nseg - 1 - k : k;
    const float4 own = s[(long)i * Q];
    s[(long)i * Q] = w;
    const float f = d[i];
    w = make_float4(fmaf(f, w.x, own.x), fmaf(f, w.y, own.y), fmaf(f, w.z, own.z), fmaf(f, w.w, own.w));
  }
}

// Streams that do not fill the card are cut until they do.
int gated_segments(int64_t streams, int chunks, bool backward) {
  constexpr int SMS = 148, LEAST = 4;  // (chunks per segment: a segment's states and its second reading must be worth it)
  if (streams >= SMS) return 1;
  const int64_t want = ((backward ? 2 : 3) * SMS) / streams;
  const int64_t most = chunks / LEAST;
  return (int)(want < most ? want : most > 1 ? most : 1);
}

template <typename T, int F, bool SAVE, bool STATE, bool REV>
static cudaError_t launch_one(const GatedMaps& maps, const GatedParams& p, int grid, cudaStream_t st) {
  auto kfn = ttt_gated_fwd_kernel<T, F, SAVE, STATE, REV>;
  constexpr size_t smem = GatedFwdSmem<T, F, STATE>::BYTES;
  static DeviceValue ready;
  int unused;
  cudaError_t e = ready.get(0, &unused, [&](int* v) {
    *v = 0;
    return cudaFuncSetAttribute(kfn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  });
  if (e != cudaSuccess) return e;
  kfn<<<grid, GF_THREADS, smem, st>>>(maps, p);
  return cudaGetLastError();
}

template <typename T, int F>
static cudaError_t launch_gated(const GatedMaps& maps, GatedParams p, bool save, cudaStream_t st) {
  if (p.nseg > 1) {
    cudaError_t e = launch_one<T, F, false, true, false>(maps, p, p.nstreams * p.nseg, st);
    if (e != cudaSuccess) return e;
    ttt_gated_join_kernel<F, false><<<(int)(((long)p.nstreams * (F * F / 4) + 255) / 256), 256, 0, st>>>(p);
    if ((e = cudaGetLastError()) != cudaSuccess) return e;
  }
  if (save) return launch_one<T, F, true, false, false>(maps, p, p.nstreams * p.nseg, st);
  return launch_one<T, F, false, false, false>(maps, p, p.nstreams * p.nseg, st);
}
cudaError_t launch_gated_fwd(int dtype, int F, const GatedMaps& maps, const GatedParams& p, bool save, cudaStream_t st) {
  if (F == 64) return dtype == 1 ? launch_gated<__nv_bfloat16, 64>(maps, p, save, st) : launch_gated<float, 64>(maps, p, save, st);
  return dtype == 1 ? launch_gated<__nv_bfloat16, 32>(maps, p, save, st) : launch_gated<float, 32>(maps, p, save, st);
}

// The gradient's states behind every segment: maps 1 and 2 are the queries and the output's gradient
template <typename T, int F>
static cudaError_t launch_rev(const GatedMaps& maps, const GatedParams& p, cudaStream_t st) {
  cudaError_t e = launch_one<T, F, false, true, true>(maps, p, p.nstreams * p.nseg, st);
  if (e != cudaSuccess) return e;
  ttt_gated_join_kernel<F, true><<<(int)(((long)p.nstreams * (F * F / 4) + 255) / 256), 256, 0, st>>>(p);
  return cudaGetLastError();
}
cudaError_t launch_gated_segments_rev(int dtype, int F, const GatedMaps& maps, const GatedParams& p, cudaStream_t st) {
  if (F == 64) return dtype == 1 ? launch_rev<__nv_bfloat16, 64>(maps, p, st) : launch_rev<float, 64>(maps, p, st);
  return dtype == 1 ? launch_rev<__nv_bfloat16, 32>(maps, p, st) : launch_rev<float, 32>(maps, p, st);
}

}  // namespace ttt
