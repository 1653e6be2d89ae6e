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
  static constexpr uint32_t BAR = GATES + 2 * sizeof(ChunkGates), BYTES = BAR + 32 + 1024;  // (1024: the base is aligned by hand)
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
  if (STATE && (int)blockIdx.x % p.nseg == (REV ? 0 : p.nseg - 1)) return;  // nothing follows it
  const uint32_t bar = base + SM::BAR;
  volatile int* const shared = reinterpret_cast<volatile int*>(mem + SM::BAR + 16);  // a wait has run out; this block's range
  if (tid == 0) {
    shared[0] = 0;
    shared[1] = !STATE && p.slots > 0 ? atomicAdd(p.flags + p.slots, 1) : (int)blockIdx.x;
    mbar_init(bar, 1);
    mbar_init(bar + 8, 1);
    fence_mbar_init();
  }
  __syncthreads();
  GatedWalk walk{};
  walk.set(p, shared[1], REV);
  const int n = walk.n;
  const GatedWalk::Step first = walk.part(0);
  auto chunk_of = [&](const GatedWalk::Step& s) { return REV ? p.NC - 1 - s.pos : s.pos; };
  auto fetch = [&](const GatedWalk::Step& s) {  // thread 0
    const int i = s.i;
    const int slot = BF ? i & 1 : 0;
    const uint32_t at = bar + 8 * slot, dst = base + (BF ? SM::TILES + slot * SM::NIN * SM::TILE : SM::RAWS);
    constexpr uint32_t bytes = BF ? SM::TILE : SM::RAW;
    const int b = s.stream / p.H, h = s.stream - b * p.H;
    mbar_expect_tx(at, SM::NIN * bytes);
#pragma unroll
    for (int m = 0; m < SM::NIN; ++m) tma_load_4d(dst + m * bytes, &maps.m[(STATE ? 1 : 0) + m], chunk_of(s) * GC, h, b, at);
  };
  if (tid == 0) {
    fetch(first);
    if (BF && n > 1) fetch(walk.next(first));
  }
  ChunkGates* const gates = reinterpret_cast<ChunkGates*>(mem + SM::GATES);
  auto gates_of = [&](const GatedWalk::Step& s, float2& g, float2& beta) {
    const size_t row = (size_t)s.stream * p.T;
    g = load_gates(p.g + row, chunk_of(s) * GC, p.T, lane, 0.f);
    beta = load_gates(p.beta != nullptr ? p.beta + row : nullptr, chunk_of(s) * GC, p.T, lane, 1.f);
  };
  if (w == 0) {
    float2 g0, b0;
    gates_of(first, g0, b0);
    make_chunk_gates(gates[0], lane, g0, b0);
  }

  // this warp's share of the state
  const int row0 = 16 * (w % SH::SLABS), part = w / SH::SLABS, col0 = part * SH::COLS;
  float W[SH::NT][4];
  // the state before walk step i: operand of its q W, and what the backward reads back.  Where a stream or a part of one starts,
  // from memory; false: the wait for it ran out
  auto publish = [&](const GatedWalk::Step& s) {
    const int i = s.i;
    if constexpr (STATE) {
      if (i == 0) load_state<F>(W, nullptr, row0, col0, lane);
    } else {
        bool ok = true;
      if (s.starts) {
        const float* w0 = p.w0 != nullptr ? p.w0 + (size_t)s.stream * F * F : nullptr;
        if (s.pos > 0) {
          if (p.slots > 0) {
            if (lane == 0) ok = wait_record(p.flags, walk.slot - 1);
            ok = __shfl_sync(0xffffffffu, ok, 0);
            w0 = p.records + (size_t)(walk.slot - 1) * F * F;
          } else {
            w0 = p.seg_state + (size_t)walk.slot * F * F;
          }
        }
        load_state<F>(W, w0, row0, col0, lane);
      }
      put_state<F, NP>(W, row0, col0, base + SM::W + (i & 1) * NP * GTile<F>::STATE_BYTES, lane);
      if (SAVE) put_fragments<F>(reinterpret_cast<float4*>(p.saved + ((size_t)s.stream * p.NC + s.pos) * F * F * 4), W, w, lane);
      return ok;
    }
    return true;
  };
  float total = 1.f;  // what is left of the state before the segment after it
  if (!publish(first)) shared[0] = 1;
  __syncthreads();
  const uint32_t low = GTile<F>::low(lane), high = GTile<F>::high(lane);

  for (GatedWalk::Step st = first, nx; st.i < n; st = nx) {
    nx = walk.next(st);
    const int i = st.i;
    const int slot = BF ? i & 1 : 0, t0 = chunk_of(st) * GC;
    const bool ahead = w == ((i + 1) & 3) && i + 1 < n;
    float2 g_next, b_next;
    if (ahead) gates_of(nx, g_next, b_next);
    if (!STATE && shared[0]) {
      if (tid == 0) report_timeout(p.status, 24, (uint32_t)i);
      return;
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
      if (tid == 0 && i + 1 < n) fetch(nx);
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
      store_rows<T, F>(static_cast<T*>(p.out) + ((size_t)st.stream * p.T + t0) * F, 16 * w, p.T - t0, o, lane);
    if constexpr (!STATE) {
      if (st.ends) {
        if (st.pos == p.NC - 1) {
          store_state<F>(p.w_out + (size_t)st.stream * F * F, W, row0, col0, lane);
        } else if (p.slots > 0) {
          store_state<F>(p.records + (size_t)walk.slot * F * F, W, row0, col0, lane);
          __threadfence();
          __syncthreads();
          if (tid == 0) set_record(p.flags, walk.slot);
        }
      }
    }
    if (i + 1 < n && !publish(nx)) shared[0] = 1;
    if (ahead) make_chunk_gates(gates[(i + 1) & 1], lane, g_next, b_next);
    __syncthreads();  // the tiles and this chunk's state and gates are free, the next one's are there
    if (BF && tid == 0 && i + 2 < n) fetch(walk.next(nx));
  }
  if constexpr (STATE) {
    store_state<F>(p.seg_state + (size_t)walk.slot * F * F, W, row0, col0, lane);
    if (tid == 0) p.seg_decay[walk.slot] = total;
  }
}

// The segments' own states to the states before them, along the sequence (REV: gradients, from the last segment to the first):
// state[s] <- W_s, W_{s+1} = decay[s] W_s + own[s].  Every thread carries one float2 of a stream's state; the loads of JOIN_AHEAD
// segments are on their way at once (one after the other, 37 segments of 12 streams took 60 us).
constexpr int JOIN_AHEAD = 12, JOIN_THREADS = 128;
template <int F, bool REV>
__global__ void __launch_bounds__(JOIN_THREADS) ttt_gated_join_kernel(const GatedParams p) {
  constexpr int Q = F * F / 2;
  const long e = (long)blockIdx.x * JOIN_THREADS + threadIdx.x;  // (a multiple of the threads)
  const long stream = e / Q;
  const int at = (int)(e - stream * Q);
  float2* s = reinterpret_cast<float2*>(p.seg_state) + stream * p.nseg * Q + at;
  const float* d = p.seg_decay + stream * p.nseg;
  float2 w = make_float2(0.f, 0.f);
  if (p.w0 != nullptr) w = reinterpret_cast<const float2*>(p.w0)[stream * Q + at];
  for (int k0 = 0; k0 < p.nseg; k0 += JOIN_AHEAD) {
    float2 own[JOIN_AHEAD];
    float f[JOIN_AHEAD];
#pragma unroll
    for (int k = 0; k < JOIN_AHEAD; ++k) {
      const int i = REV ? p.nseg - 1 - (k0 + k) : k0 + k;
      if (k0 + k < p.nseg - 1) {  // (nothing follows the last: it has no state of its own)
        own[k] = s[(long)i * Q];
        f[k] = d[i];
      }
    }
#pragma unroll
    for (int k = 0; k < JOIN_AHEAD; ++k) {
      const int i = REV ? p.nseg - 1 - (k0 + k) : k0 + k;
      if (k0 + k < p.nseg) s[(long)i * Q] = w;
      if (k0 + k < p.nseg - 1) w = make_float2(fmaf(f[k], w.x, own[k].x), fmaf(f[k], w.y, own[k].y));
    }
  }
}
static_assert(32 * 32 / 2 % JOIN_THREADS == 0, "whole blocks per stream");

// Streams that do not fill the card are cut into segments until they do; more streams than blocks are resident are cut into as
// many ranges as blocks are.
void gated_split(int64_t streams, int chunks, int dtype, bool backward, int* nseg, int* slots) {
  constexpr int SMS = 148, LEAST = 4;  // (chunks per segment: a segment's states and its second reading must be worth it)
  const int resident = dtype == 1 ? (backward ? 2 : 3) : 1;
  *nseg = 1;
  *slots = 0;
  if (streams > (int64_t)SMS * resident) *slots = SMS * resident;
  if (streams >= SMS) return;
  const int64_t want = ((backward ? 2 : 3) * SMS) / streams, most = chunks / LEAST;
  *nseg = (int)(want < most ? want : most > 1 ? most : 1);
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
    ttt_gated_join_kernel<F, false><<<(int)((long)p.nstreams * (F * F / 2) / JOIN_THREADS), JOIN_THREADS, 0, st>>>(p);
    if ((e = cudaGetLastError()) != cudaSuccess) return e;
  }
  const int grid = p.slots > 0 ? p.slots : p.nstreams * p.nseg;
  if (p.slots > 0) {
    const cudaError_t e = cudaMemsetAsync(p.flags, 0, (p.slots + 1) * sizeof(int), st);
    if (e != cudaSuccess) return e;
  }
  if (save) return launch_one<T, F, true, false, false>(maps, p, grid, st);
  return launch_one<T, F, false, false, false>(maps, p, grid, st);
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
  ttt_gated_join_kernel<F, true><<<(int)((long)p.nstreams * (F * F / 2) / JOIN_THREADS), JOIN_THREADS, 0, st>>>(p);
  return cudaGetLastError();
}
cudaError_t launch_gated_segments_rev(int dtype, int F, const GatedMaps& maps, const GatedParams& p, cudaStream_t st) {
  if (F == 64) return dtype == 1 ? launch_rev<__nv_bfloat16, 64>(maps, p, st) : launch_rev<float, 64>(maps, p, st);
  return dtype == 1 ? launch_rev<__nv_bfloat16, 32>(maps, p, st) : launch_rev<float, 32>(maps, p, st);
}

}  // namespace ttt
