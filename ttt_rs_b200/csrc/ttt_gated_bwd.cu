// Gated linear recurrence, backward (definitions and the chunked forward: ttt_gated.cuh).
//
// With dW the gradient of the state behind the chunk, W the saved state before it, D_ij = e^{G_i - G_j} (i >= j), u the output's
// gradient:
//   dq_i = sum_{j <= i} D_ij beta_j (u_i . v_j) k_j  +  e^{G_i} W u_i
//   dk_j = beta_j [ sum_{i >= j} D_ij (u_i . v_j) q_i  +  e^{G_end - G_j} dW v_j ]
//   dv_j = beta_j [ sum_{i >= j} D_ij (q_i . k_j) u_i  +  e^{G_end - G_j} dW^T k_j ]
//   dW'  = e^{G_end} dW + sum_i e^{G_i} q_i^T u_i                        (the gradient of the state before the chunk)
// The gradient of a gate is the sum over all ways from a written token to a read one that lead across it.  With
// N_ij = D_ij (q_i . k_j)(u_i . v_j), r_i = e^{G_i} q_i W u_i^T, s_j = e^{G_end - G_j} k_j dW v_j^T:
//   dbeta_j = sum_{i >= j} N_ij + s_j
//   dg_t    = sum_{j < t <= i} beta_j N_ij + sum_{i >= t} r_i + sum_{j < t} beta_j s_j + e^{G_end} <W, dW>
// summed way by way: no sum is taken as the difference of two others.  (g's gradient as a running sum of q dq - k dk leaves the
// rounding of the whole sequence behind, and where nothing leads across a token, noise instead of zero.)
//
// 384 streams of 2048 tokens, F = 64, bf16: 385 us, 2.3 TB/s, in passes back to back (alone with cold caches, under the profiler, 411).
// 1680 instructions per warp and chunk at 41 % of the issue slots (two blocks per SM, for registers and shared memory), shared-memory pipe 71 %, tensor pipe 43 %.
// What an operand holds is read from its tile again where it is used (keys, values, u): registers are short, and with fragments kept
// from use to use the training of 384 streams of 2048 tokens took 573 us, not 540.
//
// One CTA of eight warps per stream (or segment) walks the chunks from the last.  Warps 0-3 own 16 queries each: dq, and the
// float32 dW in their registers with its update.  Warps 4-7 own 16 keys each: dk, dv and the gates' sums.  Per chunk two
// barriers: all warps at its end, and the second group once more before it reads dW, which the first publishes when it has
// read the state (their third planes share their bytes).
#include <type_traits>

#include "ttt_kernels.h"
#include "ttt_gated.cuh"
#include "ttt_stage.cuh"

namespace ttt {

constexpr int GB_THREADS = 2 * 32 * GATED_WARPS;
__device__ __forceinline__ void block_sync() { asm volatile("bar.sync 0, %0;" ::"n"(GB_THREADS) : "memory"); }

struct ChunkSums {
  float r[GC], s[GC];               // r_i; beta_j s_j
  // the ways inside the chunk, from the block of 16 tokens that they start in to the one they end in:
  float c[GC];                      // sum over the blocks behind j's of beta_j N_ij
  float rows[GATED_WARPS - 1][GC];  // sum over the j of a block (= a warp) before i's of beta_j N_ij
  float block[GC];                  // those within a block that lead across token t
  float through[GATED_WARPS];       // e^{G_end} <W, dW>, by warp
};

template <typename T, int F>
struct GatedBwdSmem {
  static constexpr bool BF = sizeof(T) == 2;
  static constexpr int NP = BF ? 1 : 3, NS = 3;
  static constexpr uint32_t PLANE = GTile<F>::BYTES, TILE = NP * PLANE, RAW = GC * F * 4, WRAW = F * F * 4;
  static constexpr uint32_t SP = GTile<F>::STATE_BYTES;
  static constexpr uint32_t STAGES = BF ? 2 : 1;
  static constexpr uint32_t TILES = 0, RAWS = TILES + STAGES * 4 * TILE;
  static constexpr uint32_t WSAVED = RAWS + (BF ? 0 : 2 * RAW);  // as it was saved; bf16: its planes take the same bytes
  // planes of W upwards from W, of dW from DW in steps of DWS.  bf16: the third ones take the same bytes one after the other (both do
  // not fit beside the tiles of two chunks, two blocks per SM), dW from the last plane down
  static constexpr uint32_t W = BF ? WSAVED : WSAVED + WRAW, DW = W + (BF ? 4 : 3) * SP, DWS = BF ? 0u - SP : SP;
  static constexpr uint32_t GATES = W + (BF ? 5 : 6) * SP;
  static constexpr uint32_t SUMS = GATES + 2 * sizeof(ChunkGates);
  static constexpr uint32_t BAR = SUMS + 2 * sizeof(ChunkSums), BYTES = BAR + 48 + 1024;
  static_assert(!BF || 2 * SP == WRAW, "two planes of bf16 are as long as the float32 state");
};

template <typename T, int F>
__global__ void __launch_bounds__(GB_THREADS, sizeof(T) == 2 ? 2 : 1)
    ttt_gated_bwd_kernel(const __grid_constant__ GatedMaps maps, const GatedBwdParams p) {
  using SM = GatedBwdSmem<T, F>;
  using SH = StateShare<F>;
  using TL = GTile<F>;
  constexpr bool BF = SM::BF;
  constexpr int NP = SM::NP, NS = SM::NS, KS = F / 16;
  extern __shared__ uint8_t gated_smem[];
  const uint32_t raw = smem_u32(gated_smem), base = (raw + 1023) & ~1023u;
  uint8_t* const mem = gated_smem + (base - raw);
  const int tid = threadIdx.x, lane = tid & 31, w = (tid >> 5) & 3, g = lane >> 2, t4 = lane & 3;
  const bool queries = tid < GB_THREADS / 2;
  const uint32_t bar = base + SM::BAR, bar_w = bar + 16;
  volatile int* const shared = reinterpret_cast<volatile int*>(mem + SM::BAR + 24);  // a wait has run out; this block's range
  volatile int* const copies = shared + 2;  // (three barriers)
  const GatedWaits waits{shared, p.status};
  if (tid == 0) {
    shared[0] = copies[0] = copies[1] = copies[2] = 0;
    shared[1] = p.slots > 0 ? atomicAdd(p.flags + p.slots, 1) + p.first_slot : (int)blockIdx.x;
    mbar_init(bar, 1);
    mbar_init(bar + 8, 1);
    mbar_init(bar_w, 1);
    fence_mbar_init();
  }
  __syncthreads();
  if (p.slots > 0 && shared[1] >= p.slots) return;  // (first_slot)
  GatedWalk walk_{};
  walk_.set(p, shared[1], true);
  const int n = walk_.n;
  const GatedWalk::Step first = walk_.part(0);
  auto chunk_of = [&](const GatedWalk::Step& s) { return p.NC - 1 - s.pos; };
  // thread 0.  bf16: q, k, v, u of a chunk; float32: two of them at a time, through the same rows of shared memory
  auto fetch = [&](const GatedWalk::Step& s, int first, int count) {
    if (!waits.ok()) return;
    const int slot = BF ? s.i & 1 : 0;
    const uint32_t at = bar + 8 * slot, dst = base + (BF ? SM::TILES + slot * 4 * SM::TILE : SM::RAWS);
    constexpr uint32_t bytes = BF ? SM::TILE : SM::RAW;
    waits.started(copies, slot, BF ? (s.i >> 1) & 1 : first != 0);
    mbar_expect_tx(at, count * bytes);
    const int b = s.stream / p.H, h = s.stream - b * p.H;
    for (int m = 0; m < count; ++m) tma_load_4d(dst + m * bytes, &maps.m[first + m], chunk_of(s) * GC, h, b, at);
  };
  auto fetch_w = [&](const GatedWalk::Step& s) {
    if (!waits.ok()) return;
    waits.started(copies, 2, s.i & 1);
    mbar_expect_tx(bar_w, SM::WRAW);
    bulk_load_1d(base + SM::WSAVED, p.saved + ((size_t)s.stream * p.NC + chunk_of(s)) * SM::WRAW, SM::WRAW, bar_w);
  };
  if (tid == 0) {
    fetch(first, 0, BF ? 4 : 2);
    if (BF && n > 1) fetch(walk_.next(first), 0, 4);
    fetch_w(first);
  }
  auto gates_of = [&](const GatedWalk::Step& s, float2& g, float2& beta) {
    const size_t row = (size_t)s.stream * p.T;
    g = load_gates(p.g + row, chunk_of(s) * GC, p.T, lane, 0.f);
    beta = load_gates(p.beta != nullptr ? p.beta + row : nullptr, chunk_of(s) * GC, p.T, lane, 1.f);
  };
  ChunkGates* const gates = reinterpret_cast<ChunkGates*>(mem + SM::GATES);
  ChunkSums* const sums = reinterpret_cast<ChunkSums*>(mem + SM::SUMS);
  if (tid < 32) {
    float2 g0, b0;
    gates_of(first, g0, b0);
    make_chunk_gates<false>(gates[0], lane, g0, b0);
  }
  const int row0 = 16 * (w % SH::SLABS), part = w / SH::SLABS, col0 = part * SH::COLS;
  __syncthreads();

  const uint32_t low = TL::low(lane), high = TL::high(lane);
  // the gradients of the gates of walk step i, from the sums its warps left (one warp)
  auto finish_gates = [&](const GatedWalk::Step& st) {
    const int i = st.i;
    const ChunkSums& cs = sums[i & 1];
    const size_t row = (size_t)st.stream * p.T;
    const int t0 = chunk_of(st) * GC, a = 2 * lane;
    const float through = (cs.through[0] + cs.through[1]) + (cs.through[2] + cs.through[3]);
    const int blk = lane >> 3;
    float x[2], far1 = 0.f, far2 = 0.f;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float rows[GATED_WARPS - 1];
#pragma unroll
      for (int k = 0; k < GATED_WARPS - 1; ++k) rows[k] = k < blk ? cs.rows[k][a + e] : 0.f;
      x[e] = rows[0] + rows[1] + rows[2];
      if (blk >= 2) far1 += rows[0];            // over all of block 1
      if (blk == 3) far2 += rows[0] + rows[1];  // over all of block 2
    }
    const float2 r = *reinterpret_cast<const float2*>(&cs.r[a]), y = *reinterpret_cast<const float2*>(&cs.s[a]);
    const float2 c = *reinterpret_cast<const float2*>(&cs.c[a]), own = *reinterpret_cast<const float2*>(&cs.block[a]);
    // sums over the lanes behind this one (of the chunk, of the block) and before it
    float ends = r.x + r.y, ends_b = x[0] + x[1], starts = y.x + y.y, starts_b = c.x + c.y;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const float d0 = __shfl_down_sync(0xffffffffu, ends, o), u0 = __shfl_up_sync(0xffffffffu, starts, o);
      if (lane + o < 32) ends += d0;
      if (lane >= o) starts += u0;
      if (o < 8) {
        const float d1 = __shfl_down_sync(0xffffffffu, ends_b, o, 8), u1 = __shfl_up_sync(0xffffffffu, starts_b, o, 8);
        if ((lane & 7) + o < 8) ends_b += d1;
        if ((lane & 7) >= o) starts_b += u1;
      }
      far1 += __shfl_xor_sync(0xffffffffu, far1, o);
      far2 += __shfl_xor_sync(0xffffffffu, far2, o);
    }
    auto next = [&](float v, int width) {
      const float z = __shfl_down_sync(0xffffffffu, v, 1, width);
      return (lane & (width - 1)) == width - 1 ? 0.f : z;
    };
    auto prev = [&](float v, int width) {
      const float z = __shfl_up_sync(0xffffffffu, v, 1, width);
      return (lane & (width - 1)) == 0 ? 0.f : z;
    };
    const float ends1 = next(ends, 32) + r.y, ends_b1 = next(ends_b, 8) + x[1];
    const float starts0 = prev(starts, 32), starts_b0 = prev(starts_b, 8);
    const float base = through + (blk == 1 ? far1 : blk == 2 ? far2 : 0.f);
    const float d[2] = {base + ((ends + starts0) + (ends_b + starts_b0) + own.x),
                        base + ((ends1 + (starts0 + y.x)) + (ends_b1 + (starts_b0 + c.x)) + own.y)};
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int t = t0 + a + e;
      if (t < p.T) p.dg[row + t] = expf(p.g[row + t]) == 0.f ? 0.f : d[e];
    }
  };

  // One walk per group, so that neither carries the other's registers; the groups meet at barriers by number.
  auto walk = [&](auto group) {
  constexpr bool QUERIES = decltype(group)::value;
  float dW[QUERIES ? SH::NT : 1][4];
#pragma unroll 1
  for (GatedWalk::Step st = first, nx; st.i < n; st = nx) {
    nx = walk_.next(st);
    const int i = st.i;
    const int stream = st.stream;
    const int slot = BF ? i & 1 : 0, t0 = chunk_of(st) * GC, rows = p.T - t0;
    const bool ahead = QUERIES && w == 0 && i + 1 < n;
    float2 g_next, b_next;
    if (ahead) gates_of(nx, g_next, b_next);
    if constexpr (QUERIES) {
      if (st.starts) {  // the gradient of the state behind this stream, or behind this part of it
        const float* d0 = p.dw_out != nullptr ? p.dw_out + (size_t)stream * F * F : nullptr;
        if (st.pos > 0) {
          if (p.slots > 0) {
            if (tid == 0 && waits.ok() && !wait_record(p.flags, walk_.slot - 1, p.polls)) waits.fail(23, i);
            asm volatile("bar.sync 2, %0;" ::"n"(GB_THREADS / 2) : "memory");
            d0 = p.records + (size_t)(walk_.slot - 1) * F * F;
          } else {
            d0 = p.seg_state + (size_t)walk_.slot * F * F;
          }
        }
        load_state<F>(dW, d0, row0, col0, lane);
      }
    }
    const uint32_t tiles = base + SM::TILES + slot * 4 * SM::TILE;
    const uint32_t tq = tiles, tk = tq + SM::TILE, tv = tk + SM::TILE, tu = tv + SM::TILE;
    const uint32_t tw = base + SM::W, tdw = base + SM::DW;
    const ChunkGates& cg = gates[i & 1];
    ChunkSums& cs = sums[i & 1];
    waits.wait(bar + 8 * slot, BF ? (i >> 1) & 1 : 0, 21, i);
    if constexpr (!BF) {
      auto split2 = [&](uint32_t dst) {
        for (int m = 0; m < 2; ++m)
          split_rows<F>(dst + m * SM::TILE, SM::PLANE, reinterpret_cast<const float*>(mem + SM::RAWS + m * SM::RAW), GC, tid, GB_THREADS);
      };
      split2(tq);
      block_sync();
      if (tid == 0) fetch(st, 2, 2);
      waits.wait(bar, 1, 21, i);
      split2(tv);
      block_sync();
      if (tid == 0 && i + 1 < n) fetch(nx, 0, 2);
    }
    if constexpr (QUERIES) {
      const int ia = 16 * w + g;
      float dq[F / 8][4];
#pragma unroll
      for (int k = 0; k < F / 8; ++k) dq[k][0] = dq[k][1] = dq[k][2] = dq[k][3] = 0.f;
      const uint32_t uq = tu + 16 * w * TL::ROW + low;
      // from the state before the chunk: this thread's share as it was saved, for the ways that cross the whole chunk, and its
      // planes as an operand for all four warps
      const float all = cg.all;
      waits.wait(bar_w, i & 1, 22, i);
      {
        float W[SH::NT][4];
        get_fragments<F>(W, reinterpret_cast<const float4*>(mem + SM::WSAVED), w, lane);
        F2 cross = f2(0.f);
#pragma unroll
        for (int k = 0; k < SH::NT; ++k)
#pragma unroll
          for (int half = 0; half < 2; ++half) cross = f2fma(pr(W[k], half), pr(dW[k], half), cross);
        float through = f2hsum(cross);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) through += __shfl_xor_sync(0xffffffffu, through, o);
        if (lane == 0) cs.through[w] = through * all;
        asm volatile("bar.sync 2, %0;" ::"n"(GB_THREADS / 2) : "memory");
        put_state<F, NS>(W, row0, col0, tw, lane);
        asm volatile("bar.sync 2, %0;" ::"n"(GB_THREADS / 2) : "memory");
      }
      // W u, for r and, from the start of this warp's block on, for dq
#pragma unroll 1
      for (int k = 0; k < KS; ++k) {
        Pk<NP> v[4];
        ldsm_np<NP>(v, uq ^ (k << 5), SM::PLANE, false);
#pragma unroll
        for (int m = 0; m < KS; ++m) {
          Pk<NS> f[4];
          ldsm_np<NS>(f, (tw + 16 * m * TL::ROW + high) ^ (k << 5), TL::STATE_BYTES, false);
          mma_planes<NP, NS>(dq[2 * m], dq[2 * m + 1], v, f);
        }
      }
      if (BF) fence_proxy_async_smem();  // (the next saved state lands where this one's planes were written)
      asm volatile("bar.sync 2, %0;" ::"n"(GB_THREADS / 2) : "memory");
      if (tid == 0 && i + 1 < n) fetch_w(nx);
      put_state<F, NS>(dW, row0, col0, tdw, lane, SM::DWS);  // dW behind this chunk, for the other group
      asm volatile("bar.arrive 1, %0;" ::"n"(GB_THREADS) : "memory");
      F2 sa = f2(0.f), sb = f2(0.f);
#pragma unroll
      for (int m = 0; m < KS; ++m) {  // (an A fragment is two accumulator tiles)
        Pk<NP> q[4];
        ldsm_np<NP>(q, (tq + 16 * w * TL::ROW + low) ^ (m << 5), SM::PLANE, false);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          sa = f2fma(pr(dq[2 * m + e], 0), make_float2(pk_lo(q[2 * e]), pk_hi(q[2 * e])), sa);
          sb = f2fma(pr(dq[2 * m + e], 1), make_float2(pk_lo(q[2 * e + 1]), pk_hi(q[2 * e + 1])), sb);
        }
      }
      const float r0 = quad_sum(f2hsum(sa)) * cg.from[ia], r1 = quad_sum(f2hsum(sb)) * cg.from[ia + 8];
      if (t4 == 0) {
        cs.r[ia] = r0;
        cs.r[ia + 8] = r1;
      }
      const float first = cg.starts[w];
#pragma unroll
      for (int k = 0; k < F / 8; ++k) scale_rows(dq[k], first, first);
      // inside the chunk: the blocks before this warp's, then its own
      const float ra = cg.into[ia], rb = cg.into[ia + 8];
#pragma unroll 1
      for (int jt = 0; jt <= w; ++jt) {
        float s0[4] = {}, s1[4] = {};
#pragma unroll
        for (int k = 0; k < KS; ++k) {
          Pk<NP> u[4], f[4];
          ldsm_np<NP>(u, uq ^ (k << 5), SM::PLANE, false);
          ldsm_np<NP>(f, (tv + 16 * jt * TL::ROW + high) ^ (k << 5), SM::PLANE, false);
          mma_planes<NP, NP>(s0, s1, u, f);
        }
        const int j0 = 16 * jt + 2 * t4;
        if (jt < w) {
          const F2 between = f2(cg.blocks[jt][w - 1]);
          scale_cols(s0, f2mul(ld2(&cg.out_b[j0]), between));
          scale_cols(s1, f2mul(ld2(&cg.out_b[j0 + 8]), between));
        } else {
#pragma unroll
          for (int k = 0; k < F / 8; ++k) scale_rows(dq[k], ra, rb);
          float d[2][4];
          block_decays<true>(d, cg, w, g, t4);
          const float2 b0 = ld2(&cg.beta[j0]), b1 = ld2(&cg.beta[j0 + 8]);
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            s0[2 * half] = d[half][0] > 0.f ? s0[2 * half] * (d[half][0] * b0.x) : 0.f;
            s0[2 * half + 1] = d[half][1] > 0.f ? s0[2 * half + 1] * (d[half][1] * b0.y) : 0.f;
            s1[2 * half] = d[half][2] > 0.f ? s1[2 * half] * (d[half][2] * b1.x) : 0.f;
            s1[2 * half + 1] = d[half][3] > 0.f ? s1[2 * half + 1] * (d[half][3] * b1.y) : 0.f;
          }
        }
        Pk<NP> a[4];
        as_operand<NP>(a, s0, s1);
#pragma unroll
        for (int m = 0; m < KS; ++m) {
          Pk<NP> f[4];
          ldsm_np<NP>(f, (tk + 16 * jt * TL::ROW + low) ^ (m << 5), SM::PLANE, true);
          mma_planes<NP, NP>(dq[2 * m], dq[2 * m + 1], a, f);
        }
      }
      store_rows<T, F>(static_cast<T*>(p.dq) + ((size_t)stream * p.T + t0) * F, 16 * w, rows, dq, lane);
      // dW before the chunk
      float sum[SH::NT][4];  // (the tensor cores truncate as they add: not onto dW)
#pragma unroll
      for (int k = 0; k < SH::NT; ++k) sum[k][0] = sum[k][1] = sum[k][2] = sum[k][3] = 0.f;
#pragma unroll 1
      for (int it = 0; it < GC / 16; ++it) {
        Pk<3> qt[4];
        {
          Pk<NP> f[4];
          ldsm_np<NP>(f, (tq + 16 * it * TL::ROW + high) ^ (row0 << 1), SM::PLANE, true);
          scale_a_cols<3, NP>(qt, f, ld2(&cg.from[16 * it + 2 * t4]), ld2(&cg.from[16 * it + 2 * t4 + 8]));
        }
#pragma unroll
        for (int k = 0; k < SH::NT / 2; ++k) {
          Pk<NP> f[4];
          ldsm_np<NP>(f, (tu + 16 * it * TL::ROW + low) ^ ((col0 + 16 * k) << 1), SM::PLANE, true);
          mma_planes<3, NP>(sum[2 * k], sum[2 * k + 1], qt, f);
        }
      }
#pragma unroll
      for (int k = 0; k < SH::NT; ++k) scale_add(dW[k], all, sum[k]);
    } else {
      const int ja = 16 * w + g;
      const float oa = cg.out[ja], ob = cg.out[ja + 8], ba = cg.beta[ja], bb = cg.beta[ja + 8];
      const float wa = cg.out_b[ja], wb = cg.out_b[ja + 8];
      const uint32_t kq = tk + 16 * w * TL::ROW + low, vq = tv + 16 * w * TL::ROW + low;
      // keys . queries and values . u of this warp's 16 tokens against those of block `it`
      auto products = [&](int it, float (&s0)[4], float (&s1)[4], float (&v0)[4], float (&v1)[4]) {
#pragma unroll
        for (int x = 0; x < 4; ++x) s0[x] = s1[x] = v0[x] = v1[x] = 0.f;
        const uint32_t q = tq + 16 * it * TL::ROW + high, u = tu + 16 * it * TL::ROW + high;
#pragma unroll
        for (int k = 0; k < KS; ++k) {
          Pk<NP> a[4], f[4];
          ldsm_np<NP>(a, kq ^ (k << 5), SM::PLANE, false);
          ldsm_np<NP>(f, q ^ (k << 5), SM::PLANE, false);
          mma_planes<NP, NP>(s0, s1, a, f);
          ldsm_np<NP>(a, vq ^ (k << 5), SM::PLANE, false);
          ldsm_np<NP>(f, u ^ (k << 5), SM::PLANE, false);
          mma_planes<NP, NP>(v0, v1, a, f);
        }
      };
      // sums over the eight row pairs of the warp: halve the columns that a lane carries with each exchange
      auto column_sums = [&](const float (&col)[4], float* to) {
        const bool up4 = lane & 4, up8 = lane & 8;
        float k0 = up4 ? col[2] : col[0], k1 = up4 ? col[3] : col[1];
        k0 += __shfl_xor_sync(0xffffffffu, up4 ? col[0] : col[2], 4);
        k1 += __shfl_xor_sync(0xffffffffu, up4 ? col[1] : col[3], 4);
        float k = up8 ? k1 : k0;
        k += __shfl_xor_sync(0xffffffffu, up8 ? k0 : k1, 8);
        k += __shfl_xor_sync(0xffffffffu, k, 16);
        if (lane < 16) to[2 * t4 + (up4 ? 8 : 0) + (up8 ? 1 : 0)] = k;
      };
      // sums of N: over the blocks behind j's without what is left of j behind its own block (na, nb), and within the block
      float na = 0.f, nb = 0.f, own_a = 0.f, own_b = 0.f;
      Pk<NP> as[4][4], av[4][4];  // the operands of dv and dk: 0 the own block, d the one d blocks behind it
#pragma unroll
      for (int d = 1; d < 4; ++d) {
        const int it = w + d;
        if (it < 4) {
          float s0[4], s1[4], v0[4], v1[4];
          products(it, s0, s1, v0, v1);
          const F2 between = f2(cg.blocks[w][it - 1]);
          const F2 f0 = f2mul(ld2(&cg.into[16 * it + 2 * t4]), between), f1 = f2mul(ld2(&cg.into[16 * it + 2 * t4 + 8]), between);
          scale_cols(s0, f0);
          scale_cols(s1, f1);
          const F2 p0 = f2mul(pr(s0, 0), pr(v0, 0)), p1 = f2mul(pr(s0, 1), pr(v0, 1));
          const F2 p2 = f2mul(pr(s1, 0), pr(v1, 0)), p3 = f2mul(pr(s1, 1), pr(v1, 1));
          na += f2hsum(f2add(p0, p2));
          nb += f2hsum(f2add(p1, p3));
          const F2 x0 = f2fma(p0, f2(wa), f2mul(p1, f2(wb))), x1 = f2fma(p2, f2(wa), f2mul(p3, f2(wb)));
          const float col[4] = {x0.x, x0.y, x1.x, x1.y};
          column_sums(col, cs.rows[w] + 16 * it);
          scale_cols(v0, f0);
          scale_cols(v1, f1);
          as_operand<NP>(as[d], s0, s1);
          as_operand<NP>(av[d], v0, v1);
        }
      }
      {
        float s0[4], s1[4], v0[4], v1[4], d[2][4], M[2][4], col[4];
        products(w, s0, s1, v0, v1);
        block_decays<false>(d, cg, w, g, t4);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const float beta = half ? bb : ba;
          float sum = 0.f;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float &s = (e < 2 ? s0 : s1)[2 * half + (e & 1)], &v = (e < 2 ? v0 : v1)[2 * half + (e & 1)];
            const float x = d[half][e];
            const float n_ij = x > 0.f ? s * v * x : 0.f;
            sum += n_ij;
            M[half][e] = 2 * t4 + (e & 1) + 8 * (e >> 1) > g + 8 * half ? beta * n_ij : 0.f;
            s = x > 0.f ? s * (x * beta) : 0.f;
            v = x > 0.f ? v * (x * beta) : 0.f;
          }
          (half ? own_b : own_a) = sum;
        }
        as_operand<NP>(as[0], s0, s1);
        as_operand<NP>(av[0], v0, v1);
        // the ways within the block across token t: over j < t the sums of i >= t
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          float(&m)[4] = M[half];
          float lo = m[0] + m[1], hi = m[2] + m[3];
#pragma unroll
          for (int o = 1; o < 4; o <<= 1) {
            const float l = __shfl_down_sync(0xffffffffu, lo, o, 4), h = __shfl_down_sync(0xffffffffu, hi, o, 4);
            if (t4 + o < 4) {
              lo += l;
              hi += h;
            }
          }
          const float l = __shfl_down_sync(0xffffffffu, lo, 1, 4), h = __shfl_down_sync(0xffffffffu, hi, 1, 4);
          const float upper = __shfl_sync(0xffffffffu, hi, 0, 4);
          m[3] += t4 == 3 ? 0.f : h;
          m[2] += m[3];
          m[1] += (t4 == 3 ? 0.f : l) + upper;
          m[0] += m[1];
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int t = 2 * t4 + (e & 1) + 8 * (e >> 1);
          col[e] = (t > g ? M[0][e] : 0.f) + (t > g + 8 ? M[1][e] : 0.f);
        }
        column_sums(col, cs.block + 16 * w);
      }
      na = quad_sum(na);
      nb = quad_sum(nb);
      own_a = quad_sum(own_a);
      own_b = quad_sum(own_b);
      // adds to rows that hold what comes from behind the chunk: up to the end of this block, the sums over the blocks behind of
      // operand . tile; what is left of the row's token there; the own block
      auto gather = [&](float (&r)[F / 8][4], const Pk<NP> (&a)[4][4], uint32_t tile) {
        const float last = cg.blocks[w][3];
#pragma unroll
        for (int k = 0; k < F / 8; ++k) scale_rows(r[k], last, last);
#pragma unroll
        for (int d = 3; d >= 0; --d) {
          if (d == 0) {
#pragma unroll
            for (int k = 0; k < F / 8; ++k) scale_rows(r[k], wa, wb);
          }
          if (w + d < 4) {
            const uint32_t at = tile + 16 * (w + d) * TL::ROW + low;
#pragma unroll
            for (int m = 0; m < KS; ++m) {
              Pk<NP> f[4];
              ldsm_np<NP>(f, at ^ (m << 5), SM::PLANE, true);
              mma_planes<NP, NP>(r[2 * m], r[2 * m + 1], a[d], f);
            }
          }
        }
      };
      asm volatile("bar.sync 1, %0;" ::"n"(GB_THREADS) : "memory");
      {
        float dv[F / 8][4];
#pragma unroll
        for (int k = 0; k < F / 8; ++k) dv[k][0] = dv[k][1] = dv[k][2] = dv[k][3] = 0.f;
#pragma unroll 1
        for (int k = 0; k < KS; ++k) {  // (dv is a result of the inputs' type: bf16 takes the leading plane of dW)
          Pk<NP> a[4];
          ldsm_np<NP>(a, kq ^ (k << 5), SM::PLANE, false);
#pragma unroll
          for (int m = 0; m < KS; ++m) {
            Pk<NP> f[4];
            ldsm_np<NP>(f, (tdw + 16 * k * TL::ROW + low) ^ (m << 5), SM::DWS, true);
            mma_planes<NP, NP>(dv[2 * m], dv[2 * m + 1], a, f);
          }
        }
        gather(dv, as, tu);
        store_rows<T, F>(static_cast<T*>(p.dv) + ((size_t)stream * p.T + t0) * F, 16 * w, rows, dv, lane);
      }
      F2 sa = f2(0.f), sb = f2(0.f);
      {
        float dk[F / 8][4];
#pragma unroll
        for (int k = 0; k < F / 8; ++k) dk[k][0] = dk[k][1] = dk[k][2] = dk[k][3] = 0.f;
#pragma unroll 1
        for (int k = 0; k < KS; ++k) {
          Pk<NP> v[4];
          ldsm_np<NP>(v, vq ^ (k << 5), SM::PLANE, false);
#pragma unroll
          for (int m = 0; m < KS; ++m) {
            Pk<NS> f[4];
            ldsm_np<NS>(f, (tdw + 16 * m * TL::ROW + high) ^ (k << 5), SM::DWS, false);
            mma_planes<NP, NS>(dk[2 * m], dk[2 * m + 1], v, f);
          }
        }
#pragma unroll
        for (int m = 0; m < KS; ++m) {  // (an A fragment is two accumulator tiles)
          Pk<NP> a[4];
          ldsm_np<NP>(a, kq ^ (m << 5), SM::PLANE, false);
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            sa = f2fma(pr(dk[2 * m + e], 0), make_float2(pk_lo(a[2 * e]), pk_hi(a[2 * e])), sa);
            sb = f2fma(pr(dk[2 * m + e], 1), make_float2(pk_lo(a[2 * e + 1]), pk_hi(a[2 * e + 1])), sb);
          }
        }
        gather(dk, av, tq);
        store_rows<T, F>(static_cast<T*>(p.dk) + ((size_t)stream * p.T + t0) * F, 16 * w, rows, dk, lane);
      }
      const float ea = cg.end[ja], eb = cg.end[ja + 8];
      const float s0 = quad_sum(f2hsum(sa)) * ea, s1 = quad_sum(f2hsum(sb)) * eb;
      if (t4 == 0) {
        cs.s[ja] = s0 * ba;
        cs.s[ja + 8] = s1 * bb;
        cs.c[ja] = na * wa;
        cs.c[ja + 8] = nb * wb;
        if (p.dbeta != nullptr) {
          float* d = p.dbeta + (size_t)stream * p.T + t0;
          if (ja < rows) d[ja] = fmaf(na, oa, own_a) + s0;
          if (ja + 8 < rows) d[ja + 8] = fmaf(nb, ob, own_b) + s1;
        }
      }
    }
    if (ahead) make_chunk_gates<false>(gates[(i + 1) & 1], lane, g_next, b_next);
    if constexpr (QUERIES) {
      if (st.ends) {
        if (st.pos == p.NC - 1) {
          store_state<F>(p.dw0 + (size_t)stream * F * F, dW, row0, col0, lane);
        } else if (p.slots > 0) {
          store_state<F>(p.records + (size_t)walk_.slot * F * F, dW, row0, col0, lane);
          __threadfence();
          asm volatile("bar.sync 2, %0;" ::"n"(GB_THREADS / 2) : "memory");
          if (tid == 0) set_record(p.flags, walk_.slot);
        }
      }
    }
    block_sync();  // this chunk's tiles, states and sums are complete and free
    if (QUERIES && tid == 0) {
      if (BF && i + 2 < n) fetch(walk_.next(nx), 0, 4);
    }
    if (!QUERIES && w == GATED_WARPS - 1) finish_gates(st);
  }
  };
  if (queries) walk(std::true_type{});
  else walk(std::false_type{});
  // copies that may still be on their way (the walk ends with a barrier, and thread 0 starts them all)
  if (tid == 0 && !waits.ok()) waits.drain(copies, 3, bar);
}

template <typename T, int F>
static cudaError_t launch_one(const GatedMaps& maps, const GatedBwdParams& p, cudaStream_t st) {
  auto kfn = ttt_gated_bwd_kernel<T, F>;
  constexpr size_t smem = GatedBwdSmem<T, F>::BYTES;
  static_assert(smem <= (sizeof(T) == 2 ? 113 : 227) * 1024, "shared memory");
  static DeviceValue ready;
  int unused;
  cudaError_t e = ready.get(0, &unused, [&](int* v) {
    *v = 0;
    return cudaFuncSetAttribute(kfn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  });
  if (e != cudaSuccess) return e;
  if (p.slots > 0 && (e = cudaMemsetAsync(p.flags, 0, (p.slots + 1) * sizeof(int), st)) != cudaSuccess) return e;
  kfn<<<p.slots > 0 ? p.slots : p.nstreams * p.nseg, GB_THREADS, smem, st>>>(maps, p);
  return cudaGetLastError();
}
cudaError_t launch_gated_bwd(int dtype, int F, const GatedMaps& maps, const GatedBwdParams& p, cudaStream_t st) {
  if (F == 64) return dtype == 1 ? launch_one<__nv_bfloat16, 64>(maps, p, st) : launch_one<float, 64>(maps, p, st);
  return dtype == 1 ? launch_one<__nv_bfloat16, 32>(maps, p, st) : launch_one<float, 32>(maps, p, st);
}

}  // namespace ttt
