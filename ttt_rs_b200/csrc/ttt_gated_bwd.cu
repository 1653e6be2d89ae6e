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
// One CTA of eight warps per stream (or segment) walks the chunks from the last.  Warps 0-3 own 16 queries each: dq, and the
// float32 dW in their registers with its update.  Warps 4-7 own 16 keys each: dk, dv and the gates' sums.  Per chunk two
// barriers: all warps at its end, and the second group once more before it reads dW, which the first publishes after the first
// barrier.
#include "ttt_kernels.h"
#include "ttt_gated.cuh"
#include "ttt_stage.cuh"

namespace ttt {

constexpr int GB_THREADS = 2 * 32 * GATED_WARPS;

struct ChunkSums {
  float r[GC], s[GC];               // r_i; beta_j s_j
  // the ways inside the chunk, from the block of 16 tokens that they start in to the one they end in:
  float c[GC];                      // sum over the blocks behind j's of beta_j N_ij
  float rows[GATED_WARPS][GC];      // sum over the j of a block (= a warp) before i's of beta_j N_ij
  float block[GC];                  // those within a block that lead across token t
  float through[GATED_WARPS];       // e^{G_end} <W, dW>, by warp
};

template <typename T, int F>
struct GatedBwdSmem {
  static constexpr bool BF = sizeof(T) == 2;
  static constexpr int NP = BF ? 1 : 3, NS = BF ? 2 : 3;
  static constexpr uint32_t PLANE = GTile<F>::BYTES, TILE = NP * PLANE, RAW = GC * F * 4, WRAW = F * F * 4;
  static constexpr uint32_t STATE = NS * GTile<F>::STATE_BYTES;
  static constexpr uint32_t STAGES = BF ? 2 : 1;
  static constexpr uint32_t TILES = 0, RAWS = TILES + STAGES * 4 * TILE;
  static constexpr uint32_t WSAVED = RAWS + (BF ? 0 : 2 * RAW);  // as it was saved (bf16: the planes themselves)
  static constexpr uint32_t W = BF ? WSAVED : WSAVED + WRAW, DW = W + STATE;
  static constexpr uint32_t GATES = DW + STATE;
  static constexpr uint32_t SUMS = GATES + 2 * sizeof(ChunkGates);
  static constexpr uint32_t BAR = SUMS + 2 * sizeof(ChunkSums), BYTES = BAR + 32 + 1024;
  static_assert(!BF || STATE == WRAW, "two planes of bf16 are as long as the float32 state");
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
  const int stream = blockIdx.x / p.nseg, seg = blockIdx.x - stream * p.nseg;
  const int c_lo = seg * p.seg_chunks, c_hi = min(p.NC, c_lo + p.seg_chunks), n = c_hi - c_lo;
  const int h = stream % p.H, b = stream / p.H;
  const uint32_t bar = base + SM::BAR, bar_w = bar + 16;
  if (tid == 0) {
    mbar_init(bar, 1);
    mbar_init(bar + 8, 1);
    mbar_init(bar_w, 1);
    fence_mbar_init();
  }
  __syncthreads();
  auto chunk_of = [&](int i) { return c_hi - 1 - i; };
  // thread 0.  bf16: q, k, v, u of a chunk; float32: two of them at a time, through the same rows of shared memory
  auto fetch = [&](int i, int first, int count) {
    const int slot = BF ? i & 1 : 0;
    const uint32_t at = bar + 8 * slot, dst = base + (BF ? SM::TILES + slot * 4 * SM::TILE : SM::RAWS);
    constexpr uint32_t bytes = BF ? SM::TILE : SM::RAW;
    mbar_expect_tx(at, count * bytes);
    for (int m = 0; m < count; ++m) tma_load_4d(dst + m * bytes, &maps.m[first + m], chunk_of(i) * GC, h, b, at);
  };
  const uint8_t* saved = p.saved + (size_t)stream * p.NC * SM::WRAW;
  auto fetch_w = [&](int i) {
    mbar_expect_tx(bar_w, SM::WRAW);
    bulk_load_1d(base + SM::WSAVED, saved + (size_t)chunk_of(i) * SM::WRAW, SM::WRAW, bar_w);
  };
  if (tid == 0) {
    fetch(0, 0, BF ? 4 : 2);
    if (BF && n > 1) fetch(1, 0, 4);
    fetch_w(0);
  }
  const float* gp = p.g + (size_t)stream * p.T;
  const float* bp = p.beta != nullptr ? p.beta + (size_t)stream * p.T : nullptr;
  ChunkGates* const gates = reinterpret_cast<ChunkGates*>(mem + SM::GATES);
  ChunkSums* const sums = reinterpret_cast<ChunkSums*>(mem + SM::SUMS);
  if (tid < 32) {
    const int t0 = chunk_of(0) * GC;
    make_chunk_gates(gates[0], lane, load_gates(gp, t0, p.T, lane, 0.f), load_gates(bp, t0, p.T, lane, 1.f));
  }
  const int row0 = 16 * (w % SH::SLABS), part = w / SH::SLABS, col0 = part * SH::COLS;
  float dW[SH::NT][4];
  if (queries) {
    const float* d0 = seg < p.nseg - 1 ? p.seg_state + ((size_t)stream * p.nseg + seg) * F * F
                      : p.dw_out != nullptr ? p.dw_out + (size_t)stream * F * F : nullptr;
    load_state<F>(dW, d0, row0, col0, lane);
  }
  __syncthreads();

  // the gradients of the gates of walk step i, from the sums its warps left (one warp)
  auto finish_gates = [&](int i) {
    const ChunkSums& cs = sums[i & 1];
    const int t0 = chunk_of(i) * GC, a = 2 * lane;
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
      if (t < p.T) p.dg[(size_t)stream * p.T + t] = expf(gp[t]) == 0.f ? 0.f : d[e];
    }
  };

  for (int i = 0; i < n; ++i) {
    const int slot = BF ? i & 1 : 0, t0 = chunk_of(i) * GC, rows = p.T - t0;
    const bool ahead = tid < 32 && i + 1 < n;
    float2 g_next, b_next;
    if (ahead) {
      g_next = load_gates(gp, chunk_of(i + 1) * GC, p.T, lane, 0.f);
      b_next = load_gates(bp, chunk_of(i + 1) * GC, p.T, lane, 1.f);
    }
    const uint32_t tiles = base + SM::TILES + slot * 4 * SM::TILE;
    const uint32_t tq = tiles, tk = tq + SM::TILE, tv = tk + SM::TILE, tu = tv + SM::TILE;
    const uint32_t tw = base + SM::W, tdw = base + SM::DW;
    const ChunkGates& cg = gates[i & 1];
    ChunkSums& cs = sums[i & 1];
    if (queries) {  // dW behind this chunk, for the other group
      put_state<F, NS>(dW, row0, col0, tdw, nullptr, lane);
      asm volatile("bar.arrive 1, %0;" ::"n"(GB_THREADS) : "memory");
    }
    bool ok = mbar_wait_bounded(bar + 8 * slot, BF ? (i >> 1) & 1 : 0);
    if constexpr (!BF) {
      auto split2 = [&](uint32_t dst) {
        for (int m = 0; m < 2; ++m)
          split_rows<F>(dst + m * SM::TILE, SM::PLANE, reinterpret_cast<const float*>(mem + SM::RAWS + m * SM::RAW), GC, tid, GB_THREADS);
      };
      split2(tq);
      __syncthreads();
      if (tid == 0 && ok) fetch(i, 2, 2);
      ok = ok && mbar_wait_bounded(bar, 1) && mbar_wait_bounded(bar_w, i & 1);
      split2(tv);
      split_rows<F>(tw, TL::STATE_BYTES, reinterpret_cast<const float*>(mem + SM::WSAVED), F, tid, GB_THREADS);
      __syncthreads();
      if (tid == 0 && ok && i + 1 < n) {
        fetch(i + 1, 0, 2);
        fetch_w(i + 1);
      }
    }
    if (!ok) {
      if (tid == 0) report_timeout(p.status, 21, (uint32_t)i);
      return;
    }
    if (queries) {
      const int ia = 16 * w + g;
      float dq[F / 8][4];
#pragma unroll
      for (int k = 0; k < F / 8; ++k) dq[k][0] = dq[k][1] = dq[k][2] = dq[k][3] = 0.f;
      Pk<NP> u[KS][4];
#pragma unroll
      for (int k = 0; k < KS; ++k) ldsm_np<NP>(u[k], tu + TL::a_mk(lane, 16 * w, 16 * k), SM::PLANE, false);
      // inside the chunk
      const float ha = cg.hi[ia], la = cg.lo[ia], hb = cg.hi[ia + 8], lb = cg.lo[ia + 8];
#pragma unroll
      for (int jt = 0; jt < GC / 16; ++jt) {
        if (jt > w) break;
        float s0[4] = {}, s1[4] = {};
#pragma unroll
        for (int k = 0; k < KS; ++k) {
          Pk<NP> f[4];
          ldsm_np<NP>(f, tv + TL::b_nk(lane, 16 * jt, 16 * k), SM::PLANE, false);
          mma_planes<NP, NP>(s0, s1, u[k], f);
        }
        const int j0 = 16 * jt + 2 * t4;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int j = j0 + (e & 1) + 8 * (e >> 1);
          const float hj = cg.hi[j], lj = cg.lo[j], bj = cg.beta[j];
          float* s = e < 2 ? s0 : s1;
          s[e & 1] = j <= ia ? s[e & 1] * (exp2f((ha - hj) + (la - lj)) * bj) : 0.f;
          s[2 + (e & 1)] = j <= ia + 8 ? s[2 + (e & 1)] * (exp2f((hb - hj) + (lb - lj)) * bj) : 0.f;
        }
        const Pk<NP> a[4] = {split_pack<NP>(s0[0], s0[1]), split_pack<NP>(s0[2], s0[3]), split_pack<NP>(s1[0], s1[1]),
                             split_pack<NP>(s1[2], s1[3])};
#pragma unroll
        for (int m = 0; m < KS; ++m) {
          Pk<NP> f[4];
          ldsm_np<NP>(f, tk + TL::b_kn(lane, 16 * m, 16 * jt), SM::PLANE, true);
          mma_planes<NP, NP>(dq[2 * m], dq[2 * m + 1], a, f);
        }
      }
      // from the state before the chunk
      if constexpr (BF) {
        if (!mbar_wait_bounded(bar_w, i & 1)) {
          if (tid == 0) report_timeout(p.status, 22, (uint32_t)i);
          ok = false;
        }
      }
      const float fa = cg.from[ia], fb = cg.from[ia + 8];
      float ra = 0.f, rb = 0.f;
#pragma unroll
      for (int m = 0; m < KS; ++m) {
        float c0[4] = {}, c1[4] = {};
#pragma unroll
        for (int k = 0; k < KS; ++k) {
          Pk<NS> f[4];
          ldsm_np<NS>(f, tw + TL::b_nk(lane, 16 * m, 16 * k), TL::STATE_BYTES, false);
          mma_planes<NP, NS>(c0, c1, u[k], f);
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float* c = e ? c1 : c0;
          const int col = 16 * m + 8 * e + 2 * t4;
          Pk<NP> qa, qb;
#pragma unroll
          for (int pl = 0; pl < NP; ++pl) {
            qa.p[pl] = ld_shared_b32(tq + pl * SM::PLANE + TL::off(ia, col));
            qb.p[pl] = ld_shared_b32(tq + pl * SM::PLANE + TL::off(ia + 8, col));
          }
          c[0] *= fa;
          c[1] *= fa;
          c[2] *= fb;
          c[3] *= fb;
          ra = fmaf(c[0], pk_lo(qa), fmaf(c[1], pk_hi(qa), ra));
          rb = fmaf(c[2], pk_lo(qb), fmaf(c[3], pk_hi(qb), rb));
#pragma unroll
          for (int x = 0; x < 4; ++x) dq[2 * m + e][x] += c[x];
        }
      }
      ra = quad_sum(ra);
      rb = quad_sum(rb);
      if (t4 == 0) {
        cs.r[ia] = ra;
        cs.r[ia + 8] = rb;
      }
      store_rows<T, F>(static_cast<T*>(p.dq) + ((size_t)stream * p.T + t0) * F, 16 * w, rows, dq, lane);
      // ways that cross the whole chunk
      float through = 0.f;
#pragma unroll
      for (int k = 0; k < SH::NT; ++k)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          Pk<NS> s;
#pragma unroll
          for (int pl = 0; pl < NS; ++pl)
            s.p[pl] = ld_shared_b32(tw + pl * TL::STATE_BYTES + TL::off(row0 + g + 8 * half, col0 + 8 * k + 2 * t4));
          through = fmaf(pk_lo(s), dW[k][2 * half], fmaf(pk_hi(s), dW[k][2 * half + 1], through));
        }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) through += __shfl_xor_sync(0xffffffffu, through, o);
      const float all = cg.all;
      if (lane == 0) cs.through[w] = through * all;
      // dW before the chunk
#pragma unroll
      for (int k = 0; k < SH::NT; ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e) dW[k][e] *= all;
#pragma unroll
      for (int it = 0; it < GC / 16; ++it) {
        Pk<NS> qt[4];
        {
          Pk<NP> f[4];
          ldsm_np<NP>(f, tq + TL::a_km(lane, row0, 16 * it), SM::PLANE, true);
          scale_a_cols<NS, NP>(qt, f, *reinterpret_cast<const float2*>(&cg.from[16 * it + 2 * t4]),
                               *reinterpret_cast<const float2*>(&cg.from[16 * it + 2 * t4 + 8]));
        }
#pragma unroll
        for (int k = 0; k < SH::NT / 2; ++k) {
          Pk<NP> f[4];
          ldsm_np<NP>(f, tu + TL::b_kn(lane, col0 + 16 * k, 16 * it), SM::PLANE, true);
          mma_planes<NS, NP>(dW[2 * k], dW[2 * k + 1], qt, f);
        }
      }
    } else {
      const int ja = 16 * w + g;
      float dk[F / 8][4], dv[F / 8][4];
#pragma unroll
      for (int k = 0; k < F / 8; ++k)
#pragma unroll
        for (int x = 0; x < 4; ++x) dk[k][x] = dv[k][x] = 0.f;
      const float ha = cg.hi[ja], la = cg.lo[ja], hb = cg.hi[ja + 8], lb = cg.lo[ja + 8];
      const float ba = cg.beta[ja], bb = cg.beta[ja + 8];
      float na = 0.f, nb = 0.f, ca = 0.f, cb = 0.f;  // sums of N over i >= j and over the blocks behind
#pragma unroll
      for (int it = 0; it < GC / 16; ++it) {
        if (it < w) continue;
        float s0[4] = {}, s1[4] = {}, v0[4] = {}, v1[4] = {};
#pragma unroll
        for (int k = 0; k < KS; ++k) {
          Pk<NP> a[4], f[4];
          ldsm_np<NP>(a, tk + TL::a_mk(lane, 16 * w, 16 * k), SM::PLANE, false);
          ldsm_np<NP>(f, tq + TL::b_nk(lane, 16 * it, 16 * k), SM::PLANE, false);
          mma_planes<NP, NP>(s0, s1, a, f);
          ldsm_np<NP>(a, tv + TL::a_mk(lane, 16 * w, 16 * k), SM::PLANE, false);
          ldsm_np<NP>(f, tu + TL::b_nk(lane, 16 * it, 16 * k), SM::PLANE, false);
          mma_planes<NP, NP>(v0, v1, a, f);
        }
        const int i0 = 16 * it + 2 * t4;
        float col[4];  // sums over this warp's j of beta_j N_ij, columns i0, i0 + 1, i0 + 8, i0 + 9
        float Ma[4], Mb[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int ii = i0 + (e & 1) + 8 * (e >> 1);
          const float hi = cg.hi[ii], li = cg.lo[ii];
          float *s = e < 2 ? s0 : s1, *v = e < 2 ? v0 : v1;
          const int x = e & 1;
          const float da = ii >= ja ? exp2f((hi - ha) + (li - la)) : 0.f, db = ii >= ja + 8 ? exp2f((hi - hb) + (li - lb)) : 0.f;
          const float Na = ii >= ja ? s[x] * v[x] * da : 0.f, Nb = ii >= ja + 8 ? s[2 + x] * v[2 + x] * db : 0.f;
          na += Na;
          nb += Nb;
          if (it > w) {
            ca += Na;
            cb += Nb;
            col[e] = fmaf(ba, Na, bb * Nb);
          } else {
            Ma[e] = ii > ja ? ba * Na : 0.f;
            Mb[e] = ii > ja + 8 ? bb * Nb : 0.f;
          }
          s[x] = ii >= ja ? s[x] * (da * ba) : 0.f;
          v[x] = ii >= ja ? v[x] * (da * ba) : 0.f;
          s[2 + x] = ii >= ja + 8 ? s[2 + x] * (db * bb) : 0.f;
          v[2 + x] = ii >= ja + 8 ? v[2 + x] * (db * bb) : 0.f;
        }
        if (it == w) {  // the ways within the block across token t: over j < t the sums of i >= t
          auto behind = [&](float (&m)[4]) {
            float lo = m[0] + m[1], hi = m[2] + m[3];
#pragma unroll
            for (int o = 1; o < 4; o <<= 1) {
              const float l = __shfl_down_sync(0xffffffffu, lo, o, 4), u = __shfl_down_sync(0xffffffffu, hi, o, 4);
              if (t4 + o < 4) {
                lo += l;
                hi += u;
              }
            }
            const float l = __shfl_down_sync(0xffffffffu, lo, 1, 4), u = __shfl_down_sync(0xffffffffu, hi, 1, 4);
            const float upper = __shfl_sync(0xffffffffu, hi, 0, 4), lo1 = t4 == 3 ? 0.f : l, hi1 = t4 == 3 ? 0.f : u;
            m[3] += hi1;
            m[2] += m[3];
            m[1] += lo1 + upper;
            m[0] += m[1];
          };
          behind(Ma);
          behind(Mb);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int t = i0 + (e & 1) + 8 * (e >> 1);
            col[e] = (t > ja ? Ma[e] : 0.f) + (t > ja + 8 ? Mb[e] : 0.f);
          }
        }
        {  // over the eight row pairs of the warp: halve the columns that a lane carries with each exchange
          const bool up4 = lane & 4, up8 = lane & 8;
          float k0 = up4 ? col[2] : col[0], k1 = up4 ? col[3] : col[1];
          k0 += __shfl_xor_sync(0xffffffffu, up4 ? col[0] : col[2], 4);
          k1 += __shfl_xor_sync(0xffffffffu, up4 ? col[1] : col[3], 4);
          float k = up8 ? k1 : k0;
          k += __shfl_xor_sync(0xffffffffu, up8 ? k0 : k1, 8);
          k += __shfl_xor_sync(0xffffffffu, k, 16);
          if (lane < 16) (it > w ? cs.rows[w] : cs.block)[i0 + (up4 ? 8 : 0) + (up8 ? 1 : 0)] = k;
        }
        const Pk<NP> as[4] = {split_pack<NP>(s0[0], s0[1]), split_pack<NP>(s0[2], s0[3]), split_pack<NP>(s1[0], s1[1]),
                              split_pack<NP>(s1[2], s1[3])};
        const Pk<NP> av[4] = {split_pack<NP>(v0[0], v0[1]), split_pack<NP>(v0[2], v0[3]), split_pack<NP>(v1[0], v1[1]),
                              split_pack<NP>(v1[2], v1[3])};
#pragma unroll
        for (int m = 0; m < KS; ++m) {
          Pk<NP> f[4];
          ldsm_np<NP>(f, tu + TL::b_kn(lane, 16 * m, 16 * it), SM::PLANE, true);
          mma_planes<NP, NP>(dv[2 * m], dv[2 * m + 1], as, f);
          ldsm_np<NP>(f, tq + TL::b_kn(lane, 16 * m, 16 * it), SM::PLANE, true);
          mma_planes<NP, NP>(dk[2 * m], dk[2 * m + 1], av, f);
        }
      }
      na = quad_sum(na);
      nb = quad_sum(nb);
      ca = quad_sum(ca);
      cb = quad_sum(cb);
      // from the state's gradient behind the chunk
      asm volatile("bar.sync 1, %0;" ::"n"(GB_THREADS) : "memory");
      const float ta = cg.to[ja], tb = cg.to[ja + 8], wa = ta * ba, wb = tb * bb;
      Pk<NP> fr[KS][4];
#pragma unroll
      for (int k = 0; k < KS; ++k) ldsm_np<NP>(fr[k], tk + TL::a_mk(lane, 16 * w, 16 * k), SM::PLANE, false);
#pragma unroll
      for (int m = 0; m < KS; ++m) {
        float c0[4] = {}, c1[4] = {};
#pragma unroll
        for (int k = 0; k < KS; ++k) {  // (dv is a result of the inputs' type: bf16 takes the leading plane of dW)
          Pk<NP> f[4];
          ldsm_np<NP>(f, tdw + TL::b_kn(lane, 16 * m, 16 * k), TL::STATE_BYTES, true);
          mma_planes<NP, NP>(c0, c1, fr[k], f);
        }
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          dv[2 * m][x] = fmaf(x < 2 ? wa : wb, c0[x], dv[2 * m][x]);
          dv[2 * m + 1][x] = fmaf(x < 2 ? wa : wb, c1[x], dv[2 * m + 1][x]);
        }
      }
      store_rows<T, F>(static_cast<T*>(p.dv) + ((size_t)stream * p.T + t0) * F, 16 * w, rows, dv, lane);
#pragma unroll
      for (int k = 0; k < KS; ++k) ldsm_np<NP>(fr[k], tv + TL::a_mk(lane, 16 * w, 16 * k), SM::PLANE, false);
      float sa = 0.f, sb = 0.f;
#pragma unroll
      for (int m = 0; m < KS; ++m) {
        float c0[4] = {}, c1[4] = {};
#pragma unroll
        for (int k = 0; k < KS; ++k) {
          Pk<NS> f[4];
          ldsm_np<NS>(f, tdw + TL::b_nk(lane, 16 * m, 16 * k), TL::STATE_BYTES, false);
          mma_planes<NP, NS>(c0, c1, fr[k], f);
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float* c = e ? c1 : c0;
          const int col = 16 * m + 8 * e + 2 * t4;
          Pk<NP> ka, kb;
#pragma unroll
          for (int pl = 0; pl < NP; ++pl) {
            ka.p[pl] = ld_shared_b32(tk + pl * SM::PLANE + TL::off(ja, col));
            kb.p[pl] = ld_shared_b32(tk + pl * SM::PLANE + TL::off(ja + 8, col));
          }
          sa = fmaf(c[0], pk_lo(ka), fmaf(c[1], pk_hi(ka), sa));
          sb = fmaf(c[2], pk_lo(kb), fmaf(c[3], pk_hi(kb), sb));
#pragma unroll
          for (int x = 0; x < 4; ++x) dk[2 * m + e][x] = fmaf(x < 2 ? wa : wb, c[x], dk[2 * m + e][x]);
        }
      }
      store_rows<T, F>(static_cast<T*>(p.dk) + ((size_t)stream * p.T + t0) * F, 16 * w, rows, dk, lane);
      sa = quad_sum(sa) * ta;
      sb = quad_sum(sb) * tb;
      if (t4 == 0) {
        cs.s[ja] = sa * ba;
        cs.s[ja + 8] = sb * bb;
        cs.c[ja] = ca * ba;
        cs.c[ja + 8] = cb * bb;
        if (p.dbeta != nullptr) {
          float* d = p.dbeta + (size_t)stream * p.T + t0;
          if (ja < rows) d[ja] = na + sa;
          if (ja + 8 < rows) d[ja + 8] = nb + sb;
        }
      }
    }
    if (ahead) make_chunk_gates(gates[(i + 1) & 1], lane, g_next, b_next);
    ok = __syncthreads_and(ok);  // this chunk's tiles, states and sums are complete and free
    if (!ok) return;
    if (BF && tid == 0) {
      if (i + 2 < n) fetch(i + 2, 0, 4);
      if (i + 1 < n) fetch_w(i + 1);
    }
    if (tid >= GB_THREADS - 32) finish_gates(i);
  }
  if (queries && seg == 0) store_state<F>(p.dw0 + (size_t)stream * F * F, dW, row0, col0, lane);
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
  kfn<<<p.nstreams * p.nseg, GB_THREADS, smem, st>>>(maps, p);
  return cudaGetLastError();
}
cudaError_t launch_gated_bwd(int dtype, int F, const GatedMaps& maps, const GatedBwdParams& p, cudaStream_t st) {
  if (F == 64) return dtype == 1 ? launch_one<__nv_bfloat16, 64>(maps, p, st) : launch_one<float, 64>(maps, p, st);
  return dtype == 1 ? launch_one<__nv_bfloat16, 32>(maps, p, st) : launch_one<float, 32>(maps, p, st);
}

}  // namespace ttt
