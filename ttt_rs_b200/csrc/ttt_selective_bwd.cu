// Selective state space scan, backward (definitions: ttt_selective.cuh).
//
//   g = dout SiLU(z);   dh_t = C_t g_t + exp(d_{t+1} A) dh_{t+1};   e_t = dh_t exp(d_t A) h_{t-1}
//   dx = d <dh, B> + D g,   dd = <e, A> + <dh, B> x,   dA = sum_t e d,   dB = sum_channels dh d x,   dC = sum_channels g h
//   ddt = dd / (1 + exp(-dt - bias)),   dz = dout (<C, h> + D x) SiLU'(z)
// A tile of SEL_TILE tokens at a time, from the last: its states again from the saved one before it, kept in registers, then the
// gradients token by token.  Sums over a channel's states are dealt out over its lanes, sums over channels over the lanes with
// channels of their own, then over the block's warps through shared memory; the blocks' shares of dB, dC, dA, dD and the bias's
// gradient go to the workspace and are joined in a fixed order.  Segments: as in the forward, from the last token on.
#include "ttt_selective.cuh"

namespace ttt {

template <typename T, int NP, bool FULL>
struct SelBwdSmem {
  using S = SelShape<NP>;
  alignas(16) T raw[2][FULL ? 4 : 3][SEL_TILE][S::CH];  // dt, gradient of y, z, x
  alignas(16) T raw_bc[2][FULL ? 2 : 1][SEL_TILE][NP];  // c, b
  alignas(16) float4 du[SEL_TILE][S::PAIRS];            // (step, step x) of two channels
  alignas(16) float g[SEL_TILE][S::CH];
  alignas(16) float bc[FULL ? 2 : 1][SEL_TILE][NP];     // c, b
  alignas(16) float res[FULL ? 3 : 1][FULL ? SEL_TILE : 1][S::PITCH];  // <dh, B>, <e, A log2 e>, <C, h>
  alignas(16) float part[FULL ? SEL_THREADS / 32 : 1][FULL ? SEL_TILE : 1][2 * NP];  // dB, dC
};

// FULL false: a segment's gradient of its first state, from zero behind it.  MARKS: there are starts (else the kernel knows none).
template <typename T, int NP, bool FULL, bool MARKS>
__global__ void __launch_bounds__(SEL_THREADS, FULL ? 2 : 4) ttt_selective_bwd_kernel(const SelParams p) {
  using S = SelShape<NP>;
  using Smem = SelBwdSmem<T, NP, FULL>;
  extern __shared__ __align__(16) unsigned char sel_smem[];
  Smem& sm = *reinterpret_cast<Smem*>(sel_smem);
  const SelPlace<NP> at(p, FULL ? 0 : 1, FULL ? p.nseg : p.nseg - 1);
  const SelLane<NP> me;
  const T* x = static_cast<const T*>(p.x) + at.b * p.xs[0] + at.c0;
  const T* dt = static_cast<const T*>(p.dt) + at.b * p.ds[0] + at.c0;
  const T* gy = static_cast<const T*>(p.gy) + at.b * p.gs[0] + at.c0;
  const T* z = p.z != nullptr ? static_cast<const T*>(p.z) + at.b * p.zs[0] + at.c0 : nullptr;
  const T* bm = static_cast<const T*>(p.b) + at.b * p.bs[0] + at.g * p.bs[2];
  const T* cm = static_cast<const T*>(p.c) + at.b * p.cs[0] + at.g * p.cs[2];
  const uint8_t* starts = MARKS ? p.starts + at.b * p.T : nullptr;
  const int64_t tiles = (p.T + SEL_TILE - 1) / SEL_TILE;
  auto fetch = [&](int64_t t0, int k) {
    copy_rows<T, S::CH>(threadIdx.x, &sm.raw[k][0][0][0], dt, p.ds[1], t0, at.t_hi, at.have, p.xg);
    copy_rows<T, S::CH>(threadIdx.x, &sm.raw[k][1][0][0], gy, p.gs[1], t0, at.t_hi, at.have, p.xg);
    if (z != nullptr) copy_rows<T, S::CH>(threadIdx.x, &sm.raw[k][2][0][0], z, p.zs[1], t0, at.t_hi, at.have, p.xg);
    copy_rows<T, NP>(threadIdx.x, &sm.raw_bc[k][0][0][0], cm, p.cs[1], t0, at.t_hi, p.N, p.bg);
    if constexpr (FULL) {
      copy_rows<T, S::CH>(threadIdx.x, &sm.raw[k][FULL ? 3 : 0][0][0], x, p.xs[1], t0, at.t_hi, at.have, p.xg);
      copy_rows<T, NP>(threadIdx.x, &sm.raw_bc[k][FULL ? 1 : 0][0][0], bm, p.bs[1], t0, at.t_hi, p.N, p.bg);
    }
    copy_commit();
  };
  const int64_t t_last = at.t_lo + (at.t_hi - at.t_lo - 1) / SEL_TILE * SEL_TILE;
  fetch(t_last, 0);

  F2 A[S::CC][2], dh[S::CC][2];
  [[maybe_unused]] F2 dA[S::CC][2];
  me.load(A, p.A + (int64_t)at.c0 * p.N, p.N, at.have);
#pragma unroll
  for (int k = 0; k < S::CC; ++k)
#pragma unroll
    for (int i = 0; i < 2; ++i) A[k][i] = f2mul(A[k][i], f2(LOG2E)), dh[k][i] = f2(0.f);
  if constexpr (FULL) {
#pragma unroll
    for (int k = 0; k < S::CC; ++k) dA[k][0] = dA[k][1] = f2(0.f);
    me.load(dh, p.gstate_out != nullptr ? p.gstate_out + (at.b * p.C + at.c0) * p.N : nullptr, p.N, at.have);
    for (int j = p.nseg - 1; j > at.seg; --j) {  // the segments behind, from the last
      const int64_t row = (at.b * p.nseg + j) * p.C + at.c0;
      F2 own[S::CC][2];
      me.load_padded(own, p.seg_state + row * NP, at.have);
#pragma unroll
      for (int k = 0; k < S::CC; ++k) {
        const float sum = me.ch + k < at.have ? p.seg_sum[row + me.ch + k] : 0.f;
        const bool cut = sum == INFINITY;
#pragma unroll
        for (int i = 0; i < 2; ++i) dh[k][i] = cut ? own[k][i] : f2fma(ex2(f2mul(A[k][i], f2(sum))), dh[k][i], own[k][i]);
      }
    }
  }
  const int pr = threadIdx.x % S::PAIRS, row0 = threadIdx.x / S::PAIRS, pair_have = at.have - 2 * pr;
  float2 bias = make_float2(0.f, 0.f), skip = make_float2(0.f, 0.f);
  if (p.bias != nullptr) {
    if (pair_have > 0) bias.x = p.bias[at.c0 + 2 * pr];
    if (pair_have > 1) bias.y = p.bias[at.c0 + 2 * pr + 1];
  }
  if (FULL && p.D != nullptr) {
    if (pair_have > 0) skip.x = p.D[at.c0 + 2 * pr];
    if (pair_have > 1) skip.y = p.D[at.c0 + 2 * pr + 1];
  }
  const bool whole = pair_have > 1 && p.xg >= 4 && (sizeof(T) == 2 || p.xg == 16);
  float2 s0 = make_float2(0.f, 0.f), s1 = make_float2(0.f, 0.f);  // FULL: of dD and the bias's gradient; else of steps
  bool any_start = false;

  int buf = 0;
  for (int64_t t0 = t_last; t0 >= at.t_lo; t0 -= SEL_TILE, buf ^= 1) {
    uint32_t mark = 0;
    if constexpr (MARKS) {
      const int64_t t = t0 + (me.lane & (SEL_TILE - 1));
      mark = __ballot_sync(0xffffffffu, t < at.t_hi && starts[t] != 0) & ((1u << SEL_TILE) - 1);
      any_start = any_start || mark != 0;
    }
    [[maybe_unused]] F2 h[S::CC][2];
    if constexpr (FULL) me.load_padded(h, p.saved + ((at.b * tiles + t0 / SEL_TILE) * p.C + at.c0) * NP, at.have);
    copy_wait_all();
    __syncthreads();
    if (t0 - SEL_TILE >= at.t_lo) fetch(t0 - SEL_TILE, buf ^ 1);
#pragma unroll
    for (int r = row0; r < SEL_TILE; r += S::ROWS) {
      const float2 dv = pair_of(&sm.raw[buf][0][r][2 * pr]);
      float2 gv = pair_of(&sm.raw[buf][1][r][2 * pr]);
      F2 d = f2add(dv, bias);
      if (p.softplus) d = softplus_of(d);
      if (t0 + r >= at.t_hi || pair_have < 1) d.x = 0.f;
      if (t0 + r >= at.t_hi || pair_have < 2) d.y = 0.f;
      if (z != nullptr) {
        const float2 zv = pair_of(&sm.raw[buf][2][r][2 * pr]);
        gv.x *= act_of(zv.x, ACT_SILU), gv.y *= act_of(zv.y, ACT_SILU);
      }
      float2 xv = make_float2(0.f, 0.f);
      if constexpr (FULL) xv = pair_of(&sm.raw[buf][FULL ? 3 : 0][r][2 * pr]);
      else s0.x += d.x, s0.y += d.y;
      sm.du[r][pr] = make_float4(d.x, d.x * xv.x, d.y, d.y * xv.y);
      *reinterpret_cast<float2*>(&sm.g[r][2 * pr]) = gv;
    }
#pragma unroll
    for (int i = threadIdx.x; i < (FULL ? 2 : 1) * SEL_TILE * NP; i += SEL_THREADS)
      (&sm.bc[0][0][0])[i] = ld_as_float<T>(&sm.raw_bc[buf][0][0][0], i);
    __syncthreads();
    auto steps = [&](int r) {
      if constexpr (S::CC == 2) {
        return sm.du[r][me.ch / 2];
      } else {
        const float2 one = *reinterpret_cast<const float2*>(reinterpret_cast<const float*>(&sm.du[r][0]) + 2 * me.ch);
        return make_float4(one.x, one.y, 0.f, 0.f);
      }
    };
    auto grads = [&](int r) {
      if constexpr (S::CC == 2) return *reinterpret_cast<const float2*>(&sm.g[r][me.ch]);
      else return make_float2(sm.g[r][me.ch], 0.f);
    };
    if constexpr (!FULL) {
#pragma unroll 4
      for (int r = SEL_TILE - 1; r >= 0; --r) {
        const float4 q = steps(r), c = *reinterpret_cast<const float4*>(&sm.bc[0][r][4 * me.sl]);
        const float2 g = grads(r);
#pragma unroll
        for (int k = 0; k < S::CC; ++k) {
          const F2 d = f2(k ? q.z : q.x), gk = f2(k ? g.y : g.x);
          dh[k][0] = f2mul(f2fma(gk, f2(c.x, c.y), dh[k][0]), ex2(f2mul(A[k][0], d)));
          dh[k][1] = f2mul(f2fma(gk, f2(c.z, c.w), dh[k][1]), ex2(f2mul(A[k][1], d)));
        }
        if (MARKS && mark >> r & 1) {
#pragma unroll
          for (int k = 0; k < S::CC; ++k) dh[k][0] = dh[k][1] = f2(0.f);
        }
      }
    } else {
      F2 before[SEL_TILE][S::CC][2];  // the state that token r finds
#pragma unroll
      for (int r = 0; r < SEL_TILE; ++r) {
        const float4 q = steps(r), b = *reinterpret_cast<const float4*>(&sm.bc[FULL ? 1 : 0][r][4 * me.sl]);
#pragma unroll
        for (int k = 0; k < S::CC; ++k) {
          const F2 d = f2(k ? q.z : q.x), v = f2(k ? q.w : q.y);
          before[r][k][0] = h[k][0], before[r][k][1] = h[k][1];
          if (MARKS && mark >> r & 1) h[k][0] = h[k][1] = f2(0.f);
          h[k][0] = f2fma(ex2(f2mul(A[k][0], d)), h[k][0], f2mul(v, f2(b.x, b.y)));
          h[k][1] = f2fma(ex2(f2mul(A[k][1], d)), h[k][1], f2mul(v, f2(b.z, b.w)));
        }
      }
      constexpr int DEAL = S::SL > 4 ? 4 : S::SL > S::CC ? S::SL : S::CC, TOKENS = DEAL / S::CC;
#pragma unroll
      for (int r0 = SEL_TILE - TOKENS; r0 >= 0; r0 -= TOKENS) {
        float into[DEAL], rate[DEAL], yd[DEAL];
#pragma unroll
        for (int u = TOKENS - 1; u >= 0; --u) {
          const int r = r0 + u;
          const float4 q = steps(r);
          const float4 c = *reinterpret_cast<const float4*>(&sm.bc[0][r][4 * me.sl]), b = *reinterpret_cast<const float4*>(&sm.bc[FULL ? 1 : 0][r][4 * me.sl]);
          const float2 g = grads(r);
          const F2 cv[2] = {f2(c.x, c.y), f2(c.z, c.w)}, bv[2] = {f2(b.x, b.y), f2(b.z, b.w)};
          F2 db[2], dc[2];
#pragma unroll
          for (int k = 0; k < S::CC; ++k) {
            const F2 d = f2(k ? q.z : q.x), v = f2(k ? q.w : q.y), gk = f2(k ? g.y : g.x);
            F2 in, ra, ys;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              dh[k][i] = f2fma(gk, cv[i], dh[k][i]);
              db[i] = k ? f2fma(dh[k][i], v, db[i]) : f2mul(dh[k][i], v);
              dc[i] = k ? f2fma(gk, h[k][i], dc[i]) : f2mul(gk, h[k][i]);
              in = i ? f2fma(dh[k][i], bv[i], in) : f2mul(dh[k][i], bv[i]);
              ys = i ? f2fma(h[k][i], cv[i], ys) : f2mul(h[k][i], cv[i]);
              dh[k][i] = f2mul(dh[k][i], ex2(f2mul(A[k][i], d)));
              h[k][i] = before[r][k][i];
              F2 way = f2mul(dh[k][i], h[k][i]);
              if (MARKS && mark >> r & 1) dh[k][i] = way = f2(0.f);
              ra = i ? f2fma(way, A[k][i], ra) : f2mul(way, A[k][i]);
              dA[k][i] = f2fma(way, d, dA[k][i]);
            }
            into[u * S::CC + k] = f2hsum(in);
            rate[u * S::CC + k] = f2hsum(ra);
            yd[u * S::CC + k] = f2hsum(ys);
          }
          float sums[8] = {db[0].x, db[0].y, db[1].x, db[1].y, dc[0].x, dc[0].y, dc[1].x, dc[1].y};
          sum_and_deal<8, S::CL, S::SL>(sums, me.lane);
          // lane cl has sums [cl 8 / CL, ...); more lanes than sums: one each of lanes 0, CL / 8, ...
          constexpr int GOT = S::CL >= 8 ? 1 : 8 / S::CL, SHARED = S::CL >= 8 ? S::CL / 8 : 1;
          const int cl = me.lane / S::SL, first = S::CL >= 8 ? cl / SHARED : cl * GOT;
          if (SHARED == 1 || cl % SHARED == 0) {
#pragma unroll
            for (int i = 0; i < GOT; ++i) {
              const int e = first + i;  // dB of states 4 sl .. 4 sl + 3, then dC of them
              sm.part[threadIdx.x >> 5][r][(e >= 4 ? NP : 0) + 4 * me.sl + (e & 3)] = sums[i];
            }
          }
        }
        sum_and_deal<DEAL, S::SL, 1>(into, me.lane);
        sum_and_deal<DEAL, S::SL, 1>(rate, me.lane);
        sum_and_deal<DEAL, S::SL, 1>(yd, me.lane);
        if constexpr (S::SL == 1) {
          sm.res[0][r0][me.ch] = into[0], sm.res[1][r0][me.ch] = rate[0], sm.res[2][r0][me.ch] = yd[0];
        } else {
          constexpr int EACH = S::SL / DEAL;  // lanes with the same result
          const int e = me.sl / EACH, r = r0 + e / S::CC, c = me.ch + e % S::CC;
          if (EACH == 1 || me.sl % EACH == 0) sm.res[0][r][c] = into[0], sm.res[1][r][c] = rate[0], sm.res[2][r][c] = yd[0];
        }
      }
      __syncthreads();
#pragma unroll
      for (int r = row0; r < SEL_TILE; r += S::ROWS) {
        if (t0 + r >= at.t_hi || pair_have < 1) continue;
        const float2 xv = pair_of(&sm.raw[buf][FULL ? 3 : 0][r][2 * pr]), dv = pair_of(&sm.raw[buf][0][r][2 * pr]);
        const float2 go = pair_of(&sm.raw[buf][1][r][2 * pr]), gv = *reinterpret_cast<const float2*>(&sm.g[r][2 * pr]);
        const float2 in = *reinterpret_cast<const float2*>(&sm.res[0][r][2 * pr]), ra = *reinterpret_cast<const float2*>(&sm.res[1][r][2 * pr]);
        const float4 q = sm.du[r][pr];
        float2 sig = make_float2(1.f, 1.f);
        if (p.softplus) sig = make_float2(sigmoid_of(dv.x + bias.x), sigmoid_of(dv.y + bias.y));
        const float2 dx = make_float2(fmaf(skip.x, gv.x, q.x * in.x), fmaf(skip.y, gv.y, q.z * in.y));
        const float2 dd = make_float2(fmaf(LN2, ra.x, in.x * xv.x) * sig.x, fmaf(LN2, ra.y, in.y * xv.y) * sig.y);
        s0.x = fmaf(gv.x, xv.x, s0.x), s0.y = fmaf(gv.y, xv.y, s0.y);
        s1.x += dd.x, s1.y += dd.y;
        const int64_t row = (at.b * p.T + t0 + r) * p.C + at.c0 + 2 * pr;
        put_pair<T>(static_cast<T*>(p.gx) + row, dx, pair_have, whole);
        put_pair<T>(static_cast<T*>(p.gdt) + row, dd, pair_have, whole);
        if (z != nullptr) {
          const float2 zv = pair_of(&sm.raw[buf][2][r][2 * pr]), yv = *reinterpret_cast<const float2*>(&sm.res[2][r][2 * pr]);
          float2 slope;
          act_and_slope(zv.x, ACT_SILU, slope.x), act_and_slope(zv.y, ACT_SILU, slope.y);
          put_pair<T>(static_cast<T*>(p.gz) + row, make_float2(go.x * fmaf(skip.x, xv.x, yv.x) * slope.x, go.y * fmaf(skip.y, xv.y, yv.y) * slope.y),
                      pair_have, whole);
        }
      }
      const int blocks = (p.C / p.G + S::CH - 1) / S::CH;
      float* out = p.part_bc + (((at.b * p.G + at.g) * blocks + at.block) * p.T + t0) * 2 * NP;
#pragma unroll
      for (int i = threadIdx.x; i < SEL_TILE * 2 * NP; i += SEL_THREADS) {
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < SEL_THREADS / 32; ++w) v += (&sm.part[w][0][0])[i];
        if (t0 + i / (2 * NP) < at.t_hi) out[i] = v;
      }
    }
  }
  float* sums = reinterpret_cast<float*>(&sm.du[0][0]);  // [2][ROWS][CH], or [ROWS][CH]
  __syncthreads();
  sums[row0 * S::CH + 2 * pr] = s0.x;
  sums[row0 * S::CH + 2 * pr + 1] = s0.y;
  if constexpr (FULL) {
    sums[(S::ROWS + row0) * S::CH + 2 * pr] = s1.x;
    sums[(S::ROWS + row0) * S::CH + 2 * pr + 1] = s1.y;
  }
  __syncthreads();
  const int64_t row = at.b * p.nseg + at.seg;
  for (int i = threadIdx.x; i < (FULL ? 2 : 1) * at.have; i += SEL_THREADS) {
    const int m = i / at.have, c = i - m * at.have;
    float v = 0.f;
    for (int r = 0; r < S::ROWS; ++r) v += sums[(m * S::ROWS + r) * S::CH + c];
    if constexpr (FULL) p.part_d[(row * 2 + m) * p.C + at.c0 + c] = v;
    else p.seg_sum[row * p.C + at.c0 + c] = any_start ? INFINITY : v;
  }
  if constexpr (FULL) {
    me.store(dA, p.part_a + (row * p.C + at.c0) * NP, NP, at.have);
    if (at.seg == 0 && p.gstate != nullptr) me.store(dh, p.gstate + (at.b * p.C + at.c0) * p.N, p.N, at.have);
  } else {
    me.store(dh, p.seg_state + (row * p.C + at.c0) * NP, NP, at.have);
  }
}

// The blocks' shares of dB and dC, [B][G][blocks][T][2][NP] -> [B][T][G][N] each
template <typename T>
__global__ void __launch_bounds__(256) ttt_selective_bc_kernel(const SelParams p, int NP, int blocks) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;  // (b G + g) T 2 NP + t 2 NP + ...
  const int64_t per = p.T * 2 * NP;
  if (i >= p.B * p.G * per) return;
  const int64_t bg = i / per, e = i - bg * per;
  const float* src = p.part_bc + bg * blocks * per + e;
  float v = 0.f;
  for (int k = 0; k < blocks; ++k) v += src[k * per];
  const int64_t t = e / (2 * NP);
  const int n = (int)(e - t * 2 * NP), which = n / NP, s = n - which * NP;
  if (s >= p.N) return;
  const int64_t b = bg / p.G, g = bg - b * p.G;
  st_from_float<T>(which ? p.gc : p.gb, ((b * p.T + t) * p.G + g) * p.N + s, v);
}
// rows of partial sums [rows][pitch] (row r at r row_pitch) -> out: [n / NP][N] of [n / NP][NP]
__global__ void __launch_bounds__(256) ttt_selective_rows_kernel(const float* partials, int64_t rows, int64_t row_pitch, int64_t n, int NP, int N,
                                                                 float* out) {
  __shared__ float part[8][33];
  const int64_t col = (int64_t)blockIdx.x * 32 + (threadIdx.x & 31);
  const int share = threadIdx.x >> 5;
  float v = 0.f;
  if (col < n)
    for (int64_t r = share; r < rows; r += 8) v += partials[r * row_pitch + col];
  part[share][threadIdx.x & 31] = v;
  __syncthreads();
  if (share != 0 || col >= n) return;
#pragma unroll
  for (int k = 1; k < 8; ++k) v += part[k][threadIdx.x & 31];
  const int64_t c = col / NP;
  const int s = (int)(col - c * NP);
  if (s < N) out[c * N + s] = v;
}

template <typename T, int NP, bool FULL>
static cudaError_t run(const SelParams& p, int64_t blocks, cudaStream_t st) {
  constexpr int bytes = sizeof(SelBwdSmem<T, NP, FULL>);
  void (*kernel)(SelParams) = p.starts != nullptr ? ttt_selective_bwd_kernel<T, NP, FULL, true> : ttt_selective_bwd_kernel<T, NP, FULL, false>;
  if (bytes > 48 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != cudaSuccess) return e;
  }
  kernel<<<(unsigned)blocks, SEL_THREADS, bytes, st>>>(p);
  return cudaGetLastError();
}
template <typename T, int NP>
static cudaError_t run_all(const SelParams& p, cudaStream_t st) {
  const int each = p.C / p.G, channel_blocks = (each + SelShape<NP>::CH - 1) / SelShape<NP>::CH;
  const int64_t blocks = p.B * p.G * channel_blocks, rows = p.B * p.nseg;
  cudaError_t e;
  if (p.nseg > 1 && (e = run<T, NP, false>(p, blocks * (p.nseg - 1), st)) != cudaSuccess) return e;
  if ((e = run<T, NP, true>(p, blocks * p.nseg, st)) != cudaSuccess) return e;
  ttt_selective_bc_kernel<T><<<(unsigned)((p.B * p.G * p.T * 2 * NP + 255) / 256), 256, 0, st>>>(p, NP, channel_blocks);
  if ((e = cudaGetLastError()) != cudaSuccess) return e;
  const int64_t n = (int64_t)p.C * NP;
  ttt_selective_rows_kernel<<<(unsigned)((n + 31) / 32), 256, 0, st>>>(p.part_a, rows, n, n, NP, p.N, p.ga);
  if ((e = cudaGetLastError()) != cudaSuccess) return e;
  for (int m = 0; m < 2; ++m) {
    float* out = m ? p.gbias : p.gd;
    if (out == nullptr) continue;
    ttt_selective_rows_kernel<<<(p.C + 31) / 32, 256, 0, st>>>(p.part_d + m * p.C, rows, 2 * (int64_t)p.C, p.C, 1, 1, out);
    if ((e = cudaGetLastError()) != cudaSuccess) return e;
  }
  return cudaSuccess;
}
template <typename T>
static cudaError_t run_np(const SelParams& p, cudaStream_t st) {
  switch (sel_padded(p.N)) {
    case 4: return run_all<T, 4>(p, st);
    case 8: return run_all<T, 8>(p, st);
    case 16: return run_all<T, 16>(p, st);
    case 32: return run_all<T, 32>(p, st);
    default: return run_all<T, 64>(p, st);
  }
}
cudaError_t launch_selective_bwd(int dtype, const SelParams& p, cudaStream_t st) {
  return dtype == 1 ? run_np<__nv_bfloat16>(p, st) : run_np<float>(p, st);
}

}  // namespace ttt
