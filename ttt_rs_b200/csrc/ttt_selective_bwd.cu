// Selective state space scan, backward (definitions: ttt_selective.cuh).
//
//   g = dout SiLU(z);   dh_t = C_t g_t + exp(d_{t+1} A) dh_{t+1};   e_t = dh_t exp(d_t A) h_{t-1}
//   dx = d <dh, B> + D g,   dd = <e, A> + <dh, B> x,   dA = sum_t e d,   dB = sum_channels dh d x,   dC = sum_channels g h
//   ddt = dd / (1 + exp(-dt - bias)),   dz = dout (<C, h> + D x) SiLU'(z)
// Half a tile of SEL_TILE tokens at a time, from the last: its states again from the saved one before the tile, every second one
// kept in registers, like all decays, then the gradients token by token.  Sums over channels are dealt out over the lanes with channels
// of their own, then joined over the block's scanning warps through shared memory; a channel's shares of its sums over states go to the
// other warps through shared memory; the blocks' shares of dB, dC, dA, dD and the bias's gradient go to the workspace and are joined in
// a fixed order.  Segments: as in the forward, from the last token on.
//
// bf16, 16 x 2048 tokens of 1536 channels, 16 states: 1198 us (+ 22 us for dB and dC over the 24 blocks of channels), from 2349 us with
// all warps doing everything.  Whole tiles at once, twice the code: 1647 us, a quarter of the stalls instruction fetches; halves, which
// walk the first half's states once more: 1345 us.  Steps and gradients once instead of twice in shared memory, 12 of 50 wavefronts per
// token: 1329 -> 1243 us.  Registers for three blocks per SM (no decays kept): 1196 us for these 384 blocks, but 399 us instead of 343
// for an SM's every block.  Without the sums over channels 230 us less, without the results' pass 190, without the tiles' 125: no part
// is the whole of it.
#include "ttt_selective.cuh"

namespace ttt {

constexpr int SEL_HALF = SEL_TILE / 2;

template <typename T, int NP>
struct SelBwdSmem {
  using S = SelShape<NP>;
  alignas(16) T raw[SEL_STAGES][4][SEL_TILE][S::CH];    // dt, gradient of y, z, x
  alignas(16) T raw_bc[SEL_STAGES][2][SEL_TILE][NP];    // c, b
  alignas(16) float2 du[2][SEL_TILE][S::CH];            // step, step x
  alignas(16) float g[2][SEL_TILE][S::CH];              // gradient of the result before the gate
  alignas(16) float bc[2][2][SEL_TILE][NP];             // c, b
  alignas(16) float res[2][3][SEL_HALF][S::SHARES]; // shares of <dh, B>, <e, A log2 e>, <C, h>, as the scanning lanes lie
  alignas(16) float part[2][SEL_THREADS / 32][SEL_HALF][2 * NP];  // dB, dC
  uint32_t mark[2];
};

// The state's gradient behind a segment: the given one, and what the segments behind carry back, from the last
template <int NP>
__device__ __forceinline__ void gradient_behind(F2 (&dh)[SelShape<NP>::CC][2], const F2 (&A)[SelShape<NP>::CC][2], const SelLane<NP>& me,
                                                const SelPlace<NP>& at, const SelParams& p) {
  using S = SelShape<NP>;
  me.load(dh, p.gstate_out != nullptr ? p.gstate_out + (at.b * p.C + at.c0) * p.N : nullptr, p.N, at.have);
  for (int j = p.nseg - 1; j > at.seg; --j) {
    const int64_t row = (at.b * p.nseg + j) * p.C + at.c0;
    F2 own[S::CC][2];
    me.load_padded(own, p.seg_state + row * NP, at.have);
#pragma unroll
    for (int k = 0; k < S::CC; ++k) {
      const float sum = me.ch + k < at.have ? p.seg_sum[row + me.ch + k] : 0.f;
      const bool cut = sum == INFINITY;
#pragma unroll
      for (int i = 0; i < 2; ++i) dh[k][i] = cut ? own[k][i] : f2fma(decay_of(A[k][i], sum), dh[k][i], own[k][i]);
    }
  }
}

// The launch's 128 registers per thread are shared out: the scanning warps take 176, the others keep 80; with MARKS 200 and
// 56, for 176 spill there (16 x 2048 x 1536, bf16: 1503 us against 1806; without starts 32 and 64 states spill 64 and 32 bytes).
// build.py checks the 128.
// MARKS: there are starts (else the kernel knows none).
template <typename T, int NP, bool MARKS>
__global__ void __launch_bounds__(2 * SEL_THREADS, 2) ttt_selective_bwd_kernel(const SelParams p) {
  using S = SelShape<NP>;
  using Smem = SelBwdSmem<T, NP>;
  extern __shared__ __align__(16) unsigned char sel_smem[];
  Smem& sm = *reinterpret_cast<Smem*>(sel_smem);
  const SelPlace<NP> at(p, 0, p.nseg);
  const int tiles = (int)((at.t_hi - at.t_lo + SEL_TILE - 1) / SEL_TILE);
  if (threadIdx.x < SEL_THREADS) {
    // ---- scan
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(MARKS ? 200 : 176));
    const SelLane<NP> me;
    const int my_share = share_at<NP>(me.ch / S::CC, me.sl);
    F2 A[S::CC][2], dh[S::CC][2], dA[S::CC][2];
    me.load_rates(A, p.A + (int64_t)at.c0 * p.N, p.N, at.have);
#pragma unroll
    for (int k = 0; k < S::CC; ++k) dA[k][0] = dA[k][1] = f2(0.f);
    gradient_behind<NP>(dh, A, me, at, p);
    const float* saved = p.saved + ((at.b * ((p.T + SEL_TILE - 1) / SEL_TILE) + at.t_lo / SEL_TILE + tiles - 1) * p.C + at.c0) * NP;
    F2 next[S::CC][2];
    me.load_padded(next, saved, at.have);
    __syncthreads();
    for (int i = 0; i < tiles; ++i) {
      const uint32_t marks = MARKS ? sm.mark[i & 1] : 0;
      F2 h0[S::CC][2];
#pragma unroll
      for (int k = 0; k < S::CC; ++k) h0[k][0] = next[k][0], h0[k][1] = next[k][1];
      if (i + 1 < tiles) {
        saved -= (int64_t)p.C * NP;
        me.load_padded(next, saved, at.have);
      }
#pragma unroll 1
      for (int half = 1; half >= 0; --half) {
        const int k2 = half ^ 1;  // results alternate
        F2 h[S::CC][2], before[SEL_HALF / 2][S::CC][2];  // the states that the half's tokens 0, 2, 4, 6 find
        F2 decay[SEL_HALF][S::CC][2], dA_half[S::CC][2];  // (sums of sums: thousands of tokens one by one would lose ten times as much)
#pragma unroll
        for (int k = 0; k < S::CC; ++k) dA_half[k][0] = dA_half[k][1] = f2(0.f);
#pragma unroll
        for (int k = 0; k < S::CC; ++k) h[k][0] = h0[k][0], h[k][1] = h0[k][1];
        const float2* du = &sm.du[i & 1][0][me.ch];
        const float* bp = &sm.bc[i & 1][1][0][4 * me.sl];
        uint32_t mark = marks;
        auto channels = [&](float2 (&q)[S::CC], const float2* at) {  // of the thread's channels
          if constexpr (S::CC == 2) {
            const float4 e = *reinterpret_cast<const float4*>(at);
            q[0] = make_float2(e.x, e.y), q[1] = make_float2(e.z, e.w);
          } else {
            q[0] = *at;
          }
        };
        auto step = [&](int r, F2 (&a)[S::CC][2]) {
          const float4 b = *reinterpret_cast<const float4*>(bp + r * NP);
          float2 q[S::CC];
          channels(q, du + r * S::CH);
#pragma unroll
          for (int k = 0; k < S::CC; ++k) {
            if (MARKS && mark >> r & 1) h[k][0] = h[k][1] = f2(0.f);
#pragma unroll
            for (int n = 0; n < 2; ++n) {
              a[k][n] = decay_of(A[k][n], q[k].x);
              h[k][n] = f2fma(a[k][n], h[k][n], f2mul(f2(q[k].y), n ? f2(b.z, b.w) : f2(b.x, b.y)));
            }
          }
        };
        if (half) {
#pragma unroll 4
          for (int r = 0; r < SEL_HALF; ++r) step(r, decay[0]);
          du += SEL_HALF * S::CH;
          bp += SEL_HALF * NP;
          mark >>= SEL_HALF;
        }
        const float* cp = bp - SEL_TILE * NP;
        const float* gp = &sm.g[i & 1][half * SEL_HALF][me.ch];
#pragma unroll
        for (int r = 0; r < SEL_HALF; ++r) {
          if (r % 4 == 0) asm volatile("" ::: "memory");  // (the loads of all tokens at once would not fit in the registers)
          if (r % 2 == 0)
#pragma unroll
            for (int k = 0; k < S::CC; ++k) before[r / 2][k][0] = h[k][0], before[r / 2][k][1] = h[k][1];
          step(r, decay[r]);
        }
#pragma unroll
        for (int r0 = SEL_HALF - 2; r0 >= 0; r0 -= 2) {
          asm volatile("" ::: "memory");
          F2 mid[S::CC][2];  // the state behind token r0
          {
            const float4 b = *reinterpret_cast<const float4*>(bp + r0 * NP);
            float2 q[S::CC];
            channels(q, du + r0 * S::CH);
#pragma unroll
            for (int k = 0; k < S::CC; ++k) {
#pragma unroll
              for (int n = 0; n < 2; ++n) {
                mid[k][n] = f2mul(f2(q[k].y), n ? f2(b.z, b.w) : f2(b.x, b.y));
                if (!(MARKS && mark >> r0 & 1)) mid[k][n] = f2fma(decay[r0][k][n], before[r0 / 2][k][n], mid[k][n]);
              }
            }
          }
#pragma unroll
          for (int u = 1; u >= 0; --u) {
            const int r = r0 + u;
            const float4 c = *reinterpret_cast<const float4*>(cp + r * NP), b = *reinterpret_cast<const float4*>(bp + r * NP);
            const F2 cv[2] = {f2(c.x, c.y), f2(c.z, c.w)}, bv[2] = {f2(b.x, b.y), f2(b.z, b.w)};
            float2 q[S::CC];
            channels(q, du + r * S::CH);
            float g[S::CC];
            if constexpr (S::CC == 2) {
              const float2 e = *reinterpret_cast<const float2*>(gp + r * S::CH);
              g[0] = e.x, g[1] = e.y;
            } else {
              g[0] = gp[r * S::CH];
            }
            F2 db[2], dc[2];
            float share[3][S::CC];
#pragma unroll
            for (int k = 0; k < S::CC; ++k) {
              const F2 d = f2(q[k].x), v = f2(q[k].y), gk = f2(g[k]);
              F2 in, ra, ys;
#pragma unroll
              for (int n = 0; n < 2; ++n) {
                dh[k][n] = f2fma(gk, cv[n], dh[k][n]);
                db[n] = k ? f2fma(dh[k][n], v, db[n]) : f2mul(dh[k][n], v);
                dc[n] = k ? f2fma(gk, h[k][n], dc[n]) : f2mul(gk, h[k][n]);
                in = n ? f2fma(dh[k][n], bv[n], in) : f2mul(dh[k][n], bv[n]);
                ys = n ? f2fma(h[k][n], cv[n], ys) : f2mul(h[k][n], cv[n]);
                h[k][n] = u ? mid[k][n] : before[r0 / 2][k][n];
                dh[k][n] = f2mul(dh[k][n], decay[r][k][n]);
                F2 way = f2mul(dh[k][n], h[k][n]);
                if (MARKS && mark >> r & 1) dh[k][n] = way = f2(0.f);
                ra = n ? f2fma(way, A[k][n], ra) : f2mul(way, A[k][n]);
                dA_half[k][n] = f2fma(way, d, dA_half[k][n]);
              }
              share[0][k] = f2hsum(in);
              share[1][k] = f2hsum(ra);
              share[2][k] = f2hsum(ys);
            }
#pragma unroll
            for (int m = 0; m < 3; ++m) {
              if constexpr (S::CC == 2) *reinterpret_cast<float2*>(&sm.res[k2][m][r][my_share]) = make_float2(share[m][0], share[m][1]);
              else sm.res[k2][m][r][my_share] = share[m][0];
            }
            float sums[8] = {db[0].x, db[0].y, db[1].x, db[1].y, dc[0].x, dc[0].y, dc[1].x, dc[1].y};
            sum_and_deal<8, S::CL, S::SL>(sums, me.lane);
            // lane cl has sums [cl 8 / CL, ...); more lanes than sums: one each of lanes 0, CL / 8, ...
            constexpr int GOT = S::CL >= 8 ? 1 : 8 / S::CL, SHARED = S::CL >= 8 ? S::CL / 8 : 1;
            const int cl = me.lane / S::SL, first = S::CL >= 8 ? cl / SHARED : cl * GOT;
            if (SHARED == 1 || cl % SHARED == 0) {
#pragma unroll
              for (int e0 = 0; e0 < GOT; ++e0) {
                const int e = first + e0;  // dB of states 4 sl .. 4 sl + 3, then dC of them
                sm.part[k2][threadIdx.x >> 5][r][(e >= 4 ? NP : 0) + 4 * me.sl + (e & 3)] = sums[e0];
              }
            }
          }
        }
#pragma unroll
        for (int k = 0; k < S::CC; ++k) dA[k][0] = f2add(dA[k][0], dA_half[k][0]), dA[k][1] = f2add(dA[k][1], dA_half[k][1]);
        __syncthreads();
      }
    }
    me.store(dA, p.part_a + ((at.b * p.nseg + at.seg) * p.C + at.c0) * NP, NP, at.have);
    if (at.seg == 0 && p.gstate != nullptr) me.store(dh, p.gstate + (at.b * p.C + at.c0) * p.N, p.N, at.have);
    return;
  }
  // ---- what is done once per token and channel, pair of channels by pair
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(MARKS ? 56 : 80));
  const int tid = threadIdx.x - SEL_THREADS, pr = tid % S::PAIRS, row0 = tid / S::PAIRS, pair_have = at.have - 2 * pr;
  bool first[2] = {false, false};  // lane r of a warp: a start at token r of the next tile to be made ready, and of the one behind it
  auto fetch = [&](int i) {
    const int k = i % SEL_STAGES;
    const int64_t t0 = at.t_lo + (int64_t)(tiles - 1 - i) * SEL_TILE;
    copy_rows<T, S::CH, 1>(tid, &sm.raw[k][0][0][0], static_cast<const T*>(p.dt) + at.b * p.ds[0] + at.c0, p.ds[1], t0, at.t_hi, at.have, p.xg);
    copy_rows<T, S::CH, 1>(tid, &sm.raw[k][1][0][0], static_cast<const T*>(p.gy) + at.b * p.gs[0] + at.c0, p.gs[1], t0, at.t_hi, at.have, p.xg);
    if (p.z != nullptr)
      copy_rows<T, S::CH, 1>(tid, &sm.raw[k][2][0][0], static_cast<const T*>(p.z) + at.b * p.zs[0] + at.c0, p.zs[1], t0, at.t_hi, at.have, p.xg);
    copy_rows<T, S::CH, 1>(tid, &sm.raw[k][3][0][0], static_cast<const T*>(p.x) + at.b * p.xs[0] + at.c0, p.xs[1], t0, at.t_hi, at.have, p.xg);
    copy_rows<T, NP, 1>(tid, &sm.raw_bc[k][0][0][0], static_cast<const T*>(p.c) + at.b * p.cs[0] + at.g * p.cs[2], p.cs[1], t0, at.t_hi, p.N, p.bg);
    copy_rows<T, NP, 1>(tid, &sm.raw_bc[k][1][0][0], static_cast<const T*>(p.b) + at.b * p.bs[0] + at.g * p.bs[2], p.bs[1], t0, at.t_hi, p.N, p.bg);
    copy_commit();
    if constexpr (MARKS) {
      const int64_t t = t0 + (tid & 31);
      first[1] = (tid & 31) < SEL_TILE && t < at.t_hi && p.starts[at.b * p.T + t] != 0;
    }
  };
  float2 bias = make_float2(0.f, 0.f), skip = make_float2(0.f, 0.f);
  if (p.bias != nullptr) {
    if (pair_have > 0) bias.x = p.bias[at.c0 + 2 * pr];
    if (pair_have > 1) bias.y = p.bias[at.c0 + 2 * pr + 1];
  }
  if (p.D != nullptr) {
    if (pair_have > 0) skip.x = p.D[at.c0 + 2 * pr];
    if (pair_have > 1) skip.y = p.D[at.c0 + 2 * pr + 1];
  }
  const bool whole = pair_have > 1 && p.xg >= 4 && (sizeof(T) == 2 || p.xg == 16);
  float2 s0 = make_float2(0.f, 0.f), s1 = make_float2(0.f, 0.f);  // of dD and of the bias's gradient
  auto make_ready = [&](int i) {
    const int k = i % SEL_STAGES, left = (int)(at.t_hi - at.t_lo) - (tiles - 1 - i) * SEL_TILE;
#pragma unroll(MARKS ? 2 : SEL_TILE)
    for (int r = row0; r < SEL_TILE; r += S::ROWS) {
      F2 d = f2add(pair_of(&sm.raw[k][0][r][2 * pr]), bias), gv = pair_of(&sm.raw[k][1][r][2 * pr]);
      if (p.softplus) d = softplus_of(d);
      if (r >= left || pair_have < 1) d.x = 0.f;
      if (r >= left || pair_have < 2) d.y = 0.f;
      if (p.z != nullptr) {
        const float2 zv = pair_of(&sm.raw[k][2][r][2 * pr]);
        gv = f2mul(gv, f2(act_of(zv.x, ACT_SILU), act_of(zv.y, ACT_SILU)));
      }
      const F2 v = f2mul(d, pair_of(&sm.raw[k][3][r][2 * pr]));
      *reinterpret_cast<float4*>(&sm.du[i & 1][r][2 * pr]) = make_float4(d.x, v.x, d.y, v.y);
      *reinterpret_cast<float2*>(&sm.g[i & 1][r][2 * pr]) = gv;
    }
#pragma unroll
    for (int e = tid; e < 2 * SEL_TILE * NP; e += SEL_THREADS) (&sm.bc[i & 1][0][0][0])[e] = ld_as_float<T>(&sm.raw_bc[k][0][0][0], e);
    if constexpr (MARKS) {
      const uint32_t mark = __ballot_sync(0xffffffffu, first[0]);
      if (tid == 0) sm.mark[i & 1] = mark;
      first[0] = first[1];
    }
  };
  auto finish = [&](int i, int half) {
    const int k = i % SEL_STAGES, k2 = half ^ 1, base = half * SEL_HALF;
    const int64_t t0 = at.t_lo + (int64_t)(tiles - 1 - i) * SEL_TILE + base;
    const int left = (int)min((int64_t)SEL_HALF, at.t_hi - t0);
    if (pair_have > 0) {
#pragma unroll(MARKS ? 2 : SEL_HALF)
      for (int r = row0; r < SEL_HALF; r += S::ROWS) {
        if (r >= left) break;
        const F2 xv = pair_of(&sm.raw[k][3][base + r][2 * pr]), gv = *reinterpret_cast<const float2*>(&sm.g[i & 1][base + r][2 * pr]);
        const F2 in = sum_shares<NP>(sm.res[k2][0][r], pr);
        const float4 q = *reinterpret_cast<const float4*>(&sm.du[i & 1][base + r][2 * pr]);
        const int64_t row = (at.b * p.T + t0 + r) * p.C + at.c0 + 2 * pr;
        put_pair<T>(static_cast<T*>(p.gx) + row, f2fma(f2(q.x, q.z), in, f2mul(skip, gv)), pair_have, whole);
        F2 dd = f2fma(sum_shares<NP>(sm.res[k2][1][r], pr), f2(LN2), f2mul(in, xv));
        if (p.softplus) {
          const F2 v = f2add(pair_of(&sm.raw[k][0][base + r][2 * pr]), bias);
          dd = f2mul(dd, f2(sigmoid_of(v.x), sigmoid_of(v.y)));
        }
        put_pair<T>(static_cast<T*>(p.gdt) + row, dd, pair_have, whole);
        s0 = f2fma(gv, xv, s0);
        s1 = f2add(s1, dd);
        if (p.z != nullptr) {
          const float2 zv = pair_of(&sm.raw[k][2][base + r][2 * pr]);
          F2 slope;
          act_and_slope(zv.x, ACT_SILU, slope.x), act_and_slope(zv.y, ACT_SILU, slope.y);
          const F2 y = f2fma(skip, xv, sum_shares<NP>(sm.res[k2][2][r], pr));
          put_pair<T>(static_cast<T*>(p.gz) + row, f2mul(f2mul(pair_of(&sm.raw[k][1][base + r][2 * pr]), y), slope), pair_have, whole);
        }
      }
    }
    const int blocks = (p.C / p.G + S::CH - 1) / S::CH;
    float* out = p.part_bc + (((at.b * p.G + at.g) * blocks + at.block) * p.T + t0) * 2 * NP;
#pragma unroll 4
    for (int e = tid; e < left * 2 * NP; e += SEL_THREADS) {
      float v = 0.f;
#pragma unroll
      for (int w = 0; w < SEL_THREADS / 32; ++w) v += (&sm.part[k2][w][0][0])[e];
      out[e] = v;
    }
  };
  fetch(0);
  first[0] = first[1];
  if (tiles > 1) fetch(1);
  copy_wait_all();
  helpers_sync();
  make_ready(0);
  __syncthreads();
  for (int i = 0; i < tiles; ++i) {
    // while the second half is scanned
    if (i > 0) finish(i - 1, 0);
    copy_wait_all();
    helpers_sync();  // the copies of tile i + 1 are everybody's, and nobody reads tile i - 1 any more
    if (i + 2 < tiles) fetch(i + 2);
    __syncthreads();
    // while the first half is
    finish(i, 1);
    if (i + 1 < tiles) make_ready(i + 1);
    __syncthreads();
  }
  finish(tiles - 1, 0);
  float* sums = reinterpret_cast<float*>(&sm.du[0][0][0]);  // [2][ROWS][CH]
  helpers_sync();
  sums[row0 * S::CH + 2 * pr] = s0.x;
  sums[row0 * S::CH + 2 * pr + 1] = s0.y;
  sums[(S::ROWS + row0) * S::CH + 2 * pr] = s1.x;
  sums[(S::ROWS + row0) * S::CH + 2 * pr + 1] = s1.y;
  helpers_sync();
  for (int e = tid; e < 2 * at.have; e += SEL_THREADS) {
    const int m = e / at.have, c = e - m * at.have;
    float v = 0.f;
    for (int r = 0; r < S::ROWS; ++r) v += sums[(m * S::ROWS + r) * S::CH + c];
    p.part_d[((at.b * p.nseg + at.seg) * 2 + m) * p.C + at.c0 + c] = v;
  }
}

// A segment's gradient of its first state, from zero behind it, and its sum of steps
template <typename T, int NP>
struct SelRevSmem {
  using S = SelShape<NP>;
  alignas(16) T raw[2][3][SEL_TILE][S::CH];  // dt, gradient of y, z
  alignas(16) T raw_c[2][SEL_TILE][NP];
  alignas(16) float2 d[SEL_TILE][S::PAIRS];  // steps
  alignas(16) float g[SEL_TILE][S::CH];
  alignas(16) float c[SEL_TILE][NP];
};
template <typename T, int NP, bool MARKS>
__global__ void __launch_bounds__(SEL_THREADS) ttt_selective_rev_kernel(const SelParams p) {
  using S = SelShape<NP>;
  extern __shared__ __align__(16) unsigned char sel_smem[];
  SelRevSmem<T, NP>& sm = *reinterpret_cast<SelRevSmem<T, NP>*>(sel_smem);
  const SelPlace<NP> at(p, 1, p.nseg - 1);
  const SelLane<NP> me;
  const int tid = threadIdx.x;
  auto fetch = [&](int64_t t0, int k) {
    copy_rows<T, S::CH, 1>(tid, &sm.raw[k][0][0][0], static_cast<const T*>(p.dt) + at.b * p.ds[0] + at.c0, p.ds[1], t0, at.t_hi, at.have, p.xg);
    copy_rows<T, S::CH, 1>(tid, &sm.raw[k][1][0][0], static_cast<const T*>(p.gy) + at.b * p.gs[0] + at.c0, p.gs[1], t0, at.t_hi, at.have, p.xg);
    if (p.z != nullptr)
      copy_rows<T, S::CH, 1>(tid, &sm.raw[k][2][0][0], static_cast<const T*>(p.z) + at.b * p.zs[0] + at.c0, p.zs[1], t0, at.t_hi, at.have, p.xg);
    copy_rows<T, NP, 1>(tid, &sm.raw_c[k][0][0], static_cast<const T*>(p.c) + at.b * p.cs[0] + at.g * p.cs[2], p.cs[1], t0, at.t_hi, p.N, p.bg);
    copy_commit();
  };
  const int64_t t_last = at.t_lo + (at.t_hi - at.t_lo - 1) / SEL_TILE * SEL_TILE;
  fetch(t_last, 0);
  F2 A[S::CC][2], dh[S::CC][2];
  me.load_rates(A, p.A + (int64_t)at.c0 * p.N, p.N, at.have);
#pragma unroll
  for (int k = 0; k < S::CC; ++k) dh[k][0] = dh[k][1] = f2(0.f);
  const int pr = tid % S::PAIRS, row0 = tid / S::PAIRS, pair_have = at.have - 2 * pr;
  float2 bias = make_float2(0.f, 0.f), sum = make_float2(0.f, 0.f);
  if (p.bias != nullptr) {
    if (pair_have > 0) bias.x = p.bias[at.c0 + 2 * pr];
    if (pair_have > 1) bias.y = p.bias[at.c0 + 2 * pr + 1];
  }
  bool any_start = false;
  int buf = 0;
  for (int64_t t0 = t_last; t0 >= at.t_lo; t0 -= SEL_TILE, buf ^= 1) {
    uint32_t mark = 0;
    if constexpr (MARKS) {
      const int64_t t = t0 + (me.lane & (SEL_TILE - 1));
      mark = __ballot_sync(0xffffffffu, t < at.t_hi && p.starts[at.b * p.T + t] != 0) & ((1u << SEL_TILE) - 1);
      any_start = any_start || mark != 0;
    }
    copy_wait_all();
    __syncthreads();
    if (t0 - SEL_TILE >= at.t_lo) fetch(t0 - SEL_TILE, buf ^ 1);
#pragma unroll
    for (int r = row0; r < SEL_TILE; r += S::ROWS) {
      F2 d = f2add(pair_of(&sm.raw[buf][0][r][2 * pr]), bias), gv = pair_of(&sm.raw[buf][1][r][2 * pr]);
      if (p.softplus) d = softplus_of(d);
      if (t0 + r >= at.t_hi || pair_have < 1) d.x = 0.f;
      if (t0 + r >= at.t_hi || pair_have < 2) d.y = 0.f;
      if (p.z != nullptr) {
        const float2 zv = pair_of(&sm.raw[buf][2][r][2 * pr]);
        gv = f2mul(gv, f2(act_of(zv.x, ACT_SILU), act_of(zv.y, ACT_SILU)));
      }
      sum = f2add(sum, d);
      sm.d[r][pr] = d;
      *reinterpret_cast<float2*>(&sm.g[r][2 * pr]) = gv;
    }
#pragma unroll
    for (int e = tid; e < SEL_TILE * NP; e += SEL_THREADS) (&sm.c[0][0])[e] = ld_as_float<T>(&sm.raw_c[buf][0][0], e);
    __syncthreads();
#pragma unroll 8
    for (int r = SEL_TILE - 1; r >= 0; --r) {
      const float* dp = reinterpret_cast<const float*>(&sm.d[r][0]) + me.ch;
      const float* gp = sm.g[r] + me.ch;
      const float4 c = *reinterpret_cast<const float4*>(&sm.c[r][4 * me.sl]);
#pragma unroll
      for (int k = 0; k < S::CC; ++k) {
        const F2 dk = f2(dp[k]), gk = f2(gp[k]);
        dh[k][0] = f2mul(f2fma(gk, f2(c.x, c.y), dh[k][0]), decay_of(A[k][0], dk));
        dh[k][1] = f2mul(f2fma(gk, f2(c.z, c.w), dh[k][1]), decay_of(A[k][1], dk));
        if (MARKS && mark >> r & 1) dh[k][0] = dh[k][1] = f2(0.f);
      }
    }
  }
  const int64_t row = (at.b * p.nseg + at.seg) * p.C + at.c0;
  me.store(dh, p.seg_state + row * NP, NP, at.have);
  float* sums = reinterpret_cast<float*>(&sm.g[0][0]);  // [ROWS][CH]
  __syncthreads();
  sums[row0 * S::CH + 2 * pr] = sum.x;
  sums[row0 * S::CH + 2 * pr + 1] = sum.y;
  __syncthreads();
  for (int c = tid; c < at.have; c += SEL_THREADS) {
    float v = 0.f;
    for (int r = 0; r < S::ROWS; ++r) v += sums[r * S::CH + c];
    p.seg_sum[row + c] = any_start ? INFINITY : v;
  }
}

// The blocks' shares of dB and dC, [B][G][blocks][T][2][NP] -> [B][T][G][N] each
template <typename T>
__global__ void __launch_bounds__(256) ttt_selective_bc_kernel(const SelParams p, int NP, int blocks) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, per = p.T * NP / 2;  // four states each: (b G + g) T 2 NP / 4 + ...
  if (i >= p.B * p.G * per) return;
  const int64_t bg = i / per, e = i - bg * per;
  const float4* src = reinterpret_cast<const float4*>(p.part_bc) + bg * blocks * per + e;
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
  for (int k = 0; k < blocks; ++k) {
    const float4 w = src[k * per];
    v = make_float4(v.x + w.x, v.y + w.y, v.z + w.z, v.w + w.w);
  }
  const int64_t t = e / (NP / 2);
  const int n = 4 * (int)(e - t * (NP / 2)), which = n / NP, s = n - which * NP;
  const int64_t b = bg / p.G, g = bg - b * p.G, to = ((b * p.T + t) * p.G + g) * p.N + s;
  void* out = which ? p.gc : p.gb;
  if (s < p.N) st_from_float<T>(out, to, v.x);
  if (s + 1 < p.N) st_from_float<T>(out, to + 1, v.y);
  if (s + 2 < p.N) st_from_float<T>(out, to + 2, v.z);
  if (s + 3 < p.N) st_from_float<T>(out, to + 3, v.w);
}
// The blocks' rows of sums -> gradients of A (of [C][NP], the first blocks), D and the bias (of [C] each, blocks_c blocks)
__global__ void __launch_bounds__(ROWS_THREADS) ttt_selective_rows_kernel(const SelParams p, int64_t rows, int NP, int64_t blocks_a, int64_t blocks_c) {
  int64_t col, block = blockIdx.x;
  float v;
  if (block < blocks_a) {
    const int64_t n = (int64_t)p.C * NP;
    if (!sum_of_rows(p.part_a, rows, n, n, block, &col, &v)) return;
    const int64_t c = col / NP;
    const int s = (int)(col - c * NP);
    if (s < p.N) p.ga[c * p.N + s] = v;
    return;
  }
  block -= blocks_a;
  const bool second = block >= blocks_c;
  float* out = second ? p.gbias : p.gd;
  if (out == nullptr) return;  // (the whole block)
  if (sum_of_rows(p.part_d + (second ? p.C : 0), rows, 2 * (int64_t)p.C, p.C, second ? block - blocks_c : block, &col, &v)) out[col] = v;
}

template <typename K>
static cudaError_t run(K kernel, int bytes, int64_t blocks, int threads, const SelParams& p, cudaStream_t st) {
  if (bytes > 48 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != cudaSuccess) return e;
  }
  kernel<<<(unsigned)blocks, threads, bytes, st>>>(p);
  return cudaGetLastError();
}
template <typename T, int NP>
static cudaError_t run_all(const SelParams& p, cudaStream_t st) {
  const int each = p.C / p.G, channel_blocks = (each + SelShape<NP>::CH - 1) / SelShape<NP>::CH;
  const int64_t blocks = p.B * p.G * channel_blocks, rows = p.B * p.nseg;
  cudaError_t e;
  const bool marks = p.starts != nullptr;
  static_assert(sizeof(SelBwdSmem<T, NP>) <= 227 * 1024, "");
  if (p.nseg > 1 && (e = run(marks ? ttt_selective_rev_kernel<T, NP, true> : ttt_selective_rev_kernel<T, NP, false>, sizeof(SelRevSmem<T, NP>),
                             blocks * (p.nseg - 1), SEL_THREADS, p, st)) != cudaSuccess)
    return e;
  if ((e = run(marks ? ttt_selective_bwd_kernel<T, NP, true> : ttt_selective_bwd_kernel<T, NP, false>, sizeof(SelBwdSmem<T, NP>), blocks * p.nseg,
               2 * SEL_THREADS, p, st)) != cudaSuccess)
    return e;
  ttt_selective_bc_kernel<T><<<(unsigned)((p.B * p.G * p.T * NP / 2 + 255) / 256), 256, 0, st>>>(p, NP, channel_blocks);
  if ((e = cudaGetLastError()) != cudaSuccess) return e;
  const int64_t blocks_a = ((int64_t)p.C * NP + 31) / 32, blocks_c = (p.C + 31) / 32;
  ttt_selective_rows_kernel<<<(unsigned)(blocks_a + (p.gd != nullptr || p.gbias != nullptr ? 2 * blocks_c : 0)), ROWS_THREADS, 0, st>>>(p, rows, NP, blocks_a,
                                                                                                                                blocks_c);
  return cudaGetLastError();
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
