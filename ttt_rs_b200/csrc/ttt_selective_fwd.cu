// Selective state space scan, forward and decode step (definitions: ttt_selective.cuh).
//
// A block of eight warps owns 64 channels (N = 16) of one group of a sequence, or of a segment of it; where a group has fewer, the other
// lanes walk zeros (65536 tokens of 8 groups, 16 states, bf16: 6 channels each 468 us, 64 each 402; training 1531 and 1353).  Segments,
// where channels are too few to fill the card: every segment's own state first (from zero, with the sum of its steps, since exp(A sum d) is its whole decay), which the
// scan's blocks join along the sequence before they begin.  For training the states before every SEL_TILE tokens are kept.
//
// bf16, 16 x 2048 tokens of 1536 channels, 16 states: 390 us with the states kept (all eight warps doing everything: 519 us; a quotient
// in the step's logarithm and range handling in the exponentials: 424 us; shares of y through shuffles: 8 instructions more per token);
// one sequence of 32768 such tokens: 235 us for the segments' states, 0.77 of what their exponentials allow, and 336 us for the scan.
#include "ttt_selective.cuh"

namespace ttt {

template <typename T, int NP, bool FULL>
struct SelSmem {
  using S = SelShape<NP>;
  static constexpr int TENSORS = FULL ? 3 : 2;
  alignas(16) T raw[SEL_STAGES][TENSORS][SEL_TILE][S::CH];  // x, dt, z
  alignas(16) T raw_bc[SEL_STAGES][FULL ? 2 : 1][SEL_TILE][NP];
  alignas(16) float4 du[2][SEL_TILE][S::PAIRS];             // (step, step x) of two channels
  alignas(16) float bc[2][FULL ? 2 : 1][SEL_TILE][NP];
  alignas(16) float y[2][FULL ? SEL_TILE : 1][S::SHARES];  // shares of a result, as the scanning lanes lie
  uint32_t mark[2];                                         // starts of a tile, bit by bit
};

// FULL false: a segment's own state, from zero, and its sum of steps.  MARKS: there are starts (else the kernel knows none).
template <typename T, int NP, bool FULL, bool MARKS>
__global__ void __launch_bounds__(2 * SEL_THREADS, 3) ttt_selective_kernel(const SelParams p) {
  using S = SelShape<NP>;
  using Smem = SelSmem<T, NP, FULL>;
  extern __shared__ __align__(16) unsigned char sel_smem[];
  Smem& sm = *reinterpret_cast<Smem*>(sel_smem);
  const SelPlace<NP> at(p, 0, FULL ? p.nseg : p.nseg - 1);
  const int tiles = (int)((at.t_hi - at.t_lo + SEL_TILE - 1) / SEL_TILE);
  if (threadIdx.x < SEL_THREADS) {
    // ---- scan
    const SelLane<NP> me;
    [[maybe_unused]] const int my_share = share_at<NP>(me.ch / S::CC, me.sl);
    F2 A[S::CC][2], h[S::CC][2];
    me.load_rates(A, p.A + (int64_t)at.c0 * p.N, p.N, at.have);
    if constexpr (FULL) {
      if (p.nseg == 1) me.load(h, p.state != nullptr ? p.state + (at.b * p.C + at.c0) * p.N : nullptr, p.N, at.have);
      else me.load_padded(h, p.seg_state + ((p.B * p.nseg + at.b) * p.C + at.c0) * NP, at.have);
      for (int j = 0; j < at.seg; ++j) {  // the segments before, in their order
        const int64_t row = (at.b * p.nseg + j) * p.C + at.c0;
        F2 own[S::CC][2];
        me.load_padded(own, p.seg_state + row * NP, at.have);
#pragma unroll
        for (int k = 0; k < S::CC; ++k) {
          const float sum = me.ch + k < at.have ? p.seg_sum[row + me.ch + k] : 0.f;
          const bool cut = sum == INFINITY;
#pragma unroll
          for (int i = 0; i < 2; ++i) h[k][i] = cut ? own[k][i] : f2fma(decay_of(A[k][i], f2(sum)), h[k][i], own[k][i]);
        }
      }
    } else {
      // (the given state may be where the new one goes, which other blocks of the scan write: the scan reads it from here)
      if (at.seg == 0) {
        me.load(h, p.state != nullptr ? p.state + (at.b * p.C + at.c0) * p.N : nullptr, p.N, at.have);
        me.store(h, p.seg_state + ((p.B * p.nseg + at.b) * p.C + at.c0) * NP, NP, at.have);
      }
#pragma unroll
      for (int k = 0; k < S::CC; ++k) h[k][0] = h[k][1] = f2(0.f);
    }
    float* saved = nullptr;
    if (FULL && p.saved != nullptr) saved = p.saved + ((at.b * ((p.T + SEL_TILE - 1) / SEL_TILE) + at.t_lo / SEL_TILE) * p.C + at.c0) * NP;
    __syncthreads();
    for (int i = 0; i < tiles; ++i) {
      if (saved != nullptr) {
        me.store(h, saved, NP, at.have);
        saved += (int64_t)p.C * NP;
      }
      const uint32_t mark = MARKS ? sm.mark[i & 1] : 0;
#pragma unroll 8
      for (int r = 0; r < SEL_TILE; ++r) {
        float4 q;
        if constexpr (S::CC == 2) {
          q = sm.du[i & 1][r][me.ch / 2];
        } else {
          const float2 one = *reinterpret_cast<const float2*>(reinterpret_cast<const float*>(&sm.du[i & 1][r][0]) + 2 * me.ch);
          q = make_float4(one.x, one.y, 0.f, 0.f);
        }
        const float4 b = *reinterpret_cast<const float4*>(&sm.bc[i & 1][0][r][4 * me.sl]);
        if (MARKS && mark >> r & 1) {
#pragma unroll
          for (int k = 0; k < S::CC; ++k) h[k][0] = h[k][1] = f2(0.f);
        }
        [[maybe_unused]] float4 c;
        [[maybe_unused]] float part[2];
        if constexpr (FULL) c = *reinterpret_cast<const float4*>(&sm.bc[i & 1][FULL ? 1 : 0][r][4 * me.sl]);
#pragma unroll
        for (int k = 0; k < S::CC; ++k) {
          const F2 d = f2(k ? q.z : q.x), v = f2(k ? q.w : q.y);
          h[k][0] = f2fma(decay_of(A[k][0], d), h[k][0], f2mul(v, f2(b.x, b.y)));
          h[k][1] = f2fma(decay_of(A[k][1], d), h[k][1], f2mul(v, f2(b.z, b.w)));
          if constexpr (FULL) part[k] = f2hsum(f2fma(h[k][0], f2(c.x, c.y), f2mul(h[k][1], f2(c.z, c.w))));
        }
        if constexpr (FULL) {
          if constexpr (S::CC == 2) *reinterpret_cast<float2*>(&sm.y[i & 1][r][my_share]) = make_float2(part[0], part[1]);
          else sm.y[i & 1][r][my_share] = part[0];
        }
      }
      __syncthreads();
    }
    if constexpr (FULL) {
      if (at.t_hi == p.T) me.store(h, p.state_out + (at.b * p.C + at.c0) * p.N, p.N, at.have);
    } else {
      me.store(h, p.seg_state + ((at.b * p.nseg + at.seg) * p.C + at.c0) * NP, NP, at.have);
    }
    return;
  }
  // ---- what is done once per token and channel, pair of channels by pair
  const int tid = threadIdx.x - SEL_THREADS, pr = tid % S::PAIRS, row0 = tid / S::PAIRS, pair_have = at.have - 2 * pr;
  const T* x = static_cast<const T*>(p.x) + at.b * p.xs[0] + at.c0;
  const T* dt = static_cast<const T*>(p.dt) + at.b * p.ds[0] + at.c0;
  const T* z = FULL && p.z != nullptr ? static_cast<const T*>(p.z) + at.b * p.zs[0] + at.c0 : nullptr;
  const T* bm = static_cast<const T*>(p.b) + at.b * p.bs[0] + at.g * p.bs[2];
  const T* cm = static_cast<const T*>(p.c) + at.b * p.cs[0] + at.g * p.cs[2];
  const uint8_t* starts = MARKS ? p.starts + at.b * p.T : nullptr;
  bool first[2] = {false, false};  // lane r of a warp: a start at token r of the next tile to be made ready, and of the one behind it
  bool any_start = false;
  auto fetch = [&](int i) {
    const int k = i % SEL_STAGES;
    const int64_t t0 = at.t_lo + (int64_t)i * SEL_TILE;
    copy_rows<T, S::CH, 8>(tid, &sm.raw[k][0][0][0], x, p.xs[1], t0, at.t_hi, at.have, p.xg);
    copy_rows<T, S::CH, 8>(tid, &sm.raw[k][1][0][0], dt, p.ds[1], t0, at.t_hi, at.have, p.xg);
    copy_rows<T, NP, 8>(tid, &sm.raw_bc[k][0][0][0], bm, p.bs[1], t0, at.t_hi, p.N, p.bg);
    if constexpr (FULL) {
      if (z != nullptr) copy_rows<T, S::CH, 8>(tid, &sm.raw[k][Smem::TENSORS - 1][0][0], z, p.zs[1], t0, at.t_hi, at.have, p.xg);
      copy_rows<T, NP, 8>(tid, &sm.raw_bc[k][FULL ? 1 : 0][0][0], cm, p.cs[1], t0, at.t_hi, p.N, p.bg);
    }
    copy_commit();
    if constexpr (MARKS) {
      const int64_t t = t0 + (tid & 31);
      first[1] = (tid & 31) < SEL_TILE && t < at.t_hi && starts[t] != 0;
    }
  };
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
  float2 sum = make_float2(0.f, 0.f);  // (FULL false: of the pair's steps over this thread's tokens)
  auto make_ready = [&](int i) {
    const int k = i % SEL_STAGES, left = (int)(at.t_hi - at.t_lo) - i * SEL_TILE;
#pragma unroll
    for (int r = row0; r < SEL_TILE; r += S::ROWS) {
      const float2 xv = pair_of(&sm.raw[k][0][r][2 * pr]), dv = pair_of(&sm.raw[k][1][r][2 * pr]);
      F2 d = f2add(dv, bias);
      if (p.softplus) d = softplus_of(d);
      if (r >= left || pair_have < 1) d.x = 0.f;
      if (r >= left || pair_have < 2) d.y = 0.f;
      sm.du[i & 1][r][pr] = make_float4(d.x, d.x * xv.x, d.y, d.y * xv.y);
      if (!FULL) sum = f2add(sum, d);
    }
#pragma unroll
    for (int e = tid; e < (FULL ? 2 : 1) * SEL_TILE * NP; e += SEL_THREADS)
      (&sm.bc[i & 1][0][0][0])[e] = ld_as_float<T>(&sm.raw_bc[k][0][0][0], e);
    if constexpr (MARKS) {
      const uint32_t mark = __ballot_sync(0xffffffffu, first[0]);
      if (tid == 0) sm.mark[i & 1] = mark;
      any_start = any_start || mark != 0;
      first[0] = first[1];
    }
  };
  auto finish = [&](int i) {
    const int k = i % SEL_STAGES, left = (int)(at.t_hi - at.t_lo) - i * SEL_TILE;
    if (pair_have < 1) return;
    T* y = static_cast<T*>(p.y) + (at.b * p.T + at.t_lo + (int64_t)i * SEL_TILE + row0) * p.C + at.c0 + 2 * pr;
#pragma unroll
    for (int r = row0; r < SEL_TILE; r += S::ROWS, y += (int64_t)S::ROWS * p.C) {
      if (r >= left) break;
      F2 v = sum_shares<NP>(sm.y[i & 1][r], pr);
      v = f2fma(skip, pair_of(&sm.raw[k][0][r][2 * pr]), v);
      if (z != nullptr) {
        const float2 zv = pair_of(&sm.raw[k][Smem::TENSORS - 1][r][2 * pr]);
        v = f2mul(v, f2(act_of(zv.x, ACT_SILU), act_of(zv.y, ACT_SILU)));
      }
      put_pair<T>(y, v, pair_have, whole);
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
    if (FULL && i > 0) finish(i - 1);
    copy_wait_all();
    helpers_sync();  // the copies of tile i + 1 are everybody's, and nobody reads tile i - 1 any more
    if (i + 2 < tiles) fetch(i + 2);
    if (i + 1 < tiles) make_ready(i + 1);
    __syncthreads();
  }
  if constexpr (FULL) {
    finish(tiles - 1);
  } else {
    float* sums = reinterpret_cast<float*>(&sm.du[0][0][0]);  // [ROWS][CH]
    helpers_sync();
    sums[row0 * S::CH + 2 * pr] = sum.x;
    sums[row0 * S::CH + 2 * pr + 1] = sum.y;
    helpers_sync();
    for (int c = tid; c < at.have; c += SEL_THREADS) {
      float v = 0.f;
      for (int r = 0; r < S::ROWS; ++r) v += sums[r * S::CH + c];
      p.seg_sum[(at.b * p.nseg + at.seg) * p.C + at.c0 + c] = any_start ? INFINITY : v;
    }
  }
}

// Up to 16 tokens against the resident state: a thread per channel and EACH states, no shared memory.  Bound by the state's read and
// write where sequences are many, by the launch and one chain of loads where not.  Four states per thread are the shortest chain; where
// so many threads would not be resident at once, eight: what is done once per channel is then done by two lanes, not by four.
// 128 sequences of 1536 channels of 16 states: 14.5 us with four, 11.8 with eight, 12.7 with sixteen, 18 with fewer threads that walk
// the sequences; 8 sequences: 3.9 us with four.
template <typename T, int SL, int EACH>
__global__ void __launch_bounds__(SEL_THREADS) ttt_selective_step_kernel(const SelParams p) {
  const uint32_t i = blockIdx.x * SEL_THREADS + threadIdx.x;
  const int n0 = (int)(i % SL) * EACH;
  const bool live = i / SL < (uint32_t)p.C;
  const int c = live ? (int)(i / SL) : 0, g = p.G == 1 ? 0 : c / (p.C / p.G);
  const bool quads = p.N % 4 == 0;
  auto load = [&](const float* at, float (&v)[EACH]) {
#pragma unroll
    for (int k = 0; k < EACH; k += 4) {
      float4 e = make_float4(0.f, 0.f, 0.f, 0.f);
      if (quads) {
        if (at != nullptr && n0 + k < p.N) e = *reinterpret_cast<const float4*>(at + n0 + k);
      } else if (at != nullptr) {
        if (n0 + k < p.N) e.x = at[n0 + k];
        if (n0 + k + 1 < p.N) e.y = at[n0 + k + 1];
        if (n0 + k + 2 < p.N) e.z = at[n0 + k + 2];
        if (n0 + k + 3 < p.N) e.w = at[n0 + k + 3];
      }
      v[k] = e.x, v[k + 1] = e.y, v[k + 2] = e.z, v[k + 3] = e.w;
    }
  };
  const bool words = quads && sizeof(T) == 2 && p.bg >= 4;  // b's and c's rows on 4 bytes: two bf16 at a time
  auto states = [&](const T* at, float (&v)[EACH]) {
    if (words) {
#pragma unroll
      for (int k = 0; k < EACH; k += 2) {
        const uint32_t e = n0 + k < p.N ? reinterpret_cast<const uint32_t*>(at)[(n0 + k) / 2] : 0;
        v[k] = bf16_lo(e), v[k + 1] = bf16_hi(e);
      }
    } else {
#pragma unroll
      for (int k = 0; k < EACH; ++k) v[k] = n0 + k < p.N ? ld_as_float<T>(at, n0 + k) : 0.f;
    }
  };
  float a[EACH];
  load(p.A + (int64_t)c * p.N, a);
#pragma unroll
  for (int k = 0; k < EACH; ++k) a[k] = rate_of(a[k]);
  const float bias = p.bias != nullptr ? p.bias[c] : 0.f, skip = p.D != nullptr ? p.D[c] : 0.f;
  for (int64_t b = blockIdx.y; b < p.B; b += gridDim.y) {
    float h[EACH];
    load(p.state != nullptr ? p.state + (b * p.C + c) * p.N : nullptr, h);
    for (int t = 0; t < (int)p.T; ++t) {
      float bv[EACH], cv[EACH], d = ld_as_float<T>(p.dt, b * p.ds[0] + t * p.ds[1] + c) + bias;
      const float xv = ld_as_float<T>(p.x, b * p.xs[0] + t * p.xs[1] + c);
      const float zv = p.z != nullptr ? ld_as_float<T>(p.z, b * p.zs[0] + t * p.zs[1] + c) : 0.f;
      states(static_cast<const T*>(p.b) + b * p.bs[0] + t * p.bs[1] + g * p.bs[2], bv);
      states(static_cast<const T*>(p.c) + b * p.cs[0] + t * p.cs[1] + g * p.cs[2], cv);
      const bool start = p.starts != nullptr && p.starts[b * p.T + t] != 0;
      if (p.softplus) d = softplus_of(f2(d)).x;
      const float u = d * xv;
      float s = 0.f;
#pragma unroll
      for (int k = 0; k < EACH; ++k) {
        h[k] = fmaf(decay_of(f2(a[k]), d).x, start ? 0.f : h[k], u * bv[k]);
        s = fmaf(h[k], cv[k], s);
      }
#pragma unroll
      for (int o = 1; o < SL; o <<= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
      s = fmaf(skip, xv, s);
      if (p.z != nullptr) s *= act_of(zv, ACT_SILU);
      if (live && n0 == 0) st_from_float<T>(p.y, (b * p.T + t) * p.C + c, s);
    }
    if (!live) continue;
    float* out = p.state_out + (b * p.C + c) * p.N + n0;
#pragma unroll
    for (int k = 0; k < EACH; k += 4) {
      if (quads) {
        if (n0 + k < p.N) *reinterpret_cast<float4*>(out + k) = make_float4(h[k], h[k + 1], h[k + 2], h[k + 3]);
      } else {
#pragma unroll
        for (int e = k; e < k + 4; ++e)
          if (n0 + e < p.N) out[e] = h[e];
      }
    }
  }
}

int sel_padded(int N) {
  int n = SEL_EACH;
  while (n < N) n *= 2;
  return n;
}
SelCut sel_cut(int64_t B, int64_t T, int C, int G, int N, bool bwd) {
  const int NP = sel_padded(N), CH = NP == 4 ? 128 : NP == 8 ? 64 : 1024 / NP, each = C / G;
  SelCut k{};
  k.channel_blocks = (each + CH - 1) / CH;
  const int64_t blocks = B * G * k.channel_blocks, tiles = (T + SEL_TILE - 1) / SEL_TILE;
  // Forward: three blocks per SM in all.  Backward: four, which shares the last round of those resident out; eight where a block per SM
  // leaves little idle anyway, and none there with 64 states, whose gradients carried back cost more.  Segments of two tiles at least, of
  // four beyond 32 of them: a block joins all that are before it.  The rule does not ask how many blocks are resident.  By their shared
  // memory that is, forward, three per SM in bf16 with more than 4 states and in float32 with 5 to 8, two in bf16 with up to 4 and in float32
  // with more than 8, one in float32 with up to 4; backward two with 5 to 8 states and in bf16 with 9 to 32, one otherwise.  Where it is
  // fewer than three and two, the segments run in more rounds than the sweeps below, of 16 states in bf16, were made for.
  // us, 16 states: 1 x 32768 x 1536: 18 segments 580, 12 623, 24 615, 36 574; backward 24 1373, 12 1439, 32 1517.  2 x 4096 x 1536: 9
  // segments 161, 6 169, 12 179; backward 12 392, 6 396, 8 441.  4 x 2048 x 2048: 3 segments 201, 1 229, 4 220; backward 9 to 12
  // 500, 1 550, 4 523.  1 x 512 x 512: 16 segments 21, 8 27; backward 16 46, 8 62.  (64 states, 2 x 2048 x 1024: backward 1 611, 8 654.)
  // Between one block per SM and four thirds of that, three segments both ways: the second round would leave most SMs idle, and two
  // segments do not mend that.  192 blocks, 1 / 2 / 3 segments: 8 x 2048 x 1536 float32 forward 322 / 387 / 322, backward 1103 / 1010 /
  // 899; 4 states, 16 x 2048 x 1536 bf16 360 / 440 / 336 and 1280 / 1130 / 1003; 64 states, 2 x 2048 x 1536 backward 1145 / 1018 / 911.
  // 224 blocks: 285 / 375 / 338 and 795 / 936 / 844.  Not the best there throughout: 160 blocks of 16 states in bf16, three segments 287 and
  // 666, eight 241 and 593.
  const bool thirds = blocks > 148 && blocks <= 197;
  int64_t wanted = thirds ? 3 : blocks > 197 ? 1 : 444 / blocks;
  if (bwd && !thirds) wanted = blocks < 100 ? 592 / blocks : blocks <= 148 && NP < 64 ? 1184 / blocks : 1;
  int64_t most = tiles / 4 > 32 ? tiles / 4 : 32;
  if (most > tiles / 2) most = tiles / 2;
  if (wanted > most) wanted = most;
  k.nseg = wanted > 1 ? (int)wanted : 1;
  k.seg_tiles = (int)((tiles + k.nseg - 1) / k.nseg);
  k.nseg = (int)((tiles + k.seg_tiles - 1) / k.seg_tiles);
  return k;
}

template <typename T, int NP, bool FULL>
static cudaError_t run(const SelParams& p, int64_t blocks, cudaStream_t st) {
  constexpr int bytes = sizeof(SelSmem<T, NP, FULL>);
  void (*kernel)(SelParams) = p.starts != nullptr ? ttt_selective_kernel<T, NP, FULL, true> : ttt_selective_kernel<T, NP, FULL, false>;
  if (bytes > 48 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != cudaSuccess) return e;
  }
  kernel<<<(unsigned)blocks, 2 * SEL_THREADS, bytes, st>>>(p);
  return cudaGetLastError();
}
template <typename T, int NP>
static cudaError_t run_all(const SelParams& p, cudaStream_t st) {
  const int each = p.C / p.G;
  const int64_t blocks = p.B * p.G * ((each + SelShape<NP>::CH - 1) / SelShape<NP>::CH);
  if (p.nseg > 1) {  // (the last segment's own state is nobody's)
    const cudaError_t e = run<T, NP, false>(p, blocks * (p.nseg - 1), st);
    if (e != cudaSuccess) return e;
  }
  return run<T, NP, true>(p, blocks * p.nseg, st);
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
cudaError_t launch_selective(int dtype, const SelParams& p, cudaStream_t st) {
  return dtype == 1 ? run_np<__nv_bfloat16>(p, st) : run_np<float>(p, st);
}
template <typename T, int NP>
static cudaError_t step(const SelParams& p, cudaStream_t st) {
  constexpr int WIDE = NP < 8 ? NP : 8;
  const bool wide = (int64_t)p.C * (NP / SEL_EACH) * p.B > (int64_t)148 * 1024;
  const int lanes = wide ? NP / WIDE : NP / SEL_EACH;
  const dim3 grid((unsigned)(((int64_t)p.C * lanes + SEL_THREADS - 1) / SEL_THREADS), (unsigned)(p.B < 65535 ? p.B : 65535));
  if (wide) ttt_selective_step_kernel<T, NP / WIDE, WIDE><<<grid, SEL_THREADS, 0, st>>>(p);
  else ttt_selective_step_kernel<T, NP / SEL_EACH, SEL_EACH><<<grid, SEL_THREADS, 0, st>>>(p);
  return cudaGetLastError();
}
template <typename T>
static cudaError_t step_np(const SelParams& p, cudaStream_t st) {
  switch (sel_padded(p.N)) {
    case 4: return step<T, 4>(p, st);
    case 8: return step<T, 8>(p, st);
    case 16: return step<T, 16>(p, st);
    case 32: return step<T, 32>(p, st);
    default: return step<T, 64>(p, st);
  }
}
cudaError_t launch_selective_step(int dtype, const SelParams& p, cudaStream_t st) {
  return dtype == 1 ? step_np<__nv_bfloat16>(p, st) : step_np<float>(p, st);
}

}  // namespace ttt
