// Gated linear recurrence, forward (the mathematics and its chunked form: ttt_gated.cuh).
//
// One CTA of four warps per stream (or segment, or range of streams) walks its chunks.  A warp owns 16 rows of the float32 state,
// in accumulator layout, and updates them with the transposed and scaled keys of every chunk; and 16 queries of the chunk, another
// 16 in every chunk, since the last ones meet four blocks of keys and the first ones one: for each block of 16 tokens the
// decayed products of queries and keys become, in registers, the A operand of the product with the block's values.  q W comes
// last: the state before the chunk is there once all warps have left the chunk before, and until then a warp works on what needs only
// this chunk's inputs, so that no warp waits for the others of its chunk.  The next chunk is on its way meanwhile (TMA, rows
// behind the sequence read as zeros), fetched when all warps have left the chunk before.
//
// 384 streams of 2048 tokens, F = 64, bf16, with the states saved: 155 us, 3.7 TB/s, in passes back to back (alone with cold caches, under the
// profiler, 158); float32, without saved states, 616 us.  1170 instructions per warp and chunk at 41 % of the issue slots (three blocks per SM, for the registers), tensor pipe 47 %, shared-memory pipe 54 %: bound by the latencies of a
// warp's own chain of products and changes of form, which stay in registers because every way through memory is longer.
//
// Few streams are cut into segments: a first launch leaves every segment's own state (as if it began with none) and its decay, a
// second one joins them along the sequence, and the third is this kernel with a CTA per segment.
#include "ttt_kernels.h"
#include "ttt_gated.cuh"
#include "ttt_stage.cuh"

namespace ttt {

constexpr int GF_THREADS = 32 * GATED_WARPS;

// STATE: only keys and values (or queries and gradients) come in, and no state goes out before the end
template <typename T, int F, bool STATE>
struct GatedFwdSmem {
  static constexpr bool BF = sizeof(T) == 2;
  static constexpr int NP = BF ? 1 : 3, NIN = STATE ? 2 : 3;
  static constexpr uint32_t PLANE = GTile<F>::BYTES, TILE = NP * PLANE;
  static constexpr uint32_t RAW = GC * F * 4;  // float32 rows as they arrive
  static constexpr uint32_t STAGES = BF ? 2 : 1;
  static constexpr uint32_t TILES = 0, RAWS = TILES + STAGES * NIN * TILE;
  static constexpr uint32_t W = RAWS + (BF ? 0 : NIN * RAW);
  static constexpr uint32_t GATES = W + (STATE ? 0 : 2 * NP * GTile<F>::STATE_BYTES);
  static constexpr uint32_t BAR = GATES + 3 * sizeof(ChunkGates), BYTES = BAR + 48 + 1024;  // (1024: the base is aligned by hand)
};

// What both kernels do with a chunk's inputs, gates and the state's update
template <typename T, int F, bool STATE, bool REV, int THREADS>
struct GatedFwdBlock {
  using SM = GatedFwdSmem<T, F, STATE>;
  using SH = StateShare<F>;
  using TL = GTile<F>;
  static constexpr bool BF = SM::BF;
  static constexpr int NP = SM::NP, NS = 3, KS = F / 16;  // planes of inputs, of scaled keys
  const GatedMaps& maps;
  const GatedParams& p;
  uint8_t* mem;
  uint32_t base, bar;
  ChunkGates* gates;
  GatedWaits waits;
  int tid, lane, w;
  GatedWalk walk;

  __device__ __forceinline__ int chunk_of(const GatedWalk::Step& s) const { return REV ? p.NC - 1 - s.pos : s.pos; }
  __device__ __forceinline__ void fetch(const GatedWalk::Step& s) const {  // one thread
    if (!waits.ok()) return;
    const int slot = BF ? s.i & 1 : 0;
    const uint32_t at = bar + 8 * slot, dst = base + (BF ? SM::TILES + slot * SM::NIN * SM::TILE : SM::RAWS);
    constexpr uint32_t bytes = BF ? SM::TILE : SM::RAW;
    const int b = s.stream / p.H, h = s.stream - b * p.H;
    waits.started(copies(), slot, (BF ? s.i >> 1 : s.i) & 1);
    mbar_expect_tx(at, SM::NIN * bytes);
#pragma unroll
    for (int m = 0; m < SM::NIN; ++m) tma_load_4d(dst + m * bytes, &maps.m[(STATE ? 1 : 0) + m], chunk_of(s) * GC, h, b, at);
  }
  __device__ __forceinline__ void gates_of(const GatedWalk::Step& s, float2& g, float2& beta) const {  // one warp
    const size_t row = (size_t)s.stream * p.T;
    g = load_gates(p.g + row, chunk_of(s) * GC, p.T, lane, 0.f);
    beta = load_gates(p.beta != nullptr ? p.beta + row : nullptr, chunk_of(s) * GC, p.T, lane, 1.f);
  }
  // this chunk's tiles, in their planes
  __device__ __forceinline__ uint32_t tiles(const GatedWalk::Step& st, const GatedWalk::Step& nx) const {
    const int slot = BF ? st.i & 1 : 0;
    const uint32_t at = base + SM::TILES + slot * SM::NIN * SM::TILE;
    waits.wait(bar + 8 * slot, (BF ? st.i >> 1 : st.i) & 1, 20, st.i);
    if constexpr (!BF) {
#pragma unroll
      for (int m = 0; m < SM::NIN; ++m)
        split_rows<F>(at + m * SM::TILE, SM::PLANE, reinterpret_cast<const float*>(mem + SM::RAWS + m * SM::RAW), GC, tid, THREADS);
      block_sync();
      if (tid == 0 && nx.i < walk.n) fetch(nx);
    }
    return at;
  }
  // a warp has left step i; all warps have left the step before i (its tiles and gates are free, what it wrote is complete)
  __device__ __forceinline__ void leave(int i) const {
    __syncwarp();
    if (lane == 0) mbar_arrive(bar + 16 + 8 * (i & 1));
  }
  __device__ __forceinline__ void settled(int i) const {
    if (i > 0) waits.wait(bar + 16 + 8 * ((i - 1) & 1), ((i - 1) >> 1) & 1, 25, i);
  }
  __device__ __forceinline__ volatile int* copies() const { return reinterpret_cast<volatile int*>(mem + SM::BAR + 40); }
  __device__ __forceinline__ void drain() const {  // copies that may still be on their way
    block_sync();
    if (tid == 0 && !waits.ok()) waits.drain(copies(), 2, bar);
  }
  static __device__ __forceinline__ void block_sync() { asm volatile("bar.sync 0, %0;" ::"n"(THREADS) : "memory"); }
  // W <- e^{G_end} W + sum of scaled keys^T values (REV: queries^T gradients, scaled by what is left at the token)
  __device__ __forceinline__ void update(float (&W)[SH::NT][4], uint32_t tk, uint32_t tv, const ChunkGates& cg, int row0, int col0) const {
    const uint32_t low = TL::low(lane), high = TL::high(lane);
    float sum[SH::NT][4];  // (the tensor cores truncate as they add: not onto the state)
#pragma unroll
    for (int k = 0; k < SH::NT; ++k) sum[k][0] = sum[k][1] = sum[k][2] = sum[k][3] = 0.f;
    const float* scale = REV ? cg.from : cg.end;
#pragma unroll 1
    for (int jt = 0; jt < GC / 16; ++jt) {
      const int j0 = 16 * jt + 2 * (lane & 3);
      Pk<NS> kt[4];
      {
        Pk<NP> f[4];
        ldsm_np<NP>(f, (tk + 16 * jt * TL::ROW + high) ^ (row0 << 1), SM::PLANE, true);
        scale_a_cols<NS, NP>(kt, f, ld2(scale + j0), ld2(scale + j0 + 8));
      }
      const uint32_t v = tv + 16 * jt * TL::ROW + low;
#pragma unroll
      for (int m = 0; m < SH::NT / 2; ++m) {
        Pk<NP> f[4];
        ldsm_np<NP>(f, v ^ ((col0 << 1) + (m << 5)), SM::PLANE, true);
        mma_planes<NS, NP>(sum[2 * m], sum[2 * m + 1], kt, f);
      }
    }
    const float all = cg.all;
#pragma unroll
    for (int k = 0; k < SH::NT; ++k) scale_add(W[k], all, sum[k]);
  }
};

template <typename T, int F, bool SAVE>
__global__ void __launch_bounds__(GF_THREADS, sizeof(T) == 2 ? 3 : 1)
    ttt_gated_fwd_kernel(const __grid_constant__ GatedMaps maps, const GatedParams p) {
  using BK = GatedFwdBlock<T, F, false, false, GF_THREADS>;
  using SM = typename BK::SM;
  using SH = StateShare<F>;
  using TL = GTile<F>;
  constexpr bool BF = BK::BF;
  constexpr int NP = BK::NP, KS = BK::KS;
  extern __shared__ uint8_t gated_smem[];
  const uint32_t raw = smem_u32(gated_smem), base = (raw + 1023) & ~1023u;
  uint8_t* const mem = gated_smem + (base - raw);
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5, g = lane >> 2, t4 = lane & 3;
  volatile int* const shared = reinterpret_cast<volatile int*>(mem + SM::BAR + 32);  // a wait has run out; this block's range
  BK bk{maps, p, mem, base, base + SM::BAR, reinterpret_cast<ChunkGates*>(mem + SM::GATES), {shared, p.status}, tid, lane, w, {}};
  if (tid == 0) {
    shared[0] = bk.copies()[0] = bk.copies()[1] = 0;
    shared[1] = p.slots > 0 ? atomicAdd(p.flags + p.slots, 1) + p.first_slot : (int)blockIdx.x;
    mbar_init(bk.bar, 1);
    mbar_init(bk.bar + 8, 1);
    mbar_init(bk.bar + 16, GATED_WARPS);
    mbar_init(bk.bar + 24, GATED_WARPS);
    fence_mbar_init();
  }
  __syncthreads();
  if (p.slots > 0 && shared[1] >= p.slots) return;  // (first_slot)
  bk.walk.set(p, shared[1], false);
  const int n = bk.walk.n;
  const GatedWalk::Step first = bk.walk.part(0), second = bk.walk.next(first);
  if (tid == 0) {
    bk.fetch(first);
    if (BF && n > 1) bk.fetch(second);
  }
  if (w < 2 && w < n) {
    float2 g0, b0;
    bk.gates_of(w == 0 ? first : second, g0, b0);
    make_chunk_gates<true>(bk.gates[w], lane, g0, b0);
  }
  const uint32_t low = TL::low(lane), high = TL::high(lane);
  const int row0 = 16 * (w % SH::SLABS), col0 = w / SH::SLABS * SH::COLS;
  float W[SH::NT][4];
  // the state before a step: operand of its q W, and what the backward reads back.  Where a stream or a part of one starts, from
  // memory
  auto publish = [&](const GatedWalk::Step& s) {
    if (s.starts) {
      const float* w0 = p.w0 != nullptr ? p.w0 + (size_t)s.stream * F * F : nullptr;
      if (s.pos > 0) {
        if (p.slots > 0) {
          if (lane == 0 && bk.waits.ok() && !wait_record(p.flags, bk.walk.slot - 1, p.polls)) bk.waits.fail(24, s.i);
          __syncwarp();
          w0 = p.records + (size_t)(bk.walk.slot - 1) * F * F;
        } else {
          w0 = p.seg_state + (size_t)bk.walk.slot * F * F;
        }
      }
      load_state<F>(W, w0, row0, col0, lane);
    }
    put_state<F, NP>(W, row0, col0, base + SM::W + (s.i & 1) * NP * TL::STATE_BYTES, lane);
    if (SAVE) put_fragments<F>(reinterpret_cast<float4*>(p.saved + ((size_t)s.stream * p.NC + s.pos) * F * F * 4), W, w, lane);
  };
  publish(first);
  __syncthreads();
  int slot3 = 0;  // i modulo 3
#pragma unroll 1
  for (GatedWalk::Step st = first, nx = second, fa; st.i < n; st = nx, nx = fa) {
    fa = bk.walk.next(nx);
    const int i = st.i, r = (w + i) & 3, slot3n = slot3 == 0 ? 2 : slot3 - 1;  // r: this warp's queries; (i + 2) modulo 3
    const bool ahead = r == 0 && fa.i < n;  // (the warp with one block)
    float2 g_next, b_next;
    if (ahead) bk.gates_of(fa, g_next, b_next);
    if (!BF) bk.settled(i);  // (one set of planes)
    const uint32_t tq = bk.tiles(st, nx), tk = tq + SM::TILE, tv = tk + SM::TILE, tw = base + SM::W + (i & 1) * NP * TL::STATE_BYTES;
    const ChunkGates& cg = bk.gates[slot3];
    float o[F / 8][4];
    Pk<NP> q[KS][4];
#pragma unroll
    for (int k = 0; k < F / 8; ++k) o[k][0] = o[k][1] = o[k][2] = o[k][3] = 0.f;
#pragma unroll
    for (int k = 0; k < KS; ++k) ldsm_np<NP>(q[k], (tq + 16 * r * TL::ROW + low) ^ (k << 5), SM::PLANE, false);
#pragma unroll 1
    for (int jt = 0; jt <= r; ++jt) {
      const int j0 = 16 * jt + 2 * t4;
      float s0[4] = {}, s1[4] = {};
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        Pk<NP> f[4];
        ldsm_np<NP>(f, (tk + 16 * jt * TL::ROW + high) ^ (k << 5), SM::PLANE, false);
        mma_planes<NP, NP>(s0, s1, q[k], f);
      }
      if (jt < r) {
        const F2 between = f2(cg.blocks[jt][r - 1]);
        scale_cols(s0, f2mul(ld2(&cg.out_b[j0]), between));
        scale_cols(s1, f2mul(ld2(&cg.out_b[j0 + 8]), between));
      } else {
        // what came from the blocks before, to each token of this one; then the block itself
        const float ra = cg.into[16 * r + g], rb = cg.into[16 * r + g + 8];
#pragma unroll
        for (int k = 0; k < F / 8; ++k) scale_rows(o[k], ra, rb);
        float d[2][4];
        block_decays<true>(d, cg, r, g, t4);
        const float2 b0 = ld2(&cg.beta[j0]), b1 = ld2(&cg.beta[j0 + 8]);
#pragma unroll
        for (int half = 0; half < 2; ++half) {  // (a select, not a product: what is not there may be infinite)
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
        ldsm_np<NP>(f, (tv + 16 * jt * TL::ROW + low) ^ (m << 5), SM::PLANE, true);
        mma_planes<NP, NP>(o[2 * m], o[2 * m + 1], a, f);
      }
    }
    bk.update(W, tk, tv, cg, row0, col0);
    if (BF) bk.settled(i);
    if (BF && r == 0 && lane == 0 && i > 0 && nx.i < n) bk.fetch(nx);
    if (ahead) make_chunk_gates<true>(bk.gates[slot3n], lane, g_next, b_next);
    const float fra = cg.from[16 * r + g], frb = cg.from[16 * r + g + 8];
#pragma unroll
    for (int k = 0; k < KS; ++k) ldsm_np<NP>(q[k], (tq + 16 * r * TL::ROW + low) ^ (k << 5), SM::PLANE, false);  // (again: the registers)
#pragma unroll
    for (int half = 0; half < 2; ++half) {  // (columns in two halves, for the registers)
      float c[F / 16][4];
#pragma unroll
      for (int k = 0; k < F / 16; ++k) c[k][0] = c[k][1] = c[k][2] = c[k][3] = 0.f;
#pragma unroll
      for (int k = 0; k < KS; ++k)
#pragma unroll
        for (int m = 0; m < KS / 2; ++m) {
          Pk<NP> f[4];
          ldsm_np<NP>(f, (tw + 16 * k * TL::ROW + low) ^ ((half * (KS / 2) + m) << 5), TL::STATE_BYTES, true);
          mma_planes<NP, NP>(c[2 * m], c[2 * m + 1], q[k], f);
        }
#pragma unroll
      for (int k = 0; k < F / 16; ++k) add_rows(o[half * (F / 16) + k], c[k], fra, frb);
    }
    if (st.ends) {
      if (st.pos == p.NC - 1) {
        store_state<F>(p.w_out + (size_t)st.stream * F * F, W, row0, col0, lane);
      } else if (p.slots > 0) {
        store_state<F>(p.records + (size_t)bk.walk.slot * F * F, W, row0, col0, lane);
        __threadfence();
        asm volatile("bar.sync 1, %0;" ::"n"(GF_THREADS) : "memory");
        if (tid == 0) set_record(p.flags, bk.walk.slot);
      }
    }
    if (nx.i < n) publish(nx);
    const int t0 = st.pos * GC;
    T* const out = static_cast<T*>(p.out) + ((size_t)st.stream * p.T + t0) * F;
    if constexpr (BF) {  // through this warp's rows of the queries' tile, which no other warp reads: whole lines at a time
      constexpr int VEC = F / 8, AT_ONCE = 32 / VEC;  // 16-byte pieces of a row; rows per store
      const uint32_t mine = tq + 16 * r * TL::ROW;
#pragma unroll
      for (int k = 0; k < F / 8; k += 2)
        stsm_x4((mine + low) ^ (k << 4), pack_bf16(o[k][0], o[k][1]), pack_bf16(o[k][2], o[k][3]), pack_bf16(o[k + 1][0], o[k + 1][1]),
                pack_bf16(o[k + 1][2], o[k + 1][3]));
      __syncwarp();
      uint4 v[16 / AT_ONCE];
#pragma unroll
      for (int k = 0; k < 16 / AT_ONCE; ++k) v[k] = ld_shared_v4(mine + TL::off(AT_ONCE * k + lane / VEC, lane % VEC * 8));
      fence_proxy_async_smem();  // (a later chunk's queries land where these rows were written)
      bk.leave(i);
#pragma unroll
      for (int k = 0; k < 16 / AT_ONCE; ++k) {
        const int row = 16 * r + AT_ONCE * k + lane / VEC;
        if (row < p.T - t0) *reinterpret_cast<uint4*>(out + (size_t)row * F + lane % VEC * 8) = v[k];
      }
    } else {
      bk.leave(i);
      store_rows<T, F>(out, 16 * r, p.T - t0, o, lane);
    }
    slot3 = slot3 == 2 ? 0 : slot3 + 1;
  }
  bk.drain();
}

// Every segment's own state, and what is left behind it of the state before it.  No warp needs another's rows: they share the tiles
// and the gates, made two chunks ahead.
// (Three blocks per SM: gated_split makes no more segments.  With registers for five, 96 instead of 140, 12 streams of 32768 tokens take
// 119 us, not 113.)
template <typename T, int F, bool REV>
__global__ void __launch_bounds__(GF_THREADS, sizeof(T) == 2 || F == 32 ? 3 : 2)
    ttt_gated_state_kernel(const __grid_constant__ GatedMaps maps, const GatedParams p) {
  using BK = GatedFwdBlock<T, F, true, REV, GF_THREADS>;
  using SM = typename BK::SM;
  using SH = StateShare<F>;
  constexpr bool BF = BK::BF;
  if ((int)blockIdx.x % p.nseg == (REV ? 0 : p.nseg - 1)) return;  // nothing follows it
  extern __shared__ uint8_t gated_smem[];
  const uint32_t raw = smem_u32(gated_smem), base = (raw + 1023) & ~1023u;
  uint8_t* const mem = gated_smem + (base - raw);
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
  volatile int* const failed = reinterpret_cast<volatile int*>(mem + SM::BAR + 32);
  BK bk{maps, p, mem, base, base + SM::BAR, reinterpret_cast<ChunkGates*>(mem + SM::GATES), {failed, p.status}, tid, lane, w, {}};
  if (tid == 0) {
    *failed = bk.copies()[0] = bk.copies()[1] = 0;
    mbar_init(bk.bar, 1);
    mbar_init(bk.bar + 8, 1);
    mbar_init(bk.bar + 16, GATED_WARPS);
    mbar_init(bk.bar + 24, GATED_WARPS);
    fence_mbar_init();
  }
  bk.walk.set(p, (int)blockIdx.x, REV);
  const int n = bk.walk.n;
  const GatedWalk::Step first = bk.walk.part(0), second = bk.walk.next(first);
  if (tid == 0) {
    bk.fetch(first);
    if (BF && n > 1) bk.fetch(second);
  }
  if (w < 2 && w < n) {
    float2 g0, b0;
    bk.gates_of(w == 0 ? first : second, g0, b0);
    make_chunk_gates<true>(bk.gates[w], lane, g0, b0);
  }
  __syncthreads();
  const int row0 = 16 * (w % SH::SLABS), col0 = w / SH::SLABS * SH::COLS;
  float W[SH::NT][4], total = 1.f;
  load_state<F>(W, nullptr, row0, col0, lane);
  int slot3 = 0;  // i modulo 3
#pragma unroll 1
  for (GatedWalk::Step st = first, nx = second, fa; st.i < n; st = nx, nx = fa) {
    fa = bk.walk.next(nx);
    const int i = st.i;
    const bool turn = w == (i & 3), ahead = turn && fa.i < n;
    float2 g_next, b_next;
    if (ahead) bk.gates_of(fa, g_next, b_next);
    bk.settled(BF ? i - 1 : i);  // (float32: one set of planes)
    const uint32_t tk = bk.tiles(st, nx);
    const ChunkGates& cg = bk.gates[slot3];
    total *= cg.all;
    bk.update(W, tk, tk + SM::TILE, cg, row0, col0);
    if (turn) {
      if (BF) bk.settled(i);
      if (BF && lane == 0 && i > 0 && nx.i < n) bk.fetch(nx);
      if (ahead) make_chunk_gates<true>(bk.gates[slot3 == 0 ? 2 : slot3 - 1], lane, g_next, b_next);
    }
    bk.leave(i);
    slot3 = slot3 == 2 ? 0 : slot3 + 1;
  }
  store_state<F>(p.seg_state + (size_t)bk.walk.slot * F * F, W, row0, col0, lane);
  if (tid == 0) p.seg_decay[bk.walk.slot] = total;
  bk.drain();
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

// Fewer streams than SMs are cut into segments; more streams than blocks are resident are cut into as many ranges as blocks are; between
// the two (148 to 444, backward 296; float32 none) there is a block per stream, whatever room that leaves.  Segments of at least LEAST
// chunks (2 against 4: 36 streams of 1201 tokens 28.7 and 32.8 us), in bf16 no more of them than blocks run at once (twice as many: 12
// streams of 32768 tokens 12 % slower).  float32 is cut into as many, of which one per SM runs at a time with F = 64 (178 KB of shared
// memory forward): two or three rounds; its ranges are counted for one block per SM, though the forward of F = 32 has room for two.  Ranges against a block per stream: training of
// 384 streams of 32 chunks 17 % faster, as no last round runs half empty.
void gated_split(int64_t streams, int chunks, int dtype, bool backward, int* nseg, int* slots) {
  constexpr int SMS = 148, LEAST = 2;  // (chunks per segment: a segment's states and its second reading must be worth it)
  const int resident = dtype == 1 ? (backward ? 2 : 3) : 1;
  *nseg = 1;
  *slots = 0;
  if (streams > (int64_t)SMS * resident) *slots = SMS * resident;
  if (streams >= SMS) return;
  const int64_t want = ((backward ? 2 : 3) * SMS) / streams, most = chunks / LEAST;
  *nseg = (int)(want < most ? want : most > 1 ? most : 1);
}

template <typename Fn>
static cudaError_t launch_one(Fn kfn, DeviceValue& ready, const GatedMaps& maps, const GatedParams& p, int grid, int threads, size_t smem,
                              cudaStream_t st) {
  int unused;
  const cudaError_t e = ready.get(0, &unused, [&](int* v) {
    *v = 0;
    return cudaFuncSetAttribute(kfn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  });
  if (e != cudaSuccess) return e;
  kfn<<<grid, threads, smem, st>>>(maps, p);
  return cudaGetLastError();
}
// The states before every segment (REV: the gradients of those behind)
template <typename T, int F, bool REV>
static cudaError_t launch_states(const GatedMaps& maps, const GatedParams& p, cudaStream_t st) {
  static DeviceValue ready;
  const cudaError_t e = launch_one(ttt_gated_state_kernel<T, F, REV>, ready, maps, p, p.nstreams * p.nseg, GF_THREADS,
                                   GatedFwdSmem<T, F, true>::BYTES, st);
  if (e != cudaSuccess) return e;
  ttt_gated_join_kernel<F, REV><<<(int)((long)p.nstreams * (F * F / 2) / JOIN_THREADS), JOIN_THREADS, 0, st>>>(p);
  return cudaGetLastError();
}

template <typename T, int F>
static cudaError_t launch_gated(const GatedMaps& maps, const GatedParams& p, bool save, cudaStream_t st) {
  cudaError_t e = cudaSuccess;
  if (p.nseg > 1) e = launch_states<T, F, false>(maps, p, st);
  else if (p.slots > 0) e = cudaMemsetAsync(p.flags, 0, (p.slots + 1) * sizeof(int), st);
  if (e != cudaSuccess) return e;
  static DeviceValue ready_save, ready;
  const int grid = p.slots > 0 ? p.slots : p.nstreams * p.nseg;
  constexpr size_t smem = GatedFwdSmem<T, F, false>::BYTES;
  return save ? launch_one(ttt_gated_fwd_kernel<T, F, true>, ready_save, maps, p, grid, GF_THREADS, smem, st)
              : launch_one(ttt_gated_fwd_kernel<T, F, false>, ready, maps, p, grid, GF_THREADS, smem, st);
}
cudaError_t launch_gated_fwd(int dtype, int F, const GatedMaps& maps, const GatedParams& p, bool save, cudaStream_t st) {
  if (F == 64) return dtype == 1 ? launch_gated<__nv_bfloat16, 64>(maps, p, save, st) : launch_gated<float, 64>(maps, p, save, st);
  return dtype == 1 ? launch_gated<__nv_bfloat16, 32>(maps, p, save, st) : launch_gated<float, 32>(maps, p, save, st);
}

// The gradient's states behind every segment: maps 1 and 2 are the queries and the output's gradient
cudaError_t launch_gated_segments_rev(int dtype, int F, const GatedMaps& maps, const GatedParams& p, cudaStream_t st) {
  if (F == 64) return dtype == 1 ? launch_states<__nv_bfloat16, 64, true>(maps, p, st) : launch_states<float, 64, true>(maps, p, st);
  return dtype == 1 ? launch_states<__nv_bfloat16, 32, true>(maps, p, st) : launch_states<float, 32, true>(maps, p, st);
}

}  // namespace ttt
