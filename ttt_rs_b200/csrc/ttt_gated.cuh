// Building blocks of the gated linear recurrence's kernels (ttt_gated_fwd.cu, ttt_gated_bwd.cu).
//
//   W_t = a_t W_{t-1} + beta_t k_t^T v_t,   o_t = q_t W_t,   a_t = exp(g_t)          (W is F x F, per (batch, head) stream)
//
// Tokens are taken in chunks of GC = 64.  With G_i = sum of g over the chunk up to and including token i and W the state
// before the chunk,
//   o_i  = e^{G_i} q_i W + sum_{j <= i} e^{G_i - G_j} beta_j (q_i . k_j) v_j
//   W'   = e^{G_end} W + sum_j (e^{G_end - G_j} beta_j k_j)^T v_j
// so everything but one product per chunk is a matrix product of 64-row tiles, and no exponent is ever positive for g <= 0:
// decays are formed as exponentials of differences, never as quotients.  The sums G are taken in 64 bits and carried as two
// floats, because a decay of zero (g = -inf: a new sequence begins) counts as one of 2^-160 (zero in float32), after which G is
// large and its differences would keep few digits.
//
// Operands.  bf16 inputs go to the tensor cores as they are; what a result of the inputs' type alone depends on is rounded to bf16 where
// it becomes an operand (the decayed products, the state in q W).  What float32 results depend on is not: the scaled keys and
// queries whose products make up the state and its gradient are carried as three bf16 planes (24 bits of mantissa, as float32; two
// planes left 2.5e-6 of the state, three 5e-7, for 4 % of the forward's time), and so are the state and its gradient in the sums for
// the gates' gradients (two planes: 1.9e-6 of those, three 4e-7, for 8 % of the training pass).  float32 inputs are carried as three planes
// throughout, as in the other float32 kernels.  A chunk's part of the state is a sum of its own, added to the decayed state by a fused
// multiply-add: the tensor cores truncate as they add, and onto the state itself that lost 2e-5 of it in 128 chunks of weak decay.
#pragma once

#include "ttt_common.cuh"
#include "ttt_stage.cuh"

namespace ttt {

constexpr int GC = 64;            // tokens per chunk
constexpr int GATED_WARPS = 4;    // warps that share the rows of a chunk, 16 each
constexpr float GATED_ZERO = -160.f;  // log2 of a decay that is zero

template <>
__device__ __forceinline__ Pk<2> split_pack<2>(float x, float y) {
  Pk<2> r;
  r.p[0] = pack_bf16(x, y);
  const float2 rest = __ffma2_rn(make_float2(bf16_lo(r.p[0]), bf16_hi(r.p[0])), make_float2(-1.f, -1.f), make_float2(x, y));
  r.p[1] = pack_bf16(rest.x, rest.y);
  return r;
}

// 2^x; results below 2^-126 are zero (exp2f spends three instructions more on those)
__device__ __forceinline__ float pow2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// A bf16 tile of rows of F elements (128 or 64 bytes) in the swizzle of TMA: rows 0..63, any multiple of 8 columns
template <int F>
struct GTile {
  static constexpr uint32_t ROW = F * 2, BYTES = GC * ROW, STATE_BYTES = F * ROW;
  static __device__ __forceinline__ uint32_t off(int row, int col) {
    const int x = F == 64 ? (row & 7) : ((row >> 1) & 3);
    return (uint32_t)(row * (int)ROW + (((col >> 3) ^ x) << 4) + ((col & 7) << 1));
  }
  // Lane addresses of ldmatrix.x4 within 16 rows: the address of a 16 x 16 block at row r (a multiple of 16) and column 16 c is
  // (tile + r * ROW + lane part) ^ (c << 5), the tile on 128 bytes: the swizzle is an exclusive or with the row.
  // low: matrices 0..3 at (0, 0), (8, 0), (0, 8), (8, 8): A operands stored [row][k], B operands stored [k][n] (.trans)
  static __device__ __forceinline__ uint32_t low(int lane) { return off((lane & 7) + ((lane >> 3) & 1) * 8, (lane >> 4) * 8); }
  // high: at (0, 0), (0, 8), (8, 0), (8, 8): B operands stored [n][k], A operands stored [k][row] (.trans)
  static __device__ __forceinline__ uint32_t high(int lane) { return off((lane & 7) + (lane >> 4) * 8, ((lane >> 3) & 1) * 8); }
};

// c0 += a . b[0..1], c1 += a . b[2..3]: the products of planes whose weight is at least 2^-16 of the leading one
template <int NA, int NB>
__device__ __forceinline__ void mma_planes(float (&c0)[4], float (&c1)[4], const Pk<NA> (&a)[4], const Pk<NB> (&b)[4]) {
  if constexpr (NA == 3 && NB == 3) {
    const Pk<3> b0[2] = {b[0], b[1]}, b1[2] = {b[2], b[3]};
    mma_np2<3>(c0, a, b0, c1, a, b1);
  } else {
    static_assert(NA == 1 || NB == 1, "planes");
#pragma unroll
    for (int i = NA * NB - 1; i >= 0; --i) {  // the small planes first
      const int pa = NA > 1 ? i : 0, pb = NB > 1 ? i : 0;
      mma_bf16(c0, a[0].p[pa], a[1].p[pa], a[2].p[pa], a[3].p[pa], b[0].p[pb], b[1].p[pb]);
      mma_bf16(c1, a[0].p[pa], a[1].p[pa], a[2].p[pa], a[3].p[pa], b[2].p[pb], b[3].p[pb]);
    }
  }
}

// rows g and g + 8 of an accumulator tile times a factor each; its column pair times a pair
__device__ __forceinline__ void scale_rows(float (&c)[4], float a, float b) {
  const F2 x = f2mul(make_float2(c[0], c[1]), f2(a)), y = f2mul(make_float2(c[2], c[3]), f2(b));
  c[0] = x.x, c[1] = x.y, c[2] = y.x, c[3] = y.y;
}
__device__ __forceinline__ void scale_cols(float (&c)[4], F2 f) {
  const F2 x = f2mul(make_float2(c[0], c[1]), f), y = f2mul(make_float2(c[2], c[3]), f);
  c[0] = x.x, c[1] = x.y, c[2] = y.x, c[3] = y.y;
}
// c = c times a factor + d
__device__ __forceinline__ void scale_add(float (&c)[4], float a, const float (&d)[4]) {
  const F2 x = f2fma(make_float2(c[0], c[1]), f2(a), make_float2(d[0], d[1]));
  const F2 y = f2fma(make_float2(c[2], c[3]), f2(a), make_float2(d[2], d[3]));
  c[0] = x.x, c[1] = x.y, c[2] = y.x, c[3] = y.y;
}
// d += rows of c times a factor each
__device__ __forceinline__ void add_rows(float (&d)[4], const float (&c)[4], float a, float b) {
  const F2 x = f2fma(make_float2(c[0], c[1]), f2(a), make_float2(d[0], d[1]));
  const F2 y = f2fma(make_float2(c[2], c[3]), f2(b), make_float2(d[2], d[3]));
  d[0] = x.x, d[1] = x.y, d[2] = y.x, d[3] = y.y;
}
// two accumulator tiles (16 rows x 16 columns) as an A operand
template <int NP>
__device__ __forceinline__ void as_operand(Pk<NP> (&a)[4], const float (&c0)[4], const float (&c1)[4]) {
  a[0] = split_pack<NP>(c0[0], c0[1]);
  a[1] = split_pack<NP>(c0[2], c0[3]);
  a[2] = split_pack<NP>(c1[0], c1[1]);
  a[3] = split_pack<NP>(c1[2], c1[3]);
}
__device__ __forceinline__ float2 ld2(const float* p) { return *reinterpret_cast<const float2*>(p); }

template <int NP>
__device__ __forceinline__ float pk_lo(const Pk<NP>& v) {
  float s = 0.f;
#pragma unroll
  for (int i = NP - 1; i >= 0; --i) s += bf16_lo(v.p[i]);
  return s;
}
template <int NP>
__device__ __forceinline__ float pk_hi(const Pk<NP>& v) {
  float s = 0.f;
#pragma unroll
  for (int i = NP - 1; i >= 0; --i) s += bf16_hi(v.p[i]);
  return s;
}
// an A fragment (lane 4g + t: columns 2t, 2t+1 in [0], [1]; 2t+8, 2t+9 in [2], [3]) with its columns scaled
template <int NO, int NI>
__device__ __forceinline__ void scale_a_cols(Pk<NO> (&o)[4], const Pk<NI> (&a)[4], float2 lo, float2 hi) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 v = f2mul(make_float2(pk_lo(a[i]), pk_hi(a[i])), i < 2 ? lo : hi);
    o[i] = split_pack<NO>(v.x, v.y);
  }
}

// The gates of a chunk, for all warps of a block.  A decay between tokens of different blocks of 16 is the product of what is
// left at the end of the first one's block, of the blocks between, and at the second one from the start of its block: factors
// of rows, of pairs of blocks and of columns, none above 1 for g <= 0.  Only pairs within a block take an exponential each.
struct ChunkGates {
  float hi[GC], lo[GC];  // G_i in units of log2, in two floats
  float from[GC];        // e^{G_i}: what is left at token i of the state before the chunk
  float into[GC];        // the same of the state before i's block
  float out[GC];         // what is left of token i behind its block
  float out_b[GC];       // that times beta_i
  float end[GC];         // what is left of token i behind the chunk (forward: times beta_i)
  float beta[GC];
  float blocks[4][4];    // [a][b]: from the end of block a to the end of block b >= a
  float starts[4];       // e^G before block a
  float all;             // e^{G_end}
  float pad[3];
};
// FORWARD: `end` comes with the factor beta.  One warp; lane l brings tokens 2l and 2l + 1 of the chunk.  Tokens behind the sequence:
// g = 0, beta = 0.
template <bool FORWARD>
__device__ __forceinline__ void make_chunk_gates(ChunkGates& s, int lane, float2 g, float2 beta) {
  auto log2_of = [](float x) {
    const double v = (double)x * 1.4426950408889634;
    return v < (double)GATED_ZERO ? (double)GATED_ZERO : v;  // (a NaN stays one)
  };
  const double g0 = log2_of(g.x), g1 = log2_of(g.y);
  double sum = g0 + g1;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const double up = __shfl_up_sync(0xffffffffu, sum, o);
    if (lane >= o) sum += up;
  }
  const int blk = lane >> 3;
  const double G0 = sum - g1, G1 = sum, end = __shfl_sync(0xffffffffu, sum, 31);
  double ends[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) ends[k] = __shfl_sync(0xffffffffu, sum, 8 * k + 7);
  const double mine = blk == 0 ? ends[0] : blk == 1 ? ends[1] : blk == 2 ? ends[2] : ends[3];
  const double before = blk == 0 ? 0.0 : blk == 1 ? ends[0] : blk == 2 ? ends[1] : ends[2];
  auto put = [&](float* a, float x, float y) { *reinterpret_cast<float2*>(a + 2 * lane) = make_float2(x, y); };
  const float h0 = (float)G0, h1 = (float)G1;
  put(s.hi, h0, h1);
  put(s.lo, (float)(G0 - h0), (float)(G1 - h1));
  put(s.from, pow2((float)G0), pow2((float)G1));
  put(s.into, pow2((float)(G0 - before)), pow2((float)(G1 - before)));
  const float o0 = pow2((float)(mine - G0)), o1 = pow2((float)(mine - G1));
  const float e0 = pow2((float)(end - G0)), e1 = pow2((float)(end - G1));
  put(s.out, o0, o1);
  put(s.out_b, o0 * beta.x, o1 * beta.y);
  put(s.end, FORWARD ? e0 * beta.x : e0, FORWARD ? e1 * beta.y : e1);
  put(s.beta, beta.x, beta.y);
  if (lane < 16) {
    const int a = lane >> 2, b = lane & 3;
    double ga = ends[0], gb = ends[0];
#pragma unroll
    for (int k = 1; k < 4; ++k) {
      if (a == k) ga = ends[k];
      if (b == k) gb = ends[k];
    }
    s.blocks[a][b] = b >= a ? pow2((float)(gb - ga)) : 0.f;
    if (b == 0) s.starts[a] = a == 0 ? 1.f : pow2((float)(a == 1 ? ends[0] : a == 2 ? ends[1] : ends[2]));
  }
  if (lane == 0) s.all = pow2((float)end);
}
// Decays e^{G_i - G_j} of the 16 x 16 pairs of block `blk` with row r (g, g + 8) and column c (2t, 2t + 1, 2t + 8, 2t + 9) of a
// lane's accumulators: [row half][column]; rows are i (ROWS_LATE) or j.  Zero where i < j.
template <bool ROWS_LATE>
__device__ __forceinline__ void block_decays(float (&d)[2][4], const ChunkGates& s, int blk, int g, int t4) {
  const int r0 = 16 * blk + g, c0 = 16 * blk + 2 * t4;
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const int r = r0 + 8 * half;
    const float hr = s.hi[r], lr = s.lo[r];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int c = c0 + (e & 1) + 8 * (e >> 1);
      const float x = (hr - s.hi[c]) + (lr - s.lo[c]);
      d[half][e] = (ROWS_LATE ? c <= r : c >= r) ? pow2(ROWS_LATE ? x : -x) : 0.f;
    }
  }
}
// what lane `lane` brings for the chunk that starts at token t0
__device__ __forceinline__ float2 load_gates(const float* x, int t0, int T, int lane, float none) {
  const int t = t0 + 2 * lane;
  float2 v = make_float2(0.f, 0.f);
  if (t < T) v.x = x != nullptr ? x[t] : none;
  if (t + 1 < T) v.y = x != nullptr ? x[t + 1] : none;
  return v;
}

// Accumulators of 16 rows x F columns to global rows base[row * F], rows below `rows`: the four lanes of a row store
// 32 bytes side by side (bf16 in 64, after more shuffles: 1 % of the training pass slower).
template <typename T, int F>
__device__ __forceinline__ void store_rows(T* base, int row0, int rows, const float (&c)[F / 8][4], int lane) {
  const int g = lane >> 2, t = lane & 3;
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const int row = row0 + g + 8 * half;
    if constexpr (sizeof(T) == 2) {
#pragma unroll
      for (int n = 0; n < F / 8; n += 2) {  // two lanes swap halves of two tiles: 8 bytes each, whole sectors of 32
        const uint32_t x = pack_bf16(c[n][2 * half], c[n][2 * half + 1]), y = pack_bf16(c[n + 1][2 * half], c[n + 1][2 * half + 1]);
        const bool odd = lane & 1;
        const uint32_t got = __shfl_xor_sync(0xffffffffu, odd ? x : y, 1);
        if (row < rows)
          *reinterpret_cast<uint2*>(base + (size_t)row * F + 8 * (n + (t & 1)) + 4 * (t >> 1)) = odd ? make_uint2(got, y) : make_uint2(x, got);
      }
    } else if (row < rows) {
#pragma unroll
      for (int n = 0; n < F / 8; ++n)
        *reinterpret_cast<float2*>(base + (size_t)row * F + 8 * n + 2 * t) = make_float2(c[n][2 * half], c[n][2 * half + 1]);
    }
  }
}

// float32 rows as TMA lays them ([rows][F], no swizzle) -> three planes of bf16 tiles
template <int F>
__device__ __forceinline__ void split_rows(uint32_t planes, uint32_t plane_stride, const float* src, int rows, int tid, int threads) {
  constexpr int Q = F / 4;
  for (int e = tid; e < rows * Q; e += threads) {
    const int row = e / Q, col = 4 * (e - row * Q);
    const float4 v = *reinterpret_cast<const float4*>(src + 4 * e);
    const Pk<3> a = split_pack<3>(v.x, v.y), b = split_pack<3>(v.z, v.w);
#pragma unroll
    for (int i = 0; i < 3; ++i)
      asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(planes + i * plane_stride + GTile<F>::off(row, col)), "r"(a.p[i]),
                   "r"(b.p[i])
                   : "memory");
  }
}
__device__ __forceinline__ uint4 ld_shared_v4(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}

// 4-D TMA load: features, tokens, heads, batch
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* tm, int y, int z, int w, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
      "l"(tm), "r"(0), "r"(y), "r"(z), "r"(w), "r"(bar)
      : "memory");
}

__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}

// What a block walks: steps of one chunk each.  A stream's chunks are numbered in walk order (`pos`; the backward walks from the
// last chunk).  With p.slots = 0 a block has one segment of one stream.  Else (more streams than blocks are resident) all steps
// of all streams, stream after stream, are cut into p.slots equal ranges, of at least a stream's length each: a block's range is
// the end of one stream, whole streams, and the beginning of another.  It begins with that beginning, whose state it hands on
// to the block of the next range, and ends with the end of the first stream, whose state it gets from the block of the range before:
// by then that block is long past it.  Ranges are numbered in the order in which blocks start, so that what a block waits for
// has always started.
struct GatedWalk {
  int slot, n;            // range; steps
  int head, head_n;       // stream and steps of the beginning
  int mid, mid_n;         // first whole stream, steps of all of them
  int tail, tail_pos;     // stream and first chunk of the end
  int NC;
  struct Step {
    int i, stream, pos;
    bool starts, ends;  // a stream or a part of one starts, ends with this step
  };
  template <class P>
  __device__ __forceinline__ void set(const P& p, int slot_, bool rev) {
    slot = slot_;
    NC = p.NC;
    head = mid = tail = head_n = mid_n = tail_pos = 0;
    if (p.slots == 0) {
      tail = slot / p.nseg;
      const int seg = slot - tail * p.nseg, lo = seg * p.seg_chunks, hi = min(NC, lo + p.seg_chunks);
      tail_pos = rev ? NC - hi : lo;
      n = hi - lo;
      return;
    }
    const long long total = (long long)p.nstreams * NC;
    const long long a = total * slot / p.slots, b = total * (slot + 1) / p.slots;
    const int sa = (int)(a / NC), pa = (int)(a - (long long)sa * NC), sb = (int)(b / NC), pb = (int)(b - (long long)sb * NC);
    n = (int)(b - a);
    tail = sa;
    tail_pos = pa;
    head = sb;
    head_n = pb;
    mid = pa > 0 ? sa + 1 : sa;
    mid_n = (sb - mid) * NC;
  }
  __device__ __forceinline__ Step part(int i) const {  // the step that a part starts with
    Step s;
    s.i = i;
    s.starts = true;
    s.stream = i < head_n ? head : tail;
    s.pos = i < head_n ? 0 : tail_pos;
    if (i >= head_n && i < head_n + mid_n) {
      s.stream = mid + (i - head_n) / NC;
      s.pos = 0;
    }
    s.ends = last(s);
    return s;
  }
  __device__ __forceinline__ bool last(const Step& s) const { return s.pos + 1 == NC || s.i + 1 == head_n || s.i + 1 == n; }
  __device__ __forceinline__ Step next(const Step& s) const {  // (behind the last step: one that is not used)
    if (s.ends) return part(s.i + 1);
    Step t = s;
    ++t.i;
    ++t.pos;
    t.starts = false;
    t.ends = last(t);
    return t;
  }
};
// Waits of a block.  One that runs out is reported, and from then on no wait waits and no copy starts: every warp still passes all the
// barriers that the others meet it at, on its way to the end, and what the launch writes is not valid.
struct GatedWaits {
  volatile int* failed;  // shared memory
  uint32_t* status;
  __device__ __forceinline__ bool ok() const { return *failed == 0; }
  __device__ __forceinline__ void fail(uint32_t where, int step) const {
    report_timeout(status, where, (uint32_t)step);
    *failed = 1;
  }
  __device__ __forceinline__ void wait(uint32_t bar, uint32_t parity, uint32_t where, int step) const {
    if (ok() && !mbar_wait_bounded(bar, parity)) fail(where, step);
  }
  // The last copy that was started on barrier k of `copies`: its parity, and 2.  Written before the copy starts, by the thread that
  // starts it.
  __device__ __forceinline__ void started(volatile int* copies, int k, uint32_t parity) const { copies[k] = (int)parity | 2; }
  // One thread, behind a barrier of all threads after a wait has run out: the block ends only with its copies complete
  __device__ __forceinline__ void drain(volatile const int* copies, int count, uint32_t bar) const {
    for (int k = 0; k < count; ++k)
      if (copies[k] != 0) mbar_wait_bounded(bar + 8 * k, copies[k] & 1);
  }
};

// One thread: the record of range `slot` has been handed on (false: the wait ran out)
__device__ __forceinline__ bool wait_record(const int* flags, int slot, uint32_t polls) {
  for (uint32_t i = 0; i < polls; ++i) {
    int v;
    asm volatile("ld.acquire.gpu.global.s32 %0, [%1];" : "=r"(v) : "l"(flags + slot) : "memory");
    if (v != 0) return true;
    __nanosleep(100);
  }
  return false;
}
__device__ __forceinline__ void set_record(int* flags, int slot) {
  asm volatile("st.release.gpu.global.s32 [%0], %1;" ::"l"(flags + slot), "r"(1) : "memory");
}

// How the F x F state lies in the registers of four warps: warp w holds rows 16 (w % SLABS).. and the columns of its part
template <int F>
struct StateShare {
  static constexpr int SLABS = F / 16, PARTS = GATED_WARPS / SLABS, COLS = F / PARTS, NT = COLS / 8;
};

// A warp's share of the state (rows row0.., columns col0..) as NP bf16 planes (`stride` bytes apart) in the tile layout of shared
// memory
template <int F, int NP>
__device__ __forceinline__ void put_state(const float (&w)[StateShare<F>::NT][4], int row0, int col0, uint32_t smem, int lane,
                                          uint32_t stride = GTile<F>::STATE_BYTES) {
  const uint32_t at = smem + row0 * GTile<F>::ROW + GTile<F>::low(lane);
#pragma unroll
  for (int n = 0; n < StateShare<F>::NT; n += 2) {
    Pk<NP> v[4];
    as_operand<NP>(v, w[n], w[n + 1]);
#pragma unroll
    for (int i = 0; i < NP; ++i)
      stsm_x4((at ^ ((col0 + 8 * n) << 1)) + i * stride, v[0].p[i], v[1].p[i], v[2].p[i], v[3].p[i]);
  }
}
// The same share as the threads hold it, 16 bytes a thread side by side (what the forward saves for the backward)
template <int F>
__device__ __forceinline__ void put_fragments(float4* m, const float (&w)[StateShare<F>::NT][4], int warp, int lane) {
#pragma unroll
  for (int n = 0; n < StateShare<F>::NT; ++n)
    m[(warp * StateShare<F>::NT + n) * 32 + lane] = make_float4(w[n][0], w[n][1], w[n][2], w[n][3]);
}
template <int F>
__device__ __forceinline__ void get_fragments(float (&w)[StateShare<F>::NT][4], const float4* m, int warp, int lane) {
#pragma unroll
  for (int n = 0; n < StateShare<F>::NT; ++n) {
    const float4 v = m[(warp * StateShare<F>::NT + n) * 32 + lane];
    w[n][0] = v.x, w[n][1] = v.y, w[n][2] = v.z, w[n][3] = v.w;
  }
}
// The same share to and from a float32 matrix [F][F]
template <int F>
__device__ __forceinline__ void store_state(float* m, const float (&w)[StateShare<F>::NT][4], int row0, int col0, int lane) {
#pragma unroll
  for (int n = 0; n < StateShare<F>::NT; ++n)
#pragma unroll
    for (int half = 0; half < 2; ++half)
      *reinterpret_cast<float2*>(m + (size_t)(row0 + (lane >> 2) + 8 * half) * F + col0 + 8 * n + 2 * (lane & 3)) =
          make_float2(w[n][2 * half], w[n][2 * half + 1]);
}
template <int F>
__device__ __forceinline__ void load_state(float (&w)[StateShare<F>::NT][4], const float* m, int row0, int col0, int lane) {
#pragma unroll
  for (int n = 0; n < StateShare<F>::NT; ++n)
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      float2 v = make_float2(0.f, 0.f);
      if (m != nullptr)
        v = *reinterpret_cast<const float2*>(m + (size_t)(row0 + (lane >> 2) + 8 * half) * F + col0 + 8 * n + 2 * (lane & 3));
      w[n][2 * half] = v.x;
      w[n][2 * half + 1] = v.y;
    }
}

}  // namespace ttt
