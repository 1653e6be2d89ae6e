// C ABI of the operators of a selective state space layer (include/ttt_b200.h): causal convolution, the scan, group norm with channels last.
// Argument checks and launches.
#include <cstdarg>
#include <cstdio>
#include <initializer_list>

#include "../../include/ttt_b200.h"
#include "ttt_kernels.h"

namespace ttt {
int abi_error(int code, const char* message);  // ttt_abi.cu: the thread's last error
}

namespace {

int fail(int code, const char* fmt, ...) {
  char message[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(message, sizeof(message), fmt, ap);
  va_end(ap);
  return ttt::abi_error(code, message);
}
int launched(cudaError_t e, const char* what) {
  return e == cudaSuccess ? TTT_OK : fail(TTT_ERR_CUDA, "%s launch failed: %s", what, cudaGetErrorString(e));
}

constexpr int64_t kMostChannels = 1 << 20;
constexpr int64_t kFarthest = (int64_t)1 << 58;  // elements that one stride reaches: three of them are still an int64 of bytes

int check_sizes(int64_t B, int64_t T, int64_t C, int dtype) {
  if (B <= 0 || T <= 0 || C <= 0) return fail(TTT_ERR_SHAPE, "batch, seq_len and channels must be positive");
  if (dtype != TTT_F32 && dtype != TTT_BF16) return fail(TTT_ERR_UNSUPPORTED, "unknown dtype %d", dtype);
  if (C > kMostChannels) return fail(TTT_ERR_UNSUPPORTED, "at most %lld channels", (long long)kMostChannels);
  if (B >= (int64_t)1 << 31 || T >= (int64_t)1 << 31 || B * T >= (int64_t)1 << 31) return fail(TTT_ERR_SHAPE, "batch*seq_len must be below 2^31");
  return TTT_OK;
}
int check_bytes(size_t have, size_t need, const void* p, const char* name) {
  if (need == 0) return TTT_OK;
  if (p == nullptr || have < need) return fail(TTT_ERR_WORKSPACE, "%s has %zu bytes, %zu needed", name, p == nullptr ? (size_t)0 : have, need);
  if ((reinterpret_cast<uintptr_t>(p) & 15u) != 0) return fail(TTT_ERR_ALIGN, "%s is not 16-byte aligned", name);
  return TTT_OK;
}

// Tensors [B,T,C] (or shorter) with contiguous channels: widest vector of channels that all of them allow, and the bytes they span.
struct Spans {
  int64_t B, T, C;
  int es;
  uintptr_t low = 0;  // OR of the addresses and strides in bytes: what they are multiples of
  int rc = TTT_OK;
  void align(const char* name, const void* p) {
    if (rc != TTT_OK || p == nullptr) return;
    if (reinterpret_cast<uintptr_t>(p) % es != 0) rc = fail(TTT_ERR_ALIGN, "%s is not aligned to its elements", name);
    low |= reinterpret_cast<uintptr_t>(p);
  }
  void need(const char* name, const void* p) {
    if (rc == TTT_OK && p == nullptr) rc = fail(TTT_ERR_NULL, "%s is null", name);
    align(name, p);
  }
  // strides of batch and token of tensor `i` (null: contiguous), 0 where there is one row only
  void rows(const char* name, const void* p, const int64_t* strides, int i, int64_t (&out)[2], bool optional = false) {
    out[0] = out[1] = 0;
    if (optional && p == nullptr) return;
    need(name, p);
    const int64_t dense[2] = {T * C, C}, size[2] = {B, T};
    for (int k = 0; k < 2; ++k) {
      out[k] = size[k] == 1 ? 0 : strides != nullptr ? strides[2 * i + k] : dense[k];
      low |= (uintptr_t)(out[k] * es);
      if (rc == TTT_OK && out[k] < 0) rc = fail(TTT_ERR_SHAPE, "the strides of %s must not be negative", name);
      if (rc == TTT_OK && out[k] > kFarthest / size[k]) rc = fail(TTT_ERR_SHAPE, "the strides of %s are out of range", name);
    }
  }
  int64_t bytes(const int64_t (&s)[2]) const { return ((B - 1) * s[0] + (T - 1) * s[1] + C) * es; }
  bool contiguous(const int64_t (&s)[2]) const { return (B == 1 || s[0] == T * C) && (T == 1 || s[1] == C); }
};
// Bytes of a tensor of the call, and its kinds, bit by bit
struct Region {
  const char* name;
  const void* p;
  int64_t bytes;
  unsigned kinds;
};
// Results (contiguous) share nothing with one another, nor with an input, except that a result may be an input, all of it, of one of its
// kinds: those are read, by the thread that writes in their place or by an earlier launch, before they are written.
int check_apart(std::initializer_list<Region> results, std::initializer_list<Region> inputs) {
  auto meet = [](const Region& a, const Region& b) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a.p), y = reinterpret_cast<uintptr_t>(b.p);
    return a.p != nullptr && b.p != nullptr && x < y + (uintptr_t)b.bytes && y < x + (uintptr_t)a.bytes;
  };
  for (const Region& r : results) {
    for (const Region& in : inputs)
      if (meet(r, in) && !((r.kinds & in.kinds) != 0 && r.p == in.p && r.bytes == in.bytes))
        return fail(TTT_ERR_SHAPE, "%s lies over %s", r.name, in.name);
    for (const Region& other : results) {
      if (&other == &r) break;
      if (meet(r, other)) return fail(TTT_ERR_SHAPE, "%s lies over %s", r.name, other.name);
    }
  }
  return TTT_OK;
}

int check_conv(int64_t B, int64_t T, int64_t C, int taps, int dtype, int activation) {
  const int rc = check_sizes(B, T, C, dtype);
  if (rc != TTT_OK) return rc;
  if (taps < 2 || taps > 4) return fail(TTT_ERR_UNSUPPORTED, "Unsupported taps=%d (supported: 2, 3, 4)", taps);
  if (activation != ttt::ACT_NONE && activation != ttt::ACT_SILU)
    return fail(TTT_ERR_UNSUPPORTED, "unknown activation %d (0: none, 1: SiLU)", activation);
  return TTT_OK;
}

int conv_width(uintptr_t low, int64_t channels, int es) {
  if (low % (4 * es) == 0 && channels % 4 == 0) return 4;
  return es == 2 && low % 4 == 0 && channels % 2 == 0 ? 2 : 1;
}

}  // namespace

extern "C" int ttt_layer_causal_conv(int64_t batch, int64_t seq_len, int64_t channels, int taps, int dtype, int activation, const void* x,
                                     const int64_t* x_strides, const void* weight, const void* bias, const void* state,
                                     const void* starts, void* y, void* state_out, void* stream) {
  int rc = check_conv(batch, seq_len, channels, taps, dtype, activation);
  if (rc != TTT_OK) return rc;
  const int es = dtype == TTT_BF16 ? 2 : 4;
  ttt::ConvParams p{};
  Spans s{batch, seq_len, channels, es};
  s.rows("x", x, x_strides, 0, p.xs);
  s.need("y", y);
  s.need("state_out", state_out);
  s.align("state", state);
  s.need("weight", weight);
  const int width = conv_width(s.low, channels, es);
  s.align("bias", bias);
  if (s.rc != TTT_OK) return s.rc;
  const int64_t held = batch * (taps - 1) * channels * es, n = batch * seq_len * channels * es;
  if ((rc = check_apart({{"state_out", state_out, held, 1}, {"y", y, n, 0}},
                        {{"x", x, s.bytes(p.xs), 0}, {"weight", weight, channels * taps * es, 0}, {"bias", bias, channels * es, 0},
                         {"state", state, held, 1}, {"starts", starts, batch * seq_len, 0}})) != TTT_OK)
    return rc;
  p.x = x, p.w = weight, p.bias = bias, p.state = state, p.starts = static_cast<const uint8_t*>(starts);
  p.y = y, p.state_out = state_out;
  p.B = batch, p.T = seq_len, p.C = (int)channels, p.act = activation;
  return launched(ttt::launch_conv(dtype, p, taps, width, false, static_cast<cudaStream_t>(stream)), "causal convolution");
}

extern "C" size_t ttt_layer_causal_conv_backward_workspace_bytes(int64_t batch, int64_t seq_len, int64_t channels, int taps, int dtype) {
  if (check_conv(batch, seq_len, channels, taps, dtype, 0) != TTT_OK) return 0;
  return sizeof(float) * ttt::conv_partial_floats(batch, seq_len, (int)channels, taps);
}

extern "C" int ttt_layer_causal_conv_backward(int64_t batch, int64_t seq_len, int64_t channels, int taps, int dtype, int activation,
                                              const void* x, const void* grad_y, const int64_t* strides, const void* weight,
                                              const void* bias, const void* state, const void* starts, const void* grad_state_out,
                                              void* grad_x, void* grad_weight, void* grad_bias, void* grad_state, void* workspace,
                                              size_t workspace_bytes, void* stream) {
  int rc = check_conv(batch, seq_len, channels, taps, dtype, activation);
  if (rc != TTT_OK) return rc;
  const int es = dtype == TTT_BF16 ? 2 : 4;
  ttt::ConvParams p{};
  Spans s{batch, seq_len, channels, es};
  s.rows("x", x, strides, 0, p.xs);
  s.rows("grad_y", grad_y, strides, 1, p.gs);
  s.need("grad_x", grad_x);
  s.align("state", state);
  s.align("grad_state_out", grad_state_out);
  s.align("grad_state", grad_state);
  s.need("weight", weight);
  const int width = conv_width(s.low, channels, es);
  s.align("bias", bias);
  s.align("grad_weight", grad_weight);
  s.align("grad_bias", grad_bias);
  if (s.rc != TTT_OK) return s.rc;
  const size_t need =
      grad_weight != nullptr || grad_bias != nullptr ? ttt_layer_causal_conv_backward_workspace_bytes(batch, seq_len, channels, taps, dtype) : 0;
  if ((rc = check_bytes(workspace_bytes, need, workspace, "workspace")) != TTT_OK) return rc;
  const int64_t held = batch * (taps - 1) * channels * es, n = batch * seq_len * channels * es, taps_bytes = channels * taps * es;
  if ((rc = check_apart({{"grad_x", grad_x, n, 0}, {"grad_state", grad_state, held, 1}, {"grad_weight", grad_weight, taps_bytes, 2},
                         {"grad_bias", grad_bias, channels * es, 4}, {"workspace", need != 0 ? workspace : nullptr, (int64_t)need, 0}},
                        {{"x", x, s.bytes(p.xs), 0}, {"grad_y", grad_y, s.bytes(p.gs), 0}, {"weight", weight, taps_bytes, 2},
                         {"bias", bias, channels * es, 4}, {"state", state, held, 1}, {"starts", starts, batch * seq_len, 0},
                         {"grad_state_out", grad_state_out, held, 0}})) != TTT_OK)
    return rc;
  p.x = x, p.w = weight, p.bias = bias, p.state = state, p.starts = static_cast<const uint8_t*>(starts);
  p.gy = grad_y, p.gstate_out = grad_state_out, p.gx = grad_x, p.gstate = grad_state, p.gw = grad_weight, p.gbias = grad_bias;
  p.partials = need != 0 ? static_cast<float*>(workspace) : nullptr;
  p.B = batch, p.T = seq_len, p.C = (int)channels, p.act = activation;
  return launched(ttt::launch_conv(dtype, p, taps, width, true, static_cast<cudaStream_t>(stream)), "causal convolution backward");
}

namespace {

int check_norm(int64_t B, int64_t T, int64_t C, int G, int over, int dtype, int activation, float eps) {
  const int rc = check_sizes(B, T, C, dtype);
  if (rc != TTT_OK) return rc;
  if (G <= 0 || C % G != 0) return fail(TTT_ERR_SHAPE, "channels=%lld are not a multiple of groups=%d", (long long)C, G);
  if (over != TTT_OVER_TOKEN && over != TTT_OVER_SEQUENCE) return fail(TTT_ERR_UNSUPPORTED, "over=%d (0: tokens, 1: sequences)", over);
  if (over == TTT_OVER_TOKEN && C / G > ttt::NORM_TOKEN_CHANNELS)
    return fail(TTT_ERR_UNSUPPORTED, "groups of up to %d channels are normed token by token (got %lld)", ttt::NORM_TOKEN_CHANNELS, (long long)(C / G));
  if (activation < ttt::ACT_NONE || activation > ttt::ACT_GELU)
    return fail(TTT_ERR_UNSUPPORTED, "unknown activation %d (0: none, 1: SiLU, 2: GELU)", activation);
  if (!(eps >= 0.f)) return fail(TTT_ERR_SHAPE, "epsilon must be >= 0");
  if (over == TTT_OVER_SEQUENCE && B * C >= (int64_t)1 << 34) return fail(TTT_ERR_SHAPE, "batch*channels must be below 2^34");
  return TTT_OK;
}
void norm_dims(ttt::NormParams* p, int64_t B, int64_t T, int64_t C, int G, int activation, float eps) {
  p->B = B, p->T = T, p->tokens = B * T, p->C = (int)C, p->G = G, p->c = (int)(C / G), p->act = activation, p->eps = eps;
  p->inv_c = 1.f / (float)p->c;
}
int norm_width(uintptr_t low, int c, int es) {
  if (low % 16 == 0 && c % (16 / es) == 0) return 16 / es;
  return low % (2 * es) == 0 && c % 2 == 0 ? 2 : 1;
}

}  // namespace

extern "C" size_t ttt_layer_group_norm_workspace_bytes(int64_t batch, int64_t seq_len, int64_t channels, int groups, int over, int dtype) {
  if (check_norm(batch, seq_len, channels, groups, over, dtype, 0, 0.f) != TTT_OK) return 0;
  return sizeof(float) * ttt::norm_forward_floats(batch, seq_len, (int)channels, groups, over == TTT_OVER_SEQUENCE, dtype == TTT_BF16 ? 2 : 4);
}
extern "C" size_t ttt_layer_group_norm_backward_workspace_bytes(int64_t batch, int64_t seq_len, int64_t channels, int groups, int over, int dtype) {
  if (check_norm(batch, seq_len, channels, groups, over, dtype, 0, 0.f) != TTT_OK) return 0;
  return sizeof(float) * ttt::norm_backward_floats(batch, seq_len, (int)channels, groups, over == TTT_OVER_SEQUENCE, dtype == TTT_BF16 ? 2 : 4);
}

extern "C" int ttt_layer_group_norm(int64_t batch, int64_t seq_len, int64_t channels, int groups, int over, int dtype, int activation,
                                    float epsilon, const void* x, const void* gate, const int64_t* strides, const void* weight,
                                    const void* bias, void* y, float* stats, void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check_norm(batch, seq_len, channels, groups, over, dtype, activation, epsilon);
  if (rc != TTT_OK) return rc;
  ttt::NormParams p{};
  norm_dims(&p, batch, seq_len, channels, groups, activation, epsilon);
  const int es = dtype == TTT_BF16 ? 2 : 4;
  Spans s{batch, seq_len, channels, es};
  s.rows("x", x, strides, 0, p.xs);
  s.rows("gate", gate, strides, 1, p.gates, true);
  s.need("y", y);
  s.align("weight", weight);
  s.align("bias", bias);
  if (s.rc != TTT_OK) return s.rc;
  if ((reinterpret_cast<uintptr_t>(stats) & 3u) != 0) return fail(TTT_ERR_ALIGN, "stats is not aligned to its elements");
  const size_t need = ttt_layer_group_norm_workspace_bytes(batch, seq_len, channels, groups, over, dtype);
  if ((rc = check_bytes(workspace_bytes, need, workspace, "workspace")) != TTT_OK) return rc;
  const bool sequence = over == TTT_OVER_SEQUENCE;
  const int64_t n = batch * seq_len * channels * es, wide = channels * es;
  if ((rc = check_apart({{"y", y, n, 1}, {"stats", sequence ? stats : nullptr, batch * groups * 8, 0},
                         {"workspace", need != 0 ? workspace : nullptr, (int64_t)need, 0}},
                        {{"x", x, s.bytes(p.xs), s.contiguous(p.xs)}, {"gate", gate, s.bytes(p.gates), s.contiguous(p.gates)},
                         {"weight", weight, wide, 0}, {"bias", bias, wide, 0}})) != TTT_OK)
    return rc;
  p.x = x, p.gate = gate, p.w = weight, p.bias = bias, p.y = y, p.stats = stats, p.moments = static_cast<float*>(workspace);
  return launched(ttt::launch_norm(dtype, p, norm_width(s.low, p.c, es), sequence, false, static_cast<cudaStream_t>(stream)),
                  "group norm");
}

extern "C" int ttt_layer_group_norm_backward(int64_t batch, int64_t seq_len, int64_t channels, int groups, int over, int dtype,
                                             int activation, float epsilon, const void* x, const void* gate, const void* grad_y,
                                             const int64_t* strides, const void* weight, const void* bias, const float* stats,
                                             void* grad_x, void* grad_gate, void* grad_weight, void* grad_bias, void* workspace,
                                             size_t workspace_bytes, void* stream) {
  int rc = check_norm(batch, seq_len, channels, groups, over, dtype, activation, epsilon);
  if (rc != TTT_OK) return rc;
  ttt::NormParams p{};
  norm_dims(&p, batch, seq_len, channels, groups, activation, epsilon);
  const int es = dtype == TTT_BF16 ? 2 : 4;
  const bool sequence = over == TTT_OVER_SEQUENCE;
  Spans s{batch, seq_len, channels, es};
  s.rows("x", x, strides, 0, p.xs);
  s.rows("gate", gate, strides, 1, p.gates, true);
  s.rows("grad_y", grad_y, strides, 2, p.gys);
  s.need("grad_x", grad_x);
  if (gate != nullptr) s.need("grad_gate", grad_gate);
  s.align("weight", weight);
  s.align("bias", bias);
  const int width = norm_width(s.low, p.c, es);
  s.align("grad_weight", grad_weight);
  s.align("grad_bias", grad_bias);
  if (s.rc != TTT_OK) return s.rc;
  if (sequence && stats == nullptr) return fail(TTT_ERR_NULL, "stats is null");
  if ((reinterpret_cast<uintptr_t>(stats) & 3u) != 0) return fail(TTT_ERR_ALIGN, "stats is not aligned to its elements");
  const size_t need = sequence || grad_weight != nullptr || grad_bias != nullptr
                          ? ttt_layer_group_norm_backward_workspace_bytes(batch, seq_len, channels, groups, over, dtype)
                          : 0;
  if ((rc = check_bytes(workspace_bytes, need, workspace, "workspace")) != TTT_OK) return rc;
  const int64_t n = batch * seq_len * channels * es, wide = channels * es;
  if ((rc = check_apart({{"grad_x", grad_x, n, 1}, {"grad_gate", gate != nullptr ? grad_gate : nullptr, n, 1}, {"grad_weight", grad_weight, wide, 2},
                         {"grad_bias", grad_bias, wide, 4}, {"workspace", need != 0 ? workspace : nullptr, (int64_t)need, 0}},
                        {{"x", x, s.bytes(p.xs), s.contiguous(p.xs)}, {"gate", gate, s.bytes(p.gates), s.contiguous(p.gates)},
                         {"grad_y", grad_y, s.bytes(p.gys), s.contiguous(p.gys)}, {"weight", weight, wide, 2}, {"bias", bias, wide, 4},
                         {"stats", sequence ? stats : nullptr, batch * groups * 8, 0}})) != TTT_OK)
    return rc;
  p.x = x, p.gate = gate, p.gy = grad_y, p.w = weight, p.bias = bias, p.stats = const_cast<float*>(stats);
  p.gx = grad_x, p.ggate = grad_gate, p.gw = grad_weight, p.gb = grad_bias;
  p.partials = need != 0 ? static_cast<float*>(workspace) : nullptr;
  return launched(ttt::launch_norm(dtype, p, width, sequence, true, static_cast<cudaStream_t>(stream)), "group norm backward");
}

namespace {

struct SelDims {
  int64_t B, T, C;
  int G, N, dtype;
  int NP, es;
  int64_t tiles;
  ttt::SelCut cut(bool backward) const { return ttt::sel_cut(B, T, (int)C, G, N, backward); }
};
int sel_dims(SelDims* d, int64_t B, int64_t T, int64_t C, int G, int N, int dtype) {
  const int rc = check_sizes(B, T, C, dtype);
  if (rc != TTT_OK) return rc;
  if (G <= 0 || C % G != 0) return fail(TTT_ERR_SHAPE, "channels=%lld are not a multiple of groups=%d", (long long)C, G);
  if (N < 1 || N > ttt::SEL_STATES) return fail(TTT_ERR_UNSUPPORTED, "Unsupported states=%d (supported: 1..%d)", N, ttt::SEL_STATES);
  if (B * C >= (int64_t)1 << 31) return fail(TTT_ERR_SHAPE, "batch*channels must be below 2^31");
  if (B * T * G >= (int64_t)1 << 32) return fail(TTT_ERR_SHAPE, "batch*seq_len*groups must be below 2^32");
  d->B = B, d->T = T, d->C = C, d->G = G, d->N = N, d->dtype = dtype;
  d->NP = ttt::sel_padded(N);
  d->es = dtype == TTT_BF16 ? 2 : 4;
  d->tiles = (T + ttt::SEL_TILE - 1) / ttt::SEL_TILE;
  return TTT_OK;
}
int64_t up4(int64_t n) { return (n + 3) & ~(int64_t)3; }
// floats of a cut's segment states (and the first one's start) and sums
int64_t seg_floats(const SelDims& d, const ttt::SelCut& k) {
  return k.nseg == 1 ? 0 : d.B * (k.nseg + 1) * d.C * d.NP + up4(d.B * k.nseg * d.C);
}
int64_t saved_floats(const SelDims& d) { return d.B * d.tiles * d.C * d.NP; }
int64_t backward_floats(const SelDims& d, const ttt::SelCut& k) {
  const int64_t rows = d.B * k.nseg;
  return d.B * d.G * k.channel_blocks * d.T * 2 * d.NP + rows * d.C * d.NP + up4(rows * 2 * d.C) + seg_floats(d, k);
}
void set_segments(ttt::SelParams* p, const SelDims& d, const ttt::SelCut& k, float* at) {
  p->nseg = k.nseg, p->seg_tiles = k.seg_tiles;
  if (k.nseg > 1) p->seg_state = at, p->seg_sum = at + d.B * (k.nseg + 1) * d.C * d.NP;
}

// The tensors that both directions read.  strides: batch and token of x, dt, z and (backward) grad_y, then batch, token and group of b, c.
int sel_inputs(ttt::SelParams* p, const SelDims& d, const void* x, const void* dt, const float* a, const void* b, const void* c, const float* skip,
               const void* z, const float* bias, const float* state, const void* starts, const void* gy, bool backward, const int64_t* strides,
               const void* y, const void* gx, const void* gdt, const void* gz) {
  Spans s{d.B, d.T, d.C, d.es};
  s.rows("x", x, strides, 0, p->xs);
  s.rows("dt", dt, strides, 1, p->ds);
  s.rows("z", z, strides, 2, p->zs, true);
  if (backward) {
    s.rows("grad_y", gy, strides, 3, p->gs);
    s.need("grad_x", gx);
    s.need("grad_dt", gdt);
    if (z != nullptr) s.need("grad_z", gz);
  } else {
    s.need("y", y);
  }
  const int64_t each = d.C / d.G * d.es;
  p->xg = s.low % 16 == 0 && each % 16 == 0 ? 16 : s.low % 4 == 0 && each % 4 == 0 ? 4 : d.es;
  Spans m{d.B, d.T, (int64_t)d.G * d.N, d.es};
  const int64_t* at = strides != nullptr ? strides + (backward ? 8 : 6) : nullptr;
  const void* bases[2] = {b, c};
  int64_t(*out[2])[3] = {&p->bs, &p->cs};
  const char* names[2] = {"b", "c"};
  for (int k = 0; k < 2; ++k) {
    const int64_t two[2] = {at != nullptr ? at[3 * k] : d.T * d.G * d.N, at != nullptr ? at[3 * k + 1] : (int64_t)d.G * d.N};
    int64_t rows[2];
    m.rows(names[k], bases[k], two, 0, rows);
    const int64_t group = d.G == 1 ? 0 : at != nullptr ? at[3 * k + 2] : d.N;
    m.low |= (uintptr_t)(group * d.es);
    if (m.rc == TTT_OK && (group < 0 || group > kFarthest / d.G)) m.rc = fail(TTT_ERR_SHAPE, "the strides of %s are out of range", names[k]);
    (*out[k])[0] = rows[0], (*out[k])[1] = rows[1], (*out[k])[2] = group;
  }
  const int64_t wide = (int64_t)d.N * d.es;
  p->bg = m.low % 16 == 0 && wide % 16 == 0 ? 16 : m.low % 4 == 0 && wide % 4 == 0 ? 4 : d.es;
  if (s.rc != TTT_OK) return s.rc;
  if (m.rc != TTT_OK) return m.rc;
  const struct {
    const char* name;
    const void* p;
    unsigned align;
    bool needed;
  } plain[] = {{"a", a, 16, true}, {"d", skip, 4, false}, {"dt_bias", bias, 4, false}, {"state", state, 16, false}};
  for (const auto& q : plain) {
    if (q.needed && q.p == nullptr) return fail(TTT_ERR_NULL, "%s is null", q.name);
    if (reinterpret_cast<uintptr_t>(q.p) % q.align != 0) return fail(TTT_ERR_ALIGN, "%s is not %u-byte aligned", q.name, q.align);
  }
  p->x = x, p->dt = dt, p->z = z, p->b = b, p->c = c, p->A = a, p->D = skip, p->bias = bias, p->state = state;
  p->starts = static_cast<const uint8_t*>(starts);
  p->B = d.B, p->T = d.T, p->C = (int)d.C, p->G = d.G, p->N = d.N;
  return TTT_OK;
}
// bytes that b or c spans
int64_t states_bytes(const SelDims& d, const int64_t (&s)[3]) { return ((d.B - 1) * s[0] + (d.T - 1) * s[1] + (d.G - 1) * s[2] + d.N) * d.es; }
bool states_contiguous(const SelDims& d, const int64_t (&s)[3]) {
  return (d.B == 1 || s[0] == d.T * d.G * d.N) && (d.T == 1 || s[1] == (int64_t)d.G * d.N) && (d.G == 1 || s[2] == d.N);
}
int need16(const char* name, const void* p, bool optional) {
  if (p == nullptr && !optional) return fail(TTT_ERR_NULL, "%s is null", name);
  if ((reinterpret_cast<uintptr_t>(p) & 15u) != 0) return fail(TTT_ERR_ALIGN, "%s is not 16-byte aligned", name);
  return TTT_OK;
}

}  // namespace

extern "C" size_t ttt_linear_selective_saved_bytes(int64_t batch, int64_t seq_len, int64_t channels, int groups, int states, int dtype) {
  SelDims d;
  return sel_dims(&d, batch, seq_len, channels, groups, states, dtype) == TTT_OK ? sizeof(float) * saved_floats(d) : 0;
}
extern "C" size_t ttt_linear_selective_forward_workspace_bytes(int64_t batch, int64_t seq_len, int64_t channels, int groups, int states,
                                                               int dtype) {
  SelDims d;
  return sel_dims(&d, batch, seq_len, channels, groups, states, dtype) == TTT_OK ? sizeof(float) * seg_floats(d, d.cut(false)) : 0;
}
extern "C" size_t ttt_linear_selective_backward_workspace_bytes(int64_t batch, int64_t seq_len, int64_t channels, int groups, int states,
                                                                int dtype) {
  SelDims d;
  return sel_dims(&d, batch, seq_len, channels, groups, states, dtype) == TTT_OK ? sizeof(float) * backward_floats(d, d.cut(true)) : 0;
}

extern "C" int ttt_linear_selective_forward(int64_t batch, int64_t seq_len, int64_t channels, int groups, int states, int dtype, int softplus,
                                            const void* x, const void* dt, const float* a, const void* b, const void* c, const float* d_skip,
                                            const void* z, const float* dt_bias, const float* state, const void* starts,
                                            const int64_t* strides, void* y, float* state_out, void* saved, size_t saved_bytes,
                                            void* workspace, size_t workspace_bytes, void* stream) {
  SelDims d;
  ttt::SelParams p{};
  int rc = sel_dims(&d, batch, seq_len, channels, groups, states, dtype);
  if (rc != TTT_OK ||
      (rc = sel_inputs(&p, d, x, dt, a, b, c, d_skip, z, dt_bias, state, starts, nullptr, false, strides, y, nullptr, nullptr, nullptr)) != TTT_OK ||
      (rc = need16("state_out", state_out, false)) != TTT_OK)
    return rc;
  p.softplus = softplus != 0;
  p.y = y, p.state_out = state_out;
  const bool step = saved == nullptr && seq_len <= 16;
  const ttt::SelCut cut = d.cut(false);
  const int64_t need = step ? 0 : 4 * seg_floats(d, cut);
  if (saved != nullptr && (rc = check_bytes(saved_bytes, sizeof(float) * saved_floats(d), saved, "saved")) != TTT_OK) return rc;
  if ((rc = check_bytes(workspace_bytes, need, workspace, "workspace")) != TTT_OK) return rc;
  const Spans s{d.B, d.T, d.C, d.es};
  const int64_t held = d.B * d.C * d.N * 4;
  if ((rc = check_apart({{"state_out", state_out, held, 1}, {"y", y, d.B * d.T * d.C * d.es, 0}, {"saved", saved, 4 * saved_floats(d), 0},
                         {"workspace", need != 0 ? workspace : nullptr, need, 0}},
                        {{"x", x, s.bytes(p.xs), 0}, {"dt", dt, s.bytes(p.ds), 0}, {"z", z, s.bytes(p.zs), 0}, {"a", a, d.C * d.N * 4, 0},
                         {"b", b, states_bytes(d, p.bs), 0}, {"c", c, states_bytes(d, p.cs), 0}, {"d", d_skip, d.C * 4, 0},
                         {"dt_bias", dt_bias, d.C * 4, 0}, {"state", state, held, 1}, {"starts", starts, d.B * d.T, 0}})) != TTT_OK)
    return rc;
  if (step) return launched(ttt::launch_selective_step(dtype, p, static_cast<cudaStream_t>(stream)), "selective step");
  p.saved = static_cast<float*>(saved);
  set_segments(&p, d, cut, static_cast<float*>(workspace));
  return launched(ttt::launch_selective(dtype, p, static_cast<cudaStream_t>(stream)), "selective scan");
}

extern "C" int ttt_linear_selective_backward(int64_t batch, int64_t seq_len, int64_t channels, int groups, int states, int dtype, int softplus,
                                             const void* x, const void* dt, const float* a, const void* b, const void* c, const float* d_skip,
                                             const void* z, const float* dt_bias, const void* starts, const void* grad_y,
                                             const int64_t* strides, const void* saved, size_t saved_bytes, const float* grad_state_out,
                                             void* grad_x, void* grad_dt, float* grad_a, void* grad_b, void* grad_c, float* grad_d,
                                             void* grad_z, float* grad_dt_bias, float* grad_state, void* workspace, size_t workspace_bytes,
                                             void* stream) {
  SelDims d;
  ttt::SelParams p{};
  int rc = sel_dims(&d, batch, seq_len, channels, groups, states, dtype);
  if (rc != TTT_OK || (rc = sel_inputs(&p, d, x, dt, a, b, c, d_skip, z, dt_bias, nullptr, starts, grad_y, true, strides, nullptr, grad_x, grad_dt,
                                       grad_z)) != TTT_OK)
    return rc;
  if (saved == nullptr) return fail(TTT_ERR_NULL, "saved is null");
  if ((rc = check_bytes(saved_bytes, sizeof(float) * saved_floats(d), saved, "saved")) != TTT_OK ||
      (rc = need16("grad_state_out", grad_state_out, true)) != TTT_OK || (rc = need16("grad_a", grad_a, false)) != TTT_OK ||
      (rc = need16("grad_state", grad_state, true)) != TTT_OK)
    return rc;
  const struct {
    const char* name;
    const void* p;
    unsigned align;
    bool needed;
  } plain[] = {{"grad_b", grad_b, (unsigned)d.es, true}, {"grad_c", grad_c, (unsigned)d.es, true}, {"grad_d", grad_d, 4, false}, {"grad_dt_bias", grad_dt_bias, 4, false}};
  for (const auto& q : plain) {
    if (q.needed && q.p == nullptr) return fail(TTT_ERR_NULL, "%s is null", q.name);
    if (reinterpret_cast<uintptr_t>(q.p) % q.align != 0) return fail(TTT_ERR_ALIGN, "%s is not aligned to its elements", q.name);
  }
  const ttt::SelCut cut = d.cut(true);
  const int64_t need = 4 * backward_floats(d, cut);
  if ((rc = check_bytes(workspace_bytes, need, workspace, "workspace")) != TTT_OK) return rc;
  const Spans s{d.B, d.T, d.C, d.es};
  const int64_t n = d.B * d.T * d.C * d.es, held = d.B * d.C * d.N * 4, bc = d.B * d.T * d.G * d.N * d.es, wide = d.C * 4, rates = wide * d.N;
  if ((rc = check_apart({{"grad_x", grad_x, n, 1}, {"grad_dt", grad_dt, n, 1}, {"grad_z", z != nullptr ? grad_z : nullptr, n, 1}, {"grad_a", grad_a, rates, 2},
                         {"grad_b", grad_b, bc, 4}, {"grad_c", grad_c, bc, 4}, {"grad_d", grad_d, wide, 8}, {"grad_dt_bias", grad_dt_bias, wide, 16},
                         {"grad_state", grad_state, held, 0}, {"workspace", workspace, need, 0}},
                        {{"x", x, s.bytes(p.xs), s.contiguous(p.xs)}, {"dt", dt, s.bytes(p.ds), s.contiguous(p.ds)},
                         {"z", z, s.bytes(p.zs), s.contiguous(p.zs)}, {"grad_y", grad_y, s.bytes(p.gs), s.contiguous(p.gs)}, {"a", a, rates, 2},
                         {"b", b, states_bytes(d, p.bs), states_contiguous(d, p.bs) ? 4u : 0u},
                         {"c", c, states_bytes(d, p.cs), states_contiguous(d, p.cs) ? 4u : 0u}, {"d", d_skip, wide, 8},
                         {"dt_bias", dt_bias, wide, 16}, {"starts", starts, d.B * d.T, 0}, {"saved", saved, 4 * saved_floats(d), 0},
                         {"grad_state_out", grad_state_out, held, 0}})) != TTT_OK)
    return rc;
  float* ws = static_cast<float*>(workspace);
  const int64_t rows = d.B * cut.nseg;
  p.part_bc = ws, ws += d.B * d.G * cut.channel_blocks * d.T * 2 * d.NP;
  p.part_a = ws, ws += rows * d.C * d.NP;
  p.part_d = ws, ws += up4(rows * 2 * d.C);
  set_segments(&p, d, cut, ws);
  p.softplus = softplus != 0;
  p.saved = static_cast<float*>(const_cast<void*>(saved));
  p.gy = grad_y, p.gstate_out = grad_state_out, p.gx = grad_x, p.gdt = grad_dt, p.gz = grad_z, p.ga = grad_a, p.gb = grad_b, p.gc = grad_c;
  p.gd = grad_d, p.gbias = grad_dt_bias, p.gstate = grad_state;
  return launched(ttt::launch_selective_bwd(dtype, p, static_cast<cudaStream_t>(stream)), "selective scan backward");
}
