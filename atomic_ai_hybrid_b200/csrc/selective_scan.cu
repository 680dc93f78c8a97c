// Mamba2's short causal convolution and selective scan with state carried between calls (prompts of
// any length and single tokens), for serving (the layer's mathematics: reference `model.py:391-525`).
//
//   xc_t = sanitize(silu(sum_j w_j x_{t-3+j} + b)),  dt_t = clamp(softplus(dtraw_t), dt_min, dt_max)
//   S_t[c,:] = e^{max(dt_t A_h, -20)} S_{t-1}[c,:] + dt_t xc_t B_t ,   y_t[c] = <C_t, S_t[c,:]>
#include "launchers.h"
#include "mma.cuh"
#include "packed.cuh"
#include "recurrent.cuh"
#include <algorithm>

namespace {
using namespace ahb;

struct ScanArgs {
  const void *x, *dt, *Bm, *Cm, *conv_w;
  int64_t xs, dts, bs, cs;  // row strides in elements
  const float *A, *conv_b;
  void* conv_state;
  float* state;
  const int *cu, *slots;
  void* y;
  int B, L, T, C, P, S;
  float dt_min, dt_max;
};

constexpr float kClip = 1e3f, kMinDA = -20.f;

AHB_DEVICE float dt_of(float raw, float lo, float hi) {
  return raw != raw ? 0.f : fminf(fmaxf(softplusf_(raw), lo), hi);
}

// Sums v[0..R) over the warp; lane l gets the sum number `sum_index<R>(l)`: every step adds half of the values'
// halves across lanes, so R sums take R - 1 + 5 - log2 R shuffles.
template <int R>
AHB_DEVICE float warp_sums(float (&v)[R]) {
  const int lane = threadIdx.x & 31;
  int w = 16;
#pragma unroll
  for (int r = R / 2; r >= 1; r /= 2, w /= 2) {
    const bool hi = lane & w;
#pragma unroll
    for (int i = 0; i < r; ++i) {
      const float give = hi ? v[i] : v[i + r], keep = hi ? v[i + r] : v[i];
      v[i] = keep + __shfl_xor_sync(0xffffffffu, give, w);
    }
  }
#pragma unroll
  for (; w >= 1; w /= 2) v[0] += __shfl_xor_sync(0xffffffffu, v[0], w);
  return v[0];
}
template <int R>
AHB_DEVICE int sum_index(int lane) {
  int at = 0, w = 16;
#pragma unroll
  for (int r = R / 2; r >= 1; r /= 2, w /= 2) at += lane & w ? r : 0;
  return at;
}

// ---------------------------------------------------------------- a few tokens per sequence, or fp32
// Bound by the chain from token to token: 0.5 us each (2048 channels, 64 tokens in bf16 or 1024 in fp32; 0.7 us in 8192,
// whose rows come from HBM), the state read and written once a call.
// One warp carries CH channels of one sequence through its tokens: lane l holds states
// [l V, l V + V) of each channel in registers (N = 32 V), lanes 0..CH-1 also hold the convolution
// window of one channel and turn its row into (decay, dt xc).
template <typename T, typename W, int N, int CH, int WARPS>
__global__ void __launch_bounds__(WARPS * 32) scan_token_kernel(ScanArgs p) {
  constexpr int V = N / 32;
  const int lane = threadIdx.x & 31, b = blockIdx.y;
  if (blockIdx.x * WARPS * CH >= p.C) {  // beside the channels, in calls with offsets
    const OpenRows open(p.cu, p.B, p.T);
    for (int i = b; i < open.count; i += p.B)
      for (int c = threadIdx.x; c < p.C; c += WARPS * 32) static_cast<T*>(p.y)[(int64_t)open.row(i) * p.C + c] = from_f<T>(0.f);
    return;
  }
  const int c0 = (blockIdx.x * WARPS + (threadIdx.x >> 5)) * CH;
  if (c0 >= p.C) return;
  const SeqRange r = seq_range(p.cu, b, p.L, p.T);
  const int slot = seq_slot(p.slots, b, p.S);
  const int c = c0 + lane;
  const bool mine = lane < CH && c < p.C;
  T* y = static_cast<T*>(p.y);
  if (slot < 0) {
    for (int t = r.start; t < r.end; ++t)
      if (mine) y[(int64_t)t * p.C + c] = from_f<T>(0.f);
    return;
  }
  if (r.start == r.end) return;

  float h[CH][V];
  float* S0 = p.state + ((int64_t)slot * p.C + c0) * N + lane * V;
#pragma unroll
  for (int j = 0; j < CH; ++j)
#pragma unroll
    for (int i = 0; i < V; ++i) h[j][i] = c0 + j < p.C ? S0[j * N + i] : 0.f;

  float w[4] = {0.f, 0.f, 0.f, 0.f}, bias = 0.f, A = 0.f, x0 = 0.f, x1 = 0.f, x2 = 0.f;
  T* win = static_cast<T*>(p.conv_state) + (int64_t)slot * 3 * p.C + c;
  if (mine) {
    load_taps(w, static_cast<const W*>(p.conv_w) + (int64_t)c * 4);
    bias = p.conv_b ? p.conv_b[c] : 0.f;
    A = p.A[c / p.P];
    x0 = to_f(win[0]);
    x1 = to_f(win[p.C]);
    x2 = to_f(win[2 * p.C]);
  }
  const T* Bm = static_cast<const T*>(p.Bm);
  const T* Cm = static_cast<const T*>(p.Cm);
  // a token's values are loaded while the one before is worked on
  T xn, dn, Bn[V], Cn[V];
  auto fetch = [&](int t) {
    if (mine) {
      xn = static_cast<const T*>(p.x)[(int64_t)t * p.xs + c];
      dn = static_cast<const T*>(p.dt)[(int64_t)t * p.dts + c];
    }
#pragma unroll
    for (int i = 0; i < V; ++i) {
      Bn[i] = Bm[(int64_t)t * p.bs + lane * V + i];
      Cn[i] = Cm[(int64_t)t * p.cs + lane * V + i];
    }
  };
  fetch(r.start);
  for (int t = r.start; t < r.end; ++t) {
    float a = 0.f, u = 0.f;
    if (mine) {
      const float x3 = to_f(xn), dt = dt_of(to_f(dn), p.dt_min, p.dt_max);
      a = exp_decay(fmaxf(dt * A, kMinDA));
      u = dt * sanitize(conv_silu(w, bias, x0, x1, x2, x3), kClip);
      x0 = x1;
      x1 = x2;
      x2 = x3;
    }
    float Bv[V], Cv[V], sum[CH];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      Bv[i] = sanitize(to_f(Bn[i]), kClip);
      Cv[i] = sanitize(to_f(Cn[i]), kClip);
    }
    if (t + 1 < r.end) fetch(t + 1);
#pragma unroll
    for (int j = 0; j < CH; ++j) {
      const float aj = __shfl_sync(0xffffffffu, a, j), uj = __shfl_sync(0xffffffffu, u, j);
      sum[j] = 0.f;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        h[j][i] = fmaf(aj, h[j][i], uj * Bv[i]);
        sum[j] = fmaf(Cv[i], h[j][i], sum[j]);
      }
    }
    const float out = warp_sums<CH>(sum);
    const int at = c0 + sum_index<CH>(lane);
    if (lane % (32 / CH) == 0 && at < p.C) y[(int64_t)t * p.C + at] = from_f<T>(out);
  }
#pragma unroll
  for (int j = 0; j < CH; ++j)
    if (c0 + j < p.C) {
#pragma unroll
      for (int i = 0; i < V; ++i) S0[j * N + i] = h[j][i];
    }
  if (mine) {
    win[0] = from_f<T>(x0);
    win[p.C] = from_f<T>(x1);
    win[2 * p.C] = from_f<T>(x2);
  }
}

// ---------------------------------------------------------------- one token per sequence
// Bound by the state's bytes, read once and written once.  A warp takes G groups of R channels of one
// sequence; the next group's rows are on their way while one is worked on.  Lane c of the first R G turns
// channel c's row into (decay, dt xc).  64 sequences of 2048 channels and 128 states: 25 us, 0.84 of the copy
// rate (33 us with 8 channels a warp); 200 of 1536 in fp32: 56 us, 0.88; one sequence: 2.9 us.

template <int V> struct Floats;
template <> struct Floats<4> { using type = float4; };
template <> struct Floats<2> { using type = float2; };
template <> struct Floats<1> { using type = float; };

template <int V>
AHB_DEVICE void load_states(float (&h)[V], const float* p) {
  const auto r = __ldcs(reinterpret_cast<const typename Floats<V>::type*>(p));
#pragma unroll
  for (int i = 0; i < V; ++i) h[i] = reinterpret_cast<const float*>(&r)[i];
}
template <int V>
AHB_DEVICE void store_states(float* p, const float (&h)[V]) {
  typename Floats<V>::type r;
#pragma unroll
  for (int i = 0; i < V; ++i) reinterpret_cast<float*>(&r)[i] = h[i];
  __stcs(reinterpret_cast<typename Floats<V>::type*>(p), r);
}

template <typename T, typename W, int N, int R, int G>
__global__ void __launch_bounds__(128) scan_step_kernel(ScanArgs p) {
  constexpr int V = N / 32;
  const int lane = threadIdx.x & 31, b = blockIdx.y;
  const int c0 = (blockIdx.x * 4 + (threadIdx.x >> 5)) * R * G;
  if (c0 >= p.C) return;
  const int slot = seq_slot(p.slots, b, p.S), c = c0 + lane;
  const bool mine = lane < R * G && c < p.C;
  T* y = static_cast<T*>(p.y) + (int64_t)b * p.C;
  if (slot < 0) {
    if (mine) y[c] = from_f<T>(0.f);
    return;
  }
  float* S0 = p.state + ((int64_t)slot * p.C + c0) * N + lane * V;
  float h[2][R][V];
  auto fetch = [&](int k) {
#pragma unroll
    for (int j = 0; j < R; ++j)
      if (c0 + k * R + j < p.C) load_states<V>(h[k & 1][j], S0 + (k * R + j) * N);
  };
  fetch(0);
  float a = 0.f, u = 0.f;
  if (mine) {
    T* win = static_cast<T*>(p.conv_state) + (int64_t)slot * 3 * p.C + c;
    float w[4];
    load_taps(w, static_cast<const W*>(p.conv_w) + (int64_t)c * 4);
    const float bias = p.conv_b ? p.conv_b[c] : 0.f, A = p.A[c / p.P];
    const float x0 = to_f(win[0]), x1 = to_f(win[p.C]), x2 = to_f(win[2 * p.C]);
    const T x = static_cast<const T*>(p.x)[(int64_t)b * p.xs + c];
    const float dt = dt_of(to_f(static_cast<const T*>(p.dt)[(int64_t)b * p.dts + c]), p.dt_min, p.dt_max);
    a = exp_decay(fmaxf(dt * A, kMinDA));
    u = dt * sanitize(conv_silu(w, bias, x0, x1, x2, to_f(x)), kClip);
    win[0] = from_f<T>(x1);
    win[p.C] = from_f<T>(x2);
    win[2 * p.C] = x;
  }
  float Bv[V], Cv[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    Bv[i] = sanitize(to_f(static_cast<const T*>(p.Bm)[(int64_t)b * p.bs + lane * V + i]), kClip);
    Cv[i] = sanitize(to_f(static_cast<const T*>(p.Cm)[(int64_t)b * p.cs + lane * V + i]), kClip);
  }
#pragma unroll
  for (int k = 0; k < G; ++k) {
    if (k + 1 < G) fetch(k + 1);
    float sum[R];
#pragma unroll
    for (int j = 0; j < R; ++j) {
      const float aj = __shfl_sync(0xffffffffu, a, k * R + j), uj = __shfl_sync(0xffffffffu, u, k * R + j);
      sum[j] = 0.f;
      if (c0 + k * R + j < p.C) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          h[k & 1][j][i] = fmaf(aj, h[k & 1][j][i], uj * Bv[i]);
          sum[j] = fmaf(Cv[i], h[k & 1][j][i], sum[j]);
        }
        store_states<V>(S0 + (k * R + j) * N, h[k & 1][j]);
      }
    }
    const float out = warp_sums<R>(sum);
    const int at = c0 + k * R + sum_index<R>(lane);
    if (lane % (32 / R) == 0 && at < p.C) y[at] = from_f<T>(out);
  }
}

template <typename T, typename W, int N, int R, int G>
void launch_step(const ScanArgs& p, cudaStream_t st) {
  const dim3 grid((p.C + 4 * R * G - 1) / (4 * R * G), p.B);
  scan_step_kernel<T, W, N, R, G><<<grid, 128, 0, st>>>(p);
}

template <typename T, typename W, int N>
void launch_token(const ScanArgs& p, cudaStream_t st) {
  if (p.cu == nullptr && p.L == 1) {
    // 32 channels a warp use every lane and keep two groups of rows on their way; where that leaves an SM
    // fewer than 8 warps, 8 channels a warp spread the loads
    if ((int64_t)p.B * p.C < 32 * 8 * 148) launch_step<T, W, N, 8, 1>(p, st);
    else launch_step<T, W, N, 1024 / N, N / 32>(p, st);
    return;
  }
  constexpr int CH = 8, WARPS = 4;
  const dim3 grid((p.C + CH * WARPS - 1) / (CH * WARPS) + (p.cu != nullptr), p.B);
  scan_token_kernel<T, W, N, CH, WARPS><<<grid, WARPS * 32, 0, st>>>(p);
}

// ---------------------------------------------------------------- prompt form (bf16)
// The recurrence of a block of 32 tokens as products over the block.  With c_t = sum_{r <= t} log2(e) dA_r
// from the block's start, m = c after 16 tokens and E_t = c_t - m per channel p,
//   Y[t,p]  = 2^{E_t} ( C_t . (2^m S) + sum_{s <= t} (C_t . B_s) V_s )       V_s = 2^{-E_s} u_s
//   S'      = 2^{E_end} ( 2^m S + sum_s V_s B_s )
// so one factor V serves the output and the state, and C B^T is shared by all channels.  The factors
// stay below 2^kSpan as long as neither half block decays by more: 2^76 times the largest u (2^10), C . B
// (2^27) and 32 terms is far from the floats' end.  Channels that decay faster (over 3.3 nats a token on
// average; none of 2.1 M channel-blocks at dt around 0.06 and A up to -16) take their block token by
// token.  Both sums run on m16n8k16 bf16 products with fp32 accumulators:
// two warps keep the fp32 state of 16 channels as accumulators (channels are rows), which the next
// block's C S product takes back as its left operand without leaving the registers.  B and C are bf16
// already; the fp32 factors go in as bf16 terms: V in three (24 bits, the state loses nothing), S and
// C B^T in two (2^-17, for outputs rounded to bf16).  Sums of exponents up to
// kSpan carry 2^-18 each: the state of a channel that loses 4 powers of two a token is good to about 3e-6, that of
// the usual ones (under 0.5) to 3e-7.  A form on tcgen05 with the state in TMEM as accumulator and as tf32 operand
// was built and measured: its 22 products of 128 x 32 a block take about 60 cycles each, four times their
// arithmetic (the left operand's read), and 128 channels a group meet the token-by-token case more
// often: 416 us in place of 559 for 8 prompts of 2048 x 4096 channels, but 200 for 215, 104 for 98 on
// ragged ones, and 32 for 12 on 16 tokens that decay fast; its outputs carry 2^-11 where these carry 2^-17.
//
// What all channels share, the clipped rows of B and C and C B^T, is made first (scan_rows_kernel; made by every
// block of channels instead it costs 10 %).  Long sequences are cut into segments of `seg` tokens: a launch
// finds every segment's state from zero and its decay, the next one hands the states on from segment to
// segment (scan_join_kernel), and the last one runs the segments from their true states with outputs.
//
// One prompt of 8192 tokens, 2048 channels, 128 states: 215 us (5.9 ms token by token, in fp32), 8 of 2048 tokens with
// 4096 channels: 559 us.  Neither HBM (8 %) nor the tensor pipe (38 %) is the end of it: 1.9 thousand
// instructions for 16 channels of a block issue 47 % of the time at the 16 warps that 128 registers leave.
struct PromptArgs {
  ScanArgs a;
  int seg;        // tokens per segment, a multiple of 32
  float* states;  // (segments, C, N): the segments' own end states, then their start states
  float* decays;  // (segments, C): log2 of a segment's decay
  __nv_bfloat16* rows;  // (blocks, BlockRows<N>): what all channels share of a block
};

constexpr float kSpan = 76.f, kLog2e = 1.4426950408889634f;

struct Segment {  // sequence, its first segment's number, its segments, which one, the blocks of 32 tokens before it
  int b, first, count, index, blocks;
  SeqRange seq;
};

AHB_DEVICE int offset_of(const ScanArgs& p, int b) { return min(max(__ldg(p.cu + b), 0), p.T); }

// Sequences b0 + lane of packed rows.  A sequence starts at the largest offset up to its own (`reach`: up to b0, then
// up to b0 + 32): where offsets fall it is empty, so all sequences together never have more than T tokens and their
// segments and blocks fit their places.
AHB_DEVICE SeqRange rising_ranges(const ScanArgs& p, int b0, int& reach) {
  const int lane = threadIdx.x & 31;
  int end = max(reach, b0 + lane < p.B ? offset_of(p, b0 + lane + 1) : 0);
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, end, o);
    if (lane >= o) end = max(end, v);
  }
  const int before = __shfl_up_sync(0xffffffffu, end, 1);
  const SeqRange r{lane == 0 ? reach : before, end};
  reach = __shfl_sync(0xffffffffu, end, 31);
  return r;
}
AHB_DEVICE SeqRange range_of_lane(SeqRange q, int lane) {
  return {__shfl_sync(0xffffffffu, q.start, lane), __shfl_sync(0xffffffffu, q.end, lane)};
}

// Segment number `id` over all sequences in order; b = -1 past the last.  Every warp looks by itself.
AHB_DEVICE Segment find_segment(const ScanArgs& p, int seg, int id) {
  Segment r{-1, 0, 0, 0, 0, {0, 0}};
  if (p.cu == nullptr) {
    const int n = (p.L + seg - 1) / seg;
    if (n > 0 && id < n * p.B) {
      r.b = id / n;
      r.first = r.b * n;
      r.count = n;
      r.index = id - r.first;
      r.blocks = r.b * ((p.L + 31) / 32);
      r.seq = seq_range(p.cu, r.b, p.L, p.T);
    }
    return r;
  }
  const int lane = threadIdx.x & 31;
  int base = 0, reach = offset_of(p, 0);
  for (int b0 = 0; b0 < p.B; b0 += 32) {
    const SeqRange q = rising_ranges(p, b0, reach);
    const int n = (q.end - q.start + seg - 1) / seg, blocks = (q.end - q.start + 31) / 32;
    int incl = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    const uint32_t hit = __ballot_sync(0xffffffffu, id < base + incl);
    if (hit) {
      const int src = __ffs(hit) - 1;
      r.b = b0 + src;
      r.count = __shfl_sync(0xffffffffu, n, src);
      r.first = base + __shfl_sync(0xffffffffu, incl, src) - r.count;
      r.index = id - r.first;
      r.blocks += __reduce_add_sync(0xffffffffu, lane < src ? blocks : 0);
      r.seq = range_of_lane(q, src);
      return r;
    }
    base += __shfl_sync(0xffffffffu, incl, 31);
    r.blocks += __reduce_add_sync(0xffffffffu, blocks);
  }
  return r;
}

// log(1 + e^x) to about 2^-22: max(x, 0) + log1p(z) with z = e^{-|x|}, log1p(z) = 2 atanh(z / (2 + z)) as
// its power series (the argument is at most 1/3; the first term left out is below 2e-7 of the sum)
AHB_DEVICE float2 softplus2(float2 x) {
  const float2 z = make_float2(ex2(-fabsf(x.x) * kLog2e), ex2(-fabsf(x.y) * kLog2e)), d = add2(z, both(2.f));
  const float2 s = mul2(z, make_float2(rcp(d.x), rcp(d.y))), w = mul2(s, s);
  float2 p = fma2(w, both(2.f / 11.f), both(2.f / 9.f));
  p = fma2(w, p, both(2.f / 7.f));
  p = fma2(w, p, both(2.f / 5.f));
  p = fma2(w, p, both(2.f / 3.f));
  p = fma2(w, p, both(2.f));
  return fma2(s, p, max2(x, 0.f));
}

AHB_DEVICE void ldsm4(uint32_t r[4], const void* p) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"((uint32_t)__cvta_generic_to_shared(p)) : "memory");
}
AHB_DEVICE void ldsm4_t(uint32_t r[4], const void* p) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"((uint32_t)__cvta_generic_to_shared(p)) : "memory");
}

// clip to +-1000 (exact in bf16), NaN to 0, on two bf16
AHB_DEVICE uint32_t clip2(uint32_t x) {
  const __nv_bfloat162 v = *reinterpret_cast<const __nv_bfloat162*>(&x);
  const __nv_bfloat162 c = __hmin2(__hmax2(v, __floats2bfloat162_rn(-kClip, -kClip)), __floats2bfloat162_rn(kClip, kClip));
  return __heq2_mask(v, v) & *reinterpret_cast<const uint32_t*>(&c);
}

AHB_DEVICE float lo16(uint32_t x) { return __uint_as_float(x << 16); }
AHB_DEVICE float hi16(uint32_t x) { return __uint_as_float(x & 0xffff0000u); }

AHB_DEVICE float2 both16(uint32_t x) { return make_float2(lo16(x), hi16(x)); }

// the next bf16 term of two floats, which keep what it leaves
AHB_DEVICE uint32_t term2(float2& v) {
  const uint32_t h = pack2(v.x, v.y);
  v.x -= lo16(h);
  v.y -= hi16(h);
  return h;
}

using bf16 = __nv_bfloat16;

// Channels c, c + 1 of a row as two bf16 (0 past the last); `pairs`: both exist, in one 4-byte access
AHB_DEVICE uint32_t load_pair(const bf16* row, int c, int C, bool pairs) {
  if (pairs) return __ldg(reinterpret_cast<const unsigned int*>(row + c));
  if (c >= C) return 0u;
  const uint16_t* r = reinterpret_cast<const uint16_t*>(row) + c;
  return __ldg(r) | (c + 1 < C ? (uint32_t)__ldg(r + 1) << 16 : 0u);
}
AHB_DEVICE void store_pair(bf16* row, int c, int C, bool pairs, uint32_t v) {
  if (pairs && c < C) {
    *reinterpret_cast<uint32_t*>(row + c) = v;
  } else if (c < C) {
    uint16_t* r = reinterpret_cast<uint16_t*>(row) + c;
    r[0] = (uint16_t)v;
    if (c + 1 < C) r[1] = (uint16_t)(v >> 16);
  }
}

// Two warps share 16 channels: each makes V for its 16 of the block's 32 tokens and keeps half of the
// states (32 accumulator registers a thread at N = 128, so that 16 warps fit an SM and hide each other's
// latencies: 12 warps with whole states were issuing 42 % of the time).
constexpr int kBlock = 32, kGroups = 4, kWarps = 2 * kGroups, kChan = 16 * kGroups;

// A block's rows of B and C, clipped, zeros past the sequence's end, and C B^T up to the diagonal in two bf16
// terms: made once (scan_rows_kernel), read by every group of channels.
template <int N>
struct BlockRows {
  bf16 b[kBlock][N], c[kBlock][N], cb[2][kBlock][kBlock];
};

template <int N>
__global__ void __launch_bounds__(192) scan_rows_kernel(PromptArgs pa) {
  constexpr int LD = N + 8;
  __shared__ bf16 sb[kBlock][LD], sc[kBlock][LD];
  const ScanArgs& p = pa.a;
  const Segment sg = find_segment(p, kBlock, blockIdx.x);
  if (sg.b < 0) return;
  BlockRows<N>& out = reinterpret_cast<BlockRows<N>*>(pa.rows)[blockIdx.x];
  const int tid = threadIdx.x, t0 = sg.seq.start + sg.index * kBlock;
  const bool wide = ((p.bs | p.cs) & 7) == 0 && ((reinterpret_cast<uintptr_t>(p.Bm) | reinterpret_cast<uintptr_t>(p.Cm)) & 15) == 0;
  for (int piece = tid; piece < kBlock * N / 8; piece += 192) {
    const int row = piece / (N / 8), col = piece % (N / 8) * 8;
    uint4 v[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
    if (t0 + row < sg.seq.end) {
      const bf16* from[2] = {static_cast<const bf16*>(p.Bm) + (int64_t)(t0 + row) * p.bs + col,
                             static_cast<const bf16*>(p.Cm) + (int64_t)(t0 + row) * p.cs + col};
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        if (wide) {
          v[m] = __ldg(reinterpret_cast<const uint4*>(from[m]));
        } else {
          const uint16_t* f = reinterpret_cast<const uint16_t*>(from[m]);
          v[m] = make_uint4(f[0] | (uint32_t)f[1] << 16, f[2] | (uint32_t)f[3] << 16, f[4] | (uint32_t)f[5] << 16, f[6] | (uint32_t)f[7] << 16);
        }
        v[m] = make_uint4(clip2(v[m].x), clip2(v[m].y), clip2(v[m].z), clip2(v[m].w));
      }
    }
    *reinterpret_cast<uint4*>(&sb[row][col]) = *reinterpret_cast<uint4*>(&out.b[row][col]) = v[0];
    *reinterpret_cast<uint4*>(&sc[row][col]) = *reinterpret_cast<uint4*>(&out.c[row][col]) = v[1];
  }
  __syncthreads();
  // one warp each: 16 x 8 pieces of (0,0), (16,0), (16,16); nothing reads the fourth quarter
  const int lane = tid & 31, warp = tid >> 5, g = lane >> 2, q = lane & 3;
  const int tb = warp < 2 ? 0 : 16, cb = (warp < 4 ? 0 : 16) + (warp & 1) * 8;
  float acc[2][4];
  zero_acc<2>(acc);
#pragma unroll
  for (int k = 0; k < N; k += 32) {
    uint32_t a[4], b[4];
    ldsm4(b, &sb[cb + (lane & 7)][k + (lane >> 3) * 8]);
    ldsm4(a, &sc[tb + (lane & 15)][k + (lane >> 4) * 8]);
    mma16816(acc[0], a, b);
    ldsm4(a, &sc[tb + (lane & 15)][k + 16 + (lane >> 4) * 8]);
    mma16816(acc[1], a, b + 2);
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int t = tb + g + 8 * h, c = cb + 2 * q;
    float2 v = make_float2(c <= t ? acc[0][2 * h] + acc[1][2 * h] : 0.f, c + 1 <= t ? acc[0][2 * h + 1] + acc[1][2 * h + 1] : 0.f);
    *reinterpret_cast<uint32_t*>(&out.cb[0][t][c]) = term2(v);
    *reinterpret_cast<uint32_t*>(&out.cb[1][t][c]) = pack2(v.x, v.y);
  }
}

template <int N>
struct BlockSmem {
  static constexpr int LD = N + 8;    // row strides that spread ldmatrix rows over the banks
  static constexpr int LT = kBlock + 4, LV = kBlock + 8;
  bf16 b[2][kBlock][LD];
  bf16 c[2][kBlock][LD];
  bf16 cb[2][2][kBlock][LV];          // C B^T up to the diagonal: high and low terms
  bf16 v[kGroups][3][16][LV];         // the terms of V per channel and token
  float y[kGroups][2][16][LT];        // both warps' parts of the outputs
  float u[kGroups][16][LT];           // a group's inputs and decays where it goes token by token
  float d[kGroups][16][LT];
  float span[kGroups][2][16];         // log2 decay of each half block
};

// Multiplies the accumulator rows (channels) by factors that lane l holds for channel l % 16.
template <int NT>
AHB_DEVICE void scale_rows(float (*S)[4], float f) {
  const int g = (threadIdx.x & 31) >> 2;
  const float2 r0 = both(__shfl_sync(0xffffffffu, f, g)), r1 = both(__shfl_sync(0xffffffffu, f, g + 8));
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    const float2 u = mul2(make_float2(S[j][0], S[j][1]), r0), v = mul2(make_float2(S[j][2], S[j][3]), r1);
    S[j][0] = u.x;
    S[j][1] = u.y;
    S[j][2] = v.x;
    S[j][3] = v.y;
  }
}

// FAST: 4-byte access to channel pairs, whole groups of 16 channels (the other form takes any alignment,
// stride and number of channels).
template <typename W, int N, bool STATE, bool FAST>
__global__ void __launch_bounds__(kWarps * 32, 2) scan_block_kernel(PromptArgs pa) {
  constexpr int M = N / 2, NT = M / 8;      // this warp's states, their accumulator tiles
  using Smem = BlockSmem<N>;
  extern __shared__ __align__(16) unsigned char raw[];
  Smem& sm = *reinterpret_cast<Smem*>(raw);
  const ScanArgs& p = pa.a;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, grp = warp >> 1, half = warp & 1;
  const int g = lane >> 2, q = lane & 3;    // accumulator rows g, g + 8; columns 2 q, 2 q + 1
  const int i = lane & 7, tg = lane >> 3;   // channels 2 i, 2 i + 1 of tokens tk .. tk + 3
  const int tk = half * 16 + tg * 4;
  // with whole groups, those past the last channel repeat its group and store nothing
  const int c1 = blockIdx.y * kChan + grp * 16, c0 = FAST ? min(c1, p.C - 16) : c1, ca = c0 + 2 * i;
  const bool mine = !FAST || c1 < p.C;
  const Segment sg = find_segment(p, pa.seg, blockIdx.x);
  if (!STATE && p.cu != nullptr) {  // every block clears some of the rows without a sequence
    const OpenRows open(p.cu, p.B, p.T);
    const int c = blockIdx.y * kChan + 2 * lane;
    for (int i = blockIdx.x * kWarps + warp; i < open.count; i += gridDim.x * kWarps)
      store_pair(static_cast<bf16*>(p.y) + (int64_t)open.row(i) * p.C, c, p.C, FAST || (p.C & 1) == 0, 0u);
  }
  if (sg.b < 0) return;
  if (STATE && sg.index == sg.count - 1) return;  // its end state comes with its outputs
  const int slot = seq_slot(p.slots, sg.b, p.S);
  const int start = sg.seq.start + sg.index * pa.seg, end = min(start + pa.seg, sg.seq.end);
  bf16* const y = static_cast<bf16*>(p.y);
  const bf16* const x = static_cast<const bf16*>(p.x);
  const bf16* const dt = static_cast<const bf16*>(p.dt);
  const bool ypairs = FAST || (p.C & 1) == 0;
  const bool pairs = FAST;
  if (slot < 0) {
    if (!STATE && mine)
      for (int t = start + half * 4 + tg; t < end; t += 8) store_pair(y + (int64_t)t * p.C, ca, p.C, ypairs, 0u);
    return;
  }

  float2 w[4], bias, A2;
  {
    const bool h0 = ca < p.C, h1 = ca + 1 < p.C;
    const W* taps = static_cast<const W*>(p.conv_w) + (int64_t)ca * 4;
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = make_float2(h0 ? to_f(taps[j]) : 0.f, h1 ? to_f(taps[4 + j]) : 0.f);
    bias = make_float2(h0 && p.conv_b ? p.conv_b[ca] : 0.f, h1 && p.conv_b ? p.conv_b[ca + 1] : 0.f);
    A2 = make_float2(h0 ? p.A[ca / p.P] * kLog2e : 0.f, h1 ? p.A[(ca + 1) / p.P] * kLog2e : 0.f);
  }
  bf16* const win = static_cast<bf16*>(p.conv_state) + (int64_t)slot * 3 * p.C;

  float S[NT][4];
  float* const slot_state = p.state + (int64_t)slot * p.C * N;
  float* const seg_state = pa.states + (int64_t)(sg.first + sg.index) * p.C * N;
  const bool has0 = FAST || c0 + g < p.C, has1 = FAST || c0 + g + 8 < p.C;
  const int64_t at_state = (int64_t)(c0 + g) * N + half * M + 2 * q;
  {
    const float* src = (sg.count == 1 ? slot_state : seg_state) + at_state;
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      float2 u = make_float2(0.f, 0.f), v = u;
      if (!STATE && has0) u = *reinterpret_cast<const float2*>(src + 8 * j);
      if (!STATE && has1) v = *reinterpret_cast<const float2*>(src + 8 * N + 8 * j);
      S[j][0] = u.x;
      S[j][1] = u.y;
      S[j][2] = v.x;
      S[j][3] = v.y;
    }
  }

  const int block0 = sg.blocks + sg.index * (pa.seg / kBlock);
  auto copy_block = [&](int block, int buf) {
    const BlockRows<N>& from = reinterpret_cast<const BlockRows<N>*>(pa.rows)[block];
    auto copy = [&](bf16* to, const bf16* f) {
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(to)), "l"(f) : "memory");
    };
#pragma unroll
    for (int piece = tid; piece < kBlock * N / 8; piece += kWarps * 32) {
      const int row = piece / (N / 8), col = piece % (N / 8) * 8;
      copy(&sm.b[buf][row][col], &from.b[row][col]);
      if (!STATE) copy(&sm.c[buf][row][col], &from.c[row][col]);
    }
    if (!STATE) {
      const int m = tid >> 7, row = (tid >> 2) & 31, col = (tid & 3) * 8;  // 2 x 32 x 4 pieces, one a thread
      copy(&sm.cb[buf][m][row][col], &from.cb[m][row][col]);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  // this lane's tokens; lanes of the warp's first tokens also hold the three rows before them
  uint32_t xr[4], dr[4], hr[3];
  auto load_tokens = [&](int t0) {
    const bf16* xp = x + (int64_t)(t0 + tk) * p.xs + ca;
    const bf16* dp = dt + (int64_t)(t0 + tk) * p.dts + ca;
    if (FAST && t0 + kBlock <= end && (half == 1 || t0 > sg.seq.start)) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        xr[k] = __ldg(reinterpret_cast<const unsigned int*>(xp + k * p.xs));
        dr[k] = __ldg(reinterpret_cast<const unsigned int*>(dp + k * p.dts));
      }
      if (tg == 0) {
#pragma unroll
        for (int j = 0; j < 3; ++j) hr[j] = __ldg(reinterpret_cast<const unsigned int*>(xp + (j - 3) * p.xs));
      }
      return;
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const bool in = t0 + tk + k < end;
      xr[k] = in ? load_pair(xp - ca + k * p.xs, ca, p.C, pairs) : 0u;
      dr[k] = in ? load_pair(dp - ca + k * p.dts, ca, p.C, pairs) : 0u;
    }
    if (tg == 0) {
#pragma unroll
      for (int j = 0; j < 3; ++j) {
        const int t = t0 + tk + j - 3, back = t - sg.seq.start;
        hr[j] = back < 0 ? load_pair(win + (back + 3) * p.C, ca, p.C, pairs)
                         : t < end ? load_pair(x + (int64_t)t * p.xs, ca, p.C, pairs) : 0u;
      }
    }
  };

  copy_block(block0, 0);
  load_tokens(start);
  float pend = 0.f, total = 0.f;  // of channel lane % 16: log2 of the scale S still lacks, of the segment's decay
  int buf = 0;
  for (int t0 = start; t0 < end; t0 += kBlock, buf ^= 1) {
    const int n = min(kBlock, end - t0);
    // convolution, step and input of this lane's channels and tokens
    float2 E[4], u[4];
    {
      uint32_t xs[7];
#pragma unroll
      for (int j = 0; j < 3; ++j) {
        const uint32_t last = __shfl_up_sync(0xffffffffu, xr[1 + j], 8);
        xs[j] = tg == 0 ? hr[j] : last;
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) xs[3 + k] = xr[k];
      float2 odd = both(0.f);  // NaN as soon as an input is not finite
      float most = 0.f;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        float2 a = bias;
#pragma unroll
        for (int j = 0; j < 4; ++j) a = fma2(w[j], both16(xs[k + j]), a);
        const float2 t = mul2(a, both(-kLog2e)), d = add2(make_float2(ex2(t.x), ex2(t.y)), both(1.f));
        u[k] = mul2(a, make_float2(rcp(d.x), rcp(d.y)));
        most = fmaxf(most, fmaxf(fabsf(u[k].x), fabsf(u[k].y)));
        const float2 r = both16(dr[k]), sp = softplus2(r);
        E[k] = make_float2(fminf(fmaxf(sp.x, p.dt_min), p.dt_max), fminf(fmaxf(sp.y, p.dt_min), p.dt_max));
        odd = fma2(add2(a, r), both(0.f), odd);
      }
      if (__any_sync(0xffffffffu, (odd.x != odd.x) | (odd.y != odd.y) | (most > kClip))) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float2 r = both16(dr[k]);
          u[k] = make_float2(sanitize(u[k].x, kClip), sanitize(u[k].y, kClip));
          E[k] = make_float2(r.x != r.x ? 0.f : E[k].x, r.y != r.y ? 0.f : E[k].y);
        }
      }
      if (n < kBlock) {
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (tk + k >= n) E[k] = both(0.f);
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        u[k] = mul2(u[k], E[k]);
        E[k] = max2(mul2(E[k], A2), kMinDA * kLog2e);
      }
    }
    if (t0 + kBlock < end) load_tokens(t0 + kBlock);
    // decays summed along the warp's half block, over the four lanes of a channel
    const float2 sum = add2(add2(E[0], E[1]), add2(E[2], E[3]));
    float2 incl = sum, v = make_float2(__shfl_up_sync(0xffffffffu, sum.x, 8), __shfl_up_sync(0xffffffffu, sum.y, 8));
    if (tg >= 1) incl = add2(incl, v);
    v = make_float2(__shfl_up_sync(0xffffffffu, incl.x, 16), __shfl_up_sync(0xffffffffu, incl.y, 16));
    if (tg >= 2) incl = add2(incl, v);
    const float2 whole = make_float2(__shfl_sync(0xffffffffu, incl.x, 24 + i), __shfl_sync(0xffffffffu, incl.y, 24 + i));
    if (tg == 0) *reinterpret_cast<float2*>(&sm.span[grp][half][2 * i]) = whole;
    asm volatile("bar.sync %0, 64;" ::"r"(grp + 1) : "memory");  // the pair's spans are there
    const float mid = sm.span[grp][0][lane & 15], tail = sm.span[grp][1][lane & 15];
    const bool heavy = __any_sync(0xffffffffu, fmaxf(fabsf(mid), fabsf(tail)) > kSpan);
    if (heavy) {  // V would leave the floats' range: the group goes token by token, on these
      *reinterpret_cast<float4*>(&sm.u[grp][2 * i][tk]) = make_float4(u[0].x, u[1].x, u[2].x, u[3].x);
      *reinterpret_cast<float4*>(&sm.u[grp][2 * i + 1][tk]) = make_float4(u[0].y, u[1].y, u[2].y, u[3].y);
      *reinterpret_cast<float4*>(&sm.d[grp][2 * i][tk]) = make_float4(E[0].x, E[1].x, E[2].x, E[3].x);
      *reinterpret_cast<float4*>(&sm.d[grp][2 * i + 1][tk]) = make_float4(E[0].y, E[1].y, E[2].y, E[3].y);
    } else {
      // E: the first half ends at the reference, the second starts from it
      float2 run = add2(incl, make_float2(-sum.x, -sum.y));
      if (half == 0) run = add2(run, make_float2(-whole.x, -whole.y));
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        run = add2(run, E[k]);
        u[k] = mul2(u[k], make_float2(ex2(-run.x), ex2(-run.y)));
        E[k] = run;
      }
      float2 V0[2] = {{u[0].x, u[1].x}, {u[2].x, u[3].x}}, V1[2] = {{u[0].y, u[1].y}, {u[2].y, u[3].y}};
#pragma unroll
      for (int m = 0; m < 3; ++m) {
        *reinterpret_cast<uint2*>(&sm.v[grp][m][2 * i][tk]) = make_uint2(term2(V0[0]), term2(V0[1]));
        *reinterpret_cast<uint2*>(&sm.v[grp][m][2 * i + 1][tk]) = make_uint2(term2(V1[0]), term2(V1[1]));
      }
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();  // the block's rows are there, and V; every warp is done with the other buffer
    if (t0 + kBlock < end) copy_block(block0 + (t0 - start) / kBlock + 1, buf ^ 1);
    total += mid + tail;
    // S takes the scale it lacks and goes to the block's reference.  S itself may stand at 2^kSpan, so the two
    // scales go in one after the other where their product would leave the floats' range.
    if (__any_sync(0xffffffffu, fabsf(pend + mid) > 120.f)) {
      scale_rows<NT>(S, ex2(pend));
      pend = 0.f;
    }
    scale_rows<NT>(S, ex2(heavy ? pend : pend + mid));
    pend = heavy ? 0.f : tail;

    const int mrow = lane & 15, mcol = (lane >> 4) * 8;  // ldmatrix: rows of a 16 x 16 piece, its column half
    const int xrow = (lane & 7) + (lane >> 4) * 8, xcol = ((lane >> 3) & 1) * 8;  // two 8-row halves, each with both column halves

    // A product waits for the one before it on the same accumulators, so consecutive ones go to different ones.
    float Y[4][4];
    if (!STATE) zero_acc<4>(Y);
    if (!heavy) {
      if (!STATE) {
#pragma unroll
        for (int k = 0; k < M / 16; ++k) {  // Y += S C^T over this warp's states
          uint32_t sh[4], sl[4], cf[2][4];
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            float2 v = make_float2(S[2 * k + (r >> 1)][(r & 1) * 2], S[2 * k + (r >> 1)][(r & 1) * 2 + 1]);
            sh[r] = term2(v);
            sl[r] = pack2(v.x, v.y);
          }
#pragma unroll
          for (int h = 0; h < 2; ++h) ldsm4(cf[h], &sm.c[buf][16 * h + xrow][half * M + 16 * k + xcol]);
#pragma unroll
          for (int j = 0; j < 4; ++j) mma16816(Y[j], sh, cf[j >> 1] + 2 * (j & 1));
#pragma unroll
          for (int j = 0; j < 4; ++j) mma16816(Y[j], sl, cf[j >> 1] + 2 * (j & 1));
        }
      }
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
        uint32_t vf[3][4];
#pragma unroll
        for (int m = 0; m < 3; ++m) ldsm4(vf[m], &sm.v[grp][m][mrow][16 * ks + mcol]);
        if (!STATE) {  // Y += V (C B^T)^T: the pieces (0,0) and (16,16) by one warp, (16,0) by the other
          if (half == 0 || ks == 0) {
            const int tb = half == 0 ? 16 * ks : 16;
            uint32_t bh[4], bl[4];
            ldsm4(bh, &sm.cb[buf][0][tb + xrow][16 * ks + xcol]);
            ldsm4(bl, &sm.cb[buf][1][tb + xrow][16 * ks + xcol]);
            if (tb == 0) {
#pragma unroll
              for (int m = 0; m < 3; ++m)
#pragma unroll
                for (int j = 0; j < 2; ++j) mma16816(Y[j], vf[m == 2], (m == 1 ? bl : bh) + 2 * j);
            } else {
#pragma unroll
              for (int m = 0; m < 3; ++m)
#pragma unroll
                for (int j = 0; j < 2; ++j) mma16816(Y[2 + j], vf[m == 2], (m == 1 ? bl : bh) + 2 * j);
            }
          }
        }
        uint32_t bf[M / 16][4];  // S += V^T B
#pragma unroll
        for (int j = 0; j < M / 16; ++j) ldsm4_t(bf[j], &sm.b[buf][16 * ks + mrow][half * M + 16 * j + mcol]);
#pragma unroll
        for (int m = 0; m < 3; ++m)
#pragma unroll
          for (int j = 0; j < NT; ++j) mma16816(S[j], vf[m], bf[j >> 1] + 2 * (j & 1));
      }
      if (!STATE) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          *reinterpret_cast<float2*>(&sm.y[grp][half][g][8 * j + 2 * q]) = make_float2(Y[j][0], Y[j][1]);
          *reinterpret_cast<float2*>(&sm.y[grp][half][g + 8][8 * j + 2 * q]) = make_float2(Y[j][2], Y[j][3]);
        }
      }
    } else {
      for (int t = 0; t < n; ++t) {
        const float a0 = ex2(sm.d[grp][g][t]), a1 = ex2(sm.d[grp][g + 8][t]), u0 = sm.u[grp][g][t], u1 = sm.u[grp][g + 8][t];
        float y0 = 0.f, y1 = 0.f;
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          const float2 bb = both16(*reinterpret_cast<const uint32_t*>(&sm.b[buf][t][half * M + 8 * j + 2 * q]));
          S[j][0] = fmaf(a0, S[j][0], u0 * bb.x);
          S[j][1] = fmaf(a0, S[j][1], u0 * bb.y);
          S[j][2] = fmaf(a1, S[j][2], u1 * bb.x);
          S[j][3] = fmaf(a1, S[j][3], u1 * bb.y);
          if (!STATE) {
            const float2 cc = both16(*reinterpret_cast<const uint32_t*>(&sm.c[buf][t][half * M + 8 * j + 2 * q]));
            y0 = fmaf(cc.x, S[j][0], fmaf(cc.y, S[j][1], y0));
            y1 = fmaf(cc.x, S[j][2], fmaf(cc.y, S[j][3], y1));
          }
        }
        if (!STATE) {
          y0 += __shfl_xor_sync(0xffffffffu, y0, 1);
          y1 += __shfl_xor_sync(0xffffffffu, y1, 1);
          y0 += __shfl_xor_sync(0xffffffffu, y0, 2);
          y1 += __shfl_xor_sync(0xffffffffu, y1, 2);
          if (q == 0) {
            sm.y[grp][half][g][t] = y0;
            sm.y[grp][half][g + 8][t] = y1;
          }
        }
      }
    }
    // the pair's outputs are there, and it is done with V, u and d
    asm volatile("bar.sync %0, 64;" ::"r"(grp + 1) : "memory");
    if (!STATE) {
      const float4 a0 = *reinterpret_cast<const float4*>(&sm.y[grp][0][2 * i][tk]), b0 = *reinterpret_cast<const float4*>(&sm.y[grp][1][2 * i][tk]);
      const float4 a1 = *reinterpret_cast<const float4*>(&sm.y[grp][0][2 * i + 1][tk]), b1 = *reinterpret_cast<const float4*>(&sm.y[grp][1][2 * i + 1][tk]);
      const float2 o[4] = {{a0.x + b0.x, a1.x + b1.x}, {a0.y + b0.y, a1.y + b1.y}, {a0.z + b0.z, a1.z + b1.z}, {a0.w + b0.w, a1.w + b1.w}};
      bf16* row = y + (int64_t)(t0 + tk) * p.C;
#pragma unroll
      for (int k = 0; k < 4; ++k, row += p.C) {
        const float2 r = heavy ? o[k] : mul2(o[k], make_float2(ex2(E[k].x), ex2(E[k].y)));
        if (mine && tk + k < n) store_pair(row, ca, p.C, ypairs, pack2(r.x, r.y));
      }
    }
  }

  // the end state, with the scale it lacks
  if (mine && (STATE || sg.index == sg.count - 1)) {
    scale_rows<NT>(S, ex2(pend));
    float* dst = (STATE ? seg_state : slot_state) + at_state;
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      if (has0) *reinterpret_cast<float2*>(dst + 8 * j) = make_float2(S[j][0], S[j][1]);
      if (has1) *reinterpret_cast<float2*>(dst + 8 * N + 8 * j) = make_float2(S[j][2], S[j][3]);
    }
    if (STATE && half == 0 && lane < 16 && c0 + lane < p.C) pa.decays[(int64_t)(sg.first + sg.index) * p.C + c0 + lane] = total;
  }
  // the first segment's block alone reads the window, so it may write it
  if (!STATE && mine && sg.index == 0 && half == 0 && tg == 0) {
    const int len = sg.seq.end - sg.seq.start;
    uint32_t nw[3];
#pragma unroll
    for (int j = 0; j < 3; ++j) {
      const int at = len + j - 3;
      nw[j] = at >= 0 ? load_pair(x + (int64_t)(sg.seq.start + at) * p.xs, ca, p.C, pairs) : load_pair(win + (3 + at) * p.C, ca, p.C, pairs);
    }
#pragma unroll
    for (int j = 0; j < 3; ++j) store_pair(win + j * p.C, ca, p.C, pairs, nw[j]);
  }
}

// Hands the state on along the segments of every sequence with more than one: start states replace the
// end states from zero.  One thread per four states of a channel.
template <int N>
__global__ void __launch_bounds__(256) scan_join_kernel(PromptArgs pa) {
  const ScanArgs& p = pa.a;
  const int b = blockIdx.y;
  const int slot = seq_slot(p.slots, b, p.S);
  if (slot < 0) return;
  SeqRange r = seq_range(nullptr, b, p.L, p.T);
  int first = 0;
  if (p.cu != nullptr) {
    const int lane = threadIdx.x & 31;
    int reach = offset_of(p, 0);
    for (int b0 = 0; b0 <= b; b0 += 32) {
      const SeqRange q = rising_ranges(p, b0, reach);
      first += __reduce_add_sync(0xffffffffu, b0 + lane < b ? (q.end - q.start + pa.seg - 1) / pa.seg : 0);
      r = range_of_lane(q, b & 31);
    }
  }
  const int count = (r.end - r.start + pa.seg - 1) / pa.seg;
  if (p.cu == nullptr) first = b * count;
  if (count < 2) return;
  const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (at >= (int64_t)p.C * (N / 4)) return;
  const int c = (int)(at / (N / 4));
  float4 run = reinterpret_cast<const float4*>(p.state + (int64_t)slot * p.C * N)[at];
  constexpr int AHEAD = 8;  // segments whose end states are on the way together
  for (int s0 = 0; s0 < count; s0 += AHEAD) {
    float4 own[AHEAD];
    float f[AHEAD];
#pragma unroll
    for (int k = 0; k < AHEAD; ++k)
      if (s0 + k < count - 1) {
        own[k] = *(reinterpret_cast<const float4*>(pa.states + (int64_t)(first + s0 + k) * p.C * N) + at);
        f[k] = ex2(pa.decays[(int64_t)(first + s0 + k) * p.C + c]);
      }
#pragma unroll
    for (int k = 0; k < AHEAD; ++k)
      if (s0 + k < count) {
        *(reinterpret_cast<float4*>(pa.states + (int64_t)(first + s0 + k) * p.C * N) + at) = run;
        if (s0 + k < count - 1)
          run = make_float4(fmaf(f[k], run.x, own[k].x), fmaf(f[k], run.y, own[k].y), fmaf(f[k], run.z, own[k].z), fmaf(f[k], run.w, own[k].w));
      }
  }
}

// Segments of T tokens in B sequences: as many as any packing of them can have (a sequence of l tokens has fewer than
// l / seg + 1)
int64_t max_segments(int B, int L, int T, bool packed, int seg) {
  return packed ? (int64_t)T / seg + B : (int64_t)B * ((L + seg - 1) / seg);
}

template <typename W, int N, bool FAST>
int launch_prompt(const ScanArgs& a, int seg, float* work, cudaStream_t st) {
  static bool ready[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev >= 64) return -3;
  const int bytes = (int)sizeof(BlockSmem<N>);
  if (!ready[dev]) {
    if (cudaFuncSetAttribute(scan_block_kernel<W, N, true, FAST>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess ||
        cudaFuncSetAttribute(scan_block_kernel<W, N, false, FAST>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess)
      return -3;
    ready[dev] = true;
  }
  const bool packed = a.cu != nullptr;
  const int64_t segs = max_segments(a.B, a.L, a.T, packed, seg), blocks = max_segments(a.B, a.L, a.T, packed, kBlock);
  float* const states = work + blocks * (int64_t)(sizeof(BlockRows<N>) / 4);
  const PromptArgs p{a, seg, states, states + segs * a.C * N, reinterpret_cast<bf16*>(work)};
  const dim3 grid((unsigned)segs, (unsigned)((a.C + kChan - 1) / kChan));
  scan_rows_kernel<N><<<(unsigned)blocks, 192, 0, st>>>(p);
  if (segs > a.B) {
    scan_block_kernel<W, N, true, FAST><<<grid, kWarps * 32, bytes, st>>>(p);
    scan_join_kernel<N><<<dim3((unsigned)(((int64_t)a.C * (N / 4) + 255) / 256), (unsigned)a.B), 256, 0, st>>>(p);
  }
  scan_block_kernel<W, N, false, FAST><<<grid, kWarps * 32, bytes, st>>>(p);
  return 0;
}

template <typename W, int N>
int launch_prompt(const ScanArgs& a, int seg, float* work, cudaStream_t st) {
  const auto low = [](const void* p) { return reinterpret_cast<uintptr_t>(p); };
  const bool fast = a.C % 16 == 0 && ((a.xs | a.dts) & 1) == 0 && ((low(a.x) | low(a.dt) | low(a.conv_state)) & 3) == 0;
  return fast ? launch_prompt<W, N, true>(a, seg, work, st) : launch_prompt<W, N, false>(a, seg, work, st);
}

template <typename T, typename W>
int by_state(const ScanArgs& p, int N, int seg, float* work, cudaStream_t st) {
  if constexpr (sizeof(T) == 2) {
    if (seg > 0) {
      if (N == 128) return launch_prompt<W, 128>(p, seg, work, st);
      if (N == 64) return launch_prompt<W, 64>(p, seg, work, st);
      if (N == 32) return launch_prompt<W, 32>(p, seg, work, st);
      return -1;
    }
  }
  if (N == 128) launch_token<T, W, 128>(p, st);
  else if (N == 64) launch_token<T, W, 64>(p, st);
  else if (N == 32) launch_token<T, W, 32>(p, st);
  else return -1;
  return 0;
}

}  // namespace

int ahb_selective_scan_plan(int B, int L, int T, int C, int N, int packed, int dtype, int64_t* floats, int* kernels) {
  *floats = 0;
  *kernels = T == 0 || B == 0 ? 0 : 1;
  // Blocks from 16 tokens a sequence on average (the host knows no more of packed ones, so a prompt among many single
  // tokens goes token by token: 512 tokens beside 64 of them 286 us, alone 59).  One sequence of 2048
  // channels: 8 tokens 7.3 us token by token and 10.4 us in blocks, 16 tokens 11.2 and 10.4, 32 tokens 19 and 11;
  // 128 sequences: 123 and 190, 212 and 194, 395 and 203 us.
  if (dtype != AHB_BF16 || B == 0 || T < 16 * (int64_t)B) return 0;
  // Two blocks of 64 channels run on an SM.  Sequences that fill them stay whole (a segment more costs
  // another state pass over it); others are cut so that one wave of blocks holds all segments.  Of several packed
  // sequences the host knows the mean length: they are cut by their tokens' share of a wave, and at the mean
  // where that is not much longer (4 of 512 tokens, 4096 channels: 84 us whole, 136 us cut at their share of 448).
  const int64_t groups = (C + kChan - 1) / kChan, wave = 2 * 148;
  int64_t seg;
  if (packed && B > 1) {
    const int64_t mean = (T + B - 1) / B;
    seg = T * groups / wave;
    if (4 * seg > 3 * mean) seg = std::max(seg, mean);
  } else {
    const int64_t n = packed ? T : L, cuts = std::max<int64_t>(1, wave / (B * groups));
    seg = (n + cuts - 1) / cuts;
  }
  seg = std::min<int64_t>(1 << 30, std::max<int64_t>(128, (seg + kBlock - 1) / kBlock * kBlock));
  const int64_t segs = max_segments(B, L, T, packed != 0, (int)seg);
  *kernels = segs > B ? 4 : 2;
  const int64_t rows = (int64_t)(2 * kBlock * N + 2 * kBlock * kBlock) / 2;  // of a block, in floats
  *floats = max_segments(B, L, T, packed != 0, kBlock) * rows + (segs > B ? segs * C * (N + 1) : 0);
  return (int)seg;
}

int ahb_selective_scan(const void* x, int64_t xs, const void* dt, int64_t dts, const float* A, const void* Bm,
                       int64_t bs, const void* Cm, int64_t cs, const void* conv_w, int wdtype, const float* conv_b,
                       void* conv_state, float* state, const int* cu, const int* slots, void* y, int B, int L, int T,
                       int C, int P, int N, int S, int dtype, float dt_min, float dt_max, int seg, float* work,
                       cudaStream_t st) {
  if (T == 0 || B == 0) return 0;
  if (B > 65535) return -2;
  const ScanArgs p{x, dt, Bm, Cm, conv_w, xs, dts, bs, cs, A, conv_b, conv_state, state, cu, slots, y,
                   B, L, T, C, P, S, dt_min, dt_max};
  const bool wb = wdtype == AHB_BF16;
  if (dtype == AHB_BF16)
    return wb ? by_state<__nv_bfloat16, __nv_bfloat16>(p, N, seg, work, st) : by_state<__nv_bfloat16, float>(p, N, seg, work, st);
  return wb ? by_state<float, __nv_bfloat16>(p, N, 0, nullptr, st) : by_state<float, float>(p, N, 0, nullptr, st);
}
