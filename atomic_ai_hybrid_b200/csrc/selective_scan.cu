// Mamba2's short causal convolution and selective scan with state carried between calls (prompts of
// any length and single tokens), for serving (the layer's mathematics: reference `model.py:391-525`).
//
//   xc_t = sanitize(silu(sum_j w_j x_{t-3+j} + b)),  dt_t = clamp(softplus(dtraw_t), dt_min, dt_max)
//   S_t[c,:] = e^{max(dt_t A_h, -20)} S_{t-1}[c,:] + dt_t xc_t B_t ,   y_t[c] = <C_t, S_t[c,:]>
#include "launchers.h"
#include "mma.cuh"
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

// ---------------------------------------------------------------- token form
// One warp carries CH channels of one sequence through its tokens: lane l holds states
// [l V, l V + V) of each channel in registers (N = 32 V), lanes 0..CH-1 also hold the convolution
// window of one channel and turn its row into (decay, dt xc).
template <typename T, typename W, int N, int CH, int WARPS>
__global__ void __launch_bounds__(WARPS * 32) scan_token_kernel(ScanArgs p) {
  constexpr int V = N / 32;
  const int lane = threadIdx.x & 31, b = blockIdx.y;
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
  for (int t = r.start; t < r.end; ++t) {
    float a = 0.f, u = 0.f;
    if (mine) {
      const float x3 = to_f(static_cast<const T*>(p.x)[(int64_t)t * p.xs + c]);
      const float dt = dt_of(to_f(static_cast<const T*>(p.dt)[(int64_t)t * p.dts + c]), p.dt_min, p.dt_max);
      a = exp_decay(fmaxf(dt * A, kMinDA));
      u = dt * sanitize(conv_silu(w, bias, x0, x1, x2, x3), kClip);
      x0 = x1;
      x1 = x2;
      x2 = x3;
    }
    float Bv[V], Cv[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      Bv[i] = sanitize(to_f(Bm[(int64_t)t * p.bs + lane * V + i]), kClip);
      Cv[i] = sanitize(to_f(Cm[(int64_t)t * p.cs + lane * V + i]), kClip);
    }
    float out = 0.f;
#pragma unroll
    for (int j = 0; j < CH; ++j) {
      const float aj = __shfl_sync(0xffffffffu, a, j), uj = __shfl_sync(0xffffffffu, u, j);
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        h[j][i] = fmaf(aj, h[j][i], uj * Bv[i]);
        s = fmaf(Cv[i], h[j][i], s);
      }
      s = warp_sum(s);
      if (lane == j) out = s;
    }
    if (mine) y[(int64_t)t * p.C + c] = from_f<T>(out);
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

template <typename T, typename W, int N>
void launch_token(const ScanArgs& p, cudaStream_t st) {
  constexpr int CH = 8, WARPS = 4;
  const dim3 grid((p.C + CH * WARPS - 1) / (CH * WARPS), p.B);
  scan_token_kernel<T, W, N, CH, WARPS><<<grid, WARPS * 32, 0, st>>>(p);
}

// ---------------------------------------------------------------- prompt form (bf16)
// The recurrence of a block of 32 tokens as products over the block.  With c_t = sum_{r <= t} log2(e) dA_r
// from the block's start, m = c after 16 tokens and E_t = c_t - m per channel p,
//   Y[t,p]  = 2^{E_t} ( C_t . (2^m S) + sum_{s <= t} (C_t . B_s) V_s )       V_s = 2^{-E_s} u_s
//   S'      = 2^{E_end} ( 2^m S + sum_s V_s B_s )
// so one factor V serves the output and the state, and C B^T is shared by all channels.  The exponents
// stay below 2^kSpan as long as neither half block decays by more; a warp whose channels do
// takes its block token by token instead.  Both sums run on m16n8k16 bf16 products with fp32 accumulators:
// a warp keeps the fp32 state of 16 channels as accumulators (channels are rows), which the next
// block's C S product takes back as its left operand without leaving the registers.  B and C are bf16
// already; the fp32 factors go in as bf16 terms: V in three (24 bits, the state loses nothing), S and
// C B^T in two (2^-17, for outputs rounded to bf16).  tcgen05 would have the state in TMEM, where
// rescaling it per channel and block costs a round trip through the registers it is spared here.
//
// Long sequences are cut into segments of `seg` tokens.  A first launch finds every segment's state from
// zero and its decay, a second one hands the states on from segment to segment (scan_join_kernel), a
// third one runs the segments from their true states with outputs.
struct PromptArgs {
  ScanArgs a;
  int seg;        // tokens per segment, a multiple of 32
  int segments;   // that `states` and `decays` have room for
  float* states;  // (segments, C, N): the segments' own end states, then their start states
  float* decays;  // (segments, C): log2 of a segment's decay
};

constexpr int kBlock = 32, kWarps = 4, kChan = 16 * kWarps;
constexpr float kSpan = 86.f, kLog2e = 1.4426950408889634f;

struct Segment { int b, first, count, index; SeqRange seq; };  // sequence, its first segment's number, its segments, which one

// Segment number `id` over all sequences in order; b = -1 past the last.  Every warp looks by itself.
AHB_DEVICE Segment find_segment(const ScanArgs& p, int seg, int id) {
  Segment r{-1, 0, 0, 0, {0, 0}};
  if (p.cu == nullptr) {
    const int n = (p.L + seg - 1) / seg;
    if (n > 0 && id < n * p.B) {
      r.b = id / n;
      r.first = r.b * n;
      r.count = n;
      r.index = id - r.first;
      r.seq = seq_range(p.cu, r.b, p.L, p.T);
    }
    return r;
  }
  const int lane = threadIdx.x & 31;
  int base = 0;
  for (int b0 = 0; b0 < p.B; b0 += 32) {
    int n = 0;
    if (b0 + lane < p.B) {
      const SeqRange q = seq_range(p.cu, b0 + lane, p.L, p.T);
      n = (q.end - q.start + seg - 1) / seg;
    }
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
      r.seq = seq_range(p.cu, r.b, p.L, p.T);
      return r;
    }
    base += __shfl_sync(0xffffffffu, incl, 31);
  }
  return r;
}

AHB_DEVICE float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// log(1 + e^x) to about 2^-22: max(x, 0) + log1p(z) with z = e^{-|x|}, log1p(z) = 2 atanh(z / (2 + z)) as
// its power series (the argument is at most 1/3; the first term left out is below 5e-9 of the sum)
AHB_DEVICE float softplus_series(float x) {
  const float z = ex2(-fabsf(x) * kLog2e), s = __fdividef(z, 2.f + z), w = s * s;
  float p = fmaf(w, 2.f / 13.f, 2.f / 11.f);
  p = fmaf(w, p, 2.f / 9.f);
  p = fmaf(w, p, 2.f / 7.f);
  p = fmaf(w, p, 2.f / 5.f);
  p = fmaf(w, p, 2.f / 3.f);
  p = fmaf(w, p, 2.f);
  return fmaf(s, p, fmaxf(x, 0.f));
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

// the next bf16 term of two floats, which keep what it leaves
AHB_DEVICE uint32_t term2(float& x, float& y) {
  const uint32_t h = pack2(x, y);
  x -= lo16(h);
  y -= hi16(h);
  return h;
}

using bf16 = __nv_bfloat16;

// Channels c, c + 1 of a row as two bf16; `pairs`: both in one 4-byte access
AHB_DEVICE uint32_t load_pair(const bf16* row, int c, int C, bool pairs) {
  if (c >= C) return 0u;
  if (pairs) return __ldg(reinterpret_cast<const unsigned int*>(row + c));
  const uint16_t* r = reinterpret_cast<const uint16_t*>(row) + c;
  return __ldg(r) | (c + 1 < C ? (uint32_t)__ldg(r + 1) << 16 : 0u);
}
AHB_DEVICE void store_pair(bf16* row, int c, int C, bool pairs, uint32_t v) {
  if (c >= C) return;
  if (pairs) {
    *reinterpret_cast<uint32_t*>(row + c) = v;
  } else {
    uint16_t* r = reinterpret_cast<uint16_t*>(row) + c;
    r[0] = (uint16_t)v;
    if (c + 1 < C) r[1] = (uint16_t)(v >> 16);
  }
}

template <int N>
struct BlockSmem {
  static constexpr int LD = N + 8;    // row strides that spread ldmatrix rows over the banks
  static constexpr int LT = kBlock + 4;
  bf16 b[2][kBlock][LD];
  bf16 c[2][kBlock][LD];
  bf16 cb[2][kBlock][kBlock + 8];     // C B^T below the diagonal: high and low terms
  float v[kWarps][16][LT];            // a warp's V (or u) per channel and token, then its outputs
  float d[kWarps][16][LT];            // decays for a warp that goes token by token
};

// Multiplies the accumulator rows (channels) by factors that lane l holds for channels 2 (l % 8) + {0, 1}.
template <int NT>
AHB_DEVICE void scale_rows(float (*S)[4], float f0, float f1) {
  const int g = (threadIdx.x & 31) >> 2;
  const float a0 = __shfl_sync(0xffffffffu, f0, g >> 1), a1 = __shfl_sync(0xffffffffu, f1, g >> 1);
  const float b0 = __shfl_sync(0xffffffffu, f0, 4 + (g >> 1)), b1 = __shfl_sync(0xffffffffu, f1, 4 + (g >> 1));
  const float r0 = g & 1 ? a1 : a0, r1 = g & 1 ? b1 : b0;
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    S[j][0] *= r0;
    S[j][1] *= r0;
    S[j][2] *= r1;
    S[j][3] *= r1;
  }
}

template <typename W, int N, bool STATE>
__global__ void __launch_bounds__(kWarps * 32, 3) scan_block_kernel(PromptArgs pa) {
  constexpr int NT = N / 8;
  using Smem = BlockSmem<N>;
  extern __shared__ __align__(16) unsigned char raw[];
  Smem& sm = *reinterpret_cast<Smem*>(raw);
  const ScanArgs& p = pa.a;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, q = lane & 3;    // accumulator rows g, g + 8; columns 2 q, 2 q + 1
  const int i = lane & 7, tg = lane >> 3;   // channels 2 i, 2 i + 1 of tokens [8 tg, 8 tg + 8)
  const int c0 = blockIdx.y * kChan + warp * 16, ca = c0 + 2 * i;
  const Segment sg = find_segment(p, pa.seg, blockIdx.x);
  if (sg.b < 0) return;
  if (STATE && sg.index == sg.count - 1) return;  // its end state comes with its outputs
  const int slot = seq_slot(p.slots, sg.b, p.S);
  const int start = sg.seq.start + sg.index * pa.seg, end = min(start + pa.seg, sg.seq.end);
  bf16* const y = static_cast<bf16*>(p.y);
  const bf16* const x = static_cast<const bf16*>(p.x);
  const bf16* const dt = static_cast<const bf16*>(p.dt);
  const bool ypairs = (p.C & 1) == 0;
  const bool pairs = ypairs && ((p.xs | p.dts) & 1) == 0 &&
                     ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(dt) | reinterpret_cast<uintptr_t>(p.conv_state)) & 3) == 0;
  if (slot < 0) {
    if (!STATE)
      for (int t = start + tg; t < end; t += 4) store_pair(y + (int64_t)t * p.C, ca, p.C, ypairs, 0u);
    return;
  }

  float w[2][4], bias[2], A2[2];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const bool has = ca + e < p.C;
#pragma unroll
    for (int j = 0; j < 4; ++j) w[e][j] = has ? to_f(static_cast<const W*>(p.conv_w)[(int64_t)(ca + e) * 4 + j]) : 0.f;
    bias[e] = has && p.conv_b ? p.conv_b[ca + e] : 0.f;
    A2[e] = has ? p.A[(ca + e) / p.P] * kLog2e : 0.f;
  }
  // the three rows of x before the segment
  bf16* const win = static_cast<bf16*>(p.conv_state) + (int64_t)slot * 3 * p.C;
  uint32_t before[3], carry[3];
#pragma unroll
  for (int j = 0; j < 3; ++j)
    before[j] = carry[j] = sg.index == 0 ? load_pair(win + j * p.C, ca, p.C, pairs)
                                         : load_pair(x + (int64_t)(start - 3 + j) * p.xs, ca, p.C, pairs);

  float S[NT][4];
  float* const slot_state = p.state + (int64_t)slot * p.C * N;
  float* const seg_state = pa.states + (int64_t)(sg.first + sg.index) * p.C * N;
  const bool has0 = c0 + g < p.C, has1 = c0 + g + 8 < p.C;
  {
    const float* src = (sg.count == 1 ? slot_state : seg_state) + (int64_t)(c0 + g) * N + 2 * q;
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

  // block rows of B and C: every thread copies, and later clips, the same 16-byte pieces
  constexpr int PIECES = kBlock * N / 8 / (kWarps * 32);
  const bool wide = (((p.bs | p.cs) & 7) == 0) && ((reinterpret_cast<uintptr_t>(p.Bm) | reinterpret_cast<uintptr_t>(p.Cm)) & 15) == 0;
  auto copy_rows = [&](const void* from, int64_t stride, bf16 (*to)[Smem::LD], int t0) {
#pragma unroll
    for (int m = 0; m < PIECES; ++m) {
      const int piece = tid + m * kWarps * 32, row = piece / (N / 8), col = piece % (N / 8) * 8;
      const bf16* src = static_cast<const bf16*>(from) + (int64_t)(t0 + row) * stride + col;
      if (t0 + row >= end) {
        *reinterpret_cast<uint4*>(&to[row][col]) = make_uint4(0, 0, 0, 0);
      } else if (wide) {
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(&to[row][col])), "l"(src) : "memory");
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) to[row][col + k] = src[k];
      }
    }
  };
  auto clip_rows = [&](bf16 (*rows)[Smem::LD]) {
#pragma unroll
    for (int m = 0; m < PIECES; ++m) {
      const int piece = tid + m * kWarps * 32;
      uint4* at = reinterpret_cast<uint4*>(&rows[piece / (N / 8)][piece % (N / 8) * 8]);
      const uint4 r = *at;
      *at = make_uint4(clip2(r.x), clip2(r.y), clip2(r.z), clip2(r.w));
    }
  };
  auto copy_block = [&](int t0, int buf) {
    copy_rows(p.Bm, p.bs, sm.b[buf], t0);
    if (!STATE) copy_rows(p.Cm, p.cs, sm.c[buf], t0);
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  uint32_t xr[8], dr[8];
  auto load_tokens = [&](int t0) {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int t = t0 + tg * 8 + k;
      xr[k] = t < end ? load_pair(x + (int64_t)t * p.xs, ca, p.C, pairs) : 0u;
      dr[k] = t < end ? load_pair(dt + (int64_t)t * p.dts, ca, p.C, pairs) : 0u;
    }
  };

  copy_block(start, 0);
  load_tokens(start);
  float pend[2] = {0.f, 0.f}, total[2] = {0.f, 0.f};  // log2 of the scale S still lacks, of the segment's decay
  float (*const vt)[Smem::LT] = sm.v[warp];
  float (*const dl)[Smem::LT] = sm.d[warp];
  int buf = 0;
  for (int t0 = start; t0 < end; t0 += kBlock, buf ^= 1) {
    const int n = min(kBlock, end - t0);
    // convolution, step and input of this lane's channels and tokens
    float E[8][2], u[8][2];
    {
      uint32_t xs[11];
#pragma unroll
      for (int j = 0; j < 3; ++j) {
        const uint32_t last = __shfl_sync(0xffffffffu, xr[5 + j], (lane + 24) & 31);
        xs[j] = tg == 0 ? carry[j] : last;
        carry[j] = last;
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) xs[3 + k] = xr[k];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const bool in = tg * 8 + k < n;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float a = bias[e];
#pragma unroll
          for (int j = 0; j < 4; ++j) a = fmaf(w[e][j], e ? hi16(xs[k + j]) : lo16(xs[k + j]), a);
          const float xc = sanitize(__fdividef(a, 1.f + ex2(-a * kLog2e)), kClip);
          const float r = e ? hi16(dr[k]) : lo16(dr[k]);
          float step = fminf(fmaxf(softplus_series(r), p.dt_min), p.dt_max);
          step = in && r == r ? step : 0.f;
          E[k][e] = fmaxf(step * A2[e], kMinDA * kLog2e);
          u[k][e] = step * xc;
        }
      }
    }
    if (t0 + kBlock < end) load_tokens(t0 + kBlock);
    // decays summed along the tokens, over the four lanes of a channel
    float mid[2], last[2], off[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float sum = 0.f;
#pragma unroll
      for (int k = 0; k < 8; ++k) sum += E[k][e];
      float incl = sum, v = __shfl_up_sync(0xffffffffu, incl, 8);
      if (tg >= 1) incl += v;
      v = __shfl_up_sync(0xffffffffu, incl, 16);
      if (tg >= 2) incl += v;
      mid[e] = __shfl_sync(0xffffffffu, incl, 8 + i);
      last[e] = __shfl_sync(0xffffffffu, incl, 24 + i);
      off[e] = incl - sum - mid[e];
      total[e] += last[e];
    }
    const bool heavy = __any_sync(0xffffffffu, (mid[0] < -kSpan) | (mid[1] < -kSpan) | (last[0] - mid[0] < -kSpan) | (last[1] - mid[1] < -kSpan));
    __syncwarp();  // the previous block's outputs have left vt
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float v[8];
      if (heavy) {
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = E[k][e];
        *reinterpret_cast<float4*>(&dl[2 * i + e][8 * tg]) = make_float4(v[0], v[1], v[2], v[3]);
        *reinterpret_cast<float4*>(&dl[2 * i + e][8 * tg + 4]) = make_float4(v[4], v[5], v[6], v[7]);
      }
      float run = off[e];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        run += E[k][e];
        E[k][e] = run;
        v[k] = heavy ? u[k][e] : u[k][e] * ex2(-run);
      }
      *reinterpret_cast<float4*>(&vt[2 * i + e][8 * tg]) = make_float4(v[0], v[1], v[2], v[3]);
      *reinterpret_cast<float4*>(&vt[2 * i + e][8 * tg + 4]) = make_float4(v[4], v[5], v[6], v[7]);
    }
    // S takes the scale it lacks and goes to the block's reference.  S itself may stand at 2^kSpan, so the two
    // scales go in one after the other where their product would leave the floats' range.
    if (__any_sync(0xffffffffu, (pend[0] + mid[0] < -120.f) | (pend[1] + mid[1] < -120.f))) {
      scale_rows<NT>(S, ex2(pend[0]), ex2(pend[1]));
      pend[0] = pend[1] = 0.f;
    }
    scale_rows<NT>(S, ex2(pend[0] + (heavy ? 0.f : mid[0])), ex2(pend[1] + (heavy ? 0.f : mid[1])));
#pragma unroll
    for (int e = 0; e < 2; ++e) pend[e] = heavy ? 0.f : last[e] - mid[e];
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    clip_rows(sm.b[buf]);
    if (!STATE) clip_rows(sm.c[buf]);
    __syncthreads();  // the block's rows are there; every warp is done with the other buffer and with cb
    if (t0 + kBlock < end) copy_block(t0 + kBlock, buf ^ 1);

    const int mrow = lane & 15, mcol = (lane >> 4) * 8;  // ldmatrix: rows of a 16 x 16 piece, its column half
    const int xrow = (lane & 7) + (lane >> 4) * 8, xcol = ((lane >> 3) & 1) * 8;  // two 8-row halves, each with both column halves
    if (!STATE) {
      // C B^T, 16 x 16 pieces (0,0), (16,0), (16,16) by warps 0 to 2
      if (warp < 3) {
        const int tb = warp == 0 ? 0 : 16, sb = warp == 2 ? 16 : 0;
        float acc[2][4];
        zero_acc<2>(acc);
#pragma unroll
        for (int k = 0; k < N; k += 16) {
          uint32_t a[4], b[4];
          ldsm4(a, &sm.c[buf][tb + mrow][k + mcol]);
          ldsm4(b, &sm.b[buf][sb + xrow][k + xcol]);
          mma16816(acc[0], a, b);
          mma16816(acc[1], a, b + 2);
        }
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int t = tb + g + 8 * h, s = sb + 8 * j + 2 * q;
            float v0 = s <= t ? acc[j][2 * h] : 0.f, v1 = s + 1 <= t ? acc[j][2 * h + 1] : 0.f;
            *reinterpret_cast<uint32_t*>(&sm.cb[0][t][s]) = term2(v0, v1);
            *reinterpret_cast<uint32_t*>(&sm.cb[1][t][s]) = pack2(v0, v1);
          }
      }
      __syncthreads();
    } else {
      __syncwarp();
    }

    if (!heavy) {
      // V as left operands: rows are channels, columns tokens
      uint32_t vf[2][3][4];
#pragma unroll
      for (int ks = 0; ks < 2; ++ks)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          float2 v = *reinterpret_cast<const float2*>(&vt[g + (r & 1) * 8][ks * 16 + (r >> 1) * 8 + 2 * q]);
          vf[ks][0][r] = term2(v.x, v.y);
          vf[ks][1][r] = term2(v.x, v.y);
          vf[ks][2][r] = pack2(v.x, v.y);
        }
      if (!STATE) {
        float Y[4][4];
        zero_acc<4>(Y);
#pragma unroll
        for (int k = 0; k < N / 16; ++k) {  // S C^T
          uint32_t sh[4], sl[4], b[4];
          float s8[8] = {S[2 * k][0], S[2 * k][1], S[2 * k][2], S[2 * k][3], S[2 * k + 1][0], S[2 * k + 1][1], S[2 * k + 1][2], S[2 * k + 1][3]};
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            sh[r] = term2(s8[2 * r], s8[2 * r + 1]);
            sl[r] = pack2(s8[2 * r], s8[2 * r + 1]);
          }
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            ldsm4(b, &sm.c[buf][16 * h + xrow][16 * k + xcol]);
            mma16816(Y[2 * h], sh, b);
            mma16816(Y[2 * h + 1], sh, b + 2);
            mma16816(Y[2 * h], sl, b);
            mma16816(Y[2 * h + 1], sl, b + 2);
          }
        }
#pragma unroll
        for (int pc = 0; pc < 3; ++pc) {  // V (C B^T)^T, the same three pieces
          const int h = pc == 0 ? 0 : 1, ks = pc == 2 ? 1 : 0;
          uint32_t bh[4], bl[4];
          ldsm4(bh, &sm.cb[0][16 * h + xrow][16 * ks + xcol]);
          ldsm4(bl, &sm.cb[1][16 * h + xrow][16 * ks + xcol]);
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            mma16816(Y[2 * h + j], vf[ks][0], bh + 2 * j);
            mma16816(Y[2 * h + j], vf[ks][0], bl + 2 * j);
            mma16816(Y[2 * h + j], vf[ks][1], bh + 2 * j);
          }
        }
        __syncwarp();  // V has been read by every lane
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          *reinterpret_cast<float2*>(&vt[g][8 * j + 2 * q]) = make_float2(Y[j][0], Y[j][1]);
          *reinterpret_cast<float2*>(&vt[g + 8][8 * j + 2 * q]) = make_float2(Y[j][2], Y[j][3]);
        }
      }
#pragma unroll
      for (int j = 0; j < N / 16; ++j)  // S += V^T B
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
          uint32_t b[4];
          ldsm4_t(b, &sm.b[buf][16 * ks + mrow][16 * j + mcol]);
#pragma unroll
          for (int m = 0; m < 3; ++m) {
            mma16816(S[2 * j], vf[ks][m], b);
            mma16816(S[2 * j + 1], vf[ks][m], b + 2);
          }
        }
    } else {
      for (int t = 0; t < n; ++t) {
        const float a0 = ex2(dl[g][t]), a1 = ex2(dl[g + 8][t]), u0 = vt[g][t], u1 = vt[g + 8][t];
        float y0 = 0.f, y1 = 0.f;
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          const uint32_t bb = *reinterpret_cast<const uint32_t*>(&sm.b[buf][t][8 * j + 2 * q]);
          S[j][0] = fmaf(a0, S[j][0], u0 * lo16(bb));
          S[j][1] = fmaf(a0, S[j][1], u0 * hi16(bb));
          S[j][2] = fmaf(a1, S[j][2], u1 * lo16(bb));
          S[j][3] = fmaf(a1, S[j][3], u1 * hi16(bb));
          if (!STATE) {
            const uint32_t cc = *reinterpret_cast<const uint32_t*>(&sm.c[buf][t][8 * j + 2 * q]);
            y0 = fmaf(lo16(cc), S[j][0], fmaf(hi16(cc), S[j][1], y0));
            y1 = fmaf(lo16(cc), S[j][2], fmaf(hi16(cc), S[j][3], y1));
          }
        }
        if (!STATE) {
          y0 += __shfl_xor_sync(0xffffffffu, y0, 1);
          y1 += __shfl_xor_sync(0xffffffffu, y1, 1);
          y0 += __shfl_xor_sync(0xffffffffu, y0, 2);
          y1 += __shfl_xor_sync(0xffffffffu, y1, 2);
          if (q == 0) {  // the four lanes have read u there
            vt[g][t] = y0;
            vt[g + 8][t] = y1;
          }
        }
      }
    }
    if (!STATE) {
      __syncwarp();
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int t = 8 * tg + k;
        const float y0 = vt[2 * i][t], y1 = vt[2 * i + 1][t];
        if (t < n)
          store_pair(y + (int64_t)(t0 + t) * p.C, ca, p.C, ypairs, heavy ? pack2(y0, y1) : pack2(y0 * ex2(E[k][0]), y1 * ex2(E[k][1])));
      }
    }
  }

  // the end state, with the scale it lacks
  if (STATE || sg.index == sg.count - 1) {
    scale_rows<NT>(S, ex2(pend[0]), ex2(pend[1]));
    float* dst = (STATE ? seg_state : slot_state) + (int64_t)(c0 + g) * N + 2 * q;
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      if (has0) *reinterpret_cast<float2*>(dst + 8 * j) = make_float2(S[j][0], S[j][1]);
      if (has1) *reinterpret_cast<float2*>(dst + 8 * N + 8 * j) = make_float2(S[j][2], S[j][3]);
    }
    if (STATE && tg == 0) {
#pragma unroll
      for (int e = 0; e < 2; ++e)
        if (ca + e < p.C) pa.decays[(int64_t)(sg.first + sg.index) * p.C + ca + e] = total[e];
    }
  }
  // the first segment's block alone reads the window, so it may write it
  if (!STATE && sg.index == 0 && tg == 0) {
    const int len = sg.seq.end - sg.seq.start;
    uint32_t nw[3];
#pragma unroll
    for (int j = 0; j < 3; ++j) {
      const int at = len + j - 3;
      nw[j] = at >= 0 ? load_pair(x + (int64_t)(sg.seq.start + at) * p.xs, ca, p.C, pairs) : at == -2 ? before[1] : before[2];
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
  const SeqRange r = seq_range(p.cu, b, p.L, p.T);
  const int count = (r.end - r.start + pa.seg - 1) / pa.seg;
  if (count < 2) return;
  int first = b * count;
  if (p.cu != nullptr) {
    const int lane = threadIdx.x & 31;
    first = 0;
    for (int o = lane; o < b; o += 32) {
      const SeqRange q = seq_range(p.cu, o, p.L, p.T);
      first += (q.end - q.start + pa.seg - 1) / pa.seg;
    }
    first = __reduce_add_sync(0xffffffffu, first);
  }
  if (first + count > pa.segments) return;  // offsets that overlap
  const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (at >= (int64_t)p.C * (N / 4)) return;
  const int c = (int)(at / (N / 4));
  float4 run = reinterpret_cast<const float4*>(p.state + (int64_t)slot * p.C * N)[at];
  for (int s = first; s < first + count; ++s) {
    float4* seg = reinterpret_cast<float4*>(pa.states + (int64_t)s * p.C * N) + at;
    if (s == first + count - 1) {
      *seg = run;
      break;
    }
    const float4 own = *seg;
    const float f = ex2(pa.decays[(int64_t)s * p.C + c]);
    *seg = run;
    run = make_float4(fmaf(f, run.x, own.x), fmaf(f, run.y, own.y), fmaf(f, run.z, own.z), fmaf(f, run.w, own.w));
  }
}

// Segments of T tokens in B sequences: as many as any packing of them can have
int64_t max_segments(int B, int L, int T, bool packed, int seg) {
  return packed ? (int64_t)T / seg + B : (int64_t)B * ((L + seg - 1) / seg);
}

template <typename W, int N>
int launch_prompt(const ScanArgs& a, int seg, float* work, cudaStream_t st) {
  static bool ready[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev >= 64) return -3;
  const int bytes = (int)sizeof(BlockSmem<N>);
  if (!ready[dev]) {
    if (cudaFuncSetAttribute(scan_block_kernel<W, N, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess ||
        cudaFuncSetAttribute(scan_block_kernel<W, N, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess)
      return -3;
    ready[dev] = true;
  }
  const int64_t segs = max_segments(a.B, a.L, a.T, a.cu != nullptr, seg);
  const PromptArgs p{a, seg, (int)segs, work, work + segs * a.C * N};
  const dim3 grid((unsigned)segs, (unsigned)((a.C + kChan - 1) / kChan));
  if (segs > a.B) {
    scan_block_kernel<W, N, true><<<grid, kWarps * 32, bytes, st>>>(p);
    scan_join_kernel<N><<<dim3((unsigned)(((int64_t)a.C * (N / 4) + 255) / 256), (unsigned)a.B), 256, 0, st>>>(p);
  }
  scan_block_kernel<W, N, false><<<grid, kWarps * 32, bytes, st>>>(p);
  return 0;
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

int ahb_selective_scan_plan(int B, int L, int T, int C, int N, int packed, int dtype, int64_t* floats) {
  *floats = 0;
  if (dtype != AHB_BF16 || B == 0 || T < 4 * (int64_t)B) return 0;
  const int64_t groups = (C + kChan - 1) / kChan;
  int64_t seg = T * groups / (2 * 3 * 148);
  seg = std::min<int64_t>(1 << 30, std::max<int64_t>(256, (seg + kBlock - 1) / kBlock * kBlock));
  const int64_t segs = max_segments(B, L, T, packed != 0, (int)seg);
  if (segs > B) *floats = segs * C * (N + 1);
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
