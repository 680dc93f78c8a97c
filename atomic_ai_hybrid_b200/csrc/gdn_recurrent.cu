// GDN-2's convolutions, gates and delta rule, token by token, with state carried between calls
// (serving: single tokens and a few at once; the layer's mathematics: reference `model.py:564-653`).
//
//   q, k, v = silu(conv(.)),  v clipped to +-50,  q, k divided by their norm over the head
//   beta = sigmoid(b), omega = sigmoid(w),  alpha = exp(max(-e^a softplus(f), -1e3))     per channel
//   h <- diag(alpha) h;  n = omega v - (beta k)^T h;  h <- h + k n^T;  o = q^T h         h (D, D) per head
#include "launchers.h"
#include "packed.cuh"
#include "recurrent.cuh"

namespace {
using namespace ahb;

struct GdnArgs {
  const void* in[6];  // q, k, v, b, w, f pre-activations
  int64_t rs[6];      // row strides in elements
  const void* conv_w[3];
  const float* conv_b[3];
  const float* decay_a;
  void* conv_state;  // (S, 3, 3, d)
  float* state;      // (S, H, D, D)
  const int *cu, *slots;
  void* y;
  int B, L, T, H, S;
};

// Both kernels: one block of 2 D threads per (head, sequence).  Thread (g, m) = (tid / (D / 4), tid % (D / 4))
// has rows [g D/8, g D/8 + D/8) of columns [4 m, 4 m + 4) of the head's state, so state rows move in 16-byte
// pieces, a row's factors are one broadcast from shared memory for four columns, and sums over k end in
// eight partial rows.  With n = omega v - (beta k)^T alpha h the output is
//   o = q^T (alpha h + k n^T) = q^T alpha h + (q . k) n
// so one sweep over the state gives both sums, and the rank-1 update needs no sum after it.

// The normalised factors of a token's channel
AHB_DEVICE float unit(float x, float sumsq) { return sanitize(x * rsqrtf(sumsq + 1e-12f), 1e3f); }
AHB_DEVICE float decay_of(float rate, float f) {
  const float lg = -rate * softplusf_(f);
  return exp_decay(lg != lg ? 0.f : fmaxf(lg, -1e3f));
}
AHB_DEVICE float rate_of(float a) { return __expf(fminf(fmaxf(a, -20.f), 20.f)); }
AHB_DEVICE float gate_of(float x) { return sanitize(sigmoidf_(x), 1.f); }

// One channel of one of the three convolutions: its taps and the rows before the call
struct Channel {
  float w[4], bias, win[3];
  template <typename T, typename W>
  AHB_DEVICE void load(const GdnArgs& p, int e, int ch, int d, const T* cs) {
    load_taps(w, static_cast<const W*>(p.conv_w[e]) + (int64_t)ch * 4);
    bias = p.conv_b[e] ? p.conv_b[e][ch] : 0.f;
#pragma unroll
    for (int j = 0; j < 3; ++j) win[j] = to_f(cs[(e * 3 + j) * d]);
  }
};

AHB_DEVICE float2 lo2(const float4& v) { return make_float2(v.x, v.y); }
AHB_DEVICE float2 hi2(const float4& v) { return make_float2(v.z, v.w); }
AHB_DEVICE float4 join(float2 a, float2 b) { return make_float4(a.x, a.y, b.x, b.y); }
AHB_DEVICE float4 operator*(const float4& a, float b) { return join(mul2(lo2(a), both(b)), mul2(hi2(a), both(b))); }
AHB_DEVICE float4 fma4(float a, const float4& b, const float4& c) {
  return join(fma2(both(a), lo2(b), lo2(c)), fma2(both(a), hi2(b), hi2(c)));
}
AHB_DEVICE float4 operator+(const float4& a, const float4& b) { return join(add2(lo2(a), lo2(b)), add2(hi2(a), hi2(b))); }

template <typename T>
AHB_DEVICE void store4(T* p, const float4& v) {
  p[0] = from_f<T>(v.x);
  p[1] = from_f<T>(v.y);
  p[2] = from_f<T>(v.z);
  p[3] = from_f<T>(v.w);
}

// ---------------------------------------------------------------- one token per sequence
// Bound by the state's bytes.  The state waits in shared memory (asynchronous copies, 64 KB at D = 128), not
// in registers, so that three blocks share an SM and one's arithmetic hides behind the others' copies: 128
// sequences of 16 heads take 55 us, 0.78 of the copy rate (72 us from registers with two blocks an SM).  One
// sequence: 5.5 us, its 16 blocks' chain of loads, sums and stores.
template <typename T, typename W, int D>
__global__ void __launch_bounds__(2 * D, 3) gdn_token_kernel(GdnArgs p) {
  constexpr int Q = D / 4, R = D / 8, NW = D / 32;
  extern __shared__ __align__(16) float4 state[];  // [R][2 D]: row i of every thread
  __shared__ float4 kk[D];                         // alpha, beta k, k, q of every row
  __shared__ __align__(16) float wv[D];
  __shared__ float norms[2][NW], dots[NW];
  __shared__ float4 part[2][8][Q];                 // partial erase sums, partial outputs
  float (*raw)[D] = reinterpret_cast<float (*)[D]>(part);  // before them: q and k not yet normalised
  const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, d = p.H * D;
  const int slot = seq_slot(p.slots, b, p.S);
  T* y = static_cast<T*>(p.y) + (int64_t)b * d + h * D;
  if (slot < 0) {
    if (tid < D) y[tid] = from_f<T>(0.f);
    return;
  }
  const int g = tid / Q, m = tid % Q;
  float4* st = reinterpret_cast<float4*>(p.state + ((int64_t)slot * p.H + h) * D * D) + g * R * Q + m;
#pragma unroll
  for (int i = 0; i < R; ++i)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(&state[i * 2 * D + tid])), "l"(st + i * Q) : "memory");
  asm volatile("cp.async.commit_group;" ::: "memory");

  // threads below D: q, v and the write gate of channel c; the others: k, the erase gate and the decay
  const int half = tid / D, c = tid - half * D, ch = h * D + c;
  T* cs = static_cast<T*>(p.conv_state) + (int64_t)slot * 9 * d + ch;
  auto in = [&](int e) { return to_f(static_cast<const T*>(p.in[e])[(int64_t)b * p.rs[e] + ch]); };
  Channel a, v;
  a.template load<T, W>(p, half, ch, d, cs);
  const float xa = in(half), gate = in(half ? 3 : 4);
  float xv = 0.f, f = 0.f, rate = 0.f;
  if (half == 0) {
    v.template load<T, W>(p, 2, ch, d, cs);
    xv = in(2);
  } else {
    f = in(5);
    rate = rate_of(p.decay_a[h]);
  }
  const float qk = conv_silu(a.w, a.bias, a.win[0], a.win[1], a.win[2], xa);
  const float sum = warp_sum(qk * qk);
  raw[half][c] = qk;
  if ((tid & 31) == 0) norms[half][c >> 5] = sum;
  float alpha = 0.f;
  if (half == 0)
    wv[c] = gate_of(gate) * sanitize(conv_silu(v.w, v.bias, v.win[0], v.win[1], v.win[2], xv), 50.f);
  else
    alpha = decay_of(rate, f);
  __syncthreads();
  float sq = 0.f, sk = 0.f;
#pragma unroll
  for (int i = 0; i < NW; ++i) {
    sq += norms[0][i];
    sk += norms[1][i];
  }
  const float k = unit(raw[1][c], sk);
  if (half == 0) {
    const float q = unit(qk, sq), dot = warp_sum(q * k);
    kk[c].w = q;
    if ((tid & 31) == 0) dots[c >> 5] = dot;
  } else {
    kk[c].x = alpha;
    kk[c].y = gate_of(gate) * k;
    kk[c].z = k;
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");  // a thread reads only what it copied
  __syncthreads();
  float4 er = make_float4(0.f, 0.f, 0.f, 0.f), o = er;
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const float4 r = kk[g * R + i], s = state[i * 2 * D + tid] * r.x;
    er = fma4(r.y, s, er);
    o = fma4(r.w, s, o);
  }
  part[0][g][m] = er;
  part[1][g][m] = o;
  __syncthreads();
  float4 n = reinterpret_cast<const float4*>(wv)[m];
#pragma unroll
  for (int i = 0; i < 8; ++i) n = n + part[0][i][m] * -1.f;
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const float4 r = kk[g * R + i];
    __stcs(st + i * Q, fma4(r.z, n, state[i * 2 * D + tid] * r.x));
  }
  if (g == 0) {
    float dot = 0.f;
#pragma unroll
    for (int i = 0; i < NW; ++i) dot += dots[i];
    o = n * dot;
#pragma unroll
    for (int i = 0; i < 8; ++i) o = o + part[1][i][m];
    store4(y + 4 * m, o);
  }
  // the windows move on by one row
  cs[half * 3 * d] = from_f<T>(a.win[1]);
  cs[(half * 3 + 1) * d] = from_f<T>(a.win[2]);
  cs[(half * 3 + 2) * d] = from_f<T>(xa);
  if (half == 0) {
    cs[6 * d] = from_f<T>(v.win[1]);
    cs[7 * d] = from_f<T>(v.win[2]);
    cs[8 * d] = from_f<T>(xv);
  }
}

// ---------------------------------------------------------------- a few tokens per sequence
// The state stays in registers from token to token.  The tokens' convolutions, norms and gates depend on
// no state and are made for up to TB tokens at once while the state is on its way; then each token costs one
// sweep (the last token's update, this one's decay and both sums) and one barrier.  16 sequences of 1 to 8 tokens,
// 6 heads: 14.2 us, the dependent sweeps (1.1 us each) of 96 blocks.
constexpr int TB = 8;

template <typename T, typename W, int D>
__global__ void __launch_bounds__(2 * D, 2) gdn_tokens_kernel(GdnArgs p) {
  constexpr int Q = D / 4, R = D / 8, NW = D / 32;
  extern __shared__ __align__(16) float4 state[];  // [R][2 D]: row i of every thread, on its way to registers
  __shared__ float4 kk[TB][D];                     // alpha, beta k, k, q of every row
  __shared__ __align__(16) float wv[TB][D];
  __shared__ float norms[2][TB][NW], dots[TB][NW];
  __shared__ float4 part[2][2][8][Q];  // by parity of the token: partial erase sums and outputs
  const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, d = p.H * D;
  const SeqRange r = seq_range(p.cu, b, p.L, p.T);
  const int slot = seq_slot(p.slots, b, p.S);
  T* y = static_cast<T*>(p.y) + h * D;
  auto clear_open = [&] {  // last, when nothing of the recurrence is held: 0.4 us of 15 (0.5 to 2 us at other places)
    if (p.cu == nullptr || tid >= D) return;
    const OpenRows open(p.cu, p.B, p.T);
    for (int i = b; i < open.count; i += p.B) y[(int64_t)open.row(i) * d + tid] = from_f<T>(0.f);
  };
  if (slot < 0 || r.start == r.end) {
    for (int t = r.start; t < r.end; ++t)
      if (tid < D) y[(int64_t)t * d + tid] = from_f<T>(0.f);
    clear_open();
    return;
  }
  const int g = tid / Q, m = tid % Q;
  float4* st = reinterpret_cast<float4*>(p.state + ((int64_t)slot * p.H + h) * D * D) + g * R * Q + m;
#pragma unroll
  for (int i = 0; i < R; ++i)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(&state[i * 2 * D + tid])), "l"(st + i * Q) : "memory");
  asm volatile("cp.async.commit_group;" ::: "memory");

  // threads below D: q, v and the write gate of channel c; the others: k, the erase gate and the decay
  const int half = tid / D, c = tid - half * D, ch = h * D + c, len = r.end - r.start;
  T* cs = static_cast<T*>(p.conv_state) + (int64_t)slot * 9 * d + ch;
  auto in = [&](int e, int t) { return to_f(static_cast<const T*>(p.in[e])[(int64_t)(r.start + t) * p.rs[e] + ch]); };
  // row t of convolution e, the window's for t < 0
  auto seen = [&](int e, int t) { return t >= 0 ? in(e, t) : to_f(cs[(e * 3 + 3 + t) * d]); };

  float4 s[R], n = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int t0 = 0; t0 < len; t0 += TB) {
    const int cnt = min(TB, len - t0);
    // the channel's parameters are read again every TB tokens rather than held beside the state
    Channel a, v;
    a.template load<T, W>(p, half, ch, d, cs);
    if (half == 0) v.template load<T, W>(p, 2, ch, d, cs);
    if (t0) {
#pragma unroll
      for (int j = 0; j < 3; ++j) {
        a.win[j] = in(half, t0 - 3 + j);
        if (half == 0) v.win[j] = in(2, t0 - 3 + j);
      }
    }
    const float rate = rate_of(p.decay_a[h]);
    float qk[TB], gate[TB], other[TB];  // all on their way together; past the last token its values again
#pragma unroll
    for (int t = 0; t < TB; ++t) {
      const int at = t0 + min(t, cnt - 1);
      qk[t] = in(half, at);
      gate[t] = in(half ? 3 : 4, at);
      other[t] = in(half ? 5 : 2, at);
    }
#pragma unroll
    for (int t = 0; t < TB; ++t)
      if (t < cnt) {
        const float x = qk[t];
        qk[t] = conv_silu(a.w, a.bias, a.win[0], a.win[1], a.win[2], x);
        a.win[0] = a.win[1];
        a.win[1] = a.win[2];
        a.win[2] = x;
        gate[t] = gate_of(gate[t]);
        if (half == 0) {
          wv[t][c] = gate[t] * sanitize(conv_silu(v.w, v.bias, v.win[0], v.win[1], v.win[2], other[t]), 50.f);
          v.win[0] = v.win[1];
          v.win[1] = v.win[2];
          v.win[2] = other[t];
        } else {
          kk[t][c].x = decay_of(rate, other[t]);
          kk[t][c].z = qk[t];
        }
        const float sum = warp_sum(qk[t] * qk[t]);
        if ((tid & 31) == 0) norms[half][t][c >> 5] = sum;
      }
    __syncthreads();
#pragma unroll
    for (int t = 0; t < TB; ++t)
      if (t < cnt) {
        float sq = 0.f, sk = 0.f;
#pragma unroll
        for (int i = 0; i < NW; ++i) {
          sq += norms[0][t][i];
          sk += norms[1][t][i];
        }
        if (half == 0) {
          const float q = unit(qk[t], sq), dot = warp_sum(q * unit(kk[t][c].z, sk));
          kk[t][c].w = q;
          if ((tid & 31) == 0) dots[t][c >> 5] = dot;
        } else {
          qk[t] = unit(qk[t], sk);
          kk[t][c].y = gate[t] * qk[t];
        }
      }
    __syncthreads();  // the raw k have been read
    if (half == 1) {
#pragma unroll
      for (int t = 0; t < TB; ++t)
        if (t < cnt) kk[t][c].z = qk[t];
    }
    if (t0 == 0) {
      asm volatile("cp.async.wait_group 0;" ::: "memory");  // a thread reads only what it copied
#pragma unroll
      for (int i = 0; i < R; ++i) s[i] = state[i * 2 * D + tid];
    }
    __syncthreads();
    for (int t = 0; t < cnt; ++t) {
      float4 er = make_float4(0.f, 0.f, 0.f, 0.f), o = er;
#pragma unroll
      for (int i = 0; i < R; ++i) {
        const float4 f = kk[t][g * R + i];
        if (t) s[i] = fma4(kk[t - 1][g * R + i].z, n, s[i]);
        s[i] = s[i] * f.x;
        er = fma4(f.y, s[i], er);
        o = fma4(f.w, s[i], o);
      }
      part[t & 1][0][g][m] = er;
      part[t & 1][1][g][m] = o;
      __syncthreads();
      n = reinterpret_cast<const float4*>(wv[t])[m];
#pragma unroll
      for (int i = 0; i < 8; ++i) n = n + part[t & 1][0][i][m] * -1.f;
      if (g == (t & 7)) {  // one group of threads a token adds the output up
        float dot = 0.f;
#pragma unroll
        for (int i = 0; i < NW; ++i) dot += dots[t][i];
        o = n * dot;
#pragma unroll
        for (int i = 0; i < 8; ++i) o = o + part[t & 1][1][i][m];
        store4(y + (int64_t)(r.start + t0 + t) * d + 4 * m, o);
      }
    }
#pragma unroll
    for (int i = 0; i < R; ++i) s[i] = fma4(kk[cnt - 1][g * R + i].z, n, s[i]);
    __syncthreads();  // the next tokens' factors take these ones' places
  }
#pragma unroll
  for (int i = 0; i < R; ++i) st[i * Q] = s[i];
  float wa[3], wv3[3];
#pragma unroll
  for (int j = 0; j < 3; ++j) {
    wa[j] = seen(half, len - 3 + j);
    wv3[j] = half == 0 ? seen(2, len - 3 + j) : 0.f;
  }
#pragma unroll
  for (int j = 0; j < 3; ++j) {
    cs[(half * 3 + j) * d] = from_f<T>(wa[j]);
    if (half == 0) cs[(6 + j) * d] = from_f<T>(wv3[j]);
  }
  clear_open();
}

template <typename T, typename W, int D>
int launch(const GdnArgs& p, cudaStream_t st) {
  constexpr int bytes = D * D * 4;
  static bool ready[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev >= 64) return -3;
  if (!ready[dev]) {
    if (cudaFuncSetAttribute(gdn_token_kernel<T, W, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess ||
        cudaFuncSetAttribute(gdn_tokens_kernel<T, W, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess)
      return -3;
    ready[dev] = true;
  }
  if (p.cu == nullptr && p.L == 1)
    gdn_token_kernel<T, W, D><<<dim3(p.H, p.B), 2 * D, bytes, st>>>(p);
  else
    gdn_tokens_kernel<T, W, D><<<dim3(p.H, p.B), 2 * D, bytes, st>>>(p);
  return 0;
}

template <typename T, typename W>
int by_head(const GdnArgs& p, int D, cudaStream_t st) {
  if (D == 128) return launch<T, W, 128>(p, st);
  if (D == 96) return launch<T, W, 96>(p, st);
  if (D == 64) return launch<T, W, 64>(p, st);
  return -1;
}

}  // namespace

int ahb_gdn_recurrent(const void* const in[6], const int64_t rs[6], const void* const conv_w[3], int wdtype,
                      const float* const conv_b[3], const float* decay_a, void* conv_state, float* state,
                      const int* cu, const int* slots, void* y, int B, int L, int T, int H, int D, int S, int dtype,
                      cudaStream_t st) {
  if (T == 0 || B == 0) return 0;
  if (B > 65535) return -2;
  GdnArgs p{};
  for (int i = 0; i < 6; ++i) {
    p.in[i] = in[i];
    p.rs[i] = rs[i];
  }
  for (int i = 0; i < 3; ++i) {
    p.conv_w[i] = conv_w[i];
    p.conv_b[i] = conv_b[i];
  }
  p.decay_a = decay_a;
  p.conv_state = conv_state;
  p.state = state;
  p.cu = cu;
  p.slots = slots;
  p.y = y;
  p.B = B;
  p.L = L;
  p.T = T;
  p.H = H;
  p.S = S;
  const bool wb = wdtype == AHB_BF16;
  if (dtype == AHB_BF16)
    return wb ? by_head<__nv_bfloat16, __nv_bfloat16>(p, D, st) : by_head<__nv_bfloat16, float>(p, D, st);
  return wb ? by_head<float, __nv_bfloat16>(p, D, st) : by_head<float, float>(p, D, st);
}
