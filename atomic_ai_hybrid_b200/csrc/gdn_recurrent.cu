// GDN-2's convolutions, gates and delta rule, token by token, with state carried between calls
// (serving: single tokens and a few at once; the layer's mathematics: reference `model.py:564-653`).
//
//   q, k, v = silu(conv(.)),  v clipped to +-50,  q, k divided by their norm over the head
//   beta = sigmoid(b), omega = sigmoid(w),  alpha = exp(max(-e^a softplus(f), -1e3))     per channel
//   h <- diag(alpha) h;  n = omega v - (beta k)^T h;  h <- h + k n^T;  o = q^T h         h (D, D) per head
#include "launchers.h"
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

// One block of 2 D threads per (head, sequence): thread (g, m) = (tid / (D / 4), tid % (D / 4)) keeps rows
// [g D/8, g D/8 + D/8) of columns [4 m, 4 m + 4) of the head's state in registers, so state rows move in
// 16-byte pieces, a row's four factors are one broadcast from shared memory for four columns, and the
// sums over k end in eight partial rows.  The state's loads are issued first and fly while the tokens'
// convolutions, norms and gates, which depend on no state, are made for up to TB tokens at once.
constexpr int TB = 8;

template <typename T, typename W, int D>
__global__ void __launch_bounds__(2 * D, 2) gdn_recurrent_kernel(GdnArgs p) {
  constexpr int Q = D / 4, R = D / 8, NW = D / 32;
  __shared__ float4 kk[TB][D];  // alpha, beta k, k, q of every row
  __shared__ __align__(16) float wv[TB][D];
  __shared__ float2 norms[TB][NW];
  __shared__ float4 part[2][8][Q];  // partial erase sums, partial outputs
  const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x;
  const int d = p.H * D;
  const SeqRange r = seq_range(p.cu, b, p.L, p.T);
  const int slot = seq_slot(p.slots, b, p.S);
  T* y = static_cast<T*>(p.y) + h * D;
  if (slot < 0) {
    for (int t = r.start; t < r.end; ++t)
      for (int c = tid; c < D; c += 2 * D) y[(int64_t)t * d + c] = from_f<T>(0.f);
    return;
  }
  if (r.start == r.end) return;
  const int g = tid / Q, m = tid % Q;
  float4* st = reinterpret_cast<float4*>(p.state + ((int64_t)slot * p.H + h) * D * D) + g * R * Q + m;
  float4 s[R];
#pragma unroll
  for (int i = 0; i < R; ++i) s[i] = st[i * Q];

  // channel c of the tokens of one parity
  const int c = tid % D, half = tid / D, ch = h * D + c;
  const int len = r.end - r.start;
  const float ea = __expf(fminf(fmaxf(p.decay_a[h], -20.f), 20.f));
  T* cs = static_cast<T*>(p.conv_state) + (int64_t)slot * 9 * d + ch;
  float win[3][3], cw[3][4], cb[3];
#pragma unroll
  for (int e = 0; e < 3; ++e) {
    load_taps(cw[e], static_cast<const W*>(p.conv_w[e]) + (int64_t)ch * 4);
    cb[e] = p.conv_b[e] ? p.conv_b[e][ch] : 0.f;
#pragma unroll
    for (int j = 0; j < 3; ++j) win[e][j] = to_f(cs[(e * 3 + j) * d]);
  }
  // row `i` of the sequence preceded by its window, -3 .. len - 1
  auto input = [&](int e, int i) {
    if (i >= 0) return to_f(static_cast<const T*>(p.in[e])[(int64_t)(r.start + i) * p.rs[e] + ch]);
    return i == -3 ? win[e][0] : i == -2 ? win[e][1] : win[e][2];
  };

  for (int t0 = 0; t0 < len; t0 += TB) {
    const int n = min(TB, len - t0);
    if (t0) __syncthreads();  // the previous tokens' factors have been read
    for (int t = half; t < n; t += 2) {
      float qkv[3];
#pragma unroll
      for (int e = 0; e < 3; ++e)
        qkv[e] = conv_silu(cw[e], cb[e], input(e, t0 + t - 3), input(e, t0 + t - 2), input(e, t0 + t - 1), input(e, t0 + t));
      float gate[3];
#pragma unroll
      for (int e = 0; e < 3; ++e) gate[e] = to_f(static_cast<const T*>(p.in[3 + e])[(int64_t)(r.start + t0 + t) * p.rs[3 + e] + ch]);
      const float sq = warp_sum(qkv[0] * qkv[0]), sk = warp_sum(qkv[1] * qkv[1]);
      if ((tid & 31) == 0) norms[t][c >> 5] = make_float2(sq, sk);
      float lg = -ea * softplusf_(gate[2]);
      lg = lg != lg ? 0.f : fmaxf(lg, -1e3f);
      kk[t][c] = make_float4(exp_decay(lg), sanitize(sigmoidf_(gate[0]), 1.f), qkv[1], qkv[0]);
      wv[t][c] = sanitize(sigmoidf_(gate[1]), 1.f) * sanitize(qkv[2], 50.f);
    }
    __syncthreads();
    for (int t = half; t < n; t += 2) {
      float sq = 0.f, sk = 0.f;
#pragma unroll
      for (int i = 0; i < NW; ++i) {
        const float2 a = norms[t][i];
        sq += a.x;
        sk += a.y;
      }
      float4 f = kk[t][c];
      f.z = sanitize(f.z * rsqrtf(sk + 1e-12f), 1e3f);
      f.w = sanitize(f.w * rsqrtf(sq + 1e-12f), 1e3f);
      f.y *= f.z;
      kk[t][c] = f;
    }
    __syncthreads();
    for (int t = 0; t < n; ++t) {
      float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int i = 0; i < R; ++i) {
        const float2 f = *reinterpret_cast<const float2*>(&kk[t][g * R + i]);
        s[i].x *= f.x;
        s[i].y *= f.x;
        s[i].z *= f.x;
        s[i].w *= f.x;
        a.x = fmaf(f.y, s[i].x, a.x);
        a.y = fmaf(f.y, s[i].y, a.y);
        a.z = fmaf(f.y, s[i].z, a.z);
        a.w = fmaf(f.y, s[i].w, a.w);
      }
      part[0][g][m] = a;
      __syncthreads();
      float4 nv = reinterpret_cast<const float4*>(wv[t])[m];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        a = part[0][i][m];
        nv.x -= a.x;
        nv.y -= a.y;
        nv.z -= a.z;
        nv.w -= a.w;
      }
      a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int i = 0; i < R; ++i) {
        const float2 f = *(reinterpret_cast<const float2*>(&kk[t][g * R + i]) + 1);
        s[i].x = fmaf(f.x, nv.x, s[i].x);
        s[i].y = fmaf(f.x, nv.y, s[i].y);
        s[i].z = fmaf(f.x, nv.z, s[i].z);
        s[i].w = fmaf(f.x, nv.w, s[i].w);
        a.x = fmaf(f.y, s[i].x, a.x);
        a.y = fmaf(f.y, s[i].y, a.y);
        a.z = fmaf(f.y, s[i].z, a.z);
        a.w = fmaf(f.y, s[i].w, a.w);
      }
      part[1][g][m] = a;
      __syncthreads();
      if (tid < D) {
        float o = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) o += reinterpret_cast<const float*>(part[1][i])[tid];
        y[(int64_t)(r.start + t0 + t) * d + tid] = from_f<T>(o);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < R; ++i) st[i * Q] = s[i];
  if (half == 0) {
#pragma unroll
    for (int e = 0; e < 3; ++e) {
      float last[3];
#pragma unroll
      for (int j = 0; j < 3; ++j) last[j] = input(e, len - 3 + j);
#pragma unroll
      for (int j = 0; j < 3; ++j) cs[(e * 3 + j) * d] = from_f<T>(last[j]);
    }
  }
}

template <typename T, typename W>
int by_head(const GdnArgs& p, int D, cudaStream_t st) {
  const dim3 grid(p.H, p.B);
  if (D == 128) gdn_recurrent_kernel<T, W, 128><<<grid, 256, 0, st>>>(p);
  else if (D == 96) gdn_recurrent_kernel<T, W, 96><<<grid, 192, 0, st>>>(p);
  else if (D == 64) gdn_recurrent_kernel<T, W, 64><<<grid, 128, 0, st>>>(p);
  else return -1;
  return 0;
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
