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

// One block per (head, sequence).  A warp holds 8 VC columns of the head's state in registers: lane
// (g, m) = (lane / 8, lane % 8) has rows k = 4 i + g of columns [VC m, VC m + VC), so a state row is
// read in 32 VC-byte pieces and both sums over k end in two shuffles.
template <typename T, typename W, int D, int VC>
__global__ void __launch_bounds__(D / (8 * VC) * 32, 1) gdn_recurrent_kernel(GdnArgs p) {
  constexpr int NT = D / (8 * VC) * 32, R = D / 4;
  __shared__ float4 kk[D];  // alpha, beta k, k, q of every row
  __shared__ float wv[D];
  __shared__ float red[2 * (NT / 32)];
  const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
  const int d = p.H * D;
  const SeqRange r = seq_range(p.cu, b, p.L, p.T);
  const int slot = seq_slot(p.slots, b, p.S);
  T* y = static_cast<T*>(p.y);
  if (slot < 0) {
    for (int t = r.start; t < r.end; ++t)
      for (int c = tid; c < D; c += NT) y[(int64_t)t * d + h * D + c] = from_f<T>(0.f);
    return;
  }
  if (r.start == r.end) return;
  const int g = lane >> 3, col = wid * 8 * VC + (lane & 7) * VC;
  float* st = p.state + ((int64_t)slot * p.H + h) * D * D + col;
  float s[R][VC];
#pragma unroll
  for (int i = 0; i < R; ++i)
#pragma unroll
    for (int j = 0; j < VC; ++j) s[i][j] = st[(4 * i + g) * D + j];

  // channel threads: NT may be under or over D, each handles its channels in turn
  constexpr int PER = (D + NT - 1) / NT;
  float win[PER][3][3], cw[PER][3][4], cb[PER][3];
  const float ea = __expf(fminf(fmaxf(p.decay_a[h], -20.f), 20.f));
  T* cs = static_cast<T*>(p.conv_state) + (int64_t)slot * 9 * d + h * D;
#pragma unroll
  for (int e = 0; e < PER; ++e) {
    const int c = tid + e * NT;
    if (c < D) {
#pragma unroll
      for (int m = 0; m < 3; ++m) {
        load_taps(cw[e][m], static_cast<const W*>(p.conv_w[m]) + (int64_t)(h * D + c) * 4);
        cb[e][m] = p.conv_b[m] ? p.conv_b[m][h * D + c] : 0.f;
#pragma unroll
        for (int j = 0; j < 3; ++j) win[e][m][j] = to_f(cs[(m * 3 + j) * d + c]);
      }
    }
  }
  for (int t = r.start; t < r.end; ++t) {
    float qkv[PER][3], gate[PER][3], sq = 0.f, sk = 0.f;
#pragma unroll
    for (int e = 0; e < PER; ++e) {
      const int c = tid + e * NT;
      if (c < D) {
#pragma unroll
        for (int m = 0; m < 3; ++m) {
          const float xn = to_f(static_cast<const T*>(p.in[m])[(int64_t)t * p.rs[m] + h * D + c]);
          qkv[e][m] = conv_silu(cw[e][m], cb[e][m], win[e][m][0], win[e][m][1], win[e][m][2], xn);
          win[e][m][0] = win[e][m][1];
          win[e][m][1] = win[e][m][2];
          win[e][m][2] = xn;
          gate[e][m] = to_f(static_cast<const T*>(p.in[3 + m])[(int64_t)t * p.rs[3 + m] + h * D + c]);
        }
        sq = fmaf(qkv[e][0], qkv[e][0], sq);
        sk = fmaf(qkv[e][1], qkv[e][1], sk);
      }
    }
    sq = warp_sum(sq);
    sk = warp_sum(sk);
    if (lane == 0) {
      red[2 * wid] = sq;
      red[2 * wid + 1] = sk;
    }
    __syncthreads();
    sq = sk = 0.f;
#pragma unroll
    for (int i = 0; i < NT / 32; ++i) {
      sq += red[2 * i];
      sk += red[2 * i + 1];
    }
    const float rq = rsqrtf(sq + 1e-12f), rk = rsqrtf(sk + 1e-12f);
#pragma unroll
    for (int e = 0; e < PER; ++e) {
      const int c = tid + e * NT;
      if (c < D) {
        const float q = sanitize(qkv[e][0] * rq, 1e3f), k = sanitize(qkv[e][1] * rk, 1e3f);
        const float v = sanitize(qkv[e][2], 50.f);
        float lg = -ea * softplusf_(gate[e][2]);
        lg = lg != lg ? 0.f : fmaxf(lg, -1e3f);
        kk[c] = make_float4(exp_decay(lg), sanitize(sigmoidf_(gate[e][0]), 1.f) * k, k, q);
        wv[c] = sanitize(sigmoidf_(gate[e][1]), 1.f) * v;
      }
    }
    __syncthreads();
    float er[VC];
#pragma unroll
    for (int j = 0; j < VC; ++j) er[j] = 0.f;
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const float2 ab = *reinterpret_cast<const float2*>(&kk[4 * i + g]);
#pragma unroll
      for (int j = 0; j < VC; ++j) {
        s[i][j] *= ab.x;
        er[j] = fmaf(ab.y, s[i][j], er[j]);
      }
    }
    float o[VC];
#pragma unroll
    for (int j = 0; j < VC; ++j) {
      er[j] += __shfl_xor_sync(0xffffffffu, er[j], 8);
      er[j] += __shfl_xor_sync(0xffffffffu, er[j], 16);
      er[j] = wv[col + j] - er[j];
      o[j] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const float2 kq = *(reinterpret_cast<const float2*>(&kk[4 * i + g]) + 1);
#pragma unroll
      for (int j = 0; j < VC; ++j) {
        s[i][j] = fmaf(kq.x, er[j], s[i][j]);
        o[j] = fmaf(kq.y, s[i][j], o[j]);
      }
    }
#pragma unroll
    for (int j = 0; j < VC; ++j) {
      o[j] += __shfl_xor_sync(0xffffffffu, o[j], 8);
      o[j] += __shfl_xor_sync(0xffffffffu, o[j], 16);
      if (g == 0) y[(int64_t)t * d + h * D + col + j] = from_f<T>(o[j]);
    }
    __syncthreads();  // kk / wv / red are rewritten for the next token
  }
#pragma unroll
  for (int i = 0; i < R; ++i)
#pragma unroll
    for (int j = 0; j < VC; ++j) st[(4 * i + g) * D + j] = s[i][j];
#pragma unroll
  for (int e = 0; e < PER; ++e) {
    const int c = tid + e * NT;
    if (c < D) {
#pragma unroll
      for (int m = 0; m < 3; ++m)
#pragma unroll
        for (int j = 0; j < 3; ++j) cs[(m * 3 + j) * d + c] = from_f<T>(win[e][m][j]);
    }
  }
}

template <typename T, typename W>
int by_head(const GdnArgs& p, int D, cudaStream_t st) {
  const dim3 grid(p.H, p.B);
  if (D == 128) gdn_recurrent_kernel<T, W, 128, 1><<<grid, 512, 0, st>>>(p);
  else if (D == 96) gdn_recurrent_kernel<T, W, 96, 1><<<grid, 384, 0, st>>>(p);
  else if (D == 64) gdn_recurrent_kernel<T, W, 64, 1><<<grid, 256, 0, st>>>(p);
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
