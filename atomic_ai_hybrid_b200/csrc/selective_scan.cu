// Mamba2's short causal convolution and selective scan with state carried between calls (prompts of
// any length and single tokens), for serving (the layer's mathematics: reference `model.py:391-525`).
//
//   xc_t = sanitize(silu(sum_j w_j x_{t-3+j} + b)),  dt_t = clamp(softplus(dtraw_t), dt_min, dt_max)
//   S_t[c,:] = e^{max(dt_t A_h, -20)} S_{t-1}[c,:] + dt_t xc_t B_t ,   y_t[c] = <C_t, S_t[c,:]>
#include "launchers.h"
#include "recurrent.cuh"

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

template <typename T, typename W>
int by_state(const ScanArgs& p, int N, cudaStream_t st) {
  if (N == 128) launch_token<T, W, 128>(p, st);
  else if (N == 64) launch_token<T, W, 64>(p, st);
  else if (N == 32) launch_token<T, W, 32>(p, st);
  else return -1;
  return 0;
}

}  // namespace

int ahb_selective_scan(const void* x, int64_t xs, const void* dt, int64_t dts, const float* A, const void* Bm,
                       int64_t bs, const void* Cm, int64_t cs, const void* conv_w, int wdtype, const float* conv_b,
                       void* conv_state, float* state, const int* cu, const int* slots, void* y, int B, int L, int T,
                       int C, int P, int N, int S, int dtype, float dt_min, float dt_max, cudaStream_t st) {
  if (T == 0 || B == 0) return 0;
  if (B > 65535) return -2;
  const ScanArgs p{x, dt, Bm, Cm, conv_w, xs, dts, bs, cs, A, conv_b, conv_state, state, cu, slots, y,
                   B, L, T, C, P, S, dt_min, dt_max};
  const bool wb = wdtype == AHB_BF16;
  if (dtype == AHB_BF16)
    return wb ? by_state<__nv_bfloat16, __nv_bfloat16>(p, N, st) : by_state<__nv_bfloat16, float>(p, N, st);
  return wb ? by_state<float, __nv_bfloat16>(p, N, st) : by_state<float, float>(p, N, st);
}
