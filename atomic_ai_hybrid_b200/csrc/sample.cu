// The next token of every row from its logits and given Exp(1) noise, with temperature, top-k, top-p
// and min-p per row (the reference has no sampler).
//
// With d_i = (max l - l_i) / T and m_i = e^{-d_i}, tokens are ranked by (logit descending, index
// ascending).  A token is kept if its rank is below top_k, the mass ranked before it is below
// top_p sum m (rank 0 always), and m_i >= min_p; each rule looks at the whole tempered row, so their
// order does not matter.  The token is argmax over the kept ones of -d_i - log q_i, which picks i with
// probability m_i over the kept mass; logprob = -d_i - log sum m.
//
// No sort: the kept tokens are a prefix of the ranking, so if the winner of the race over some longer
// prefix is kept, it is the winner over the kept tokens; if not, nothing ranked after it is kept either
// and the race is run again over what is ranked before it.  The first prefix comes from a histogram
// of d in 512 bins (counts only: integer atomics, so no result depends on their order): a bin is left out
// when the counts before it reach top_k, or when the least mass they can stand for reaches top_p.  What
// remains is the kept tokens and at most a bin more, so one race is nearly always enough, and
// noise is read for these tokens alone.
//
// A row is split over a cluster of 1 to 8 CTAs which keep it in shared memory (as loaded, NaN and
// infinities replaced), so the logits leave HBM once; partial results meet through distributed shared
// memory and every CTA combines them in the same order.
#include "launchers.h"
#include "common.cuh"
#include "sm100.cuh"
#include <cfloat>
#include <climits>

namespace {
using namespace ahb;
using namespace ahb::sm100;

struct SampleArgs {
  const void* logits;
  int64_t ls;  // row stride in elements
  const float* noise;
  int64_t ns;
  const float *temperature, *top_p, *min_p;
  const int* top_k;
  int64_t* tokens;
  float* logprobs;
  int V;
  int chunk;     // 16-byte vectors per CTA
  int resident;  // the CTA's part of the row fits in shared memory
};

constexpr int kBins = 512;
constexpr float kBinsPerLog2 = 12.f;  // bins of 6 % in probability over the top 2^-42; finer for a flatter row
constexpr float kSlack = 1e-5f;       // rounding of the fp32 mass sums

struct alignas(16) Part {
  float v;
  int i;
  float l, w;
};

AHB_DEVICE float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// larger value, then lower index
AHB_DEVICE bool beats(float v, int i, const Part& b) { return v > b.v || (v == b.v && i < b.i); }

AHB_DEVICE Part shfl_xor(const Part& p, int o) {
  return {__shfl_xor_sync(0xffffffffu, p.v, o), __shfl_xor_sync(0xffffffffu, p.i, o),
          __shfl_xor_sync(0xffffffffu, p.l, o), __shfl_xor_sync(0xffffffffu, p.w, o)};
}
// winner of (v, i) with its l; sum of w
struct TakeBest {
  AHB_DEVICE static Part none() { return {-INFINITY, INT_MAX, 0.f, 0.f}; }
  AHB_DEVICE Part operator()(Part a, const Part& b) const {
    const float w = a.w + b.w;
    if (beats(b.v, b.i, a)) a = b;
    a.w = w;
    return a;
  }
};
// larger v, then lower i; smaller l
struct TakeRange {
  AHB_DEVICE static Part none() { return {-INFINITY, INT_MAX, INFINITY, 0.f}; }
  AHB_DEVICE Part operator()(Part a, const Part& b) const {
    const float l = fminf(a.l, b.l);
    if (beats(b.v, b.i, a)) a = b;
    a.l = l;
    return a;
  }
};
// sums of i and w
struct TakeSum {
  AHB_DEVICE static Part none() { return {0.f, 0, 0.f, 0.f}; }
  AHB_DEVICE Part operator()(Part a, const Part& b) const {
    a.i += b.i;
    a.w += b.w;
    return a;
  }
};

template <typename T> struct Vec;
template <> struct Vec<__nv_bfloat16> {
  static constexpr int N = 8;
  AHB_DEVICE static float get(const uint4& r, int j) {
    const uint32_t w = j < 2 ? r.x : j < 4 ? r.y : j < 6 ? r.z : r.w;
    return __uint_as_float(j & 1 ? w & 0xffff0000u : w << 16);
  }
  AHB_DEVICE static void put(uint4& r, int j, float v) {
    uint32_t& w = j < 2 ? r.x : j < 4 ? r.y : j < 6 ? r.z : r.w;
    const uint32_t h = __float_as_uint(v) >> 16;
    w = j & 1 ? (w & 0xffffu) | (h << 16) : (w & 0xffff0000u) | h;
  }
  // +inf counts as the largest value of the type
  AHB_DEVICE static float most() { return __uint_as_float(0x7f7f0000u); }
};
template <> struct Vec<float> {
  static constexpr int N = 4;
  AHB_DEVICE static float get(const uint4& r, int j) {
    return __uint_as_float(j == 0 ? r.x : j == 1 ? r.y : j == 2 ? r.z : r.w);
  }
  AHB_DEVICE static void put(uint4& r, int j, float v) {
    (j == 0 ? r.x : j == 1 ? r.y : j == 2 ? r.z : r.w) = __float_as_uint(v);
  }
  AHB_DEVICE static float most() { return FLT_MAX; }
};

// Combines the threads' parts, then the CTAs' in rank order; every thread gets the result.  `mine` are
// two slots used in turn: one is rewritten only after the barrier that follows its last reading.
template <int NT, class Op>
AHB_DEVICE Part combine(Part p, Op op, Part* warps, Part* mine, int turn, int ctas) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) p = op(p, shfl_xor(p, o));
  if (lane == 0) warps[threadIdx.x >> 5] = p;
  __syncthreads();
  if (threadIdx.x < 32) {
    p = lane < NT / 32 ? warps[lane] : Op::none();
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) p = op(p, shfl_xor(p, o));
    if (lane == 0) mine[turn] = p;
  }
  cluster_sync();
  p = Op::none();
  for (int r = 0; r < ctas; ++r) {
    const uint32_t a = mapa_shared(&mine[turn], r);
    uint32_t x, y, z, w;
    asm volatile("ld.shared::cluster.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(x), "=r"(y), "=r"(z), "=r"(w) : "r"(a) : "memory");
    p = op(p, Part{__uint_as_float(x), (int)y, __uint_as_float(z), __uint_as_float(w)});
  }
  return p;
}

template <typename T, int NT>
__global__ void __launch_bounds__(NT) sample_kernel(SampleArgs p, int ctas) {
  using X = Vec<T>;
  constexpr int N = X::N;
  extern __shared__ __align__(16) uint4 keep[];
  __shared__ Part warps[NT / 32], mine[2];
  __shared__ int hist[kBins];
  __shared__ int count_to[kBins];    // tokens in bins up to and with this one
  __shared__ float most_to[kBins];   // and the most mass they can stand for
  __shared__ float2 wsum[kBins / 32];
  __shared__ int wcnt[kBins / 32];
  __shared__ int first_out;
  const int tid = threadIdx.x, rank = (int)cluster_ctarank();
  const int64_t row = blockIdx.x / ctas;
  const T* l = static_cast<const T*>(p.logits) + row * p.ls;
  const float* q = p.noise + row * p.ns;
  const float temp = p.temperature[row];
  const bool greedy = !(temp > 0.f);
  const float inv = greedy ? 1.f : fminf(fmaxf(1.f / temp, 1e-30f), 1e30f);
  const float c = inv * 1.4426950408889634f;  // logits to log2 of a probability
  const int kr = p.top_k[row], k = kr <= 0 || kr > p.V ? p.V : kr;
  const float top_p = p.top_p[row], min_p = fminf(p.min_p[row], 1.f);
  const float most_x = min_p > 0.f ? -__log2f(min_p) : INFINITY;
  const bool by_rank = !greedy && k < p.V, by_mass = !greedy && top_p < 1.f;
  int turn = 0;

  // vectors [v0, v1) of the row in 16-byte lines; its first element is element `skew` of line 0
  const int skew = (int)((reinterpret_cast<uintptr_t>(l) & 15) / sizeof(T));
  const int v0 = rank * p.chunk, v1 = min(v0 + p.chunk, (skew + p.V + N - 1) / N);
  auto fetch = [&](int v) {
    uint4 r = make_uint4(0, 0, 0, 0);
    const int i = v * N - skew;
    if (i >= 0 && i + N <= p.V) return __ldg(reinterpret_cast<const uint4*>(l + i));
#pragma unroll
    for (int j = 0; j < N; ++j) X::put(r, j, i + j >= 0 && i + j < p.V ? to_f(l[i + j]) : -INFINITY);
    return r;
  };
  auto clean = [&](uint4& r) {  // NaN never drawn, +inf as the largest value
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const float x = X::get(r, j);
      if (!(x < INFINITY)) X::put(r, j, x != x ? -INFINITY : X::most());
    }
  };
  auto line = [&](int v) {
    if (p.resident) return keep[v - v0];
    uint4 r = fetch(v);
    clean(r);
    return r;
  };

  // pass 1: the row into shared memory, its largest and least values
  for (int b = tid; b < kBins; b += NT) hist[b] = 0;
  if (tid == 0) first_out = kBins;
  Part range = TakeRange::none();
  for (int v = v0 + tid; v < v1; v += 4 * NT) {
    uint4 r[4];
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (v + u * NT < v1) r[u] = fetch(v + u * NT);
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (v + u * NT < v1) {
        clean(r[u]);
        if (p.resident) keep[v + u * NT - v0] = r[u];
#pragma unroll
        for (int j = 0; j < N; ++j) {
          const float x = X::get(r[u], j);
          if (x > range.v) {
            range.v = x;
            range.i = (v + u * NT) * N - skew + j;
          }
          if (x > -INFINITY) range.l = fminf(range.l, x);
        }
      }
  }
  range = combine<NT>(range, TakeRange(), warps, mine, turn ^= 1, ctas);
  const float top = range.v;
  const int top_i = range.i;
  if (top == -INFINITY) {  // nothing can be drawn
    if (rank == 0 && tid == 0) {
      p.tokens[row] = -1;
      p.logprobs[row] = -INFINITY;
    }
    cluster_sync();  // the other CTAs may still be reading this one's part
    return;
  }
  const float bins = fmaxf(kBinsPerLog2, (kBins - 1) / fmaxf((top - range.l) * c, 1e-20f));

  // the race over tokens ranked before (bound_l, bound_i), in bins before `out`
  float out = INFINITY, bound_l = -INFINITY;
  int bound_i = INT_MAX;
  auto race_line = [&](const uint4& r, int i0, Part& best) {
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const float x = X::get(r, j), x2 = (top - x) * c;
      if (x2 * bins < out && x2 <= most_x && (x > bound_l || (x == bound_l && i0 + j < bound_i))) {
        float s = -x2 - __log2f(__ldg(q + i0 + j));
        s = s != s ? -INFINITY : s;
        if (beats(s, i0 + j, best)) best = {s, i0 + j, x, best.w};
      }
    }
  };
  // pass 2: the mass beside the first token's, and the histogram where a rule needs one, else the race
  const bool binned = by_rank || by_mass;
  Part best = TakeBest::none();
  for (int v = v0 + tid; v < v1; v += NT) {
    const uint4 r = line(v);
    const int i0 = v * N - skew;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const float x2 = (top - X::get(r, j)) * c, e = ex2(-x2);
      best.w += i0 + j == top_i ? 0.f : e;
      if (binned && x2 < INFINITY) atomicAdd(&hist[(int)fminf(x2 * bins, kBins - 1)], 1);
    }
    if (!binned && !greedy) race_line(r, i0, best);
  }
  best = combine<NT>(best, TakeBest(), warps, mine, turn ^= 1, ctas);
  const float rest = best.w, z = 1.f + rest;

  if (binned) {
    // counts of all CTAs, summed up to each bin; the least and the most mass they can stand for
    int n = 0;
    float lo = 0.f, hi = 0.f;
    int cn = 0;
    if (tid < kBins) {
      for (int r = 0; r < ctas; ++r) {
        int a;
        asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(a) : "r"(mapa_shared(&hist[tid], r)) : "memory");
        n += a;
      }
      cn = n;
      lo = tid == kBins - 1 ? 0.f : n * ex2(-(tid + 1) / bins);
      hi = n * ex2(-tid / bins);
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int a = __shfl_up_sync(0xffffffffu, cn, o);
        const float b = __shfl_up_sync(0xffffffffu, lo, o), d = __shfl_up_sync(0xffffffffu, hi, o);
        if ((tid & 31) >= o) {
          cn += a;
          lo += b;
          hi += d;
        }
      }
      if ((tid & 31) == 31) {
        wcnt[tid >> 5] = cn;
        wsum[tid >> 5] = make_float2(lo, hi);
      }
    }
    __syncthreads();
    if (tid < kBins) {
      for (int w = 0; w < (tid >> 5); ++w) {
        cn += wcnt[w];
        lo += wsum[w].x;
        hi += wsum[w].y;
      }
      count_to[tid] = cn;
      most_to[tid] = hi;
      // everything in the bins after this one is out if the bins up to it already fill a rule
      if ((by_rank && cn >= k) || (by_mass && lo >= top_p * z * (1.f + kSlack))) atomicMin(&first_out, tid + 1);
    }
    __syncthreads();
    out = first_out < kBins ? (float)first_out : INFINITY;
  }

  float won_l = top;
  int won_i = top_i;
  for (bool again = binned; !greedy;) {
    if (again) {
      best = TakeBest::none();
      for (int v = v0 + tid; v < v1; v += NT) race_line(line(v), v * N - skew, best);
      best = combine<NT>(best, TakeBest(), warps, mine, turn ^= 1, ctas);
    }
    if (best.i == INT_MAX || best.i == top_i) break;
    won_l = best.l;
    won_i = best.i;
    if (!binned) break;
    const float x2 = (top - won_l) * c;
    const int bin = (int)fminf(x2 * bins, kBins - 1);
    if ((!by_rank || count_to[bin] <= k) && (!by_mass || most_to[bin] * (1.f + kSlack) < top_p * z)) break;
    Part before = TakeSum::none();
    for (int v = v0 + tid; v < v1; v += NT) {
      const uint4 r = line(v);
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const float x = X::get(r, j);
        if (x > won_l || (x == won_l && v * N - skew + j < won_i)) {
          before.i += 1;
          before.w += ex2(-(top - x) * c);
        }
      }
    }
    before = combine<NT>(before, TakeSum(), warps, mine, turn ^= 1, ctas);
    if ((!by_rank || before.i < k) && (!by_mass || before.w < top_p * z)) break;
    bound_l = won_l;
    bound_i = won_i;
    won_l = top;
    won_i = top_i;
    again = true;
  }
  if (rank == 0 && tid == 0) {
    p.tokens[row] = won_i;
    p.logprobs[row] = -(top - won_l) * inv - log1pf(rest);
  }
  cluster_sync();  // the other CTAs may still be reading this one's part
}

constexpr int kMaxSlice = 200 * 1024;

template <typename T, int NT>
int launch(SampleArgs& p, int B, int ctas, size_t smem, cudaStream_t st) {
  static bool ready[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev >= 64) return -3;
  if (!ready[dev]) {
    if (cudaFuncSetAttribute(sample_kernel<T, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSlice) != cudaSuccess) return -3;
    ready[dev] = true;
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(B * ctas));
  cfg.blockDim = dim3(NT);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = ctas;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, sample_kernel<T, NT>, p, ctas) == cudaSuccess ? 0 : -4;
}

}  // namespace

int ahb_sample(const void* logits, int64_t ls, int dtype, const float* noise, int64_t ns, const float* temperature,
               const int* top_k, const float* top_p, const float* min_p, int64_t* tokens, float* logprobs, int B, int V,
               cudaStream_t st) {
  if (B == 0) return 0;
  if (B > (1 << 27)) return -2;
  SampleArgs p{logits, ls, noise, ns, temperature, top_p, min_p, top_k, tokens, logprobs, V, 0, 0};
  const int N = dtype == AHB_BF16 ? 8 : 4;
  const int lines = (V + N - 1) / N + 1;  // one more where a row starts inside a line
  // Split a row while its part would keep a second CTA off the SM (over 96 KB), or while the rows alone do
  // not fill the SMs and a part still has four lines for every thread.
  int ctas = 1;
  while (ctas < 8 && ((lines / ctas) * 16 > 96 * 1024 || (B * ctas < 148 && lines / ctas >= 2048))) ctas *= 2;
  p.chunk = (lines + ctas - 1) / ctas;
  size_t smem = (size_t)p.chunk * 16;
  p.resident = smem <= (size_t)kMaxSlice;
  if (!p.resident) smem = 0;
  if (dtype == AHB_BF16) return launch<__nv_bfloat16, 512>(p, B, ctas, smem, st);
  return launch<float, 512>(p, B, ctas, smem, st);
}
