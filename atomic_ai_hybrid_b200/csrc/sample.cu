// The next token of every row from its logits and given Exp(1) noise, with temperature, top-k, top-p
// and min-p per row (the reference has no sampler).
//
// With d_i = (max l - l_i) / T and m_i = e^{-d_i}, tokens are ranked by (logit descending, index
// ascending).  A token is kept if its rank is below top_k, the mass ranked before it is below
// top_p sum m (rank 0 always), and m_i >= min_p; each rule looks at the whole tempered row, so their
// order does not matter.  The token is argmax over the kept ones of -d_i - log q_i, which picks i with
// probability m_i over the kept mass; logprob = -d_i - log sum m.
//
// No sort and no search for thresholds: the kept tokens are a prefix of the ranking, so if the winner of
// the race over some prefix is kept, it is the winner over the kept tokens; if not, nothing ranked
// after it is kept either and the race is run again over what is ranked before it.
#include "launchers.h"
#include "common.cuh"
#include <cfloat>

namespace {
using namespace ahb;

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
};

constexpr int kThreads = 512, kWarps = kThreads / 32;

struct Best {
  float s;
  int i;
};
AHB_DEVICE Best better(Best a, Best b) { return b.s > a.s || (b.s == a.s && b.i < a.i) ? b : a; }

AHB_DEVICE Best warp_best(Best v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = better(v, Best{__shfl_xor_sync(0xffffffffu, v.s, o), __shfl_xor_sync(0xffffffffu, v.i, o)});
  return v;
}

AHB_DEVICE Best block_best(Best v, Best* sh) {
  v = warp_best(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
  __syncthreads();
  const int lane = threadIdx.x & 31;
  return warp_best(lane < kWarps ? sh[lane] : Best{-INFINITY, INT_MAX});
}

// NaN counts as -inf (never drawn), +inf as the largest finite value
AHB_DEVICE float logit_of(float l) { return l != l ? -INFINITY : fminf(l, FLT_MAX); }

template <typename T>
__global__ void __launch_bounds__(kThreads) sample_kernel(SampleArgs p) {
  __shared__ Best shb[kWarps];
  __shared__ float shf[kWarps];
  const int64_t row = blockIdx.x;
  const T* l = static_cast<const T*>(p.logits) + row * p.ls;
  const float* q = p.noise + row * p.ns;
  const float temp = p.temperature[row];
  const bool greedy = !(temp > 0.f);
  const float inv = greedy ? 1.f : 1.f / temp;
  const int kr = p.top_k[row], k = greedy ? 1 : (kr <= 0 ? p.V : kr);
  const float top_p = p.top_p[row], min_p = fminf(p.min_p[row], 1.f);

  Best top{-INFINITY, INT_MAX};
  for (int i = threadIdx.x; i < p.V; i += kThreads) top = better(top, Best{logit_of(to_f(l[i])), i});
  top = block_best(top, shb);
  if (top.s == -INFINITY) {  // nothing can be drawn
    if (threadIdx.x == 0) {
      p.tokens[row] = -1;
      p.logprobs[row] = -INFINITY;
    }
    return;
  }
  float z = 0.f;
  for (int i = threadIdx.x; i < p.V; i += kThreads) z += __expf((logit_of(to_f(l[i])) - top.s) * inv);
  z = block_sum(z, shf);

  Best bound{-INFINITY, INT_MAX};  // tokens ranked before (logit, index)
  Best won = top;
  while (k > 1) {
    Best race{-INFINITY, INT_MAX};
    for (int i = threadIdx.x; i < p.V; i += kThreads) {
      const float li = logit_of(to_f(l[i]));
      if (!(li > bound.s || (li == bound.s && i < bound.i)) || li == -INFINITY) continue;
      const float nd = (li - top.s) * inv;
      if (__expf(nd) < min_p) continue;
      float s = nd - __logf(q[i]);
      race = better(race, Best{s != s ? -INFINITY : s, i});
    }
    race = block_best(race, shb);
    won = race.i == INT_MAX ? top : Best{logit_of(to_f(l[race.i])), race.i};
    if (won.i == top.i) break;
    float before = 0.f, mass = 0.f;
    for (int i = threadIdx.x; i < p.V; i += kThreads) {
      const float li = logit_of(to_f(l[i]));
      if (li > won.s || (li == won.s && i < won.i)) {
        before += 1.f;
        mass += __expf((li - top.s) * inv);
      }
    }
    before = block_sum(before, shf);
    mass = block_sum(mass, shf);
    if (before < (float)k && (mass < top_p * z)) break;
    bound = won;
  }
  if (threadIdx.x == 0) {
    p.tokens[row] = won.i;
    p.logprobs[row] = (won.s - top.s) * inv - __logf(z);
  }
}

}  // namespace

int ahb_sample(const void* logits, int64_t ls, int dtype, const float* noise, int64_t ns, const float* temperature,
               const int* top_k, const float* top_p, const float* min_p, int64_t* tokens, float* logprobs, int B, int V,
               cudaStream_t st) {
  if (B == 0) return 0;
  const SampleArgs p{logits, ls, noise, ns, temperature, top_p, min_p, top_k, tokens, logprobs, V};
  if (dtype == AHB_BF16) sample_kernel<__nv_bfloat16><<<B, kThreads, 0, st>>>(p);
  else sample_kernel<float><<<B, kThreads, 0, st>>>(p);
  return 0;
}
