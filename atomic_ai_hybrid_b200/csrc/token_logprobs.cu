// Log-probabilities of given tokens, entropies and the likeliest alternatives of rows of logits, and their gradient.
//
//   d_v = (x_v - max x) / T,  S = sum e^{d_v},  log p_v = d_v - log S,  H = log S - sum e^{d_v} d_v / S
//   dx_v = (g ([v = y] - p_v) - gH p_v (log p_v + H)) / T
//
// Sums run over differences from the running maximum, in which nothing is lost to the size of the logits.
//
// Forward: one block a row, one pass over it.  Every thread keeps its largest logit (the lowest index where equal).
// The k-th largest of the 64 eight-lane groups' best is a bound that at least k logits reach, and only a thread
// whose own best reaches it can hold one of them: those few read their share of the row again, and what reaches the
// bound is ranked by counting.
#include "common.cuh"
#include "launchers.h"
#include "packed.cuh"

using namespace ahb;
using bf16 = __nv_bfloat16;

namespace {

constexpr int NT = 512, CAND = 1024;
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f, BIG = 3.4028234663852886e38f;
constexpr float FLOOR = -200.f;  // 2^-200 is 0 in fp32, and 0 times -200 is 0 where 0 times -inf is NaN

template <typename T>
struct Vec {
  static constexpr int N = 16 / sizeof(T);
};
AHB_DEVICE void unpack(const uint4& u, float (&x)[8]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = __uint_as_float(w[i] << 16);
    x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}
AHB_DEVICE void unpack(const uint4& u, float (&x)[4]) {
  x[0] = __uint_as_float(u.x), x[1] = __uint_as_float(u.y), x[2] = __uint_as_float(u.z), x[3] = __uint_as_float(u.w);
}

// NaN as -inf, +inf as the largest finite number
AHB_DEVICE float clean(float x) { return x != x ? -INFINITY : fminf(x, BIG); }

// order of (logit, index): larger logit first, then the lower index; 0 is below every logit with a probability
AHB_DEVICE uint64_t rank_of(float x, int v) {
  if (x == -INFINITY) return 0;
  const uint32_t b = __float_as_uint(x + 0.f);
  const uint32_t k = (b & 0x80000000u) ? ~b : b | 0x80000000u;
  return (static_cast<uint64_t>(k) << 32) | (0xffffffffu - (uint32_t)v);
}
AHB_DEVICE int index_of(uint64_t r) { return (int)(0xffffffffu - (uint32_t)r); }
AHB_DEVICE float logit_of(uint64_t r) {
  const uint32_t k = (uint32_t)(r >> 32);
  return __uint_as_float((k & 0x80000000u) ? k & 0x7fffffffu : ~k);
}

struct Sums {
  float m, s, z;  // maximum, sum 2^d, sum 2^d d with d = (x - m) c
  AHB_DEVICE void move(float mn, float c) {
    if (m == -INFINITY) {
      m = mn;
      return;
    }
    const float d = fmaxf((m - mn) * c, FLOOR), f = ex2(d);
    z = f * (z + s * d);
    s *= f;
    m = mn;
  }
  AHB_DEVICE void add(float x, float c) {
    const float d = fminf(fmaxf((x - m) * c, FLOOR), 0.f), e = ex2(d);  // NaN: no mass; +inf: as the largest
    s += e;
    z += e * d;
  }
  AHB_DEVICE void join(const Sums& o, float c) {
    if (o.m == -INFINITY) return;
    Sums b = o;
    const float mn = fmaxf(m, o.m);
    if (m != mn) move(mn, c);
    if (b.m != mn) b.move(mn, c);
    s += b.s;
    z += b.z;
  }
};

// A row's elements as this thread sees them: f(x, v) in rising v, in vectors where the row is aligned.
template <typename T>
struct Row {
  const T* p;
  int V, head, vecs;  // elements before the first 16-byte boundary, whole vectors from there
  AHB_DEVICE Row(const T* row, int n) : p(row), V(n) {
    head = min(n, (int)(((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / sizeof(T)));
    vecs = (n - head) / Vec<T>::N;
  }
  AHB_DEVICE int tail() const { return head + vecs * Vec<T>::N; }
  AHB_DEVICE uint4 vec(int i) const { return reinterpret_cast<const uint4*>(p + head)[i]; }
};

template <typename T>
__global__ void __launch_bounds__(NT) logprobs_fwd(const T* __restrict__ logits, int64_t ls, const int64_t* __restrict__ tokens,
                                                   int V, int top, float c, float* __restrict__ lp, float* __restrict__ entropy,
                                                   float4* __restrict__ stats, int64_t* __restrict__ top_tok,
                                                   float* __restrict__ top_lp) {
  constexpr int N = Vec<T>::N, UN = 4;
  __shared__ Sums sums[NT / 32];
  __shared__ uint64_t best_sh[64], cand[CAND], bound_sh;
  __shared__ int count;
  const int64_t r = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
  const Row<T> row(logits + r * ls, V);
  Sums a{-INFINITY, 0.f, 0.f};
  uint64_t best = 0;
  auto one = [&](int v) {  // the few elements outside the vectors
    const float x = clean(to_f(row.p[v]));
    if (x == -INFINITY) return;
    if (x > a.m) a.move(x, c);
    a.add(x, c);
    const uint64_t k = rank_of(x, v);
    best = k > best ? k : best;
  };
  if (tid < row.head) one(tid);
  if (row.tail() + tid < V) one(row.tail() + tid);
  float top_x = -INFINITY;
  int top_v = 0;
  for (int i0 = tid; i0 < row.vecs; i0 += NT * UN) {
    uint4 u[UN];
#pragma unroll
    for (int j = 0; j < UN; ++j)
      if (i0 + j * NT < row.vecs) u[j] = row.vec(i0 + j * NT);
#pragma unroll
    for (int j = 0; j < UN; ++j) {
      if (i0 + j * NT >= row.vecs) break;
      float x[N];
      unpack(u[j], x);
      float mx = -INFINITY;
#pragma unroll
      for (int e = 0; e < N; ++e) mx = fmaxf(mx, x[e]);  // NaN is passed over
      if (mx > top_x) {  // seldom, but for a thread's first vectors
        mx = fminf(mx, BIG);
        if (mx > a.m) a.move(mx, c);
        if (mx > top_x) {
          top_x = mx;
#pragma unroll
          for (int e = N - 1; e >= 0; --e)
            if (clean(x[e]) == mx) top_v = row.head + (i0 + j * NT) * N + e;
        }
      }
      if (a.m > -INFINITY) {
#pragma unroll
        for (int e = 0; e < N; ++e) a.add(x[e], c);
      }
    }
  }
  {
    const uint64_t k = rank_of(top_x, top_v);
    best = k > best ? k : best;
  }
  const uint64_t mine = best;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    Sums b{__shfl_xor_sync(0xffffffffu, a.m, o), __shfl_xor_sync(0xffffffffu, a.s, o), __shfl_xor_sync(0xffffffffu, a.z, o)};
    a.join(b, c);
  }
  if (lane == 0) sums[w] = a;
  if (top > 0) {
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) {
      const uint64_t b = __shfl_xor_sync(0xffffffffu, best, o);
      best = b > best ? b : best;
    }
    if ((lane & 7) == 0) best_sh[tid >> 3] = best;
    if (tid == 0) count = 0;
  }
  __syncthreads();
  a = sums[0];
#pragma unroll
  for (int i = 1; i < NT / 32; ++i) a.join(sums[i], c);
  const bool some = a.m > -INFINITY;
  const float log2s = some ? log2f(a.s) : 0.f;
  auto logprob = [&](float x) { return x == -INFINITY || !some ? -INFINITY : ((x - a.m) * c - log2s) * LN2; };
  if (tid == 0) {
    const int64_t y = tokens[r];
    lp[r] = y >= 0 && y < V ? logprob(clean(to_f(row.p[y]))) : 0.f;
    const float H = some ? (log2s - a.z / a.s) * LN2 : 0.f;
    entropy[r] = H;
    stats[r] = make_float4(a.m, log2s, H, 0.f);
  }
  if (top == 0) return;
  if (tid < 64) {
    const uint64_t b = best_sh[tid];
    int above = 0;
    for (int i = 0; i < 64; ++i) above += best_sh[i] > b || (best_sh[i] == b && i < tid);
    if (above == top - 1) bound_sh = b;
  }
  __syncthreads();
  const uint64_t bound = bound_sh > 0 ? bound_sh : 1;
  auto take = [&](float x, int v) {
    const uint64_t k = rank_of(x, v);
    if (k < bound) return;
    const int at = atomicAdd(&count, 1);
    if (at < CAND) cand[at] = k;
  };
  if (mine >= bound) {
    const float least = logit_of(bound);
    if (tid < row.head) take(clean(to_f(row.p[tid])), tid);
    if (row.tail() + tid < V) take(clean(to_f(row.p[row.tail() + tid])), row.tail() + tid);
    for (int i0 = tid; i0 < row.vecs; i0 += NT * UN) {
      uint4 u[UN];
#pragma unroll
      for (int j = 0; j < UN; ++j)
        if (i0 + j * NT < row.vecs) u[j] = row.vec(i0 + j * NT);
#pragma unroll
      for (int j = 0; j < UN; ++j) {
        if (i0 + j * NT >= row.vecs) break;
        float x[N];
        unpack(u[j], x);
#pragma unroll
        for (int e = 0; e < N; ++e)
          if (bound == 1 || x[e] >= least) take(clean(x[e]), row.head + (i0 + j * NT) * N + e);
      }
    }
  }
  __syncthreads();
  int n = count;
  if (n > CAND) {  // logits in an order that puts the largest into few threads: one pass for each alternative
    uint64_t last = ~0ull;
    for (int k = 0; k < top; ++k) {
      uint64_t b = 0;
      for (int v = tid; v < V; v += NT) {
        const uint64_t q = rank_of(clean(to_f(row.p[v])), v);
        if (q < last && q > b) b = q;
      }
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint64_t q = __shfl_xor_sync(0xffffffffu, b, o);
        b = q > b ? q : b;
      }
      __syncthreads();
      if (lane == 0) best_sh[w] = b;
      __syncthreads();
      for (int i = 0; i < NT / 32; ++i) b = best_sh[i] > b ? best_sh[i] : b;
      last = b;
      if (tid == 0) cand[k] = b;
    }
    n = top;
    __syncthreads();
  }
  for (int i = tid; i < n; i += NT) {
    const uint64_t b = cand[i];
    int above = 0;
    for (int j = 0; j < n; ++j) above += cand[j] > b;
    if (above < top) {
      const float p = b ? logprob(logit_of(b)) : -INFINITY;
      top_tok[r * top + above] = p > -INFINITY ? index_of(b) : -1;
      top_lp[r * top + above] = p;
    }
  }
  for (int i = n + tid; i < top; i += NT) {  // fewer logits with a probability than asked for
    top_tok[r * top + i] = -1;
    top_lp[r * top + i] = -INFINITY;
  }
}

// Elementwise over the row's part; logits and gradient in vectors where both lie alike.
template <typename T>
__global__ void __launch_bounds__(256) logprobs_bwd(const T* __restrict__ logits, int64_t ls, const int64_t* __restrict__ tokens,
                                                    const float4* __restrict__ stats, const float* __restrict__ g,
                                                    const float* __restrict__ ge, int V, float c, float inv_t, int part,
                                                    T* __restrict__ dx) {
  constexpr int N = Vec<T>::N;
  const int64_t r = blockIdx.y;
  const T* x = logits + r * ls;
  T* d = dx + r * V;
  const float4 st = stats[r];
  const int64_t y64 = tokens[r];
  const int y = y64 >= 0 && y64 < V ? (int)y64 : -1;
  const bool some = st.x > -INFINITY;
  const float gy = y >= 0 ? g[r] * inv_t : 0.f, gh = ge[r] * inv_t;
  auto grad = [&](float v, int i) {
    v = clean(v);
    if (v == -INFINITY || !some) return 0.f;
    const float q = fmaxf((v - st.x) * c - st.y, -1e30f), p = ex2(q);
    return (i == y ? gy : 0.f) - p * (gy + gh * (q * LN2 + st.z));
  };
  const int b = blockIdx.x * part, e = min(V, b + part);
  const Row<T> row(x + b, e - b);
  const bool alike = ((reinterpret_cast<uintptr_t>(x + b) ^ reinterpret_cast<uintptr_t>(d + b)) & 15) == 0;
  if (alike) {
    for (int i = threadIdx.x; i < row.vecs; i += 256) {
      const uint4 u = row.vec(i);
      float v[N];
      unpack(u, v);
      const int at = b + row.head + i * N;
      alignas(16) T o[N];
#pragma unroll
      for (int k = 0; k < N; ++k) o[k] = from_f<T>(grad(v[k], at + k));
      *reinterpret_cast<uint4*>(d + at) = *reinterpret_cast<uint4*>(o);
    }
    if ((int)threadIdx.x < row.head) d[b + threadIdx.x] = from_f<T>(grad(to_f(x[b + threadIdx.x]), b + threadIdx.x));
    const int t = b + row.tail() + threadIdx.x;
    if (t < e) d[t] = from_f<T>(grad(to_f(x[t]), t));
  } else {
    for (int i = b + threadIdx.x; i < e; i += 256) d[i] = from_f<T>(grad(to_f(x[i]), i));
  }
}

}  // namespace

void ahb_token_logprobs_fwd(const void* logits, int64_t ls, int dtype, const int64_t* tokens, int64_t R, int V, int top,
                            float temperature, float* lp, float* entropy, void* stats, int64_t* top_tok, float* top_lp,
                            cudaStream_t st) {
  if (R == 0) return;
  const float c = LOG2E / temperature;
  if (dtype == AHB_BF16)
    logprobs_fwd<<<(unsigned)R, NT, 0, st>>>((const bf16*)logits, ls, tokens, V, top, c, lp, entropy, (float4*)stats, top_tok,
                                             top_lp);
  else
    logprobs_fwd<<<(unsigned)R, NT, 0, st>>>((const float*)logits, ls, tokens, V, top, c, lp, entropy, (float4*)stats, top_tok,
                                             top_lp);
}

void ahb_token_logprobs_bwd(const void* logits, int64_t ls, int dtype, const int64_t* tokens, const void* stats,
                            const float* g, const float* ge, int64_t R, int V, float temperature, void* dx,
                            cudaStream_t st) {
  if (R == 0) return;
  const float c = LOG2E / temperature, inv_t = 1.f / temperature;
  const int part = 16384;
  for (int64_t r = 0; r < R; r += 65535) {  // the grid's second extent
    const int64_t n = R - r < 65535 ? R - r : 65535;
    const dim3 grid((V + part - 1) / part, (unsigned)n);
    if (dtype == AHB_BF16)
      logprobs_bwd<<<grid, 256, 0, st>>>((const bf16*)logits + r * ls, ls, tokens + r, (const float4*)stats + r, g + r, ge + r, V,
                                         c, inv_t, part, (bf16*)dx + r * V);
    else
      logprobs_bwd<<<grid, 256, 0, st>>>((const float*)logits + r * ls, ls, tokens + r, (const float4*)stats + r, g + r, ge + r, V,
                                         c, inv_t, part, (float*)dx + r * V);
  }
}
