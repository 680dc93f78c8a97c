// Log-probabilities of given tokens, entropies and the likeliest alternatives of rows of logits, and their gradient.
//
//   d_v = (x_v - max x) / T,  S = sum e^{d_v},  log p_v = d_v - log S,  H = log S - sum e^{d_v} d_v / S
//   dx_v = (g ([v = y] - p_v) - gH p_v (log p_v + H)) / T
//
// Sums run over differences from the running maximum, in which nothing is lost to the size of the logits.  Two values
// at a time where the GPU has instructions for it: a bf16 logit costs eleven all told (2048 x 128256: 93.1 M issued by warps), as many
// as the SMs issue while the copy would bring it.
//
// Forward: one pass over a row, by one block or, where rows are few, by a cluster of up to eight.  A warp's sums refer
// to its own running maximum, which moves a handful of times (with one for each thread some lane of a warp had a new one at
// almost every step: 2048 x 128256 logits 156 to 191 us).  Every thread keeps its largest logit: the k-th largest of 64
// groups' is a bound that at least k logits reach, and only a thread whose own reaches it can hold one of them: the
// shares of those few are read again, by all threads, and what reaches the bound is ranked by counting.
// 2048 x 128256 bf16 logits with 8 alternatives take 138 us, 0.59 of the copy's rate, 62 % of the issue slots; 300 x 151936 fp32
// 48 us.  Backward: one read and one write, 4096 x 50304 bf16 in 128 us, 0.94 of that rate; fp32 54 us.
#include <cooperative_groups.h>
#include "common.cuh"
#include "launchers.h"
#include "packed.cuh"

using namespace ahb;
using bf16 = __nv_bfloat16;

namespace {

constexpr int NT = 256, CAND = 1024, MAX_TOP = 64;
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
  float m, s, z;  // maximum, sum 2^d, sum 2^d d with d = (x - m) c, c = log2(e) / T
  AHB_DEVICE void move(float mn, float c) {
    if (m != -INFINITY) {
      const float d = fmaxf((m - mn) * c, FLOOR), f = ex2(d);
      z = f * (z + s * d);
      s *= f;
    }
    m = mn;
  }
  AHB_DEVICE void add(float x, float c) {
    const float d = fmaxf((x - m) * c, FLOOR), e = ex2(d);
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

// A vector's elements with NaN and what lies below LOW as LOW, and the largest of them.
constexpr float LOW = -1e30f;
AHB_DEVICE float unpack_low(const uint4& u, float (&x)[8]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
  const __nv_bfloat162* in = reinterpret_cast<const __nv_bfloat162*>(w);
  const __nv_bfloat162 low = __float2bfloat162_rn(LOW);
  uint4 v;
  __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&v);
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = __hmax2(in[i], low);
  const float2 f = __bfloat1622float2(__hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3])));
  unpack(v, x);
  return fmaxf(f.x, f.y);
}
AHB_DEVICE float unpack_low(const uint4& u, float (&x)[4]) {
  unpack(u, x);
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = fmaxf(x[i], LOW);
  return fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
}

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

// C: blocks of a row's cluster, each with a part of it
template <typename T, int C>
__global__ void __launch_bounds__(NT, 4) logprobs_fwd(const T* __restrict__ logits, int64_t ls, const int64_t* __restrict__ tokens,
                                                      int V, int top, float c, float* __restrict__ lp, float* __restrict__ entropy,
                                                      float4* __restrict__ stats, int64_t* __restrict__ top_tok,
                                                      float* __restrict__ top_lp) {
  constexpr int N = Vec<T>::N, UN = 4, GL = NT / 64;  // GL: lanes of a group
  __shared__ Sums sums[NT / 32];
  __shared__ uint64_t best_sh[NT / 32], cand[CAND];
  __shared__ float group_max[64], bound_sh;
  __shared__ int count, who[NT], n_who;
  struct Part {
    Sums sums;
    uint64_t best[MAX_TOP];
  };
  __shared__ Part part;  // what the cluster's first block reads
  const int64_t r = blockIdx.x / C;
  const int rank = blockIdx.x % C, tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
  const T* p = logits + r * ls;
  // parts of whole 64-element pieces
  const int each = C == 1 ? V : ((V + C - 1) / C + 63) & ~63, v0 = min(V, rank * each), v1 = min(V, v0 + each);
  const Row<T> row(p + v0, v1 - v0);
  Sums a{-INFINITY, 0.f, 0.f};
  float best = -INFINITY;  // this thread's largest, where it is above LOW
  // Up to this maximum (m - LOW) c is finite: 0 times a weight's infinite exponent would be NaN.  It is the temperature
  // below 4e-9 and the logits above 1e38 that go the way of `Sums::add`.
  const float limit = fminf(BIG, 3e38f / c + LOW);
  auto one = [&](int v) {  // the few elements outside the vectors, and all where the maximum is infinite or below LOW
    const float x = clean(v < row.V ? to_f(row.p[v]) : -INFINITY);
    const float mx = warp_max(x);
    best = fmaxf(best, x);
    if (mx > a.m) a.move(mx, c);
    if (x > -INFINITY) a.add(x, c);
  };
  if (w == 0) one(lane < row.head ? lane : row.V);
  if (w == 1) one(row.tail() + lane);
  auto vec = [&](const uint4& u, int i) {
    float x[N];
    const bool in = i < row.vecs;
    const float mx = in ? unpack_low(u, x) : -INFINITY;
    if (__any_sync(0xffffffffu, mx > a.m)) {
      float y[N], top_y = -INFINITY;
      unpack(u, y);
#pragma unroll
      for (int e = 0; e < N; ++e) top_y = fmaxf(top_y, clean(y[e]));
      top_y = warp_max(in ? top_y : -INFINITY);
      if (top_y > a.m) a.move(top_y, c);
    }
    if (!in) return;
    best = fmaxf(best, mx);
    if (!(a.m > 0.1f * LOW && a.m < limit)) {
      unpack(u, x);
#pragma unroll
      for (int e = 0; e < N; ++e)
        if (clean(x[e]) > -INFINITY) a.add(clean(x[e]), c);
      return;
    }
    const float2 neg = both(-a.m), cc = both(c);
    float2 s2 = both(0.f), z2 = both(0.f);
#pragma unroll
    for (int e = 0; e < N; e += 2) {
      const float2 d = mul2(add2(make_float2(x[e], x[e + 1]), neg), cc);
      const float2 q = make_float2(ex2(d.x), ex2(d.y));
      s2 = add2(s2, q);
      z2 = fma2(q, d, z2);
    }
    a.s += s2.x + s2.y;
    a.z += z2.x + z2.y;
  };
  int i0 = tid;
  for (; i0 - lane + 31 + (UN - 1) * NT < row.vecs; i0 += NT * UN) {  // whole warps
    uint4 u[UN];
#pragma unroll
    for (int j = 0; j < UN; ++j) u[j] = row.vec(i0 + j * NT);
#pragma unroll
    for (int j = 0; j < UN; ++j) vec(u[j], i0 + j * NT);
  }
  for (; i0 - lane < row.vecs; i0 += NT) vec(i0 < row.vecs ? row.vec(i0) : make_uint4(0, 0, 0, 0), i0);
  best = fminf(best, BIG);
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {  // the maximum is the warp's already
    a.s += __shfl_xor_sync(0xffffffffu, a.s, o);
    a.z += __shfl_xor_sync(0xffffffffu, a.z, o);
  }
  if (lane == 0) sums[w] = a;
  if (top > 0) {
    float b = best;
#pragma unroll
    for (int o = 1; o < GL; o <<= 1) b = fmaxf(b, __shfl_xor_sync(0xffffffffu, b, o));
    if (tid % GL == 0) group_max[tid / GL] = b;
    if (tid == 0) count = n_who = 0;
  }
  __syncthreads();
  a = sums[0];
#pragma unroll
  for (int i = 1; i < NT / 32; ++i) a.join(sums[i], c);
  int n = 0;  // candidates for the row's likeliest, in `cand`
  if (top > 0) {
    if (tid < 64) {
      const float b = group_max[tid];
      int above = 0;
      for (int i = 0; i < 64; ++i) above += group_max[i] > b || (group_max[i] == b && i < tid);
      if (above == top - 1) bound_sh = b;
    }
    __syncthreads();
    // a bound that says nothing (few logits above LOW): all with a probability
    const float bound = bound_sh > LOW ? bound_sh : -INFINITY;
    auto take = [&](float x, int v) {
      if (!(x >= bound) || x == -INFINITY) return;
      const int at = atomicAdd(&count, 1);
      if (at < CAND) cand[at] = rank_of(x, v);
    };
    if (w == 0 && lane < row.head) take(clean(to_f(row.p[lane])), v0 + lane);
    if (w == 1 && row.tail() + lane < row.V) take(clean(to_f(row.p[row.tail() + lane])), v0 + row.tail() + lane);
    if (best >= bound) who[atomicAdd(&n_who, 1)] = tid;
    __syncthreads();
    const int turns = (row.vecs + NT - 1) / NT, all = n_who * turns;
    for (int x0 = tid; x0 < all; x0 += NT * UN) {
      uint4 u[UN];
      int i[UN];
#pragma unroll
      for (int j = 0; j < UN; ++j) {
        const int x = x0 + j * NT;
        i[j] = x < all ? who[x / turns] + (x % turns) * NT : row.vecs;
        if (i[j] < row.vecs) u[j] = row.vec(i[j]);
      }
#pragma unroll
      for (int j = 0; j < UN; ++j) {
        if (i[j] >= row.vecs) continue;
        float x[N];
        unpack(u[j], x);
#pragma unroll
        for (int e = 0; e < N; ++e) take(clean(x[e]), v0 + row.head + i[j] * N + e);
      }
    }
    __syncthreads();
    n = count;
    if (n > CAND) {  // many equal ones, or an order that puts the largest into few threads: one pass for each alternative
      uint64_t last = ~0ull;
      for (int k = 0; k < top; ++k) {
        uint64_t b = 0;
        for (int v = tid; v < row.V; v += NT) {
          const uint64_t q = rank_of(clean(to_f(row.p[v])), v0 + v);
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
  }
  if (C > 1) {  // the parts meet in the cluster's first block: sums, and each one's likeliest in order
    namespace cg = cooperative_groups;
    auto cluster = cg::this_cluster();
    if (tid == 0) part.sums = a;
    for (int i = tid; i < top; i += NT)
      if (i >= n) part.best[i] = 0;
    for (int i = tid; i < n; i += NT) {
      int above = 0;
      for (int j = 0; j < n; ++j) above += cand[j] > cand[i];
      if (above < top) part.best[above] = cand[i];
    }
    cluster.sync();
    if (rank == 0) {
      for (int k = 1; k < C; ++k) a.join(cluster.map_shared_rank(&part, k)->sums, c);
      for (int i = tid; i < C * top; i += NT) cand[i] = cluster.map_shared_rank(&part, i / top)->best[i % top];
      n = C * top;
    }
    cluster.sync();  // no part leaves before it has been read
    if (rank != 0) return;
  }
  const bool some = a.m > -INFINITY;
  const float log2s = some ? log2f(a.s) : 0.f;
  // without the floor, and not by way of c: a logit however far below has a log-probability
  const float inv_t = c * LN2;
  auto logprob = [&](float x) { return x == -INFINITY || !some ? -INFINITY : (x - a.m) * inv_t - log2s * LN2; };
  if (tid == 0) {
    const int64_t y = tokens[r];
    lp[r] = y >= 0 && y < V ? logprob(clean(to_f(p[y]))) : 0.f;
    const float H = some ? (log2s - a.z / a.s) * LN2 : 0.f;
    entropy[r] = H;
    stats[r] = make_float4(a.m, log2s, H, 0.f);
  }
  auto place = [&](int at, uint64_t b) {
    const float q = b ? logprob(logit_of(b)) : -INFINITY;
    top_tok[r * top + at] = q > -INFINITY ? index_of(b) : -1;
    top_lp[r * top + at] = q;
  };
  for (int i = tid; i < n; i += NT) {
    const uint64_t b = cand[i];
    int above = 0;
    for (int j = 0; j < n; ++j) above += cand[j] > b || (cand[j] == b && j < i);
    if (above < top) place(above, b);
  }
  for (int i = n + tid; i < top; i += NT) place(i, 0);  // fewer logits with a probability than asked for
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
  const bool some = st.x > -INFINITY, plain = some && st.x < BIG;
  const float gy = y >= 0 ? g[r] * inv_t : 0.f, gh = ge[r] * inv_t;
  auto grad = [&](float v, int i) {
    v = clean(v);
    if (v == -INFINITY || !some) return 0.f;
    const float q = fmaxf((v - st.x) * c - st.y, FLOOR), p = ex2(q);
    return (i == y ? gy : 0.f) - p * (gy + gh * (q * LN2 + st.z));
  };
  const int b = blockIdx.x * part, e = min(V, b + part);
  const Row<T> row(x + b, e - b);
  const bool alike = ((reinterpret_cast<uintptr_t>(x + b) ^ reinterpret_cast<uintptr_t>(d + b)) & 15) == 0;
  if (alike) {
    constexpr int UN = 4;
    for (int i0 = threadIdx.x; i0 < row.vecs; i0 += 256 * UN) {
      uint4 u[UN];
#pragma unroll
      for (int j = 0; j < UN; ++j)
        if (i0 + j * 256 < row.vecs) u[j] = row.vec(i0 + j * 256);
#pragma unroll
      for (int j = 0; j < UN; ++j) {
        if (i0 + j * 256 >= row.vecs) break;
        float v[N];
        unpack(u[j], v);
        const int at = b + row.head + (i0 + j * 256) * N;
        alignas(16) T o[N];
        if ((y >= at && y < at + N) || !plain) {  // the given token's, or an unusual row
#pragma unroll
          for (int k = 0; k < N; ++k) o[k] = from_f<T>(grad(v[k], at + k));
        } else {
#pragma unroll
          for (int k = 0; k < N; k += 2) {
            const float2 q = max2(fma2(add2(make_float2(v[k], v[k + 1]), both(-st.x)), both(c), both(-st.y)), FLOOR);
            const float2 g2 = mul2(make_float2(ex2(q.x), ex2(q.y)), fma2(q, both(-gh * LN2), both(-gy - gh * st.z)));
            o[k] = from_f<T>(g2.x);
            o[k + 1] = from_f<T>(g2.y);
          }
        }
        *reinterpret_cast<uint4*>(d + at) = *reinterpret_cast<uint4*>(o);
      }
    }
    if ((int)threadIdx.x < row.head) d[b + threadIdx.x] = from_f<T>(grad(to_f(x[b + threadIdx.x]), b + threadIdx.x));
    const int t = b + row.tail() + threadIdx.x;
    if (t < e) d[t] = from_f<T>(grad(to_f(x[t]), t));
  } else {
    for (int i = b + threadIdx.x; i < e; i += 256) d[i] = from_f<T>(grad(to_f(x[i]), i));
  }
}

// Few rows are cut for as many blocks as two an SM: a row alone on a block takes its 10 us however few there are (64 rows of
// 50304 logits with 5 alternatives: 15.6 us whole, 12.3 with four blocks a row).  A part keeps 4096 logits at least.
template <typename T>
int launch_fwd(const T* logits, int64_t ls, const int64_t* tokens, int64_t R, int V, int top, float c, float* lp, float* entropy,
               float4* stats, int64_t* top_tok, float* top_lp, cudaStream_t st) {
  int dev = 0, sms = 148;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return -1;
  int C = 1;
  while (C < 8 && R * 2 * C <= 2 * sms && V / (2 * C) >= 4096) C *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(R * C));
  cfg.blockDim = dim3(NT);
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim = {(unsigned)C, 1, 1};
  cfg.attrs = at;
  cfg.numAttrs = 1;
  auto go = [&](auto kernel) {
    return cudaLaunchKernelEx(&cfg, kernel, logits, ls, tokens, V, top, c, lp, entropy, stats, top_tok, top_lp) == cudaSuccess ? 0 : -2;
  };
  switch (C) {
    case 8: return go(logprobs_fwd<T, 8>);
    case 4: return go(logprobs_fwd<T, 4>);
    case 2: return go(logprobs_fwd<T, 2>);
    default: return go(logprobs_fwd<T, 1>);
  }
}

}  // namespace

int ahb_token_logprobs_fwd(const void* logits, int64_t ls, int dtype, const int64_t* tokens, int64_t R, int V, int top,
                           float temperature, float* lp, float* entropy, void* stats, int64_t* top_tok, float* top_lp,
                           cudaStream_t st) {
  if (R == 0) return 0;
  const float c = LOG2E / temperature;
  return dtype == AHB_BF16 ? launch_fwd((const bf16*)logits, ls, tokens, R, V, top, c, lp, entropy, (float4*)stats, top_tok, top_lp, st)
                           : launch_fwd((const float*)logits, ls, tokens, R, V, top, c, lp, entropy, (float4*)stats, top_tok, top_lp, st);
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
