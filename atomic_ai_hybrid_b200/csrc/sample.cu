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
//
// 1 x 151936 with every rule 10.1 us, 64 x 50304 16 us: three passes over shared memory and four meetings of the
// cluster, one after another.  256 x 128256 fp32 119 us (greedy 57 us): 56 instructions a value; the noise of
// tokens that are cut is not read, 200 MB move in place of 263.
#include "launchers.h"
#include "packed.cuh"
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

constexpr int kBins = 512, kMaxCtas = 8;
constexpr float kBinsPerLog2 = 24.f;  // bins of 3 % in probability down to 2^-21 of the largest; finer for a flatter row
constexpr float kSlack = 1e-5f;       // rounding of the fp32 mass sums

// What the threads of a cluster bring together: the race's leader as an ordered key (score, then lowest
// index) with its logit, a mass, an index and a count, the largest and least logit.
struct alignas(16) Part {
  uint32_t score, place;  // order_of(score), ~index; 0: none
  float logit, mass;
  int first, count;
  float most, least;
  AHB_DEVICE static Part none() { return {0u, 0u, 0.f, 0.f, INT_MAX, 0, -INFINITY, INFINITY}; }
  AHB_DEVICE int index() const { return (int)~place; }
  template <int F>
  AHB_DEVICE void take(const Part& b);
};
enum { RACE = 1, MASS = 2, FIRST = 4, COUNT = 8, RANGE = 16 };

template <int F>
AHB_DEVICE void Part::take(const Part& b) {
  if (F & RACE) {
    const bool t = b.score > score || (b.score == score && b.place > place);
    logit = t ? b.logit : logit;
    score = t ? b.score : score;
    place = t ? b.place : place;
  }
  if (F & MASS) mass += b.mass;
  if (F & FIRST) first = min(first, b.first);
  if (F & COUNT) count += b.count;
  if (F & RANGE) {
    most = fmaxf(most, b.most);
    least = fminf(least, b.least);
  }
}

// monotone maps between floats (no NaN) and unsigned / signed integers
AHB_DEVICE uint32_t order_of(float x) {
  const uint32_t b = __float_as_uint(x);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
AHB_DEVICE float value_of(uint32_t o) { return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o); }

// The fields F over a warp; every lane gets the result (the same bits: the additions are symmetric).
template <int F>
AHB_DEVICE Part warp_part(Part p) {
  constexpr uint32_t all = 0xffffffffu;
  if (F & RACE) {
    const uint32_t score = __reduce_max_sync(all, p.score);
    const uint32_t place = __reduce_max_sync(all, p.score == score ? p.place : 0u);
    const uint32_t who = __ballot_sync(all, p.score == score && p.place == place);
    p.logit = __shfl_sync(all, p.logit, __ffs(who) - 1);
    p.score = score;
    p.place = place;
  }
  if (F & MASS) p.mass = warp_sum(p.mass);
  if (F & FIRST) p.first = __reduce_min_sync(all, p.first);
  if (F & COUNT) p.count = __reduce_add_sync(all, p.count);
  if (F & RANGE) {
    p.most = value_of(__reduce_max_sync(all, order_of(p.most)));
    p.least = value_of(__reduce_min_sync(all, order_of(p.least)));
  }
  return p;
}

// 16 bytes of logits
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
  // NaN becomes -inf, +inf the largest value of the type (max and min return the operand that is not NaN)
  AHB_DEVICE static void clean(uint4& r) {
    const uint32_t lo = 0xff80ff80u, hi = 0x7f7f7f7fu;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      uint32_t& w = k == 0 ? r.x : k == 1 ? r.y : k == 2 ? r.z : r.w;
      asm("max.bf16x2 %0, %0, %1;\n\tmin.bf16x2 %0, %0, %2;" : "+r"(w) : "r"(lo), "r"(hi));
    }
  }
};
template <> struct Vec<float> {
  static constexpr int N = 4;
  AHB_DEVICE static float get(const uint4& r, int j) {
    return __uint_as_float(j == 0 ? r.x : j == 1 ? r.y : j == 2 ? r.z : r.w);
  }
  AHB_DEVICE static void put(uint4& r, int j, float v) {
    (j == 0 ? r.x : j == 1 ? r.y : j == 2 ? r.z : r.w) = __float_as_uint(v);
  }
  AHB_DEVICE static void clean(uint4& r) {
#pragma unroll
    for (int j = 0; j < 4; ++j) put(r, j, fminf(fmaxf(get(r, j), -INFINITY), FLT_MAX));
  }
};
template <typename T>
AHB_DEVICE float largest(const uint4& r) {
  float m = Vec<T>::get(r, 0);
#pragma unroll
  for (int j = 1; j < Vec<T>::N; ++j) m = fmaxf(m, Vec<T>::get(r, j));
  return m;
}

// Combines the parts of all threads of the cluster; every thread gets the result.  Each warp puts its
// part into every CTA's shared memory before the barrier, and every warp combines them all after it from
// its own: one barrier, and no remote read waits.  `parts` are two sets of slots used in turn: one is
// rewritten only after the barrier that follows its last reading.
template <int F, int NT>
AHB_DEVICE Part combine(Part p, Part (*parts)[kMaxCtas * NT / 32], int turn, int rank, int ctas) {
  constexpr int NW = NT / 32;
  const int lane = threadIdx.x & 31, at = rank * NW + (threadIdx.x >> 5);
  p = warp_part<F>(p);
  if (ctas == 1) {
    if (lane == 0) parts[turn][at] = p;
    __syncthreads();
  } else {
    if (lane < ctas) {
      const uint32_t a = mapa_shared(&parts[turn][at], lane);
      if (F & (RACE | MASS))
        asm volatile("st.shared::cluster.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(a), "r"(p.score), "r"(p.place),
                     "r"(__float_as_uint(p.logit)), "r"(__float_as_uint(p.mass)) : "memory");
      if (F & (FIRST | COUNT | RANGE))
        asm volatile("st.shared::cluster.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(a + 16), "r"((uint32_t)p.first),
                     "r"((uint32_t)p.count), "r"(__float_as_uint(p.most)), "r"(__float_as_uint(p.least)) : "memory");
    }
    cluster_sync();
  }
  p = Part::none();
#pragma unroll
  for (int u = 0; u < kMaxCtas * NW / 32; ++u)
    if (u * 32 + lane < ctas * NW) p.take<F>(parts[turn][u * 32 + lane]);
  return warp_part<F>(p);
}

template <typename T, int NT>
__global__ void __launch_bounds__(NT) sample_kernel(SampleArgs p, int ctas) {
  using X = Vec<T>;
  constexpr int N = X::N, U = 16 / N;
  extern __shared__ __align__(16) uint4 keep[];
  __shared__ Part parts[2][kMaxCtas * NT / 32];
  __shared__ int hist[kBins + 32];   // then a place per lane for what is beyond the bins
  __shared__ int count_to[kBins];    // tokens in bins up to and with this one
  __shared__ float most_to[kBins];   // and the most mass they can stand for
  __shared__ float2 wsum[kBins / 32];
  __shared__ int wcnt[kBins / 32];
  __shared__ int first_out;
  const int tid = threadIdx.x, rank = (int)cluster_ctarank();
  if (ctas > 1) cluster_arrive();  // this CTA has started: the others may write into its shared memory
  const int64_t row = blockIdx.x / ctas;
  const T* l = static_cast<const T*>(p.logits) + row * p.ls;
  const float* noise = p.noise + row * p.ns;
  const float temp = p.temperature[row];
  const bool greedy = !(temp > 0.f);
  const float inv = greedy ? 1.f : fminf(fmaxf(1.f / temp, 1e-30f), 1e30f);
  const float c = inv * 1.4426950408889634f;  // logits to log2 of a probability
  const int kr = p.top_k[row], k = kr <= 0 || kr > p.V ? p.V : kr;
  const float top_p = p.top_p[row], min_p = p.min_p[row];
  const bool only_first = !(top_p > 0.f) || !(min_p <= 1.f);  // nothing else passes such a rule, NaN among them
  const bool by_rank = !greedy && k < p.V, by_mass = !greedy && top_p < 1.f;
  int turn = 0;

  // vectors [v0, v1) of the row in 16-byte lines; its first element is element `skew` of line 0
  const int skew = (int)((reinterpret_cast<uintptr_t>(l) & 15) / sizeof(T));
  const int v0 = rank * p.chunk, v1 = min(v0 + p.chunk, (skew + p.V + N - 1) / N);
  const bool q4 = (reinterpret_cast<uintptr_t>(noise - skew) & 15) == 0;  // noise in 16-byte pieces beside it
  auto fetch = [&](int v) {
    const int i = v * N - skew;
    if (i >= 0 && i + N <= p.V) return __ldg(reinterpret_cast<const uint4*>(l + i));
    uint4 r = make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int j = 0; j < N; ++j) X::put(r, j, i + j >= 0 && i + j < p.V ? to_f(l[i + j]) : -INFINITY);
    return r;
  };
  auto line = [&](int v) {
    if (p.resident) return keep[v - v0];
    uint4 r = fetch(v);
    X::clean(r);
    return r;
  };

  // pass 1: the row into shared memory, its largest and least values
  for (int b = tid; b < kBins; b += NT) hist[b] = 0;
  if (tid == 0) first_out = kBins;
  Part range = Part::none();
  auto take = [&](uint4 r) {
    range.most = fmaxf(range.most, largest<T>(r));
    const float x = X::get(r, 0);  // one value a line is enough to size the bins
    range.least = fminf(range.least, x == -INFINITY ? INFINITY : x);
  };
  if (p.resident) {  // all on their way at once; a thread reads only the lines it copied
    for (int v = v0 + tid; v < v1; v += NT) {
      const int i = v * N - skew;
      if (i >= 0 && i + N <= p.V)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(&keep[v - v0])), "l"(l + i) : "memory");
      else
        keep[v - v0] = fetch(v);
    }
    asm volatile("cp.async.commit_group;\n\tcp.async.wait_group 0;" ::: "memory");
    for (int v = v0 + tid; v < v1; v += NT) {
      uint4 r = keep[v - v0];
      X::clean(r);
      keep[v - v0] = r;
      take(r);
    }
  } else {
    for (int v = v0 + tid; v < v1; v += NT) take(line(v));
  }
  if (ctas > 1) cluster_wait();  // for the others' start, which the copy of the row has covered
  range = combine<RANGE, NT>(range, parts, turn ^= 1, rank, ctas);
  const float top = range.most;
  if (top == -INFINITY) {  // nothing can be drawn
    if (rank == 0 && tid == 0) {
      p.tokens[row] = -1;
      p.logprobs[row] = -INFINITY;
    }
    cluster_sync();  // the other CTAs may still be reading this one's part
    return;
  }
  const float bins = range.least < INFINITY ? fminf(fmaxf(kBinsPerLog2, (kBins - 1) / fmaxf((top - range.least) * c, 1e-20f)), 1e6f) : kBinsPerLog2;

  // The race over line r: tokens with y = (top - x) c bins below `limit` (bins left in, min_p) and, in
  // later rounds, ranked before (bound_l, bound_i).
  float limit = only_first ? -1.f : min_p > 0.f ? -__log2f(min_p) * bins * (1.f + 1e-6f) + 1e-30f : INFINITY;
  float bound_l = 0.f;
  int bound_i = 0;
  bool bounded = false;
  float best_s, best_l;
  int best_i;
  auto race_lines = [&](int v) {  // lines v, v + NT, ... of this thread, their noise on the way together
    uint4 r[U];
    float q[U][N];
    bool in[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int w = v + u * NT, i0 = w * N - skew;
      in[u] = w < v1;
      if (in[u]) {
        r[u] = line(w);
        in[u] = (top - largest<T>(r[u])) * c * bins < limit;
      }
      if (in[u]) {
        if (q4 && i0 >= 0 && i0 + N <= p.V) {
#pragma unroll
          for (int j = 0; j < N; j += 4) {
            const float4 f = __ldg(reinterpret_cast<const float4*>(noise + i0 + j));
            q[u][j] = f.x;
            q[u][j + 1] = f.y;
            q[u][j + 2] = f.z;
            q[u][j + 3] = f.w;
          }
        } else {
#pragma unroll
          for (int j = 0; j < N; ++j) q[u][j] = (unsigned)(i0 + j) < (unsigned)p.V ? __ldg(noise + i0 + j) : 1.f;
        }
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (!in[u]) continue;
      const int i0 = (v + u * NT) * N - skew;
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const float x = X::get(r[u], j), x2 = (top - x) * c, s = -x2 - __log2f(q[u][j]);
        bool win = (x2 * bins < limit) & (s > best_s);  // a thread's indices ascend: ties stay with the lowest
        if (bounded) win = win & ((x > bound_l) | ((x == bound_l) & (i0 + j < bound_i)));
        best_s = win ? s : best_s;
        best_i = win ? i0 + j : best_i;
        best_l = win ? x : best_l;
      }
    }
  };

  // pass 2: the mass beside one first token's, the first token's index, and the histogram where a rule
  // needs it, else the race itself
  const bool binned = by_rank || by_mass;
  Part best = Part::none();
  best_s = -INFINITY;
  auto weigh = [&](const uint4& r, int i0) {
    float e[N];
#pragma unroll
    for (int j = 0; j < N; ++j) e[j] = ex2((X::get(r, j) - top) * c);
    if (binned) {
#pragma unroll
      for (int j = 0; j < N; ++j) {  // floor(y) from the sum with 2^23, rounded towards zero
        const float y = (top - X::get(r, j)) * c * bins;
        const int at = __float_as_int(__fadd_rz(y, 8388608.f)) - 0x4b000000;
        atomicAdd(&hist[y < (float)(kBins - 1) ? at : kBins + (tid & 31)], 1);
      }
    }
    if (largest<T>(r) == top) {
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (X::get(r, j) == top) {
          e[j] = 0.f;
          ++best.count;
          best.first = min(best.first, i0 + j);
        }
    }
#pragma unroll
    for (int j = 1; j < N; ++j) e[0] += e[j];
    best.mass += e[0];
  };
  int v = v0 + tid;
  for (; v + (U - 1) * NT < v1; v += U * NT) {  // several lines' arithmetic side by side
    uint4 r[U];
#pragma unroll
    for (int u = 0; u < U; ++u) r[u] = line(v + u * NT);
#pragma unroll
    for (int u = 0; u < U; ++u) weigh(r[u], (v + u * NT) * N - skew);
  }
  for (; v < v1; v += NT) weigh(line(v), v * N - skew);
  if (!binned && !greedy)
    for (int v = v0 + tid; v < v1; v += U * NT) race_lines(v);
  auto leader = [&](Part& p) {
    if (best_s > -INFINITY) {
      p.score = order_of(best_s);
      p.place = ~(uint32_t)best_i;
      p.logit = best_l;
    }
  };
  leader(best);
  best = combine<RACE | MASS | FIRST | COUNT, NT>(best, parts, turn ^= 1, rank, ctas);
  // tokens as likely as the first count 1 each; the first itself stays out so that `rest` keeps its bits
  const int top_i = best.first;
  const float rest = best.mass + (float)(best.count - 1), z = 1.f + rest;

  if (binned) {
    // counts of all CTAs, summed up to each bin; the least and the most mass they can stand for
    constexpr int PB = NT < kBins ? kBins / NT : 1;  // consecutive bins of a thread
    int cn[PB], c_all = 0;
    float lo[PB], hi[PB], lo_all = 0.f, hi_all = 0.f;
    const int bin0 = tid * PB;
    if (bin0 < kBins) {
#pragma unroll
      for (int u = 0; u < PB; ++u) {
        int a[kMaxCtas], n = 0;
#pragma unroll
        for (int r = 0; r < kMaxCtas; ++r) {
          a[r] = 0;
          if (r < ctas) asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(a[r]) : "r"(mapa_shared(&hist[bin0 + u], r)));
        }
#pragma unroll
        for (int r = 0; r < kMaxCtas; ++r) n += a[r];
        cn[u] = c_all += n;
        lo[u] = lo_all += n * ex2(-(bin0 + u + 1) / bins);
        hi[u] = hi_all += n * ex2(-(bin0 + u) / bins);
      }
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int a = __shfl_up_sync(0xffffffffu, c_all, o);
        const float b = __shfl_up_sync(0xffffffffu, lo_all, o), d = __shfl_up_sync(0xffffffffu, hi_all, o);
        if ((tid & 31) >= o) {
          c_all += a;
          lo_all += b;
          hi_all += d;
        }
      }
      if ((tid & 31) == 31) {
        wcnt[tid >> 5] = c_all;
        wsum[tid >> 5] = make_float2(lo_all, hi_all);
      }
      // up to and without this thread's bins
      c_all -= cn[PB - 1];
      lo_all -= lo[PB - 1];
      hi_all -= hi[PB - 1];
    }
    __syncthreads();
    if (bin0 < kBins) {
      for (int w = 0; w < (tid >> 5); ++w) {
        c_all += wcnt[w];
        lo_all += wsum[w].x;
        hi_all += wsum[w].y;
      }
#pragma unroll
      for (int u = 0; u < PB; ++u) {
        count_to[bin0 + u] = c_all + cn[u];
        most_to[bin0 + u] = hi_all + hi[u];
        // everything in the bins after this one is out if the bins up to it already fill a rule
        if ((by_rank && c_all + cn[u] >= k) || (by_mass && lo_all + lo[u] >= top_p * z * (1.f + kSlack)))
          atomicMin(&first_out, bin0 + u + 1);
      }
    }
    __syncthreads();
    if (first_out < kBins - 1) limit = fminf(limit, (float)first_out);
  }

  float won_l = top;
  int won_i = top_i;
  for (bool again = binned; !greedy;) {
    if (again) {
      best = Part::none();
      best_s = -INFINITY;
      for (int v = v0 + tid; v < v1; v += U * NT) race_lines(v);
      leader(best);
      best = combine<RACE, NT>(best, parts, turn ^= 1, rank, ctas);
    }
    if (best.score == 0u || best.index() == top_i) break;
    if (binned) {
      // surely kept by the histogram's bounds, or ranked exactly
      const float y = (top - best.logit) * c * bins;
      const int bin = y < (float)(kBins - 1) ? (int)y : kBins - 1;
      if (bin == kBins - 1 || (by_rank && count_to[bin] > k) || (by_mass && most_to[bin] * (1.f + kSlack) >= top_p * z)) {
        Part before = Part::none();
        for (int v = v0 + tid; v < v1; v += NT) {
          const uint4 r = line(v);
          if (largest<T>(r) < best.logit) continue;
#pragma unroll
          for (int j = 0; j < N; ++j) {
            const float x = X::get(r, j);
            if ((x > best.logit) | ((x == best.logit) & (v * N - skew + j < best.index()))) {
              before.count += 1;
              before.mass += ex2(-(top - x) * c);
            }
          }
        }
        before = combine<MASS | COUNT, NT>(before, parts, turn ^= 1, rank, ctas);
        if ((by_rank && before.count >= k) || (by_mass && !(before.mass < top_p * z))) {
          bound_l = best.logit;
          bound_i = best.index();
          bounded = again = true;
          continue;
        }
      }
    }
    won_l = best.logit;
    won_i = best.index();
    break;
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
  // not fill the SMs and a part still has four lines for every thread.  1 x 151936 bf16: 8 CTAs 10.1 us, 4 12.9,
  // 2 18.3; 64 x 50304: 4 CTAs 16 us, 2 17.2, 8 17.8.  256 x 128256 fp32 (501 KB a row): 8 CTAs 119 us, 4 148, 2 218.
  int ctas = 1;
  while (ctas < 8 && ((lines / ctas) * 16 > 96 * 1024 || (B * ctas < 148 && lines / ctas >= 2048))) ctas *= 2;
  p.chunk = (lines + ctas - 1) / ctas;
  size_t smem = (size_t)p.chunk * 16;
  p.resident = smem <= (size_t)kMaxSlice;
  if (!p.resident) smem = 0;
  // 512 threads while all CTAs are on the SMs at once: more warps to hide each other's latency (1 x 151936: 10.1 us,
  // 256 threads 10.9).  Beyond that 256, so that more clusters overlap (256 x 128256 fp32: 119 us, 512 threads 223).
  if (B * ctas <= 2 * 148)
    return dtype == AHB_BF16 ? launch<__nv_bfloat16, 512>(p, B, ctas, smem, st) : launch<float, 512>(p, B, ctas, smem, st);
  return dtype == AHB_BF16 ? launch<__nv_bfloat16, 256>(p, B, ctas, smem, st) : launch<float, 256>(p, B, ctas, smem, st);
}
