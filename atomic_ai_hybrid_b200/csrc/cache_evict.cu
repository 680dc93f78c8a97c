// Thins a slot's cache out to `keep` rows per key head: the newest `recent` rows and then those with the largest
// mass stay, the lower row first where masses are equal.
//
// One block a (slot, head).  A row's rank is a 32-bit key (the newest ones above all others, then the mass in an
// order-preserving integer form); four passes over the keys in shared memory, eight bits each, find the key of the
// last kept row and how many rows with that key stay.  Every thread then owns a stretch of rows, and one scan over
// the threads gives the rows given up below `keep` and the kept ones behind, each in order: the i-th of
// these moves to the i-th of those.  Sources lie at or behind `keep`, targets below it, so no move waits for another, and
// only rows that have to move are touched (a cache cut back by a few rows moves a few, not all).
//
// Many heads are bound by HBM (64 conversations of 16 heads of 128 from 1024 to 512 rows: 272 MB in 65 us, 0.65 of the copy's rate:
// rows of 256 bytes, found only after the passes), few by the passes one after another (6 heads of 1152 rows: 17 us).
#include "common.cuh"
#include "launchers.h"

using namespace ahb;

namespace {

constexpr int NT = 256;

AHB_DEVICE uint32_t rank_key(float mass, int held, int64_t newest) {
  if (held >= newest) return 0xffffffffu;
  if (mass != mass) return 0u;
  const uint32_t b = __float_as_uint(mass + 0.f);  // -0 ranks as 0
  const uint32_t k = (b & 0x80000000u) ? ~b : b | 0x80000000u;
  return k == 0x007fffffu ? 0u : k;                // -inf ranks as NaN
}

// exclusive sum over the block's threads; `total` for all
AHB_DEVICE int block_sum_before(int v, int* sh, int& total) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  int s = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, s, o);
    if (lane >= o) s += u;
  }
  __syncthreads();
  if (lane == 31) sh[w] = s;
  __syncthreads();
  int before = 0;
  total = 0;
#pragma unroll
  for (int i = 0; i < NT / 32; ++i) {
    before += i < w ? sh[i] : 0;
    total += sh[i];
  }
  return before + s - v;
}

// SMEM: the keys fit into shared memory; else they are made again from the mass in every pass.
template <bool SMEM>
__global__ void __launch_bounds__(NT) evict_kernel(char* __restrict__ kc, char* __restrict__ vc, float* __restrict__ mass,
                                                   int* __restrict__ held, const int* __restrict__ lengths,
                                                   const int* __restrict__ seen, const int* __restrict__ slots, int S,
                                                   int Hk, int M, int row_bytes, int keep, int recent, int* __restrict__ lists,
                                                   int cap) {
  extern __shared__ uint32_t keys[];
  __shared__ int hist[256], sh[NT / 32], found[2];
  const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x;
  const int slot = slots ? slots[b] : b;
  if ((unsigned)slot >= (unsigned)S) return;
  const int n = lengths[slot];
  if (n <= keep || n > M) return;
  if (slots) {  // one given twice is the first one's
    bool twice = false;
    for (int i = tid; i < b; i += NT) twice |= slots[i] == slot;
    if (__syncthreads_or(twice)) return;
  }
  const int64_t newest = (int64_t)seen[slot] - recent, base = ((int64_t)slot * Hk + h) * M;
  float* ms = mass + base;
  int* hd = held + base;
  auto key = [&](int i) { return SMEM ? keys[i] : rank_key(ms[i], hd[i], newest); };
  if (SMEM)
    for (int i = tid; i < n; i += NT) keys[i] = rank_key(ms[i], hd[i], newest);
  uint32_t prefix = 0, mask = 0;
  int left = keep;
  for (int shift = 24; shift >= 0; shift -= 8) {
    hist[tid] = 0;
    __syncthreads();
    for (int i = tid; i < n; i += NT) {
      const uint32_t k = key(i);
      if ((k & mask) == prefix) atomicAdd(&hist[(k >> shift) & 255], 1);
    }
    __syncthreads();
    if (tid < 32) {  // the bin, from the top, in which the count reaches `left`
      int c[8], sum = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        c[e] = hist[255 - (8 * tid + e)];
        sum += c[e];
      }
      int upto = sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, upto, o);
        if (tid >= o) upto += u;
      }
      int before = upto - sum;
      if (before < left && left <= upto) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          if (before < left && left <= before + c[e]) {
            found[0] = 255 - (8 * tid + e);
            found[1] = left - before;
          }
          before += c[e];
        }
      }
    }
    __syncthreads();
    prefix |= (uint32_t)found[0] << shift;
    mask |= 255u << shift;
    left = found[1];
  }
  // a stretch of an odd number of rows a thread: neighbours then read different banks
  const int per = ((n + NT - 1) / NT) | 1, i0 = min(n, tid * per), i1 = min(n, i0 + per);
  int equal = 0, total;
  for (int i = i0; i < i1; ++i) equal += key(i) == prefix;
  const int equal_before = block_sum_before(equal, sh, total);
  int seen_equal = equal_before, holes = 0, movers = 0;
  for (int i = i0; i < i1; ++i) {
    const uint32_t k = key(i);
    const bool kept = k > prefix || (k == prefix && seen_equal++ < left);
    holes += !kept && i < keep;
    movers += kept && i >= keep;
  }
  int moves;
  int hole_at = block_sum_before(holes, sh, moves), mover_at = block_sum_before(movers, sh, moves);
  int* to = lists + ((int64_t)b * Hk + h) * 2 * cap;
  int* from = to + cap;
  seen_equal = equal_before;
  for (int i = i0; i < i1; ++i) {
    const uint32_t k = key(i);
    const bool kept = k > prefix || (k == prefix && seen_equal++ < left);
    if (!kept && i < keep) to[hole_at++] = i;
    if (kept && i >= keep) from[mover_at++] = i;
  }
  __syncthreads();
  for (int x = tid; x < moves; x += NT) {
    ms[to[x]] = ms[from[x]];
    hd[to[x]] = hd[from[x]];
  }
  const int chunks = row_bytes >> 4;
  uint4* kr = reinterpret_cast<uint4*>(kc) + base * chunks;
  uint4* vr = reinterpret_cast<uint4*>(vc) + base * chunks;
  constexpr int UN = 4;  // pieces of 16 bytes of k and of v that a thread has on their way
  for (int x0 = tid; x0 < moves * chunks; x0 += NT * UN) {
    uint4 k[UN], v[UN];
    int64_t dst[UN];
#pragma unroll
    for (int j = 0; j < UN; ++j) {
      const int x = x0 + j * NT;
      if (x >= moves * chunks) break;
      const int r = x / chunks, c = x - r * chunks;
      const int64_t src = (int64_t)from[r] * chunks + c;
      dst[j] = (int64_t)to[r] * chunks + c;
      k[j] = kr[src];
      v[j] = vr[src];
    }
#pragma unroll
    for (int j = 0; j < UN; ++j) {
      if (x0 + j * NT >= moves * chunks) break;
      kr[dst[j]] = k[j];
      vr[dst[j]] = v[j];
    }
  }
}

constexpr int SMEM_KEYS = 200 * 1024 / 4;

}  // namespace

int64_t ahb_cache_evict_bytes(int slots, int Hk, int M, int keep) {
  const int64_t cap = keep < M - keep ? keep : M - keep;
  return cap > 0 ? (int64_t)slots * Hk * 2 * cap * 4 : 0;
}

int ahb_cache_evict(void* kc, void* vc, float* mass, int* held, const int* lengths, const int* seen, const int* slots,
                    int n_slots, int S, int Hk, int M, int row_bytes, int keep, int recent, void* work, cudaStream_t st) {
  const int cap = keep < M - keep ? keep : M - keep;
  if (cap <= 0 || n_slots == 0) return 0;
  const dim3 grid(Hk, n_slots);
  if (M <= SMEM_KEYS) {
    const int bytes = M * 4;
    if (bytes > 40 * 1024 &&
        cudaFuncSetAttribute(evict_kernel<true>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess)
      return -1;
    evict_kernel<true><<<grid, NT, bytes, st>>>((char*)kc, (char*)vc, mass, held, lengths, seen, slots, S, Hk, M, row_bytes,
                                                keep, recent, (int*)work, cap);
  } else {
    evict_kernel<false><<<grid, NT, 0, st>>>((char*)kc, (char*)vc, mass, held, lengths, seen, slots, S, Hk, M, row_bytes,
                                             keep, recent, (int*)work, cap);
  }
  return 0;
}
